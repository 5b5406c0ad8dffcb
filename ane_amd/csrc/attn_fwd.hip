// attn_fwd.hip — causal attention, forward, and the plan of packed rows (attention.h has the mathematics).
#include "attention.h"

namespace {

// ---- forward --------------------------------------------------------------------------------------------------------------------

// Two products of 2 * hd operations for each allowed pair, three where weights are pairs.  What bounds it: at 4096 positions of 16 heads, 128
// channels, bfloat16, 133 to 142 us or 500 TFLOP/s of the two, the walk of the last block over its 64 tiles, 2.1 us each: products (34 cycles for
// 32 x 32 x 16), exponentials, the weights' second halves and the reads of LDS that feed all take turns in a wave, and two waves to a SIMD
// overlap part of it.  At 256 positions of 256 heads (50 MB) 18 us or 2.8 TB/s: start, first loads and stores of one round of workgroups.
// One sequence of 256 positions, 12 heads of 64 channels, fp32: 10.4 us.
// A panel has 64 keys (32 in fp32) and is fetched while the one before is used; four waves of 32 queries share it.
constexpr float FAR = 16777216.f;           // 2^24

// One position block.  CAREFUL: see below; else false where that is needed.  k and v have `pitch` values between rows (PanelStream), q and o S.
template <typename T, int HDB, int POS, bool CAREFUL>
__device__ __forceinline__ bool fwd_block(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale2, T *__restrict__ o, float *__restrict__ lse, int batch, int blocks, lds_char *lds_) {
    typedef Mma<T> M;
    constexpr int TEAMS = 4 / POS, STAGES = stages_for(HDB, TEAMS), QT = 32 * POS, BYTES = HDB * 32 * PANEL_ROW, STEPS = HDB * 32 / M::STEP;
    char *lds = (char *)lds_;
    int *firsts = reinterpret_cast<int *>(lds + TEAMS * STAGES * 2 * BYTES);
    const Place at = place(blocks, heads, batch, true);
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = uniform(threadIdx.x >> 6), pos = wave % POS, team = wave / POS;
    const int q0 = at.block * QT, wq = q0 + pos * 32, mine = wq + (lane & 31);
    int start = S;
    if (mine < S) start = bounds ? max(bounds[(size_t)at.b * 2 * S + mine], 0) : 0;
    const bool active = mine < S && start <= mine;
    int wfrom = 0, wfull = 0;               // keys below wfrom meet none of the wave's queries, from wfull on all that are not behind
    if (bounds) {
        wfrom = uniform(wave_min_int(active ? start : S));
        wfull = uniform(wave_max_int(active ? start : 0));
    } else if (wq >= S) wfrom = S;
    int from = wfrom;
    if constexpr (POS > 1) {
        if (lane == 0 && team == 0) firsts[pos] = wfrom;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < POS; w++) from = min(from, uniform(firsts[w]));
    }
    if (from >= S) return true;
    const int to = min(q0 + QT, S);
    const int kvh = at.h / (heads / kv_heads);
    const size_t slab = ((size_t)at.b * heads + at.h) * hd * S;
    PanelStream<T, HDB * 32, POS> ks, vs;
    ks.begin(k + ((size_t)at.b * kv_heads + kvh) * hd * pitch, pitch, hd, pos);
    vs.begin(v + ((size_t)at.b * kv_heads + kvh) * hd * pitch, pitch, hd, pos);
    const int t0 = from / M::COLS, t1 = (to - 1) / M::COLS;
    // the team's tiles are t0 + team, + TEAMS, ...; its panels lie side by side, those of one stage behind those of the other
    const char *panels = lds + team * 2 * BYTES;
    const unsigned place = lds_place(lds) + team * 2 * BYTES;
    auto load = [&](int i) __attribute__((always_inline)) {
        const int t = t0 + i * TEAMS + team;
        if (t > t1) return;
        ks.load(place + i % STAGES * (TEAMS * 2 * BYTES), t * M::COLS, from, to);
        vs.load(place + i % STAGES * (TEAMS * 2 * BYTES) + BYTES, t * M::COLS, from, to);
    };
    constexpr bool EARLY = sizeof(T) == 4 || STAGES == 2;       // (own positions need the place of the second stage)
    if (EARLY) load(0);

    typename M::Frag qf[1][STEPS];
    own_columns<T, HDB, POS, 1, STEPS>(qf, lds + (EARLY ? TEAMS * 2 * BYTES : 0), {q + slab}, S, hd, q0, S, pos);
    if (!EARLY) load(0);

    v16f acc[HDB];
    float m, l;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < HDB; d++) acc[d] = v16_zero();
    const int count = (t1 - t0) / TEAMS + 1;
    for (int i = 0; i < count; i++) {
        // what this tile needs is there; everybody is done with the tile before it
        loads_and_barrier<0, 0>();
        const char *kp = panels + i % STAGES * (TEAMS * 2 * BYTES), *vp = kp + BYTES;
        if (STAGES == 2) load(i + 1);
        const int t = t0 + i * TEAMS + team;
        const int c0 = t * M::COLS;
        if (t <= t1 && c0 <= wq + 31 && c0 + M::COLS > wfrom) {
            const bool masked = c0 + M::COLS - 1 > wq || c0 < wfull;
            const unsigned long long odd = CAREFUL && (masked || sizeof(T) == 2) ? odd_columns<T, HDB * 32>(vp) : 0;
            v16f s[M::SUBS];
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < M::SUBS; u++) {
                s[u] = over_channels<T, STEPS>(kp, u, qf[0], v16_zero());
            }
            if (masked) {
#pragma unroll
                for (int u = 0; u < M::SUBS; u++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int key = c0 + u * 32 + acc_row(r) + 4 * h;
                        s[u][r] = key <= mine && key >= start ? s[u][r] : -INFINITY;
                    }
            }
#pragma unroll
            for (int u = 0; u < M::SUBS; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[u][r]);
            mx = fmaxf(mx, lane_xor<32>(mx)) * scale2;
            if (__any(mx > m)) {        // the running maximum moves: what is there is brought to the new one
                const float to_m = fmaxf(m, mx), f = to_m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to_m);
                l *= f;
#pragma unroll
                for (int d = 0; d < HDB; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[d][r] *= f;
                m = to_m;
            }
            const float base = m == -INFINITY ? 0.f : m;
            // m is rounded and the fused product is not: their difference, up to 2^-24 m, is in every weight of a row and in its sum alike,
            // until it is beyond what an exponential holds.  From FAR on products are rounded as m is, and the largest is exactly 0 off.
            float by = scale2;
            if (__any(fabsf(base) > FAR)) {
                const bool far = fabsf(base) > FAR;
#pragma unroll
                for (int u = 0; u < M::SUBS; u++)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[u][r] = far ? s[u][r] * scale2 : s[u][r];
                by = far ? 1.f : scale2;
            }
#pragma unroll
            for (int u = 0; u < M::SUBS; u++) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], by, -base));
                    l += s[u][r];
                }
                const typename M::Packed p = M::template pack<CAREFUL>(s[u]);
                if (odd) {
                    over_positions<T, HDB, true>(acc, vp, u, p);
                    add_odd<T, HDB>(acc, vp, u, s[u], odd, [&](int c) { return c0 + c <= mine && c0 + c >= start; });
                } else {
                    over_positions<T, HDB, false>(acc, vp, u, p);
                }
            }
        }
        if (STAGES == 1) {
            __syncthreads();
            load(i + 1);
        }
    }
    __syncthreads();
    l += lane_xor<32>(l);
    if constexpr (TEAMS > 1) {          // brought to the largest of the teams' maxima, then added up
        float *ms = reinterpret_cast<float *>(lds);
        ms[(wave * 64 + lane) * 2] = m;
        ms[(wave * 64 + lane) * 2 + 1] = l;
        __syncthreads();
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < TEAMS; w++) top = fmaxf(top, ms[((w * POS + pos) * 64 + lane) * 2]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < TEAMS; w++) sum += ms[((w * POS + pos) * 64 + lane) * 2 + 1] * __builtin_amdgcn_exp2f(ms[((w * POS + pos) * 64 + lane) * 2] - base);
        const float f = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l = sum;
#pragma unroll
        for (int d = 0; d < HDB; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[d][r] *= f;
        __syncthreads();
    }
    if (!store_sums<T, HDB, POS, 1>({o + slab}, S, hd, {&acc}, {1.f / l}, wq, active, lds, pos, team, CAREFUL)) return false;
    if (active && lse && h == 0 && team == 0) lse[((size_t)at.b * heads + at.h) * S + mine] = (m + __builtin_amdgcn_logf(l)) * LN2;
    return true;
}

// An infinity or a NaN among the values of positions that the mask hides makes 0 * inf of their weights, and so does an infinity that counts
// of the second half of a bfloat16 weight.  A block that ends with a NaN is computed again, with those values taken out of the products
// (fp32: where something is masked) and added for the pairs that count.  It is a function of its own, for its
// registers not to be the kernel's.
template <typename T, int HDB, int POS>
__device__ __attribute__((noinline)) void fwd_block_again(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale2, T *__restrict__ o, float *__restrict__ lse, int batch, int blocks, lds_char *lds) {
    fwd_block<T, HDB, POS, true>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale2, o, lse, batch, blocks, lds);
}

template <typename T, int HDB, int POS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(waves_per_simd<T>(HDB, POS)))) void attn_fwd_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale2, T *__restrict__ o, float *__restrict__ lse, int batch, int blocks) {
    __shared__ __attribute__((aligned(16))) char lds[panel_bytes(HDB, POS) + 16];
    if (!fwd_block<T, HDB, POS, false>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale2, o, lse, batch, blocks, (lds_char *)lds))
        fwd_block_again<T, HDB, POS>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale2, o, lse, batch, blocks, (lds_char *)lds);
}

// ---- the plan of packed rows ----------------------------------------------------------------------------------------------------

// One thread to a position: the last offset at or below it, by bisection.
__global__ void attn_plan_kernel(int *__restrict__ bounds, const int *__restrict__ cu, int n_seqs, int S) {
    const int s = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (s >= S) return;
    const int *c = cu + (size_t)b * (n_seqs + 1);
    int lo = 0, hi = n_seqs + 1;            // offsets below lo are <= s, from hi on > s
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (c[mid] <= s) lo = mid + 1;
        else hi = mid;
    }
    const bool in = lo > 0 && lo <= n_seqs;
    bounds[(size_t)b * 2 * S + s] = in ? max(c[lo - 1], 0) : S;
    bounds[((size_t)b * 2 + 1) * S + s] = in ? min(c[lo], S) : 0;
}

template <typename T>
int attn_fwd(const char *who, T *o, float *lse, const T *q, const T *k, const T *v, const int32_t *bounds, int heads, int kv_heads, int hd,
             int S, int batch, float scale) {
    if (!mi355_ready(who)) return -1;
    if (!o || !q || !k || !v) return mi355_fail("%s: NULL pointer", who);
    if (!shape_ok(who, heads, kv_heads, hd, S, batch, scale)) return -1;
    const size_t n = (size_t)heads * batch;
    int pitch = S;
    if (!streams_directly(k, S) || !streams_directly(v, S)) {
        const size_t rows = (size_t)batch * kv_heads * hd;
        void *ws = mi355_ws(2 * packed_bytes<T>(rows, S));
        if (!ws || pack_rows(who, &k, &v, rows, S, &pitch, ws)) return -1;
    }
    return dispatch(hd, waves_for(n, S, TWO_FROM_QUERIES<T>), [&](auto hdb, auto waves) {
        constexpr int HDB = decltype(hdb)::value, W = decltype(waves)::value;
        const int blocks = (int)ceil_div(S, 32 * W);
        attn_fwd_kernel<T, HDB, W><<<(unsigned)(blocks * n), 256, 0, g_ctx.stream>>>(q, k, v, bounds, S, pitch, heads, kv_heads, hd,
                                                                                        scale * LOG2E, o, lse, batch, blocks);
        LAUNCH_OK(who);
        return 0;
    });
}

}  // namespace

MI355_API int mi355_attn_plan_dev(int32_t *bounds, const int32_t *cu, int n_seqs, int S, int batch) {
    if (!mi355_ready("attn_plan")) return -1;
    if (!bounds || !cu) return mi355_fail("attn_plan: NULL pointer");
    if (n_seqs <= 0 || S <= 0 || batch <= 0 || S > 1 << 30 || n_seqs > 1 << 30 || batch > 65535)
        return mi355_fail("attn_plan: bad shape n_seqs=%d S=%d batch=%d", n_seqs, S, batch);
    attn_plan_kernel<<<dim3((unsigned)ceil_div(S, 256), (unsigned)batch), 256, 0, g_ctx.stream>>>(bounds, cu, n_seqs, S);
    LAUNCH_OK("attn_plan");
    return 0;
}

MI355_API int mi355_attn_fwd_dev(float *o, float *lse, const float *q, const float *k, const float *v, const int32_t *bounds, int heads,
                                 int kv_heads, int hd, int S, int batch, float scale) {
    return attn_fwd<float>("attn_fwd", o, lse, q, k, v, bounds, heads, kv_heads, hd, S, batch, scale);
}
MI355_API int mi355_attn_fwd_bf16_dev(uint16_t *o, float *lse, const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                      const int32_t *bounds, int heads, int kv_heads, int hd, int S, int batch, float scale) {
    return attn_fwd<bf16_t>("attn_fwd_bf16", o, lse, q, k, v, bounds, heads, kv_heads, hd, S, batch, scale);
}
