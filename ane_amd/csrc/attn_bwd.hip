// attn_bwd.hip — causal attention, backward: dq and delta, then the entry points (attention.h has the mathematics, attn_dkv.hip dk and dv).
#include "attention.h"

namespace {

// ---- backward: dq and delta -----------------------------------------------------------------------------------------------------

// Three products of 2 * hd operations for each allowed pair, four where score gradients are pairs.  bfloat16, 4096 positions of 16 heads, 128
// channels: 173 us in a kernel trace (167 to 184), 600 TFLOP/s of the three, bound like the forward pass by a tile's products, exponentials
// and reads of LDS in turn.  fp32, 256 positions of 128 heads, 128 channels: 53 us (61 TFLOP/s of 150: two rounds of workgroups, each 128 KB
// of LDS, whose start and end nothing overlaps).
// One position block; CAREFUL as in the forward pass.  k and v have `pitch` values between rows (PanelStream), the others S.
template <typename T, int HDB, int POS, bool CAREFUL>
__device__ __forceinline__ bool dq_block(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale, const T *__restrict__ o, const T *__restrict__ d_o, const float *__restrict__ lse, T *__restrict__ dq, float *__restrict__ delta,
    int batch, int blocks, lds_char *lds_) {
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
    int wfrom = 0, wfull = 0;
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
    const size_t slab = ((size_t)at.b * heads + at.h) * hd * S, row = ((size_t)at.b * heads + at.h) * S;
    const int t0 = from / M::COLS, t1 = (to - 1) / M::COLS;

    PanelStream<T, HDB * 32, POS> ks, vs;
    ks.begin(k + ((size_t)at.b * kv_heads + kvh) * hd * pitch, pitch, hd, pos);
    vs.begin(v + ((size_t)at.b * kv_heads + kvh) * hd * pitch, pitch, hd, pos);
    // the team's tiles are t0 + team, + TEAMS, ...; its panels lie side by side, those of one stage behind those of the other
    const char *panels = lds + team * 2 * BYTES;
    const unsigned place = lds_place(lds) + team * 2 * BYTES;
    auto load = [&](int i) __attribute__((always_inline)) {
        const int t = t0 + i * TEAMS + team;
        if (t > t1) return;
        ks.load(place + i % STAGES * (TEAMS * 2 * BYTES), t * M::COLS, from, to);
        vs.load(place + i % STAGES * (TEAMS * 2 * BYTES) + BYTES, t * M::COLS, from, to);
    };
    // Own positions: those of fp32 come without LDS and behind the first panels; those of bfloat16 by way of the panels' places, all three
    // by the second stage's where that is large enough, else two before the first panels and q by the second stage's.
    constexpr int OWN = own_panels<T, POS>();
    constexpr bool DIRECT = sizeof(T) == 4, ALL = STAGES == 2 && 3 * OWN <= TEAMS * 2;
    char *second = lds + (STAGES == 2 ? TEAMS * 2 * BYTES : 0);
    typename M::Frag own[3][STEPS];         // of d_o, o and q
    if constexpr (DIRECT || ALL) {
        load(0);
        own_columns<T, HDB, POS, 3, STEPS>(own, second, {d_o + slab, o + slab, q + slab}, S, hd, q0, S, pos);
    } else {
        static_assert(2 * OWN <= STAGES * TEAMS * 2 && OWN <= TEAMS * 2, "they fit the panels' places");
        typename M::Frag two[2][STEPS], one[1][STEPS];
        own_columns<T, HDB, POS, 2, STEPS>(two, lds, {d_o + slab, o + slab}, S, hd, q0, S, pos);
        if (STAGES == 2) load(0);
        own_columns<T, HDB, POS, 1, STEPS>(one, second, {q + slab}, S, hd, q0, S, pos);
        if (STAGES == 1) load(0);
#pragma unroll
        for (int s = 0; s < STEPS; s++) own[0][s] = two[0][s], own[1][s] = two[1][s], own[2][s] = one[0][s];
    }
    // delta from the fragments: two lanes share a query, each has half of the channels
    float dlt = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; i++) dlt = M::dot(own[1][i], own[0][i], dlt);
    dlt += lane_xor<32>(dlt);
    const float lse2 = active ? lse[row + mine] * LOG2E : 0.f;
    if (active && h == 0 && team == 0) delta[row + mine] = dlt;
    const float scale2 = scale * LOG2E;
    // A query with a single key has p = 1 whatever its score: do.v and delta are the same sum in two orders, and what is left of their
    // difference by rounding is taken out.  (A product, for NaNs to stay.)
    const float only = start == mine ? 0.f : 1.f;

    v16f acc[HDB];
#pragma unroll
    for (int d = 0; d < HDB; d++) acc[d] = v16_zero();
    if constexpr (waves_per_simd<T>(HDB, POS) == 1) in_agprs(acc);
    const int count = (t1 - t0) / TEAMS + 1;
    for (int i = 0; i < count; i++) {
        // what this tile needs is there; everybody is done with the tile before it
        loads_and_barrier<0, 0>();
        if constexpr (waves_per_simd<T>(HDB, POS) == 1) in_agprs(acc);
        const char *kp = panels + i % STAGES * (TEAMS * 2 * BYTES), *vp = kp + BYTES;
        if (STAGES == 2) load(i + 1);
        const int t = t0 + i * TEAMS + team;
        const int c0 = t * M::COLS;
        if (t <= t1 && c0 <= wq + 31 && c0 + M::COLS > wfrom) {
            const bool masked = c0 + M::COLS - 1 > wq || c0 < wfull;
            const unsigned long long odd = CAREFUL && (masked || sizeof(T) == 2) ? odd_columns<T, HDB * 32>(kp) : 0;
#pragma unroll
            for (int u = 0; u < M::SUBS; u++) {
                v16f s = over_channels<T, STEPS>(kp, u, own[2], v16_zero()), g = over_channels<T, STEPS>(vp, u, own[0], v16_zero());
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale2, -lse2));
                    s[r] = p * (g[r] - dlt);
                }
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int key = c0 + u * 32 + acc_row(r) + 4 * h;
                        s[r] = key <= mine && key >= start ? s[r] * only : 0.f;
                    }
                }
                const typename M::Packed p = M::template pack<CAREFUL>(s);
                if (odd) {
                    over_positions<T, HDB, true>(acc, kp, u, p);
                    add_odd<T, HDB>(acc, kp, u, s, odd, [&](int c) { return c0 + c <= mine && c0 + c >= start; });
                } else {
                    over_positions<T, HDB, false>(acc, kp, u, p);
                }
            }
        }
        if (STAGES == 1) {
            __syncthreads();
            load(i + 1);
        }
    }
    __syncthreads();
    if (!store_sums<T, HDB, POS, 1>({dq + slab}, S, hd, {&acc}, {scale}, wq, active, lds, pos, team, CAREFUL)) return false;
    return true;
}
template <typename T, int HDB, int POS>
__device__ __attribute__((noinline)) void dq_block_again(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale, const T *__restrict__ o, const T *__restrict__ d_o, const float *__restrict__ lse, T *__restrict__ dq, float *__restrict__ delta,
    int batch, int blocks, lds_char *lds) {
    dq_block<T, HDB, POS, true>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale, o, d_o, lse, dq, delta, batch, blocks, lds);
}

template <typename T, int HDB, int POS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(waves_per_simd<T>(HDB, POS)))) void attn_dq_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale, const T *__restrict__ o, const T *__restrict__ d_o, const float *__restrict__ lse, T *__restrict__ dq, float *__restrict__ delta,
    int batch, int blocks) {
    __shared__ __attribute__((aligned(16))) char lds[panel_bytes(HDB, POS) + 16];
    if (!dq_block<T, HDB, POS, false>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale, o, d_o, lse, dq, delta, batch, blocks, (lds_char *)lds))
        dq_block_again<T, HDB, POS>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale, o, d_o, lse, dq, delta, batch, blocks, (lds_char *)lds);
}

template <typename T>
int attn_bwd(const char *who, T *dq, T *dk, T *dv, const T *d_o, const T *q, const T *k, const T *v, const T *o, const float *lse,
             const int32_t *bounds, int heads, int kv_heads, int hd, int S, int batch, float scale) {
    if (!mi355_ready(who)) return -1;
    if (!dq || !dk || !dv || !d_o || !q || !k || !v || !o || !lse) return mi355_fail("%s: NULL pointer", who);
    if (!shape_ok(who, heads, kv_heads, hd, S, batch, scale)) return -1;
    const size_t n = (size_t)heads * batch;
    // Workspace: delta; the streamed tensors (k and v here, q and d_o in the launch for dk and dv) where their rows are no whole chunks, at
    // the same place one after the other.
    const size_t delta_bytes = (n * S * sizeof(float) + 255) & ~(size_t)255;
    const bool pack_kv = !streams_directly(k, S) || !streams_directly(v, S), pack_q = !streams_directly(q, S) || !streams_directly(d_o, S);
    const size_t packed = 2 * (packed_bytes<T>((size_t)batch * (pack_q ? heads : kv_heads) * hd, S));
    char *ws = (char *)mi355_ws(delta_bytes + (pack_q || pack_kv ? packed : 0));
    if (!ws) return -1;
    float *delta = (float *)ws;
    int pitch = S;
    const T *ks = k, *vs = v;
    if (pack_kv && pack_rows(who, &ks, &vs, (size_t)batch * kv_heads * hd, S, &pitch, ws + delta_bytes)) return -1;
    int rc = dispatch(hd, waves_for(n, S, TWO_FROM_QUERIES<T>), [&](auto hdb, auto waves) {
        constexpr int HDB = decltype(hdb)::value, W = decltype(waves)::value;
        const int blocks = (int)ceil_div(S, 32 * W);
        attn_dq_kernel<T, HDB, W><<<(unsigned)(blocks * n), 256, 0, g_ctx.stream>>>(q, ks, vs, bounds, S, pitch, heads, kv_heads, hd,
                                                                                       scale, o, d_o, lse, dq, delta, batch, blocks);
        LAUNCH_OK(who);
        return 0;
    });
    if (rc) return rc;
    pitch = S;
    const T *qs = q, *gs = d_o;
    if (pack_q && pack_rows(who, &qs, &gs, n * hd, S, &pitch, ws + delta_bytes)) return -1;
    return mi355_attn_dkv(who, dk, dv, gs, qs, k, v, lse, delta, bounds, heads, kv_heads, hd, S, pitch, batch, scale);
}

}  // namespace

MI355_API int mi355_attn_bwd_dev(float *dq, float *dk, float *dv, const float *d_o, const float *q, const float *k, const float *v,
                                 const float *o, const float *lse, const int32_t *bounds, int heads, int kv_heads, int hd, int S,
                                 int batch, float scale) {
    return attn_bwd<float>("attn_bwd", dq, dk, dv, d_o, q, k, v, o, lse, bounds, heads, kv_heads, hd, S, batch, scale);
}
MI355_API int mi355_attn_bwd_bf16_dev(uint16_t *dq, uint16_t *dk, uint16_t *dv, const uint16_t *d_o, const uint16_t *q, const uint16_t *k,
                                      const uint16_t *v, const uint16_t *o, const float *lse, const int32_t *bounds, int heads,
                                      int kv_heads, int hd, int S, int batch, float scale) {
    return attn_bwd<bf16_t>("attn_bwd_bf16", dq, dk, dv, d_o, q, k, v, o, lse, bounds, heads, kv_heads, hd, S, batch, scale);
}
