// attn_dkv.hip — causal attention, backward: dk and dv (attention.h has the mathematics).
#include "attention.h"

namespace {

// ---- backward: dk and dv --------------------------------------------------------------------------------------------------------

// bfloat16 and up to 64 channels: what a wave keeps fits 256 registers, so two workgroups share a compute unit if their LDS lets them, which
// four teams' panels for two tiles do not.  One tile at a time and two workgroups: 1024 positions of 96 heads 115 us (all gradients) where
// one workgroup with two tiles took 133; 16 heads for 48, 69.5 and 76.5; packed rows of 997 positions, 16 for 48, 71 and 75.
template <typename T>
constexpr bool two_workgroups(int hdb) { return sizeof(T) == 2 && hdb == 2; }
template <typename T>
constexpr int dkv_stages(int hdb, int teams) { return two_workgroups<T>(hdb) && teams == 4 ? 1 : stages_for(hdb, teams); }

// Four products of 2 * hd operations for each allowed pair, six where weights and score gradients are pairs, and two accumulators: one wave to
// a SIMD beyond 64 channels of bfloat16.  bfloat16, 4096 positions of 16 heads over 8, 128 channels: 277 us in a kernel trace (262 to 298; both
// kernels are slower there than in the 386 us that an untraced call takes), 500 TFLOP/s of the four; what a tile does comes one after the other
// in that wave.  fp32, 256 positions of 128 heads over 64: 68 us, 64 TFLOP/s of 150 in two rounds of workgroups, each 37 us: 23 the walk, 11
// own positions, first loads, the teams' sums and stores.
// One position block; CAREFUL as in the forward pass.  q and d_o have `pitch` values between rows (PanelStream), the others S.
template <typename T, int HDB, int POS, bool CAREFUL>
__device__ __forceinline__ bool dkv_block(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale, const T *__restrict__ d_o, const float *__restrict__ lse, const float *__restrict__ delta, T *__restrict__ dk, T *__restrict__ dv,
    int batch, int blocks, lds_char *lds_) {
    typedef Mma<T> M;
    constexpr int TEAMS = 4 / POS, STAGES = dkv_stages<T>(HDB, TEAMS), KT = 32 * POS, BYTES = HDB * 32 * PANEL_ROW, STEPS = HDB * 32 / M::STEP;
    char *lds = (char *)lds_;
    typedef float Rows[TEAMS][2][M::COLS];          // [team][lse * log2(e), delta][query], of a stage
    Rows *rows = reinterpret_cast<Rows *>(lds + TEAMS * STAGES * 2 * BYTES);
    int *lasts = reinterpret_cast<int *>(rows + STAGES);
    const Place at = place(blocks, kv_heads, batch, false);
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = uniform(threadIdx.x >> 6), pos = wave % POS, team = wave / POS;
    const int k0 = at.block * KT, wk = k0 + pos * 32, mine = wk + (lane & 31);
    int end = 0;
    if (mine < S) end = bounds ? min(bounds[((size_t)at.b * 2 + 1) * S + mine], S) : S;
    const bool active = mine < S && end > mine;
    int wto = S, wfull = S;                 // queries from wto on meet none of the wave's keys, below wfull all that are not before
    if (bounds) {
        wto = uniform(wave_max_int(active ? end : 0));
        wfull = uniform(wave_min_int(active ? end : S));
    } else if (wk >= S) wto = 0;
    int to = wto;
    if constexpr (POS > 1) {
        if (lane == 0 && team == 0) lasts[pos] = wto;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < POS; w++) to = max(to, uniform(lasts[w]));
    }
    if (to <= k0) return true;
    const int group = heads / kv_heads;
    const size_t slab = ((size_t)at.b * kv_heads + at.h) * hd * S;
    const size_t head0 = (size_t)at.b * heads + (size_t)at.h * group;

    typename M::Frag own[2][STEPS];         // of k and v
    static_assert(sizeof(T) == 4 || 2 * own_panels<T, POS>() <= STAGES * TEAMS * 2, "they fit the panels' places");
    own_columns<T, HDB, POS, 2, STEPS>(own, lds, {k + slab, v + slab}, S, hd, k0, S, pos);
    const float scale2 = scale * LOG2E;
    // the query at this lane's position, if this key is its only one (attn_bwd.hip)
    const int first = mine < S && (bounds ? max(bounds[(size_t)at.b * 2 * S + mine], 0) == mine : mine == 0) ? mine : -1;

    v16f ak[HDB], av[HDB];
    const int t0 = k0 / M::COLS, tiles = (to - 1) / M::COLS - t0 + 1, steps = tiles * group;
    const int count = (steps + TEAMS - 1) / TEAMS;
    const char *panels = lds + team * 2 * BYTES;
    const unsigned place = lds_place(lds) + team * 2 * BYTES;
#pragma unroll
    for (int d = 0; d < HDB; d++) ak[d] = v16_zero(), av[d] = v16_zero();
    if constexpr (!two_workgroups<T>(HDB)) in_agprs(ak), in_agprs(av);
    PanelStream<T, HDB * 32, POS> qs, gs;
    float lr[2] = {0.f, 0.f};
    // The walk goes over a group's heads one after the other, each over its queries; the team takes every TEAMS-th of all tiles.  What of
    // lse and delta a thread loads goes to LDS when the tile before is done.
    int head = team / tiles, tile = team % tiles;           // of the load to come
    auto load = [&](int stage) __attribute__((always_inline)) {
        if (head >= group) return;
        const size_t hh = head0 + head;
        const int t = t0 + tile, at_q = t * M::COLS + lane;
        if (pos == 0) {
            lr[0] = lane < M::COLS && at_q < S ? lse[hh * S + at_q] * LOG2E : 0.f;
            lr[1] = lane < M::COLS && at_q < S ? delta[hh * S + at_q] : 0.f;
        }
        const unsigned p = place + stage * (TEAMS * 2 * BYTES);
        qs.begin(q + hh * hd * pitch, pitch, hd, pos);
        gs.begin(d_o + hh * hd * pitch, pitch, hd, pos);
        qs.load(p, t * M::COLS, k0, to);
        gs.load(p + BYTES, t * M::COLS, k0, to);
    };
    auto store_rows = [&](int stage) {
        if (pos == 0 && lane < M::COLS) rows[stage][team][0][lane] = lr[0], rows[stage][team][1][lane] = lr[1];
    };
    load(0);
    store_rows(0);
    for (int i = 0; i < count; i++) {
        // what this tile needs is there; everybody is done with the tile before it
        loads_and_barrier<0, 0>();
        if constexpr (!two_workgroups<T>(HDB)) in_agprs(ak), in_agprs(av);
        const char *qp = panels + i % STAGES * (TEAMS * 2 * BYTES), *gp = qp + BYTES;
        const float *ls_row = rows[i % STAGES][team][0], *dl_row = rows[i % STAGES][team][1];
        const int c0 = head < group ? (t0 + tile) * M::COLS : to;
        tile += TEAMS;
        while (tile >= tiles && head < group) tile -= tiles, head++;
        if (STAGES == 2) load((i + 1) % STAGES);
        if (c0 + M::COLS > wk && c0 < wto) {
            const bool masked = c0 < wk + 31 || c0 + M::COLS > wfull;
            const unsigned long long odd = CAREFUL && (masked || sizeof(T) == 2) ? odd_columns<T, HDB * 32>(qp) | odd_columns<T, HDB * 32>(gp) : 0;
#pragma unroll
            for (int u = 0; u < M::SUBS; u++) {
                v16f s = over_channels<T, STEPS>(qp, u, own[0], v16_zero()), g = over_channels<T, STEPS>(gp, u, own[1], v16_zero());
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const v4f ls = *reinterpret_cast<const v4f *>(ls_row + u * 32 + 8 * j + 4 * h);
                    const v4f dl = *reinterpret_cast<const v4f *>(dl_row + u * 32 + 8 * j + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = 4 * j + e;
                        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale2, -ls[e]));
                        g[r] = s[r] * (g[r] - dl[e]);
                    }
                }
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int qq = c0 + u * 32 + acc_row(r) + 4 * h;
                        const bool ok = qq >= mine && qq < end;
                        s[r] = ok ? s[r] : 0.f;
                        g[r] = ok ? qq == first ? g[r] * 0.f : g[r] : 0.f;
                    }
                }
                const typename M::Packed ps = M::template pack<CAREFUL>(s), pg = M::template pack<CAREFUL>(g);
                if (odd) {
                    over_positions<T, HDB, true>(av, gp, u, ps);
                    over_positions<T, HDB, true>(ak, qp, u, pg);
                    auto ok = [&](int c) { return c0 + c >= mine && c0 + c < end; };
                    add_odd<T, HDB>(av, gp, u, s, odd, ok);
                    add_odd<T, HDB>(ak, qp, u, g, odd, ok);
                } else {
                    over_positions<T, HDB, false>(av, gp, u, ps);
                    over_positions<T, HDB, false>(ak, qp, u, pg);
                }
            }
        }
        if (STAGES == 1) {
            __syncthreads();
            load(0);
        }
        store_rows((i + 1) % STAGES);
    }
    __syncthreads();
    if (!store_sums<T, HDB, POS, 2>({dk + slab, dv + slab}, S, hd, {&ak, &av}, {scale, 1.f}, wk, active, lds, pos, team, CAREFUL)) return false;
    return true;
}
template <typename T, int HDB, int POS>
__device__ __attribute__((noinline)) void dkv_block_again(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale, const T *__restrict__ d_o, const float *__restrict__ lse, const float *__restrict__ delta, T *__restrict__ dk, T *__restrict__ dv,
    int batch, int blocks, lds_char *lds) {
    dkv_block<T, HDB, POS, true>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale, d_o, lse, delta, dk, dv, batch, blocks, lds);
}

template <typename T, int HDB, int POS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(two_workgroups<T>(HDB) ? 2 : 1))) void attn_dkv_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ bounds, int S, int pitch, int heads, int kv_heads,
    int hd, float scale, const T *__restrict__ d_o, const float *__restrict__ lse, const float *__restrict__ delta, T *__restrict__ dk, T *__restrict__ dv,
    int batch, int blocks) {
    constexpr int TEAMS = 4 / POS, STAGES = dkv_stages<T>(HDB, TEAMS), ROWS = STAGES * TEAMS * 2 * Mma<T>::COLS * 4;
    __shared__ __attribute__((aligned(16))) char lds[TEAMS * STAGES * 2 * HDB * 32 * PANEL_ROW + ROWS + 16];
    if (!dkv_block<T, HDB, POS, false>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale, d_o, lse, delta, dk, dv, batch, blocks, (lds_char *)lds))
        dkv_block_again<T, HDB, POS>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale, d_o, lse, delta, dk, dv, batch, blocks, (lds_char *)lds);
}

template <typename T>
int launch_dkv(const char *who, T *dk, T *dv, const T *d_o, const T *q, const T *k, const T *v, const float *lse, const float *delta,
               const int32_t *bounds, int heads, int kv_heads, int hd, int S, int pitch, int batch, float scale) {
    const size_t nk = (size_t)kv_heads * batch;
    return dispatch(hd, waves_for(nk, S, TWO_FROM), [&](auto hdb, auto waves) {
        constexpr int HDB = decltype(hdb)::value, W = decltype(waves)::value;
        const int blocks = (int)ceil_div(S, 32 * W);
        attn_dkv_kernel<T, HDB, W><<<(unsigned)(blocks * nk), 256, 0, g_ctx.stream>>>(q, k, v, bounds, S, pitch, heads, kv_heads, hd, scale, d_o,
                                                                                         lse, delta, dk, dv, batch, blocks);
        LAUNCH_OK(who);
        return 0;
    });
}


}  // namespace

int mi355_attn_dkv(const char *who, float *dk, float *dv, const float *d_o, const float *q, const float *k, const float *v, const float *lse,
                   const float *delta, const int32_t *bounds, int heads, int kv_heads, int hd, int S, int pitch, int batch, float scale) {
    return launch_dkv<float>(who, dk, dv, d_o, q, k, v, lse, delta, bounds, heads, kv_heads, hd, S, pitch, batch, scale);
}
int mi355_attn_dkv(const char *who, bf16_t *dk, bf16_t *dv, const bf16_t *d_o, const bf16_t *q, const bf16_t *k, const bf16_t *v,
                   const float *lse, const float *delta, const int32_t *bounds, int heads, int kv_heads, int hd, int S, int pitch, int batch, float scale) {
    return launch_dkv<bf16_t>(who, dk, dv, d_o, q, k, v, lse, delta, bounds, heads, kv_heads, hd, S, pitch, batch, scale);
}
