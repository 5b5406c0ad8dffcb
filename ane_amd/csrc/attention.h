// attention.h — causal attention over whole prompts, forward and backward: q [batch][heads*hd][S], k and v [batch][kv_heads*hd][S].
// Not among the reference's CPU ops (its attention runs in MIL kernels, training/training_dynamic/mil_dynamic.h); it stands between
// mi355_qknorm_rope_fwd_dev / mi355_rope_dev and the output projection, and its gradients go on into mi355_qknorm_rope_bwd_dev.
//
//   p[s][t] = exp(scale q_s.k_t - lse_s) for start_s <= t <= s,  o_s = sum_t p[s][t] v_t,  lse_s = log sum_t exp(scale q_s.k_t)
//   delta_s = do_s.o_s,  ds[s][t] = p[s][t] (do_s.v_t - delta_s)
//   dv_t = sum_s p[s][t] do_s,  dq_s = scale sum_t ds[s][t] k_t,  dk_t = scale sum_s ds[s][t] q_s   (dk, dv: over a group's heads)
//
// Positions are the contiguous axis, so a 32 x 32 product of scores is laid out with one position to a lane and the positions of the
// other side in its registers: running maxima and sums are a lane's own (two lanes share a position), the accumulators of o, dq, dk and
// dv have the same position in the lane, and scores go into the second product as they lie (mma.h).  The forward pass and dq have a
// query to the lane and walk over the keys, dk and dv a key to the lane and walk over the queries: seven products in place of five, and
// no gradient is added up by atomics.
#pragma once
#include "mma.h"

#include <math.h>

// dk and dv from lse and delta (attn_dkv.hip): the second launch of the backward entry points, which have checked the arguments.
int mi355_attn_dkv(const char *who, float *dk, float *dv, const float *d_o, const float *q, const float *k, const float *v, const float *lse,
                   const float *delta, const int32_t *bounds, int heads, int kv_heads, int hd, int S, int batch, float scale);
int mi355_attn_dkv(const char *who, bf16_t *dk, bf16_t *dv, const bf16_t *d_o, const bf16_t *q, const bf16_t *k, const bf16_t *v,
                   const float *lse, const float *delta, const int32_t *bounds, int heads, int kv_heads, int hd, int S, int batch, float scale);

namespace {

constexpr float LOG2E = 1.44269502162933349609375f, LN2 = 0.693147182464599609375f;

__device__ __forceinline__ int wave_min_int(int v) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) v = min(v, __shfl_xor(v, m, 64));
    return v;
}
__device__ __forceinline__ int wave_max_int(int v) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) v = max(v, __shfl_xor(v, m, 64));
    return v;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Columns of a panel that hold an infinity or a NaN in one of their ROWS rows (the same mask in every lane).
template <typename T, int ROWS>
__device__ unsigned long long odd_columns(const char *panel) {
    bool odd = false;
    const int col = threadIdx.x & (Mma<T>::COLS - 1);
#pragma unroll 1
    for (int row = 0; row < ROWS; row++) odd |= !is_finite(Mma<T>::value(panel, row, col));
    return __ballot(odd) & (Mma<T>::COLS == 64 ? ~0ull : (1ull << (Mma<T>::COLS & 63)) - 1);
}
// acc += w * panel over the infinities and NaNs of the panel's 32 columns `sub`, for the pairs that the mask leaves: what a product that
// takes them as zeros leaves out.  weights: a product's registers, the panel's columns in its rows.
template <typename T, int HDB, typename Allowed>
__device__ void add_odd(v16f (&acc)[HDB], const char *panel, int sub, const v16f &weights, unsigned long long odd, Allowed allowed) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll 1
    for (int c = 0; c < 32; c++) {
        if (!(odd >> (sub * 32 + c) & 1)) continue;
        float w = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r++)
            if (acc_row(r) == (c & ~4)) w = weights[r];
        w = __shfl(w, (lane & 31) + ((c >> 2 & 1) << 5), 64);
        if (!allowed(sub * 32 + c)) continue;
#pragma unroll
        for (int d = 0; d < HDB; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float x = Mma<T>::value(panel, d * 32 + acc_row(r) + 4 * h, sub * 32 + c);
                if (!is_finite(x)) acc[d][r] += w * x;
            }
    }
}

template <int HDB>
__device__ __forceinline__ bool has_nan(const v16f (&acc)[HDB]) {
    float s = 0.f;      // (infinities of both signs count too: that costs time, nothing else)
#pragma unroll
    for (int d = 0; d < HDB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) s += acc[d][r];
    return s != s;
}

// acc[channel][position] * f to rows of a tensor; `pos` is the lane's own column of it
template <typename T, int HDB>
__device__ __forceinline__ void store_columns(T *dst, size_t pitch, int hd, const v16f (&acc)[HDB], float f) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int d = 0; d < HDB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int row = d * 32 + acc_row(r) + 4 * h;
            if (row < hd) dst[(size_t)row * pitch] = Mma<T>::narrow(acc[d][r] * f);
        }
}

// The 32 columns of this wave, of 32 * WAVES from col0 on, as fragments of a product over the channels.  Needs as many panels of LDS as
// the columns fill; ends with a barrier.
template <typename T, int HDB, int WAVES, int STEPS>
__device__ __forceinline__ void own_columns(typename Mma<T>::Frag (&f)[STEPS], char *lds, const T *src, size_t pitch, int hd, int col0, int S) {
    typedef Mma<T> M;
    constexpr int PANELS = (32 * WAVES + M::COLS - 1) / M::COLS, BYTES = HDB * 32 * PANEL_ROW;
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int p = 0; p < PANELS; p++) {
        PanelLoad<T, HDB * 32, WAVES * 64> ld;
        ld.load(src, pitch, hd, col0 + p * M::COLS, 0, S);
        ld.store(lds + p * BYTES);
    }
    __syncthreads();
    const char *panel = lds + (wave * 32 / M::COLS) * BYTES;
#pragma unroll
    for (int s = 0; s < STEPS; s++) f[s] = M::columns(panel, wave * 32 % M::COLS / 32, s);
    __syncthreads();
}

// Which position block of which head a workgroup has: blocks in the given order, heads of one KV group on one XCD where the heads deal
// out evenly (their L2 then holds the group's keys and values once).
struct Place { int block, b, h; };
__device__ __forceinline__ Place place(int blocks, int heads, int batch, bool last_first) {
    const int n = heads * batch, bid = (int)blockIdx.x;
    Place p;
    p.block = bid / n;
    if (last_first) p.block = blocks - 1 - p.block;
    int i = bid % n;
    if ((n & 7) == 0) i = xcd_remap(i, n);
    p.b = i / heads;
    p.h = i % heads;
    return p;
}

// ---- host side ------------------------------------------------------------------------------------------------------------------

bool shape_ok(const char *who, int heads, int kv_heads, int hd, int S, int batch, float scale) {
    if (heads <= 0 || kv_heads <= 0 || hd <= 0 || S <= 0 || batch <= 0) {
        mi355_fail("%s: bad shape heads=%d kv_heads=%d hd=%d S=%d batch=%d", who, heads, kv_heads, hd, S, batch);
        return false;
    }
    if (heads % kv_heads) {
        mi355_fail("%s: heads=%d is no multiple of kv_heads=%d", who, heads, kv_heads);
        return false;
    }
    if (hd > 128) {
        mi355_fail("%s: head size %d (at most 128)", who, hd);
        return false;
    }
    if (!(scale > 0.f) || !isfinite(scale)) {
        mi355_fail("%s: scale must be positive and finite", who);
        return false;
    }
    // what a launch can number (2^32 threads, two waves to 64 positions), and 32-bit positions
    if (S > 1 << 30 || (double)heads * batch * ceil_div(S, 64) > (double)((1 << 25) - 1)) {
        mi355_fail("%s: heads * batch * ceil(S / 64) = %.0f (at most 2^25 - 1), S = %d (at most 2^30)", who, (double)heads * batch * ceil_div(S, 64), S);
        return false;
    }
    return true;
}

// Waves (32 positions each) to a workgroup: four share the panels that they read, unless that leaves compute units without work.
int waves_for(size_t heads_batch, int S) {
    return ceil_div(S, 128) * heads_batch >= (size_t)g_ctx.num_cu ? 4 : 2;
}

template <typename F>
int dispatch(int hd, int waves, F go) {
    auto by_waves = [&](auto hdb) {
        if (waves == 4) return go(hdb, std::integral_constant<int, 4>());
        return go(hdb, std::integral_constant<int, 2>());
    };
    if (hd <= 64) return by_waves(std::integral_constant<int, 2>());
    if (hd <= 96) return by_waves(std::integral_constant<int, 3>());
    return by_waves(std::integral_constant<int, 4>());
}

}  // namespace
