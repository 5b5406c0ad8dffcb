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
//
// In bfloat16 p and ds go into the second product as pairs of bfloat16 values that are off by 2^-15 of them (mma.h): the matrix cores take
// no other operand beside bfloat16 values, and one value each, off by 2^-8, is as much again as the rounding of the results.  The second
// half costs a product more for each of those: 4096 positions of 16 heads, 128 channels, forward 107 -> 133 us, all gradients 311 -> 391;
// 256 positions of 256 heads, forward 17.5 -> 19.7.  Scores, statistics, sums, delta and all accumulators are fp32.  delta is of o as it is
// stored, and has the rounding of that in it, which shows where keys are few: dq and dk against 64 bits 0.0032 off for sequences of two
// positions, 0.0024 of eight, 0.0020 of 32, 0.0018 of 256, 0.0017 being the rounding of the results.  (From the weights themselves it would
// take a walk of its own before dq's.)
#pragma once
#include "mma.h"

#include <math.h>

// dk and dv from lse and delta (attn_dkv.hip): the second launch of the backward entry points, which have checked the arguments.
int mi355_attn_dkv(const char *who, float *dk, float *dv, const float *d_o, const float *q, const float *k, const float *v, const float *lse,
                   const float *delta, const int32_t *bounds, int heads, int kv_heads, int hd, int S, int pitch, int batch, float scale);
int mi355_attn_dkv(const char *who, bf16_t *dk, bf16_t *dv, const bf16_t *d_o, const bf16_t *q, const bf16_t *k, const bf16_t *v,
                   const float *lse, const float *delta, const int32_t *bounds, int heads, int kv_heads, int hd, int S, int pitch, int batch, float scale);

namespace {

constexpr float LOG2E = 1.44269502162933349609375f, LN2 = 0.693147182464599609375f;

typedef __attribute__((address_space(3))) char lds_char;

// Panels for two tiles of each team, or for one where two would not fit the 160 KB of a compute unit beside what else there is; their bytes;
// and how many waves to a SIMD they leave room for.
constexpr int stages_for(int hdb, int teams) { return 2 * 2 * teams * hdb * 32 * PANEL_ROW <= 128 * 1024 ? 2 : 1; }
constexpr int panel_bytes(int hdb, int pos) { return 4 / pos * stages_for(hdb, 4 / pos) * 2 * hdb * 32 * PANEL_ROW; }
template <typename T>
constexpr int waves_per_simd(int hdb, int pos) { return panel_bytes(hdb, pos) <= 72 * 1024 && (sizeof(T) == 2 || hdb == 2) ? 2 : 1; }

// Keeps accumulators where a kernel of one wave to a SIMD has its products write them.  Without it each tile copied them out of those
// registers and back: dkv of bf16, 128 channels: 993 vector instructions a tile for 736 with it.
template <int HDB>
__device__ __forceinline__ void in_agprs(v16f (&acc)[HDB]) {
#pragma unroll
    for (int d = 0; d < HDB; d++) asm("" : "+a"(acc[d]));
}

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

// A panel of ROWS rows on its way from memory to LDS by way of registers, from any alignment: the chunks of one thread.  src: row 0, column 0 of a tensor with `pitch` values
// between rows; columns [lo, hi) and rows below `rows` are read, the others become zero.
template <typename T, int ROWS, int THREADS>
struct PanelLoad {
    static constexpr int N = ROWS * 8 / THREADS;
    static_assert(N * THREADS == ROWS * 8, "whole chunks per thread");
    v4u w[N];
    __device__ __forceinline__ void load(const T *src, size_t pitch, int rows, int col0, int lo, int hi) {
        typedef Mma<T> M;
        const bool whole = rows >= ROWS && col0 >= lo && col0 + M::COLS <= hi;       // the same for every thread
        if (whole) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int t = threadIdx.x + i * THREADS;
                const T *p = src + (size_t)(t >> 3) * pitch + col0 + (t & 7) * M::EPC;
                w[i] = *reinterpret_cast<const typename M::Any16 *>(p);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int t = threadIdx.x + i * THREADS, row = t >> 3, col = col0 + (t & 7) * M::EPC;
                v4u v = {0u, 0u, 0u, 0u};
                if (row < rows) {
                    const T *p = src + (size_t)row * pitch + col;
                    if (col >= lo && col + M::EPC <= hi) v = *reinterpret_cast<const typename M::Any16 *>(p);
                    else if (col < hi && col + M::EPC > lo) {
                        unsigned e[M::EPC];
#pragma unroll
                        for (int j = 0; j < M::EPC; j++) e[j] = col + j >= lo && col + j < hi ? bits(p[j]) : 0u;
                        if constexpr (M::EPC == 4) v = v4u{e[0], e[1], e[2], e[3]};
                        else v = v4u{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
                    }
                }
                w[i] = v;
            }
        }
    }
    __device__ __forceinline__ void store(char *panel) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int t = threadIdx.x + i * THREADS;
            *reinterpret_cast<v4u *>(panel + panel_at(t >> 3, t & 7)) = w[i];
        }
    }

private:
    static __device__ __forceinline__ unsigned bits(bf16_t v) { return v; }
    static __device__ __forceinline__ unsigned bits(float v) { return __float_as_uint(v); }
};

template <int HDB>
__device__ __forceinline__ bool has_nan(const v16f (&acc)[HDB]) {
    float s = 0.f;      // (infinities of both signs count too: that costs time, nothing else)
#pragma unroll
    for (int d = 0; d < HDB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) s += acc[d][r];
    return s != s;
}

// acc[channel][position] * f to the columns pos0 .. pos0 + 31 of `dst` whose lanes are active.  fp32: as they lie, a row of 32 columns to
// half a wave.  bfloat16: through LDS that is the wave's own, [position][channel], which the transposing read gives back as eight
// positions of a channel to a lane (rows of 64 bytes; two bytes a lane and a store for each register without it).
template <typename T, int HDB>
__device__ __forceinline__ void store_columns(T *dst, size_t pitch, int hd, const v16f (&acc)[HDB], float f, int pos0, bool active, char *lds) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (sizeof(T) == 4) {
        // offsets into the head's rows: 64-bit addresses and a condition for each row took ten times as long
        const unsigned row_bytes = (unsigned)pitch * 4, voff = active ? 4 * h * row_bytes + (pos0 + (lane & 31)) * 4 : OUTSIDE;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(dst, 0, (int)(hd * row_bytes), 0x00027000);
        const bool whole = hd >= HDB * 32;
#pragma unroll
        for (int d = 0; d < HDB; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int row = d * 32 + acc_row(i);
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(acc[d][i] * f), r, (int)(whole || row + 4 * h < hd ? voff : OUTSIDE), (int)(row * row_bytes), 0);
            }
    } else {
        constexpr int ROW = HDB * 64 + 16;          // (the 16 bytes spread the rows over the banks)
        typedef unsigned v2u __attribute__((ext_vector_type(2)));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int d = 0; d < HDB; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<v2u *>(lds + (lane & 31) * ROW + (d * 32 + acc_row(r) + 4 * h) * 2) =
                    v2u{f2_to_bf2(acc[d][r] * f, acc[d][r + 1] * f), f2_to_bf2(acc[d][r + 2] * f, acc[d][r + 3] * f)};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const unsigned mask = (unsigned)__ballot(active) >> (lane >> 4) * 8 & 0xff;       // the lane's eight positions
        const int i = lane & 15, q = (lane >> 4) * 8;
        const char *at = lds + (q + (i >> 2)) * ROW + (i & 3) * 8;
#pragma unroll
        for (int c = 0; c < HDB * 2; c++) {
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(at + c * 32));
            const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(at + c * 32 + 4 * ROW));
            const v8s v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            const int row = c * 16 + i;
            T *p = dst + (size_t)row * pitch + pos0 + q;
            if (row >= hd) continue;
            if (mask == 0xff) *reinterpret_cast<v4u_any *>(p) = __builtin_bit_cast(v4u, v);
            else
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (mask >> j & 1) p[j] = (T)v[j];
        }
    }
}

// The 32 positions of this wave (number `pos` of POS side by side, from col0 on) in N tensors, as fragments of a product over the channels.
// All their loads are under way together.  bfloat16: through LDS, as many panels of a tensor as the positions fill; begins when all waves
// are done with that place, ends with a barrier.  fp32: a fragment is a value of each lane, rows of 32 positions, straight from memory.
template <typename T, int POS>
constexpr int own_panels() { return (32 * POS + Mma<T>::COLS - 1) / Mma<T>::COLS; }
template <typename T, int HDB, int POS, int N, int STEPS>
__device__ __forceinline__ void own_columns(typename Mma<T>::Frag (&f)[N][STEPS], char *lds, const T *const (&src)[N], size_t pitch, int hd, int col0, int S,
                                            int pos) {
    typedef Mma<T> M;
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 4) {
        // as offsets into the head's rows: no load is behind a condition, or has an address of its own (positions behind the row's end: the
        // last one again, whose results nobody keeps)
        const int h = lane >> 5;
        const unsigned row_bytes = (unsigned)pitch * 4, voff = h * row_bytes + min(col0 + pos * 32 + (lane & 31), S - 1) * 4;
        const bool whole = hd >= 2 * STEPS;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(src[n]), 0, (int)(hd * row_bytes), 0x00027000);
#pragma unroll
            for (int s = 0; s < STEPS; s++)
                f[n][s] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)(whole || 2 * s + h < hd ? voff : OUTSIDE), (int)(2 * s * row_bytes), 0));
        }
    } else {
        constexpr int PANELS = own_panels<T, POS>(), BYTES = HDB * 32 * PANEL_ROW;
        PanelLoad<T, HDB * 32, 256> ld[N][PANELS];
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int p = 0; p < PANELS; p++) ld[n][p].load(src[n], pitch, hd, col0 + p * M::COLS, 0, S);
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int p = 0; p < PANELS; p++) ld[n][p].store(lds + (n * PANELS + p) * BYTES);
        __syncthreads();
        const char *panel = lds + (pos * 32 / M::COLS) * BYTES;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int s = 0; s < STEPS; s++) f[n][s] = M::columns(panel + n * PANELS * BYTES, pos * 32 % M::COLS / 32, s);
        __syncthreads();
    }
}

// The panels of a head on their way into LDS, one after the other: columns col0 .. col0 + COLS, whole chunks outside of [from, to) and rows
// from hd on zero.  `pitch` values between rows, a multiple of a chunk, as is the address of the first.  Loaded by WAVES waves, of which
// this is number `wave`.
template <typename T, int ROWS, int WAVES>
struct PanelStream {
    static constexpr int LOADS = ROWS / (8 * WAVES);
    static_assert(LOADS * 8 * WAVES == ROWS, "whole instructions per wave");
    rsrc_t r;
    unsigned voff, odd_voff, row_bytes;         // odd_voff: for one wave, whose rows of odd eights have another swizzle
    int hd, row, wave;
    __device__ __forceinline__ int chunk_of(int r) { return (threadIdx.x & 7) ^ panel_swz(r); }
    __device__ __forceinline__ void begin(const T *head, int pitch, int channels, int wave_) {
        wave = wave_;
        row = wave * 8 + ((threadIdx.x & 63) >> 3);
        hd = channels;
        row_bytes = (unsigned)pitch * sizeof(T);
        r = buffer_at(head, (unsigned long long)channels * row_bytes);
        voff = row * row_bytes + chunk_of(row) * 16;
        odd_voff = row * row_bytes + chunk_of(row + 8) * 16;
    }
    __device__ __forceinline__ void load(unsigned panel, int col0, int from, int to) {
        panel += wave * 1024;
        const unsigned soff = (unsigned)col0 * sizeof(T);
        if (col0 >= from && col0 + Mma<T>::COLS <= to && hd == ROWS) {
#pragma unroll
            for (int j = 0; j < LOADS; j++)
                load_to_lds(r, WAVES == 1 && (j & 1) ? odd_voff : voff, soff + j * 8 * WAVES * row_bytes, panel + j * WAVES * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < LOADS; j++) {
                const int at = row + j * 8 * WAVES, col = col0 + chunk_of(at) * Mma<T>::EPC;
                const unsigned v = WAVES == 1 && (j & 1) ? odd_voff : voff;
                load_to_lds(r, at < hd && col < to && col + Mma<T>::EPC > from ? v : OUTSIDE, soff + j * 8 * WAVES * row_bytes, panel + j * WAVES * 1024);
            }
        }
    }
};

// A position block's results, N of them: the accumulators of a position's teams added up in the order of the teams, and stored times f.
// A team does that for its share of the channels.  False if a sum is NaN, and nothing is stored then; `anyway` stores it.  Begins with
// everybody done with LDS, of which it takes N * HDB * 16 KB.
template <typename T, int HDB, int POS, int N>
__device__ __forceinline__ bool store_sums(T *const (&dst)[N], size_t pitch, int hd, const v16f (*const (&acc)[N])[HDB], const float (&f)[N], int pos0,
                                           bool active, char *lds, int pos, int team, bool anyway) {
    constexpr int TEAMS = 4 / POS, MINE = (HDB + TEAMS - 1) / TEAMS;       // blocks of 32 channels to a team
    char *own = lds + (threadIdx.x >> 6) * ((MINE * 64 + 16) * 32);
    bool odd = false;
    if constexpr (TEAMS == 1) {
#pragma unroll
        for (int n = 0; n < N; n++) odd |= has_nan(*acc[n]);
        if (!anyway && __syncthreads_or(active && odd)) return false;
#pragma unroll
        for (int n = 0; n < N; n++) store_columns<T, HDB>(dst[n], pitch, hd, *acc[n], f[n], pos0, active, own);
    } else {
        const int lane = threadIdx.x & 63, first = team * MINE * 32;
        auto at = [&](int n, int t, int d, int r) { return reinterpret_cast<v4f *>(lds) + ((((n * TEAMS + t) * POS + pos) * HDB + d) * 4 + r) * 64 + lane; };
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int d = 0; d < HDB; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const v16f &v = (*acc[n])[d];
                    *at(n, team, d, r) = v4f{v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]};
                }
        __syncthreads();
        v16f sum[N][MINE];
#pragma unroll
        for (int n = 0; n < N; n++) {
#pragma unroll
            for (int j = 0; j < MINE; j++) {
                const int d = min(team * MINE + j, HDB - 1);        // (a block behind the last: nobody stores it)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    v4f v = *at(n, 0, d, r);
#pragma unroll
                    for (int t = 1; t < TEAMS; t++) {
                        const v4f o = *at(n, t, d, r);
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e] += o[e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) sum[n][j][4 * r + e] = v[e];
                }
            }
            odd |= has_nan(sum[n]);
        }
        if (__syncthreads_or(active && odd) && !anyway) return false;
        if (first < hd)
#pragma unroll
            for (int n = 0; n < N; n++) store_columns<T, MINE>(dst[n] + (size_t)first * pitch, pitch, hd - first, sum[n], f[n], pos0, active, own);
    }
    return true;
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
    if (!(scale > 0.f) || !isfinite(scale * LOG2E)) {          // (exponents are of base 2)
        mi355_fail("%s: scale must be positive, and finite times log2(e)", who);
        return false;
    }
    // what a launch can number (2^32 threads, 256 to 64 positions at most), and 32-bit offsets into a head
    if (S > 1 << 22 || (double)heads * batch * ceil_div(S, 64) > (double)((1 << 24) - 1)) {
        mi355_fail("%s: heads * batch * ceil(S / 64) = %.0f (at most 2^24 - 1), S = %d (at most 2^22)", who, (double)heads * batch * ceil_div(S, 64), S);
        return false;
    }
    return true;
}

// Whether rows of S values can be loaded in whole chunks of 16 bytes as they lie.
template <typename T>
bool streams_directly(const T *p, int S) { return aligned16(p) && S % (16 / sizeof(T)) == 0; }

// Rows of S values into rows of whole chunks, zeros behind: up to two tensors of as many rows.
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(T *__restrict__ out0, T *__restrict__ out1, const T *__restrict__ in0, const T *__restrict__ in1,
                                                        size_t rows, int S, int pitch) {
    constexpr int EPC = Mma<T>::EPC;
    const T *in = blockIdx.y ? in1 : in0;
    T *out = blockIdx.y ? out1 : out0;
    const int chunks = pitch / EPC;
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x, row = t / chunks;
    const int col = (int)(t - row * chunks) * EPC;
    if (row >= rows) return;
    const T *p = in + row * S + col;
    if (col + EPC <= S) {
        *reinterpret_cast<v4u *>(out + row * pitch + col) = *reinterpret_cast<const typename Mma<T>::Any16 *>(p);
    } else
#pragma unroll
        for (int j = 0; j < EPC; j++) out[row * pitch + col + j] = col + j < S ? p[j] : (T)0;
}
template <typename T>
size_t packed_bytes(size_t rows, int S) {
    constexpr int EPC = Mma<T>::EPC;
    return (rows * ((S + EPC - 1) / EPC * EPC) * sizeof(T) + 255) & ~(size_t)255;
}
// Two tensors to `ws`, packed_bytes() for each.
template <typename T>
int pack_rows(const char *who, const T **a, const T **b, size_t rows, int S, int *pitch, void *ws) {
    constexpr int EPC = Mma<T>::EPC;
    *pitch = (S + EPC - 1) / EPC * EPC;
    const size_t threads = rows * (*pitch / EPC);
    if (ceil_div(threads, 256) > 0xffffff) return mi355_fail("%s: %zu rows of %d positions, which are no whole 16 bytes, are too many", who, rows, S);
    T *d0 = (T *)ws, *d1 = (T *)((char *)ws + packed_bytes<T>(rows, S));
    pack_rows_kernel<T><<<dim3((unsigned)ceil_div(threads, 256), 2), 256, 0, g_ctx.stream>>>(d0, d1, *a, *b, rows, S, *pitch);
    LAUNCH_OK(who);
    *a = d0;
    *b = d1;
    return 0;
}

// How many waves of a workgroup stand side by side (32 positions each, sharing the panels that they read), and in how many teams, which
// share the walk: team i takes every TEAMS-th tile of it, with panels of its own.  Four side by side where that gives every compute unit two
// workgroups; else two by two, where that gives it `two_from` half workgroups; else one position block to four teams.  Measured on 256
// compute units with four / two / one side by side, us:
//   four blocks of 512, 1024 of two: forward, bfloat16, 128 channels, 4096 positions of 16 heads 141 / 181 / 242
//   192, 384: forward, 64 channels, 256 positions of 96 heads: bfloat16 10.2 / 7.9 / 17.5, fp32 25.2 / 19.0 / 26.2; all gradients: bfloat16
//             32 / 21.6 / 37, fp32 76 / 57 / 72
//   128, 256: 128 channels, 512 positions of 32 heads, bfloat16: forward 20.0 / 15.4 / 19.3, all gradients (only dq changed) 57 / 51 /
//             56; but all gradients (only dk and dv changed), 64 channels, 1024 positions of 16 heads for 48: 140 / 89 / 74, and fp32, 2048
//             positions of 8 heads: forward 158 / 83 / 58, all gradients (both changed) 491 / 258 / 164
//   32, 64:   forward, bfloat16, 96 channels, 1024 positions of 4 heads 29.0 / 20.6 / 14.7
constexpr int TWO_FROM = 3;                                                     // half workgroups to a compute unit
template <typename T>
constexpr int TWO_FROM_QUERIES = sizeof(T) == 2 ? 2 : TWO_FROM;                 // (the forward pass and dq)
int waves_for(size_t heads_batch, int S, int two_from) {
    if (ceil_div(S, 128) * heads_batch >= 2 * (size_t)g_ctx.num_cu) return 4;
    return 2 * ceil_div(S, 64) * heads_batch >= two_from * (size_t)g_ctx.num_cu ? 2 : 1;
}
template <typename F>
int dispatch(int hd, int waves, F go) {
    auto by_waves = [&](auto hdb) {
        if (waves == 4) return go(hdb, std::integral_constant<int, 4>());
        if (waves == 2) return go(hdb, std::integral_constant<int, 2>());
        return go(hdb, std::integral_constant<int, 1>());
    };
    if (hd <= 64) return by_waves(std::integral_constant<int, 2>());
    if (hd <= 96) return by_waves(std::integral_constant<int, 3>());
    return by_waves(std::integral_constant<int, 4>());
}

}  // namespace
