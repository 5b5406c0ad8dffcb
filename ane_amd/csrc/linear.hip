// linear.hip — the products of a layer on bfloat16 storage: y = res + alpha * act(w x + bias) and its gradients, channel-first:
// x [batch][K][S], w [M][K], y [batch][M][S].  The reference runs them inside its MIL kernels (1x1 convolutions with their weights baked
// in or handed over, training/training_dynamic/mil_dynamic.h) and as cblas_sgemm (training/training_dynamic/train.m:490-508, 577-685).
//
// With n = (sequence, position) running over all columns of the batch:
//   forward    C[m][n] = sum_k w[m][k] x[k][n]            w by rows (the sum along them), x by columns
//   dx         C[k][n] = sum_m w[m][k] dy[m][n]           both by columns
//   dw         C[m][k] = sum_n dy[m][n] x[k][n]           both by rows
// so a tensor is always read as rows of consecutive columns, 64 of them to a panel of LDS (mma.h); what differs is which way the panel is
// read.  A workgroup forms a tile of C over a slice of the sum; sums are fp32 in the matrix cores' registers, slices (where C has too few
// tiles for the compute units) are added in a fixed order by a second launch, which then has the epilogue.
#include "mma.h"

#include <initializer_list>
#include <math.h>

namespace {

typedef Mma<bf16_t> M16;

// A tensor of the product: rows of `S` consecutive values, `batch` slabs of them side by side as columns b * S + s.
struct Mat {
    const bf16_t *p;
    int rows, S, cols;      // cols = batch * S
};

enum { FORWARD = 0, DX = 1, DW = 2 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

struct Epilogue {
    int act;
    float alpha;
    const float *bias;          // forward: [M]
    const bf16_t *res;          // forward: [batch][M][S]
    const bf16_t *pre;          // dx: what the activation below was applied to
    bf16_t *pre_out;            // forward: w x + bias
    bf16_t *out;                // forward, dx
    float *dw;
    int accumulate;
};

constexpr float GELU_C = 0.797884583473205566406f;      // sqrt(2 / pi)

// GELU in its tanh form, through tanh(y) = 2 sigmoid(2y) - 1.  Far below zero the exponential is infinite and the sigmoid zero, as it should.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }      // (1 / inf is 0 there too)
template <int ACT>
__device__ __forceinline__ float act_value(float x) {
    if (ACT == ACT_RELU) return x < 0.f ? 0.f : x;      // (a NaN stays one)
    if (ACT == ACT_SILU) return x * sigmoid(x);
    if (ACT == ACT_GELU) return x * sigmoid(2.f * GELU_C * (x + 0.044715f * x * x * x));
    return x;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float x) {
    if (ACT == ACT_RELU) return x > 0.f ? 1.f : (x == x ? 0.f : x);
    if (ACT == ACT_SILU) {
        const float g = sigmoid(x);
        return g * (1.f + x * (1.f - g));
    }
    if (ACT == ACT_GELU) {
        x = __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, 16.f), -16.f);       // the slope's limits, long reached; x^2 stays finite
        const float g = sigmoid(2.f * GELU_C * (x + 0.044715f * x * x * x));
        return g + x * (2.f * g * (1.f - g)) * GELU_C * (1.f + 0.134145f * x * x);
    }
    return 1.f;
}
// One branch for many values: with one for each, the epilogue of a 256 x 256 tile took four times as long.
template <typename F>
__device__ __forceinline__ void by_act(int act, F f) {
    if (act == ACT_NONE) f(std::integral_constant<int, ACT_NONE>());
    else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>());
    else if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>());
    else f(std::integral_constant<int, ACT_GELU>());
}

// Eight values of row `m` of C from column n on (fewer at the end of a row) to where they belong.
template <int KIND>
__device__ __forceinline__ void finish(const Epilogue &e, float (&v)[8], int m, int rows, int n, int cols, int S) {
    if (KIND == DW) {
        float *p = e.dw + (size_t)m * cols + n;
        const int k = min(8, cols - n);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= e.alpha;
        if (k == 8) {
            if (e.accumulate) {
                const v4f a = ld4(p), b = ld4(p + 4);
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] += a[j], v[4 + j] += b[j];
            }
            st4(p, v4f{v[0], v[1], v[2], v[3]});
            st4(p + 4, v4f{v[4], v[5], v[6], v[7]});
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < k) p[j] = e.accumulate ? p[j] + v[j] : v[j];
        }
        return;
    }
    const int b = n / S, s = n - b * S;
    const float bias = KIND == FORWARD && e.bias ? e.bias[m] : 0.f;
    if (s + 8 <= S) {
        const size_t at = ((size_t)b * rows + m) * S + s;
        if (KIND == FORWARD) {
            if (e.bias) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] += bias;
            }
            if (e.pre_out) stb<8>(e.pre_out + at, v);
            float r[8];
            if (e.res) ldb<8, true>(r, e.res + at);
            by_act(e.act, [&](auto act) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = e.alpha * act_value<decltype(act)::value>(v[j]);
            });
            if (e.res) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] += r[j];
            }
        } else {
            float r[8];
            if (e.act != ACT_NONE) ldb<8, true>(r, e.pre + at);
            by_act(e.act, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    v[j] *= e.alpha;
                    if (ACT != ACT_NONE) v[j] *= act_slope<ACT>(r[j]);
                }
            });
        }
        stb<8>(e.out + at, v);
        return;
    }
    // the columns go over into the next sequence, or end
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (n + j >= cols) break;
        const int bj = (n + j) / S, sj = n + j - bj * S;
        const size_t at = ((size_t)bj * rows + m) * S + sj;
        float x = v[j];
        if (KIND == FORWARD) {
            if (e.bias) x += bias;
            if (e.pre_out) e.pre_out[at] = (bf16_t)f_to_bf(x);
            by_act(e.act, [&](auto act) { x = e.alpha * act_value<decltype(act)::value>(x); });
            if (e.res) x += bf_to_f(e.res[at]);
        } else {
            x *= e.alpha;
            if (e.act != ACT_NONE) by_act(e.act, [&](auto act) { x *= act_slope<decltype(act)::value>(bf_to_f(e.pre[at])); });
        }
        e.out[at] = (bf16_t)f_to_bf(x);
    }
}

// Tensors go straight into LDS (load_to_lds).  They are aligned: base and S in units of eight values; repack() brings others to that.
// An operand's 64 steps of the sum for B indexes (PanelWalk has the offsets).
template <int B, bool COLUMNS, int THREADS>
struct Operand {
    typedef PanelWalk<B, COLUMNS, THREADS> Walk;
    static constexpr int BYTES = B * PANEL_ROW, LOADS = Walk::PANELS * Walk::PER;       // of a stage; a wave's instructions to it
    static constexpr int READS = COLUMNS ? 2 : 1;           // reads of LDS to a fragment
    rsrc_t r;
    Walk walk;
    unsigned wave_at;

    // index0: the tile's first index; sum0: where the sum starts
    __device__ __forceinline__ void begin(const Mat &a, int index0, int sum0) {
        wave_at = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
        const unsigned long long skip = walk.begin(a.rows, a.S, a.cols, index0, sum0, threadIdx.x);
        r = buffer_at((const char *)a.p + skip, walk.bytes);
    }
    // the next 64 steps of the sum, `left` of which exist, to a stage of LDS; moves on
    __device__ __forceinline__ void load(unsigned lds, int left) {
        lds += wave_at;
        if (walk.plain(left)) {
#pragma unroll
            for (int i = 0; i < Walk::PANELS; i++)
#pragma unroll
                for (int j = 0; j < Walk::PER; j++)
                    load_to_lds(r, walk.voff[i], walk.soffset(j), lds + i * (64 * PANEL_ROW) + j * Walk::WAVES * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < Walk::PANELS; i++)
#pragma unroll
                for (int j = 0; j < Walk::PER; j++)
                    load_to_lds(r, walk.voffset(i, j, left, threadIdx.x), walk.soffset(j), lds + i * (64 * PANEL_ROW) + j * Walk::WAVES * 1024);
        }
        if (const unsigned long long move = walk.advance()) {
            const unsigned long long at = ((unsigned long long)(unsigned)r[1] << 32 | (unsigned)r[0]) + move;
            r = buffer_at((const void *)at, walk.bytes);
        }
    }
    // the fragment of indexes block*32 .. +31 at 16 steps of the sum
    static __device__ __forceinline__ M16::Frag frag(const char *lds, int block, int step) {
        if constexpr (COLUMNS) return M16::columns(lds + (block >> 1) * (64 * PANEL_ROW), block & 1, step);
        else return M16::along(lds, block, step);
    }
};

// What a wave has of C, written where it belongs.  The product is formed with C's columns in the registers (four consecutive ones at a time)
// and a row to the lane; 32 rows at a time then go through LDS that is the wave's own, so that memory sees whole rows of the tile.  The
// residual, or what the activation below was applied to, comes in by the same way.
template <int KIND, int FM, int FN>
struct WaveOut {
    static constexpr int WN = FN * 32;
    static constexpr int BYTES = 32 * (WN * 4 + 16);        // for fp32 rows; the 16 bytes behind each row spread them over the banks
    static __device__ __forceinline__ void settle() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

    static __device__ __forceinline__ void floats(char *lds, const v16f (&acc)[FN], float *out, size_t pitch, int m0, int n0, int M, int N, float alpha, bool accumulate) {
        constexpr int PITCH = WN * 4 + 16, LANES = WN / 4;
        const int lane = threadIdx.x & 63, h = lane >> 5, at = lane % LANES * 4;
        settle();
#pragma unroll
        for (int k = 0; k < FN; k++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<v4f *>(lds + (lane & 31) * PITCH + (k * 32 + 8 * q + 4 * h) * 4) =
                    v4f{acc[k][4 * q], acc[k][4 * q + 1], acc[k][4 * q + 2], acc[k][4 * q + 3]};
        settle();
        const int n = n0 + at, left = n < N ? M - m0 - lane / LANES : 0;
        float *p = out + (size_t)(m0 + lane / LANES) * pitch + n;
#pragma unroll
        for (int i = 0; i < 32; i += 64 / LANES, p += 64 / LANES * pitch) {
            v4f v = *reinterpret_cast<const v4f *>(lds + (i + lane / LANES) * PITCH + at * 4);
            if (i >= left) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] *= alpha;
            if (n + 4 <= N) {
                if (accumulate) {
                    const v4f old = ld4(p);
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] += old[j];
                }
                st4(p, v);
            } else
                for (int j = 0; n + j < N; j++) p[j] = accumulate ? p[j] + v[j] : v[j];
        }
    }

    // Eight columns of rows m, m + STEP, ... between memory and LDS: a lane's own place in each of them.  Where a sequence ends within the
    // eight, or the columns do, one by one.
    struct Columns { int n, b, s, N, S; };
    template <typename F>
    static __device__ __forceinline__ void each_row(const Columns &c, int rows, int m, int M, F f) {
        constexpr int STEP = 64 / (WN / 8);
        size_t at = ((size_t)c.b * rows + m) * c.S + c.s;
        const int left = c.n < c.N ? M - m : 0;
#pragma unroll
        for (int i = 0; i < 32 / STEP; i++, at += (unsigned)(STEP * c.S))
            f(i, at, i * STEP < left);
    }
    static __device__ __forceinline__ v4u read8(const bf16_t *src, size_t at, int rows, const Columns &c) {
        if (c.s + 8 <= c.S) return *reinterpret_cast<const v4u_any *>(src + at);
        unsigned e[8];
        int s = c.s;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            e[j] = c.n + j < c.N ? src[at] : 0u;
            at++;
            if (++s == c.S) s = 0, at += (size_t)(rows - 1) * c.S;
        }
        return v4u{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
    }
    static __device__ __forceinline__ void write8(bf16_t *dst, size_t at, int rows, const Columns &c, v4u v) {
        if (c.s + 8 <= c.S) {
            *reinterpret_cast<v4u_any *>(dst + at) = v;
            return;
        }
        int s = c.s;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (c.n + j < c.N) dst[at] = (bf16_t)(v[j >> 1] >> (j & 1) * 16);
            at++;
            if (++s == c.S) s = 0, at += (size_t)(rows - 1) * c.S;
        }
    }

    static __device__ __forceinline__ void halves(char *lds, const v16f (&acc)[FN], const Epilogue &e, int m0, int M, const Columns &c) {
        constexpr int PITCH = WN * 2 + 16, LANES = WN / 8;
        const int lane = threadIdx.x & 63, h = lane >> 5, row0 = lane / LANES;
        const bf16_t *in = KIND == FORWARD ? e.res : e.act != ACT_NONE ? e.pre : nullptr;
        char *mine = lds + (lane & 31) * PITCH + h * 8, *rows = lds + row0 * PITCH + lane % LANES * 16;
        if (in) {
            v4u w[32 * LANES / 64];
            each_row(c, M, m0 + row0, M, [&](int i, size_t at, bool there) { w[i] = there ? read8(in, at, M, c) : v4u{0u, 0u, 0u, 0u}; });
            settle();
#pragma unroll
            for (int i = 0; i < 32 * LANES / 64; i++) *reinterpret_cast<v4u *>(rows + i * (64 / LANES) * PITCH) = w[i];
        }
        settle();
        const float bias = KIND == FORWARD && e.bias && m0 + (lane & 31) < M ? e.bias[m0 + (lane & 31)] : 0.f;
        by_act(e.act, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            auto quads = [&](auto with) {           // with: whether LDS holds something of these columns
                constexpr bool IN = decltype(with)::value;
#pragma unroll
                for (int k = 0; k < FN; k++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        typedef unsigned v2u __attribute__((ext_vector_type(2)));
                        v2u *at = reinterpret_cast<v2u *>(mine + k * 64 + q * 16);
                        v2u r = {0u, 0u};
                        if (IN) r = *at;
                        float v[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float x = bf_to_f(j & 1 ? r[j >> 1] >> 16 : r[j >> 1] & 0xffffu);
                            if (KIND == FORWARD) {
                                v[j] = e.alpha * act_value<ACT>(acc[k][4 * q + j] + bias);
                                if (IN) v[j] += x;
                            } else {
                                v[j] = e.alpha * acc[k][4 * q + j];
                                if (IN) v[j] *= act_slope<ACT>(x);
                            }
                        }
                        *at = v2u{f2_to_bf2(v[0], v[1]), f2_to_bf2(v[2], v[3])};
                    }
            };
            if (KIND == DX) quads(std::integral_constant<bool, ACT != ACT_NONE>());
            else if (in) quads(std::true_type());
            else quads(std::false_type());
        });
        settle();
        each_row(c, M, m0 + row0, M, [&](int i, size_t at, bool there) {
            const v4u v = *reinterpret_cast<const v4u *>(rows + i * (64 / LANES) * PITCH);
            if (there) write8(e.out, at, M, c, v);
        });
        if (KIND == FORWARD && e.pre_out) {
            settle();
#pragma unroll
            for (int k = 0; k < FN; k++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    typedef unsigned v2u __attribute__((ext_vector_type(2)));
                    *reinterpret_cast<v2u *>(mine + k * 64 + q * 16) = v2u{f2_to_bf2(acc[k][4 * q] + bias, acc[k][4 * q + 1] + bias),
                                                                           f2_to_bf2(acc[k][4 * q + 2] + bias, acc[k][4 * q + 3] + bias)};
                }
            settle();
            each_row(c, M, m0 + row0, M, [&](int i, size_t at, bool there) {
                const v4u v = *reinterpret_cast<const v4u *>(rows + i * (64 / LANES) * PITCH);
                if (there) write8(e.pre_out, at, M, c, v);
            });
        }
    }
};

// One product of a launch: C[M][N] in tiles, each over a slice of the sum.
struct Work {
    Mat a, b;
    Epilogue e;
    float *part;                // slices of C, where there are more than one
    int M, N, out_s, sum, slice_steps, tiles_m, tiles_n, units;
};

template <int KIND, int BM, int BN, int WM, int WN, int STAGES>
constexpr int lds_bytes() {
    constexpr int waves = BM / WM * (BN / WN), out = waves * WaveOut<KIND, WM / 32, WN / 32>::BYTES, stages = STAGES * (BM + BN) * PANEL_ROW;
    return out > stages ? out : stages;
}

template <int KIND, int BM, int BN, int WM, int WN, int STAGES>
__device__ __forceinline__ void product_unit(const Work &w, int unit, char *lds) {
    const Mat &a = w.a, &b = w.b;
    const Epilogue &e = w.e;
    float *const part = w.part;
    const int M = w.M, N = w.N, out_s = w.out_s, tiles = w.tiles_m * w.tiles_n, slice = unit / tiles, tile = unit - slice * tiles;
    constexpr int WAVES_M = BM / WM, WAVES_N = BN / WN, THREADS = WAVES_M * WAVES_N * 64, FM = WM / 32, FN = WN / 32;
    typedef Operand<BM, KIND == DX, THREADS> A;
    typedef Operand<BN, KIND != DW, THREADS> B;
    typedef WaveOut<KIND, FM, FN> Out;
    constexpr int STAGE = A::BYTES + B::BYTES, LOADS = A::LOADS + B::LOADS;
    // With three stages or more the one after the present one has arrived too, so that its first fragments can be read ahead.
    constexpr bool AHEAD = STAGES > 2;
    constexpr int LEFT = LOADS * (AHEAD ? STAGES - 3 : 0), FULL = AHEAD ? STAGES - 1 : 2;
    const int m0 = tile % w.tiles_m * BM, n0 = tile / w.tiles_m * BN;
    const int sum0 = slice * w.slice_steps * 64, sum1 = min(w.sum, sum0 + w.slice_steps * 64), steps = (sum1 - sum0 + 63) / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave / WAVES_N * FM, wn = wave % WAVES_N * FN;

    const unsigned place = lds_place(lds);
    A la;
    B lb;
    la.begin(a, m0, sum0);
    lb.begin(b, n0, sum0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++)
        if (i < steps) {
            la.load(place + i * STAGE, sum1 - sum0 - i * 64);
            lb.load(place + i * STAGE + A::BYTES, sum1 - sum0 - i * 64);
        }
    v16f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = v16_zero();
    // Fragments are read DEEP steps of 16 before they are multiplied: a read takes longer than one step's products.  They are a ring.
    constexpr int DEEP = AHEAD ? 2 : 1, RING = DEEP == 2 ? 4 : 2;
    M16::Frag fa[RING][FM], fb[RING][FN];
    auto fetch = [&](int set, const char *p, int s) {
#pragma unroll
        for (int j = 0; j < FM; j++) fa[set][j] = A::frag(p, wm + j, s);
#pragma unroll
        for (int j = 0; j < FN; j++) fb[set][j] = B::frag(p + A::BYTES, wn + j, s);
    };
    if (AHEAD) {
        if (steps >= STAGES - 1) loads_and_barrier<LOADS *(STAGES - 2), 0>();
        else loads_and_barrier<0, 0>();
        __builtin_amdgcn_s_waitcnt(0xc07f);     // lgkmcnt(0), for the compiler to know that no scalar load is under way in the loop
        fetch(0, lds, 0);
        fetch(1, lds, 1);
    }
    // reads of the stage to come that are under way at the barrier; all before them are done when no more than these are
    constexpr int READS = AHEAD ? DEEP * (FM * A::READS + FN * B::READS) : 0, READS_LEFT = READS < 15 ? READS : 15;
    int at = 0, next = STAGES - 1;              // the stages that are read and written
    for (int i = 0; i < steps; i++) {
        // everybody is done with the stage before `at`, which is filled again
        if (steps - i >= FULL) loads_and_barrier<LEFT, READS_LEFT>();
        else loads_and_barrier<0, READS_LEFT>();
        if (i + STAGES - 1 < steps) {
            la.load(place + next * STAGE, sum1 - sum0 - (i + STAGES - 1) * 64);
            lb.load(place + next * STAGE + A::BYTES, sum1 - sum0 - (i + STAGES - 1) * 64);
        }
        const char *p = lds + at * STAGE;
        at = at + 1 == STAGES ? 0 : at + 1;
        next = next + 1 == STAGES ? 0 : next + 1;
        const char *p1 = lds + at * STAGE;
        if (!AHEAD) fetch(0, p, 0);
#pragma unroll
        for (int s = 0; s < 4; s++) {
            // (past the last stage: read, not used)
            if (s + DEEP < 4) fetch((s + DEEP) & (RING - 1), p, s + DEEP);
            else if (AHEAD) fetch((s + DEEP) & (RING - 1), p1, s + DEEP - 4);
            __builtin_amdgcn_sched_barrier(0);      // (left alone, the compiler puts each read right before the product that needs it)
#pragma unroll
            for (int j = 0; j < FM; j++)
#pragma unroll
                for (int k = 0; k < FN; k++) acc[j][k] = M16::mul(fb[s & (RING - 1)][k], fa[s & (RING - 1)][j], acc[j][k]);
        }
    }
    __syncthreads();
    char *mine = lds + wave * Out::BYTES;
    const int n = n0 + wn * 32 + lane % (FN * 4) * 8, slab = KIND == DW ? 0 : n / out_s;
    const typename Out::Columns cols = {n, slab, n - slab * out_s, N, out_s};
#pragma unroll 1
    for (int i = 0; i < FM; i++) {              // (one copy of the code for all blocks of 32 rows)
        v16f cur[FN];
#pragma unroll
        for (int j = 0; j < FM; j++)
            if (i == j) {
#pragma unroll
                for (int k = 0; k < FN; k++) cur[k] = acc[j][k];
            }
        const int m = m0 + (wm + i) * 32;
        if (part || KIND == DW)
            Out::floats(mine, cur, part ? part + (size_t)slice * M * N : e.dw, N, m, n0 + wn * 32, M, N, part ? 1.f : e.alpha, !part && e.accumulate);
        else Out::halves(mine, cur, e, m, M, cols);
    }
}

// What bounds it: 256 x 256 tiles, 32000 x 4096 results of 768 terms 270 to 290 us, 720 TFLOP/s (a library product of that size 205 to 208; in a
// kernel trace, whose calls follow one another less closely, 278 to 354): a tile takes 26 us of which 18 are the sum's products at 1.5
// times what the matrix cores alone need, 7.3 the way of its 128 KB of results to memory, and its successor starts 3.5 later, with nobody
// else on the compute unit.  128 x 128 tiles: 1024 x 4096 results of 2048 terms with the residual 25 to 29 us from one card to another, 640
// TFLOP/s (the library's product alone 24.6).  Both gradients of that layer 53 to 62 us, 600 TFLOP/s, of which 9 for the slices and row sums.
// The units of one or two products, a workgroup to each, neighbours on one XCD (xcd_remap).  (As many workgroups as run
// at once, each with several units: 278 -> 297 us for 32000 x 4096 results.  A unit's first loads then come behind the stores of the one
// before, and so does the wait for them.)
template <int KIND0, int KIND1, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(BM / WM *BN / WN * 64) void linear_kernel(Work w0, Work w1, int one_first) {
    constexpr int B0 = lds_bytes<KIND0, BM, BN, WM, WN, STAGES>(), B1 = lds_bytes<KIND1, BM, BN, WM, WN, STAGES>();
    __shared__ __attribute__((aligned(1024))) char lds[B0 > B1 ? B0 : B1];
    if constexpr (KIND0 == KIND1) product_unit<KIND0, BM, BN, WM, WN, STAGES>(w0, xcd_remap(blockIdx.x, gridDim.x), lds);
    else {
        // The longer product's units come first, on every XCD.  (With one run of both for all XCDs the first of these had all of the long
        // units: gradients of 1024 x 2048 weights over 4096 columns 73.5 us for 62, of 512 x 2800 over 2048 columns 38 for 28.)
        const DealtUnit d = xcd_deal(blockIdx.x, one_first ? w1.units : w0.units, gridDim.x);
        if (d.second == (one_first != 0)) product_unit<KIND0, BM, BN, WM, WN, STAGES>(w0, d.unit, lds);
        else product_unit<KIND1, BM, BN, WM, WN, STAGES>(w1, d.unit, lds);
    }
}

// (8 rows of 197 positions x 768 channels: 4 to 6 us, of 21.4 for the whole call; read from there as often as tiles need it.)
// A tensor whose rows begin at any value, as one of [rows][cols8] whose rows begin at multiples of eight: zeros from its last column on.
__global__ __launch_bounds__(256) void repack_kernel(bf16_t *__restrict__ out, Mat a, int cols8) {
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int groups = cols8 / 8;
    if (t >= (size_t)a.rows * groups) return;
    const int row = (int)(t / groups), col = (int)(t % groups) * 8;
    int b = col / a.S, s = col - b * a.S;
    v4u v;
    if (col + 8 <= a.cols && s + 8 <= a.S) v = *reinterpret_cast<const v4u_any *>(a.p + ((size_t)b * a.rows + row) * a.S + s);
    else {
        unsigned e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            e[j] = col + j < a.cols ? a.p[((size_t)b * a.rows + row) * a.S + s] : 0u;
            if (++s == a.S) s = 0, b++;
        }
        v = v4u{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
    }
    *reinterpret_cast<v4u *>(out + (size_t)row * cols8 + col) = v;
}

// The slices of a product added up in their order, and its epilogue: eight columns of a row to a thread.
template <int KIND>
__device__ __forceinline__ void join(const Work &w, size_t t) {
    const int groups = (w.N + 7) / 8, N = w.N, slices = w.units / (w.tiles_m * w.tiles_n);
    const int m = (int)(t / groups), n = (int)(t % groups) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0.f;
    const float *p = w.part + (size_t)m * N + n;
    if (n + 8 <= N) {
#pragma unroll 4
        for (int i = 0; i < slices; i++, p += (size_t)w.M * N) {
            const v4f a = ld4(p), b = ld4(p + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] += a[j], v[4 + j] += b[j];
        }
    } else {
        for (int i = 0; i < slices; i++, p += (size_t)w.M * N)
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < N) v[j] += p[j];
    }
    finish<KIND>(w.e, v, m, w.M, n, N, w.out_s);
}
// dbias[m] (+)= alpha * sum of row m of dy over the batch: a wave to a row, a fixed tree.
struct RowSums {
    float *out;
    const bf16_t *dy;
    int M, S, batch, accumulate;
    float alpha;
};
__device__ __forceinline__ void row_sum(const RowSums &r, int m) {
    const int lane = threadIdx.x & 63;
    const int chunks = (r.S + 7) / 8, total = r.batch * chunks;
    float s = 0.f;
#pragma unroll 4
    for (int c = lane; c < total; c += 64) {
        const int b = c / chunks, i = (c - b * chunks) * 8;
        const bf16_t *p = r.dy + ((size_t)b * r.M + m) * r.S + i;
        if (i + 8 <= r.S) {
            float v[8];
            ldb<8, false>(v, p);
#pragma unroll
            for (int j = 0; j < 8; j++) s += v[j];
        } else
            for (int j = 0; i + j < r.S; j++) s += bf_to_f(p[j]);
    }
    s = wave_sum_far_first(s) * r.alpha;
    if (lane == 0) r.out[m] = r.accumulate ? r.out[m] + s : s;
}

// What comes after the products: workgroups for the first one's slices, for the second one's, for the row sums.
template <int KIND0, int KIND1>
__global__ __launch_bounds__(256) void linear_join_kernel(Work w0, Work w1, RowSums r, int groups0, int groups1) {
    const int g = blockIdx.x;
    if (KIND1 != KIND0 && g >= groups0 + groups1) {
        const int m = (g - groups0 - groups1) * 4 + (threadIdx.x >> 6);
        if (m < r.M) row_sum(r, m);
    } else if (KIND1 != KIND0 && g >= groups0) {
        const size_t t = (size_t)(g - groups0) * 256 + threadIdx.x;
        if (t < (size_t)w1.M * ((w1.N + 7) / 8)) join<KIND1>(w1, t);
    } else {
        const size_t t = (size_t)g * 256 + threadIdx.x;
        if (t < (size_t)w0.M * ((w0.N + 7) / 8)) join<KIND0>(w0, t);
    }
}

// Few columns: y is bound by reading w once, in rows.  A wave takes rows of w, its lanes eight steps of the sum at a time; x, as fp32 in LDS
// [column][step], serves all rows of the workgroup.  NC columns at once.
constexpr int GEMV_MAX = 4;
template <int NC>
__global__ __launch_bounds__(256) void gemv_kernel(const bf16_t *__restrict__ w, const bf16_t *__restrict__ x, Epilogue e, int M, int K, int N, int S,
                                                   int kpad) {
    extern __shared__ __attribute__((aligned(16))) float xs[];
    size_t column[NC];
#pragma unroll
    for (int n = 0; n < NC; n++) column[n] = n < N ? (size_t)(n / S) * K * S + n % S : 0;
#pragma unroll 4
    for (int k = threadIdx.x; k < kpad; k += 256)
#pragma unroll
        for (int n = 0; n < NC; n++) xs[n * kpad + k] = n < N && k < K ? bf_to_f(x[column[n] + (size_t)k * S]) : 0.f;
    __syncthreads();
    const int lane = threadIdx.x & 63;
    for (int m = blockIdx.x * 4 + (threadIdx.x >> 6); m < M; m += gridDim.x * 4) {
        float acc[NC];
#pragma unroll
        for (int n = 0; n < NC; n++) acc[n] = 0.f;
        const bf16_t *row = w + (size_t)m * K;
#pragma unroll 4
        for (int k = lane * 8; k < kpad; k += 512) {
            float v[8];
            if (k + 8 <= K) ldb<8, true>(v, row + k);
            else
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = k + j < K ? bf_to_f(row[k + j]) : 0.f;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                const v4f a = *reinterpret_cast<const v4f *>(xs + n * kpad + k), b = *reinterpret_cast<const v4f *>(xs + n * kpad + k + 4);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[n] = __builtin_fmaf(v[4 + j], b[j], __builtin_fmaf(v[j], a[j], acc[n]));
            }
        }
        float mine = 0.f;
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const float s = wave_sum_far_first(acc[n]);
            mine = lane == n ? s : mine;
        }
        if (lane < N && lane < NC) {
            const int b = lane / S;
            const size_t at = ((size_t)b * M + m) * S + (lane - b * S);
            if (e.bias) mine += e.bias[m];
            if (e.pre_out) e.pre_out[at] = (bf16_t)f_to_bf(mine);
            by_act(e.act, [&](auto act) { mine = e.alpha * act_value<decltype(act)::value>(mine); });
            if (e.res) mine += bf_to_f(e.res[at]);
            e.out[at] = (bf16_t)f_to_bf(mine);
        }
    }
}

// dpre may be dy: a thread loads what it writes before it does.  Three tensors once: 2^20 values 3.7 us, 2^25 33.5 or 6.0 TB/s, 2^27 125 or 6.5.
__global__ __launch_bounds__(256) void act_bwd_kernel(bf16_t *dpre, const bf16_t *dy, const bf16_t *__restrict__ pre, float alpha, int act, size_t n) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i + 8 <= n) {
        float g[8], x[8];
        ldb<8, true>(g, dy + i);
        ldb<8, true>(x, pre + i);
        by_act(act, [&](auto a) {
#pragma unroll
            for (int j = 0; j < 8; j++) g[j] = alpha * g[j] * act_slope<decltype(a)::value>(x[j]);
        });
        stb<8>(dpre + i, g);
    } else
        for (size_t j = i; j < n; j++)
            by_act(act, [&](auto a) { dpre[j] = (bf16_t)f_to_bf(alpha * bf_to_f(dy[j]) * act_slope<decltype(a)::value>(bf_to_f(pre[j]))); });
}

// Whether linear_kernel can read a tensor as it is: chunks of eight values that begin at multiples of 16 bytes, and one slab, or 32-bit offsets
// over those that 256 columns (or 64 of the sum) reach from where they begin.
bool direct(const Mat &a) {
    return aligned16(a.p) && a.S % 8 == 0 && (a.cols == a.S || ((double)(256 / a.S + 2) * a.rows + 256) * a.S * 2 < 4e9);
}
size_t repacked_bytes(const Mat &a) { return direct(a) ? 0 : ((size_t)a.rows * ((a.cols + 7) & ~7) * 2 + 255) & ~(size_t)255; }
int repack(const char *who, Mat &a, char *&ws) {
    if (direct(a)) return 0;
    const int cols8 = (a.cols + 7) & ~7;
    const size_t threads = (size_t)a.rows * (cols8 / 8);
    if (ceil_div(threads, 256) > 0xffffff) return mi355_fail("%s: %d rows of %d columns, which do not begin at whole 16 bytes, are too many", who, a.rows, a.cols);
    repack_kernel<<<(unsigned)ceil_div(threads, 256), 256, 0, g_ctx.stream>>>((bf16_t *)ws, a, cols8);
    LAUNCH_OK(who);
    const size_t bytes = repacked_bytes(a);
    a = Mat{(bf16_t *)ws, a.rows, cols8, cols8};
    ws += bytes;
    return 0;
}

// Tiles of C: 256 x 256 (eight waves, the fewest reads of LDS to a product), 128 x 128 or 64 x 64, the largest of which there are enough.
// In `need`, how many quarters of a round of the compute units that is, for 256 and for 128; a backward call counts both products' tiles.
// Measured, us, with 64 / 128 / 256:
//   forward, sums of 1024: 8192 x 4096 results 165 / 101 / 92, 4096 x 5120 101 / 59 / 75, 4096 x 4096 82 / 45 / 43, 1024 x 2048 10.9 / 14 / 36;
//            sums of 2048: 768 x 4096 28 / 23.5 / 41; sums of 4096 and 8192: 1024 x 2048 31 / 31 / 43 and 57 / 49 / 55
//   both gradients: weights of 768 x 2048, 2048 columns 29 / 26 / 44, 768 x 768, 4096 columns 28 / 24 / 41, 1024 columns 9.8 / 14 / 36;
//            with 128 / 256, tiles of 256: 1024 x 4096, 4096 columns (320) 91 / 104, 2048 x 2048, 8192 columns (320) 142 / 153, 300 x 4200,
//            4531 columns (340) 76 / 108, 2048 x 4096, 4096 columns (384) 157 / 158, 4096 x 4096, 2048 columns (384) 160 / 156,
//            32000 x 768, 4096 columns (423) 486 / 447, 4096 x 4096, 4096 columns (512) 306 / 254
struct Shape { int m, n; };
int tile_for(std::initializer_list<Shape> products, const int (&need)[2]) {
    const size_t cu = g_ctx.num_cu;
    auto enough = [&](int t, int quarters) {
        size_t tiles = 0;
        for (const Shape &p : products) tiles += ceil_div(p.m, t) * ceil_div(p.n, t);
        return 4 * tiles >= quarters * cu;
    };
    return enough(256, need[0]) ? 256 : enough(128, need[1]) ? 128 : 64;
}
// C of M x N from a sum of `sum` terms; `share`: how many compute units' worth of work it should make.
Work work(const Mat &a, const Mat &b, const Epilogue &e, int M, int N, int out_s, int sum, int tile, size_t share) {
    Work w = {};
    w.a = a; w.b = b; w.e = e; w.M = M; w.N = N; w.out_s = out_s; w.sum = sum;
    w.tiles_m = (int)ceil_div(M, tile);
    w.tiles_n = (int)ceil_div(N, tile);
    const size_t tiles = (size_t)w.tiles_m * w.tiles_n, steps = ceil_div(sum, 64);
    // Slices of the sum until every compute unit has work, each with at least four panels of the sum, and only where a workgroup's walk gets
    // 16 panels shorter: joining them is a launch and two ways through memory.  Forward, 1024 x 2048 results, sums of 4096 in two slices 34.6 us and
    // in one 39.8, of 1024 12.0 and 11.3; both gradients of 768 x 768 over 256 columns, in three slices 9.6 us, in one 7.4 to 8.1.
    size_t slices = share / tiles;
    if (slices > steps / 4) slices = steps / 4;
    if (slices < 1 || steps - ceil_div(steps, slices) < 16) slices = 1;
    w.slice_steps = (int)ceil_div(steps, slices);
    slices = ceil_div(steps, w.slice_steps);
    w.units = tiles * slices <= 0xffffff ? (int)(tiles * slices) : -1;
    return w;
}
int slices_of(const Work &w) { return w.M ? w.units / (w.tiles_m * w.tiles_n) : 0; }
size_t part_bytes(const Work &w) { return slices_of(w) > 1 ? ((size_t)slices_of(w) * w.M * w.N * sizeof(float) + 255) & ~(size_t)255 : 0; }

// The products' tensors are direct(); ws: room for the slices of both.
template <int KIND0, int KIND1>
int run(const char *who, Work w0, Work w1, const RowSums &r, int tile, char *ws) {
    if (w0.units < 0 || w1.units < 0) return mi355_fail("%s: too many results", who);
    for (Work *w : {&w0, &w1})
        if (part_bytes(*w)) {
            w->part = (float *)ws;
            ws += part_bytes(*w);
        }
    const unsigned grid = (unsigned)(w0.units + w1.units);
    if (grid > 0x7fffff) return mi355_fail("%s: too many results", who);
    const int one_first = w1.units && w1.slice_steps > w0.slice_steps;
    if (grid) {
        if (tile == 256) linear_kernel<KIND0, KIND1, 256, 256, 128, 64, 2><<<grid, 512, 0, g_ctx.stream>>>(w0, w1, one_first);
        // 128 x 128: with two stages two workgroups share a compute unit, with four one of them reads further ahead.  512 units 25.8 us
        // with two, 31.6 with four; 256 units of twice the sum 28.1 and 26.0.
        else if (tile == 128 && grid > (unsigned)g_ctx.num_cu) linear_kernel<KIND0, KIND1, 128, 128, 64, 32, 2><<<grid, 512, 0, g_ctx.stream>>>(w0, w1, one_first);
        else if (tile == 128) linear_kernel<KIND0, KIND1, 128, 128, 64, 32, 4><<<grid, 512, 0, g_ctx.stream>>>(w0, w1, one_first);
        else linear_kernel<KIND0, KIND1, 64, 64, 32, 32, 4><<<grid, 256, 0, g_ctx.stream>>>(w0, w1, one_first);
        LAUNCH_OK(who);
    }
    // (few results to a sum that is cut into slices: their groups are far from what an int holds)
    const int g0 = w0.part ? (int)ceil_div((size_t)w0.M * ceil_div(w0.N, 8), 256) : 0, g1 = w1.part ? (int)ceil_div((size_t)w1.M * ceil_div(w1.N, 8), 256) : 0;
    const int g2 = (r.M + 3) / 4;
    if (g0 + g1 + g2) {
        linear_join_kernel<KIND0, KIND1><<<(unsigned)(g0 + g1 + g2), 256, 0, g_ctx.stream>>>(w0, w1, r, g0, g1);
        LAUNCH_OK(who);
    }
    return 0;
}

bool sizes_ok(const char *who, int M, int K, int S, int batch, int act) {
    if (M <= 0 || K <= 0 || S <= 0 || batch <= 0) {
        mi355_fail("%s: bad shape M=%d K=%d S=%d batch=%d", who, M, K, S, batch);
        return false;
    }
    if ((double)S * batch > 1 << 22 || M > 1 << 22 || K > 1 << 22) {        // (256 rows of that many values: 32-bit offsets)
        mi355_fail("%s: M, K and batch * S are at most 2^22", who);
        return false;
    }
    if (act < ACT_NONE || act > ACT_GELU) {
        mi355_fail("%s: act=%d (0 none, 1 ReLU, 2 SiLU, 3 GELU)", who, act);
        return false;
    }
    return true;
}

}  // namespace

MI355_API int mi355_linear_fwd_bf16_dev(uint16_t *y, uint16_t *pre, const uint16_t *x, const uint16_t *w, const float *bias, int act,
                                        const uint16_t *res, float alpha, int M, int K, int S, int batch) {
    if (!mi355_ready("linear_fwd_bf16")) return -1;
    if (!y || !x || !w) return mi355_fail("linear_fwd_bf16: NULL pointer");
    if (!sizes_ok("linear_fwd_bf16", M, K, S, batch, act)) return -1;
    Epilogue e = {};
    e.act = act; e.alpha = alpha; e.bias = bias; e.res = res; e.pre_out = pre; e.out = y;
    const int N = batch * S, kpad = (K + 7) & ~7;
    const size_t xs = (size_t)(N <= 1 ? 1 : N <= 2 ? 2 : 4) * kpad * sizeof(float);
    // Few columns: 2048 x 1024 weights and 1, 2, 4 columns 4.6, 4.9 and 7.2 us with gemv_kernel, 10.4 to 10.7 with tiles; 4096 x 4096 and 2 columns
    // 16.2 and 14.8; 2048 x 4096 and 4 columns 20 and 15: it multiplies without the matrix cores.  One column alone has no such clear limit:
    // 4096 x 4096 10.4 and 14.4, 32000 x 768 15.5 and 14.3, 8192 x 4096 16.4 and 18.4, 32000 x 2048 27.5 and 24.5, 151936 x 1024 66 and 116.
    if (N <= GEMV_MAX && (double)M * K * N <= 1 << 24 && xs <= 64 * 1024) {
        // at most four workgroups to a compute unit: each fetches x for itself
        const unsigned grid = (unsigned)(ceil_div(M, 4) < 4 * (size_t)g_ctx.num_cu ? ceil_div(M, 4) : 4 * (size_t)g_ctx.num_cu);
        if (N <= 1) gemv_kernel<1><<<grid, 256, xs, g_ctx.stream>>>(w, x, e, M, K, N, S, kpad);
        else if (N <= 2) gemv_kernel<2><<<grid, 256, xs, g_ctx.stream>>>(w, x, e, M, K, N, S, kpad);
        else gemv_kernel<4><<<grid, 256, xs, g_ctx.stream>>>(w, x, e, M, K, N, S, kpad);
        LAUNCH_OK("linear_fwd_bf16");
        return 0;
    }
    Mat a = {w, M, K, K}, b = {x, K, S, N};
    const int tile = tile_for({{M, N}}, {8, K >= 2048 ? 2 : 3});
    const size_t packed = repacked_bytes(a) + repacked_bytes(b), need = packed + part_bytes(work(a, b, e, M, N, S, K, tile, g_ctx.num_cu));
    char *ws = nullptr;
    if (need && !(ws = (char *)mi355_ws(need))) return -1;
    if (repack("linear_fwd_bf16", a, ws) || repack("linear_fwd_bf16", b, ws)) return -1;
    return run<FORWARD, FORWARD>("linear_fwd_bf16", work(a, b, e, M, N, S, K, tile, g_ctx.num_cu), Work{}, RowSums{}, tile, ws);
}

MI355_API int mi355_linear_bwd_bf16_dev(uint16_t *dx, float *dw, float *dbias, const uint16_t *dy, const uint16_t *x, const uint16_t *w,
                                        float alpha, int act, const uint16_t *x_pre, int accumulate, int M, int K, int S, int batch) {
    if (!mi355_ready("linear_bwd_bf16")) return -1;
    if (!dy || (dx && !w) || (dw && !x) || (!dx && !dw && !dbias)) return mi355_fail("linear_bwd_bf16: NULL pointer");
    if (!sizes_ok("linear_bwd_bf16", M, K, S, batch, act)) return -1;
    if (dx && act != ACT_NONE && !x_pre) return mi355_fail("linear_bwd_bf16: act=%d needs x_pre", act);
    Epilogue e = {};
    e.act = act; e.alpha = alpha; e.pre = x_pre; e.out = dx; e.dw = dw; e.accumulate = accumulate;
    const int N = batch * S;
    Mat g = {dy, M, S, N}, wm = {w, M, K, K}, xm = {x, K, S, N};
    const size_t packed = (dx || dw ? repacked_bytes(g) : 0) + (dx ? repacked_bytes(wm) : 0) + (dw ? repacked_bytes(xm) : 0);
    // both products in one launch and one size of tile; the sum over N columns is as long when they are repacked
    const int tile = tile_for({{dx ? K : 0, dx ? N : 0}, {dw ? M : 0, dw ? K : 0}}, {6, 3});
    auto works = [&](Work &w0, Work &w1) {
        const size_t cu = g_ctx.num_cu;
        w0 = dx ? work(wm, g, e, K, N, S, M, tile, cu) : Work{};
        w1 = dw ? work(g, xm, e, M, K, K, g.cols, tile, cu) : Work{};
    };
    Work w0, w1;
    works(w0, w1);
    const size_t need = packed + part_bytes(w0) + part_bytes(w1);
    char *ws = nullptr;
    if (need && !(ws = (char *)mi355_ws(need))) return -1;
    if ((dx || dw) && repack("linear_bwd_bf16", g, ws)) return -1;
    if (dx && repack("linear_bwd_bf16", wm, ws)) return -1;
    if (dw && repack("linear_bwd_bf16", xm, ws)) return -1;
    works(w0, w1);
    RowSums r = {};
    if (dbias) {
        r.out = dbias; r.dy = dy; r.M = M; r.S = S; r.batch = batch; r.accumulate = accumulate; r.alpha = alpha;
    }
    return run<DX, DW>("linear_bwd_bf16", w0, w1, r, tile, ws);
}

MI355_API int mi355_act_bwd_bf16_dev(uint16_t *dpre, const uint16_t *dy, const uint16_t *pre, float alpha, int act, size_t n) {
    if (!mi355_ready("act_bwd_bf16")) return -1;
    if (!dpre || !dy || !pre) return mi355_fail("act_bwd_bf16: NULL pointer");
    if (act < ACT_NONE || act > ACT_GELU) return mi355_fail("act_bwd_bf16: act=%d (0 none, 1 ReLU, 2 SiLU, 3 GELU)", act);
    if (ceil_div(n, 2048) > 0xffffff) return mi355_fail("act_bwd_bf16: n=%zu is too large", n);
    if (!n) return 0;
    act_bwd_kernel<<<(unsigned)ceil_div(n, 2048), 256, 0, g_ctx.stream>>>(dpre, dy, pre, alpha, act, n);
    LAUNCH_OK("act_bwd_bf16");
    return 0;
}
