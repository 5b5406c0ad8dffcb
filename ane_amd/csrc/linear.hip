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
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }
__device__ __forceinline__ float act_value(int act, float x) {
    if (act == ACT_RELU) return x < 0.f ? 0.f : x;      // (a NaN stays one)
    if (act == ACT_SILU) return x * sigmoid(x);
    if (act == ACT_GELU) return x * sigmoid(2.f * GELU_C * (x + 0.044715f * x * x * x));
    return x;
}
__device__ __forceinline__ float act_slope(int act, float x) {
    if (act == ACT_RELU) return x > 0.f ? 1.f : (x == x ? 0.f : x);
    if (act == ACT_SILU) {
        const float g = sigmoid(x);
        return g * (1.f + x * (1.f - g));
    }
    if (act == ACT_GELU) {
        x = __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, 16.f), -16.f);       // the slope's limits, long reached; x^2 stays finite
        const float g = sigmoid(2.f * GELU_C * (x + 0.044715f * x * x * x));
        return g + x * (2.f * g * (1.f - g)) * GELU_C * (1.f + 0.134145f * x * x);
    }
    return 1.f;
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
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[j] = e.alpha * act_value(e.act, v[j]);
                if (e.res) v[j] += r[j];
            }
        } else {
            float r[8];
            if (e.act != ACT_NONE) ldb<8, true>(r, e.pre + at);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[j] *= e.alpha;
                if (e.act != ACT_NONE) v[j] *= act_slope(e.act, r[j]);
            }
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
            x = e.alpha * act_value(e.act, x);
            if (e.res) x += bf_to_f(e.res[at]);
        } else {
            x *= e.alpha;
            if (e.act != ACT_NONE) x *= act_slope(e.act, bf_to_f(e.pre[at]));
        }
        e.out[at] = (bf16_t)f_to_bf(x);
    }
}

// Rows [row0, row0 + ROWS) and columns [col0, col0 + 64) of a tensor on their way to LDS; zero outside.
template <int ROWS, int THREADS>
struct Stage {
    static constexpr int N = ROWS * 8 / THREADS;
    v4u w[N];
    __device__ __forceinline__ void load(const Mat &a, int row0, int col0) {
        const int chunk = threadIdx.x & 7, col = col0 + chunk * 8;
        const int b = col / a.S, s = col - b * a.S;
        const bf16_t *p = a.p + ((size_t)b * a.rows + row0 + (threadIdx.x >> 3)) * a.S + s;
        const bool vec = s + 8 <= a.S && col < a.cols;
        const int left = a.rows - row0 - (int)(threadIdx.x >> 3);
#pragma unroll
        for (int i = 0; i < N; i++) {
            v4u v = {0u, 0u, 0u, 0u};
            if (i * (THREADS / 8) < left) {
                const bf16_t *q = p + (size_t)(i * (THREADS / 8)) * a.S;
                if (vec) v = *reinterpret_cast<const v4u_any *>(q);
                else if (col < a.cols) v = pieces(a, row0 + (int)(threadIdx.x >> 3) + i * (THREADS / 8), col);
            }
            w[i] = v;
        }
    }
    static __device__ __forceinline__ v4u pieces(const Mat &a, int row, int col) {
        unsigned e[8];
        int b = col / a.S, s = col - b * a.S;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            e[j] = col + j < a.cols ? a.p[((size_t)b * a.rows + row) * a.S + s] : 0u;
            if (++s == a.S) s = 0, b++;
        }
        return v4u{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
    }
    __device__ __forceinline__ void store(char *panel) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int t = threadIdx.x + i * THREADS;
            *reinterpret_cast<v4u *>(panel + panel_at(t >> 3, t & 7)) = w[i];
        }
    }
};

// An operand's 64 steps of the sum for B indexes: by columns B / 64 panels of 64 rows (the sum) x 64 columns, else one of B rows.
template <int B, bool COLUMNS, int THREADS>
struct Operand {
    static constexpr int PANELS = COLUMNS ? B / 64 : 1, ROWS = COLUMNS ? 64 : B, BYTES = B * PANEL_ROW;
    Stage<ROWS, THREADS> s[PANELS];
    __device__ __forceinline__ void load(const Mat &a, int index0, int sum0) {
#pragma unroll
        for (int p = 0; p < PANELS; p++) {
            if (COLUMNS) s[p].load(a, sum0, index0 + p * 64);
            else s[p].load(a, index0, sum0);
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int p = 0; p < PANELS; p++) s[p].store(lds + p * (ROWS * PANEL_ROW));
    }
    // the fragment of indexes block*32 .. +31 at 16 steps of the sum
    static __device__ __forceinline__ M16::Frag frag(const char *lds, int block, int step) {
        if constexpr (COLUMNS) return M16::columns(lds + (block >> 1) * (64 * PANEL_ROW), block & 1, step);
        else return M16::along(lds, block, step);
    }
};

template <int KIND, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(BM / WM *BN / WN * 64) void linear_kernel(Mat a, Mat b, Epilogue e, float *__restrict__ part, int M, int N, int steps,
                                                                       int slice_steps, int tiles_m, int tiles_n) {
    constexpr int WAVES_N = BN / WN, THREADS = BM / WM * WAVES_N * 64, FM = WM / 32, FN = WN / 32;
    typedef Operand<BM, KIND == DX, THREADS> A;
    typedef Operand<BN, KIND != DW, THREADS> B;
    constexpr int PITCH = BN + 8;               // floats between the rows of the tile of C in LDS
    constexpr int TILE = BM * PITCH * 4, PANELS = 2 * (A::BYTES + B::BYTES);
    __shared__ __attribute__((aligned(16))) char lds[TILE > PANELS ? TILE : PANELS];
    const int tile = xcd_remap(blockIdx.x, tiles_m * tiles_n);
    const int m0 = tile % tiles_m * BM, n0 = tile / tiles_m * BN;
    const int i0 = blockIdx.y * slice_steps, i1 = min(steps, i0 + slice_steps);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave / WAVES_N * FM, wn = wave % WAVES_N * FN;

    v16f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = v16_zero();
    A la;
    B lb;
    la.load(a, m0, i0 * 64);
    lb.load(b, n0, i0 * 64);
    la.store(lds);
    lb.store(lds + A::BYTES);
    __syncthreads();
    for (int i = i0; i < i1; i++) {
        const char *at = lds + ((i - i0) & 1) * (A::BYTES + B::BYTES);
        if (i + 1 < i1) {
            la.load(a, m0, (i + 1) * 64);
            lb.load(b, n0, (i + 1) * 64);
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            M16::Frag fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FM; j++) fa[j] = A::frag(at, wm + j, s);
#pragma unroll
            for (int j = 0; j < FN; j++) fb[j] = B::frag(at + A::BYTES, wn + j, s);
#pragma unroll
            for (int j = 0; j < FM; j++)
#pragma unroll
                for (int k = 0; k < FN; k++) acc[j][k] = M16::mul(fa[j], fb[k], acc[j][k]);
        }
        if (i + 1 < i1) {
            char *next = lds + ((i + 1 - i0) & 1) * (A::BYTES + B::BYTES);
            la.store(next);
            lb.store(next + A::BYTES);
        }
        __syncthreads();
    }
    // The tile goes through LDS so that a thread ends with eight columns of one row.
    float *c = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int j = 0; j < FM; j++)
#pragma unroll
        for (int k = 0; k < FN; k++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                c[((wm + j) * 32 + acc_row(r) + 4 * (lane >> 5)) * PITCH + (wn + k) * 32 + (lane & 31)] = acc[j][k][r];
    __syncthreads();
    for (int t = threadIdx.x; t < BM * BN / 8; t += THREADS) {
        const int row = t / (BN / 8), col = t % (BN / 8) * 8, m = m0 + row, n = n0 + col;
        if (m >= M || n >= N) continue;
        float v[8];
        const v4f lo = *reinterpret_cast<const v4f *>(c + row * PITCH + col), hi = *reinterpret_cast<const v4f *>(c + row * PITCH + col + 4);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = lo[j], v[4 + j] = hi[j];
        if (part) {
            float *p = part + ((size_t)blockIdx.y * M + m) * N + n;
            if (n + 8 <= N) st4(p, lo), st4(p + 4, hi);
            else
                for (int j = 0; n + j < N; j++) p[j] = v[j];
        } else finish<KIND>(e, v, m, M, n, N, KIND == DW ? N : b.S);
    }
}

// The slices of a product added up in their order, and its epilogue.
template <int KIND>
__global__ __launch_bounds__(256) void linear_join_kernel(Epilogue e, const float *__restrict__ part, int M, int N, int S, int slices) {
    const int groups = (N + 7) / 8;
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)M * groups) return;
    const int m = (int)(t / groups), n = (int)(t % groups) * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0.f;
    const float *p = part + (size_t)m * N + n;
    if (n + 8 <= N) {
        for (int i = 0; i < slices; i++, p += (size_t)M * N) {
            const v4f a = ld4(p), b = ld4(p + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] += a[j], v[4 + j] += b[j];
        }
    } else {
        for (int i = 0; i < slices; i++, p += (size_t)M * N)
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < N) v[j] += p[j];
    }
    finish<KIND>(e, v, m, M, n, N, S);
}

// dbias[m] (+)= alpha * sum of row m of dy over the batch: a workgroup to a row, a fixed tree.
__global__ __launch_bounds__(256) void row_sum_kernel(float *__restrict__ out, const bf16_t *__restrict__ dy, int M, int S, int batch, float alpha,
                                                      int accumulate) {
    __shared__ float sums[4];
    const int m = blockIdx.x;
    float s = 0.f;
    for (int b = 0; b < batch; b++) {
        const bf16_t *row = dy + ((size_t)b * M + m) * S;
        for (int i = threadIdx.x * 8; i < S; i += 2048) {
            if (i + 8 <= S) {
                float v[8];
                ldb<8, false>(v, row + i);
#pragma unroll
                for (int j = 0; j < 8; j++) s += v[j];
            } else
                for (int j = i; j < S; j++) s += bf_to_f(row[j]);
        }
    }
    s = wave_sum_far_first(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = alpha * (sums[0] + sums[1] + sums[2] + sums[3]);
        out[m] = accumulate ? out[m] + s : s;
    }
}

__global__ __launch_bounds__(256) void act_bwd_kernel(bf16_t *__restrict__ dpre, const bf16_t *__restrict__ dy, const bf16_t *__restrict__ pre,
                                                      float alpha, int act, size_t n) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i + 8 <= n) {
        float g[8], x[8];
        ldb<8, true>(g, dy + i);
        ldb<8, true>(x, pre + i);
#pragma unroll
        for (int j = 0; j < 8; j++) g[j] = alpha * g[j] * act_slope(act, x[j]);
        stb<8>(dpre + i, g);
    } else
        for (size_t j = i; j < n; j++) dpre[j] = (bf16_t)f_to_bf(alpha * bf_to_f(dy[j]) * act_slope(act, bf_to_f(pre[j])));
}

// C of M x N from a sum of `sum` terms.
template <int KIND>
int product(const char *who, const Mat &a, const Mat &b, const Epilogue &e, int M, int N, int sum) {
    const int steps = (int)ceil_div(sum, 64), cu = g_ctx.num_cu;
    const bool big = ceil_div(M, 128) * ceil_div(N, 128) >= (size_t)cu;
    const int tile = big ? 128 : 64;
    const int tm = (int)ceil_div(M, tile), tn = (int)ceil_div(N, tile);
    if ((size_t)tm * tn > 0xffffff) return mi355_fail("%s: %d x %d results are too many", who, M, N);
    // slices of the sum until every compute unit has two workgroups, each with at least four panels of the sum
    int slices = (int)(2 * (size_t)cu / ((size_t)tm * tn));
    if (slices > steps / 4) slices = steps / 4;
    if (slices < 1) slices = 1;
    const int per = (int)ceil_div(steps, slices);
    slices = (int)ceil_div(steps, per);
    float *part = nullptr;
    if (slices > 1) {
        part = (float *)mi355_ws((size_t)slices * M * N * sizeof(float));
        if (!part) return -1;
    }
    const dim3 grid((unsigned)(tm * tn), (unsigned)slices);
    if (big) linear_kernel<KIND, 128, 128, 64, 64><<<grid, 256, 0, g_ctx.stream>>>(a, b, e, part, M, N, steps, per, tm, tn);
    else linear_kernel<KIND, 64, 64, 32, 32><<<grid, 256, 0, g_ctx.stream>>>(a, b, e, part, M, N, steps, per, tm, tn);
    LAUNCH_OK(who);
    if (part) {
        const size_t threads = (size_t)M * ceil_div(N, 8);
        linear_join_kernel<KIND><<<(unsigned)ceil_div(threads, 256), 256, 0, g_ctx.stream>>>(e, part, M, N, KIND == DW ? N : b.S, slices);
        LAUNCH_OK(who);
    }
    return 0;
}

bool sizes_ok(const char *who, int M, int K, int S, int batch, int act) {
    if (M <= 0 || K <= 0 || S <= 0 || batch <= 0) {
        mi355_fail("%s: bad shape M=%d K=%d S=%d batch=%d", who, M, K, S, batch);
        return false;
    }
    if ((double)S * batch > 1 << 30 || M > 1 << 30 || K > 1 << 30) {
        mi355_fail("%s: M, K and batch * S are at most 2^30", who);
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
    const Mat a = {w, M, K, K}, b = {x, K, S, batch * S};
    return product<FORWARD>("linear_fwd_bf16", a, b, e, M, batch * S, K);
}

MI355_API int mi355_linear_bwd_bf16_dev(uint16_t *dx, float *dw, float *dbias, const uint16_t *dy, const uint16_t *x, const uint16_t *w,
                                        float alpha, int act, const uint16_t *x_pre, int accumulate, int M, int K, int S, int batch) {
    if (!mi355_ready("linear_bwd_bf16")) return -1;
    if (!dy || (dx && !w) || (dw && !x) || (!dx && !dw && !dbias)) return mi355_fail("linear_bwd_bf16: NULL pointer");
    if (!sizes_ok("linear_bwd_bf16", M, K, S, batch, act)) return -1;
    if (dx && act != ACT_NONE && !x_pre) return mi355_fail("linear_bwd_bf16: act=%d needs x_pre", act);
    const Mat g = {dy, M, S, batch * S};
    Epilogue e = {};
    e.act = act; e.alpha = alpha; e.pre = x_pre; e.out = dx; e.dw = dw; e.accumulate = accumulate;
    if (dx) {
        const Mat a = {w, M, K, K};
        if (product<DX>("linear_bwd_bf16", a, g, e, K, batch * S, M)) return -1;
    }
    if (dw) {
        const Mat b = {x, K, S, batch * S};
        if (product<DW>("linear_bwd_bf16", g, b, e, M, K, batch * S)) return -1;
    }
    if (dbias) {
        row_sum_kernel<<<(unsigned)M, 256, 0, g_ctx.stream>>>(dbias, dy, M, S, batch, alpha, accumulate);
        LAUNCH_OK("linear_bwd_bf16");
    }
    return 0;
}

MI355_API int mi355_act_bwd_bf16_dev(uint16_t *dpre, const uint16_t *dy, const uint16_t *pre, float alpha, int act, size_t n) {
    if (!mi355_ready("act_bwd_bf16")) return -1;
    if (!dpre || !dy || !pre) return mi355_fail("act_bwd_bf16: NULL pointer");
    if (act < ACT_NONE || act > ACT_GELU) return mi355_fail("act_bwd_bf16: act=%d (0 none, 1 ReLU, 2 SiLU, 3 GELU)", act);
    if (ceil_div(n, 2048) > 0x7fffffff) return mi355_fail("act_bwd_bf16: n=%zu is too large", n);
    if (!n) return 0;
    act_bwd_kernel<<<(unsigned)ceil_div(n, 2048), 256, 0, g_ctx.stream>>>(dpre, dy, pre, alpha, act, n);
    LAUNCH_OK("act_bwd_bf16");
    return 0;
}
