// beam.hip — a step of beam search: the best continuations of each group of beams.
//   candidate (n, v) = score[n] + (x[v][n] - log sum_u exp x[u][n]);  a finished beam has (n, pad) = score[n], and -inf for every other token.
// The `beams` largest of a group, equal ones in the order of (n, v); a NaN counts as -inf.
#include "tile.h"

#include <math.h>

namespace {

__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const bf16_t *p) { return bf_to_f(*p); }

// A workgroup to a column: max and log of the sum of exponentials.
template <typename T>
__global__ __launch_bounds__(256) void beam_lse_kernel(double *__restrict__ lse, const T *__restrict__ logits, int V, int S) {
    __shared__ float ms[4];
    __shared__ double ls[4];
    const size_t col = blockIdx.x, b = col / S;
    const T *x = logits + b * V * S + (col - b * S);
    float m = -INFINITY;
    for (int v = threadIdx.x; v < V; v += 256) m = __builtin_elementwise_maximum(m, load_one(x + (size_t)v * S));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, d, 64));
    if ((threadIdx.x & 63) == 0) ms[threadIdx.x >> 6] = m;
    __syncthreads();
    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(ms[0], ms[1]), __builtin_elementwise_maximum(ms[2], ms[3]));
    double l = 0.0;
    for (int v = threadIdx.x; v < V; v += 256) l += exp_neg(load_one(x + (size_t)v * S) - m);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
    if ((threadIdx.x & 63) == 0) ls[threadIdx.x >> 6] = l;
    __syncthreads();
    if (threadIdx.x == 0) lse[col] = (double)m + log(ls[0] + ls[1] + ls[2] + ls[3]);
}

// A candidate in the order of the search: larger values first, then lower indices.
struct Candidate { double value; int index; };
__device__ __forceinline__ bool before(const Candidate &a, const Candidate &b) { return a.value > b.value || (a.value == b.value && a.index < b.index); }

// A workgroup to a group: one walk over its candidates for each of the beams.
template <typename T>
__global__ __launch_bounds__(256) void beam_select_kernel(float *__restrict__ score_out, int *__restrict__ token, int *__restrict__ parent,
                                                          int *__restrict__ done_out, const T *__restrict__ logits, const float *__restrict__ score,
                                                          const int *__restrict__ done, const double *__restrict__ lse, int V, int S, int beams, int eos,
                                                          int pad) {
    __shared__ Candidate best[4];
    const int first = blockIdx.x * beams;
    Candidate last = {INFINITY, -1};
    for (int i = 0; i < beams; i++) {
        Candidate mine = {-INFINITY, 0x7fffffff};
        for (int j = threadIdx.x; j < beams * V; j += 256) {
            const int n = first + j / V, v = j % V;
            const size_t b = n / S;
            double c = (double)score[n];
            if (done && done[n]) c = v == pad ? c : -INFINITY;
            else c = c + ((double)load_one(logits + (b * V + v) * S + (n - b * S)) - lse[n]);
            if (c != c) c = -INFINITY;
            const Candidate it = {c, j};
            if (before(last, it) && before(it, mine)) mine = it;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const Candidate o = {__shfl_xor(mine.value, d, 64), __shfl_xor(mine.index, d, 64)};
            if (before(o, mine)) mine = o;
        }
        if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = mine;
        __syncthreads();
        last = best[0];
#pragma unroll
        for (int w = 1; w < 4; w++)
            if (before(best[w], last)) last = best[w];
        __syncthreads();
        if (threadIdx.x == 0) {
            const int n = first + last.index / V, v = last.index % V;
            score_out[first + i] = (float)last.value;
            token[first + i] = v;
            parent[first + i] = n;
            if (done_out) done_out[first + i] = (done && done[n]) || v == eos;
        }
    }
}

template <typename T>
int beam_step(const char *who, float *score_out, int32_t *token, int32_t *parent, int32_t *done_out, const T *logits, const float *score,
              const int32_t *done, int V, int S, int batch, int beams, int eos, int pad) {
    if (!score_out || !token || !parent || !logits || !score) return mi355_fail("%s: NULL pointer", who);
    if (V <= 0 || S <= 0 || batch <= 0 || beams <= 0 || beams > 64 || (double)S * batch > 1 << 22 || (double)V * beams >= 2147483648.0)
        return mi355_fail("%s: bad shape V=%d S=%d batch=%d beams=%d (at most 64; batch * S at most 2^22, V * beams below 2^31)", who, V, S, batch, beams);
    if (S * batch % beams) return mi355_fail("%s: %d columns are no multiple of beams=%d", who, S * batch, beams);
    if (pad < 0 || pad >= V || eos >= V) return mi355_fail("%s: pad=%d or eos=%d is no token of %d", who, pad, eos, V);
    if (score_out == score || (done_out && done_out == done)) return mi355_fail("%s: the new scores and marks must not be the old ones", who);
    if (!mi355_ready(who)) return -1;
    const size_t n = (size_t)S * batch;
    double *lse = (double *)mi355_ws(n * sizeof(double));
    if (!lse) return -1;
    beam_lse_kernel<T><<<(unsigned)n, 256, 0, g_ctx.stream>>>(lse, logits, V, S);
    LAUNCH_OK(who);
    beam_select_kernel<T><<<(unsigned)(n / beams), 256, 0, g_ctx.stream>>>(score_out, token, parent, done_out, logits, score, done, lse, V, S, beams, eos, pad);
    LAUNCH_OK(who);
    return 0;
}

}  // namespace

MI355_API int mi355_beam_step_dev(float *score_out, int32_t *token, int32_t *parent, int32_t *done_out, const float *logits, const float *score,
                                  const int32_t *done, int V, int S, int batch, int beams, int eos, int pad) {
    return beam_step<float>("beam_step", score_out, token, parent, done_out, logits, score, done, V, S, batch, beams, eos, pad);
}
MI355_API int mi355_beam_step_bf16_dev(float *score_out, int32_t *token, int32_t *parent, int32_t *done_out, const uint16_t *logits, const float *score,
                                       const int32_t *done, int V, int S, int batch, int beams, int eos, int pad) {
    return beam_step<bf16_t>("beam_step_bf16", score_out, token, parent, done_out, logits, score, done, V, S, batch, beams, eos, pad);
}
