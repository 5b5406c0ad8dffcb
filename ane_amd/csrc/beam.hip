// beam.hip — a step of beam search: the best continuations of each group of beams.
//   candidate (n, v) = score[n] + (x[v][n] - log sum_u exp x[u][n]);  a finished beam has (n, pad) = score[n], and -inf for every other token.
// The `beams` largest of a group, equal ones in the order of (n, v); a NaN counts as -inf.
//
// Two launches.  The first reads the logits once, at the rate of memory, and leaves for every block of rows of a column its largest logit and the
// sum of exponentials.  The second has a workgroup for each group: log sums; the `beams` best blocks by their largest candidates; and
// the best of these blocks' elements, which are read again.  The best `beams` elements lie in the best `beams` blocks, with equal ones in the
// order of their indices in both: each block before another has an element before all of the other's.
// Measured: 64 groups of eight beams over 151936 tokens, bfloat16, 49 us: the logits in 32 (156 MB at 4.85 TB/s; a copy of 1 GiB: 5.1), the selection, 64
// workgroups, in 12; four beams over 32000, fp32, 12 us: 4.7 and 7.8, a chain of a dozen barriers and four trips to memory.
#include "tile.h"

#include <math.h>

namespace {

constexpr int SELECT = 1024;        // threads of a group's workgroup
constexpr int LIST = 512;           // candidates that it ranks
constexpr int NONE = 0x7fffffff;    // no candidate's key
constexpr int MOST = 64;            // beams

template <int VEC> __device__ __forceinline__ void load_vec(float (&r)[VEC], const float *p) {
    if constexpr (VEC == 1) r[0] = __builtin_nontemporal_load(p);
    else ldv_nt<VEC>(r, p);
}
template <int VEC> __device__ __forceinline__ void load_vec(float (&r)[VEC], const bf16_t *p) {
    if constexpr (VEC == 1) r[0] = bf_to_f(__builtin_nontemporal_load(p));
    else ldb<VEC, true>(r, p);
}

// {largest, sum of exp(x - largest)} of two parts; -inf with a sum of 0: nothing.
__device__ __forceinline__ void join(float &m, float &l, float m2, float l2) {
    const float to = fmaxf(m, m2), base = to == -INFINITY ? 0.f : to;
    l = l * exp_neg_fast(m - base) + l2 * exp_neg_fast(m2 - base);
    m = to;
}
// The values of N rows at once.  (fmaxf passes NaNs over; the sum does not, and with it all candidates of the column are NaN.)
template <int N>
__device__ __forceinline__ void take(float &m, float &l, const float (&x)[N]) {
    float top = m;
#pragma unroll
    for (int i = 0; i < N; i++) top = fmaxf(top, x[i]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) sum += exp_neg_fast(x[i] - base);
    l = l * exp_neg_fast(m - base) + sum;
    m = top;
}

// Several columns: threads side by side take VEC columns of a row each (the last ones of a row its last VEC, some of them twice), `across` threads
// to a row; a thread takes every (256 / across)-th of the block's rows, ROWS at a time.  part[block][column].
template <typename T, int VEC>
__global__ __launch_bounds__(256) void beam_columns_kernel(float2 *__restrict__ part, const T *__restrict__ logits, int V, int S, int columns,
                                                           int across, int rows) {
    constexpr int ROWS = 8;
    __shared__ float ms[256 * VEC], ls[256 * VEC];
    const int down = 256 / across, r = threadIdx.x / across, c = threadIdx.x - r * across;
    const int first = blockIdx.x * rows, last = min(first + rows, V);
    const size_t b = blockIdx.z;
    const int col = min(((int)blockIdx.y * across + c) * VEC, S - VEC);
    float m[VEC], l[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) { m[e] = -INFINITY; l[e] = 0.f; }
    if (r < down) {
        const T *x = logits + b * V * S + col;
        for (int v = first + r; v < last; v += ROWS * down) {
            float in[ROWS][VEC];
#pragma unroll
            for (int i = 0; i < ROWS; i++) load_vec<VEC>(in[i], x + (size_t)min(v + i * down, last - 1) * S);
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                float of[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; i++) of[i] = v + i * down < last ? in[i][e] : -INFINITY;
                take(m[e], l[e], of);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) { ms[threadIdx.x * VEC + e] = m[e]; ls[threadIdx.x * VEC + e] = l[e]; }
    // the threads of a column in halves
    for (int n = down; n > 1;) {
        const int half = (n + 1) / 2;
        __syncthreads();
        if (r < n - half) {
            const int at = threadIdx.x * VEC, of = at + half * across * VEC;
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                join(m[e], l[e], ms[of + e], ls[of + e]);
                ms[at + e] = m[e];
                ls[at + e] = l[e];
            }
        }
        n = half;
    }
    if (r == 0)
#pragma unroll
        for (int e = 0; e < VEC; e++) part[(size_t)blockIdx.x * columns + b * S + col + e] = make_float2(m[e], l[e]);
}

// Columns whose logits lie one after the other (S = 1): a wave to a block of 64 * VEC * N rows.
template <typename T, int VEC, int N>
__global__ __launch_bounds__(256) void beam_rows_kernel(float2 *__restrict__ part, const T *__restrict__ logits, int V, int columns, int blocks) {
    constexpr int ROWS = 64 * VEC * N;
    const int block = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (block >= blocks) return;
    const size_t col = blockIdx.y;
    const T *x = logits + col * V;
    float in[N * VEC];
    const int first = block * ROWS;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int v = first + (i * 64 + lane) * VEC;
        float r[VEC];
        if (v + VEC <= V) load_vec<VEC>(r, x + v);
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) r[e] = v + e < V ? load_one(x + v + e) : -INFINITY;
#pragma unroll
        for (int e = 0; e < VEC; e++) in[i * VEC + e] = r[e];
    }
    float m = -INFINITY, l = 0.f;
    take(m, l, in);
    const float top = wave_max(m);
    l = wave_sum_stride<1>(l * exp_neg_fast(m - (top == -INFINITY ? 0.f : top)));
    if (lane == 0) part[(size_t)block * columns + col] = make_float2(top, l);
}

struct SelectLds {
    double lse[MOST], value[SELECT], out_value[MOST];
    int key[SELECT], out_key[MOST], count;
    float tops[64], tau;
    float m[SELECT];
    double l[SELECT];
};
__device__ __forceinline__ bool before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

// -inf.  (The compiler has set a pair of scalar registers to this double with an instruction that holds only 32 bits of it, and they were 0 then;
// here it does not see the constant.)
__device__ __forceinline__ double lowest() {
    float x = -INFINITY;
    asm("" : "+v"(x));
    return x;
}

// All of these are loaded here.  (Else each load is moved to where its value is used, behind a condition, and waited for there.)
__device__ __forceinline__ void loaded(float (&x)[4]) { asm("" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3])); }

// Of this lane's item and that of lane ^ d the lower lane keeps the first, or (back) the last.
__device__ __forceinline__ void first_of_two(double &v, int &k, int d, bool back) {
    const double x = __shfl_xor(v, d, 64);
    const int y = __shfl_xor(k, d, 64);
    if (before(v, k, x, y) != (((threadIdx.x & d) == 0) != back)) { v = x; k = y; }
}

// The `want` first of all threads' items, larger values first, equal ones by their keys: out_value, out_key in order.  own: the largest of the
// thread's items as a float (rounding keeps the order); walk(f) calls f(value, key) for each of them, item(i, load(i), value, key) has the i-th of
// `items`, key -1: none (nor is there one behind the last).
// Of 64 parts of the threads the largest ones are compared; what is not below the `want`-th of these goes into a list, in which every item counts
// those before it.  Few threads have any of those, and only they walk.  (512 at most: 1000 of them take 60 us.)
template <typename F, typename G, typename H>
__device__ __forceinline__ void first_of(SelectLds &lds, int want, float own, F walk, int items, G load, H item) {
    constexpr int PART = SELECT / 64;
    const int tid = threadIdx.x;
    float best = own;
    if constexpr (PART >= 2) best = fmaxf(best, lane_xor<1>(best));
    if constexpr (PART >= 4) best = fmaxf(best, lane_xor<2>(best));
    if constexpr (PART >= 8) best = fmaxf(best, dpp_half_mirror(best));
    if constexpr (PART >= 16) best = fmaxf(best, dpp_row_mirror(best));
    if (tid % PART == 0) lds.tops[tid / PART] = best;
    if (tid == 0) lds.count = 0;
    __syncthreads();
    {
        const float mine = lds.tops[tid / PART];
        float rank = 0.f;
#pragma unroll
        for (int i = 0; i < 64 / PART; i++) {
            const int j = tid % PART * (64 / PART) + i;
            const float t = lds.tops[j];
            rank += t > mine || (t == mine && j < tid / PART) ? 1.f : 0.f;
        }
        if ((int)group_sum<PART>(rank) == want - 1) lds.tau = mine;
    }
    __syncthreads();
    const float tau = lds.tau;
    if (own >= tau) {
        auto put = [&](double v, int k) __attribute__((always_inline)) {
            if ((float)v < tau) return;
            const int at = atomicAdd(&lds.count, 1);
            if (at < LIST) { lds.value[at] = v; lds.key[at] = k; }
        };
        walk(put);
    }
    __syncthreads();
    const int count = lds.count;
    if (count <= LIST) {
        for (int i = tid >> 4; i < count; i += SELECT / 16) {       // 16 threads to an item
            const double v = lds.value[i];
            const int k = lds.key[i];
            float rank = 0.f;
            for (int j = tid & 15; j < count; j += 16) rank += before(lds.value[j], lds.key[j], v, k) ? 1.f : 0.f;
            const int r = (int)group_sum<16>(rank);
            if (r < want && (tid & 15) == 0) { lds.out_value[r] = v; lds.out_key[r] = k; }
        }
    } else {
        // Too many equal ones, or so many of one part's: a wave has the `want` first of its threads' items in order, one to a lane, and brings in those
        // that are before the last of them, few of them one by one; then each counts those before it in all waves' lists.
        const int lane = tid & 63;
        const double low = lowest();
        double held = low, last = low;
        int held_key = NONE, last_key = NONE;
        auto of_lane = [](double x, int from) __attribute__((always_inline)) {
            const long long b = __double_as_longlong(x);
            const unsigned low_half = __builtin_amdgcn_readlane((int)b, from);
            return __longlong_as_double((long long)low_half | (long long)__builtin_amdgcn_readlane((int)(b >> 32), from) << 32);
        };
        constexpr int AT_ONCE = 4;          // items on their way
        for (int i0 = 0; i0 < items; i0 += AT_ONCE) {
            float x[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++) x[i] = load(i0 + i);
            loaded(x);
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++) {
                double v;
                int k;
                item(i0 + i, x[i], v, k);
                const bool in = k >= 0 && before(v, k, last, last_key);
                unsigned long long more = __ballot(in);
                if (__popcll(more) > 8) {
                    v = in ? v : low;
                    k = in ? k : NONE;
#pragma unroll 1
                    for (int size = 2; size <= 64; size *= 2)
#pragma unroll 1
                        for (int d = size / 2; d; d /= 2) first_of_two(v, k, d, (lane & size) != 0);
                    const double x = __shfl(v, 63 - lane, 64);
                    const int y = __shfl(k, 63 - lane, 64);
                    if (before(x, y, held, held_key)) { held = x; held_key = y; }
#pragma unroll 1
                    for (int d = 32; d; d /= 2) first_of_two(held, held_key, d, false);
                    more = 0;
                    last = of_lane(held, want - 1);
                    last_key = __builtin_amdgcn_readlane(held_key, want - 1);
                }
                while (more) {
                    const int from = __builtin_ctzll(more);
                    const double x = of_lane(v, from), above = __shfl_up(held, 1, 64);
                    const int y = __builtin_amdgcn_readlane(k, from), key_above = __shfl_up(held_key, 1, 64);
                    const int rank = __popcll(__ballot(before(held, held_key, x, y)));
                    held = lane > rank ? above : lane == rank ? x : held;
                    held_key = lane > rank ? key_above : lane == rank ? y : held_key;
                    last = of_lane(held, want - 1);
                    last_key = __builtin_amdgcn_readlane(held_key, want - 1);
                    more &= more - 1;
                    more &= __ballot(before(v, k, last, last_key));
                }
            }
        }
        lds.value[tid] = held;
        lds.key[tid] = held_key;
        __syncthreads();
        if (lane < want && held_key != NONE) {
            int rank = 0;
            for (int list = 0; list < SELECT; list += 64) {
                int n = 0;          // of the list, before this one
#pragma unroll
                for (int step = 64; step; step >>= 1)
                    if (n + step <= 64 && before(lds.value[list + n + step - 1], lds.key[list + n + step - 1], held, held_key)) n += step;
                rank += n;
            }
            if (rank < want) { lds.out_value[rank] = held; lds.out_key[rank] = held_key; }
        }
    }
    __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(SELECT) void beam_select_kernel(float *__restrict__ score_out, int *__restrict__ token, int *__restrict__ parent,
                                                             int *__restrict__ done_out, const T *__restrict__ logits, const float *__restrict__ score,
                                                             const int *__restrict__ done, const float2 *__restrict__ part, int blocks, int rows, int V, int S,
                                                             int columns, int beams, int eos, int pad) {
    __shared__ SelectLds lds;
    __shared__ float scores[MOST], tops_of[MOST];
    __shared__ int ended[MOST], beam_of[MOST], row_of[MOST];       // the last two: of the best blocks, whose beams and where they begin
    const int tid = threadIdx.x, first = blockIdx.x * beams;
    if (tid < beams) {
        scores[tid] = score[first + tid];
        ended[tid] = done ? done[first + tid] : 0;
    }
    // A thread keeps to one beam: every (SELECT / beams)-th of its blocks.
    const int side = SELECT / beams, beam = tid % beams, step = tid / beams;
    float m = -INFINITY, tops[8];       // tops: of its first eight
    double l = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) tops[i] = -INFINITY;
    if (step < side)
        for (int b = step; b < blocks; b += 8 * side) {
            float2 p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = part[(size_t)min(b + i * side, blocks - 1) * columns + first + beam];
            if (b == step)
#pragma unroll
                for (int i = 0; i < 8; i++) tops[i] = p[i].x;
            float to = m;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (b + i * side < blocks) to = fmaxf(to, p[i].x);
            const float base = to == -INFINITY ? 0.f : to;
            l *= (double)exp_neg_fast(m - base);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (b + i * side < blocks) l += (double)p[i].y * (double)exp_neg(p[i].x - base);
            m = to;
        }
    lds.m[tid] = m;
    lds.l[tid] = l;
    __syncthreads();
    for (int n = tid >> 6; n < beams; n += SELECT / 64) {
        float top = -INFINITY;
        double sum = 0.0;
        for (int i = tid & 63; i < side; i += 64) top = fmaxf(top, lds.m[i * beams + n]);
        top = wave_max(top);
        const float base = top == -INFINITY ? 0.f : top;
        for (int i = tid & 63; i < side; i += 64) sum += lds.l[i * beams + n] * (double)exp_neg(lds.m[i * beams + n] - base);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
        if ((tid & 63) == 0) { lds.value[n] = sum; tops_of[n] = top; }
    }
    __syncthreads();
    if (tid < beams) lds.lse[tid] = (double)tops_of[tid] + log(lds.value[tid]);        // (one wave's work, for all beams)
    __syncthreads();
    const double none = lowest();
    auto candidate = [&](int n, float x, bool is_pad) __attribute__((always_inline)) {
        const double s = scores[n];
        double c = ended[n] ? (is_pad ? s : none) : s + ((double)x - lds.lse[n]);
        return c == c ? c : none;
    };
    // the best blocks, as many as beams (each beam has one at least); of a beam's candidates the one with the largest logit is the largest, but an
    // ended beam has only one
    const int pad_block = pad / rows;
    float own = -INFINITY;
    if (step < side && (!ended[beam] || pad_block % side == step)) own = (float)candidate(beam, m, true);
    first_of(lds, beams, own, [&](auto f) __attribute__((always_inline)) {
        if (step >= side) return;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i * side < blocks && step + i * side < blocks) f(candidate(beam, tops[i], step + i * side == pad_block), beam * blocks + step + i * side);
        for (int b = step + 8 * side; b < blocks; b += side)
            f(candidate(beam, part[(size_t)b * columns + first + beam].x, b == pad_block), beam * blocks + b);
    }, (blocks + side - 1) / side,
    [&](int i) __attribute__((always_inline)) { return part[(size_t)min(step + i * side, blocks - 1) * columns + first + beam].x; },
    [&](int i, float x, double &v, int &k) __attribute__((always_inline)) {
        const int b = step + i * side;
        v = candidate(beam, x, b == pad_block);
        k = step < side && b < blocks ? beam * blocks + b : -1;
    });
    if (tid < beams) {
        const int n = lds.out_key[tid] / blocks;
        beam_of[tid] = n;
        row_of[tid] = (lds.out_key[tid] - n * blocks) * rows;
    }
    __syncthreads();
    // the best of their elements
    {
        constexpr int N = 4;
        const int n_elements = beams * rows;          // (at most 2^19: 64 blocks of 8192 rows)
        const float per_row = 1.f / rows;
        double value[N];
        int key[N];
        auto place = [&](int i, int &n, int &row) __attribute__((always_inline)) {
            const int at = min(i, n_elements - 1);
            int j = (int)((float)at * per_row);             // at / rows, or one off
            j -= j * rows > at;
            j += (j + 1) * rows <= at;
            n = beam_of[j];
            row = row_of[j] + (at - j * rows);
        };
        auto load_from = [&](int n, int row) __attribute__((always_inline)) {
            const int col = first + n, b = S == 1 ? col : col / S;
            return load_one(logits + ((size_t)b * V + min(row, V - 1)) * S + (col - b * S));
        };
        auto element_of = [&](int i, int n, int row, float x, double &v, int &k) __attribute__((always_inline)) {
            v = candidate(n, x, row == pad);
            k = tid + i * SELECT < n_elements && row < V ? n * V + row : -1;
        };
        auto load = [&](int i) __attribute__((always_inline)) {
            int n, row;
            place(tid + i * SELECT, n, row);
            return load_from(n, row);
        };
        auto element = [&](int i, float x, double &v, int &k) __attribute__((always_inline)) {
            int n, row;
            place(tid + i * SELECT, n, row);
            element_of(i, n, row, x, v, k);
        };
        const int items = (n_elements + SELECT - 1) / SELECT;
        float x[N];
        int n[N], row[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (i < items) place(tid + i * SELECT, n[i], row[i]);
            x[i] = i < items ? load_from(n[i], row[i]) : 0.f;
        }
        own = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; i++) {
            key[i] = -1;
            if (i < items) element_of(i, n[i], row[i], x[i], value[i], key[i]);
            if (key[i] >= 0) own = fmaxf(own, (float)value[i]);
        }
        auto rest = [&](auto f) __attribute__((always_inline)) {
            for (int i0 = N; i0 < items; i0 += N) {
                float x[N];
#pragma unroll
                for (int i = 0; i < N; i++) x[i] = load(i0 + i);
                loaded(x);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    double v;
                    int k;
                    element(i0 + i, x[i], v, k);
                    if (k >= 0) f(v, k);
                }
            }
        };
        rest([&](double v, int) __attribute__((always_inline)) { own = fmaxf(own, (float)v); });
        first_of(lds, beams, own, [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i < items && key[i] >= 0) f(value[i], key[i]);
            rest(f);
        }, items, load, element);
    }
    if (tid < beams) {
        const int n = lds.out_key[tid] / V, v = lds.out_key[tid] - n * V;
        score_out[first + tid] = (float)lds.out_value[tid];
        token[first + tid] = v;
        parent[first + tid] = first + n;
        if (done_out) done_out[first + tid] = ended[n] || v == eos;
    }
}

// Rows to a block, and the first launch.
template <typename T>
int beam_blocks(const char *who, float2 **part, int *blocks, int *rows, const T *logits, int V, int S, int batch, int beams) {
    constexpr int WIDE = 16 / (int)sizeof(T);
    const size_t columns = (size_t)S * batch;
    if (S == 1) {
        auto go = [&](auto loads) {
            constexpr int N = decltype(loads)::value;
            *rows = 64 * WIDE * N;
            *blocks = (int)ceil_div(V, *rows);
            *part = (float2 *)mi355_ws(*blocks * columns * sizeof(float2));
            if (!*part) return -1;
            for (size_t c = 0; c < columns; c += 65535) {
                const unsigned n = (unsigned)(columns - c < 65535 ? columns - c : 65535);
                beam_rows_kernel<T, WIDE, N><<<dim3((unsigned)ceil_div(*blocks, 4), n), 256, 0, g_ctx.stream>>>(*part + c, logits + c * V, V, (int)columns,
                                                                                                                      *blocks);
                LAUNCH_OK(who);
            }
            return 0;
        };
        // a launch of eight workgroups and more to a compute unit can have longer blocks
        const size_t waves = columns * ceil_div(V, 64 * WIDE);
        if (waves >= 4 * 16 * (size_t)g_ctx.num_cu) return go(std::integral_constant<int, 2>());
        return go(std::integral_constant<int, 1>());
    }
    auto go = [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        const int threads = (int)ceil_div(S, VEC), across = threads < 64 ? threads : 64, strips = (int)ceil_div(threads, across), down = 256 / across;
        // rows to a thread: eight at a time, more where there are workgroups enough
        const size_t steps = ceil_div(V, down), each = steps * strips * batch / (4 * (size_t)g_ctx.num_cu);
        *rows = down * (each >= 32 && down <= 8 ? 64 : each >= 32 ? 32 : each >= 16 ? 16 : each >= 8 ? 8 : each >= 4 ? 4 : each >= 2 ? 2 : 1);
        // The second launch looks at all blocks of a group, and then at as many blocks' rows as it has beams.  us, 4 / 1 blocks to a row at most / any number:
        // 32000 tokens, 64 beams 48 / 69 / 75, 50257, 32 beams 25 / 27 / 43, 16 beams 16.8 / 16.8 / 20.7, 151936, 64 beams 77 / 129 / 75, four beams 12.2 / - / 13.0.
        while (beams >= 4 && ceil_div(V, *rows) > 4 * (size_t)*rows) *rows *= 2;
        *blocks = (int)ceil_div(V, *rows);
        *part = (float2 *)mi355_ws(*blocks * columns * sizeof(float2));
        if (!*part) return -1;
        for (int b = 0; b < batch; b += 65535) {
            const unsigned n = (unsigned)(batch - b < 65535 ? batch - b : 65535);
            beam_columns_kernel<T, VEC><<<dim3((unsigned)*blocks, (unsigned)strips, n), 256, 0, g_ctx.stream>>>(
                *part + (size_t)b * S, logits + (size_t)b * V * S, V, S, (int)columns, across, *rows);
            LAUNCH_OK(who);
        }
        return 0;
    };
    if (S >= WIDE) return go(std::integral_constant<int, WIDE>());
    return go(std::integral_constant<int, 1>());
}

template <typename T>
int beam_step(const char *who, float *score_out, int32_t *token, int32_t *parent, int32_t *done_out, const T *logits, const float *score,
              const int32_t *done, int V, int S, int batch, int beams, int eos, int pad) {
    if (!score_out || !token || !parent || !logits || !score) return mi355_fail("%s: NULL pointer", who);
    if (V <= 0 || S <= 0 || batch <= 0 || beams <= 0 || beams > MOST || (double)S * batch >= 1 << 22 || (double)V * beams > 1 << 30)
        return mi355_fail("%s: bad shape V=%d S=%d batch=%d beams=%d (at most 64; batch * S below 2^22, V * beams at most 2^30)", who, V, S, batch, beams);
    if (S * batch % beams) return mi355_fail("%s: %d columns are no multiple of beams=%d", who, S * batch, beams);
    if (pad < 0 || pad >= V || eos >= V) return mi355_fail("%s: pad=%d or eos=%d is no token of %d", who, pad, eos, V);
    if (score_out == score || (done_out && done_out == done)) return mi355_fail("%s: the new scores and marks must not be the old ones", who);
    if (!mi355_ready(who)) return -1;
    const size_t n = (size_t)S * batch;
    float2 *part;
    int blocks, rows;
    if (beam_blocks(who, &part, &blocks, &rows, logits, V, S, batch, beams)) return -1;
    beam_select_kernel<T><<<(unsigned)(n / beams), SELECT, 0, g_ctx.stream>>>(score_out, token, parent, done_out, logits, score, done, part, blocks, rows, V, S,
                                                                             (int)n, beams, eos, pad);
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
