// kv_cache.hip — a paged cache of keys and values: new positions are appended, rows of the table follow the beams of a search.
// No counterpart in the reference, whose loops train.  The norm and the rotation are those of qknorm_rope.hip and rope.h, at positions that
// are read from memory.
#include "kv_cache.h"

namespace {

// 16 bytes of a row, and their values
__device__ __forceinline__ v4f raw_cols(const float *p) { return ld4(p); }
__device__ __forceinline__ v4u raw_cols(const bf16_t *p) { return *reinterpret_cast<const v4u_any *>(p); }
__device__ __forceinline__ void widen(float (&r)[4], v4f w) {
#pragma unroll
    for (int j = 0; j < 4; j++) r[j] = w[j];
}
__device__ __forceinline__ void widen(float (&r)[8], v4u w) {
#pragma unroll
    for (int j = 0; j < 4; j++) { r[2 * j] = bf_to_f(w[j] & 0xffffu); r[2 * j + 1] = bf_to_f(w[j] >> 16); }
}
template <int VEC> __device__ __forceinline__ void store_cols(float *p, const float (&r)[VEC]) { stv<VEC>(p, r); }
template <int VEC> __device__ __forceinline__ void store_cols(bf16_t *p, const float (&r)[VEC]) { stb<VEC>(p, r); }
typedef unsigned bf_pair __attribute__((ext_vector_type(1)));
typedef unsigned f_pair __attribute__((ext_vector_type(2)));
__device__ __forceinline__ bf_pair pair_of(float a, float b, bf16_t *) { return bf_pair(f2_to_bf2(a, b)); }
__device__ __forceinline__ f_pair pair_of(float a, float b, float *) { return f_pair{__float_as_uint(a), __float_as_uint(b)}; }

// What a column is a token of: the row of its page and of head 0, -1 if it is none.
__device__ __forceinline__ long long token_row(const int *seq, const int *pages, size_t col, int pos, int n_pages, int page, int n_seqs, int max_pages,
                                               int kv_heads, int positions) {
    const long long entry = paged_entry(seq ? seq[col] : (int)col, pos, n_seqs, max_pages, page);
    if (entry < 0 || pos >= positions) return -1;
    const int id = pages[entry];
    return paged_id_ok(id, n_pages) ? (long long)paged_row(id, 0, pos % page, kv_heads, page, 1) : -1;
}

// A wave to a head of a column, a pair of channels to a lane.  64 new tokens, 16 + 8 + 8 heads of 128, bfloat16: 6.0 us of which an empty launch takes 5.
template <typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(
    T *q_out, const T *q, const T *__restrict__ k, const T *__restrict__ v, T *__restrict__ k_cache, T *__restrict__ v_cache,
    const int *__restrict__ pages, const int *__restrict__ seq, const int *__restrict__ pos_of, const float *__restrict__ wq, const float *__restrict__ wk,
    const float *__restrict__ cos_t, const float *__restrict__ sin_t, int n_pages, int page, int n_seqs, int max_pages, int kv_heads, int hd, int heads, int S,
    int table, float eps, int columns) {
    const int lane = threadIdx.x & 63, slabs = heads + 2 * kv_heads, half = hd / 2;
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int col = (int)(unit / slabs), slab = (int)(unit - (size_t)col * slabs);
    if (col >= columns) return;
    const int b = col / S, s = col - b * S, pos = pos_of[col];
    const long long place = token_row(seq, pages, col, pos, n_pages, page, n_seqs, max_pages, kv_heads, cos_t ? table : 0x7fffffff);
    if (place < 0) return;
    const bool is_q = slab < heads, is_k = !is_q && slab < heads + kv_heads;
    const int head = is_q ? slab : is_k ? slab - heads : slab - heads - kv_heads;
    const T *in = (is_q ? q : is_k ? k : v) + ((size_t)b * (is_q ? heads : kv_heads) + head) * hd * S + s;
    const float *w = is_q ? wq : is_k ? wk : nullptr;
    const bool mine = lane < half;
    float x0 = 0.f, x1 = 0.f;
    if (mine) {
        x0 = load_one(in + (size_t)(2 * lane) * S);
        x1 = load_one(in + (size_t)(2 * lane + 1) * S);
    }
    if (w) {
        const float rr = 1.f / sqrtf(wave_sum_stride<1>(x0 * x0 + x1 * x1) * (1.f / hd) + eps);
        if (mine) {
            x0 = (x0 * rr) * w[2 * lane];
            x1 = (x1 * rr) * w[2 * lane + 1];
        }
    }
    if (!mine) return;
    if ((is_q || is_k) && cos_t) {
        const float cs = cos_t[(size_t)lane * table + pos], sn = sin_t[(size_t)lane * table + pos];
        const float y0 = x0 * cs - x1 * sn, y1 = x0 * sn + x1 * cs;
        x0 = y0;
        x1 = y1;
    }
    if (is_q) {
        T *out = q_out + ((size_t)b * heads + head) * hd * S + s;
        store_one(out + (size_t)(2 * lane) * S, x0);
        store_one(out + (size_t)(2 * lane + 1) * S, x1);
    } else {
        T *out = (is_k ? k_cache : v_cache) + (size_t)(place + head * page) * hd;
        store_one(out + 2 * lane, x0);
        store_one(out + 2 * lane + 1, x1);
    }
}

// Columns side by side: a workgroup has 64 of them and some of the heads.  As in qknorm_rope.hip a thread has whole row pairs of VEC columns, so the
// rotation needs no other lane; the angles of its pairs and columns stay in registers for all the heads.  Rotated queries go back as they came.
// A key or value is a row of the cache: 64 x hd values are turned round in LDS, 16 bytes of a row to a lane on the way out.  Chunks of 4 (fp32) or 8
// pairs of a row are exchanged by the group of columns, so that neither side meets a bank twice.
// 16 padded prompts of 256 positions, 16 + 8 + 8 heads of 128, bfloat16: 15 us (25 MB); one of 8191, 12 + 12 + 12 heads of 64, fp32: 40 us (153 MB, 3.8
// TB/s).  What bounds it is the work of a wave on a head, 2.3 us alone on its SIMD, and 4 us until it has its angles.
// (With 16 columns to a wave, each by itself and without barriers: as long for these, four prompts of 4096 60 us for 40, since a wave's loads are then
// of 32 bytes of each row.)
template <typename P>
__device__ __forceinline__ P of_kind(bool is_q, bool is_k, P q, P k, P v) { return is_q ? q : is_k ? k : v; }
// A head of the queries, the keys or the values, one after the other.
template <typename T> struct Slab { bool is_q, is_k; int head, heads; const T *in; };
template <typename T>
__device__ __forceinline__ Slab<T> slab_of(int i, int heads, int kv_heads, const T *q, const T *k, const T *v) {
    Slab<T> s;
    s.is_q = i < heads;
    s.is_k = !s.is_q && i < heads + kv_heads;
    s.head = i - (s.is_q ? 0 : s.is_k ? heads : heads + kv_heads);
    s.heads = s.is_q ? heads : kv_heads;
    s.in = of_kind(s.is_q, s.is_k, q, k, v);
    return s;
}
template <typename T, int CAP, int PPS, typename Raw>
__device__ __forceinline__ void load_slab(Raw (&r0)[CAP], Raw (&r1)[CAP], const Slab<T> s, int b, int hd, int S, int col, int p0, bool ok) {
    const T *in = s.in + ((size_t)b * s.heads + s.head) * hd * S + col;
#pragma unroll
    for (int kk = 0; kk < CAP; kk++) {
        const int rp = p0 + kk * PPS;
        r0[kk] = r1[kk] = Raw(0);
        if (2 * rp < hd && ok) {
            r0[kk] = raw_cols(in + (size_t)(2 * rp) * S);
            r1[kk] = raw_cols(in + (size_t)(2 * rp + 1) * S);
        }
    }
}
template <typename T> constexpr int PAIRS_AT_ONCE = 256 * 16 / (int)sizeof(T) / 64;

template <typename T, int CAP>
__global__ __launch_bounds__(256) void kv_append_tile_kernel(
    T *q_out, const T *q, const T *__restrict__ k, const T *__restrict__ v, T *__restrict__ k_cache, T *__restrict__ v_cache,
    const int *__restrict__ pages, const int *__restrict__ seq, const int *__restrict__ pos_of, const float *__restrict__ wq, const float *__restrict__ wk,
    const float *__restrict__ cos_t, const float *__restrict__ sin_t, int n_pages, int page, int n_seqs, int max_pages, int kv_heads, int hd, int heads, int S,
    int table, float eps, int tiles, int slabs_each, int all_tiles) {
    constexpr int VEC = 16 / (int)sizeof(T), LPR = 64 / VEC, PPS = 256 / LPR, ROW = 64;        // row pairs: of a step, of a column in LDS
    typedef unsigned pair_t __attribute__((ext_vector_type(sizeof(T) / 2)));                  // a column's values of a row pair
    __shared__ __attribute__((aligned(16))) pair_t turned[64 * ROW];
    __shared__ float sums[4 * LPR * VEC];
    __shared__ long long place[64];         // row of head 0, -1: no token
    __shared__ int at[64];
    const int tid = threadIdx.x, half = hd / 2;
    // The last tiles of padded prompts are empty, and should not be those of the same XCDs for every group of heads: in a batch each group begins at another
    // tile (16 prompts of 256 positions 20 -> 15 us).  A single row does not: an XCD then has its own tiles' angles only (one of 8191 42.7 -> 40).
    const int group = blockIdx.x / all_tiles, turn = blockIdx.x - group * all_tiles + (all_tiles > tiles ? group % all_tiles : 0);
    const int tile = turn >= all_tiles ? turn - all_tiles : turn, b = tile / tiles, s0 = (tile - b * tiles) * 64;
    bool some = false;
    if (tid < 64) {
        long long p = -1;
        int pos = 0;
        if (s0 + tid < S) {
            const size_t col = (size_t)b * S + s0 + tid;
            pos = pos_of[col];
            p = token_row(seq, pages, col, pos, n_pages, page, n_seqs, max_pages, kv_heads, cos_t ? table : 0x7fffffff);
        }
        place[tid] = p;
        at[tid] = p < 0 ? 0 : pos;
        some = p >= 0;
    }
    if (!__syncthreads_or(some)) return;        // (the end of a padded prompt)
    const int lc = tid % LPR, p0 = tid / LPR;
    const LaneCols mine = lane_cols<VEC>(s0 + lc * VEC, S);
    // the lane's columns that are its own, and tokens
    bool own[VEC], all = true, in_a_row = true;
    int pos[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const int c = mine.col + j - s0;
        own[j] = mine.ok && j >= mine.dup && place[max(c, 0)] >= 0;
        pos[j] = own[j] ? at[c] : 0;
        all &= own[j];
        in_a_row &= pos[j] == pos[0] + j;
    }
    float cs[CAP][VEC], sn[CAP][VEC];
    if (cos_t) {
#pragma unroll
        for (int kk = 0; kk < CAP; kk++) {
            const int rp = min(p0 + kk * PPS, half - 1);
            const float *pc = cos_t + (size_t)rp * table, *ps = sin_t + (size_t)rp * table;
            if (in_a_row) {
#pragma unroll
                for (int j = 0; j < VEC; j += 4) {
                    const v4f x = ld4(pc + pos[0] + j), y = ld4(ps + pos[0] + j);
#pragma unroll
                    for (int e = 0; e < 4; e++) { cs[kk][j + e] = x[e]; sn[kk][j + e] = y[e]; }
                }
            } else
#pragma unroll
                for (int j = 0; j < VEC; j++) { cs[kk][j] = pc[pos[j]]; sn[kk][j] = ps[pos[j]]; }
        }
    }
    const int slabs = heads + 2 * kv_heads, first = group * slabs_each, last = min(first + slabs_each, slabs);
    // (weights from memory inside the loop would have it wait for the next head's values too, which are asked for before them)
    float gq[2 * CAP], gk[2 * CAP];
#pragma unroll
    for (int kk = 0; kk < CAP; kk++) {
        const int rp = min(p0 + kk * PPS, half - 1);
        gq[2 * kk] = wq ? wq[2 * rp] : 0.f;
        gq[2 * kk + 1] = wq ? wq[2 * rp + 1] : 0.f;
        gk[2 * kk] = wk ? wk[2 * rp] : 0.f;
        gk[2 * kk + 1] = wk ? wk[2 * rp + 1] : 0.f;
    }
    // the next head's values are under way while one is worked on
    typedef decltype(raw_cols((const T *)nullptr)) Raw;
    Raw r0[CAP], r1[CAP];
    load_slab<T, CAP, PPS>(r0, r1, slab_of(first, heads, kv_heads, q, k, v), b, hd, S, mine.col, p0, mine.ok);
    for (int slab = first; slab < last; slab++) {
        const Slab<T> now = slab_of(slab, heads, kv_heads, q, k, v);
        const bool is_q = now.is_q, is_k = now.is_k;
        const int head = now.head;
        const bool norm = is_q ? wq != nullptr : is_k && wk != nullptr;
        float x0[CAP][VEC], x1[CAP][VEC];
#pragma unroll
        for (int kk = 0; kk < CAP; kk++) { widen(x0[kk], r0[kk]); widen(x1[kk], r1[kk]); }
        if (slab + 1 < last) load_slab<T, CAP, PPS>(r0, r1, slab_of(slab + 1, heads, kv_heads, q, k, v), b, hd, S, mine.col, p0, mine.ok);
        __syncthreads();            // (everybody is done with LDS)
        if (norm) {
            float acc[1][VEC];
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                acc[0][j] = 0.f;
#pragma unroll
                for (int kk = 0; kk < CAP; kk++) { acc[0][j] += x0[kk][j] * x0[kk][j]; acc[0][j] += x1[kk][j] * x1[kk][j]; }
            }
            // the column's sum: over the wave's lanes, then over the waves by one thread to a column, which takes the root for all
#pragma unroll
            for (int j = 0; j < VEC; j++) acc[0][j] = wave_sum_stride<LPR>(acc[0][j]);
            if ((tid & 63) < LPR)
#pragma unroll
                for (int j = 0; j < VEC; j++) sums[(tid >> 6) * 64 + lc * VEC + j] = acc[0][j];
            __syncthreads();
            if (tid < 64) sums[tid] = 1.f / sqrtf((((sums[tid] + sums[64 + tid]) + sums[128 + tid]) + sums[192 + tid]) * (1.f / hd) + eps);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VEC; j++) acc[0][j] = sums[lc * VEC + j];
#pragma unroll
            for (int kk = 0; kk < CAP; kk++) {
                const float w0 = is_q ? gq[2 * kk] : gk[2 * kk], w1 = is_q ? gq[2 * kk + 1] : gk[2 * kk + 1];
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    x0[kk][j] = (x0[kk][j] * acc[0][j]) * w0;
                    x1[kk][j] = (x1[kk][j] * acc[0][j]) * w1;
                }
            }
        }
        if ((is_q || is_k) && cos_t) {
#pragma unroll
            for (int kk = 0; kk < CAP; kk++)
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float y0 = x0[kk][j] * cs[kk][j] - x1[kk][j] * sn[kk][j];
                    x1[kk][j] = x0[kk][j] * sn[kk][j] + x1[kk][j] * cs[kk][j];
                    x0[kk][j] = y0;
                }
        }
        if (is_q) {
#pragma unroll
            for (int kk = 0; kk < CAP; kk++) {
                const int rp = p0 + kk * PPS;
                if (rp >= half) continue;
                T *out = q_out + (((size_t)b * heads + head) * hd + 2 * rp) * S + mine.col;
                if (all) {
                    store_cols<VEC>(out, x0[kk]);
                    store_cols<VEC>(out + S, x1[kk]);
                } else
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        if (own[j]) {
                            store_one(out + j, x0[kk][j]);
                            store_one(out + S + j, x1[kk][j]);
                        }
            }
            continue;
        }
        constexpr int XOR = 64 / LPR;           // pairs that a wave has of a column; the lanes of a column take other places in its row
#pragma unroll
        for (int kk = 0; kk < CAP; kk++) {
            const int rp = p0 + kk * PPS;
            if (rp >= half) continue;
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if (own[j]) {
                    const int c = mine.col + j - s0;
                    turned[c * ROW + (rp ^ (c / VEC * XOR & (ROW - 1)))] = pair_of(x0[kk][j], x1[kk][j], (T *)nullptr);
                }
        }
        __syncthreads();
        T *out = of_kind(false, is_k, k_cache, k_cache, v_cache) + (size_t)head * page * hd;
        const int chunks = hd / VEC;            // of 16 bytes
        constexpr int PER = VEC / 2;            // pairs of a chunk
        for (int i = tid; i < 64 * chunks; i += 256) {
            const int c = i / chunks, x = i - c * chunks;
            if (place[c] < 0) continue;
            const pair_t *chunk = turned + c * ROW + (x * PER ^ (c / VEC * XOR & (ROW - 1)));
            *reinterpret_cast<v4u *>(out + (size_t)place[c] * hd + x * VEC) = *reinterpret_cast<const v4u *>(chunk);
        }
    }
}

// Heads of columns from which tiles pay, where rows have 16 columns at least.  us, a wave to a head of a column / tiles, 16 + 8 + 8 heads of 128, bfloat16:
// one row of 128 new tokens 7.5 / 9.3, of 256 (8192 heads) 12.5 / 10.9, 16 rows of 16 positions 8.4 / 9.0, 32 of 32 17.6 / 13.9, 16 of 256 62 / 21.
constexpr size_t TILE_FROM = 8192;

template <typename T>
int kv_append(const char *who, const mi355_kv_cache *c, T *q_out, const T *q, const T *k, const T *v, const float *wq, const float *wk,
              const int32_t *seq, const int32_t *pos, int heads, int S, int batch, const float *cos_dev, const float *sin_dev, int table, float eps) {
    if (!kv_cache_ok(who, c)) return -1;
    if (!k || !v || !pos) return mi355_fail("%s: NULL pointer", who);
    if (!q != !q_out || !q != (heads == 0)) return mi355_fail("%s: q, q_out and heads go together", who);
    if (!cos_dev != !sin_dev || (cos_dev && table <= 0)) return mi355_fail("%s: cos, sin and the positions of their tables go together", who);
    if ((wq || wk) && !(eps >= 0.f)) return mi355_fail("%s: eps must not be negative", who);
    if (!kv_columns_ok(who, c, heads, S, batch, seq)) return -1;
    const size_t units = (size_t)S * batch * (heads + 2 * c->kv_heads);
    if (ceil_div(units, 4) > 0xffffff) return mi355_fail("%s: %zu heads of columns (at most 2^26 - 4)", who, units);
    if (!mi355_ready(who)) return -1;
    auto go = [&](auto kernel, dim3 grid, auto... more) {
        kernel<<<grid, 256, 0, g_ctx.stream>>>(q_out, q, k, v, (T *)c->k, (T *)c->v, c->pages, seq, pos, wq, wk, cos_dev, sin_dev, c->n_pages, c->page, c->n_seqs,
                                               c->max_pages, c->kv_heads, c->hd, heads, S, table, eps, more...);
        LAUNCH_OK(who);
        return 0;
    };
    if (S >= 16 && units >= TILE_FROM) {
        const int slabs = heads + 2 * c->kv_heads, tiles = (int)ceil_div(S, 64);
        // Heads to a workgroup, whose angles are then fetched once, by how many each compute unit gets.  us, one / two / four heads: 16 padded prompts of 256
        // (8 to a compute unit) 15.7 / 15.3 / 18.8, 32 of 32 14.7 / 13.2 / 15.6, one of 8191 in fp32 (18) 44 / 40 / 41, four of 4096 (32) 52 / 42 / 36.
        const size_t heads_each = (size_t)tiles * batch * slabs / g_ctx.num_cu;
        const int each = heads_each >= 24 ? 4 : heads_each >= 4 ? 2 : 1;
        const dim3 grid((unsigned)((size_t)tiles * batch * ceil_div(slabs, each)));
        constexpr int PPS = PAIRS_AT_ONCE<T>;
        if (c->hd / 2 <= 32) return go(kv_append_tile_kernel<T, 32 / PPS>, grid, tiles, each, tiles * batch);
        return go(kv_append_tile_kernel<T, 64 / PPS>, grid, tiles, each, tiles * batch);
    }
    return go(kv_append_kernel<T>, dim3((unsigned)ceil_div(units, 4)), S * batch);
}

// ---- rows that follow their parents ----------------------------------------------------------------------------------------------

// A row that is given no row, or one at another position, stays as it is.
__device__ __forceinline__ int parent_of(int n, const int *parents, const int *pos, int rows) {
    const int p = parents[n];
    return p >= 0 && p < rows && pos[p] == pos[n] ? p : n;
}

constexpr int MOVE_LAYERS = 64;
struct MoveArgs { void *cache[2 * MOVE_LAYERS]; };

// A workgroup to a row's head, in y to a tensor of a layer: its part of the tail, `words` 16-byte words to a position.  Behind the last tensor (in the first
// of several launches) the new table, a workgroup to a row; it is read by none of the copies.
// Rows that stay, and full pages, are not touched: 256 beams of 28 layers move 787 MB in 148 us, which is what a copy of as much takes.
__global__ __launch_bounds__(256) void kv_reorder_kernel(MoveArgs t, int tensors, int *__restrict__ pages_out, int *__restrict__ pos_out,
                                                         int *__restrict__ spare_out, const int *__restrict__ pages, const int *__restrict__ parents, const int *__restrict__ pos,
                                                         const int *__restrict__ spare, int rows, int max_pages, int page, int n_pages, int kv_heads,
                                                         int words, int advance) {
    const int n = blockIdx.x / kv_heads, head = blockIdx.x - n * kv_heads, at = pos[n], parent = parent_of(n, parents, pos, rows);
    const PagedMove m = paged_move(n, parent, at, page);
    // (a page that is none is passed on as it is)
    const bool moves = m.moves && m.tail < max_pages && paged_id_ok(pages[(size_t)parent * max_pages + m.tail], n_pages);
    if ((int)blockIdx.y == tensors) {
        if (head != 0) return;
        const int *from = pages + (size_t)parent * max_pages, *mine = pages + (size_t)n * max_pages;
        for (int j = threadIdx.x; j < max_pages; j += 256)
            pages_out[(size_t)n * max_pages + j] = j > m.tail ? mine[j] : j == m.tail && moves ? spare[n] : from[j];
        if (threadIdx.x == 0) {
            if (pos_out) pos_out[n] = at < 0 ? at : at + advance;
            spare_out[n] = moves ? mine[m.tail] : spare[n];
        }
        return;
    }
    if (!moves) return;
    const int from = pages[(size_t)parent * max_pages + m.tail], to = spare[n];
    if (!paged_id_ok(to, n_pages)) return;
    v4i *base = (v4i *)t.cache[blockIdx.y];
    const v4i *src = base + paged_row(from, head, 0, kv_heads, page, words);
    v4i *dst = base + paged_row(to, head, 0, kv_heads, page, words);
    for (int i = threadIdx.x; i < m.filled * words; i += 256) dst[i] = src[i];
}

int kv_reorder(const char *who, int size, const mi355_kv_cache *caches, int count, int32_t *pages_out, int32_t *pos_out, int32_t *spare_out,
               const int32_t *parent, const int32_t *pos, const int32_t *spare, int advance) {
    if (!caches || count <= 0) return mi355_fail("%s: no caches", who);
    for (int i = 0; i < count; i++) {
        const mi355_kv_cache *c = caches + i;
        if (!kv_cache_ok(who, c)) return -1;
        if (c->pages != caches->pages || c->n_pages != caches->n_pages || c->page != caches->page || c->n_seqs != caches->n_seqs ||
            c->max_pages != caches->max_pages || c->kv_heads != caches->kv_heads || c->hd != caches->hd)
            return mi355_fail("%s: cache %d is of another shape or table than the first", who, i);
    }
    if (!pages_out || !spare_out || !parent || !pos || !spare) return mi355_fail("%s: NULL pointer", who);
    if (pages_out == caches->pages || pos_out == pos || spare_out == spare)
        return mi355_fail("%s: the new table, positions and spare pages must not be the old ones", who);
    if (advance < 0) return mi355_fail("%s: advance must not be negative", who);
    const mi355_kv_cache &c = *caches;
    if ((double)c.n_seqs * c.kv_heads > (1 << 24) - 1)
        return mi355_fail("%s: n_seqs * kv_heads = %.0f (at most 2^24 - 1)", who, (double)c.n_seqs * c.kv_heads);
    if (!mi355_ready(who)) return -1;
    for (int i = 0; i < count; i += MOVE_LAYERS) {
        MoveArgs t = {};
        const int n = count - i < MOVE_LAYERS ? count - i : MOVE_LAYERS;
        for (int j = 0; j < n; j++) {
            t.cache[2 * j] = caches[i + j].k;
            t.cache[2 * j + 1] = caches[i + j].v;
        }
        kv_reorder_kernel<<<dim3((unsigned)(c.n_seqs * c.kv_heads), 2 * n + (i == 0)), 256, 0, g_ctx.stream>>>(
            t, 2 * n, pages_out, pos_out, spare_out, c.pages, parent, pos, spare, c.n_seqs, c.max_pages, c.page, c.n_pages, c.kv_heads, c.hd * size / 16,
            advance);
        LAUNCH_OK(who);
    }
    return 0;
}

}  // namespace

MI355_API int mi355_kv_append_dev(const mi355_kv_cache *cache, float *q_out, const float *q, const float *k, const float *v, const float *wq,
                                  const float *wk, const int32_t *seq, const int32_t *pos, int heads, int S, int batch, const float *cos_dev,
                                  const float *sin_dev, int table, float eps) {
    return kv_append<float>("kv_append", cache, q_out, q, k, v, wq, wk, seq, pos, heads, S, batch, cos_dev, sin_dev, table, eps);
}
MI355_API int mi355_kv_append_bf16_dev(const mi355_kv_cache *cache, uint16_t *q_out, const uint16_t *q, const uint16_t *k, const uint16_t *v,
                                       const float *wq, const float *wk, const int32_t *seq, const int32_t *pos, int heads, int S, int batch,
                                       const float *cos_dev, const float *sin_dev, int table, float eps) {
    return kv_append<bf16_t>("kv_append_bf16", cache, q_out, q, k, v, wq, wk, seq, pos, heads, S, batch, cos_dev, sin_dev, table, eps);
}
MI355_API int mi355_kv_reorder_dev(const mi355_kv_cache *caches, int count, int32_t *pages_out, int32_t *pos_out, int32_t *spare_out,
                                   const int32_t *parent, const int32_t *pos, const int32_t *spare, int advance) {
    return kv_reorder("kv_reorder", 4, caches, count, pages_out, pos_out, spare_out, parent, pos, spare, advance);
}
MI355_API int mi355_kv_reorder_bf16_dev(const mi355_kv_cache *caches, int count, int32_t *pages_out, int32_t *pos_out, int32_t *spare_out,
                                        const int32_t *parent, const int32_t *pos, const int32_t *spare, int advance) {
    return kv_reorder("kv_reorder_bf16", 2, caches, count, pages_out, pos_out, spare_out, parent, pos, spare, advance);
}
