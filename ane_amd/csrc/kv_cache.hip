// kv_cache.hip — a paged cache of keys and values: new positions are appended, rows of the table follow the beams of a search.
// No counterpart in the reference, whose loops train.  The norm and the rotation are those of qknorm_rope.hip and rope.h, at positions that
// are read from memory.
#include "kv_cache.h"

namespace {

__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const bf16_t *p) { return bf_to_f(*p); }
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16_t *p, float v) { *p = (bf16_t)f_to_bf(v); }

struct AppendArgs {
    mi355_kv_cache c;
    const float *wq, *wk, *cos_t, *sin_t;
    const int *seq, *pos;
    int heads, S, batch, table;
    float eps;
};

// A wave to a head of a column, a pair of channels to a lane.
template <typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(T *q_out, const T *q, const T *__restrict__ k, const T *__restrict__ v, AppendArgs a) {
    const int lane = threadIdx.x & 63, slabs = a.heads + 2 * a.c.kv_heads, hd = a.c.hd, half = hd / 2;
    const size_t unit = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const size_t col = unit / slabs;
    const int slab = (int)(unit - col * slabs);
    if (col >= (size_t)a.S * a.batch) return;
    const int b = (int)(col / a.S), s = (int)(col - (size_t)b * a.S), pos = a.pos[col];
    const long long entry = paged_entry(a.seq ? a.seq[col] : (int)col, pos, a.c.n_seqs, a.c.max_pages, a.c.page);
    if (entry < 0 || (a.cos_t && pos >= a.table)) return;
    const int id = a.c.pages[entry];
    if (!paged_id_ok(id, a.c.n_pages)) return;
    const bool is_q = slab < a.heads, is_k = !is_q && slab < a.heads + a.c.kv_heads;
    const int head = is_q ? slab : is_k ? slab - a.heads : slab - a.heads - a.c.kv_heads;
    const T *in = (is_q ? q : is_k ? k : v) + ((size_t)b * (is_q ? a.heads : a.c.kv_heads) + head) * hd * a.S + s;
    const float *w = is_q ? a.wq : is_k ? a.wk : nullptr;
    const bool mine = lane < half;
    float x0 = 0.f, x1 = 0.f;
    if (mine) {
        x0 = load_one(in + (size_t)(2 * lane) * a.S);
        x1 = load_one(in + (size_t)(2 * lane + 1) * a.S);
    }
    if (w) {
        const float rr = 1.f / sqrtf(wave_sum_stride<1>(x0 * x0 + x1 * x1) * (1.f / hd) + a.eps);
        if (mine) {
            x0 = (x0 * rr) * w[2 * lane];
            x1 = (x1 * rr) * w[2 * lane + 1];
        }
    }
    if (!mine) return;
    if ((is_q || is_k) && a.cos_t) {
        const float cs = a.cos_t[(size_t)lane * a.table + pos], sn = a.sin_t[(size_t)lane * a.table + pos];
        const float y0 = x0 * cs - x1 * sn, y1 = x0 * sn + x1 * cs;
        x0 = y0;
        x1 = y1;
    }
    if (is_q) {
        T *out = q_out + ((size_t)b * a.heads + head) * hd * a.S + s;
        store_one(out + (size_t)(2 * lane) * a.S, x0);
        store_one(out + (size_t)(2 * lane + 1) * a.S, x1);
    } else {
        T *out = (T *)(is_k ? a.c.k : a.c.v) + paged_row(id, head, pos % a.c.page, a.c.kv_heads, a.c.page, hd);
        store_one(out + 2 * lane, x0);
        store_one(out + 2 * lane + 1, x1);
    }
}

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
    const AppendArgs a = {*c, wq, wk, cos_dev, sin_dev, seq, pos, heads, S, batch, table, eps};
    kv_append_kernel<T><<<(unsigned)ceil_div(units, 4), 256, 0, g_ctx.stream>>>(q_out, q, k, v, a);
    LAUNCH_OK(who);
    return 0;
}

// ---- rows that follow their parents ----------------------------------------------------------------------------------------------

// A row that is given no row, or one at another position, stays as it is.
__device__ __forceinline__ int parent_of(int n, const int *parents, const int *pos, int rows) {
    const int p = parents[n];
    return p >= 0 && p < rows && pos[p] == pos[n] ? p : n;
}

// A workgroup to a row.
__global__ __launch_bounds__(256) void kv_table_kernel(int *__restrict__ pages_out, int *__restrict__ pos_out, int *__restrict__ spare_out,
                                                       const int *__restrict__ pages, const int *__restrict__ parents, const int *__restrict__ pos,
                                                       const int *__restrict__ spare, int rows, int max_pages, int page, int advance) {
    const int n = blockIdx.x, at = pos[n], parent = parent_of(n, parents, pos, rows);
    const PagedMove m = paged_move(n, parent, at, page);
    const bool moves = m.moves && m.tail < max_pages;
    const int *from = pages + (size_t)parent * max_pages, *mine = pages + (size_t)n * max_pages;
    for (int j = threadIdx.x; j < max_pages; j += 256)
        pages_out[(size_t)n * max_pages + j] = j > m.tail ? mine[j] : j == m.tail && moves ? spare[n] : from[j];
    if (threadIdx.x == 0) {
        if (pos_out) pos_out[n] = at < 0 ? at : at + advance;
        spare_out[n] = moves ? mine[m.tail] : spare[n];
    }
}

constexpr int MOVE_LAYERS = 64;
struct MoveArgs { void *cache[2 * MOVE_LAYERS]; };

// The tails: a workgroup to a head of a row and a tensor of a layer; `words` 16-byte words to a position.
__global__ __launch_bounds__(256) void kv_move_kernel(MoveArgs t, const int *__restrict__ pages, const int *__restrict__ parents,
                                                      const int *__restrict__ pos, const int *__restrict__ spare, int rows, int max_pages, int page,
                                                      int n_pages, int kv_heads, int words) {
    const int n = blockIdx.x / kv_heads, head = blockIdx.x - n * kv_heads, parent = parent_of(n, parents, pos, rows);
    const PagedMove m = paged_move(n, parent, pos[n], page);
    if (!m.moves || m.tail >= max_pages) return;
    const int from = pages[(size_t)parent * max_pages + m.tail], to = spare[n];
    if (!paged_id_ok(from, n_pages) || !paged_id_ok(to, n_pages)) return;
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
    if ((double)c.n_seqs * c.kv_heads > (1 << 24) - 1) return mi355_fail("%s: n_seqs * kv_heads = %.0f (at most 2^24 - 1)", who, (double)c.n_seqs * c.kv_heads);
    if (!mi355_ready(who)) return -1;
    for (int i = 0; i < count; i += MOVE_LAYERS) {
        MoveArgs t;
        const int n = count - i < MOVE_LAYERS ? count - i : MOVE_LAYERS;
        for (int j = 0; j < n; j++) {
            t.cache[2 * j] = caches[i + j].k;
            t.cache[2 * j + 1] = caches[i + j].v;
        }
        kv_move_kernel<<<dim3((unsigned)(c.n_seqs * c.kv_heads), 2 * n), 256, 0, g_ctx.stream>>>(t, c.pages, parent, pos, spare, c.n_seqs, c.max_pages,
                                                                                               c.page, c.n_pages, c.kv_heads, c.hd * size / 16);
        LAUNCH_OK(who);
    }
    kv_table_kernel<<<(unsigned)c.n_seqs, 256, 0, g_ctx.stream>>>(pages_out, pos_out, spare_out, c.pages, parent, pos, spare, c.n_seqs, c.max_pages,
                                                                  c.page, advance);
    LAUNCH_OK(who);
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
