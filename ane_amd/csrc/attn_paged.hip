// attn_paged.hip — attention of one new token over a paged cache of keys and values.
//   p_t = exp(scale q.k_t - lse) for 0 <= t <= pos,  o = sum_t p_t v_t,  lse = log sum_t exp(scale q.k_t)
#include "kv_cache.h"

#include <math.h>

namespace {

constexpr float LOG2E = 1.44269502162933349609375f, LN2 = 0.693147182464599609375f;

__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const bf16_t *p) { return bf_to_f(*p); }
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16_t *p, float v) { *p = (bf16_t)f_to_bf(v); }

// A wave to a head of a column; two channels to a lane.
template <typename T>
__global__ __launch_bounds__(64) void attn_paged_kernel(T *__restrict__ o, float *__restrict__ lse, const T *__restrict__ q, mi355_kv_cache c,
                                                        const int *__restrict__ seqs, const int *__restrict__ pos, int heads, int S, float scale2) {
    const int lane = threadIdx.x, hd = c.hd;
    const size_t unit = blockIdx.x, col = unit / heads;
    const int head = (int)(unit - col * heads), kvh = head / (heads / c.kv_heads), b = (int)(col / S), s = (int)(col - (size_t)b * S), at = pos[col];
    const int seq = seqs ? seqs[col] : (int)col;
    if (paged_entry(seq, at, c.n_seqs, c.max_pages, c.page) < 0) return;
    const bool mine0 = lane < hd, mine1 = lane + 64 < hd;
    const T *qp = q + ((size_t)b * heads + head) * hd * S + s;
    const float q0 = mine0 ? load_one(qp + (size_t)lane * S) : 0.f, q1 = mine1 ? load_one(qp + (size_t)(lane + 64) * S) : 0.f;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    bool any = false;
    for (int t = 0; t <= at; t++) {
        const int id = c.pages[paged_entry(seq, t, c.n_seqs, c.max_pages, c.page)];
        if (!paged_id_ok(id, c.n_pages)) continue;
        any = true;
        const size_t row = paged_row(id, kvh, t % c.page, c.kv_heads, c.page, hd);
        const T *k = (const T *)c.k + row, *v = (const T *)c.v + row;
        float z = mine0 ? q0 * load_one(k + lane) : 0.f;
        if (mine1) z += q1 * load_one(k + lane + 64);
        z = wave_sum_stride<1>(z) * scale2;
        const float top = fmaxf(m, z), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(z - base);
        m = top;
        l = l * f + p;
        o0 = o0 * f + (mine0 ? p * load_one(v + lane) : 0.f);
        o1 = o1 * f + (mine1 ? p * load_one(v + lane + 64) : 0.f);
    }
    if (!any) return;
    T *op = o + ((size_t)b * heads + head) * hd * S + s;
    if (mine0) store_one(op + (size_t)lane * S, o0 / l);
    if (mine1) store_one(op + (size_t)(lane + 64) * S, o1 / l);
    if (lse && lane == 0) lse[((size_t)b * heads + head) * S + s] = (m + __builtin_amdgcn_logf(l)) * LN2;
}

template <typename T>
int attn_paged(const char *who, const mi355_kv_cache *c, T *o, float *lse, const T *q, const int32_t *seq, const int32_t *pos, int heads, int S, int batch,
               float scale) {
    if (!kv_cache_ok(who, c)) return -1;
    if (!o || !q || !pos) return mi355_fail("%s: NULL pointer", who);
    if (heads == 0) return mi355_fail("%s: no heads", who);
    if (!kv_columns_ok(who, c, heads, S, batch, seq)) return -1;
    if (!(scale > 0.f) || !isfinite(scale * LOG2E)) return mi355_fail("%s: scale must be positive, and finite times log2(e)", who);
    const size_t units = (size_t)S * batch * heads;
    if (units > 0xffffff) return mi355_fail("%s: %zu heads of columns (at most 2^24 - 1)", who, units);
    if (!mi355_ready(who)) return -1;
    attn_paged_kernel<T><<<(unsigned)units, 64, 0, g_ctx.stream>>>(o, lse, q, *c, seq, pos, heads, S, scale * LOG2E);
    LAUNCH_OK(who);
    return 0;
}

}  // namespace

MI355_API int mi355_attn_paged_dev(const mi355_kv_cache *cache, float *o, float *lse, const float *q, const int32_t *seq, const int32_t *pos, int heads,
                                   int S, int batch, float scale) {
    return attn_paged<float>("attn_paged", cache, o, lse, q, seq, pos, heads, S, batch, scale);
}
MI355_API int mi355_attn_paged_bf16_dev(const mi355_kv_cache *cache, uint16_t *o, float *lse, const uint16_t *q, const int32_t *seq, const int32_t *pos,
                                        int heads, int S, int batch, float scale) {
    return attn_paged<bf16_t>("attn_paged_bf16", cache, o, lse, q, seq, pos, heads, S, batch, scale);
}
