// kv_cache.h — host side of the entry points that take a paged cache: what they ask of it.
#pragma once
#include "paged.h"
#include "tile.h"

static inline bool kv_cache_ok(const char *who, const mi355_kv_cache *c) {
    if (!c || !c->k || !c->v || !c->pages) { mi355_fail("%s: NULL pointer", who); return false; }
    if (c->n_pages <= 0 || c->n_seqs <= 0 || c->max_pages <= 0 || c->kv_heads <= 0 || c->page <= 0 || c->hd <= 0) {
        mi355_fail("%s: bad cache n_pages=%d page=%d n_seqs=%d max_pages=%d kv_heads=%d hd=%d", who, c->n_pages, c->page, c->n_seqs, c->max_pages,
                   c->kv_heads, c->hd);
        return false;
    }
    if (c->page % 16 || c->page > 1 << 16) { mi355_fail("%s: pages of %d positions (a multiple of 16, at most 65536)", who, c->page); return false; }
    if (c->hd % 8 || c->hd > 128) { mi355_fail("%s: head size %d (a multiple of 8, at most 128)", who, c->hd); return false; }
    if ((double)c->max_pages * c->page > 1 << 30) {
        mi355_fail("%s: max_pages * page = %.0f positions (at most 2^30)", who, (double)c->max_pages * c->page);
        return false;
    }
    if (c->kv_heads > 1 << 12) { mi355_fail("%s: kv_heads=%d (at most 4096)", who, c->kv_heads); return false; }
    if (!aligned16(c->k) || !aligned16(c->v)) { mi355_fail("%s: k and v of a cache begin at multiples of 16 bytes", who); return false; }
    return true;
}
// Columns of new tokens: `heads` query heads (0 where there are none), batch * S columns.
static inline bool kv_columns_ok(const char *who, const mi355_kv_cache *c, int heads, int S, int batch, const int32_t *seq) {
    if (heads < 0 || S <= 0 || batch <= 0 || (double)S * batch > 1 << 22 || heads > 1 << 14) {
        mi355_fail("%s: bad shape heads=%d S=%d batch=%d (batch * S at most 2^22, heads at most 2^14)", who, heads, S, batch);
        return false;
    }
    if (heads % c->kv_heads) { mi355_fail("%s: heads=%d is no multiple of kv_heads=%d", who, heads, c->kv_heads); return false; }
    if (!seq && S * batch > c->n_seqs) {
        mi355_fail("%s: %d columns of a sequence each, but the table has %d rows", who, S * batch, c->n_seqs);
        return false;
    }
    return true;
}
