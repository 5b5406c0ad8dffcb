// paged.h — where a position of a sequence lies in a paged cache of keys and values.  Plain C++, which the host and the device compile alike.
//
// k, v: [n_pages][kv_heads][page][hd], pages: [n_seqs][max_pages].  The rows of a page and head lie one after the other, a position's channels
// side by side: a new position is one row, and a reader takes whole rows whatever its page is.
#pragma once
#include <stddef.h>

// Place in the table of the page that holds position `pos` of sequence `seq`, -1 where the table has none.
constexpr __attribute__((always_inline)) long long paged_entry(int seq, int pos, int n_seqs, int max_pages, int page) {
    if (seq < 0 || seq >= n_seqs || pos < 0 || pos / page >= max_pages) return -1;
    return (long long)seq * max_pages + pos / page;
}
constexpr __attribute__((always_inline)) bool paged_id_ok(int id, int n_pages) { return id >= 0 && id < n_pages; }
// First value of a page's row, of head `head`.
constexpr __attribute__((always_inline)) size_t paged_row(int id, int head, int slot, int kv_heads, int page, int hd) {
    return (((size_t)id * kv_heads + head) * page + slot) * hd;
}

// What happens to row n of the table when it becomes the row of its parent, which is at the same position `pos`, on page `tail`: pages before the
// tail are the parent's, pages behind it stay n's own, and the tail itself is
//   the parent's page where parent == n or the page is full (nobody writes to a full page, so it is shared),
//   else n's spare page, into which the parent's rows are copied, while n's former tail, which nobody else has, becomes its spare.
struct PagedMove { bool moves; int tail, filled; };        // filled: rows of the tail that hold positions
constexpr __attribute__((always_inline)) PagedMove paged_move(int n, int parent, int pos, int page) {
    if (pos < 0) return {false, -1, 0};
    const int filled = pos % page + 1;
    return {parent != n && filled < page, pos / page, filled};
}
