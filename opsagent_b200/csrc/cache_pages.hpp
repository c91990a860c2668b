// cache_pages.hpp — host bookkeeping of a caller's paged cache (oa_page_table): growing, forking, freeing and compacting the pages of its sequences.  No GPU
// here: what has to be copied comes back as moves.  Every call checks what it is going to touch first and changes nothing where it fails.
#pragma once
#include <cstdint>
#include <cstring>
#include <vector>

#include "../../include/opsagent_b200.h"

namespace oa {

struct PageResult { int rc; const char* why; };
constexpr int TABLE_PAGE = 64;
inline int table_pages_of(int tokens) { return tokens / TABLE_PAGE + (tokens % TABLE_PAGE != 0); }
inline PageResult page_ok() { return {OA_OK, ""}; }
inline PageResult page_bad(const char* why) { return {OA_ERR_BAD_REQUEST, why}; }

inline PageResult check_table(const oa_page_table* t) {
    if (!t || !t->block_tables || !t->lens || !t->refs) return page_bad("page table: null array");
    if (t->n_rows < 1 || t->max_pages_per_seq < 1 || t->num_pages < 1) return page_bad("page table: no rows or no pages");
    return page_ok();
}
// a row that can be read: its length fits and its pages exist and are in use
inline PageResult check_row(const oa_page_table& t, int row) {
    if (row < 0 || row >= t.n_rows) return page_bad("page table: no such row");
    if (t.lens[row] < 0 || t.lens[row] > (int64_t)t.max_pages_per_seq * TABLE_PAGE) return page_bad("page table: a row's length is beyond its pages");
    const int32_t* r = t.block_tables + (size_t)row * t.max_pages_per_seq;
    for (int i = 0, n = table_pages_of(t.lens[row]); i < n; ++i)
        if (r[i] < 0 || r[i] >= t.num_pages || t.refs[r[i]] < 1) return page_bad("page table: a row names a page that is not in use");
    return page_ok();
}
// the n lowest-numbered free pages; false where there are fewer
inline bool lowest_free(const oa_page_table& t, int n, std::vector<int32_t>& out) {
    out.clear();
    for (int p = 0; p < t.num_pages && (int)out.size() < n; ++p) if (t.refs[p] == 0) out.push_back(p);
    return (int)out.size() == n;
}

// room for n_tokens more: new pages where the last one is full
inline PageResult table_grow(const oa_page_table* tp, int row, int n_tokens) {
    PageResult r = check_table(tp); if (r.rc) return r;
    const oa_page_table& t = *tp;
    if ((r = check_row(t, row)).rc) return r;
    const int len = t.lens[row], have = table_pages_of(len);
    if (n_tokens < 0 || (int64_t)len + n_tokens > INT32_MAX || (int64_t)len + n_tokens > (int64_t)t.max_pages_per_seq * TABLE_PAGE) return page_bad("page table: a row holds no more than its pages, and fewer than 2^31 tokens");
    int32_t* pages = t.block_tables + (size_t)row * t.max_pages_per_seq;
    if (n_tokens > 0 && len % TABLE_PAGE != 0 && t.refs[pages[have - 1]] > 1) return page_bad("page table: the last page is shared and not full (a fork copies it)");
    std::vector<int32_t> fresh;
    const int more = table_pages_of(len + n_tokens) - have;
    if (!lowest_free(t, more, fresh)) return {OA_ERR_OVERLOADED, "no free cache pages"};
    for (int i = 0; i < more; ++i) { pages[have + i] = fresh[i]; t.refs[fresh[i]] = 1; }
    t.lens[row] = len + n_tokens;
    return page_ok();
}

// children become copies of parent: full pages are shared, the last one, if partly filled, is copied (one move per child)
inline PageResult table_fork(const oa_page_table* tp, int parent, const int32_t* children, int n, oa_page_move* moves, int cap, int32_t* n_moves) {
    PageResult r = check_table(tp); if (r.rc) return r;
    const oa_page_table& t = *tp;
    if (n < 0 || (n > 0 && !children) || !n_moves || cap < 0 || (cap > 0 && !moves)) return page_bad("fork: bad arguments");
    if ((r = check_row(t, parent)).rc) return r;
    std::vector<bool> seen((size_t)t.n_rows, false);
    for (int i = 0; i < n; ++i) {
        const int c = children[i];
        if (c < 0 || c >= t.n_rows) return page_bad("fork: no such row");
        if (c == parent || seen[c]) return page_bad("fork: a child is its parent or named twice");
        if (t.lens[c] != 0) return page_bad("fork: a child holds tokens");
        seen[c] = true;
    }
    const int len = t.lens[parent], full = len / TABLE_PAGE, tail = len % TABLE_PAGE;
    std::vector<int32_t> fresh;
    if (tail) {
        if (cap < n) return page_bad("fork: too few moves");
        if (!lowest_free(t, n, fresh)) return {OA_ERR_OVERLOADED, "no free cache pages"};
    }
    const int32_t* from = t.block_tables + (size_t)parent * t.max_pages_per_seq;
    for (int i = 0; i < full; ++i) if (t.refs[from[i]] > INT32_MAX - n) return page_bad("fork: too many references to a page");
    for (int i = 0; i < n; ++i) {
        int32_t* to = t.block_tables + (size_t)children[i] * t.max_pages_per_seq;
        std::memcpy(to, from, (size_t)full * 4);
        if (tail) { to[full] = fresh[i]; t.refs[fresh[i]] = 1; moves[i] = oa_page_move{from[full], fresh[i], tail}; }
        t.lens[children[i]] = len;
    }
    for (int i = 0; i < full; ++i) t.refs[from[i]] += n;
    *n_moves = tail ? n : 0;
    return page_ok();
}

// rows give their references back and hold nothing; pages without one are free.  A row named twice, or empty, has nothing to give.
inline PageResult table_free(const oa_page_table* tp, const int32_t* rows, int n) {
    PageResult r = check_table(tp); if (r.rc) return r;
    const oa_page_table& t = *tp;
    if (n < 0 || (n > 0 && !rows)) return page_bad("free: bad arguments");
    for (int i = 0; i < n; ++i) if ((r = check_row(t, rows[i])).rc) return r;
    std::vector<bool> done((size_t)t.n_rows, false);
    std::vector<int32_t> left(t.refs, t.refs + t.num_pages);
    for (int i = 0; i < n; ++i) {
        if (done[rows[i]]) continue;
        done[rows[i]] = true;
        const int32_t* p = t.block_tables + (size_t)rows[i] * t.max_pages_per_seq;
        for (int k = 0, m = table_pages_of(t.lens[rows[i]]); k < m; ++k)
            if (--left[p[k]] < 0) return page_bad("free: more rows name a page than it has references");
    }
    std::memcpy(t.refs, left.data(), left.size() * 4);
    for (int i = 0; i < n; ++i) {
        int32_t* p = t.block_tables + (size_t)rows[i] * t.max_pages_per_seq;
        for (int k = 0, m = table_pages_of(t.lens[rows[i]]); k < m; ++k) p[k] = -1;
        t.lens[rows[i]] = 0;
    }
    return page_ok();
}

// the pages in use become the lowest-numbered ones: the i-th page in use beyond their count moves to the i-th free one below it, and every row names the new
// page.  Afterwards pages [0, in use) are in use and the rest is free.
inline PageResult table_compact(const oa_page_table* tp, oa_page_move* moves, int cap, int32_t* n_moves) {
    PageResult r = check_table(tp); if (r.rc) return r;
    const oa_page_table& t = *tp;
    if (!n_moves || cap < 0 || (cap > 0 && !moves)) return page_bad("compact: bad arguments");
    for (int i = 0; i < t.n_rows; ++i) if ((r = check_row(t, i)).rc) return r;
    int used = 0, high = 0;
    for (int p = 0; p < t.num_pages; ++p) { if (t.refs[p] < 0) return page_bad("compact: a negative reference count"); used += t.refs[p] > 0; }
    for (int p = used; p < t.num_pages; ++p) high += t.refs[p] > 0;
    if (high > cap) return page_bad("compact: too few moves");
    if (high > 0) {
        std::vector<int32_t> to((size_t)t.num_pages);
        for (int p = 0; p < t.num_pages; ++p) to[p] = p;
        for (int p = used, q = 0, i = 0; i < high; ++p) {
            if (t.refs[p] == 0) continue;
            while (t.refs[q] != 0) ++q;
            moves[i++] = oa_page_move{p, q, TABLE_PAGE};
            to[p] = q; t.refs[q] = t.refs[p]; t.refs[p] = 0;
        }
        for (int i = 0; i < t.n_rows; ++i) {
            int32_t* b = t.block_tables + (size_t)i * t.max_pages_per_seq;
            for (int k = 0, m = table_pages_of(t.lens[i]); k < m; ++k) b[k] = to[b[k]];
        }
    }
    *n_moves = high;
    return page_ok();
}

}  // namespace oa
