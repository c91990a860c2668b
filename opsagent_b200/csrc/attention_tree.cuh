// attention_tree.cuh — what the kernels of attention of several new tokens share (attention_tree.cu, attention_tree_many.cu): sequences, the places that their rows see, and how work is dealt out.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r . k_j)  over the places j that row r sees:
//   cached ones, j < ctx:  j < sinks or pos_r - j < window (all without a window), pos_r = ctx + the number of r's ancestors;
//   new ones, j = ctx + u:  where bit u of seen_r is set.
//
// The softmax splits over any partition of the keys: a part leaves a reference m, l = sum 2^(s - m) and O = sum 2^(s - m) v, and parts join as O = sum_i 2^(m_i - M) O_i, l likewise, M = max m_i.
// Scores, references, sums, O and parts are fp32; the reference is a maximum that scores pass by 2^8 at most before it rises.  l sums the weights unrounded.
//
// A row tile of a sequence (as many tokens' heads of a group as fit) and a key/value head are an item; an item's units are a few for itself and one for each page, or pair of pages, that a row of the
// sequence sees.  Units are dealt out contiguously, the same number to every CTA, so that what parts an item has follows from lengths alone.  The plan is made on the device, by every CTA
// for itself: lengths may come from the kernel before, a captured call serves other lengths when it is replayed, and the host waits for nothing.  An item that one CTA has whole is written by it; of the
// others a CTA begins one at most, parts go to scratch and another kernel joins them in their order: the same call gives the same bits.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"
#include "work_units.hpp"

namespace oa {

constexpr int TREE_OVER = 2;             // tiles of 128 keys that an item's beginning and end cost (trees of 3 to 40 tokens, 40 / 8 heads: 99 us with 2, 101 with 3, 102 with 4, 105 with 6)
OA_DEVINL float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }     // nothing seen: any reference will do, 2^(-inf - 0) is 0
OA_DEVINL int pages_of(int len) { return (len + CACHE_PAGE - 1) / CACHE_PAGE; }
OA_DEVINL void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {       // untiled copy of 16-byte pieces, completing on an mbarrier
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
OA_DEVINL uint32_t pack_f16x2(float a, float b) { uint32_t r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a)); return r; }
// four values of 8 bits as two pairs of fp16, exactly: (0, 1) and (2, 3), or with ALT (0, 2) and (1, 3).  int8: 1024 + 128 + x has x in its low bits
template <int FMT, bool ALT>
OA_DEVINL void to_f16(uint32_t w, uint32_t& first, uint32_t& second) {
    if (FMT == CACHE_E4M3) {
        if (ALT) w = __byte_perm(w, 0, 0x3120);
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(first) : "h"((uint16_t)w));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(second) : "h"((uint16_t)(w >> 16)));
    } else {
        w ^= 0x80808080u;
        const uint32_t a = __byte_perm(w, 0x64646464u, ALT ? 0x4240 : 0x4140), b = __byte_perm(w, 0x64646464u, ALT ? 0x4341 : 0x4342), off = 0x64806480u;
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&off)), y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&off));
        first = *reinterpret_cast<const uint32_t*>(&x); second = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// A sequence: its new rows, its cached places, where its places end and which pages any of its rows sees
struct TreeSeq {
    int row0, n, ctx, end, low_pages, skip, pages;           // pages below low_pages are seen as they are, later ones are `skip` further on
    bool wrong;
    OA_DEVINL void read(const TreeAttnArgs& a, int seq) {
        const int r0 = __ldcg(a.row_starts + seq), r1 = __ldcg(a.row_starts + seq + 1), c = __ldcg(a.ctx_lens + seq);
        const int64_t room = (int64_t)a.max_pages * CACHE_PAGE;
        wrong = r0 < 0 || r1 < r0 || r1 > a.n_rows || r1 - (int64_t)r0 > TREE_MAX_TOKENS || c < 0 || c + max(r1 - (int64_t)r0, (int64_t)0) > room;
        row0 = min(max(r0, 0), a.n_rows);
        n = min(max(min(r1, a.n_rows) - row0, 0), TREE_MAX_TOKENS);
        ctx = (int)min((int64_t)max(c, 0), room);
        end = (int)min((int64_t)ctx + n, room);
        low_pages = skip = 0;
        if (a.window > 0) {
            const int near = max(ctx - a.window + 1, 0);     // the first place that the least deep row sees beside the kept ones
            low_pages = pages_of(min(a.sinks, near));
            skip = max(near / CACHE_PAGE - low_pages, 0);
        }
        pages = n > 0 ? pages_of(end) - skip : 0;
    }
    OA_DEVINL int page(int c) const { return c < low_pages ? c : c + skip; }
    OA_DEVINL int tiles(int tile_tokens) const { return (n + tile_tokens - 1) / tile_tokens; }
};
// How many of a sequence's pages begin below a place of its window.  Some row may not see all of a page where it begins below ctx + n - window (the deepest row's window), or does not end by ctx
OA_DEVINL int pages_below(const TreeSeq& s, int place) {
    if (place <= 0) return 0;
    const int page = pages_of(place) - 1;                                        // the last one that does
    return 1 + (page < s.low_pages ? page : max(page - s.skip, s.low_pages - 1));
}
// which new tokens token t of a sequence of n sees, and the first cached place of its window
OA_DEVINL uint64_t tree_seen(const TreeAttnArgs& a, const TreeSeq& s, int t) {
    const uint64_t there = s.n < 64 ? (1ull << s.n) - 1 : ~0ull;
    return (a.seen ? __ldcg(reinterpret_cast<const unsigned long long*>(a.seen) + s.row0 + t) : (2ull << t) - 1) & there;
}
OA_DEVINL int tree_low(const TreeAttnArgs& a, const TreeSeq& s, uint64_t seen, int t) { return a.window > 0 ? max(s.ctx + __popcll(seen & ((1ull << t) - 1)) - a.window + 1, 0) : 0; }

// A place in the list of (sequence, key/value head, row tile) items.  An item's units are OVER for itself and one for each PAGES of its sequence's pages
template <int PAGES, int OVER>
struct TreeAt {
    int seq, kvh, tile, tile_tokens; int64_t unit0; TreeSeq s;                   // unit0: the item's first unit
    OA_DEVINL int steps() const { return (s.pages + PAGES - 1) / PAGES; }
    OA_DEVINL int64_t units() const { return OVER + steps(); }
    OA_DEVINL int64_t all_units(const TreeAttnArgs& a) const { return (int64_t)s.tiles(tile_tokens) * a.n_kv * units(); }      // of the sequence
    // by a whole warp
    OA_DEVINL void next(const TreeAttnArgs& a) {
        unit0 += units();
        if (++tile < s.tiles(tile_tokens)) return;
        tile = 0;
        if (++kvh < a.n_kv) return;
        kvh = 0;
        if (++seq >= a.n_seqs) { s.n = s.pages = 0; return; }
        s.read(a, seq);
        // sequences without rows, as a padded batch has behind its last one, 32 at a time: each is a latency of L2
        while (s.n == 0) {
            const int lane = threadIdx.x & 31;
            TreeSeq other; other.n = 0;
            if (seq + 1 + lane < a.n_seqs) other.read(a, seq + 1 + lane);
            const uint32_t some = __ballot_sync(0xffffffffu, other.n > 0);
            if (some) s.read(a, seq += __ffs(some)); else if ((seq += 32) >= a.n_seqs - 1) { s.n = s.pages = 0; return; }
        }
    }
    OA_DEVINL int rows(int grp) const { return min(tile_tokens, s.n - tile * tile_tokens) * grp; }
    OA_DEVINL int row0() const { return s.row0 + tile * tile_tokens; }
};
struct TreeShare { int64_t busy, total, begin, end; };                           // a CTA's units
// The plan, by a whole CTA: what its share is and the item that it begins in
template <int THREADS, int PAGES, int OVER>
OA_DEVINL TreeShare tree_share(const TreeAttnArgs& a, int tile_tokens, int64_t* sums, TreeAt<PAGES, OVER>& start) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = (a.n_seqs + THREADS - 1) / THREADS, s0 = min(a.n_seqs, (int)threadIdx.x * per), s1 = min(a.n_seqs, s0 + per);
    TreeAt<PAGES, OVER> at;
    at.tile_tokens = tile_tokens;
    int64_t units = 0; bool wrong = false;
    for (at.seq = s0; at.seq < s1; ++at.seq) { at.s.read(a, at.seq); wrong = wrong || at.s.wrong; units += at.all_units(a); }
    if (wrong && a.status) *a.status = 400;
    int64_t before = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t x = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += x; }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    before -= units;
    TreeShare share; share.total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) before += sums[w]; share.total += sums[w]; }
    share.busy = busy_ctas(gridDim.x, share.total);
    share.begin = first_unit(blockIdx.x, share.busy, share.total); share.end = first_unit(blockIdx.x + 1, share.busy, share.total);
    if (share.begin < share.end && share.begin >= before && share.begin < before + units) {          // one thread
        at.seq = s0; at.unit0 = before;
        if (s1 - s0 > 1) at.s.read(a, s0);                                               // else it is there already
        while (share.begin >= at.unit0 + at.all_units(a)) { at.unit0 += at.all_units(a); ++at.seq; at.s.read(a, at.seq); }
        const int item = (int)quotient(share.begin - at.unit0, at.units()), tiles = at.s.tiles(tile_tokens);
        at.unit0 += (int64_t)item * at.units();
        at.kvh = item / tiles; at.tile = item - at.kvh * tiles;
        start = at;
    }
    if (threadIdx.x == 0) a.joins[blockIdx.x].parts = 0;
    __syncthreads();
    return share;
}
// whether a row sees anything at all
OA_DEVINL bool tree_sees(const TreeAttnArgs& a, const TreeSeq& s, uint64_t seen, int low) {
    const uint64_t there = s.end - s.ctx < 64 ? (1ull << (s.end - s.ctx)) - 1 : ~0ull;
    return (seen & there) != 0 || (s.ctx > 0 && (a.window == 0 || a.sinks > 0 || low < s.ctx));
}
// what a part leaves in scratch: [slot][D / 4][rows][4], and m and l of each row.  Slot 2 c: of the item that CTA c begins, 2 c + 1: of one that an earlier one began.  l of -1 in the former: the row sees nothing
OA_DEVINL void tree_record(const TreeAttnArgs& a, int later, int row0, int rows, int kvh) { TreeJoin j; j.parts = later; j.row0 = row0; j.rows = rows; j.kvh = kvh; a.joins[blockIdx.x] = j; }

// tiles of 128 rows (attention_tree_many.cu)
cudaError_t launch_tree_many(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int head_dim, int format, const TreeAttnArgs& a, cudaStream_t s);

}  // namespace oa
