// attention_tree.cu — attention of several new tokens of each sequence (one, a chain, a tree of drafts) over a paged cache of bf16 or 8 bits.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r . k_j)  over the places j that row r sees:
//   cached ones, j < ctx:  j < sinks or pos_r - j < window (all without a window), pos_r = ctx + the number of r's ancestors;
//   new ones, j = ctx + u:  where bit u of seen_r is set.
//
// The softmax splits over any partition of the keys: a part leaves its maximum m, l = sum 2^(s - m) and O = sum 2^(s - m) v, and parts join as O = sum_i 2^(m_i - M) O_i, l likewise.
// Scores, maxima, sums and O are fp32.  Over a cache of bf16 the weights are rounded to bf16 for the second product.  A cache of 8 bits is multiplied in fp16, which holds e4m3 and int8 exactly: a row
// of q is scaled by a power of two that brings its largest magnitude to [2^14, 2^15), where 8 bits of a channel stay down to 2^-31 of that; a key's scale multiplies its scores, a value's scale its
// weights, over a power of two that no scale so far passes and times 2^15: at least 8 bits of a weight stay down to 2^-32 of the largest.  l sums the weights unrounded.
//
// A row tile of a sequence (its tokens' heads of a group, up to 8 or 16 rows) and a key/value head are an item; an item's units are one for itself and one for each page that a row of the sequence sees.
// Units are dealt out contiguously, the same number to every CTA, so that what parts an item has follows from lengths alone.  The plan is made on the device, by every CTA for itself.  An
// item that one CTA has whole is written by it; of the others, of which a CTA begins one at most, parts go to scratch and a second kernel joins them in their order: the same call gives the same bits.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"
#include "work_units.hpp"

namespace oa {

constexpr int TREE_CONSUMERS = 256, TREE_THREADS = TREE_CONSUMERS + 96;          // eight consumer warps; a producer, a warp that brings an item's states together, one that lays its queries out

OA_DEVINL float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }     // nothing seen: any reference will do, 2^(-inf - 0) is 0
OA_DEVINL int pages_of(int len) { return (len + CACHE_PAGE - 1) / CACHE_PAGE; }
OA_DEVINL uint32_t transpose_8x8(uint32_t v) { uint32_t r; asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v)); return r; }      // 16-bit values, a row in four lanes
OA_DEVINL void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {       // untiled copy of 16-byte pieces, completing on an mbarrier
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
OA_DEVINL void mbar_wait3(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, uint64_t* c, uint32_t pc) {        // phases that do not pass before this thread's own arrivals
    uint32_t spins = 0;
    for (;;) {
        const bool x = mbar_try_wait(a, pa), y = mbar_try_wait(b, pb), z = mbar_try_wait(c, pc);
        if (x && y && z) return;
        if (++spins > OA_MBAR_SPIN_LIMIT) { __trap(); }
    }
}
OA_DEVINL uint32_t pack_f16x2(float a, float b) { uint32_t r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a)); return r; }
OA_DEVINL void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
OA_DEVINL uint32_t mul_f16x2(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
OA_DEVINL uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) { uint32_t r; asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c)); return r; }
template <int FMT>
OA_DEVINL void mma_of(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (FMT == CACHE_BF16) mma_bf16_16816(d, a0, a1, a2, a3, b0, b1); else mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
}
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
    // whether some row may not see all of a page's places
    OA_DEVINL bool special(const TreeAttnArgs& a, int page) const { return (page + 1) * CACHE_PAGE > ctx || (a.window > 0 && page * CACHE_PAGE < ctx + n - a.window); }
};
// how many of a sequence's pages begin below a place of its window
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
    OA_DEVINL void next(const TreeAttnArgs& a) {
        unit0 += units();
        if (++tile < s.tiles(tile_tokens)) return;
        tile = 0;
        if (++kvh < a.n_kv) return;
        kvh = 0;
        do { if (++seq >= a.n_seqs) { s.n = s.pages = 0; return; } s.read(a, seq); } while (s.n == 0);
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

// =============================================================================================
// up to 16 rows of an item: the warp path
// =============================================================================================
// What eight warps do with pages: bf16, which memory bounds, take every page together, 16 tokens and half of the channels a warp; 8 bits, which issue slots bound, take pages in turn, four warps a page, 16
// tokens and all channels a warp: scores, weights and keys' fp16 once instead of twice
template <int D, int FMT, int NB, int STAGES>
struct FewCfg {
    static constexpr int ESZ = FMT == CACHE_BF16 ? 2 : 1, GROUPS = FMT == CACHE_BF16 ? 1 : 2, PARTS = 2 / GROUPS;       // groups of warps that take pages in turn; parts of the channels
    static_assert(GROUPS == 1 || STAGES % 2 == 0, "a page of the ring belongs to one group");
    static constexpr int KV_BYTES = CACHE_PAGE * D * ESZ, STAGE_BYTES = 2 * KV_BYTES, SCALE_BYTES = FMT == CACHE_BF16 ? 0 : 2 * CACHE_PAGE * 4;
    static constexpr int ROWS = 8 * NB, REGS = D / 4 * NB, STATES = 4 * GROUPS;  // output values of a lane in all parts; states of an item that meet
    static constexpr int Q_PITCH = D * 2 + (FMT == CACHE_BF16 ? 16 : 64), Q_BYTES = ROWS * Q_PITCH;      // no bank conflicts
    static constexpr int STATE_BYTES = STATES * (REGS * 32 * 4 + ROWS * 2 * 4 + 4);
    static constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + SCALE_BYTES) + 2 * (Q_BYTES + ROWS * 16 + 80) + STATE_BYTES + (2 * STAGES + 6) * 8;
    static constexpr int CTAS = FMT != CACHE_BF16 && NB == 1 ? 2 : 1;            // of an SM
};
struct TreeMeta { uint64_t seen; int low; float factor; };
struct FewItem { TreeSeq s; int c0, c1, low, high, row0, rows, kvh, later; bool first, last, more; };      // a CTA's pages of an item, special ones below `low` and from `high` on; CTAs that have later parts
static_assert(sizeof(FewItem) <= 80, "an item's place in shared memory");

template <int D>
OA_DEVINL uint32_t few_off(int r, int d) { return (uint32_t)((d >> 6) * (CACHE_PAGE * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4)); }      // bf16: halves of 64 channels
template <int D>
OA_DEVINL uint32_t few_off8(int r, int chunk) {                                  // 8 bits: chunk of 16 channels of token r
    if (D == 128) return (uint32_t)(r * 128 + ((chunk ^ (r & 7)) << 4));
    return (uint32_t)((r >> 1) * 128 + (((((r & 1) << 2) + chunk) ^ ((r >> 1) & 7)) << 4));
}

template <int D, int FMT, int NB, int STAGES>
__global__ void __launch_bounds__(TREE_THREADS, FewCfg<D, FMT, NB, STAGES>::CTAS) tree_few_kernel(const __grid_constant__ CUtensorMap tm_page, const __grid_constant__ TreeAttnArgs a) {
    using Cfg = FewCfg<D, FMT, NB, STAGES>;
    constexpr int KS = D / 16, KH = KS / Cfg::PARTS, ROWS = Cfg::ROWS, STATES = Cfg::STATES;
    constexpr bool BITS8 = FMT != CACHE_BF16;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* scales_s = smem + STAGES * Cfg::STAGE_BYTES;                                    // [stage][keys', values'][64]
    uint8_t* q_s = scales_s + STAGES * Cfg::SCALE_BYTES;                                     // [2 items][rows]
    TreeMeta* meta_s = reinterpret_cast<TreeMeta*>(q_s + 2 * Cfg::Q_BYTES);                  // [2 items][rows]
    uint8_t* item_s = reinterpret_cast<uint8_t*>(meta_s + 2 * ROWS);                         // [2 items]
    float* states = reinterpret_cast<float*>(item_s + 2 * 80);                               // [states][values][32 lanes]
    float* ml_s = states + Cfg::STATES * Cfg::REGS * 32;                                     // [states][rows][2]
    float* vref_s = ml_s + Cfg::STATES * ROWS * 2;                                           // [states]: what values' scales are taken over
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(vref_s + Cfg::STATES);
    uint64_t *empty_bar = full_bar + STAGES, *q_full = empty_bar + STAGES, *q_empty = q_full + 2, *states_full = q_empty + 2, *states_empty = states_full + 1;
    using At = TreeAt<1, 1>;
    __shared__ int64_t sums[TREE_THREADS / 32];
    __shared__ At start;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv, tile_tokens = ROWS / grp;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_page);
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], TREE_CONSUMERS / 32 / Cfg::GROUPS); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], TREE_CONSUMERS / 32 + 1); }
        mbar_init(states_full, TREE_CONSUMERS / 32); mbar_init(states_empty, 1);
        fence_barrier_init();
    }
    griddep_wait();
    const TreeShare share = tree_share<TREE_THREADS>(a, tile_tokens, sums, start);
    const int64_t u_begin = share.begin, u_end = share.end;
    if (u_begin >= u_end) { griddep_launch(); return; }
    At at = start;
    auto next = [&] { at.next(a); };

    if (warp == 8) {
        int st = 0; uint32_t ph = 0;
        for (int64_t u = u_begin; u < u_end; next()) {
            const int c0 = (int)max(u - at.unit0 - 1, (int64_t)0), c1 = (int)min((int64_t)at.s.pages, u_end - at.unit0 - 1);
            u = at.unit0 + 1 + c1;
            const int32_t* table = a.tables + (int64_t)at.seq * a.max_pages;
            int have = 0;
            for (int c = c0; c < c1; ++c) {
                if (c == c0 || (c & 31) == 0) { const int w = (c & ~31) + lane; have = w < c1 ? __ldcg(table + at.s.page(w)) : 0; }
                int page = __shfl_sync(0xffffffffu, have, c & 31);
                if (page < 0 || page >= a.num_pages) { if (lane == 0 && a.status) *a.status = 400; page = 0; }
                mbar_wait(&empty_bar[st], ph ^ 1);
                if (lane == 0) mbar_expect_tx(&full_bar[st], Cfg::STAGE_BYTES + Cfg::SCALE_BYTES);
                __syncwarp();
                // a lane a copy: one that issues them all takes longer for it than a page's warps do
                constexpr int COPIES = BITS8 ? 2 : D / 64;                                   // of keys, of values
                if (lane < 2 * COPIES) {
                    const int v = lane / COPIES, part = lane % COPIES;
                    uint8_t* dst = smem + st * Cfg::STAGE_BYTES + v * Cfg::KV_BYTES;
                    const int64_t block = (int64_t)(v * a.num_pages + page) * a.n_kv + at.kvh;
                    if (!BITS8) tma_load_2d(dst + part * (CACHE_PAGE * 128), &tm_page, &full_bar[st], part * 64, (int)(block * CACHE_PAGE), kEvictFirst);
                    else {
                        constexpr int BLOCK_BYTES = CACHE_PAGE * (D + 4);
                        if (part == 0) tma_load_2d(dst, &tm_page, &full_bar[st], 0, (int)(block * (BLOCK_BYTES / 128)), kEvictFirst);
                        else bulk_load(scales_s + st * Cfg::SCALE_BYTES + v * CACHE_PAGE * 4, reinterpret_cast<const uint8_t*>(a.cache) + block * BLOCK_BYTES + CACHE_PAGE * D, CACHE_PAGE * 4, &full_bar[st]);
                    }
                }
                __syncwarp();
                if (++st == STAGES) { st = 0; ph ^= 1; }
            }
        }
        griddep_launch();
        return;
    }
    if (warp == 10) {
        // queries of an item, and what its rows see.  8 bits: fp16 under a power of two, pieces of eight channels where the consumers' lanes find them side by side
        uint32_t k = 0;
        for (int64_t u = u_begin; u < u_end; next(), ++k) {
            const int64_t end = at.unit0 + 1 + at.s.pages;
            FewItem item;
            item.s = at.s; item.c0 = (int)max(u - at.unit0 - 1, (int64_t)0); item.c1 = (int)min((int64_t)at.s.pages, u_end - at.unit0 - 1);
            item.low = a.window > 0 ? pages_below(at.s, at.s.ctx + at.s.n - a.window) : 0; item.high = at.s.ctx / CACHE_PAGE - at.s.skip;
            item.row0 = at.row0(); item.rows = at.rows(grp); item.kvh = at.kvh;
            item.first = at.unit0 >= u_begin; item.last = end <= u_end; item.more = end < u_end;
            item.later = item.first && !item.last ? cta_of(end - 1, share.busy, share.total) - (int)blockIdx.x : 0;
            u = min(end, u_end);
            mbar_wait(&q_empty[k & 1], ((k >> 1) & 1) ^ 1);
            if (lane == 0) *reinterpret_cast<FewItem*>(item_s + (k & 1) * 80) = item;
            uint8_t* q_dst = q_s + (k & 1) * Cfg::Q_BYTES;
            TreeMeta* meta = meta_s + (k & 1) * ROWS;
            const int live = at.rows(grp), t0 = at.tile * tile_tokens;
            constexpr int W = D / 64;                                                        // words of two channels a lane
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                uint32_t w[8][W];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = b * 8 + i, token = r / grp;
                    const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(at.s.row0 + t0 + token) * a.ldq + (int64_t)(at.kvh * grp + r - token * grp) * D + lane * 2 * W;
                    if (r < live) {
                        if (W == 2) { const uint2 x = __ldcg(reinterpret_cast<const uint2*>(src)); w[i][0] = x.x; w[i][W - 1] = x.y; } else w[i][0] = __ldcg(reinterpret_cast<const uint32_t*>(src));
                    } else
#pragma unroll
                        for (int j = 0; j < W; ++j) w[i][j] = 0u;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = b * 8 + i;
                    float factor = 1.0f;
                    int place = lane * 4 * W;
                    if (BITS8) {
                        uint32_t top = 0;
#pragma unroll
                        for (int j = 0; j < W; ++j) top = max(top, max(w[i][j] << 16 & 0x7fffffffu, w[i][j] & 0x7fff0000u));
                        top = __reduce_max_sync(0xffffffffu, top);
                        const int e = top >= 0x7f800000u ? 14 : max((int)(top >> 23) - 127, -100);       // not finite: as it is
                        const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
                        factor = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
#pragma unroll
                        for (int j = 0; j < W; ++j) w[i][j] = pack_f16x2(bf16lo(w[i][j]) * up, bf16hi(w[i][j]) * up);
                        const int chunk = lane * W / 4;                                      // of eight channels: consumer lane chunk / (D / 32)'s number chunk % (D / 32)
                        place = ((chunk % (D / 32)) * 4 + chunk / (D / 32)) * 16 + (lane * W % 4) * 4;
                    }
#pragma unroll
                    for (int j = 0; j < W; ++j) *reinterpret_cast<uint32_t*>(q_dst + r * Cfg::Q_PITCH + place + j * 4) = w[i][j];
                    if (lane == 0) meta[r].factor = factor * a.scale_log2e;
                }
            }
            if (lane < ROWS) {
                uint64_t seen = 0; int low = 0x7fffffff;
                if (lane < live) { const int t = t0 + lane / grp; seen = tree_seen(a, at.s, t); low = tree_low(a, at.s, seen, t); }
                meta[lane].seen = seen; meta[lane].low = low;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[k & 1]);
        }
        griddep_launch();
        return;
    }
    if (warp == 9) {
        // An item's states under one maximum: its rows of the output where the CTA has all of it, a part elsewhere
        const int g = lane >> 2, t = lane & 3;
        for (uint32_t k = 0;; ++k) {
            mbar_wait(&q_full[k & 1], (k >> 1) & 1);
            const FewItem& item = *reinterpret_cast<const FewItem*>(item_s + (k & 1) * 80);
            const bool first = item.first, whole = item.first && item.last, more = item.more;
            const int live = item.rows, row0 = item.row0, kvh = item.kvh;
            const TreeMeta own = meta_s[(k & 1) * ROWS + (lane < ROWS ? lane : 0)];
            const uint32_t blind = __ballot_sync(0xffffffffu, lane < live && !tree_sees(a, item.s, own.seen, own.low));       // rows that see nothing
            if (lane == 0 && first && !whole) tree_record(a, item.later, row0, live, kvh);
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_empty[k & 1]);
            float* po = a.part_o + ((int64_t)blockIdx.x * 2 + !first) * (ROWS * D);
            float2* ml = reinterpret_cast<float2*>(a.part_ml) + ((int64_t)blockIdx.x * 2 + !first) * ROWS;
            mbar_wait(states_full, k & 1);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    const int row = b * 8 + 2 * t + h;
                    float2 s4[STATES]; float m = -INFINITY, l = 0.f, f[STATES];
#pragma unroll
                    for (int w = 0; w < STATES; ++w) { s4[w] = *reinterpret_cast<const float2*>(ml_s + (w * ROWS + row) * 2); m = fmaxf(m, s4[w].x); }
                    const float ref = finite_or_zero(m);
#pragma unroll
                    for (int w = 0; w < STATES; ++w) { f[w] = ex2_approx(s4[w].x - ref); l += f[w] * s4[w].y; if (BITS8) f[w] *= vref_s[w]; }
                    if (row >= live) continue;
                    const int token = row / grp;
                    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(row0 + token) * a.ldo + (int64_t)(kvh * grp + row - token * grp) * D;
                    const float inv = whole ? (blind >> row & 1 ? 0.f : 1.0f / l) : 1.0f;
                    if (!whole && g == 0) ml[row] = make_float2(m, first && (blind >> row & 1) ? -1.0f : l);
#pragma unroll 4
                    for (int r = 0; r < KS * 2; ++r) {                                       // channel block r / 2 and the one or the other of a lane's two channels there
                        const int i = r >> 1, up = r & 1, reg = (i / KH) * (Cfg::REGS / Cfg::PARTS) + (b * KH + i % KH) * 4 + 2 * up + h, d = i * 16 + (BITS8 ? 2 * g + up : 8 * up + g);
                        float o = 0.f;
#pragma unroll
                        for (int w = 0; w < STATES; ++w) o += f[w] * states[(w * Cfg::REGS + reg) * 32 + lane];
                        if (whole) out[d] = f32_to_bf16_bits(o * inv); else po[(d >> 2) * (ROWS * 4) + row * 4 + (d & 3)] = o;
                    }
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(states_empty);
            if (!more) break;
        }
        griddep_launch();
        return;
    }

    // Tokens are the 16 rows of the first product and channels those of the second, the item's rows the 8 columns of both: S^T = K Q^T, O^T = V^T P^T.  A row's reference maximum rises (and its sums are
    // rescaled) only where a score passes it by 2^8
    const int g = lane >> 2, t = lane & 3, quarter = warp & 3, half = Cfg::PARTS == 2 ? warp >> 2 : 0, group = Cfg::GROUPS == 2 ? warp >> 2 : 0;
    constexpr float kRaise = 8.0f;
    constexpr float kValueUp = 128.f;                                                        // a weight is 2^8 at most: fp16 holds it times a value's scale
    uint32_t pages = 0, n_items = 0;                                                         // of the items before
    for (bool more = true; more; ++n_items) {
        mbar_wait(&q_full[n_items & 1], (n_items >> 1) & 1);
        const FewItem& item = *reinterpret_cast<const FewItem*>(item_s + (n_items & 1) * 80);
        const TreeMeta* meta = meta_s + (n_items & 1) * ROWS;
        const int c0 = item.c0, c1 = max(item.c0, item.c1), special_below = item.low, special_from = item.high;
        more = item.more;
        float oacc[NB][KH][4], m_run[NB][2], l_run[NB][2], factor[NB][2];                    // O^T: two channels of a lane in each block of 16, rows 2 t and 2 t + 1; references, sums and score factors of these rows
        float vref = 0.f;                                                                    // 8 bits: a power of two that no value's scale so far passes
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < KH; ++i) oacc[b][i][0] = oacc[b][i][1] = oacc[b][i][2] = oacc[b][i][3] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) { m_run[b][h] = -INFINITY; l_run[b][h] = 0.f; factor[b][h] = meta[b * 8 + 2 * t + h].factor; }
        }
        const uint8_t* q_item = q_s + (n_items & 1) * Cfg::Q_BYTES;
        for (int c = c0 + (Cfg::GROUPS == 2 ? (int)((pages ^ group) & 1) : 0); c < c1; c += Cfg::GROUPS) {
            const uint32_t n = pages + (c - c0), st = n % STAGES;
            const bool special = c < special_below || c >= special_from;
            mbar_wait(&full_bar[st], (n / STAGES) & 1);
            const int key0 = special ? item.s.page(c) * CACHE_PAGE + quarter * 16 : 0;
            if (!special || key0 < item.s.end) {
                const uint8_t* stage = smem + st * Cfg::STAGE_BYTES;
                const uint32_t kbase = smem_u32(stage), vbase = kbase + Cfg::KV_BYTES;
                float sacc[NB][2][4];                                                        // even and odd steps apart: two chains of products
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sacc[b][0][e] = sacc[b][1][e] = 0.f;
                float kscale[2] = {1.f, 1.f}, vscale[2] = {1.f, 1.f};                        // of tokens g and g + 8
                if constexpr (BITS8) {
                    const float* sc = reinterpret_cast<const float*>(scales_s + st * Cfg::SCALE_BYTES) + quarter * 16 + g;
                    kscale[0] = sc[0]; kscale[1] = sc[8]; vscale[0] = sc[CACHE_PAGE]; vscale[1] = sc[CACHE_PAGE + 8];
                    const int r = quarter * 16 + g;
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {                                       // lane t's channels: D / 4 of them next to each other, four a step
                        const uint4 x0 = *reinterpret_cast<const uint4*>(stage + few_off8<D>(r, t * (D / 64) + j)), x1 = *reinterpret_cast<const uint4*>(stage + few_off8<D>(r + 8, t * (D / 64) + j));
                        const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            uint4 qf[NB];
#pragma unroll
                            for (int b = 0; b < NB; ++b) qf[b] = *reinterpret_cast<const uint4*>(q_item + (b * 8 + g) * Cfg::Q_PITCH + ((2 * j + p) * 4 + t) * 16);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                uint32_t k0, k1, k2, k3;
                                to_f16<FMT, false>(w0[2 * p + e], k0, k2);
                                to_f16<FMT, false>(w1[2 * p + e], k1, k3);
#pragma unroll
                                for (int b = 0; b < NB; ++b) mma_of<FMT>(sacc[b][e], k0, k1, k2, k3, e ? qf[b].z : qf[b].x, e ? qf[b].w : qf[b].y);
                            }
                        }
                    }
                } else {
                    const int r = quarter * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), dsel = (lane >> 4) << 3;
                    const uint32_t qbase = smem_u32(q_item) + (lane & 7) * Cfg::Q_PITCH + (lane >> 3) * 16;
#pragma unroll
                    for (int k0 = 0; k0 < KS; k0 += 4) {                                     // loads of four steps ahead of their products
                        uint32_t qf[NB][2][4], kf[4][4];
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int b = 0; b < NB; ++b) ldmatrix_x4(qbase + b * 8 * Cfg::Q_PITCH + (k0 + 2 * h) * 32, qf[b][h][0], qf[b][h][1], qf[b][h][2], qf[b][h][3]);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) ldmatrix_x4(kbase + few_off<D>(r, (k0 + ks) * 16 + dsel), kf[ks][0], kf[ks][1], kf[ks][2], kf[ks][3]);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                            for (int b = 0; b < NB; ++b) mma_of<FMT>(sacc[b][ks & 1], kf[ks][0], kf[ks][1], kf[ks][2], kf[ks][3], qf[b][ks >> 1][2 * (ks & 1)], qf[b][ks >> 1][2 * (ks & 1) + 1]);
                    }
                }
                // which rows see tokens g (bits 0 and 1 of a block's two) and g + 8 (2 and 3), and whether anyone does
                uint32_t vis = 0xffffffffu, any_lo = 0xffffffffu, any_hi = 0xffffffffu;
                if (special) {
                    vis = 0;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const TreeMeta m = meta[b * 8 + 2 * t + h];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int key = key0 + g + 8 * e, u = key - item.s.ctx;
                                const bool sees = u < 0 ? key < a.sinks || key >= m.low : key < item.s.end && u < 64 && (m.seen >> (u & 63) & 1);
                                if (sees) vis |= 1u << (b * 4 + e * 2 + h);
                            }
                        }
                    constexpr uint32_t LO = NB == 2 ? 0x33u : 0x3u;
                    any_lo = __ballot_sync(0xffffffffu, (vis & LO) != 0); any_hi = __ballot_sync(0xffffffffu, (vis & LO << 2) != 0);
                }
                float vfac[2] = {1.f, 1.f}, grown = 1.0f;                                    // a weight's factor of tokens g and g + 8; O's, where a scale passes the reference
                if constexpr (BITS8) {
                    // a bit of a token is in its four lanes together: whoever is not seen by anyone counts for nothing
                    const bool see_lo = any_lo >> (g * 4) & 0xfu, see_hi = any_hi >> (g * 4) & 0xfu;
                    const float top = fmaxf(see_lo && vscale[0] < INFINITY ? fabsf(vscale[0]) : 0.f, see_hi && vscale[1] < INFINITY ? fabsf(vscale[1]) : 0.f);
                    if (__any_sync(0xffffffffu, top >= vref)) {
                        const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
                        const float need = __uint_as_float(min(max((most & 0x7f800000u) + 0x00800000u, 0x0d800000u), 0x7e800000u));     // 2^-100 to 2^126
                        if (need > vref) { grown = vref * (1.0f / need); vref = need; }
                    }
                    const float inv = kValueUp / vref;                                       // powers of two: exact
                    vfac[0] = vscale[0] * inv; vfac[1] = vscale[1] * inv;
                }
                uint32_t pb[NB][2]; float sc[NB][2][2];
                bool raise = false;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        sc[b][h][0] = vis >> (b * 4 + h) & 1 ? (sacc[b][0][h] + sacc[b][1][h]) * (BITS8 ? kscale[0] * factor[b][h] : factor[b][h]) : -INFINITY;
                        sc[b][h][1] = vis >> (b * 4 + 2 + h) & 1 ? (sacc[b][0][2 + h] + sacc[b][1][2 + h]) * (BITS8 ? kscale[1] * factor[b][h] : factor[b][h]) : -INFINITY;
                        raise = raise || fmaxf(sc[b][h][0], sc[b][h][1]) > m_run[b][h] + kRaise;
                    }
                if (__any_sync(0xffffffffu, raise) || grown != 1.0f) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float alpha[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float mx = fmaxf(sc[b][h][0], sc[b][h][1]);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                            const float m_new = mx > m_run[b][h] + kRaise ? mx : m_run[b][h];
                            alpha[h] = m_new == m_run[b][h] ? 1.0f : ex2_approx(m_run[b][h] - finite_or_zero(m_new));
                            m_run[b][h] = m_new;
                            l_run[b][h] *= alpha[h]; alpha[h] *= grown;
                        }
#pragma unroll
                        for (int i = 0; i < KH; ++i) { oacc[b][i][0] *= alpha[0]; oacc[b][i][1] *= alpha[1]; oacc[b][i][2] *= alpha[0]; oacc[b][i][3] *= alpha[1]; }
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float pr[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float ref = finite_or_zero(m_run[b][h]);
                        const float p0 = ex2_approx(sc[b][h][0] - ref), p1 = ex2_approx(sc[b][h][1] - ref);
                        l_run[b][h] += p0 + p1;
                        // 0 of a token that the row does not see, whatever its scale
                        pr[h] = !BITS8 ? p0 : vis >> (b * 4 + h) & 1 ? p0 * vfac[0] : 0.f; pr[2 + h] = !BITS8 ? p1 : vis >> (b * 4 + 2 + h) & 1 ? p1 * vfac[1] : 0.f;
                    }
                    if (BITS8) { pb[b][0] = transpose_8x8(pack_f16x2(pr[0], pr[1])); pb[b][1] = transpose_8x8(pack_f16x2(pr[2], pr[3])); }
                    else { pb[b][0] = transpose_8x8(pack_bf16x2(pr[0], pr[1])); pb[b][1] = transpose_8x8(pack_bf16x2(pr[2], pr[3])); }
                }
                // values of tokens 2 t, 2 t + 1 and these + 8; what nobody sees may be anything, and 0 x inf is not 0
                uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                if (special) {
                    keep0 = (any_lo >> (8 * t) & 0xfu ? 0xffffu : 0u) | (any_lo >> (8 * t + 4) & 0xfu ? 0xffff0000u : 0u);
                    keep1 = (any_hi >> (8 * t) & 0xfu ? 0xffffu : 0u) | (any_hi >> (8 * t + 4) & 0xfu ? 0xffff0000u : 0u);
                }
                if constexpr (BITS8) {
                    const int r = quarter * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                    for (int i = 0; i < KH; i += 2) {
                        uint32_t w[4], vf[2][4];
                        ldmatrix_x4_trans(vbase + few_off8<D>(r, i + (lane >> 4)), w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int e = 0; e < 2; ++e) { to_f16<FMT, true>(w[2 * e], vf[e][0], vf[e][1]); to_f16<FMT, true>(w[2 * e + 1], vf[e][2], vf[e][3]); }
                        if (special)
#pragma unroll
                            for (int e = 0; e < 2; ++e) { vf[e][0] &= keep0; vf[e][1] &= keep0; vf[e][2] &= keep1; vf[e][3] &= keep1; }
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int b = 0; b < NB; ++b) mma_of<FMT>(oacc[b][i + e], vf[e][0], vf[e][1], vf[e][2], vf[e][3], pb[b][0], pb[b][1]);
                    }
                } else {
                    const int r = quarter * 16 + ((lane >> 4) << 3) + (lane & 7), dsel = ((lane >> 3) & 1) << 3;
                    uint32_t vf[KH][4];
#pragma unroll
                    for (int i = 0; i < KH; ++i) ldmatrix_x4_trans(vbase + few_off<D>(r, (half * KH + i) * 16 + dsel), vf[i][0], vf[i][1], vf[i][2], vf[i][3]);
                    if (special)
#pragma unroll
                        for (int i = 0; i < KH; ++i) { vf[i][0] &= keep0; vf[i][1] &= keep0; vf[i][2] &= keep1; vf[i][3] &= keep1; }
#pragma unroll
                    for (int i = 0; i < KH; ++i)
#pragma unroll
                        for (int b = 0; b < NB; ++b) mma_of<FMT>(oacc[b][i], vf[i][0], vf[i][1], vf[i][2], vf[i][3], pb[b][0], pb[b][1]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[st]);
        }
        pages += c1 - c0;
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[n_items & 1]);
        // the states of the quarters (of either group's), for the warp that brings them together while this one goes on
        mbar_wait(states_empty, (n_items & 1) ^ 1);
        const int state = group * 4 + quarter;
        float* mine = states + (state * Cfg::REGS + half * (Cfg::REGS / Cfg::PARTS)) * 32 + lane;                // value [part][b][i][e]
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float l = l_run[b][h];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                if (half == 0 && g == 0) *reinterpret_cast<float2*>(ml_s + (state * ROWS + b * 8 + 2 * t + h) * 2) = make_float2(m_run[b][h], l);
            }
#pragma unroll
            for (int i = 0; i < KH; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[((b * KH + i) * 4 + e) * 32] = oacc[b][i][e];
        }
        if (BITS8 && lane == 0) vref_s[state] = vref * (1.0f / kValueUp);
        __syncwarp();
        if (lane == 0) mbar_arrive(states_full);
    }
    griddep_launch();                            // not before: the next kernel's CTAs would crowd onto the SMs that are done first
}

// =============================================================================================
// more rows: tcgen05
// =============================================================================================
// 128 rows of an item (as many tokens' heads of a group as fit) x 128 keys a tile: S = Q K^T in three TMEM buffers, two tiles ahead, P over S's own columns as the second product's operand, O in
// TMEM.  Two softmax warpgroups take the tiles in turn, one row a thread; the reference maximum rises (and O is rescaled) only where a score passes it by 2^8.  Over 8 bits four warps turn tiles (and
// an item's queries) into fp16 under the swizzle that the products read, and one brings the scales of a tile's values under one power of two.
struct TrueTag { static constexpr bool value = true; };
struct FalseTag { static constexpr bool value = false; };
constexpr int TREE_OVER = 2;                                                     // tiles that an item's beginning and end cost

// what any row of an item sees: bits of new tokens, and the first cached place of the widest window
struct TreeAny {
    uint64_t seen; int low;
    OA_DEVINL bool sees(const TreeAttnArgs& a, const TreeSeq& s, int key) const {
        const int n = key - s.ctx;
        return n < 0 ? key < a.sinks || key >= low : key < s.end && n < 64 && (seen >> (n & 63) & 1);
    }
};
// A CTA's piece of an item: key tiles c0 .. c1 - 1 (none where its units are the item's own alone), of which those before s0 and from s1 on have places that some row may not see; what each row sees.  Made
// by a warp of its own, a piece ahead of the others: each of its looks into the arrays is a latency of L2
struct TreePiece {
    uint64_t seen[128]; int low[128]; float factor[128];                         // factor: of a row's scores
    TreeSeq s; TreeAny any;
    int c0, c1, s0, s1, seq, kvh, row0, rows;
    bool first, last, more;                                                      // the CTA has the item's begin, its end; another piece follows
};

template <int D, int FMT>
struct ManyCfg {
    static constexpr bool BITS8 = FMT != CACHE_BF16;
    static constexpr int KEYS = 128, HALVES = D / 64, HALF = 128 * 128;          // 128 rows x 64 channels of 2 bytes under the 128-byte swizzle: of Q, of a tile
    static constexpr int TILE_BYTES = HALVES * HALF, SLOTS = BITS8 ? (D == 128 ? 3 : 4) : D == 128 ? 5 : 8;
    static constexpr int RAW_BYTES = KEYS * D, RAW = BITS8 ? (D == 128 ? 5 : 8) : 0;         // a tile of 8 bits, and how many wait
    static constexpr int SC = 8, SC_FLOATS = 2 * KEYS + 4;                       // tiles whose scales wait: keys', values', what scores are multiplied by, what O is for larger scales of values and at its end
    static constexpr int CONV = BITS8 ? 8 : 0, THREADS = 128 + 256 + 32 * CONV;     // producer, issuer, scales, pieces; eight softmax warps; warps that convert
    static constexpr int BARS = 18 + 2 * SLOTS + 2 * RAW + (BITS8 ? 2 * SC : 0);
    static constexpr int SMEM_BYTES = TILE_BYTES + SLOTS * TILE_BYTES + RAW * RAW_BYTES + (BITS8 ? SC * SC_FLOATS * 4 : 0) + 3 * 128 * 4 + BARS * 8 + 16 + 2 * sizeof(TreePiece);
    static constexpr uint32_t O_COL = 384;                                       // TMEM: S and P of the tiles in turn at 0, 128 and 256
};
OA_DEVINL uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }
// which of the 64 places from `key` on a row sees
OA_DEVINL uint64_t tree_word(const TreeAttnArgs& a, const TreeSeq& s, uint64_t seen, int low, int key) {
    const uint64_t old = low_bits(s.ctx - key) & (low_bits(a.sinks - key) | ~low_bits(low - key));
    const int d = s.ctx - key;
    const uint64_t fresh = d >= 64 || d <= -64 ? 0ull : d >= 0 ? seen << d : seen >> -d;
    return (old | fresh) & low_bits(s.end - key);
}

// Queries in fp16, a row of a head under a power of two that brings its largest magnitude to [2^14, 2^15): a warp eight rows.  What the next kernel reads besides was written by kernels that have ended
template <int D>
__global__ void __launch_bounds__(128) tree_queries_kernel(const __grid_constant__ TreeAttnArgs a) {
    constexpr int W = D / 64, ROWS = 8;                                          // words of two channels a lane
    const int lane = threadIdx.x & 31;
    const int64_t total = (int64_t)a.n_rows * a.n_heads, r0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * ROWS;
    griddep_wait();
    griddep_launch();
    uint32_t x[ROWS][W];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int64_t token = quotient(r0 + i, a.n_heads);
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + token * a.ldq + (r0 + i - token * a.n_heads) * D + lane * 2 * W;
#pragma unroll
        for (int j = 0; j < W; ++j) x[i][j] = 0u;
        if (r0 + i < total) { if (W == 2) { const uint2 y = __ldcg(reinterpret_cast<const uint2*>(src)); x[i][0] = y.x; x[i][W - 1] = y.y; } else x[i][0] = __ldcg(reinterpret_cast<const uint32_t*>(src)); }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < W; ++j) top = max(top, max(x[i][j] << 16 & 0x7fffffffu, x[i][j] & 0x7fff0000u));
        top = __reduce_max_sync(0xffffffffu, top);
        if (r0 + i >= total) return;
        const int e = top >= 0x7f800000u ? 14 : max((int)(top >> 23) - 127, -100);           // not finite: as it is
        const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        uint32_t* dst = a.q16 + (r0 + i) * (D / 2) + lane * W;
#pragma unroll
        for (int j = 0; j < W; ++j) x[i][j] = pack_f16x2(bf16lo(x[i][j]) * up, bf16hi(x[i][j]) * up);
        if (W == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(x[i][0], x[i][W - 1]); else dst[0] = x[i][0];
        if (lane == 0) a.q_factor[r0 + i] = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
    }
}

template <int D, int FMT>
__global__ void __launch_bounds__(ManyCfg<D, FMT>::THREADS, 1) tree_many_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ TreeAttnArgs a) {
    using Cfg = ManyCfg<D, FMT>;
    using At = TreeAt<2, TREE_OVER>;
    constexpr bool BITS8 = Cfg::BITS8;
    constexpr int KEYS = Cfg::KEYS, HALVES = Cfg::HALVES, HALF = Cfg::HALF, TILE = Cfg::TILE_BYTES, SLOTS = Cfg::SLOTS, RAW = BITS8 ? Cfg::RAW : 1, SC = Cfg::SC, SOFTMAX = 256;
    constexpr int64_t BLOCK_BYTES = CACHE_PAGE * (D + 4);
    constexpr float kKeyUp = FMT == CACHE_INT8 ? 1.0f / 512.f : 64.f;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_s = smem;
    uint8_t* kv_s = q_s + TILE;
    uint8_t* raw_s = kv_s + SLOTS * TILE;
    float* sc_s = reinterpret_cast<float*>(raw_s + Cfg::RAW * Cfg::RAW_BYTES);
    float* m_s = sc_s + (BITS8 ? SC * Cfg::SC_FLOATS : 0);                                   // a row's reference maximum, and its two sums of a piece
    float* l_s = m_s + 128;
    uint64_t* bars = reinterpret_cast<uint64_t*>(l_s + 256);
    uint64_t *q_full = bars, *q_empty = bars + 1, *s_full = bars + 2, *p_full = bars + 5, *o_full = bars + 8, *full = bars + 12, *empty = full + SLOTS;
    uint64_t *piece_full = empty + SLOTS, *rows_full = piece_full + 2, *piece_empty = rows_full + 2, *raw_full = piece_empty + 2, *raw_empty = raw_full + Cfg::RAW, *sc_full = raw_empty + Cfg::RAW, *sc_empty = sc_full + SC;
    TreePiece* piece_s = reinterpret_cast<TreePiece*>(bars + Cfg::BARS);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(piece_s + 2);
    __shared__ int64_t sums[Cfg::THREADS / 32];
    __shared__ At start;
    __shared__ float sc_last;                                                    // 8 bits: what the values' scales of a piece's last tile are over

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv, tile_tokens = 128 / grp;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_q);
        if (!BITS8) tma_prefetch_desc(&tm_kv);
        mbar_init(q_full, 1); mbar_init(q_empty, 1);
        for (int i = 0; i < 3; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); }
        for (int i = 0; i < 4; ++i) mbar_init(&o_full[i], 1);
        for (int i = 0; i < 2; ++i) { mbar_init(&piece_full[i], 1); mbar_init(&rows_full[i], 1); mbar_init(&piece_empty[i], BITS8 ? 11 + Cfg::CONV : 10); }
        for (int i = 0; i < SLOTS; ++i) { mbar_init(&full[i], BITS8 ? Cfg::CONV : 1); mbar_init(&empty[i], 1); }
        if (BITS8) {
            for (int i = 0; i < RAW; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], Cfg::CONV); }
            for (int i = 0; i < SC; ++i) { mbar_init(&sc_full[i], 1); mbar_init(&sc_empty[i], 4 + Cfg::CONV); }
        }
        fence_barrier_init();
    }
    // Tensor memory is taken behind the wait: a kernel before this one that has not taken its own yet would otherwise wait for this one, and this one for it.  8 bits: the kernel before this one is the
    // queries', which takes none and has let this one start behind its own wait; only what it writes is waited for, later
    if (!BITS8) griddep_wait();
    if (warp == 1) tmem_alloc<512>(tmem_slot);
    const TreeShare share = tree_share<Cfg::THREADS>(a, tile_tokens, sums, start);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int64_t u_begin = share.begin, u_end = share.end;
    // what a warp does with each piece; p lies in shared memory until it is done.  What rows see comes a latency later
    auto pieces = [&](bool rows, auto&& work) {
        if (u_begin >= u_end) return;
        for (uint32_t k = 0;; ++k) {
            mbar_wait(&piece_full[k & 1], (k >> 1) & 1);
            const TreePiece& p = piece_s[k & 1];
            if (rows) mbar_wait(&rows_full[k & 1], (k >> 1) & 1);
            const bool more = p.more;
            work(p);
            __syncwarp();
            if (lane == 0) mbar_arrive(&piece_empty[k & 1]);
            if (!more) return;
        }
    };

    // Keys and values share one ring in the order of their products: K_0, K_1, K_2, V_0, K_3, V_1, ..: entry number of V_j is min(tiles, j + 3) + j
    // 8 bits: 96 registers a thread at launch, 480 for five warpgroups: 64 + 2 x 136 + 2 x 72.  A warpgroup's split is the same instruction for all of it, in the branch that lives by it
    if (warp < 4) {
        if constexpr (BITS8) reg_dec<64>();
        if (warp == 0) {
            constexpr int RING = BITS8 ? RAW : SLOTS;
            uint64_t *in = BITS8 ? raw_full : full, *out = BITS8 ? raw_empty : empty;
            uint32_t n = 0, seg = 0;                                                 // entries and pieces loaded
            pieces(false, [&](const TreePiece& p) {
                const int c0 = p.c0, c1 = p.c1;
                if (c1 == c0) return;
                bool q_due = true;
                auto load_q = [&] {
                    mbar_wait(q_empty, (seg & 1) ^ 1);
                    if (BITS8 && seg == 0) { griddep_wait(); fence_proxy_async_all(); }          // written by threads of the kernel before
                    if (elect_one()) {                                               // tokens behind the last row are zeros, other sequences' are not looked at
                        mbar_expect_tx(q_full, HALVES * tile_tokens * grp * 128);
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) tma_load_3d(q_s + h * HALF, &tm_q, q_full, h * 64, p.kvh * grp, p.row0, kEvictNormal);
                    }
                    __syncwarp();
                    ++seg;
                    q_due = false;
                };
                if (!BITS8) load_q();
                const int32_t* table = a.tables + (int64_t)p.seq * a.max_pages;
                int page[3][2] = {}, have = 0, later = 0;                            // pages of this tile and of the two before
                for (int kt = c0; kt < c1 + 2; ++kt) {
                    if (kt < c1 && (kt == c0 || (kt & 15) == 0)) {                   // 32 page numbers, and the next 32 on their way
                        const int w = (2 * kt & ~31) + lane, stop = min(2 * c1, p.s.pages);
                        have = kt > c0 ? later : w < stop ? __ldcg(table + p.s.page(w)) : 0;
                        later = w + 32 < stop ? __ldcg(table + p.s.page(w + 32)) : 0;
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        page[2][i] = page[1][i]; page[1][i] = page[0][i];
                        page[0][i] = __shfl_sync(0xffffffffu, have, (2 * kt + i) & 31);
                        if (kt >= c1 || 2 * kt + i >= p.s.pages) page[0][i] = 0;
                        if (page[0][i] < 0 || page[0][i] >= a.num_pages) { if (lane == 0 && a.status) *a.status = 400; page[0][i] = 0; }
                    }
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int t = kt - 2 * v;                                    // K of this tile, V of the one two before
                        if (t < c0 || t >= c1) continue;
                        const int there = min(2, p.s.pages - 2 * t);                // a missing second page is not loaded: its scores are masked, its values set to zero
                        const uint32_t slot = n % RING;
                        mbar_wait(&out[slot], ((n / RING) & 1) ^ 1);
                        if (lane == 0) mbar_expect_tx(&in[slot], there * (BITS8 ? CACHE_PAGE * D : HALVES * 8192));
                        __syncwarp();
                        constexpr int COPIES = BITS8 ? 1 : HALVES;                   // of a page, a lane each: one lane that issues them all takes longer for it than the tile does
                        if (lane < there * COPIES) {
                            const int i = lane / COPIES, h = lane % COPIES;
                            const int64_t block = ((int64_t)v * a.num_pages + (v ? (i ? page[2][1] : page[2][0]) : (i ? page[0][1] : page[0][0]))) * a.n_kv + p.kvh;
                            if (BITS8) bulk_load(raw_s + slot * Cfg::RAW_BYTES + i * CACHE_PAGE * D, reinterpret_cast<const uint8_t*>(a.cache) + block * BLOCK_BYTES, CACHE_PAGE * D, &in[slot]);
                            else tma_load_2d(kv_s + slot * TILE + h * HALF + i * 8192, &tm_kv, &in[slot], h * 64, (int)(block * CACHE_PAGE), kEvictNormal);
                        }
                        __syncwarp();
                        ++n;
                        if (BITS8 && q_due) load_q();                                // behind the first tile of keys, which takes longer to be one
                    }
                }
            });
        } else if (warp == 1) {
            // the whole warp walks the loop, an elected lane issues: descriptors stay in uniform registers
            constexpr uint32_t f16 = BITS8 ? (1u << 7) | (1u << 10) : 0u;            // both operands fp16 instead of bf16
            constexpr uint32_t idesc_s = umma_idesc_bf16(128, KEYS) ^ f16, idesc_o = umma_idesc_bf16_bmn(128, D) ^ f16;
            const uint64_t q_desc = umma_desc_sw128(smem_u32(q_s)), k_desc = umma_desc_sw128(smem_u32(kv_s));
            const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(kv_s), (uint32_t)HALF, 1024u);
            uint32_t n = 0, r = 0, seg = 0;                                          // tiles of the pieces before, entries of the ring, pieces
            auto await = [&] {                                                       // the ring's next tile
                const uint32_t slot = r % SLOTS;
                mbar_wait(&full[slot], (r / SLOTS) & 1);
                ++r;
                tcgen05_fence_after();
                return slot;
            };
            // products of one thread are carried out in the order of their issue: S of a tile goes over scores whose P a product ahead of it reads
            pieces(false, [&](const TreePiece& p) {
                const int tiles = p.c1 - p.c0;
                if (tiles == 0) return;
                mbar_wait(q_full, seg & 1);
                ++seg;
                tcgen05_fence_after();
                for (int j = -2; j < tiles; ++j) {
                    if (j + 2 < tiles) {                                             // scores two tiles ahead, under the softmaxes of the tiles before
                        const uint32_t slot = await(), to = (n + j + 2) % 3;
                        if (elect_one()) {
                            const uint64_t b = k_desc + (uint64_t)(slot * (TILE >> 4));
#pragma unroll
                            for (int ks = 0; ks < D / 16; ++ks) {
                                const int half = ks >> 2, in = (ks & 3) * 32;
                                umma_bf16(tmem_base + to * 128, q_desc + (uint64_t)((half * HALF + in) >> 4), b + (uint64_t)((half * HALF + in) >> 4), idesc_s, ks > 0 ? 1u : 0u);
                            }
                            umma_commit(&s_full[to]);
                            umma_commit(&empty[slot]);
                            if (j + 3 == tiles) umma_commit(q_empty);
                        }
                        __syncwarp();
                    }
                    if (j >= 0) {
                        const uint32_t m = n + j, from = m % 3;
                        mbar_wait(&p_full[from], (m / 3) & 1);
                        const uint32_t slot = await();
                        if (elect_one()) {
                            const uint64_t b = v_desc + (uint64_t)(slot * (TILE >> 4));
#pragma unroll
                            for (int ks = 0; ks < KEYS / 16; ++ks)
                                umma_bf16_ta(tmem_base + Cfg::O_COL, tmem_base + from * 128 + ks * 8, b + (uint64_t)(ks * (2048 >> 4)), idesc_o, (j > 0 || ks > 0) ? 1u : 0u);
                            umma_commit(&o_full[m & 3]);
                            umma_commit(&empty[slot]);
                        }
                        __syncwarp();
                    }
                }
                n += tiles;
            });
        } else if (warp == 2) {
            // A tile's scales in fp16, twice: keys' over a power of two that none of the tile passes and times 2^6 (int8: 2^-9), values' over one that none of the piece so far passes and times 2^7, which bring the
            // largest product to 28672 (0.25) and 57344; 0 of what none of the rows sees.  int8 keys u - 128 times s are the fused product u 2^-24 (a subnormal's bits) times s 2^24 less 128 s
            if constexpr (BITS8) {
                uint32_t n = 0;
                pieces(true, [&](const TreePiece& p) {
                    const int c0 = p.c0, c1 = p.c1, stop = min(2 * c1, p.s.pages);
                    const int32_t* table = a.tables + (int64_t)p.seq * a.max_pages;
                    int have = 0, later = 0;
                    auto entry = [&](int w) { return w < stop ? __ldcg(table + p.s.page(w)) : 0; };
                    // four keys' and values' scales a lane, a tile ahead; a bad page number is told where its bytes are loaded
                    auto load = [&](int kt, float4 (&x)[2]) {
                        if (kt == c0 || (kt & 15) == 0) { have = kt == c0 ? entry((2 * kt & ~31) + lane) : later; later = entry((2 * kt & ~31) + 32 + lane); }
                        const int w = 2 * kt + (lane >> 4);
                        int page = __shfl_sync(0xffffffffu, have, w & 31);
                        if (page < 0 || page >= a.num_pages) page = 0;
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            x[v] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (w < stop) x[v] = __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const uint8_t*>(a.cache) + (((int64_t)v * a.num_pages + page) * a.n_kv + p.kvh) * BLOCK_BYTES + CACHE_PAGE * D) + (lane & 15));
                        }
                    };
                    float4 ahead[2];
                    if (c0 < c1) load(c0, ahead);
                    float vref = 0.f;
                    for (int kt = c0; kt < c1; ++kt, ++n) {
                        const uint32_t buf = n % SC;
                        float* sc = sc_s + buf * Cfg::SC_FLOATS;
                        const bool sp = kt < p.s0 || kt >= p.s1;
                        const float4 in[2] = {ahead[0], ahead[1]};
                        if (kt + 1 < c1) load(kt + 1, ahead);
                        mbar_wait(&sc_empty[buf], ((n / SC) & 1) ^ 1);
                        uint32_t mask = 0xf;
                        if (sp) {
                            const int c = 2 * kt + (lane >> 4);
                            mask = 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i) if (c < p.s.pages && p.any.sees(a, p.s, p.s.page(c) * CACHE_PAGE + (4 * lane & 63) + i)) mask |= 1u << i;
                        }
                        float grown = 1.0f, ref[2] = {0.f, vref};
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            float x[4] = {in[v].x, in[v].y, in[v].z, in[v].w};
                            uint32_t top = 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (!(mask >> i & 1)) x[i] = 0.f;
                                if (fabsf(x[i]) < INFINITY) top = max(top, __float_as_uint(fabsf(x[i])));
                            }
                            top = __reduce_max_sync(0xffffffffu, top);
                            const float need = __uint_as_float(min((top & 0x7f800000u) + 0x00800000u, 0x7e800000u));             // up to 2^126
                            if (need > ref[v]) { if (ref[v] > 0.f) grown = ref[v] * (1.0f / need); ref[v] = need; }
                            const float inv = 1.0f / ref[v], up = v ? 128.f : kKeyUp;        // powers of two: exact
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float y = x[i] * inv * up;
                                w[i] = pack_f16x2(y, y);
                                if (!v && FMT == CACHE_INT8) {                       // s 2^24 and -128 s, of the same s
                                    const float r = __half2float(__float2half_rn(y * 16777216.f));
                                    w[i] = pack_f16x2(r, r * (-128.f / 16777216.f));
                                }
                            }
                            *reinterpret_cast<uint4*>(sc + v * KEYS + 4 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        vref = ref[1];
                        if (lane == 0) { sc[2 * KEYS] = ref[0] * (1.0f / kKeyUp); sc[2 * KEYS + 1] = grown; sc[2 * KEYS + 2] = vref * (1.0f / 128.f); }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sc_full[buf]);
                    }
                });
            }
        } else {
            At at;
            at = start;
            uint32_t k = 0;
            for (int64_t u = u_begin; u < u_end; at.next(a), ++k) {
                const int64_t end = at.unit0 + at.units();
                const int c0 = (int)max(u - at.unit0 - TREE_OVER, (int64_t)0), c1 = (int)max((int64_t)c0, min((int64_t)at.steps(), u_end - at.unit0 - TREE_OVER));
                u = min(end, u_end);
                mbar_wait(&piece_empty[k & 1], ((k >> 1) & 1) ^ 1);
                TreePiece& p = piece_s[k & 1];
                const int rows = at.rows(grp);
                if (lane == 0) {
                    const TreeSeq& s = at.s;
                    p.s = s;
                    p.c0 = c0; p.c1 = c1; p.seq = at.seq; p.kvh = at.kvh; p.row0 = at.row0(); p.rows = rows;
                    p.s0 = a.window > 0 ? (pages_below(s, s.ctx + s.n - a.window) + 1) / 2 : 0; p.s1 = min((s.ctx / CACHE_PAGE - s.skip) / 2, s.pages / 2);
                    p.first = at.unit0 >= u_begin; p.last = end <= u_end; p.more = end < u_end;
                    if (p.first && !p.last) tree_record(a, cta_of(end - 1, share.busy, share.total) - (int)blockIdx.x, p.row0, rows, p.kvh);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&piece_full[k & 1]);
                if (BITS8 && k == 0) griddep_wait();                             // the queries in fp16 are there
                uint64_t any = 0; int lowest = 0x7fffffff;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = i * 32 + lane, token = r / grp;
                    uint64_t seen = 0; int low = 0x7fffffff; float factor = a.scale_log2e;
                    if (r < rows) {
                        const int t = at.tile * tile_tokens + token;
                        seen = tree_seen(a, at.s, t); low = tree_low(a, at.s, seen, t);
                        if (BITS8) factor *= __ldcg(a.q_factor + (int64_t)(at.row0() + token) * a.n_heads + at.kvh * grp + r - token * grp);
                    }
                    p.seen[r] = seen; p.low[r] = low; p.factor[r] = factor;
                    any |= seen; lowest = min(lowest, low);
                }
                any = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(any >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)any);
                lowest = __reduce_min_sync(0xffffffffu, lowest);
                if (lane == 0) { p.any.seen = any; p.any.low = lowest; }
                __syncwarp();
                if (lane == 0) mbar_arrive(&rows_full[k & 1]);
            }
        }
    } else if (warp < 12) {
        if constexpr (BITS8) reg_inc<136>();
        // Two warpgroups take the tiles in turn, a row a thread: one's exponentials run under the other's loads and maxima.  A row's reference maximum goes from one to the other
        // with each tile, as soon as the tile's own maximum is known; sums stay with either, O is one for both
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t wg = (warp - 4) >> 2, lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16), o_addr = lane_addr + Cfg::O_COL;
        auto meet = [] { asm volatile("bar.sync 2, %0;" ::"n"(SOFTMAX) : "memory"); };
        auto take_turn = [](uint32_t n) {                                        // tile n - 1 has left its reference
            if (n & 1) asm volatile("bar.sync 3, %0;" ::"n"(SOFTMAX) : "memory"); else asm volatile("bar.sync 4, %0;" ::"n"(SOFTMAX) : "memory");
        };
        auto pass_turn = [](uint32_t n) {                                        // to tile n
            if (n & 1) asm volatile("bar.arrive 3, %0;" ::"n"(SOFTMAX) : "memory"); else asm volatile("bar.arrive 4, %0;" ::"n"(SOFTMAX) : "memory");
        };
        constexpr float kRaise = 8.0f;                                           // log2 units a score may pass the reference by
        constexpr float kLift = BITS8 ? 7.0f : 0.0f;                             // of the weights, which fp16 holds up to 2^16 and with 8 bits down to 2^-17
        constexpr int COLS = D / 2;
        uint32_t n0 = 0;                                                         // tiles of the pieces before
        pieces(true, [&](const TreePiece& p) {
            const TreeSeq& s = p.s;
            const int c0 = p.c0, tiles = p.c1 - p.c0;
            const bool live = row < p.rows, first = p.first;
            const uint32_t n1 = n0 + tiles;
            const uint64_t seen = p.seen[row]; const int low = p.low[row];
            const bool blind = live && !tree_sees(a, s, seen, low);
            float* po = a.part_o + ((int64_t)blockIdx.x * 2 + !first) * (128 * D) + row * 4;         // [D / 4][128 rows][4]: a warp's rows lie next to each other
            float2* ml = reinterpret_cast<float2*>(a.part_ml) + ((int64_t)blockIdx.x * 2 + !first) * 128 + row;
            if (tiles == 0) {                                                    // units of the item's own alone
                if (live)
                    for (int c = wg * COLS; c < (int)(wg + 1) * COLS; c += 4) *reinterpret_cast<float4*>(po + c * 128) = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live && wg == 0) *ml = make_float2(-INFINITY, first && blind ? -1.f : 0.f);
                return;
            }
            const float row_fac = p.factor[row];
            float undo = 1.0f;
            float m_mine = -INFINITY, l_run = 0.f;                               // the sum so far and the reference that it is under
            auto clear_unseen = [&](uint32_t n) {
                const int kt = c0 + (int)(n - n0);
                    // values that none of the rows sees may be anything, and 0 x inf is not 0: a thread looks after the key of its row's number
                    const uint32_t entry = 2 * n0 + min(tiles, kt - c0 + 3) + (kt - c0), slot = entry % SLOTS;
                    mbar_wait(&full[slot], (entry / SLOTS) & 1);
                    const int c = 2 * kt + (row >> 6);
                    if (c >= s.pages || !p.any.sees(a, s, s.page(c) * CACHE_PAGE + (row & 63))) {
#pragma unroll
                        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(kv_s + slot * TILE + (c >> 3) * HALF + row * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async();
            };
            // a warp without rows keeps the others' pace and clears the keys that it looks after
            auto pace = [&](uint32_t n, bool special) {
                const uint32_t from = n % 3;
                mbar_wait(&s_full[from], (n / 3) & 1);
                if (n > n0) take_turn(n);
                if (n > 2) mbar_wait(&o_full[(n - 3) & 3], ((n - 3) >> 2) & 1);
                if (n + 1 < n1) pass_turn(n + 1);
                if (special && !BITS8) clear_unseen(n);
                if (BITS8) undo = sc_s[n % SC * Cfg::SC_FLOATS + 2 * KEYS + 2];
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&p_full[from]); if (BITS8) mbar_arrive(&sc_empty[n % SC]); }
            };
            const bool idle = quarter * 32 >= p.rows;
            auto tile = [&](uint32_t n, auto tag) {
                constexpr bool SPECIAL = decltype(tag)::value;
                const int kt = c0 + (int)(n - n0);
                const uint32_t from = n % 3, s_addr = lane_addr + from * 128, buf = n % SC;
                uint64_t word[2] = {~0ull, ~0ull};
                if (SPECIAL) {
                    word[0] = tree_word(a, s, seen, low, s.page(2 * kt) * CACHE_PAGE);
                    word[1] = 2 * kt + 1 < s.pages ? tree_word(a, s, seen, low, s.page(2 * kt + 1) * CACHE_PAGE) : 0ull;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};     // four chains
                mbar_wait(&s_full[from], (n / 3) & 1);                           // the tile's scales, which its keys were turned with, are there too
                tcgen05_fence_after();
                float grown = 1.0f, fac = row_fac;
                if (BITS8) {
                    const float* sc = sc_s + buf * Cfg::SC_FLOATS + 2 * KEYS;
                    fac *= sc[0]; grown = sc[1]; undo = sc[2];
                }
                uint32_t v[2][32];
                auto scores = [&](int k) {                                       // of keys k .. k + 63, -inf where the row does not see
                    tmem_ld_32x32b_x32(s_addr + k, v[0]);
                    tmem_ld_32x32b_x32(s_addr + k + 32, v[1]);
                    tmem_ld_wait();
                    if (SPECIAL) {
                        const uint64_t w = k ? word[1] : word[0];
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i) if (!((uint32_t)(w >> (c * 32)) >> i & 1)) v[c][i] = 0xff800000u;
                    }
                };
#pragma unroll 1
                for (int k = KEYS - 64; k >= 0; k -= 64) {                       // the lower keys last: they stay in registers
                    scores(k);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[c][i]));
                }
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * fac;
                if (n > n0) take_turn(n);
                // A barrier's phases are seen one by one: PV of the tile three before is the last one that this tile can be sure of without a wait
                if (n > 2) mbar_wait(&o_full[(n - 3) & 3], ((n - 3) >> 2) & 1);
                const float m_last = n > n0 ? m_s[row] : -INFINITY;
                const bool raise = live && mx > m_last + kRaise;
                const float m_ref = raise ? mx : m_last;
                m_s[row] = m_ref;
                if (n + 1 < n1) pass_turn(n + 1);
                if (n > n0 && (grown != 1.0f || __any_sync(0xffffffffu, raise))) {
                    mbar_wait(&o_full[(n - 1) & 3], ((n - 1) >> 2) & 1);         // O has the products of all tiles before; this tile's are not issued before p_full
                    tcgen05_fence_after();
                    const float alpha = (raise ? exp2f(m_last - m_ref) : 1.0f) * grown;
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(o_addr + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st_32x32b_x16(o_addr + c, o);
                    }
                }
                if (SPECIAL && !BITS8) clear_unseen(n);
                if (m_mine != m_ref) { l_run *= ex2_approx(m_mine - m_ref); m_mine = m_ref; }
                const float neg_ref = kLift - finite_or_zero(m_ref);
                uint64_t sum = 0;
#pragma unroll 1
                for (int k = 0; k < KEYS; k += 64) {
                    if (k > 0) scores(k);                                        // read again: P of the keys before lies over their own scores
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = ex2_approx(fmaf(__uint_as_float(v[c][2 * i]), fac, neg_ref)), y = ex2_approx(fmaf(__uint_as_float(v[c][2 * i + 1]), fac, neg_ref));
                            sum = add_f32x2(sum, pack_f32x2(x, y));
                            w[i] = BITS8 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
                        }
                        tmem_st_32x32b_x16(s_addr + k / 2 + c * 16, w);
                    }
                }
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&p_full[from]); if (BITS8) mbar_arrive(&sc_empty[buf]); }
                float lo, hi; unpack_f32x2(sum, lo, hi);
                l_run += lo + hi;
            };
            for (uint32_t n = n0 + ((n0 ^ wg) & 1); n < n1; n += 2) {
                const int kt = c0 + (int)(n - n0);
                const bool special = kt < p.s0 || kt >= p.s1;
                if (idle) pace(n, special); else if (special) tile(n, TrueTag{}); else tile(n, FalseTag{});
            }
            n0 = n1;
            meet();                                                              // the last tile's reference is there
            const float m_ref = m_s[row];
            if (m_mine != m_ref) l_run *= ex2_approx(m_mine - m_ref);
            l_s[wg * 128 + row] = l_run;
            if (BITS8 && ((n1 - 1) & 1) == wg && row == 0) sc_last = undo;
            meet();
            const float l = l_s[row] + l_s[128 + row];
            if (BITS8) undo = sc_last;
            mbar_wait(&o_full[(n1 - 1) & 3], ((n1 - 1) >> 2) & 1);
            tcgen05_fence_after();
            const bool whole = first && p.last;
            const float mult = undo * (whole ? (blind ? 0.f : 1.0f / l) : 1.0f);
            const int token = row / grp;
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(p.row0 + token) * a.ldo + (int64_t)(p.kvh * grp + row - token * grp) * D;
#pragma unroll 1
            for (int c = wg * COLS; c < (int)(wg + 1) * COLS; c += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_addr + c, o);
                tmem_ld_wait();
                if (!live) continue;
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * mult);
                if (whole) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
#pragma unroll
                    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(out + c + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                } else
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(po + (c + i) * 128) = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
            }
            tcgen05_fence_before();
            if (live && !whole && wg == 0) *ml = make_float2(m_ref - kLift, first && blind ? -1.f : l);
            meet();                                                              // O and the sums may be written again
        });
    } else {
        if constexpr (BITS8) reg_dec<72>();
        // tiles in the ring's order, 16 channels of a key a step
        if constexpr (BITS8) {
            const int w = warp - 12, tid = w * 32 + lane;
            // 16 channels of a key a step.  Heads of 128: eight lanes take the lower half of one key and the upper of its neighbour, then the other way round, so that neither loads nor stores meet on a bank
            constexpr int STEPS = Cfg::RAW_BYTES / 16 / (32 * Cfg::CONV), AHEAD = STEPS < 4 ? STEPS : 4;
            const int ch = tid % (D / 16);
            auto key_of = [&](int i) { return D == 128 ? 2 * ((tid >> 3) + 4 * Cfg::CONV * (i >> 1)) + ((ch >> 2) ^ (i & 1)) : (tid >> 2) + 8 * Cfg::CONV * i; };
            uint32_t n = 0, g = 0;                                               // entries, tiles of the pieces before
            pieces(true, [&](const TreePiece& p) {
                const int c0 = p.c0, tiles = p.c1 - p.c0;
                if (tiles == 0) return;
#pragma unroll 1
                for (int e = 0; e < 2 * tiles + 4; ++e) {                        // K of a tile, V of the one two before
                    const int t = (e >> 1) - 2 * (e & 1);
                    if (t < 0 || t >= tiles) continue;
                    const uint32_t from = n % RAW, to = n % SLOTS;
                    const uint32_t* sc = reinterpret_cast<const uint32_t*>(sc_s + (g + t) % SC * Cfg::SC_FLOATS + (e & 1) * KEYS);
                    // keys' scales came with theirs for values.  Asked together: an answer takes 140 cycles
                    mbar_wait3(&raw_full[from], (n / RAW) & 1, &empty[to], ((n / SLOTS) & 1) ^ 1, &sc_full[(g + t) % SC], ((g + t) / SC) & 1);
                    const uint8_t* src = raw_s + from * Cfg::RAW_BYTES + ch * 16;
                    uint8_t* dst = kv_s + to * TILE + (ch >> 2) * HALF;
                    auto convert = [&](auto tag) {
                    constexpr bool KEY = decltype(tag)::value;
#pragma unroll
                    for (int h = 0; h < STEPS; h += AHEAD) {                     // loads ahead of their stores
                        uint4 x[AHEAD]; uint32_t f[AHEAD];
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i) { x[i] = *reinterpret_cast<const uint4*>(src + key_of(h + i) * D); f[i] = sc[key_of(h + i)]; }
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i) {
                            uint32_t y[8];
                            const uint32_t w4[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                            if (FMT == CACHE_INT8 && KEY) {
                                const uint32_t mul = __byte_perm(f[i], 0, 0x1010), add = __byte_perm(f[i], 0, 0x3232);
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint32_t u = w4[k] ^ 0x80808080u;
                                    y[2 * k] = fma_f16x2(__byte_perm(u, 0, 0x4140), mul, add); y[2 * k + 1] = fma_f16x2(__byte_perm(u, 0, 0x4342), mul, add);
                                }
                            } else
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    to_f16<FMT, false>(w4[k], y[2 * k], y[2 * k + 1]);
                                    y[2 * k] = mul_f16x2(y[2 * k], f[i]); y[2 * k + 1] = mul_f16x2(y[2 * k + 1], f[i]);
                                }
                            const int key = key_of(h + i);
                            *reinterpret_cast<uint4*>(dst + key * 128 + (((2 * (ch & 3)) ^ (key & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
                            *reinterpret_cast<uint4*>(dst + key * 128 + (((2 * (ch & 3) + 1) ^ (key & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
                        }
                    }
                    };
                    if (e & 1) convert(FalseTag{}); else convert(TrueTag{});
                    if ((e & 1) && (c0 + t < p.s0 || c0 + t >= p.s1))                              // values that none of the rows sees may be anything, and 0 x inf is not 0
#pragma unroll 1
                        for (int i = 0; i < STEPS; ++i) {
                            const int key = key_of(i), pg = 2 * (c0 + t) + (key >> 6);
                            if (pg < p.s.pages && p.any.sees(a, p.s, p.s.page(pg) * CACHE_PAGE + (key & 63))) continue;
                            *reinterpret_cast<uint4*>(dst + key * 128 + (((2 * (ch & 3)) ^ (key & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
                            *reinterpret_cast<uint4*>(dst + key * 128 + (((2 * (ch & 3) + 1) ^ (key & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(&raw_empty[from]); mbar_arrive(&full[to]); if (e & 1) mbar_arrive(&sc_empty[(g + t) % SC]); }
                    ++n;
                }
                g += tiles;
            });
        }
    }
    if (BITS8) griddep_wait();                   // also a CTA without units: what follows this kernel follows the queries' too
    __syncthreads();
    griddep_launch();
    if (warp == 1) { tcgen05_fence_after(); tmem_dealloc<512>(tmem_base); }
}

// =============================================================================================
// the join
// =============================================================================================
// Of the item that a CTA began and others ended: a thread eight channels of a row
constexpr int TREE_JOIN_THREADS = 128;
template <int D>
__global__ void __launch_bounds__(TREE_JOIN_THREADS) tree_join_kernel(const __grid_constant__ TreeAttnArgs a) {
    const int cta = blockIdx.x, x = blockIdx.y * TREE_JOIN_THREADS + threadIdx.x, row = x % a.rows, c = x / a.rows * 8, grp = a.n_heads / a.n_kv;
    griddep_launch();
    griddep_wait();
    const int parts = __ldcg(&a.joins[cta].parts);
    if (parts == 0 || c >= D || row >= __ldcg(&a.joins[cta].rows)) return;
    const int row0 = __ldcg(&a.joins[cta].row0), kvh = __ldcg(&a.joins[cta].kvh);
    auto slot = [&](int i) { return i == 0 ? (int64_t)cta * 2 : (int64_t)(cta + i) * 2 + 1; };
    float M = -INFINITY, l = 0.f; float acc[8] = {};
    bool blind = false;
    constexpr int MP = 4;
    for (int i0 = 0; i0 <= parts; i0 += MP) {
        float2 ml[MP]; float4 o[MP][2];
#pragma unroll
        for (int p = 0; p < MP; ++p) {
            ml[p] = make_float2(-INFINITY, 0.f); o[p][0] = o[p][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i0 + p > parts) continue;
            const int64_t at = slot(i0 + p) * a.rows;
            ml[p] = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + at + row);
#pragma unroll
            for (int h = 0; h < 2; ++h) o[p][h] = __ldcg(reinterpret_cast<const float4*>(a.part_o + at * D + (int64_t)(c / 4 + h) * (a.rows * 4) + row * 4));
        }
        if (i0 == 0) blind = ml[0].y < 0.f;
        float m = M;
#pragma unroll
        for (int p = 0; p < MP; ++p) m = fmaxf(m, ml[p].x);
        const float ref = finite_or_zero(m), f0 = ex2_approx(M - ref);
        M = m; l *= f0;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= f0;
#pragma unroll
        for (int p = 0; p < MP; ++p) {
            const float f = ex2_approx(ml[p].x - ref);
            l += f * ml[p].y;
#pragma unroll
            for (int h = 0; h < 2; ++h) { acc[4 * h] += f * o[p][h].x; acc[4 * h + 1] += f * o[p][h].y; acc[4 * h + 2] += f * o[p][h].z; acc[4 * h + 3] += f * o[p][h].w; }
        }
    }
    const float inv = blind ? 0.f : 1.0f / l;
    const int token = row / grp;
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(row0 + token) * a.ldo + (int64_t)(kvh * grp + row - token * grp) * D + c;
    *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv), pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
}
template <int D>
static cudaError_t launch_tree_join(const TreeAttnArgs& a, cudaStream_t s) {
    return launch_k(tree_join_kernel<D>, dim3(a.ctas, (a.rows * (D / 8) + TREE_JOIN_THREADS - 1) / TREE_JOIN_THREADS), dim3(TREE_JOIN_THREADS), 0, s, a);
}

// =============================================================================================
// host
// =============================================================================================
constexpr int TREE_FEW_ROWS = 16;               // of a sequence on average
TreeAttnPlan tree_attn_plan(int n_seqs, int n_rows, int n_heads, int n_kv, int head_dim, int format, int max_pages, int sms) {
    TreeAttnPlan p{};
    const int grp = n_heads / n_kv;
    const int64_t mean = ((int64_t)n_rows + n_seqs - 1) / n_seqs * grp;
    p.rows = mean > TREE_FEW_ROWS ? 128 : mean <= 8 && grp <= 8 ? 8 : 16;
    const int tile_tokens = p.rows / grp;
    const int64_t items = ((int64_t)n_rows / tile_tokens + n_seqs) * n_kv, units = items * (TREE_OVER + (int64_t)max_pages);          // no more than that, however rows fall on sequences
    const int64_t most = (int64_t)sms * (format != CACHE_BF16 && p.rows == 8 ? 2 : 1);
    p.ctas = (int)(units < most ? units : most);
    auto take = [&](size_t bytes) { const size_t at = p.bytes; p.bytes += (bytes + 255) & ~size_t(255); return at; };
    p.part_o = take((size_t)p.ctas * 2 * p.rows * head_dim * 4); p.part_ml = take((size_t)p.ctas * 2 * p.rows * 8); p.joins = take((size_t)p.ctas * sizeof(TreeJoin));
    if (p.rows == 128 && format != CACHE_BF16) { p.q16 = take((size_t)n_rows * n_heads * head_dim * 2); p.q_factor = take((size_t)n_rows * n_heads * 4); }
    return p;
}

template <int D, int FMT, int NB, int STAGES>
static cudaError_t launch_few(const CUtensorMap* tm_page, const TreeAttnArgs& a, cudaStream_t s) {
    using Cfg = FewCfg<D, FMT, NB, STAGES>;
    auto kern = tree_few_kernel<D, FMT, NB, STAGES>;
    static bool attr_done[16] = {};
    const cudaError_t e = ensure_dynamic_smem(kern, Cfg::SMEM_BYTES, attr_done);
    return e == cudaSuccess ? launch_k(kern, dim3(a.ctas), dim3(TREE_THREADS), Cfg::SMEM_BYTES, s, *tm_page, a) : e;
}
template <int D, int FMT>
static cudaError_t launch_many(const CUtensorMap* tm_q, const CUtensorMap* tm_page, const TreeAttnArgs& a, cudaStream_t s) {
    using Cfg = ManyCfg<D, FMT>;
    auto kern = tree_many_kernel<D, FMT>;
    static bool attr_done[16] = {};
    cudaError_t e = ensure_dynamic_smem(kern, Cfg::SMEM_BYTES, attr_done);
    if (e == cudaSuccess && FMT != CACHE_BF16) e = launch_k(tree_queries_kernel<D>, dim3((unsigned)(((int64_t)a.n_rows * a.n_heads + 31) / 32)), dim3(128), 0, s, a);
    return e == cudaSuccess ? launch_k(kern, dim3(a.ctas), dim3(Cfg::THREADS), Cfg::SMEM_BYTES, s, *tm_q, *tm_page, a) : e;
}
template <int D, int FMT>
static cudaError_t launch_parts(const CUtensorMap* tm_q, const CUtensorMap* tm_page, const TreeAttnArgs& a, cudaStream_t s) {
    constexpr int MORE = D == 64 ? 2 : 1;
    const cudaError_t e = a.rows == 128 ? launch_many<D, FMT>(tm_q, tm_page, a, s)
                        : a.rows == 8 ? launch_few<D, FMT, 1, (FMT == CACHE_BF16 ? 5 : 4) * MORE>(tm_page, a, s) : launch_few<D, FMT, 2, (FMT == CACHE_BF16 ? 5 : 8) * MORE>(tm_page, a, s);
    return e == cudaSuccess ? launch_tree_join<D>(a, s) : e;
}
template <int D>
static cudaError_t launch_of(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int format, const TreeAttnArgs& a, cudaStream_t s) {
    return format == CACHE_BF16 ? launch_parts<D, CACHE_BF16>(tm_q, tm_page, a, s) : format == CACHE_E4M3 ? launch_parts<D, CACHE_E4M3>(tm_q, tm_page, a, s) : launch_parts<D, CACHE_INT8>(tm_q, tm_page, a, s);
}
cudaError_t launch_tree_attention(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int head_dim, int format, const TreeAttnArgs& a, cudaStream_t s) {
    return head_dim == 64 ? launch_of<64>(tm_q, tm_page, format, a, s) : head_dim == 128 ? launch_of<128>(tm_q, tm_page, format, a, s) : cudaErrorInvalidValue;
}

}  // namespace oa
