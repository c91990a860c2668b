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
OA_DEVINL uint32_t pack_f16x2(float a, float b) { uint32_t r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a)); return r; }
OA_DEVINL void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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
// which new tokens token t of a sequence of n sees, and the first cached place of its window
OA_DEVINL uint64_t tree_seen(const TreeAttnArgs& a, const TreeSeq& s, int t) {
    const uint64_t there = s.n < 64 ? (1ull << s.n) - 1 : ~0ull;
    return (a.seen ? __ldcg(reinterpret_cast<const unsigned long long*>(a.seen) + s.row0 + t) : (2ull << t) - 1) & there;
}
OA_DEVINL int tree_low(const TreeAttnArgs& a, const TreeSeq& s, uint64_t seen, int t) { return a.window > 0 ? s.ctx + __popcll(seen & ((1ull << t) - 1)) - a.window + 1 : 0; }

// =============================================================================================
// up to 16 rows of an item: the warp path
// =============================================================================================
template <int D, int FMT, int NB, int STAGES>
struct FewCfg {
    static constexpr int ESZ = FMT == CACHE_BF16 ? 2 : 1;
    static constexpr int KV_BYTES = CACHE_PAGE * D * ESZ, STAGE_BYTES = 2 * KV_BYTES, SCALE_BYTES = FMT == CACHE_BF16 ? 0 : 2 * CACHE_PAGE * 4;
    static constexpr int ROWS = 8 * NB, REGS = D / 4 * NB;                       // output values of a lane and its twin's in the other half
    static constexpr int Q_PITCH = D * 2 + (FMT == CACHE_BF16 ? 16 : 64), Q_BYTES = ROWS * Q_PITCH;      // no bank conflicts
    static constexpr int META_BYTES = ROWS * 16;                                 // seen, first place, factor
    static constexpr int STATE_BYTES = 4 * REGS * 32 * 4 + 4 * ROWS * 2 * 4 + 16;
    static constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + SCALE_BYTES) + 2 * (Q_BYTES + META_BYTES) + STATE_BYTES + (2 * STAGES + 6) * 8;
    static constexpr int CTAS = FMT != CACHE_BF16 && NB == 1 ? 2 : 1;            // of an SM
};
struct TreeMeta { uint64_t seen; int low; float factor; };
struct FewAt { int seq, kvh, tile; int64_t unit0; TreeSeq s; };                  // an item and its first unit

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
    constexpr int KS = D / 16, KH = KS / 2, ROWS = Cfg::ROWS;
    constexpr bool BITS8 = FMT != CACHE_BF16;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* scales_s = smem + STAGES * Cfg::STAGE_BYTES;                                    // [stage][keys', values'][64]
    uint8_t* q_s = scales_s + STAGES * Cfg::SCALE_BYTES;                                     // [2 items][rows]
    TreeMeta* meta_s = reinterpret_cast<TreeMeta*>(q_s + 2 * Cfg::Q_BYTES);                  // [2 items][rows]
    float* states = reinterpret_cast<float*>(meta_s + 2 * ROWS);                             // [4 quarters][values][32 lanes]
    float* ml_s = states + 4 * Cfg::REGS * 32;                                               // [4 quarters][rows][2]
    float* vref_s = ml_s + 4 * ROWS * 2;                                                     // [4 quarters]: what values' scales are taken over
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(vref_s + 4);
    uint64_t *empty_bar = full_bar + STAGES, *q_full = empty_bar + STAGES, *q_empty = q_full + 2, *states_full = q_empty + 2, *states_empty = states_full + 1;
    __shared__ int64_t sums[TREE_THREADS / 32];
    __shared__ FewAt start;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv, tile_tokens = ROWS / grp;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_page);
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], TREE_CONSUMERS / 32); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], TREE_CONSUMERS / 32 + 1); }
        mbar_init(states_full, TREE_CONSUMERS / 32); mbar_init(states_empty, 1);
        fence_barrier_init();
    }
    griddep_wait();
    // ---- the plan ----
    const int per = (a.n_seqs + TREE_THREADS - 1) / TREE_THREADS, s0 = min(a.n_seqs, (int)threadIdx.x * per), s1 = min(a.n_seqs, s0 + per);
    FewAt at;
    auto units_of = [&](const TreeSeq& s) { return (int64_t)s.tiles(tile_tokens) * a.n_kv * (1 + s.pages); };
    int64_t units = 0; bool wrong = false;
    for (at.seq = s0; at.seq < s1; ++at.seq) { at.s.read(a, at.seq); wrong = wrong || at.s.wrong; units += units_of(at.s); }
    if (wrong && a.status) *a.status = 400;
    int64_t before = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t x = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += x; }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    before -= units;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < TREE_THREADS / 32; ++w) { if (w < warp) before += sums[w]; total += sums[w]; }
    const int64_t busy = busy_ctas(gridDim.x, total), u_begin = first_unit(blockIdx.x, busy, total), u_end = first_unit(blockIdx.x + 1, busy, total);
    if (u_begin < u_end && u_begin >= before && u_begin < before + units) {                  // one thread
        at.seq = s0; at.unit0 = before;
        for (at.s.read(a, s0); u_begin >= at.unit0 + units_of(at.s);) { at.unit0 += units_of(at.s); ++at.seq; at.s.read(a, at.seq); }
        const int item = (int)quotient(u_begin - at.unit0, 1 + at.s.pages), tiles = at.s.tiles(tile_tokens);
        at.unit0 += (int64_t)item * (1 + at.s.pages);
        at.kvh = item / tiles; at.tile = item - at.kvh * tiles;
        start = at;
    }
    if (threadIdx.x == 0) a.joins[blockIdx.x].parts = 0;
    __syncthreads();
    if (u_begin >= u_end) { griddep_launch(); return; }
    at = start;
    auto next = [&] {
        at.unit0 += 1 + at.s.pages;
        if (++at.tile < at.s.tiles(tile_tokens)) return;
        at.tile = 0;
        if (++at.kvh < a.n_kv) return;
        at.kvh = 0;
        do { if (++at.seq >= a.n_seqs) { at.s.n = at.s.pages = 0; return; } at.s.read(a, at.seq); } while (at.s.n == 0);
    };
    auto tile_rows = [&] { return min(tile_tokens, at.s.n - at.tile * tile_tokens) * grp; };

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
                if (lane == 0) {
                    uint8_t* dst = smem + st * Cfg::STAGE_BYTES;
                    mbar_expect_tx(&full_bar[st], Cfg::STAGE_BYTES + Cfg::SCALE_BYTES);
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int64_t block = (int64_t)(v * a.num_pages + page) * a.n_kv + at.kvh;
                        if (BITS8) {
                            constexpr int BLOCK_BYTES = CACHE_PAGE * (D + 4);
                            tma_load_2d(dst + v * Cfg::KV_BYTES, &tm_page, &full_bar[st], 0, (int)(block * (BLOCK_BYTES / 128)), kEvictFirst);
                            bulk_load(scales_s + st * Cfg::SCALE_BYTES + v * CACHE_PAGE * 4, reinterpret_cast<const uint8_t*>(a.cache) + block * BLOCK_BYTES + CACHE_PAGE * D, CACHE_PAGE * 4, &full_bar[st]);
                        } else
#pragma unroll
                            for (int h = 0; h < D / 64; ++h) tma_load_2d(dst + v * Cfg::KV_BYTES + h * (CACHE_PAGE * 128), &tm_page, &full_bar[st], h * 64, (int)(block * CACHE_PAGE), kEvictFirst);
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
            u = min(at.unit0 + 1 + at.s.pages, u_end);
            mbar_wait(&q_empty[k & 1], ((k >> 1) & 1) ^ 1);
            uint8_t* q_dst = q_s + (k & 1) * Cfg::Q_BYTES;
            TreeMeta* meta = meta_s + (k & 1) * ROWS;
            const int live = tile_rows(), t0 = at.tile * tile_tokens;
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
        uint32_t k = 0;
        for (int64_t u = u_begin; u < u_end; next(), ++k) {
            const int64_t end = at.unit0 + 1 + at.s.pages;
            const bool first = at.unit0 >= u_begin, last = end <= u_end;
            u = min(end, u_end);
            const int live = tile_rows(), row0 = at.s.row0 + at.tile * tile_tokens;
            mbar_wait(&q_full[k & 1], (k >> 1) & 1);
            uint32_t blind = 0;                                                              // rows that see nothing
            {
                const TreeMeta m = meta_s[(k & 1) * ROWS + (lane < ROWS ? lane : 0)];
                const uint64_t there = at.s.end - at.s.ctx < 64 ? (1ull << (at.s.end - at.s.ctx)) - 1 : ~0ull;
                const bool sees = (m.seen & there) != 0 || (at.s.ctx > 0 && (a.window == 0 || a.sinks > 0 || m.low < at.s.ctx));
                blind = __ballot_sync(0xffffffffu, lane < live && !sees);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_empty[k & 1]);
            if (lane == 0 && first && !last) { TreeJoin j; j.parts = cta_of(end - 1, busy, total) - (int)blockIdx.x; j.row0 = row0; j.rows = live; j.kvh = at.kvh; j.blind = blind; a.joins[blockIdx.x] = j; }
            float* po = a.part_o + ((int64_t)blockIdx.x * 2 + !first) * (ROWS * D);
            float2* ml = reinterpret_cast<float2*>(a.part_ml) + ((int64_t)blockIdx.x * 2 + !first) * ROWS;
            mbar_wait(states_full, k & 1);
            float vref[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) vref[w] = BITS8 ? vref_s[w] : 1.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = b * 8 + 2 * t + h;
                    float2 s4[4]; float m = -INFINITY, l = 0.f, f[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) { s4[w] = *reinterpret_cast<const float2*>(ml_s + (w * ROWS + row) * 2); m = fmaxf(m, s4[w].x); }
                    const float ref = finite_or_zero(m);
#pragma unroll
                    for (int w = 0; w < 4; ++w) { f[w] = ex2_approx(s4[w].x - ref); l += f[w] * s4[w].y; f[w] *= vref[w]; }
                    if (row >= live) continue;
                    float inv = 1.0f;
                    uint16_t* out = nullptr;
                    if (first && last) {
                        inv = blind >> row & 1 ? 0.f : 1.0f / l;
                        const int token = row / grp;
                        out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(row0 + token) * a.ldo + (int64_t)(at.kvh * grp + row - token * grp) * D;
                    } else if (g == 0) ml[row] = make_float2(m, l);
#pragma unroll 4
                    for (int r = 0; r < KS * 2; ++r) {                                       // channel block r / 2 and the one or the other of a lane's two channels there
                        const int i = r >> 1, up = r & 1, reg = (i / KH) * (Cfg::REGS / 2) + (b * KH + i % KH) * 4 + 2 * up + h, d = i * 16 + (BITS8 ? 2 * g + up : 8 * up + g);
                        float o = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; ++w) o += f[w] * states[(w * Cfg::REGS + reg) * 32 + lane];
                        if (out) out[d] = f32_to_bf16_bits(o * inv); else po[row * D + d] = o;
                    }
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(states_empty);
        }
        griddep_launch();
        return;
    }

    // Warps w and w + 4 take the same 16 tokens of every page and half of the channels each.  Tokens are the 16 rows of the first product and channels those of the second, the item's rows the 8
    // columns of both: S^T = K Q^T, O^T = V^T P^T
    const int g = lane >> 2, t = lane & 3, quarter = warp & 3, half = warp >> 2;
    int st = 0, n_items = 0; uint32_t ph = 0;
    for (int64_t u = u_begin; u < u_end; next(), ++n_items) {
        const int c0 = (int)max(u - at.unit0 - 1, (int64_t)0), c1 = (int)min((int64_t)at.s.pages, u_end - at.unit0 - 1);
        u = at.unit0 + 1 + c1;
        float oacc[NB][KH][4], m_run[NB][2], l_run[NB][2], factor[NB][2];                    // O^T: two channels of a lane in each block of 16, rows 2 t and 2 t + 1; maxima, sums and score factors of these rows
        float vref = 0.f;                                                                    // 8 bits: a power of two that no value's scale so far passes
        mbar_wait(&q_full[n_items & 1], (n_items >> 1) & 1);
        const TreeMeta* meta = meta_s + (n_items & 1) * ROWS;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < KH; ++i) oacc[b][i][0] = oacc[b][i][1] = oacc[b][i][2] = oacc[b][i][3] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) { m_run[b][h] = -INFINITY; l_run[b][h] = 0.f; factor[b][h] = meta[b * 8 + 2 * t + h].factor; }
        }
        const uint8_t* q_item = q_s + (n_items & 1) * Cfg::Q_BYTES;
        for (int c = c0; c < c1; ++c) {
            const int page = at.s.page(c), key0 = page * CACHE_PAGE + quarter * 16;
            const bool special = at.s.special(a, page);
            mbar_wait(&full_bar[st], ph);
            if (key0 < at.s.end) {
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
                                const int key = key0 + g + 8 * e, n = key - at.s.ctx;
                                const bool sees = n < 0 ? key < a.sinks || key >= m.low : key < at.s.end && n < 64 && (m.seen >> (n & 63) & 1);
                                if (sees && b * 8 + 2 * t + h < ROWS) vis |= 1u << (b * 4 + e * 2 + h);
                            }
                        }
                    constexpr uint32_t LO = NB == 2 ? 0x33u : 0x3u;
                    any_lo = __ballot_sync(0xffffffffu, (vis & LO) != 0); any_hi = __ballot_sync(0xffffffffu, (vis & LO << 2) != 0);
                }
                float vfac[2] = {1.f, 1.f}, grown = 1.0f;                                    // a weight's factor of tokens g and g + 8; O's, where a scale passes the reference
                if constexpr (BITS8) {
                    // a bit of a token is in its four lanes together: whoever is not seen by anyone counts for nothing
                    const bool see_lo = any_lo >> (g * 4) & 0xfu, see_hi = any_hi >> (g * 4) & 0xfu;
                    uint32_t top = max(see_lo && vscale[0] < INFINITY ? __float_as_uint(fabsf(vscale[0])) : 0u, see_hi && vscale[1] < INFINITY ? __float_as_uint(fabsf(vscale[1])) : 0u);
                    top = __reduce_max_sync(0xffffffffu, top);
                    const float need = __uint_as_float(min((top & 0x7f800000u) + 0x00800000u, 0x7e800000u));         // up to 2^126
                    if (need > vref) { grown = vref * (1.0f / need); vref = need; }
                    const float inv = 1.0f / vref;                                           // powers of two: exact
                    vfac[0] = vscale[0] * inv * 32768.f; vfac[1] = vscale[1] * inv * 32768.f;
                }
                uint32_t pb[NB][2]; float alpha[NB][2];
                bool same = grown == 1.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float pr[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool s0 = vis >> (b * 4 + h) & 1, s1 = vis >> (b * 4 + 2 + h) & 1;
                        const float lo = s0 ? (sacc[b][0][h] + sacc[b][1][h]) * (BITS8 ? kscale[0] * factor[b][h] : factor[b][h]) : -INFINITY;
                        const float hi = s1 ? (sacc[b][0][2 + h] + sacc[b][1][2 + h]) * (BITS8 ? kscale[1] * factor[b][h] : factor[b][h]) : -INFINITY;
                        float mx = fmaxf(lo, hi);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        const float m_new = fmaxf(m_run[b][h], mx), ref = finite_or_zero(m_new);
                        alpha[b][h] = ex2_approx(m_run[b][h] - ref);
                        const float p0 = ex2_approx(lo - ref), p1 = ex2_approx(hi - ref);
                        l_run[b][h] = l_run[b][h] * alpha[b][h] + (p0 + p1);
                        alpha[b][h] *= grown;
                        pr[h] = s0 && BITS8 ? p0 * vfac[0] : p0; pr[2 + h] = s1 && BITS8 ? p1 * vfac[1] : p1;       // 0 of a token that the row does not see, whatever its scale
                        same = same && m_new == m_run[b][h];
                        m_run[b][h] = m_new;
                    }
                    if (BITS8) { pb[b][0] = transpose_8x8(pack_f16x2(pr[0], pr[1])); pb[b][1] = transpose_8x8(pack_f16x2(pr[2], pr[3])); }
                    else { pb[b][0] = transpose_8x8(pack_bf16x2(pr[0], pr[1])); pb[b][1] = transpose_8x8(pack_bf16x2(pr[2], pr[3])); }
                }
                if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < KH; ++i) { oacc[b][i][0] *= alpha[b][0]; oacc[b][i][1] *= alpha[b][1]; oacc[b][i][2] *= alpha[b][0]; oacc[b][i][3] *= alpha[b][1]; }
                }
                // values of tokens 2 t, 2 t + 1 and these + 8
                uint32_t vf[KH][4];
                if constexpr (BITS8) {
                    const int r = quarter * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                    for (int i = 0; i < KH; i += 2) {
                        uint32_t w[4];
                        ldmatrix_x4_trans(vbase + few_off8<D>(r, half * KH + i + (lane >> 4)), w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int e = 0; e < 2; ++e) { to_f16<FMT, true>(w[2 * e], vf[i + e][0], vf[i + e][1]); to_f16<FMT, true>(w[2 * e + 1], vf[i + e][2], vf[i + e][3]); }
                    }
                } else {
                    const int r = quarter * 16 + ((lane >> 4) << 3) + (lane & 7), dsel = ((lane >> 3) & 1) << 3;
#pragma unroll
                    for (int i = 0; i < KH; ++i) ldmatrix_x4_trans(vbase + few_off<D>(r, (half * KH + i) * 16 + dsel), vf[i][0], vf[i][1], vf[i][2], vf[i][3]);
                }
                if (special) {                                                               // values that nobody sees may be anything, and 0 x inf is not 0
                    const uint32_t keep0 = (any_lo >> (8 * t) & 0xfu ? 0xffffu : 0u) | (any_lo >> (8 * t + 4) & 0xfu ? 0xffff0000u : 0u);
                    const uint32_t keep1 = (any_hi >> (8 * t) & 0xfu ? 0xffffu : 0u) | (any_hi >> (8 * t + 4) & 0xfu ? 0xffff0000u : 0u);
#pragma unroll
                    for (int i = 0; i < KH; ++i) { vf[i][0] &= keep0; vf[i][1] &= keep0; vf[i][2] &= keep1; vf[i][3] &= keep1; }
                }
#pragma unroll
                for (int i = 0; i < KH; ++i)
#pragma unroll
                    for (int b = 0; b < NB; ++b) mma_of<FMT>(oacc[b][i], vf[i][0], vf[i][1], vf[i][2], vf[i][3], pb[b][0], pb[b][1]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[st]);
            if (++st == STAGES) { st = 0; ph ^= 1; }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[n_items & 1]);
        // the four quarters' states, for the warp that brings them together while this one goes on
        mbar_wait(states_empty, (n_items & 1) ^ 1);
        float* mine = states + (quarter * Cfg::REGS + half * (Cfg::REGS / 2)) * 32 + lane;   // value [half][b][i][e]
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float l = l_run[b][h];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                if (half == 0 && g == 0) *reinterpret_cast<float2*>(ml_s + (quarter * ROWS + b * 8 + 2 * t + h) * 2) = make_float2(m_run[b][h], l);
            }
#pragma unroll
            for (int i = 0; i < KH; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[((b * KH + i) * 4 + e) * 32] = oacc[b][i][e];
        }
        if (BITS8 && half == 0 && lane == 0) vref_s[quarter] = vref * (1.0f / 32768.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(states_full);
    }
    griddep_launch();                            // not before: the next kernel's CTAs would crowd onto the SMs that are done first
}

// =============================================================================================
// the join
// =============================================================================================
// Of the item that a CTA began and others ended: eight rows a CTA, a thread four channels of a row
template <int D>
__global__ void __launch_bounds__(2 * D) tree_join_kernel(const __grid_constant__ TreeAttnArgs a) {
    const int cta = blockIdx.x, row = blockIdx.y * 8 + threadIdx.x / (D / 4), c = threadIdx.x % (D / 4) * 4, grp = a.n_heads / a.n_kv;
    griddep_launch();
    griddep_wait();
    const int parts = __ldcg(&a.joins[cta].parts);
    if (parts == 0 || row >= __ldcg(&a.joins[cta].rows)) return;
    const int row0 = __ldcg(&a.joins[cta].row0), kvh = __ldcg(&a.joins[cta].kvh);
    const bool blind = __ldcg(&a.joins[cta].blind) >> row & 1;
    auto slot = [&](int i) { return i == 0 ? (int64_t)cta * 2 : (int64_t)(cta + i) * 2 + 1; };
    float M = -INFINITY, l = 0.f; float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int MP = 8;
    for (int i0 = 0; i0 <= parts; i0 += MP) {
        float2 ml[MP]; float4 o[MP];
#pragma unroll
        for (int p = 0; p < MP; ++p) {
            ml[p] = make_float2(-INFINITY, 0.f); o[p] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i0 + p > parts) continue;
            ml[p] = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + slot(i0 + p) * a.rows + row);
            o[p] = __ldcg(reinterpret_cast<const float4*>(a.part_o + (slot(i0 + p) * a.rows + row) * D + c));
        }
        float m = M;
#pragma unroll
        for (int p = 0; p < MP; ++p) m = fmaxf(m, ml[p].x);
        const float ref = finite_or_zero(m), f0 = ex2_approx(M - ref);
        M = m; l *= f0; acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
        for (int p = 0; p < MP; ++p) {
            const float f = ex2_approx(ml[p].x - ref);
            l += f * ml[p].y; acc.x += f * o[p].x; acc.y += f * o[p].y; acc.z += f * o[p].z; acc.w += f * o[p].w;
        }
    }
    const float inv = blind ? 0.f : 1.0f / l;
    const int token = row / grp;
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(row0 + token) * a.ldo + (int64_t)(kvh * grp + row - token * grp) * D + c;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// =============================================================================================
// host
// =============================================================================================
TreeAttnPlan tree_attn_plan(int n_seqs, int n_rows, int n_heads, int n_kv, int head_dim, int format, int max_pages, int sms) {
    TreeAttnPlan p{};
    const int grp = n_heads / n_kv;
    const int64_t mean = ((int64_t)n_rows + n_seqs - 1) / n_seqs * grp;
    p.rows = mean <= 8 && grp <= 8 ? 8 : 16;
    const int tile_tokens = p.rows / grp;
    const int64_t items = ((int64_t)n_rows / tile_tokens + n_seqs) * n_kv, units = items * (1 + (int64_t)max_pages);          // no more than that, however rows fall on sequences
    const int64_t most = (int64_t)sms * (format != CACHE_BF16 && p.rows == 8 ? 2 : 1);
    p.ctas = (int)(units < most ? units : most);
    auto take = [&](size_t bytes) { const size_t at = p.bytes; p.bytes += (bytes + 255) & ~size_t(255); return at; };
    p.part_o = take((size_t)p.ctas * 2 * p.rows * head_dim * 4); p.part_ml = take((size_t)p.ctas * 2 * p.rows * 8); p.joins = take((size_t)p.ctas * sizeof(TreeJoin));
    return p;
}

template <int D, int FMT, int NB, int STAGES>
static cudaError_t launch_few(const CUtensorMap* tm_page, const TreeAttnArgs& a, cudaStream_t s) {
    using Cfg = FewCfg<D, FMT, NB, STAGES>;
    auto kern = tree_few_kernel<D, FMT, NB, STAGES>;
    static bool attr_done[16] = {};
    cudaError_t e = ensure_dynamic_smem(kern, Cfg::SMEM_BYTES, attr_done);
    if (e == cudaSuccess) e = launch_k(kern, dim3(a.ctas), dim3(TREE_THREADS), Cfg::SMEM_BYTES, s, *tm_page, a);
    if (e == cudaSuccess) e = launch_k(tree_join_kernel<D>, dim3(a.ctas, NB), dim3(2 * D), 0, s, a);
    return e;
}
template <int D, int FMT>
static cudaError_t launch_of(const CUtensorMap* tm_page, const TreeAttnArgs& a, cudaStream_t s) {
    constexpr int MORE = D == 64 ? 2 : 1;
    return a.rows == 8 ? launch_few<D, FMT, 1, 5 * MORE>(tm_page, a, s) : launch_few<D, FMT, 2, (FMT == CACHE_BF16 ? 5 : 9) * MORE>(tm_page, a, s);
}
cudaError_t launch_tree_attention(const CUtensorMap* tm_page, int head_dim, int format, const TreeAttnArgs& a, cudaStream_t s) {
    if (head_dim == 64) return format == CACHE_BF16 ? launch_of<64, CACHE_BF16>(tm_page, a, s) : format == CACHE_E4M3 ? launch_of<64, CACHE_E4M3>(tm_page, a, s) : launch_of<64, CACHE_INT8>(tm_page, a, s);
    if (head_dim == 128) return format == CACHE_BF16 ? launch_of<128, CACHE_BF16>(tm_page, a, s) : format == CACHE_E4M3 ? launch_of<128, CACHE_E4M3>(tm_page, a, s) : launch_of<128, CACHE_INT8>(tm_page, a, s);
    return cudaErrorInvalidValue;
}

}  // namespace oa
