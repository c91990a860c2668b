// attention_prefix.cu — decode attention of a batch whose sequences share prefixes: a prefix's keys and values are read once for all rows that see them.
//
//   out_i = softmax(scale q_i [K_prefix; K_own(i)]^T) [V_prefix; V_own(i)]
//
// The softmax splits over any partition of the keys: a part leaves its maximum m, l = sum 2^(s - m) and O = sum 2^(s - m) v, and parts join as
// O = sum_i 2^(m_i - M) O_i, l likewise, M = max m_i.  Scores, maxima, sums, O and parts are fp32; the weights 2^(s - m) are rounded to bf16 for the second product (2^-9 of a weight, of
// either sign; l sums them unrounded) and the result once more.  Two kernels make the parts, a third joins them:
//
//  prefix_part_kernel: all rows of a prefix against its keys is a product of matrices (128 conversations of 4 heads a group: 512 rows a key/value head), so it runs on tcgen05: 128 rows (as
//    many tokens' heads of a group as fit) x 64 or 128 keys a tile, S = Q K^T in three TMEM buffers, two tiles ahead, P over S's own columns as the second product's operand, O in TMEM.  Two
//    softmax warpgroups take the tiles in turn, one row a thread; the reference maximum rises (and O is rescaled) only where a score passes it by 2^8.  16384 keys under 4 x 8 row tiles of
//    128: 29 us, 1680 cycles a tile of 128 x 128 x 128 for 1024 of the tensor pipe's and 1024 of the exponentials' (all eight warps on one tile, as before: 1900).
//  own_part_kernel: a sequence's own keys have only its few heads as rows: streamed through shared memory by TMA and multiplied on the warp path of 16 x 8 x 16 products, a page's 64
//    tokens over four warps (and either half of its channels on one of two), with tokens and channels as the 16 rows and the heads as the 8 columns: nothing of a product is empty for 8 heads a
//    group, and O takes D / 8 registers a lane.  128 sequences of 64 to 512 tokens, 170 MB, in 28 us: 6.1 TB/s.
//  join_parts_kernel: 3 us and as much to begin.
//
// Row tiles and key/value heads are items; the prefixes' are cut into pieces of equally many key tiles, the own parts (a unit a page, and one an item) dealt out contiguously, the same number
// to every CTA: unit u is CTA floor(((u + 1) G - 1) / total)'s, so what parts an item has, and where each of them lies, follows from lengths alone.  The plan is made on the device, by every
// CTA for itself: lengths may come from the kernel before, a captured call serves other lengths when it is replayed, and the host waits for nothing.  Parts are joined in one order, whatever
// came first: the same call gives the same bits.
//
// The second kernel starts beside the first (it needs nothing of it): it streams own keys from memory while the first is busy with products, and for up to 8 heads a group their shared memory and
// registers are cut so that an SM holds one CTA of each.  For 9 to 16 heads a group they are not (the own parts' kernel has 112 to 158 registers a thread): on an SM the own parts come after the
// prefixes; 128 rows of 16 heads a group on 1536 tokens, own parts of 64 to 512: 46 us with 4 key/value heads of 128 (bytes 12.8 at the copy rate), 79 with 8 (25.6), 35 with 4 of 64 (6.4).
// Whole calls: 128 rows of 4 x 8 heads on a prefix of 1536 40 us (162 MB; 25 at the copy rate): 3 to begin, 28 of stream, 3 between the first CTA's end and the last one's, 5 for the join with its start; 8 rows of 4000 to 9000 own tokens 42 us for 221 MB.
#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"
#include "work_units.hpp"

namespace oa {

constexpr int PRE_SOFTMAX = 256;        // threads of a row tile: two softmax warpgroups
constexpr int OWN_CONSUMERS = 256, OWN_THREADS = OWN_CONSUMERS + 64;        // eight consumer warps, producer, a warp that brings an item's states together
constexpr int ROW_TILE = 128;          // rows of a prefix's products
constexpr int JOIN_THREADS = 128, JOIN_CTAS = 4;         // of an SM: 128 registers a thread

OA_DEVINL float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }        // nothing seen: any reference will do, 2^(-inf - 0) is 0
OA_DEVINL int pages_of(int len) { return (len + CACHE_PAGE - 1) / CACHE_PAGE; }
OA_DEVINL void report(const PrefixAttnArgs& a) { if (a.status) *a.status = 400; }

// The runs of rows that share a prefix: bounds that never fall, lengths that fit their tables (0 where nobody sees it)
OA_DEVINL void read_runs(const PrefixAttnArgs& a, int lane, int& row0, int& rows, int& len) {      // one warp, a lane a prefix
    int r0 = 0, r1 = 0; bool wrong = false;
    len = 0;
    if (lane < a.n_prefixes) {
        r0 = __ldcg(a.prefix_rows + lane); r1 = __ldcg(a.prefix_rows + lane + 1); len = __ldcg(a.prefix_lens + lane);
        wrong = r0 < 0 || r1 < r0 || r1 > a.n_seqs || len < 0 || len > (int64_t)a.max_prefix_pages * CACHE_PAGE;
        r0 = min(max(r0, 0), a.n_seqs); r1 = min(max(r1, 0), a.n_seqs);
        len = (int)min((int64_t)max(len, 0), (int64_t)a.max_prefix_pages * CACHE_PAGE);
    }
    if (wrong) report(a);
    for (int o = 1; o < a.n_prefixes; o <<= 1) { const int below = __shfl_up_sync(0xffffffffu, r0, o); if (lane >= o) r0 = max(r0, below); }
    r1 = max(r0, r1);
    const bool some = lane < a.n_prefixes && r1 > r0 && len > 0;
    row0 = r0; rows = some ? r1 - r0 : 0; len = some ? len : 0;
}
// What the prefixes' part looks like: a prefix's rows, tokens, row tiles and key tiles, and the pieces that its items (a row tile and a key/value head) are cut into along the keys
struct PrefixPieces { int row0[PREFIX_MAX], rows[PREFIX_MAX], len[PREFIX_MAX], tiles[PREFIX_MAX], key_tiles[PREFIX_MAX], split[PREFIX_MAX], piece0[PREFIX_MAX], pieces; };
OA_DEVINL void cut_prefixes(const PrefixAttnArgs& a, PrefixPieces& px, int lane) {      // one warp
    int row0, rows, len;
    read_runs(a, lane, row0, rows, len);
    const int tile_tokens = ROW_TILE / (a.n_heads / a.n_kv), tiles = (rows + tile_tokens - 1) / tile_tokens, key_tiles = (len + a.key_tile - 1) / a.key_tile, items = tiles * a.n_kv;
    // Pieces of at most `most` key tiles, as many as make the CTA with most work end first, where a piece costs what 384 keys do besides its own; every lane weighs
    // one number of them, up to 144 for the longest prefix.  No more pieces than CTAs and items together: the scratch has that many slots.
    const int longest = __reduce_max_sync(0xffffffffu, key_tiles), all_items = __reduce_add_sync(0xffffffffu, items);
    const int want = lane < 16 ? lane + 1 : 16 + 8 * (lane - 15), most = (max(longest, 1) + want - 1) / want;
    int64_t n = 0;
    for (int p = 0; p < a.n_prefixes; ++p) n += (int64_t)__shfl_sync(0xffffffffu, items, p) * ((__shfl_sync(0xffffffffu, key_tiles, p) + most - 1) / most);
    const int64_t cost = quotient(n + a.pre_ctas - 1, a.pre_ctas) * (most + 384 / a.key_tile);
    const unsigned key = n > (int64_t)a.pre_ctas + all_items ? 0xffffffffu : (unsigned)min(cost, (int64_t)0x3ffffff) << 5 | (unsigned)lane;
    const unsigned best = __reduce_min_sync(0xffffffffu, key);
    const int cut = __shfl_sync(0xffffffffu, most, (int)(best & 31u)), split = (key_tiles + cut - 1) / cut;
    int pieces = items * split;
    const int mine = pieces;
    for (int o = 1; o < a.n_prefixes; o <<= 1) { const int below = __shfl_up_sync(0xffffffffu, pieces, o); if (lane >= o) pieces += below; }
    px.row0[lane] = row0; px.rows[lane] = rows; px.len[lane] = len; px.tiles[lane] = tiles; px.key_tiles[lane] = key_tiles; px.split[lane] = split;
    px.piece0[lane] = pieces - mine;
    if (lane == a.n_prefixes - 1) px.pieces = pieces;
}

// =============================================================================================
// the prefixes' part
// =============================================================================================
template <int D, int KEYS, int SLOTS>          // KEYS: of a tile; SLOTS: tiles of keys or values in the ring
struct PreCfg {
    static constexpr int HALVES = D / 64;
    static constexpr int Q_HALF = ROW_TILE * 128, KV_HALF = KEYS * 128;          // rows x 64 bf16 columns under the 128-byte swizzle
    static constexpr int Q_BYTES = HALVES * Q_HALF, TILE_BYTES = HALVES * KV_HALF;
    static constexpr int THREADS = 64 + PRE_SOFTMAX;             // producer, issuer, softmax warps
    static constexpr int XCH_BYTES = 3 * 128 * 4;                // a row's reference maximum, and its two sums of a piece
    static constexpr int SMEM_BYTES = Q_BYTES + SLOTS * TILE_BYTES + 256 + XCH_BYTES;
    static constexpr uint32_t O_COL = 384;                       // TMEM: S and P of the tiles in turn at 0, 128 and 256, O at 384
};
struct PrePiece { int g, kvh, tile, k0, k1; };
OA_DEVINL PrePiece pre_piece(const PrefixPieces& px, int piece, int n_prefixes) {
    PrePiece s; s.g = 0;
    while (s.g + 1 < n_prefixes && piece >= px.piece0[s.g + 1]) ++s.g;     // prefixes without pieces begin where the next one does
    const int rem = piece - px.piece0[s.g], split = px.split[s.g], i = rem / split, k = rem - i * split;
    s.k0 = (int)quotient((int64_t)px.key_tiles[s.g] * k, split); s.k1 = (int)quotient((int64_t)px.key_tiles[s.g] * (k + 1), split);
    s.kvh = i / px.tiles[s.g]; s.tile = i - s.kvh * px.tiles[s.g];
    return s;
}

template <int D, int KEYS, int SLOTS>
// 104 registers: one CTA and one of the own parts' (96, up to 8 heads a group) fill an SM's file, two of this kernel do not fit (of 96 they would).  Started while the kernel before it leaves the SMs one by one, two
// CTAs on one SM would have the second wait for the first one's TMEM, and the own parts' CTA go elsewhere: 8 to 15 us of a call of 45
__global__ void __maxnreg__(104) prefix_part_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ PrefixAttnArgs a) {
    using Cfg = PreCfg<D, KEYS, SLOTS>;
    constexpr int HALVES = Cfg::HALVES, PAGES = KEYS / CACHE_PAGE;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_s = smem;
    uint8_t* kv_s = q_s + Cfg::Q_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(kv_s + SLOTS * Cfg::TILE_BYTES);
    uint64_t *q_full = bars, *q_empty = bars + 1, *s_full = bars + 2, *p_full = bars + 5, *o_full = bars + 8, *full = bars + 12, *empty = full + SLOTS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty + SLOTS);
    float* xch = reinterpret_cast<float*>(kv_s + SLOTS * Cfg::TILE_BYTES + 256);
    __shared__ PrefixPieces px;

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv, tile_tokens = ROW_TILE / grp;      // tokens of a row tile
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tm_q); tma_prefetch_desc(&tm_kv);
        mbar_init(q_full, 1); mbar_init(q_empty, 1);
        for (int i = 0; i < 3; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], PRE_SOFTMAX / 64); }
        for (int i = 0; i < 4; ++i) mbar_init(&o_full[i], 1);
        for (int i = 0; i < SLOTS; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc<512>(tmem_slot);
    griddep_wait();
    // Behind the wait: what the own part's kernel reads ahead of its own wait was written by kernels that have ended.  From the warp that allocates (one warp's signal is its CTA's): a later kernel
    // of the stream that takes tensor memory ahead of its own wait finds every CTA of this one with its columns
    if (warp == 1) griddep_launch();
    if (warp == 0) cut_prefixes(a, px, lane);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    // Keys and values share one ring in the order of their products: K_0 and K_1, then K_(j+2) and V_j
    if (warp == 0) {
        uint32_t n = 0, seg = 0;                                 // tiles and pieces loaded
        for (int piece = blockIdx.x; piece < px.pieces; piece += gridDim.x, ++seg) {
            const PrePiece sg = pre_piece(px, piece, a.n_prefixes);
            mbar_wait(q_empty, (seg & 1) ^ 1);
            if (elect_one()) {                                   // rows of a tile: tokens, and the group's heads within; tokens behind the last sequence are zeros, other prefixes' are not looked at
                mbar_expect_tx(q_full, HALVES * tile_tokens * grp * 128);
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
                    tma_load_3d(q_s + h * Cfg::Q_HALF, &tm_q, q_full, h * 64, sg.kvh * grp, px.row0[sg.g] + sg.tile * tile_tokens, kEvictNormal);
            }
            __syncwarp();
            const int32_t* bt = a.prefix_tables + (size_t)sg.g * a.max_prefix_pages;
            const int pages = pages_of(px.len[sg.g]);
            int page[3][PAGES] = {};                             // of this tile and of the two before
            for (int kt = sg.k0; kt < sg.k1 + 2; ++kt) {
#pragma unroll
                for (int i = 0; i < PAGES; ++i) {
                    page[2][i] = page[1][i]; page[1][i] = page[0][i];
                    page[0][i] = kt < sg.k1 && PAGES * kt + i < pages ? bt[PAGES * kt + i] : 0;
                    if (page[0][i] < 0 || page[0][i] >= a.num_pages) { if (lane == 0) report(a); page[0][i] = 0; }
                }
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int t = kt - 2 * v;                    // K of this tile, V of the one two before
                    if (t < sg.k0 || t >= sg.k1) continue;
                    const uint32_t slot = n % SLOTS;
                    mbar_wait(&empty[slot], ((n / SLOTS) & 1) ^ 1);
                    if (elect_one()) {
                        const int there = min(PAGES, pages - PAGES * t);         // a missing second page is not loaded: its scores are masked, its values set to zero
                        uint8_t* dst = kv_s + slot * Cfg::TILE_BYTES;
                        mbar_expect_tx(&full[slot], there * HALVES * 8192);
#pragma unroll
                        for (int i = 0; i < PAGES; ++i) {
                            if (i >= there) break;
                            const int row = ((v ? a.num_pages + page[2][i] : page[0][i]) * a.n_kv + sg.kvh) * CACHE_PAGE;
#pragma unroll
                            for (int h = 0; h < HALVES; ++h) tma_load_2d(dst + h * Cfg::KV_HALF + i * 8192, &tm_kv, &full[slot], h * 64, row, kEvictLast);
                        }
                    }
                    __syncwarp();
                    ++n;
                }
            }
        }
    } else if (warp == 1) {
        // the whole warp walks the loop, an elected lane issues: descriptors stay in uniform registers
        constexpr uint32_t idesc_s = umma_idesc_bf16(128, KEYS), idesc_o = umma_idesc_bf16_bmn(128, D);
        const uint64_t q_desc = umma_desc_sw128(smem_u32(q_s)), k_desc = umma_desc_sw128(smem_u32(kv_s));
        const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(kv_s), (uint32_t)Cfg::KV_HALF, 1024u);
        uint32_t n = 0, r = 0, seg = 0;                          // tiles of the pieces before, tiles of the ring, pieces
        auto await = [&] {                                       // the ring's next tile
            const uint32_t slot = r % SLOTS;
            mbar_wait(&full[slot], (r / SLOTS) & 1);
            ++r;
            tcgen05_fence_after();
            return slot;
        };
        // products of one thread are carried out in the order of their issue: S of a tile goes over scores whose P a product ahead of it reads
        for (int piece = blockIdx.x; piece < px.pieces; piece += gridDim.x, ++seg) {
            const PrePiece sg = pre_piece(px, piece, a.n_prefixes);
            const int tiles = sg.k1 - sg.k0;
            mbar_wait(q_full, seg & 1);
            tcgen05_fence_after();
            for (int j = -2; j < tiles; ++j) {
                if (j + 2 < tiles) {                                             // scores two tiles ahead, under the softmaxes of the tiles before
                    const uint32_t slot = await(), at = (n + j + 2) % 3;
                    if (elect_one()) {
                        const uint64_t b = k_desc + (uint64_t)(slot * (Cfg::TILE_BYTES >> 4));
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) {
                            const int half = ks >> 2, in = (ks & 3) * 32;
                            umma_bf16(tmem_base + at * 128, q_desc + (uint64_t)((half * Cfg::Q_HALF + in) >> 4), b + (uint64_t)((half * Cfg::KV_HALF + in) >> 4), idesc_s, ks > 0 ? 1u : 0u);
                        }
                        umma_commit(&s_full[at]);
                        umma_commit(&empty[slot]);
                        if (j + 3 == tiles) umma_commit(q_empty);
                    }
                    __syncwarp();
                }
                if (j >= 0) {
                    const uint32_t m = n + j, at = m % 3;
                    mbar_wait(&p_full[at], (m / 3) & 1);
                    const uint32_t slot = await();
                    if (elect_one()) {
                        const uint64_t b = v_desc + (uint64_t)(slot * (Cfg::TILE_BYTES >> 4));
#pragma unroll
                        for (int ks = 0; ks < KEYS / 16; ++ks)
                            umma_bf16_ta(tmem_base + Cfg::O_COL, tmem_base + at * 128 + ks * 8, b + (uint64_t)(ks * (2048 >> 4)), idesc_o, (j > 0 || ks > 0) ? 1u : 0u);
                        umma_commit(&o_full[m & 3]);
                        umma_commit(&empty[slot]);
                    }
                    __syncwarp();
                }
            }
            n += tiles;
        }
    } else {
        // Two warpgroups take the tiles in turn, a row a thread: one's exponentials run under the other's loads and maxima.  A row's reference maximum goes from one to the other
        // with each tile, as soon as the tile's own maximum is known; sums stay with either, O is one for both
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t wg = (warp - 2) >> 2, lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16), o_addr = lane_addr + Cfg::O_COL;
        float *m_s = xch, *l_s = xch + 128;
        auto meet = [] { asm volatile("bar.sync 2, %0;" ::"n"(PRE_SOFTMAX) : "memory"); };
        auto take_turn = [](uint32_t n) {                                        // tile n - 1 has left its reference
            if (n & 1) asm volatile("bar.sync 3, %0;" ::"n"(PRE_SOFTMAX) : "memory"); else asm volatile("bar.sync 4, %0;" ::"n"(PRE_SOFTMAX) : "memory");
        };
        auto pass_turn = [](uint32_t n) {                                        // to tile n
            if (n & 1) asm volatile("bar.arrive 3, %0;" ::"n"(PRE_SOFTMAX) : "memory"); else asm volatile("bar.arrive 4, %0;" ::"n"(PRE_SOFTMAX) : "memory");
        };
        constexpr float kRaise = 8.0f;                                           // log2 units a score may pass the reference by
        constexpr int COLS = D / 2;
        uint32_t n0 = 0;                                                         // tiles of the pieces before
        for (int piece = blockIdx.x; piece < px.pieces; piece += gridDim.x) {
            const PrePiece sg = pre_piece(px, piece, a.n_prefixes);
            const bool live = row < tile_tokens * grp && sg.tile * tile_tokens + row / grp < px.rows[sg.g];
            const int tiles = sg.k1 - sg.k0, len = px.len[sg.g];
            const uint32_t n1 = n0 + tiles;
            float m_mine = -INFINITY, l_run = 0.f;                               // the sum so far and the reference that it is under
            for (uint32_t n = n0 + ((n0 ^ wg) & 1); n < n1; n += 2) {
                const int valid = len - (sg.k0 + (int)(n - n0)) * KEYS;          // keys of this tile
                const uint32_t at = n % 3, s_addr = lane_addr + at * 128;
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};     // four chains
                mbar_wait(&s_full[at], (n / 3) & 1);
                tcgen05_fence_after();
                uint32_t v[2][32];
#pragma unroll 1
                for (int k = KEYS - 64; k >= 0; k -= 64) {                       // the lower keys last: they stay in registers
                    tmem_ld_32x32b_x32(s_addr + k, v[0]);
                    tmem_ld_32x32b_x32(s_addr + k + 32, v[1]);
                    tmem_ld_wait();
                    if (valid < k + 64) {                                        // keys behind the end: -inf, also for the second reading
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) if (c * 32 + i >= valid - k) v[c][i] = 0xff800000u;
                            tmem_st_32x32b_x32(s_addr + k + c * 32, v[c]);
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[c][i]));
                }
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2e;
                if (n > 0) take_turn(n);
                // A barrier's phases are seen one by one: PV of the tile three before is the last one that this tile can be sure of without a wait
                if (n > 2) mbar_wait(&o_full[(n - 3) & 3], ((n - 3) >> 2) & 1);
                const float m_last = n > n0 ? m_s[row] : -INFINITY;
                const bool raise = mx > m_last + kRaise;
                const float m_ref = raise ? mx : m_last;
                m_s[row] = m_ref;
                if (n + 1 < n1 || piece + (int)gridDim.x < px.pieces) pass_turn(n + 1);
                if (n > n0 && (valid < KEYS || __any_sync(0xffffffffu, raise))) {
                    mbar_wait(&o_full[(n - 1) & 3], ((n - 1) >> 2) & 1);         // O has the products of all tiles before; this tile's are not issued before p_full
                    tcgen05_fence_after();
                    const float alpha = raise ? exp2f(m_last - m_ref) : 1.0f;
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
                if (valid < KEYS) {
                    tmem_st_wait();
                    // values behind the end may be anything, and 0 x inf is not 0; only the last tile of a prefix ends early, and its V is the last of the pieces' tiles so far
                    const uint32_t last = 2 * n1 - 1, slot = last % SLOTS;
                    mbar_wait(&full[slot], (last / SLOTS) & 1);
                    if (row >= valid && row < KEYS) {
#pragma unroll
                        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(kv_s + slot * Cfg::TILE_BYTES + (c >> 3) * Cfg::KV_HALF + row * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async();
                }
                if (m_mine != m_ref) { l_run *= ex2_approx(m_mine - m_ref); m_mine = m_ref; }
                const float neg_ref = -finite_or_zero(m_ref);
                uint64_t sum = 0;
#pragma unroll 1
                for (int k = 0; k < KEYS; k += 64) {
                    if (k > 0) {                                                 // read again: P of the keys before lies over their own scores
                        tmem_ld_32x32b_x32(s_addr + k, v[0]);
                        tmem_ld_32x32b_x32(s_addr + k + 32, v[1]);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = ex2_approx(fmaf(__uint_as_float(v[c][2 * i]), a.scale_log2e, neg_ref)), y = ex2_approx(fmaf(__uint_as_float(v[c][2 * i + 1]), a.scale_log2e, neg_ref));
                            sum = add_f32x2(sum, pack_f32x2(x, y));
                            w[i] = pack_bf16x2(x, y);
                        }
                        tmem_st_32x32b_x16(s_addr + k / 2 + c * 16, w);
                    }
                }
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[at]);
                float lo, hi; unpack_f32x2(sum, lo, hi);
                l_run += lo + hi;
            }
            n0 = n1;
            meet();                                                              // the last tile's reference is there
            const float m_ref = m_s[row];
            if (m_mine != m_ref) l_run *= ex2_approx(m_mine - m_ref);
            l_s[wg * 128 + row] = l_run;
            mbar_wait(&o_full[(n1 - 1) & 3], ((n1 - 1) >> 2) & 1);
            tcgen05_fence_after();
            float* po = a.pre_o + (int64_t)piece * (ROW_TILE * D) + row * 4;     // [D / 4][128 rows][4]: a warp's rows lie next to each other
#pragma unroll 1
            for (int c = wg * COLS; c < (int)(wg + 1) * COLS; c += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_addr + c, o);
                tmem_ld_wait();
                if (live)
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(po + (c + i) / 4 * (ROW_TILE * 4)) = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
            }
            tcgen05_fence_before();
            meet();                                                              // O may be written again, and both sums are there
            if (live && wg == 0) *reinterpret_cast<float2*>(a.pre_ml + ((int64_t)piece * ROW_TILE + row) * 2) = make_float2(m_ref, l_run + l_s[128 + row]);
        }
    }
    __syncthreads();
    if (warp == 1) { tcgen05_fence_after(); tmem_dealloc<512>(tmem_base); }
}

// =============================================================================================
// the sequences' own part, and the join
// =============================================================================================
template <int D, bool WIDE, int STAGES>  // WIDE: 9 to 16 heads a group, two blocks of 8 columns; STAGES: pages in the ring
struct OwnCfg {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE_BYTES = CACHE_PAGE * 128;
    static constexpr int KV_BYTES = HALVES * TILE_BYTES;
    static constexpr int STAGE_BYTES = 2 * KV_BYTES;
    static constexpr int BLOCKS = WIDE ? 2 : 1, ROWS = 8 * BLOCKS, REGS = D / 4 * BLOCKS;      // output values of a lane and its twin's in the other half
    static constexpr int Q_PITCH = D * 2 + 16, Q_BYTES = ROWS * Q_PITCH;         // queries of an item, rows 16 bytes further apart than they are long: no bank conflicts
    static constexpr int SCRATCH_BYTES = 4 * REGS * 32 * 4 + 4 * ROWS * 2 * 4;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 2 * Q_BYTES + SCRATCH_BYTES + (2 * STAGES + 6) * 8;
};
template <int D>
OA_DEVINL uint32_t own_off(int r, int d) { return (uint32_t)((d >> 6) * (CACHE_PAGE * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4)); }

// transpose of an 8 x 8 matrix of 16-bit values, a row in four lanes
OA_DEVINL uint32_t transpose_8x8(uint32_t v) { uint32_t r; asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v)); return r; }
// untiled copy of 16-byte pieces from global to shared memory, completing on an mbarrier
OA_DEVINL void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// Position in the list of (sequence, key/value head) items.  An item's units are one for the item itself (its states have to meet, which takes about as long as a page)
// and one for each of its pages: those of its prefix first, where prefixes are not a kernel of their own, then its own
struct Runs { int row0[PREFIX_MAX], rows[PREFIX_MAX], len[PREFIX_MAX]; };
struct OwnAt {
    int seq, kvh, len, run, pre_len, pre_pages, pages, next_len; int64_t unit0;              // next_len: the next sequence's, read ahead (ahead()); unit0: first unit of this item
    OA_DEVINL static int length(const PrefixAttnArgs& a, int seq) { return seq < a.n_seqs ? __ldcg(a.own_lens + seq) : 0; }
    OA_DEVINL void take(const PrefixAttnArgs& a, const Runs& runs, int raw) {
        len = (int)min((int64_t)max(raw, 0), (int64_t)a.max_own_pages * CACHE_PAGE);
        run = pre_len = pre_pages = 0;
        if (a.pre_ctas == 0)
            for (int r = 0; r < a.n_prefixes; ++r)
                if (seq >= runs.row0[r] && seq < runs.row0[r] + runs.rows[r]) { run = r; pre_len = runs.len[r]; pre_pages = pages_of(pre_len); }
        pages = pre_pages + pages_of(len);
    }
    OA_DEVINL OwnAt& ahead(const PrefixAttnArgs& a) { next_len = length(a, seq + 1); return *this; }
    OA_DEVINL void next(const PrefixAttnArgs& a, const Runs& runs) {
        unit0 += 1 + pages;
        if (++kvh == a.n_kv) { kvh = 0; ++seq; take(a, runs, next_len); ahead(a); }
    }
    OA_DEVINL int tokens(int c) const { return c < pre_pages ? pre_len - c * CACHE_PAGE : len - (c - pre_pages) * CACHE_PAGE; }      // from page c on, in its part
    OA_DEVINL const int32_t* entry(const PrefixAttnArgs& a, int c) const {
        return c < pre_pages ? a.prefix_tables + (int64_t)run * a.max_prefix_pages + c : a.own_tables + (int64_t)seq * a.max_own_pages + (c - pre_pages);
    }
};

template <int D, bool WIDE, int STAGES>
__global__ void __maxnreg__(WIDE ? 168 : 96) own_part_kernel(const __grid_constant__ CUtensorMap tm_page, const __grid_constant__ PrefixAttnArgs a) {
    using Cfg = OwnCfg<D, WIDE, STAGES>;
    constexpr int KS = D / 16, ROWS = Cfg::ROWS, NB = Cfg::BLOCKS;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_s = smem + STAGES * Cfg::STAGE_BYTES;                                         // [2 items][rows]
    float* scratch = reinterpret_cast<float*>(q_s + 2 * Cfg::Q_BYTES);                       // [4 quarters][values][32 lanes]
    float* ml_s = scratch + 4 * Cfg::REGS * 32;                                              // [4 quarters][rows][2]
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(ml_s + 4 * ROWS * 2);
    uint64_t *empty_bar = full_bar + STAGES, *q_full = empty_bar + STAGES, *q_empty = q_full + 2, *states_full = q_empty + 2, *states_empty = states_full + 1;
    __shared__ Runs runs;
    __shared__ int64_t sums[OWN_THREADS / 32];
    __shared__ OwnAt start;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv;
    if (a.pre_ctas == 0) griddep_wait();
    // ---- the plan: everything read here was written before the prefixes' kernel let this one start ----
    const int per = (a.n_seqs + OWN_THREADS - 1) / OWN_THREADS, s0 = threadIdx.x * per, s1 = min(a.n_seqs, s0 + per);
    const int first_len = OwnAt::length(a, s0);
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_page);
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], OWN_CONSUMERS / 32); }
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], OWN_CONSUMERS / 32); }
        mbar_init(states_full, OWN_CONSUMERS / 32); mbar_init(states_empty, 1);
        fence_barrier_init();
    }
    if (a.pre_ctas == 0) {
        if (warp == 8) { int row0, rows, len; read_runs(a, lane, row0, rows, len); runs.row0[lane] = row0; runs.rows[lane] = rows; runs.len[lane] = len; }
        __syncthreads();
    }
    OwnAt at;
    int64_t units = 0; bool wrong = false;
    for (at.seq = s0; at.seq < s1; ++at.seq) {
        const int len = at.seq == s0 ? first_len : OwnAt::length(a, at.seq);
        wrong = wrong || len < 0 || len > (int64_t)a.max_own_pages * CACHE_PAGE;
        at.take(a, runs, len);
        units += 1 + at.pages;
    }
    if (wrong) report(a);
    int64_t before = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t x = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += x; }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    before -= units;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < OWN_THREADS / 32; ++w) { if (w < warp) before += sums[w]; total += sums[w]; }
    before *= a.n_kv; total *= a.n_kv;
    const int64_t busy = busy_ctas(gridDim.x, total), u_begin = first_unit(blockIdx.x, busy, total), u_end = first_unit(blockIdx.x + 1, busy, total);
    if (u_begin < u_end && u_begin >= before && u_begin < before + units * a.n_kv) {         // one thread
        at.seq = s0; at.unit0 = before;
        for (at.take(a, runs, first_len); u_begin >= at.unit0 + (int64_t)(1 + at.pages) * a.n_kv;) { at.unit0 += (int64_t)(1 + at.pages) * a.n_kv; ++at.seq; at.take(a, runs, OwnAt::length(a, at.seq)); }
        at.kvh = (int)quotient(u_begin - at.unit0, 1 + at.pages); at.unit0 += (int64_t)at.kvh * (1 + at.pages);
        start = at;
    }
    __syncthreads();
    if (u_begin >= u_end) { griddep_launch(); griddep_wait(); return; }

    if (warp == 8) {
        int s = 0; uint32_t ph = 0, k = 0;
        at = start;
        at.ahead(a);
        // Page numbers come 32 at a time, one a lane, and the next 32 that will be wanted are on their way meanwhile (a look one page ahead is a chain of one latency a page: 1300 cycles, as
        // long as a page takes to arrive)
        auto block_of = [&](int seq, int block, int pages) {
            const int c = block * 32 + lane;
            if (seq == at.seq) return c < at.pages ? __ldcg(at.entry(a, c)) : 0;
            return seq < a.n_seqs && c < pages ? __ldcg(a.own_tables + (int64_t)seq * a.max_own_pages + c) : 0;
        };
        int have = 0, next = 0, have_seq = -1, have_block = 0, next_seq = -1, next_block = 0;
        for (int64_t u = u_begin; u < u_end; at.next(a, runs), ++k) {
            const int c0 = (int)max(u - at.unit0 - 1, (int64_t)0), c1 = (int)min((int64_t)at.pages, u_end - at.unit0 - 1);
            u = at.unit0 + 1 + c1;
            mbar_wait(&q_empty[k & 1], ((k >> 1) & 1) ^ 1);
            if (lane == 0) {
                if (c1 > c0) {
                    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)at.seq * a.ldq + (int64_t)at.kvh * grp * D;
                    mbar_expect_tx(&q_full[k & 1], grp * D * 2);
                    for (int r = 0; r < grp; ++r) bulk_load(q_s + (k & 1) * Cfg::Q_BYTES + r * Cfg::Q_PITCH, q + r * D, D * 2, &q_full[k & 1]);
                } else mbar_arrive(&q_full[k & 1]);
            }
            for (int c = c0; c < c1; ++c) {
                const int block = c >> 5;
                if (have_seq != at.seq || have_block != block) {
                    have = next_seq == at.seq && next_block == block ? next : block_of(at.seq, block, 0);
                    have_seq = at.seq; have_block = block;
                    if (block < (c1 - 1) >> 5) { next_seq = at.seq; next_block = block + 1; }
                    else if (block > 0 && at.kvh + 1 < a.n_kv) { next_seq = at.seq; next_block = 0; }
                    else { next_seq = a.pre_ctas > 0 || a.n_prefixes == 0 ? at.seq + 1 : -1; next_block = 0; }      // with prefixes' pages first, the next sequence's are not known yet
                    if (next_seq >= 0) next = block_of(next_seq, next_block, a.max_own_pages);
                }
                int page = __shfl_sync(0xffffffffu, have, c & 31);
                if (page < 0 || page >= a.num_pages) { if (lane == 0) report(a); page = 0; }
                mbar_wait(&empty_bar[s], ph ^ 1);
                if (lane == 0) {
                    uint8_t* kdst = smem + s * Cfg::STAGE_BYTES;
                    uint8_t* vdst = kdst + Cfg::KV_BYTES;
                    const int krow = (page * a.n_kv + at.kvh) * CACHE_PAGE, vrow = krow + a.num_pages * a.n_kv * CACHE_PAGE;
                    mbar_expect_tx(&full_bar[s], Cfg::STAGE_BYTES);                          // whole pages, also those that end early: pieces of 16 tokens were 0.7 us of 40 faster for own parts of 64 to 512 tokens, 0.5 us of 25 slower for 1 to 40
#pragma unroll
                    for (int h = 0; h < Cfg::HALVES; ++h) {
                        tma_load_2d(kdst + h * Cfg::TILE_BYTES, &tm_page, &full_bar[s], h * 64, krow, kEvictFirst);
                        tma_load_2d(vdst + h * Cfg::TILE_BYTES, &tm_page, &full_bar[s], h * 64, vrow, kEvictFirst);
                    }
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
        }
        __syncwarp();
        griddep_launch();
        griddep_wait();
        return;
    }
    if (warp == 9) {
        // An item's part: O and l of the four quarters under one maximum.  The part with an item's first unit goes to the item's own place, a later one (a CTA has at most one,
        // its first) to the CTA's
        at = start;
        at.ahead(a);
        const int g = lane >> 2, t = lane & 3;
        uint32_t k = 0;
        for (int64_t u = u_begin; u < u_end; at.next(a, runs), ++k) {
            const int64_t end = at.unit0 + 1 + at.pages, item = (int64_t)at.seq * a.n_kv + at.kvh;
            const bool first = at.unit0 >= u_begin, tokens = min(end, u_end) > max(u, at.unit0 + 1);
            u = min(end, u_end);
            if (lane == 0 && first) a.own_parts[item] = make_int2(blockIdx.x + 1, end <= u_end ? 0 : cta_of(end - 1, busy, total) - (int)blockIdx.x);      // for the join: later parts, from which CTA on
            float* po = first ? a.own_o + item * grp * D : a.more_o + (int64_t)blockIdx.x * grp * D;
            float2* ml = reinterpret_cast<float2*>(first ? a.own_ml + item * grp * 2 : a.more_ml + (int64_t)blockIdx.x * grp * 2);
            mbar_wait(states_full, k & 1);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = b * 8 + 2 * t + h;
                    float2 st[4]; float m = -INFINITY, l = 0.f;
#pragma unroll
                    for (int w = 0; w < 4; ++w) { st[w] = *reinterpret_cast<const float2*>(ml_s + (w * ROWS + row) * 2); m = fmaxf(m, st[w].x); }
                    const float ref = finite_or_zero(m);
#pragma unroll
                    for (int w = 0; w < 4; ++w) { st[w].x = ex2_approx(st[w].x - ref); l += st[w].x * st[w].y; }
                    if (row >= grp) continue;
                    if (g == 0) ml[row] = make_float2(m, tokens ? l : -1.0f);                // -1: a part without tokens
#pragma unroll 4
                    for (int r = 0; r < KS * 2; ++r) {                                       // channel block r / 2 and its upper or lower 8 channels
                        const int i = r >> 1, up = r & 1, reg = (i / (KS / 2)) * (Cfg::REGS / 2) + (b * (KS / 2) + i % (KS / 2)) * 4 + 2 * up + h;
                        float o = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; ++w) o += st[w].x * scratch[(w * Cfg::REGS + reg) * 32 + lane];
                        po[row * D + i * 16 + 8 * up + g] = o;                               // [heads][D]
                    }
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(states_empty);
        }
        griddep_launch();
        griddep_wait();
        return;
    }

    // Warps w and w + 4 take the same 16 tokens of every page and half of the channels each: scores and probabilities twice, which costs less than states of eight warps that have
    // to meet.  Tokens are the 16 rows of the first product and channels those of the second, heads the 8 columns of both: S^T = K Q^T, O^T = V^T P^T
    constexpr int KH = KS / 2;
    const int g = lane >> 2, t = lane & 3, quarter = warp & 3, half = warp >> 2;
    int s = 0, n_items = 0; uint32_t ph = 0;
    {
        at = start;
        at.ahead(a);
        for (int64_t u = u_begin; u < u_end; at.next(a, runs), ++n_items) {
            const int c0 = (int)max(u - at.unit0 - 1, (int64_t)0), c1 = (int)min((int64_t)at.pages, u_end - at.unit0 - 1);
            u = at.unit0 + 1 + c1;
            float oacc[NB][KH][4], m_run[NB][2], l_run[NB][2];                               // O^T: channels 16 i + g and + 8, heads 2 t and 2 t + 1; maxima and sums of these heads
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int i = 0; i < KH; ++i) oacc[b][i][0] = oacc[b][i][1] = oacc[b][i][2] = oacc[b][i][3] = 0.f;
                m_run[b][0] = m_run[b][1] = -INFINITY; l_run[b][0] = l_run[b][1] = 0.f;
            }
            const uint32_t qbase = smem_u32(q_s + (n_items & 1) * Cfg::Q_BYTES) + (lane & 7) * Cfg::Q_PITCH + (lane >> 3) * 16;      // rows beyond the group hold anything: columns of no head
            mbar_wait(&q_full[n_items & 1], (n_items >> 1) & 1);
            for (int c = c0; c < c1; ++c) {
                const int valid = at.tokens(c) - quarter * 16;                               // tokens of this warp's quarter
                mbar_wait(&full_bar[s], ph);
                if (valid > 0) {
                    const uint32_t kbase = smem_u32(smem + s * Cfg::STAGE_BYTES), vbase = kbase + Cfg::KV_BYTES;
                    float sacc[NB][2][4];                                                    // even and odd steps apart: two chains of products
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sacc[b][0][e] = sacc[b][1][e] = 0.f;
                    {
                        const int r = quarter * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), dsel = (lane >> 4) << 3;
#pragma unroll
                        for (int k0 = 0; k0 < KS; k0 += 4) {                                 // loads of four steps ahead of their products
                            uint32_t qf[NB][2][4], kf[4][4];
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int b = 0; b < NB; ++b) ldmatrix_x4(qbase + b * 8 * Cfg::Q_PITCH + (k0 + 2 * h) * 32, qf[b][h][0], qf[b][h][1], qf[b][h][2], qf[b][h][3]);
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) ldmatrix_x4(kbase + own_off<D>(r, (k0 + ks) * 16 + dsel), kf[ks][0], kf[ks][1], kf[ks][2], kf[ks][3]);
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                                for (int b = 0; b < NB; ++b) mma_bf16_16816(sacc[b][ks & 1], kf[ks][0], kf[ks][1], kf[ks][2], kf[ks][3], qf[b][ks >> 1][2 * (ks & 1)], qf[b][ks >> 1][2 * (ks & 1) + 1]);
                        }
                    }
                    uint32_t pb[NB][2]; float alpha[NB][2];
                    bool same = true;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float pr[4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float lo = g < valid ? (sacc[b][0][h] + sacc[b][1][h]) * a.scale_log2e : -INFINITY;
                            const float hi = g + 8 < valid ? (sacc[b][0][2 + h] + sacc[b][1][2 + h]) * a.scale_log2e : -INFINITY;
                            float mx = fmaxf(lo, hi);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                            const float m_new = fmaxf(m_run[b][h], mx), ref = finite_or_zero(m_new);
                            alpha[b][h] = ex2_approx(m_run[b][h] - ref);
                            pr[h] = ex2_approx(lo - ref); pr[2 + h] = ex2_approx(hi - ref);
                            l_run[b][h] = l_run[b][h] * alpha[b][h] + (pr[h] + pr[2 + h]);
                            same = same && m_new == m_run[b][h];
                            m_run[b][h] = m_new;
                        }
                        pb[b][0] = transpose_8x8(pack_bf16x2(pr[0], pr[1])); pb[b][1] = transpose_8x8(pack_bf16x2(pr[2], pr[3]));
                    }
                    if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int i = 0; i < KH; ++i) { oacc[b][i][0] *= alpha[b][0]; oacc[b][i][1] *= alpha[b][1]; oacc[b][i][2] *= alpha[b][0]; oacc[b][i][3] *= alpha[b][1]; }
                    }
                    const int r = quarter * 16 + ((lane >> 4) << 3) + (lane & 7), dsel = ((lane >> 3) & 1) << 3;
                    uint32_t vf[KH][4];
#pragma unroll
                    for (int i = 0; i < KH; ++i) ldmatrix_x4_trans(vbase + own_off<D>(r, (half * KH + i) * 16 + dsel), vf[i][0], vf[i][1], vf[i][2], vf[i][3]);
                    if (valid < 16) {                                                        // values behind the end may be anything, and 0 x inf is not 0
                        const uint32_t keep0 = (2 * t < valid ? 0xffffu : 0u) | (2 * t + 1 < valid ? 0xffff0000u : 0u), keep1 = (2 * t + 8 < valid ? 0xffffu : 0u) | (2 * t + 9 < valid ? 0xffff0000u : 0u);
#pragma unroll
                        for (int i = 0; i < KH; ++i) { vf[i][0] &= keep0; vf[i][1] &= keep0; vf[i][2] &= keep1; vf[i][3] &= keep1; }
                    }
#pragma unroll
                    for (int i = 0; i < KH; ++i)
#pragma unroll
                        for (int b = 0; b < NB; ++b) mma_bf16_16816(oacc[b][i], vf[i][0], vf[i][1], vf[i][2], vf[i][3], pb[b][0], pb[b][1]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[s]);
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_empty[n_items & 1]);
            // the four quarters' states, for the warp that brings them together while this one goes on
            mbar_wait(states_empty, (n_items & 1) ^ 1);
            float* mine = scratch + (quarter * Cfg::REGS + half * (Cfg::REGS / 2)) * 32 + lane;          // value [half][b][i][e]
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
            __syncwarp();
            if (lane == 0) mbar_arrive(states_full);
        }
    }

    griddep_launch();                            // not before: the next kernels' CTAs would crowd onto the SMs that are done first
    griddep_wait();                              // the join waits for this kernel alone
}

// =============================================================================================
// the join
// =============================================================================================
// One warp an item (or one of SPLIT pieces of its columns), RP rows at a time, 32 / RP lanes a row.  One pass over the parts, 16 loads of 16 bytes of eight of them in flight per
// lane; what is summed up follows a maximum that rises from batch to batch.  Bound by latency: four parts a batch in fewer registers were 2 to 8 us slower (two batches one after the other),
// two rows at a time for any group 1 us (16 bytes of a row here and there).  A kernel of its own: at the end of own_part_kernel, whose CTAs have from 2 to 20 items each, the same sums took 3 to
// 11 us, and a CTA that came last for an item had to be found by a counter.
template <int D, int RP>
__global__ void __launch_bounds__(JOIN_THREADS, JOIN_CTAS) join_parts_kernel(const __grid_constant__ PrefixAttnArgs a) {
    constexpr int SPLIT = D * RP / 256 > 1 ? D * RP / 256 : 1, LANES = 32 / RP, ITERS = D / 4 / LANES / SPLIT, MP = 8;
    const int lane = threadIdx.x & 31, grp = a.n_heads / a.n_kv, tile_tokens = ROW_TILE / grp;
    __shared__ PrefixPieces px;
    griddep_launch();
    if (a.pre_ctas > 0) {                        // from the call's arguments, while the parts are being made
        if (threadIdx.x < 32) cut_prefixes(a, px, lane);
        __syncthreads();
    }
    const int64_t tasks = (int64_t)a.n_seqs * a.n_kv * SPLIT;
    int64_t task = (int64_t)blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5), item = 0, pre_slot = 0;
    int seq = 0, kvh = 0, part = 0, n_pre = 0, first_row = 0;
    auto look = [&] {                            // where the task's row and its prefix's parts are
        if (task >= tasks) return;
        item = task / SPLIT; seq = (int)quotient(item, a.n_kv); kvh = (int)(item - (int64_t)seq * a.n_kv); part = (int)(task % SPLIT) * (D / 4 / SPLIT) + lane / RP;
        n_pre = 0;
        if (a.pre_ctas == 0) return;
        const unsigned who = __ballot_sync(0xffffffffu, px.rows[lane] > 0 && seq >= px.row0[lane] && seq < px.row0[lane] + px.rows[lane]);
        if (who) {
            const int run = __ffs(who) - 1, token = seq - px.row0[run], tile = token / tile_tokens;
            n_pre = px.split[run]; first_row = (token - tile * tile_tokens) * grp;
            pre_slot = (int64_t)px.piece0[run] + (int64_t)(kvh * px.tiles[run] + tile) * n_pre;
        }
    };
    look();
    griddep_wait();
    for (; task < tasks; task += (int64_t)gridDim.x * (JOIN_THREADS / 32), look()) {
        const int2 later = __ldcg(a.own_parts + item);
        const int n = n_pre + 1;                     // the prefix's parts and the first own one: where they lie is known; later own ones follow
        for (int r0 = 0; r0 < grp; r0 += RP) {
            const int row = r0 + lane % RP, r = row < grp ? row : grp - 1;          // lanes beyond the group go along
            const float2* pre_ml = reinterpret_cast<const float2*>(a.pre_ml) + pre_slot * ROW_TILE + first_row + r;
            const float2* own_ml = reinterpret_cast<const float2*>(a.own_ml) + item * grp + r;
            const float2* more_ml = reinterpret_cast<const float2*>(a.more_ml) + (int64_t)later.x * grp + r;
            const float* pre_o = a.pre_o + pre_slot * (ROW_TILE * D) + (first_row + r) * 4 + part * (ROW_TILE * 4);
            const float* own_o = a.own_o + (item * grp + r) * D + part * 4;
            const float* more_o = a.more_o + ((int64_t)later.x * grp + r) * D + part * 4;
            float M = -INFINITY, l = 0.f; float4 acc[ITERS]; bool some = false;
#pragma unroll
            for (int k = 0; k < ITERS; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            int i0 = 0;
            do {
                float2 ml[MP]; float4 o[MP][ITERS];
#pragma unroll
                for (int p = 0; p < MP; ++p) {
                    const int i = i0 + p;
                    ml[p] = make_float2(-INFINITY, -1.f);
                    if (i >= n && i >= n + later.y) continue;
                    const float2* m = i < n_pre ? pre_ml + (int64_t)i * ROW_TILE : i < n ? own_ml : more_ml + (int64_t)(i - n) * grp;
                    const float* src = i < n_pre ? pre_o + (int64_t)i * (ROW_TILE * D) : i < n ? own_o : more_o + (int64_t)(i - n) * (grp * D);
                    const int step = i < n_pre ? ROW_TILE * 4 * LANES : 4 * LANES;
                    ml[p] = __ldcg(m);
#pragma unroll
                    for (int k = 0; k < ITERS; ++k) o[p][k] = __ldcg(reinterpret_cast<const float4*>(src + k * step));
                }
                float m = M;
#pragma unroll
                for (int p = 0; p < MP; ++p) m = fmaxf(m, ml[p].x);
                const float ref = finite_or_zero(m), f0 = ex2_approx(M - ref);
                M = m; l *= f0;
#pragma unroll
                for (int k = 0; k < ITERS; ++k) { acc[k].x *= f0; acc[k].y *= f0; acc[k].z *= f0; acc[k].w *= f0; }
#pragma unroll
                for (int p = 0; p < MP; ++p) {
                    if (ml[p].y < 0.f) continue;                                     // a part without tokens
                    const float f = ex2_approx(ml[p].x - ref);
                    l += f * ml[p].y; some = true;
#pragma unroll
                    for (int k = 0; k < ITERS; ++k) { acc[k].x += f * o[p][k].x; acc[k].y += f * o[p][k].y; acc[k].z += f * o[p][k].z; acc[k].w += f * o[p][k].w; }
                }
                i0 += MP;
            } while (i0 < n + later.y);
            if (row < grp) {
                const float inv = some ? 1.0f / l : 0.f;
                uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)seq * a.ldo + (int64_t)(kvh * grp + row) * D + part * 4;
#pragma unroll
                for (int k = 0; k < ITERS; ++k)
                    *reinterpret_cast<uint2*>(out + k * LANES * 4) = make_uint2(pack_bf16x2(acc[k].x * inv, acc[k].y * inv), pack_bf16x2(acc[k].z * inv, acc[k].w * inv));
            }
        }
    }
}

// =============================================================================================
// host
// =============================================================================================
// Prefixes are read with the sequences' own parts, once for each sequence, where that is few pages: two launches instead of three.  us with one kernel / two, heads of 64, own parts of
// 50 to 200 tokens, rows x prefix: 4 x 256 9.0 / 10.0, 8 x 1024 11.5 / 13.1, 8 x 4096 20.1 / 15.2; 16 x 256 10.6 / 11.2, 32 x 128 12.2 / 13.0, 16 x 512 11.9 / 10.8, 32 x 256 13.5 / 12.8 (128 the same way); 9 to 15
// rows were not measured
constexpr int PREFIX_INLINE_UNITS = 4, PREFIX_FEW_ROWS = 8;           // pages an SM; up to so many rows twice as many
// Heads of 128: an SM's shared memory holds tiles of 64 keys beside four of the own parts' pages, or tiles of 128 beside two.  us with 64 / 128, own parts of 20 to 600 tokens: 128 rows of
// 4 heads a group on a prefix of 1024 41.2 / 45.7, 4096 44.5 / 48.5, 8192 48.9 / 51.8; 64 rows of 8 heads a group 1024 30.6 / 31.6, 4096 33.1 / 34.1, 6144 34.9 / 35.6, 8192 40.2 / 37.1
constexpr int PREFIX_LONG_UNITS = 24;                                 // pages an SM
PrefixAttnPlan prefix_attn_plan(int n_seqs, int n_heads, int n_kv, int head_dim, int n_prefixes, int max_prefix_pages, int max_own_pages, int sms) {
    PrefixAttnPlan p{};
    const int grp = n_heads / n_kv;
    const int tile_tokens = ROW_TILE / grp;
    const int64_t work = ((int64_t)n_seqs + tile_tokens - 1) / tile_tokens * n_kv * max_prefix_pages;       // pages, if one prefix has all rows
    const bool apart = n_prefixes > 0 && (int64_t)n_seqs * n_kv * max_prefix_pages > (n_seqs <= PREFIX_FEW_ROWS ? 2 : 1) * PREFIX_INLINE_UNITS * (int64_t)sms;
    const int64_t items = apart ? ((int64_t)n_seqs / tile_tokens + n_prefixes) * n_kv : 0;                              // no more row tiles than that, however rows fall on prefixes
    const int64_t units = items * max_prefix_pages, own_units = (int64_t)n_seqs * n_kv * (1 + (int64_t)max_own_pages + (apart ? 0 : max_prefix_pages));
    p.pre_ctas = (int)(units < sms ? units : sms);                                                                      // 0: prefixes are read with the sequences' own parts
    p.own_ctas = (int)(own_units < sms ? own_units : sms);
    p.long_prefix = apart && work >= PREFIX_LONG_UNITS * (int64_t)sms;
    p.key_tile = head_dim == 64 || p.long_prefix ? 128 : 64;
    p.pre_slots = (size_t)(items + p.pre_ctas);
    auto take = [&](size_t bytes) { const size_t at = p.bytes; p.bytes += (bytes + 255) & ~size_t(255); return at; };
    p.pre_o = take(p.pre_slots * ROW_TILE * head_dim * 4); p.pre_ml = take(p.pre_slots * ROW_TILE * 8);
    const size_t own_items = (size_t)n_seqs * n_kv;
    p.own_o = take(own_items * grp * head_dim * 4); p.own_ml = take(own_items * grp * 8); p.own_parts = take(own_items * 8);
    p.more_o = take((size_t)p.own_ctas * grp * head_dim * 4); p.more_ml = take((size_t)p.own_ctas * grp * 8);
    return p;
}

// The first two kernels' CTAs share SMs: both ask for the whole carve-out, or an SM would have to be empty before it takes the other kernel's (2 us between the kernels)
template <typename K>
static cudaError_t raise_smem(K kern, int bytes, bool (&done)[16]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev >= 0 && dev < 16 && done[dev])) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e == cudaSuccess ? ensure_dynamic_smem(kern, bytes, done) : e;
}
template <int D, bool WIDE, int STAGES>
static cudaError_t launch_own(const CUtensorMap* tm_page, const PrefixAttnArgs& a, cudaStream_t s) {
    auto kern = own_part_kernel<D, WIDE, STAGES>;
    static bool attr_done[16] = {};
    { const cudaError_t e = raise_smem(kern, OwnCfg<D, WIDE, STAGES>::SMEM_BYTES, attr_done); if (e != cudaSuccess) return e; }
    return launch_k(kern, dim3(a.own_ctas), dim3(OWN_THREADS), OwnCfg<D, WIDE, STAGES>::SMEM_BYTES, s, *tm_page, a);
}
template <int D, int KEYS, int SLOTS>
static cudaError_t launch_prefixes(const CUtensorMap* tm_q, const CUtensorMap* tm_page, const PrefixAttnArgs& a, cudaStream_t s) {
    using Cfg = PreCfg<D, KEYS, SLOTS>;
    auto kern = prefix_part_kernel<D, KEYS, SLOTS>;
    static bool attr_done[16] = {};
    { const cudaError_t e = raise_smem(kern, Cfg::SMEM_BYTES, attr_done); if (e != cudaSuccess) return e; }
    return launch_k(kern, dim3(a.pre_ctas), dim3(Cfg::THREADS), Cfg::SMEM_BYTES, s, *tm_q, *tm_page, a);
}
template <int D, int RP>
static cudaError_t launch_join(const PrefixAttnArgs& a, cudaStream_t s) {
    auto kern = join_parts_kernel<D, RP>;
    static bool attr_done[16] = {};
    { const cudaError_t e = raise_smem(kern, 0, attr_done); if (e != cudaSuccess) return e; }
    const int64_t tasks = (int64_t)a.n_seqs * a.n_kv * (D * RP / 256 > 1 ? D * RP / 256 : 1);
    const int64_t ctas = (tasks + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32), most = (int64_t)JOIN_CTAS * a.sms;
    return launch_k(kern, dim3((unsigned)(ctas < most ? ctas : most)), dim3(JOIN_THREADS), 0, s, a);
}
// KEYS, SLOTS: tiles and ring of the prefixes' kernel; PAGES: ring of the own parts'
template <int D, int KEYS, int SLOTS, int PAGES>
static cudaError_t launch_parts(const CUtensorMap* tm_q, const CUtensorMap* tm_page, const PrefixAttnArgs& a, cudaStream_t s) {
    cudaError_t e = cudaSuccess;
    if (a.pre_ctas > 0) e = launch_prefixes<D, KEYS, SLOTS>(tm_q, tm_page, a, s);
    if (e == cudaSuccess) e = a.n_heads / a.n_kv > 8 ? launch_own<D, true, PAGES>(tm_page, a, s) : launch_own<D, false, PAGES>(tm_page, a, s);
    return e;
}
cudaError_t launch_prefix_attention(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int head_dim, bool long_prefix, const PrefixAttnArgs& a, cudaStream_t s) {
    if (head_dim != 64 && head_dim != 128) return cudaErrorInvalidValue;
    // An SM's shared memory goes to both kernels: heads of 128 give the prefixes three tiles of 128 keys and the own parts two pages where prefixes are most of the work, two tiles
    // of 64 keys and four pages elsewhere
    const cudaError_t e = head_dim == 64 ? launch_parts<64, 128, 3, 8>(tm_q, tm_page, a, s)
                        : long_prefix ? launch_parts<128, 128, 3, 2>(tm_q, tm_page, a, s) : launch_parts<128, 64, 2, 4>(tm_q, tm_page, a, s);
    if (e != cudaSuccess) return e;
    const int grp = a.n_heads / a.n_kv;
    if (head_dim == 64) return grp > 4 ? launch_join<64, 8>(a, s) : grp > 2 ? launch_join<64, 4>(a, s) : launch_join<64, 2>(a, s);
    return grp > 4 ? launch_join<128, 8>(a, s) : grp > 2 ? launch_join<128, 4>(a, s) : launch_join<128, 2>(a, s);
}

}  // namespace oa
