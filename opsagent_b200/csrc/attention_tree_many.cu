// attention_tree_many.cu — attention of several new tokens: tiles of 128 rows on tcgen05.  The mathematics and the plan are attention_tree.cuh's.
//
// 128 rows of an item (as many tokens' heads of a group as fit) x 128 keys a tile: S = Q K^T in three TMEM buffers, two tiles ahead, P over S's own columns as the second product's operand, O in
// TMEM.  Two softmax warpgroups take the tiles in turn, one row a thread; the reference maximum rises (and O is rescaled) only where a score passes it by 2^8.
//
// bf16: P is rounded to bf16.  8 bits: tiles are turned into fp16 under the swizzle that the products read, by eight warps of their own.  Keys and values are multiplied by their scales on the way
// (over a power of two that none of a tile's, or of a piece's so far, passes): a softmax thread that multiplied 128 scores and weights by scales from shared memory took twice as long for a tile.
// Roundings to fp16, 2^-11 each: a key or value times its scale, a weight.  Scales come in two halves: rounded to one, an error that all channels of a key share, they left 2.4e-3 to 3.6e-3 of the output for
// scores up to 20 and 80 (single rows 6.7e-3 and 2.3e-2) instead of 1.9e-3 and 2.2e-3 (3.6e-3 and 1.0e-2), at 89 and 100 us for unequal trees of 3 to 40 tokens over e4m3 and int8, 122 and 128 for 25 tokens behind
// 100001, instead of 91, 96, 127 and 139; scores times fp32 scales in the softmax threads leave 1.7e-3 at any size and took 122, 127, 148 and 155.  Keys and values go through one code: a second copy of it cost
// the unequal trees 10 us.
// Queries are scaled by a power of two as for few rows, by a kernel before.
//
// Trees of 64 tokens behind 8 sequences of 2000 to 8000 over bf16, 32 / 8 heads of 128: 54 us in a graph, for bytes 24 at the copy rate and products 23: 0.95 us a tile (1700 cycles at the 1.7 to
// 1.8 GHz that the power cap leaves: the exponentials and the tensor pipe take 1024 each), 5 to begin, 4.5 for each piece that begins inside a CTA's share (the last product, 64 KB of parts under the next
// one's first weights, the first scores), 5 for the join.  Over 8 bits a tile takes 1.35 us (e4m3) to 1.5 (int8), 800 cycles and more for either half's conversion by the eight warps, whose loads from shared memory wait beside the products' reads: 25
// tokens of 64 / 8 heads behind 100001 tokens, int8, 139 us in a graph; unequal trees of 3 to 40 tokens, e4m3, 91 (1.5 more where both warpgroups wrote a piece's end).
#include "attention_tree.cuh"

namespace oa {

OA_DEVINL void mbar_wait3(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, uint64_t* c, uint32_t pc) {        // phases that do not pass before this thread's own arrivals
    uint32_t spins = 0;
    for (;;) {
        const bool x = mbar_try_wait(a, pa), y = mbar_try_wait(b, pb), z = mbar_try_wait(c, pc);
        if (x && y && z) return;
        if (++spins > OA_MBAR_SPIN_LIMIT) { __trap(); }
    }
}
OA_DEVINL uint32_t mul_f16x2(uint32_t a, uint32_t b) { uint32_t r; asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
OA_DEVINL uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) { uint32_t r; asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c)); return r; }

struct TrueTag { static constexpr bool value = true; };
struct FalseTag { static constexpr bool value = false; };

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
    static constexpr int SC = 8, SC_FLOATS = 2 * KEYS + 4;                       // tiles whose scales wait: keys', values', what keys' are over, what O is multiplied by for larger scales of values and at its end
    static constexpr int CONV = BITS8 ? 8 : 0, THREADS = 128 + 256 + 32 * CONV;     // producer, issuer, scales, pieces; eight softmax warps; warps that convert
    static constexpr int BARS = 19 + 2 * SLOTS + 2 * RAW + (BITS8 ? 2 * SC : 0);
    static constexpr int SMEM_BYTES = TILE_BYTES + SLOTS * TILE_BYTES + RAW * RAW_BYTES + (BITS8 ? SC * SC_FLOATS * 4 : 0) + 5 * 128 * 4 + BARS * 8 + 16 + 2 * sizeof(TreePiece);
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
    constexpr float kUp = 128.f;                                                             // scales over their reference times this: the largest product is 57344 (e4m3), which fp16 holds
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_s = smem;
    uint8_t* kv_s = q_s + TILE;
    uint8_t* raw_s = kv_s + SLOTS * TILE;
    float* sc_s = reinterpret_cast<float*>(raw_s + Cfg::RAW * Cfg::RAW_BYTES);
    float* m_s = sc_s + (BITS8 ? SC * Cfg::SC_FLOATS : 0);                                   // a row's reference maximum, and a warpgroup's reference and sum of a piece [piece & 1][row]
    float2* ml_s = reinterpret_cast<float2*>(m_s + 128);
    uint64_t* bars = reinterpret_cast<uint64_t*>(ml_s + 256);
    uint64_t *q_full = bars, *q_empty = bars + 1, *s_full = bars + 2, *p_full = bars + 5, *o_full = bars + 8, *o_read = bars + 12, *full = bars + 13, *empty = full + SLOTS;
    uint64_t *piece_full = empty + SLOTS, *rows_full = piece_full + 2, *piece_empty = rows_full + 2, *raw_full = piece_empty + 2, *raw_empty = raw_full + Cfg::RAW, *sc_full = raw_empty + Cfg::RAW, *sc_empty = sc_full + SC;
    TreePiece* piece_s = reinterpret_cast<TreePiece*>(bars + Cfg::BARS);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(piece_s + 2);
    __shared__ int64_t sums[Cfg::THREADS / 32];
    __shared__ At start;

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv, tile_tokens = 128 / grp;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_q);
        if (!BITS8) tma_prefetch_desc(&tm_kv);
        mbar_init(q_full, 1); mbar_init(q_empty, 1); mbar_init(o_read, 4);
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
                        if (j == 0 && seg > 1) mbar_wait(o_read, seg & 1);           // O of the piece before has been read
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
            // A tile's scales, keys' over a power of two that none of the tile passes, values' over one that none of the piece so far passes, and either times 2^7; 0 of what none of the rows sees.  In two halves of
            // fp16: one alone would be off by 2^-11 of itself, which all of a key's channels share, so that a score would be off by as much
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
                            const float inv = 1.0f / ref[v];                         // a power of two: exact
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float y = x[i] * inv * kUp, hi = __half2float(__float2half_rn(y));
                                w[i] = pack_f16x2(hi, y == hi ? 0.f : y - hi);       // an infinite one has no second half
                            }
                            *reinterpret_cast<uint4*>(sc + v * KEYS + 4 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        vref = ref[1];
                        if (lane == 0) { sc[2 * KEYS] = ref[0]; sc[2 * KEYS + 1] = grown; sc[2 * KEYS + 2] = vref * (1.0f / kUp); }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sc_full[buf]);
                    }
                });
            }
        } else {
            At at;
            at = start;
            uint32_t k = 0;
            for (int64_t u = u_begin; u < u_end; ++k) {
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
                if (u < u_end) at.next(a);
            }
        }
    } else if (warp < 12) {
        if constexpr (BITS8) reg_inc<136>();
        // Two warpgroups take the tiles in turn, a row a thread: one's exponentials run under the other's loads and maxima.  A row's reference maximum goes from one to the other
        // with each tile, as soon as the tile's own maximum is known; sums stay with either, O is one for both
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t wg = (warp - 4) >> 2, lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16), o_addr = lane_addr + Cfg::O_COL;
        // Of a piece's end: the warpgroup that had its last tile waits for the other's sum and writes the piece, under the other's first tile of the next one.  Neither is two pieces behind the other
        auto take_sum = [](uint32_t k) { if (k & 1) asm volatile("bar.sync 5, %0;" ::"n"(SOFTMAX) : "memory"); else asm volatile("bar.sync 2, %0;" ::"n"(SOFTMAX) : "memory"); };
        auto pass_sum = [](uint32_t k) { if (k & 1) asm volatile("bar.arrive 5, %0;" ::"n"(SOFTMAX) : "memory"); else asm volatile("bar.arrive 2, %0;" ::"n"(SOFTMAX) : "memory"); };
        auto take_turn = [](uint32_t n) {                                        // tile n - 1 has left its reference
            if (n & 1) asm volatile("bar.sync 3, %0;" ::"n"(SOFTMAX) : "memory"); else asm volatile("bar.sync 4, %0;" ::"n"(SOFTMAX) : "memory");
        };
        auto pass_turn = [](uint32_t n) {                                        // to tile n
            if (n & 1) asm volatile("bar.arrive 3, %0;" ::"n"(SOFTMAX) : "memory"); else asm volatile("bar.arrive 4, %0;" ::"n"(SOFTMAX) : "memory");
        };
        constexpr float kRaise = 8.0f;                                           // log2 units a score may pass the reference by
        constexpr float kLift = BITS8 ? 7.0f : 0.0f;                             // of the weights, which fp16 holds up to 2^16 and with 8 bits down to 2^-17
        uint32_t n0 = 0, seg = 0;                                                // tiles of the pieces before, pieces
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
                    for (int c = wg * (D / 2); c < (int)(wg + 1) * (D / 2); c += 4) *reinterpret_cast<float4*>(po + c * 128) = make_float4(0.f, 0.f, 0.f, 0.f);
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
                    // Never 0, by which a masked score, -inf, would be NaN: scores of a tile whose visible keys are all zero, or whose row of queries is, are 0 times this, others so small move by less than 2^-80
                    fac = fmaxf(fac * sc[0] * (1.0f / kUp), 0x1p-126f); grown = sc[1]; undo = sc[2];
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
            float2* pair = ml_s + (seg & 1) * 128 + row;
            if (((n1 - 1) & 1) != wg) {
                *pair = make_float2(m_mine, l_run);
                pass_sum(seg++);
                return;
            }
            take_sum(seg++);
            const float2 other = *pair;
            const float m_ref = m_mine, l = l_run + (other.x == m_ref ? other.y : other.y * ex2_approx(other.x - m_ref));       // the last tile's reference is the piece's
            mbar_wait(&o_full[(n1 - 1) & 3], ((n1 - 1) >> 2) & 1);
            tcgen05_fence_after();
            const bool whole = first && p.last;
            const float mult = undo * (whole ? (blind ? 0.f : 1.0f / l) : 1.0f);
            const int token = row / grp;
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(p.row0 + token) * a.ldo + (int64_t)(p.kvh * grp + row - token * grp) * D;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
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
            __syncwarp();
            if (lane == 0) mbar_arrive(o_read);
            if (live && !whole) *ml = make_float2(m_ref - kLift, first && blind ? -1.f : l);
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
                    auto convert = [&] {                             // as a function of its own: written in line the compiler's order took 92, 98, 128.5 and 140 us
#pragma unroll
                        for (int h = 0; h < STEPS; h += AHEAD) {                     // loads ahead of their stores
                            uint4 x[AHEAD]; uint32_t f[AHEAD];
#pragma unroll
                            for (int i = 0; i < AHEAD; ++i) { x[i] = *reinterpret_cast<const uint4*>(src + key_of(h + i) * D); f[i] = sc[key_of(h + i)]; }
#pragma unroll
                            for (int i = 0; i < AHEAD; ++i) {
                                uint32_t y[8];
                                const uint32_t w4[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, hi = __byte_perm(f[i], 0, 0x1010), lo = __byte_perm(f[i], 0, 0x3232);
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    to_f16<FMT, false>(w4[k], y[2 * k], y[2 * k + 1]);
                                    y[2 * k] = fma_f16x2(y[2 * k], hi, mul_f16x2(y[2 * k], lo)); y[2 * k + 1] = fma_f16x2(y[2 * k + 1], hi, mul_f16x2(y[2 * k + 1], lo));
                                }
                                const int key = key_of(h + i);
                                *reinterpret_cast<uint4*>(dst + key * 128 + (((2 * (ch & 3)) ^ (key & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
                                *reinterpret_cast<uint4*>(dst + key * 128 + (((2 * (ch & 3) + 1) ^ (key & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
                            }
                        }
                    };
                    convert();
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

template <int D, int FMT>
static cudaError_t launch_many(const CUtensorMap* tm_q, const CUtensorMap* tm_page, const TreeAttnArgs& a, cudaStream_t s) {
    using Cfg = ManyCfg<D, FMT>;
    auto kern = tree_many_kernel<D, FMT>;
    static bool attr_done[16] = {};
    cudaError_t e = ensure_dynamic_smem(kern, Cfg::SMEM_BYTES, attr_done);
    if (e == cudaSuccess && FMT != CACHE_BF16) e = launch_k(tree_queries_kernel<D>, dim3((unsigned)(((int64_t)a.n_rows * a.n_heads + 31) / 32)), dim3(128), 0, s, a);
    return e == cudaSuccess ? launch_k(kern, dim3(a.ctas), dim3(Cfg::THREADS), Cfg::SMEM_BYTES, s, *tm_q, *tm_page, a) : e;
}
template <int D>
static cudaError_t launch_many_of(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int format, const TreeAttnArgs& a, cudaStream_t s) {
    return format == CACHE_BF16 ? launch_many<D, CACHE_BF16>(tm_q, tm_page, a, s) : format == CACHE_E4M3 ? launch_many<D, CACHE_E4M3>(tm_q, tm_page, a, s) : launch_many<D, CACHE_INT8>(tm_q, tm_page, a, s);
}
cudaError_t launch_tree_many(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int head_dim, int format, const TreeAttnArgs& a, cudaStream_t s) {
    return head_dim == 64 ? launch_many_of<64>(tm_q, tm_page, format, a, s) : head_dim == 128 ? launch_many_of<128>(tm_q, tm_page, format, a, s) : cudaErrorInvalidValue;
}

}  // namespace oa
