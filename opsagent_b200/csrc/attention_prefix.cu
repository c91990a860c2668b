// attention_prefix.cu — decode attention of a batch whose sequences share prefixes: a prefix's keys and values are read once for all rows that see them.
//
//   out_i = softmax(scale q_i [K_prefix; K_own(i)]^T) [V_prefix; V_own(i)]
//
// The softmax splits over any partition of the keys: a part leaves its maximum m, l = sum 2^(s - m) and O = sum 2^(s - m) v, and parts join as
// O = sum_i 2^(m_i - M) O_i, l likewise, M = max m_i.  Two kernels make the parts, the second also joins them:
//
//  prefix_part_kernel: all rows of a prefix against its keys is a product of matrices (128 conversations of 4 heads a group: 512 rows a key/value head), so it
//    runs on tcgen05: 128 rows (as many tokens' heads of a group as fit) x 128 keys a unit, S = Q K^T in two TMEM buffers, P over S's own columns as the second
//    product's operand, O in TMEM.  One row a thread, reference maximum raised (and O rescaled) only where a score passes it by 2^8.
//  own_part_kernel: a sequence's own keys have only its few heads as rows: streamed through shared memory by TMA and multiplied on the 16-row warp path,
//    a page's 64 tokens over four warps, like decode attention over a whole context (attention.cu).
//
// Both deal their units (128 keys of a row tile; a page of a sequence and key/value head) out contiguously, the same number to every CTA: unit u is CTA
// floor(((u + 1) G - 1) / total)'s, so what parts an item has, and in which slot (CTA + item) each of them lies, follows from lengths alone.  The plan is made on the
// device, by every CTA for itself: lengths may come from the kernel before, a captured call serves other lengths when it is replayed, and the host waits for nothing.
// Parts are joined in one order, whatever came first: the same call gives the same bits.
//
// The second kernel starts beside the first (it needs nothing of it until it joins): it streams own keys from memory while the first is busy with products.
#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"

namespace oa {

constexpr int PRE_THREADS = 192;        // producer, issuer, four softmax warps
constexpr int OWN_THREADS = 160;        // four consumer warps, producer
constexpr int KEY_TILE = 128;

OA_DEVINL float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }        // nothing seen: any reference will do, 2^(-inf - 0) is 0
OA_DEVINL int own_pages(int len) { return len > CACHE_PAGE ? (len + CACHE_PAGE - 1) / CACHE_PAGE : 1; }       // an empty sequence has a page without tokens: somebody writes its row
// of a grid's CTAs the first min(grid, total) have units, each at least one: an item's parts are those of consecutive CTAs
OA_DEVINL int64_t busy_ctas(int64_t grid, int64_t total) { return total < grid ? (total > 0 ? total : 1) : grid; }
OA_DEVINL int64_t first_unit(int64_t cta, int64_t busy, int64_t total) { return cta < busy ? total * cta / busy : total; }
OA_DEVINL int cta_of(int64_t unit, int64_t busy, int64_t total) { return (int)(((unit + 1) * busy - 1) / total); }
OA_DEVINL void report(const PrefixAttnArgs& a) { if (a.status) *a.status = 400; }

// What the prefixes' part looks like, the same in both kernels: run bounds that never fall, lengths that fit their tables
struct Prefixes {
    int row0[PREFIX_MAX], rows[PREFIX_MAX], len[PREFIX_MAX], tiles[PREFIX_MAX], key_tiles[PREFIX_MAX], item0[PREFIX_MAX];
    int64_t unit0[PREFIX_MAX], units;
};
OA_DEVINL void read_prefixes(const PrefixAttnArgs& a, Prefixes& px, int tile_tokens, int lane) {      // one warp
    int r0 = 0, r1 = 0, len = 0; bool wrong = false;
    if (lane < a.n_prefixes) {
        r0 = __ldcg(a.prefix_rows + lane); r1 = __ldcg(a.prefix_rows + lane + 1); len = __ldcg(a.prefix_lens + lane);
        wrong = r0 < 0 || r1 < r0 || r1 > a.n_seqs || len < 0 || len > (int64_t)a.max_prefix_pages * CACHE_PAGE;
        r0 = min(max(r0, 0), a.n_seqs); r1 = min(max(r1, 0), a.n_seqs);
        len = (int)min((int64_t)max(len, 0), (int64_t)a.max_prefix_pages * CACHE_PAGE);
    }
    if (wrong) report(a);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int below = __shfl_up_sync(0xffffffffu, r0, o); if (lane >= o) r0 = max(r0, below); }
    r1 = max(r0, r1);
    const bool some = lane < a.n_prefixes && r1 > r0 && len > 0;
    const int tiles = some ? (r1 - r0 + tile_tokens - 1) / tile_tokens : 0, key_tiles = some ? (len + KEY_TILE - 1) / KEY_TILE : 0;
    int items = tiles * a.n_kv; int64_t units = (int64_t)items * key_tiles;
    const int items_own = items; const int64_t units_own = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int i = __shfl_up_sync(0xffffffffu, items, o); const int64_t u = __shfl_up_sync(0xffffffffu, units, o);
        if (lane >= o) { items += i; units += u; }
    }
    px.row0[lane] = r0; px.rows[lane] = some ? r1 - r0 : 0; px.len[lane] = len; px.tiles[lane] = tiles; px.key_tiles[lane] = key_tiles;
    px.item0[lane] = items - items_own; px.unit0[lane] = units - units_own;
    if (lane == 31) px.units = units;
}

// =============================================================================================
// the prefixes' part
// =============================================================================================
template <int D>
struct PreCfg {
    static constexpr int HALVES = D / 64;
    static constexpr int HALF_BYTES = 128 * 128;                 // 128 rows x 64 bf16 columns under the 128-byte swizzle
    static constexpr int TILE_BYTES = HALVES * HALF_BYTES;       // Q, and K or V of 128 keys
    static constexpr int NK = 2, NV = 1;
    static constexpr int SMEM_BYTES = (1 + NK + NV) * TILE_BYTES + 256;
    static constexpr uint32_t O_COL = 256;                       // TMEM: S[0] and P[0] at 0, S[1] and P[1] at 128, O at 256
};
struct PreSeg { int g, kvh, tile, k0, k1, item; };
// the segment that begins at unit u, at most `left` units long; g0: a prefix at or before it
OA_DEVINL PreSeg pre_segment(const Prefixes& px, int64_t u, int64_t left, int g0, int n_prefixes) {
    PreSeg s; s.g = g0;
    while (s.g + 1 < n_prefixes && u >= px.unit0[s.g + 1]) ++s.g;          // prefixes without units begin where the next one does
    const int64_t rem = u - px.unit0[s.g];
    const int kt = px.key_tiles[s.g], i = (int)(rem / kt);
    s.k0 = (int)(rem - (int64_t)i * kt); s.k1 = (int)min((int64_t)kt, s.k0 + left);
    s.kvh = i / px.tiles[s.g]; s.tile = i - s.kvh * px.tiles[s.g]; s.item = px.item0[s.g] + i;
    return s;
}

template <int D>
__global__ void __launch_bounds__(PRE_THREADS, 1) prefix_part_kernel(const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ PrefixAttnArgs a) {
    using Cfg = PreCfg<D>;
    constexpr int HALVES = Cfg::HALVES, NK = Cfg::NK, NV = Cfg::NV;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_s = smem;
    uint8_t* k_s = q_s + Cfg::TILE_BYTES;
    uint8_t* v_s = k_s + NK * Cfg::TILE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + NV * Cfg::TILE_BYTES);
    uint64_t *q_full = bars, *s_full = bars + 1, *p_full = bars + 3, *t_full = bars + 5, *o_full = bars + 6;
    uint64_t *k_full = bars + 7, *k_empty = k_full + NK, *v_full = k_empty + NK, *v_empty = v_full + NV;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + NV);
    __shared__ Prefixes px;

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv, tile_tokens = KEY_TILE / grp;
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tm_kv);
        mbar_init(q_full, 4); mbar_init(t_full, 1); mbar_init(o_full, 1);
        for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); }
        for (int i = 0; i < NK; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < NV; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc<512>(tmem_slot);
    griddep_wait();
    griddep_launch();            // behind the wait: what the own part's kernel reads ahead of its own wait was written by kernels that have ended
    if (warp == 0) read_prefixes(a, px, tile_tokens, lane);
    for (int i = blockIdx.x * PRE_THREADS + threadIdx.x; i < a.own_ctas; i += gridDim.x * PRE_THREADS) a.counters[i] = 0;
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int64_t total = px.units, busy = busy_ctas(gridDim.x, total);
    const int64_t u_begin = first_unit(blockIdx.x, busy, total), u_end = first_unit(blockIdx.x + 1, busy, total);

    if (warp == 0) {
        uint32_t n = 0;                                          // tiles loaded
        int g = 0;
        for (int64_t u = u_begin; u < u_end;) {
            const PreSeg sg = pre_segment(px, u, u_end - u, g, a.n_prefixes); g = sg.g; u += sg.k1 - sg.k0;
            const int32_t* bt = a.prefix_tables + (size_t)sg.g * a.max_prefix_pages;
            const int pages = (px.len[sg.g] + CACHE_PAGE - 1) / CACHE_PAGE;
            for (int kt = sg.k0; kt < sg.k1; ++kt, ++n) {
                const int two = 2 * kt + 1 < pages;              // a missing second page is not loaded: its scores are masked, its values set to zero
                int page[2] = {bt[2 * kt], two ? bt[2 * kt + 1] : 0};
#pragma unroll
                for (int i = 0; i < 2; ++i) if (page[i] < 0 || page[i] >= a.num_pages) { if (lane == 0) report(a); page[i] = 0; }
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const uint32_t slot = n % (v ? NV : NK), turn = n / (v ? NV : NK);
                    uint64_t* full = (v ? v_full : k_full) + slot;
                    mbar_wait((v ? v_empty : k_empty) + slot, (turn & 1) ^ 1);
                    if (elect_one()) {
                        uint8_t* dst = (v ? v_s : k_s) + slot * Cfg::TILE_BYTES;
                        mbar_expect_tx(full, two ? Cfg::TILE_BYTES : Cfg::TILE_BYTES / 2);
                        for (int i = 0; i <= two; ++i) {
                            const int row = ((v ? a.num_pages : 0) + page[i]) * a.n_kv * CACHE_PAGE + sg.kvh * CACHE_PAGE;
#pragma unroll
                            for (int h = 0; h < HALVES; ++h) tma_load_2d(dst + h * Cfg::HALF_BYTES + i * 8192, &tm_kv, full, h * 64, row, kEvictLast);
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp == 1) {
        // the whole warp walks the loop, an elected lane issues: descriptors stay in uniform registers
        constexpr uint32_t idesc_s = umma_idesc_bf16(128, KEY_TILE), idesc_o = umma_idesc_bf16_bmn(128, D);
        const uint64_t q_desc = umma_desc_sw128(smem_u32(q_s)), k_desc = umma_desc_sw128(smem_u32(k_s));
        const uint64_t v_desc = umma_desc_sw128_mn(smem_u32(v_s), (uint32_t)Cfg::HALF_BYTES, 1024u);
        auto issue_s = [&](uint32_t n) {
            const uint32_t slot = n % NK;
            mbar_wait(&k_full[slot], (n / NK) & 1);
            tcgen05_fence_after();
            if (elect_one()) {
                const uint64_t b = k_desc + (uint64_t)(slot * (Cfg::TILE_BYTES >> 4));
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint64_t off = (uint64_t)(((ks >> 2) * Cfg::HALF_BYTES + (ks & 3) * 32) >> 4);
                    umma_bf16(tmem_base + (n & 1) * 128, q_desc + off, b + off, idesc_s, ks > 0 ? 1u : 0u);
                }
                umma_commit(&s_full[n & 1]);
                umma_commit(&k_empty[slot]);
            }
            __syncwarp();
        };
        uint32_t n = 0, seg = 0; int g = 0;
        for (int64_t u = u_begin; u < u_end; ++seg) {
            const PreSeg sg = pre_segment(px, u, u_end - u, g, a.n_prefixes); g = sg.g; u += sg.k1 - sg.k0;
            const int tiles = sg.k1 - sg.k0;
            mbar_wait(q_full, seg & 1);
            tcgen05_fence_after();
            issue_s(n);
            for (int j = 0; j < tiles; ++j, ++n) {
                if (j + 1 < tiles) issue_s(n + 1);               // S of the next tile goes over the scores of the one before, whose P the tensor core has been told to read
                const uint32_t slot = n % NV;
                mbar_wait(&p_full[n & 1], (n >> 1) & 1);
                mbar_wait(&v_full[slot], (n / NV) & 1);
                tcgen05_fence_after();
                if (elect_one()) {
                    const uint64_t b = v_desc + (uint64_t)(slot * (Cfg::TILE_BYTES >> 4));
#pragma unroll
                    for (int ks = 0; ks < KEY_TILE / 16; ++ks)
                        umma_bf16_ta(tmem_base + Cfg::O_COL, tmem_base + (n & 1) * 128 + ks * 8, b + (uint64_t)(ks * (2048 >> 4)), idesc_o, (j > 0 || ks > 0) ? 1u : 0u);
                    umma_commit(j + 1 < tiles ? t_full : o_full);
                    umma_commit(&v_empty[slot]);
                }
                __syncwarp();
            }
        }
    } else {
        const int quarter = warp & 3, row = quarter * 32 + lane;                 // this thread's row, TMEM lane of the same number
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        constexpr float kRaise = 8.0f;                                           // log2 units a score may pass the reference by
        uint32_t n = 0, seg = 0, rescaled0 = 0; int g = 0;                       // rescaled0: completions of t_full before this segment
        for (int64_t u = u_begin; u < u_end; ++seg) {
            const PreSeg sg = pre_segment(px, u, u_end - u, g, a.n_prefixes); g = sg.g; u += sg.k1 - sg.k0;
            const int tiles = sg.k1 - sg.k0, len = px.len[sg.g];
            const int token = sg.tile * tile_tokens + row / grp;
            const bool live = row < tile_tokens * grp && token < px.rows[sg.g];
            {   // Q: a row of 128 or 256 bytes a thread, zeros where there is none
                const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(px.row0[sg.g] + (live ? token : 0)) * a.ldq +
                                                                  (int64_t)(sg.kvh * grp + (live ? row % grp : 0)) * D);
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const uint4 w = live ? src[c] : make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(q_s + (c >> 3) * Cfg::HALF_BYTES + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = w;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            float m_ref = -INFINITY, l_run = 0.f;
            for (int j = 0; j < tiles; ++j, ++n) {
                const uint32_t sb = n & 1;
                const int valid = len - (sg.k0 + j) * KEY_TILE;                 // keys of this tile
                mbar_wait(&s_full[sb], (n >> 1) & 1);
                tcgen05_fence_after();
                uint32_t v[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(tmem_base + lane_addr + sb * 128 + c * 32, v[c]);
                tmem_ld_wait();
                if (valid < KEY_TILE) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) if (c * 32 + i >= valid) v[c][i] = 0xff800000u;
                    // values behind the end may be anything, and 0 x inf is not 0
                    const uint32_t slot = n % NV;
                    mbar_wait(&v_full[slot], (n / NV) & 1);
                    if (row >= valid) {
#pragma unroll
                        for (int h = 0; h < HALVES; ++h)
#pragma unroll
                            for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(v_s + slot * Cfg::TILE_BYTES + h * Cfg::HALF_BYTES + row * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async();
                }
                float mraw = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) mraw = fmaxf(mraw, __uint_as_float(v[c][i]));
                const float mx = mraw * a.scale_log2e;
                const bool raise = mx > m_ref + kRaise;
                if (__any_sync(0xffffffffu, raise)) {
                    if (j > 0) {
                        mbar_wait(t_full, (rescaled0 + j - 1) & 1);             // O has the products of the tile before; this tile's are not issued before p_full
                        tcgen05_fence_after();
                        const float alpha = raise ? exp2f(m_ref - mx) : 1.0f;
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld_32x32b_x32(tmem_base + lane_addr + Cfg::O_COL + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st_32x32b_x32(tmem_base + lane_addr + Cfg::O_COL + c, o);
                        }
                        l_run *= alpha;
                    }
                    if (raise) m_ref = mx;
                }
                const float neg_ref = -finite_or_zero(m_ref);
                uint64_t sum = 0;
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float x = ex2_approx(fmaf(__uint_as_float(v[c + (i >> 4)][(2 * i) & 31]), a.scale_log2e, neg_ref));
                        const float y = ex2_approx(fmaf(__uint_as_float(v[c + (i >> 4)][(2 * i + 1) & 31]), a.scale_log2e, neg_ref));
                        sum = add_f32x2(sum, pack_f32x2(x, y));
                        w[i] = pack_bf16x2(x, y);
                    }
                    tmem_st_32x32b_x32(tmem_base + lane_addr + sb * 128 + c * 16, w);
                }
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[sb]);
                float even, odd; unpack_f32x2(sum, even, odd);
                l_run += even + odd;
            }
            rescaled0 += tiles - 1;
            mbar_wait(o_full, seg & 1);
            tcgen05_fence_after();
            const int64_t slot = (int64_t)blockIdx.x + sg.item;
            float* po = a.pre_o + slot * (KEY_TILE * D) + row * 4;               // [D / 4][128 rows][4]: a warp's rows lie next to each other
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(tmem_base + lane_addr + Cfg::O_COL + c, o);
                tmem_ld_wait();
                if (live)
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(po + (c + i) / 4 * (KEY_TILE * 4)) = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
            }
            if (live) *reinterpret_cast<float2*>(a.pre_ml + (slot * KEY_TILE + row) * 2) = make_float2(m_ref, l_run);
            tcgen05_fence_before();
        }
    }
    __syncthreads();
    if (warp == 1) { tcgen05_fence_after(); tmem_dealloc<512>(tmem_base); }
}

// =============================================================================================
// the sequences' own part, and the join
// =============================================================================================
template <int D, bool WIDE>              // WIDE: 9 to 16 heads a group, both halves of the 16-row tile
struct OwnCfg {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE_BYTES = CACHE_PAGE * 128;
    static constexpr int KV_BYTES = HALVES * TILE_BYTES;
    static constexpr int STAGE_BYTES = 2 * KV_BYTES;
    static constexpr int STAGES = D == 128 ? 2 : 4;
    static constexpr int ROWS = WIDE ? 16 : 8;
    static constexpr int REGS = D / 4 * (WIDE ? 2 : 1);                          // output values of a lane
    static constexpr int SCRATCH_BYTES = 4 * REGS * 32 * 4 + 4 * ROWS * 2 * 4;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + SCRATCH_BYTES + 2 * STAGES * 8;
};
template <int D>
OA_DEVINL uint32_t own_off(int r, int d) { return (uint32_t)((d >> 6) * (CACHE_PAGE * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4)); }

// position in the list of (sequence, key/value head) items
struct OwnAt {
    int seq, kvh, len, pages; int64_t unit0;                                     // unit0: first unit of this item
    OA_DEVINL void read(const PrefixAttnArgs& a) {
        len = __ldcg(a.own_lens + seq);
        len = (int)min((int64_t)max(len, 0), (int64_t)a.max_own_pages * CACHE_PAGE);
        pages = own_pages(len);
    }
    OA_DEVINL void next(const PrefixAttnArgs& a) {
        unit0 += pages;
        if (++kvh == a.n_kv) { kvh = 0; if (++seq < a.n_seqs) read(a); }
    }
};

// joins the parts of one item's rows and writes them; one warp, RP rows at a time, 32 / RP lanes a row
template <int D, int RP>
OA_DEVINL void join_item(const PrefixAttnArgs& a, const Prefixes& px, const OwnAt& at, int c_first, int c_last, int grp, int tile_tokens, int lane) {
    constexpr int LANES = 32 / RP, ITERS = D / 4 / LANES;
    const int part = lane / RP;
    // the row's prefix, if it has one
    int mine = -1;
    { const bool in = px.rows[lane] > 0 && at.seq >= px.row0[lane] && at.seq < px.row0[lane] + px.rows[lane]; const unsigned who = __ballot_sync(0xffffffffu, in); if (who) mine = __ffs(who) - 1; }
    int n_pre = 0, first_row = 0; int64_t pre_slot = 0;
    if (mine >= 0) {
        const int token = at.seq - px.row0[mine], tile = token / tile_tokens, i = at.kvh * px.tiles[mine] + tile;
        const int64_t u = px.unit0[mine] + (int64_t)i * px.key_tiles[mine];
        const int64_t busy = busy_ctas(a.pre_ctas, px.units);
        const int c0 = cta_of(u, busy, px.units), c1 = cta_of(u + px.key_tiles[mine] - 1, busy, px.units);
        n_pre = c1 - c0 + 1; pre_slot = (int64_t)c0 + px.item0[mine] + i; first_row = (token - tile * tile_tokens) * grp;
    }
    const int n_own = c_last - c_first + 1;
    const int64_t own_slot = (int64_t)c_first + (int64_t)at.seq * a.n_kv + at.kvh;
    const bool nothing = at.len == 0 && mine < 0;
    for (int r0 = 0; r0 < grp; r0 += RP) {
        const int row = r0 + lane % RP, r = row < grp ? row : grp - 1;          // lanes beyond the group go along for the shuffles
        const float2* pre_ml = reinterpret_cast<const float2*>(a.pre_ml) + pre_slot * KEY_TILE + first_row + r;
        const float2* own_ml = reinterpret_cast<const float2*>(a.own_ml) + own_slot * grp + r;
        const float* pre_o = a.pre_o + pre_slot * (KEY_TILE * D) + (first_row + r) * 4 + part * (KEY_TILE * 4);
        const float* own_o = a.own_o + own_slot * (grp * D) + r * 4 + part * (grp * 4);
        float M = -INFINITY;
        for (int i = part; i < n_pre; i += LANES) M = fmaxf(M, __ldcg(pre_ml + (int64_t)i * KEY_TILE).x);
        for (int i = part; i < n_own; i += LANES) M = fmaxf(M, __ldcg(own_ml + (int64_t)i * grp).x);
#pragma unroll
        for (int o = RP; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        M = finite_or_zero(M);
        float l = 0.f; float4 acc[ITERS];
#pragma unroll
        for (int k = 0; k < ITERS; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float2 ml, const float* o, int step) {
            const float f = exp2f(ml.x - M);
            l += f * ml.y;
#pragma unroll
            for (int k = 0; k < ITERS; ++k) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(o + (int64_t)k * LANES * step));
                acc[k].x += f * x.x; acc[k].y += f * x.y; acc[k].z += f * x.z; acc[k].w += f * x.w;
            }
        };
#pragma unroll 2
        for (int i = 0; i < n_pre; ++i) add(__ldcg(pre_ml + (int64_t)i * KEY_TILE), pre_o + (int64_t)i * (KEY_TILE * D), KEY_TILE * 4);
#pragma unroll 2
        for (int i = 0; i < n_own; ++i) add(__ldcg(own_ml + (int64_t)i * grp), own_o + (int64_t)i * (grp * D), grp * 4);
        if (row < grp) {
            const float inv = nothing ? 0.f : 1.0f / l;
            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)at.seq * a.ldo + (int64_t)(at.kvh * grp + row) * D + part * 4;
#pragma unroll
            for (int k = 0; k < ITERS; ++k)
                *reinterpret_cast<uint2*>(out + k * LANES * 4) = make_uint2(pack_bf16x2(acc[k].x * inv, acc[k].y * inv), pack_bf16x2(acc[k].z * inv, acc[k].w * inv));
        }
    }
}

template <int D, bool WIDE>
__global__ void __launch_bounds__(OWN_THREADS, 2) own_part_kernel(const __grid_constant__ CUtensorMap tm_page, const __grid_constant__ CUtensorMap tm_part, const __grid_constant__ PrefixAttnArgs a) {
    using Cfg = OwnCfg<D, WIDE>;
    constexpr int STAGES = Cfg::STAGES, KS = D / 16, NT = D / 8, ROWS = Cfg::ROWS, VALS = WIDE ? 4 : 2;
    extern __shared__ __align__(1024) uint8_t smem[];
    float* scratch = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE_BYTES);             // [4 warps][values][32 lanes]
    float* ml_s = scratch + 4 * Cfg::REGS * 32;                                              // [4 warps][rows][2]
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(ml_s + 4 * ROWS * 2);
    uint64_t* empty_bar = full_bar + STAGES;
    __shared__ Prefixes px;
    __shared__ int64_t sums[OWN_THREADS / 32];
    __shared__ OwnAt start;
    __shared__ int joins[2];                                                                 // whether this CTA came last for its first and its last item

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int grp = a.n_heads / a.n_kv, tile_tokens = KEY_TILE / grp;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_page); tma_prefetch_desc(&tm_part);
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 4); }
        fence_barrier_init();
    }
    griddep_launch();
    // ---- the plan: everything read here was written before the prefixes' kernel let this one start ----
    const int per = (a.n_seqs + OWN_THREADS - 1) / OWN_THREADS, s0 = threadIdx.x * per, s1 = min(a.n_seqs, s0 + per);
    int64_t pages = 0; bool wrong = false;
    for (int s = s0; s < s1; ++s) {
        const int len = __ldcg(a.own_lens + s);
        wrong = wrong || len < 0 || len > (int64_t)a.max_own_pages * CACHE_PAGE;
        pages += own_pages((int)min((int64_t)max(len, 0), (int64_t)a.max_own_pages * CACHE_PAGE));
    }
    if (wrong) report(a);
    int64_t before = pages;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t x = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += x; }
    if (lane == 31) sums[warp] = before;
    if (warp == 4) read_prefixes(a, px, tile_tokens, lane);
    __syncthreads();
    before -= pages;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < OWN_THREADS / 32; ++w) { if (w < warp) before += sums[w]; total += sums[w]; }
    before *= a.n_kv; total *= a.n_kv;
    const int64_t busy = busy_ctas(gridDim.x, total), u_begin = first_unit(blockIdx.x, busy, total), u_end = first_unit(blockIdx.x + 1, busy, total);
    if (u_begin < u_end && u_begin >= before && u_begin < before + pages * a.n_kv) {         // one thread
        OwnAt at; at.seq = s0; at.unit0 = before;
        for (at.read(a); u_begin >= at.unit0 + (int64_t)at.pages * a.n_kv;) { at.unit0 += (int64_t)at.pages * a.n_kv; ++at.seq; at.read(a); }
        at.kvh = (int)((u_begin - at.unit0) / at.pages); at.unit0 += (int64_t)at.kvh * at.pages;
        start = at;
    }
    __syncthreads();
    if (u_begin >= u_end) { griddep_wait(); return; }

    if (warp == 4) {
        if (lane == 0) {
            int s = 0; uint32_t ph = 0;
            OwnAt at = start;
            for (int64_t u = u_begin; u < u_end; at.next(a)) {
                const int c0 = (int)(u - at.unit0), c1 = (int)min((int64_t)at.pages, u_end - at.unit0);
                u = at.unit0 + c1;
                const int32_t* bt = a.own_tables + (int64_t)at.seq * a.max_own_pages;
                int page = at.len > 0 ? __ldcg(bt + c0) : 0;
                for (int c = c0; c < c1; ++c) {
                    const int next_page = c + 1 < c1 ? __ldcg(bt + c + 1) : 0;               // looked up while this one's slot is waited for
                    if (page < 0 || page >= a.num_pages) { report(a); page = 0; }
                    const int valid = min(CACHE_PAGE, at.len - c * CACHE_PAGE);
                    mbar_wait(&empty_bar[s], ph ^ 1);
                    uint8_t* kdst = smem + s * Cfg::STAGE_BYTES;
                    uint8_t* vdst = kdst + Cfg::KV_BYTES;
                    const int krow = (page * a.n_kv + at.kvh) * CACHE_PAGE, vrow = krow + a.num_pages * a.n_kv * CACHE_PAGE;
                    if (valid > 48) {
                        mbar_expect_tx(&full_bar[s], Cfg::STAGE_BYTES);
#pragma unroll
                        for (int h = 0; h < Cfg::HALVES; ++h) {
                            tma_load_2d(kdst + h * Cfg::TILE_BYTES, &tm_page, &full_bar[s], h * 64, krow, kEvictFirst);
                            tma_load_2d(vdst + h * Cfg::TILE_BYTES, &tm_page, &full_bar[s], h * 64, vrow, kEvictFirst);
                        }
                    } else if (valid > 0) {                                                  // a page that ends early: pieces of 16 tokens
                        const int n = (valid + 15) / 16;
                        mbar_expect_tx(&full_bar[s], n * 2 * Cfg::HALVES * 16 * 128);
                        for (int i = 0; i < n; ++i)
#pragma unroll
                            for (int h = 0; h < Cfg::HALVES; ++h) {
                                tma_load_2d(kdst + h * Cfg::TILE_BYTES + i * 2048, &tm_part, &full_bar[s], h * 64, krow + i * 16, kEvictFirst);
                                tma_load_2d(vdst + h * Cfg::TILE_BYTES + i * 2048, &tm_part, &full_bar[s], h * 64, vrow + i * 16, kEvictFirst);
                            }
                    } else mbar_arrive(&full_bar[s]);
                    page = next_page;
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
        griddep_wait();
        return;
    }

    const int g = lane >> 2, t = lane & 3;
    int s = 0; uint32_t ph = 0; int n_items = 0;
    {
        OwnAt at = start;
        for (int64_t u = u_begin; u < u_end; at.next(a), ++n_items) {
            const int c0 = (int)(u - at.unit0), c1 = (int)min((int64_t)at.pages, u_end - at.unit0);
            u = at.unit0 + c1;
            uint32_t qa[KS][VALS];                                                           // rows = heads of the group, zeros beyond it
            {
                const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)at.seq * a.ldq + (int64_t)(at.kvh * grp + g) * D;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int v = 0; v < VALS; ++v) {                                         // v: columns + 8, then rows + 8
                        const int up = WIDE ? v & 1 : 0, right = WIDE ? v >> 1 : v;
                        qa[ks][v] = g + 8 * up < grp ? __ldcg(reinterpret_cast<const uint32_t*>(q + up * 8 * D + ks * 16 + right * 8 + 2 * t)) : 0u;
                    }
            }
            float oacc[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) { oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f; }
            float m_run[VALS / 2], l_run[VALS / 2];
#pragma unroll
            for (int h = 0; h < VALS / 2; ++h) { m_run[h] = -INFINITY; l_run[h] = 0.f; }
            for (int c = c0; c < c1; ++c) {
                mbar_wait(&full_bar[s], ph);
                const int valid = at.len - c * CACHE_PAGE - warp * 16;                       // tokens of this warp's quarter
                if (valid > 0) {
                    const uint32_t kbase = smem_u32(smem + s * Cfg::STAGE_BYTES), vbase = kbase + Cfg::KV_BYTES;
                    float sacc[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) { sacc[j][0] = sacc[j][1] = sacc[j][2] = sacc[j][3] = 0.f; }
                    {
                        const int r = warp * 16 + ((lane >> 4) << 3) + (lane & 7), dsel = ((lane >> 3) & 1) << 3;
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            uint32_t b0, b1, b2, b3;
                            ldmatrix_x4(kbase + own_off<D>(r, ks * 16 + dsel), b0, b1, b2, b3);
                            const uint32_t a0 = qa[ks][0], a1 = WIDE ? qa[ks][1] : 0u, a2 = qa[ks][WIDE ? 2 : 1], a3 = WIDE ? qa[ks][VALS - 1] : 0u;
                            mma_bf16_16816(sacc[0], a0, a1, a2, a3, b0, b1);
                            mma_bf16_16816(sacc[1], a0, a1, a2, a3, b2, b3);
                        }
                    }
                    uint32_t pa[4] = {0u, 0u, 0u, 0u}; float alpha[VALS / 2];
#pragma unroll
                    for (int h = 0; h < VALS / 2; ++h) {                                     // rows g, and g + 8
                        float sc[4];
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) sc[j * 2 + e] = j * 8 + 2 * t + e < valid ? sacc[j][2 * h + e] * a.scale_log2e : -INFINITY;
                        float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const float m_new = fmaxf(m_run[h], mx), ref = finite_or_zero(m_new);
                        alpha[h] = exp2f(m_run[h] - ref);
                        float pr[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) pr[e] = exp2f(sc[e] - ref);
                        l_run[h] = l_run[h] * alpha[h] + (pr[0] + pr[1] + pr[2] + pr[3]);
                        m_run[h] = m_new;
                        pa[h] = pack_bf16x2(pr[0], pr[1]); pa[2 + h] = pack_bf16x2(pr[2], pr[3]);
                    }
                    // values behind the end may be anything, and 0 x inf is not 0
                    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                    if (valid < 16) {
                        keep0 = (2 * t < valid ? 0xffffu : 0u) | (2 * t + 1 < valid ? 0xffff0000u : 0u);
                        keep1 = (2 * t + 8 < valid ? 0xffffu : 0u) | (2 * t + 9 < valid ? 0xffff0000u : 0u);
                    }
                    {
                        const int r = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), dsel = (lane >> 4) << 3;
#pragma unroll
                        for (int j = 0; j < NT; j += 2) {
                            uint32_t b0, b1, b2, b3;
                            ldmatrix_x4_trans(vbase + own_off<D>(r, j * 8 + dsel), b0, b1, b2, b3);
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int e = 0; e < VALS; ++e) oacc[j + i][e] *= alpha[e >> 1];
                            mma_bf16_16816(oacc[j], pa[0], pa[1], pa[2], pa[3], b0 & keep0, b1 & keep1);
                            mma_bf16_16816(oacc[j + 1], pa[0], pa[1], pa[2], pa[3], b2 & keep0, b3 & keep1);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[s]);
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            // ---- the four warps' states meet: each warp adds up a quarter of the columns ----
#pragma unroll
            for (int h = 0; h < VALS / 2; ++h) {
                l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
                l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
                if (t == 0) { ml_s[(warp * ROWS + g + 8 * h) * 2] = m_run[h]; ml_s[(warp * ROWS + g + 8 * h) * 2 + 1] = l_run[h]; }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < VALS; ++e) scratch[(warp * Cfg::REGS + j * VALS + e) * 32 + lane] = oacc[j][e];
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const int64_t slot = (int64_t)blockIdx.x + (int64_t)at.seq * a.n_kv + at.kvh;
#pragma unroll
            for (int h = 0; h < VALS / 2; ++h) {
                const int row = g + 8 * h;
                float f[4], m = -INFINITY, l = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) { f[w] = ml_s[(w * ROWS + row) * 2]; m = fmaxf(m, f[w]); }
                const float ref = finite_or_zero(m);
#pragma unroll
                for (int w = 0; w < 4; ++w) { f[w] = exp2f(f[w] - ref); l += f[w] * ml_s[(w * ROWS + row) * 2 + 1]; }
                if (row >= grp) continue;
                float* po = a.own_o + slot * (grp * D) + row * 4;                            // [D / 4][heads][4]
#pragma unroll
                for (int j = 0; j < NT / 4; ++j) {
                    const int jj = warp * (NT / 4) + j, col = jj * 8 + 2 * t;
                    float o[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        o[e] = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; ++w) o[e] += f[w] * scratch[(w * Cfg::REGS + jj * VALS + 2 * h + e) * 32 + lane];
                    }
                    *reinterpret_cast<float2*>(po + (col >> 2) * (grp * 4) + (col & 3)) = make_float2(o[0], o[1]);
                }
                if (warp == 0 && t == 0) *reinterpret_cast<float2*>(a.own_ml + (slot * grp + row) * 2) = make_float2(m, l);
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");                                   // scratch is free for the next item
        }
    }

    // ---- the join.  Items that lie in this CTA alone are its own; of one cut between CTAs (at most the first and the last here) the CTA that comes last joins all parts ----
    griddep_wait();                                                                          // the prefixes' parts are there, and the counters are zero
    fence_acq_rel_gpu();
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (threadIdx.x == 0) {
        OwnAt at = start;
        for (int k = 0; k < n_items; ++k, at.next(a)) {
            if (k > 0 && k + 1 < n_items) continue;
            const int c0 = cta_of(at.unit0, busy, total), c1 = cta_of(at.unit0 + at.pages - 1, busy, total);
            bool last = true;
            if (c0 != c1) {
                last = atomicAdd(a.counters + c0, 1) == c1 - c0;
                if (last) fence_acq_rel_gpu();
            }
            joins[k > 0] = last;
        }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    OwnAt at = start;
    for (int k = 0; k < n_items; ++k, at.next(a)) {
        if ((k & 3) != warp || (k == 0 && !joins[0]) || (k > 0 && k + 1 == n_items && !joins[1])) continue;
        const int c0 = cta_of(at.unit0, busy, total), c1 = cta_of(at.unit0 + at.pages - 1, busy, total);
        if (grp > 4) join_item<D, 8>(a, px, at, c0, c1, grp, tile_tokens, lane);
        else if (grp > 2) join_item<D, 4>(a, px, at, c0, c1, grp, tile_tokens, lane);
        else join_item<D, 2>(a, px, at, c0, c1, grp, tile_tokens, lane);
    }
}

// =============================================================================================
// host
// =============================================================================================
PrefixAttnPlan prefix_attn_plan(int n_seqs, int n_heads, int n_kv, int head_dim, int n_prefixes, int max_prefix_pages, int max_own_pages, int sms) {
    PrefixAttnPlan p{};
    const int grp = n_heads / n_kv, tile_tokens = KEY_TILE / grp;
    const int64_t items = n_prefixes > 0 ? ((int64_t)n_seqs / tile_tokens + n_prefixes) * n_kv : 0;                // no more row tiles than that, however rows fall on prefixes
    const int64_t units = items * ((max_prefix_pages + 1) / 2), own_units = (int64_t)n_seqs * n_kv * max_own_pages;
    p.pre_ctas = (int)(units < 1 ? 1 : units < sms ? units : sms);
    p.own_ctas = (int)(own_units < 2 * sms ? own_units : 2 * sms);
    p.pre_slots = (size_t)(items + p.pre_ctas); p.own_slots = (size_t)((int64_t)n_seqs * n_kv + p.own_ctas);
    auto take = [&](size_t bytes) { const size_t at = p.bytes; p.bytes += (bytes + 255) & ~size_t(255); return at; };
    p.pre_o = take(p.pre_slots * KEY_TILE * head_dim * 4); p.pre_ml = take(p.pre_slots * KEY_TILE * 8);
    p.own_o = take(p.own_slots * grp * head_dim * 4); p.own_ml = take(p.own_slots * grp * 8);
    p.counters = take((size_t)p.own_ctas * 4);
    return p;
}

template <int D, bool WIDE>
static cudaError_t launch_own(const CUtensorMap* tm_page, const CUtensorMap* tm_part, const PrefixAttnArgs& a, cudaStream_t s) {
    auto kern = own_part_kernel<D, WIDE>;
    static bool attr_done[16] = {};
    { const cudaError_t e = ensure_dynamic_smem(kern, OwnCfg<D, WIDE>::SMEM_BYTES, attr_done); if (e != cudaSuccess) return e; }
    return launch_k(kern, dim3(a.own_ctas), dim3(OWN_THREADS), OwnCfg<D, WIDE>::SMEM_BYTES, s, *tm_page, *tm_part, a);
}
template <int D>
static cudaError_t launch_both(const CUtensorMap* tm_page, const CUtensorMap* tm_part, const PrefixAttnArgs& a, cudaStream_t s) {
    auto kern = prefix_part_kernel<D>;
    static bool attr_done[16] = {};
    { const cudaError_t e = ensure_dynamic_smem(kern, PreCfg<D>::SMEM_BYTES, attr_done); if (e != cudaSuccess) return e; }
    const cudaError_t e = launch_k(kern, dim3(a.pre_ctas), dim3(PRE_THREADS), PreCfg<D>::SMEM_BYTES, s, *tm_page, a);
    if (e != cudaSuccess) return e;
    return a.n_heads / a.n_kv > 8 ? launch_own<D, true>(tm_page, tm_part, a, s) : launch_own<D, false>(tm_page, tm_part, a, s);
}
cudaError_t launch_prefix_attention(const CUtensorMap* tm_page, const CUtensorMap* tm_part, int head_dim, const PrefixAttnArgs& a, cudaStream_t s) {
    if (head_dim == 128) return launch_both<128>(tm_page, tm_part, a, s);
    if (head_dim == 64) return launch_both<64>(tm_page, tm_part, a, s);
    return cudaErrorInvalidValue;
}

}  // namespace oa
