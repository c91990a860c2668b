// attention_tree.cu — attention of several new tokens of each sequence (one, a chain, a tree of drafts) over a paged cache of bf16 or 8 bits: tiles of up to 16 rows, the join of parts, and which kernel
// a call takes.  The mathematics and the plan are attention_tree.cuh's.
//
// Few rows leave the keys' stream as the bound: pages come through shared memory by TMA and are multiplied on the warp path of 16 x 8 x 16 products, tokens and channels as the 16 rows and the item's
// rows as the 8 columns, so that nothing of a product is empty for 8 rows.  Over bf16 the weights are rounded to bf16 for the second product (2^-9 of a weight, of either sign).  A cache of 8 bits is
// multiplied in fp16, which holds e4m3 and int8 exactly, converted in registers: a row of q is scaled by a power of two that brings its largest magnitude to [2^14, 2^15), where 8 bits of a channel
// stay down to 2^-31 of that; a key's scale multiplies its scores, a value's scale its weights, over a power of two that no scale so far passes and times 2^7 (a weight is 2^8 at most): 8 bits of a
// weight stay down to 2^-24 of the reference, 2^-32 of what it may be passed by.
//
// 128 sequences of one token, 4 heads a group of 128, 600 to 2500 cached tokens: over e4m3 81 us in a graph for 408 MB (62 at the copy rate; 67 with the loads alone, without a product).  With either
// half of the channels on another warp, as over bf16, every score, weight and conversion was made twice: 111.  16 sequences of 4000 tokens: 47 us over bf16 (40 at the copy rate), 33 over 8 bits (21).
// Six chains of 4 over int8, heads of 64: 14 us, 12 without a product: the plan 2, tables, pages, the states, the join 4.
#include "attention_tree.cuh"

namespace oa {

constexpr int TREE_CONSUMERS = 256, TREE_THREADS = TREE_CONSUMERS + 96;          // eight consumer warps; a producer, a warp that brings an item's states together, one that lays its queries out

OA_DEVINL uint32_t transpose_8x8(uint32_t v) { uint32_t r; asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v)); return r; }      // 16-bit values, a row in four lanes
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
    static constexpr int CTAS = FMT != CACHE_BF16 && NB == 1 ? 2 : 1;            // of an SM: two leave 80 registers, of which up to 44 bytes spill, and take 81 us for the decoding step above; one with ten pages in its ring took 93
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

    if (warp == 8) {
        int st = 0; uint32_t ph = 0;
        for (int64_t u = u_begin;; at.next(a)) {
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
            if (u >= u_end) break;
        }
        griddep_launch();
        return;
    }
    if (warp == 10) {
        // queries of an item, and what its rows see.  8 bits: fp16 under a power of two, pieces of eight channels where the consumers' lanes find them side by side
        uint32_t k = 0;
        for (int64_t u = u_begin;; at.next(a), ++k) {
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
            if (u >= u_end) break;
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
// Rows of a sequence (its new tokens' heads of a group) on average that take tiles of 128.  us in a graph, few / many rows' kernel, 8 key/value heads of 128: 16 sequences of 4000 tokens, 16 rows bf16 50 / 55,
// e4m3 43 / 54; 20 rows (two tiles of few) 86 / 55, 71 / 54; 64 sequences of 500, 16 rows 35 / 38, 39 / 53; 20 rows 54 / 38, 53 / 53; two sequences of 3000, 16 rows 17.5 / 16.6, 18.9 / 19.5; 20 rows
// 18.3 / 16.6, 19.1 / 19.6
constexpr int TREE_FEW_ROWS = 16;
// Tiles of 8 rows where a sequence has no more on average and a group's heads fit: 8 rows as above 47 against 49 with tiles of 16 over bf16, 33 against 40 over e4m3, 27 against 33 for 64 sequences of 500
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
static cudaError_t launch_parts(const CUtensorMap* tm_q, const CUtensorMap* tm_page, const TreeAttnArgs& a, cudaStream_t s) {
    constexpr int MORE = D == 64 ? 2 : 1;
    const cudaError_t e = a.rows == 128 ? launch_tree_many(tm_q, tm_page, D, FMT, a, s)
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
