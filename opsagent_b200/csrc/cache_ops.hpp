// cache_ops.hpp — launch API of the operators on a caller's paged cache: rotary positions (rotary.cu), copies of pages (cache_copy.cu) and decode
// attention over shared prefixes (attention_prefix.cu).  Device pointers in, cudaError_t out; every launcher is asynchronous on the given stream.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace oa {

constexpr int CACHE_PAGE = 64;                    // tokens of a page

// ---- rotary positions ------------------------------------------------------------------------
constexpr int ROTARY_MAX_PAIRS = 128;             // rotated channels of a head: up to 256
struct RotaryArgs {
    // rows of n_heads heads of head_dim channels, pitch in elements; the first 2 * pairs channels of a head are rotated, the others copied
    const void* x; int64_t ldx; void* out; int64_t ldo;
    const int32_t* positions;                     // [T]
    int32_t T, n_heads, head_dim, pairs;
    // with a cache: n_kv heads of new keys (rotated) and values (as they are), pitch ldkv, written to row slots[t] % 64 of page slots[t] / 64 of a layer's two
    // planes [num_pages][n_kv][64][head_dim]; a negative slot: the token is not written; one beyond the cache: not written, *status = 400
    const void* k; const void* v; int64_t ldkv; void* cache; const int32_t* slots; int32_t n_kv, num_pages;
    int32_t* status;
    float amplitude;
    double turns[ROTARY_MAX_PAIRS];               // frequency / 2 pi of each pair, negative to rotate back
};
cudaError_t launch_rotary(const RotaryArgs& a, int layout, bool f32, cudaStream_t s);       // layout 0: channel 2i with 2i + 1, 1: channel i with i + pairs

// ---- copies of pages ----------------------------------------------------------------------------
struct PageMove { int32_t src, dst, tokens; };   // the first `tokens` places of page src go to page dst (the C ABI's oa_page_move)
// cache [planes][num_pages][n_kv][64][row_bytes]; no page is the target of two moves, or target and source (checked by the caller)
cudaError_t launch_cache_copy(void* cache, int planes, int num_pages, int n_kv, int row_bytes, const PageMove* moves, int n_moves, cudaStream_t s);

// ---- decode attention over shared prefixes ----------------------------------------------------------
constexpr int PREFIX_MAX = 32;                    // prefixes of a call: a warp's lanes
constexpr int PREFIX_MAX_GROUP = 16;              // query heads of a key/value head
struct PrefixAttnArgs {
    const void* q; int64_t ldq; void* out; int64_t ldo;
    const int32_t* prefix_tables; const int32_t* prefix_lens; const int32_t* prefix_rows; int32_t n_prefixes, max_prefix_pages;
    const int32_t* own_tables; const int32_t* own_lens; int32_t max_own_pages;
    int32_t n_seqs, n_heads, n_kv, num_pages;
    float scale_log2e;
    int32_t* status;
    // scratch (prefix_attn_plan): parts of the prefixes, each item's first own part, later ones by the CTA that makes them, and how many of those an item has
    float *pre_o, *pre_ml, *own_o, *own_ml, *more_o, *more_ml; int2* own_parts;
    int32_t pre_ctas, own_ctas, key_tile, sms;     // pre_ctas 0: prefixes have no kernel of their own; key_tile: keys of its tiles
};
struct PrefixAttnPlan { int pre_ctas, own_ctas, key_tile; bool long_prefix; size_t pre_slots, pre_o, pre_ml, own_o, own_ml, more_o, more_ml, own_parts, bytes; };      // CTAs, slots, byte offsets
PrefixAttnPlan prefix_attn_plan(int n_seqs, int n_heads, int n_kv, int head_dim, int n_prefixes, int max_prefix_pages, int max_own_pages, int sms);
// tm_q: box of 128 / group tokens by a group's heads over q; tm_page: box of 64 rows over the layer's cache [2 * num_pages * n_kv * 64, head_dim]
cudaError_t launch_prefix_attention(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int head_dim, bool long_prefix, const PrefixAttnArgs& a, cudaStream_t s);

}  // namespace oa
