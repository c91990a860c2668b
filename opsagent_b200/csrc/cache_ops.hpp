// cache_ops.hpp — launch API of the operators on a caller's paged cache: rotary positions (rotary.cu), copies of pages (cache_copy.cu), decode
// attention over shared prefixes (attention_prefix.cu), caches of 8 bits (cache8.cu) and attention of several new tokens of a sequence (attention_tree.cu).  Device pointers in, cudaError_t out; every launcher is asynchronous on the given stream.
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

// ---- caches of 8 bits -----------------------------------------------------------------------------------
// [planes][num_pages][n_kv] blocks of 64 * (head_dim + 4) bytes: values [64][head_dim], then fp32 scales [64]
enum CacheFormat { CACHE_BF16 = 0, CACHE_E4M3 = 1, CACHE_INT8 = 2 };
struct Rows8Args {
    // T rows of n_kv heads of keys and of values (bf16, pitch ldkv in elements) and a layer's two planes; token t is place slots[t] % 64 of page slots[t] / 64.  A negative slot: the
    // token is passed over; one beyond the cache: the same, *status = 400
    const void *k, *v; void *k_out, *v_out; int64_t ldkv; void* cache; const int32_t* slots; int32_t T, n_kv, head_dim, num_pages; int32_t* status;
    int32_t step_tokens, step_rows;                // of a thread's next row (the launchers')
};
cudaError_t launch_cache8_write(const Rows8Args& a, bool e4m3, cudaStream_t s);          // k, v -> cache
cudaError_t launch_cache8_read(const Rows8Args& a, bool e4m3, cudaStream_t s);           // cache -> k_out, v_out
cudaError_t launch_cache8_copy(void* cache, int planes, int num_pages, int n_kv, int head_dim, const PageMove* moves, int n_moves, cudaStream_t s);      // as launch_cache_copy

// ---- attention of several new tokens of a sequence -----------------------------------------------------------
constexpr int TREE_MAX_TOKENS = 64;               // new tokens of a sequence: the bits of a row of `seen`
constexpr int TREE_MAX_GROUP = 16;                // query heads of a key/value head
struct TreeJoin { int32_t parts, row0, rows, kvh; };      // an item that several CTAs share: later parts, its first row, its rows, its head
struct TreeAttnArgs {
    const void* q; int64_t ldq; void* out; int64_t ldo;
    const void* cache; const int32_t* tables; const int32_t* ctx_lens; const int32_t* row_starts; const uint64_t* seen;      // seen null: a chain
    int32_t max_pages, n_seqs, n_rows, n_heads, n_kv, num_pages, window, sinks;
    float scale_log2e;
    int32_t* status;
    // scratch (tree_attn_plan): each CTA's part of an item that it begins and others end, its part of one that another began, and who they belong to
    float *part_o, *part_ml; TreeJoin* joins;
    uint32_t* q16; float* q_factor;                // tiles of 128 rows over 8 bits: queries in fp16 [n_rows][n_heads][head_dim] and their scores' factors [n_rows][n_heads]
    int32_t ctas, rows;                            // rows: of a tile
};
struct TreeAttnPlan { int ctas, rows; size_t part_o, part_ml, joins, q16, q_factor, bytes; };
TreeAttnPlan tree_attn_plan(int n_seqs, int n_rows, int n_heads, int n_kv, int head_dim, int format, int max_pages, int sms);
// tm_page: box of 64 rows over the layer's cache [2 * num_pages * n_kv * 64, head_dim] of bf16, or of a block's values over the same of 8 bits, rows of 128 bytes; tm_q, looked at for tiles of 128 rows:
// box of 128 / group tokens by a group's heads over q, or over q16 where the cache has 8 bits
cudaError_t launch_tree_attention(const CUtensorMap* tm_q, const CUtensorMap* tm_page, int head_dim, int format, const TreeAttnArgs& a, cudaStream_t s);

}  // namespace oa
