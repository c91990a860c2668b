// capi_cache.cpp — C entry points of the operators on a caller's paged cache: rotary positions, page bookkeeping and copies, decode attention over shared
// prefixes, caches of 8 bits, attention of several new tokens of a sequence.  Every argument that the host can judge is judged before anything is enqueued; what lies on the device the kernels check against the bounds they are given.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "../../include/opsagent_b200.h"
#include "cache_ops.hpp"
#include "cache_pages.hpp"
#include "call_scratch.hpp"
#include "kernels.hpp"

using namespace oa;

static_assert(sizeof(oa_page_move) == sizeof(PageMove) && TABLE_PAGE == CACHE_PAGE, "one layout of moves, one page size");

namespace {
int bad(const char* why) { return call_failed(OA_ERR_BAD_REQUEST, why); }
int device_rc(cudaError_t e) {
    if (e == cudaSuccess) return OA_OK;
    cudaGetLastError();                          // told by the code: it does not stay behind for whoever asks next
    return call_failed(OA_ERR_INTERNAL, cudaGetErrorString(e));
}
int page_rc(const PageResult& r) { return r.rc == OA_OK ? OA_OK : call_failed(r.rc, r.why); }
#define OA_ON_DEVICE_OF(...)                                                                                 \
    CallDevice on_device({__VA_ARGS__});                                                                     \
    if (on_device.foreign()) return bad("a pointer is not memory of the device that holds the others");      \
    if (on_device.error() != cudaSuccess) return device_rc(on_device.error())

// what the two rotary entries share; cols: elements of a row that are read and written
const char* rotary_wrong(int64_t T, int64_t heads, int32_t head_dim, int32_t rot_dims, int32_t layout, const double* freqs, float amplitude, int64_t ldx, int64_t ldo) {
    if (T < 0 || heads < 1 || heads > (1 << 16)) return "rotary: bad number of rows or heads";
    if (head_dim < 2 || head_dim % 2 || head_dim > (1 << 16)) return "rotary: head_dim is even and at least 2";
    if (rot_dims < 0 || rot_dims % 2 || rot_dims > head_dim || rot_dims > 2 * ROTARY_MAX_PAIRS) return "rotary: rot_dims is even, at most head_dim and at most 256";
    if (layout != 0 && layout != 1) return "rotary: layout is 0 (neighbouring channels) or 1 (halves)";
    if (rot_dims > 0 && !freqs) return "rotary: no frequencies";
    for (int i = 0; i < rot_dims / 2; ++i) if (!std::isfinite(freqs[i])) return "rotary: a frequency is not finite";
    if (!std::isfinite(amplitude)) return "rotary: the amplitude is not finite";
    if (ldx < heads * head_dim || ldo < heads * head_dim) return "rotary: a row is longer than its pitch";
    return nullptr;
}
// T rows whose last one no device's memory holds beside the first: 2^39 elements, below which products of rows, pitches and element sizes stay in 64 bits and a tensor map takes the pitch
bool beyond_memory(int64_t T, int64_t ld) { return T > 1 && ld >= ((int64_t)1 << 39) / (T - 1); }
// a cache of 2^40 bytes or more: below, offsets of its blocks stay in 64 bits and CTAs of a launch in 31
bool cache_beyond_memory(int64_t planes, int64_t num_pages, int64_t page_bytes) { return planes >= ((int64_t)1 << 40) / page_bytes / num_pages; }
// rows of T x wa and T x wb elements share no memory: they are other memory, or other columns of the same rows
bool apart(const void* x, int64_t ldx, int64_t wa, const void* y, int64_t ldy, int64_t wb, int64_t T, int64_t esz) {
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
    if (a + ((T - 1) * ldx + wa) * esz <= b || b + ((T - 1) * ldy + wb) * esz <= a) return true;
    if (ldx != ldy || T == 1) return false;                  // a single row has no pitch
    const int64_t pitch = ldx * esz, off = b >= a ? (int64_t)((b - a) % (uintptr_t)pitch) : (pitch - (int64_t)((a - b) % (uintptr_t)pitch)) % pitch;
    return off >= wa * esz && off + wb * esz <= pitch;
}
bool apart_or_same(const void* x, int64_t ldx, const void* out, int64_t ldo, int64_t T, int64_t cols, int64_t esz) {
    return (x == out && (ldx == ldo || T == 1)) || apart(x, ldx, cols, out, ldo, cols, T, esz);
}
// rows of bf16 have nothing of a layer's two planes
bool outside_cache(const void* cache, int64_t num_pages, int64_t n_kv, int64_t head_dim, const void* x, int64_t ldx, int64_t cols, int64_t T) {
    const uintptr_t c = (uintptr_t)cache, p = (uintptr_t)x;
    return p + ((T - 1) * ldx + cols) * 2 <= c || c + 2 * num_pages * n_kv * CACHE_PAGE * head_dim * 2 <= p;
}
// whether n bytes at x lie in m bytes at y or the other way round (none of a null pointer's)
bool meet(const void* x, uintptr_t n, const void* y, uintptr_t m) { return x && y && (uintptr_t)x < (uintptr_t)y + m && (uintptr_t)y < (uintptr_t)x + n; }
// a list of moves that one launch can carry out in any order (may throw)
const char* moves_wrong(int32_t num_pages, const oa_page_move* moves, int32_t n_moves) {
    if (n_moves < 0 || (n_moves > 0 && !moves)) return "cache copy: no moves";
    std::vector<unsigned char> role((size_t)num_pages, 0);              // 1: a source, 2: a target
    for (int i = 0; i < n_moves; ++i) {
        const oa_page_move& m = moves[i];
        if (m.src < 0 || m.src >= num_pages || m.dst < 0 || m.dst >= num_pages || m.tokens < 0 || m.tokens > CACHE_PAGE) return "cache copy: a move is outside the cache or its pages";
        if (role[m.dst]) return "cache copy: a page is the target of two moves, or a target and a source";
        role[m.dst] = 2;
        if (role[m.src] == 2) return "cache copy: a page is the target of two moves, or a target and a source";
        role[m.src] = 1;
    }
    return nullptr;
}
// what the entries on a cache of 8 bits share
const char* cache8_wrong(int32_t num_pages, int32_t n_kv, int32_t head_dim) {
    if (head_dim < 16 || head_dim % 16 || head_dim > 256) return "8-bit cache: head_dim is a multiple of 16, up to 256";
    if (n_kv < 1 || n_kv > 4096 || num_pages < 1) return "8-bit cache: a page or more, of 1 to 4096 heads";
    return nullptr;
}
const char* rows8_wrong(const void* k, const void* v, int64_t ldkv, const void* cache, int32_t num_pages, const int32_t* slots, int32_t T, int32_t n_kv, int32_t head_dim, int32_t format, const int32_t* status) {
    if (const char* wrong = cache8_wrong(num_pages, n_kv, head_dim)) return wrong;
    if (format != CACHE_E4M3 && format != CACHE_INT8) return "8-bit cache: format is 1 (e4m3) or 2 (int8)";
    const int64_t cols = (int64_t)n_kv * head_dim;
    if (T < 0 || ldkv < cols) return "8-bit cache: bad number of rows, or a row is longer than its pitch";
    if (T == 0) return nullptr;
    if (!k || !v || !cache || !slots) return "8-bit cache: null pointer";
    if (((uintptr_t)k | (uintptr_t)v) % 2 || (uintptr_t)cache % 16 || ((uintptr_t)slots | (uintptr_t)status) % 4) return "8-bit cache: a pointer is not aligned (the cache to 16 bytes)";
    if (beyond_memory(T, ldkv)) return "8-bit cache: rows further apart than memory reaches";
    const uintptr_t bytes = 2ull * num_pages * n_kv * CACHE_PAGE * (head_dim + 4), row_bytes = ((T - 1) * ldkv + cols) * 2;
    for (const void* p : {k, v}) {
        if (meet(p, row_bytes, cache, bytes)) return "8-bit cache: rows overlap the cache";
        if (meet(p, row_bytes, slots, 4ull * T) || meet(p, row_bytes, status, 4)) return "8-bit cache: rows overlap slots or status";
    }
    if (meet(cache, bytes, slots, 4ull * T) || meet(cache, bytes, status, 4) || meet(slots, 4ull * T, status, 4)) return "8-bit cache: the cache, slots and status overlap";
    return nullptr;
}
void rotary_turns(RotaryArgs& a, const double* freqs, int32_t rot_dims, float amplitude, bool transpose) {
    a.pairs = rot_dims / 2; a.amplitude = amplitude;
    for (int i = 0; i < a.pairs; ++i) a.turns[i] = (transpose ? -freqs[i] : freqs[i]) / 6.283185307179586476925;
}
}  // namespace

extern "C" {

int oa_host_rotary_freqs(int32_t rot_dims, double base, int32_t scaling, double factor, double first, double second, int32_t original, double* freqs_out, float* amplitude_out) {
    if (rot_dims < 0 || rot_dims % 2 || rot_dims > 2 * ROTARY_MAX_PAIRS || (rot_dims > 0 && !freqs_out) || !amplitude_out) return bad("rotary: rot_dims is even and at most 256, with room for its frequencies");
    if (!(base > 0) || !std::isfinite(base)) return bad("rotary: the base is positive");
    if (scaling < 0 || scaling > 3) return bad("rotary: scaling is 0, 1 (linear), 2 (llama3) or 3 (YaRN)");
    if (scaling > 0 && (!(factor > 0) || !std::isfinite(factor))) return bad("rotary: the factor is positive");
    if (scaling >= 2 && (original < 1 || !(first > 0) || !(second > 0) || !std::isfinite(first) || !std::isfinite(second))) return bad("rotary: scaling needs a length and two numbers of turns");
    if (scaling == 2 && !(second > first)) return bad("rotary: the high frequency factor is above the low one");
    if (scaling == 3 && (base == 1.0 || !(factor >= 1))) return bad("rotary: YaRN takes a factor of at least 1, and another base than 1");
    const double two_pi = 6.283185307179586476925;
    double lo = 0.0, hi = 0.0;
    if (scaling == 3) {
        auto where = [&](double turns) { return rot_dims * std::log(original / (two_pi * turns)) / (2.0 * std::log(base)); };
        lo = std::max(std::floor(where(first)), 0.0); hi = std::min(std::ceil(where(second)), (double)(rot_dims - 1));
    }
    for (int i = 0; i < rot_dims / 2; ++i) {
        double f = std::pow(base, -2.0 * i / (double)rot_dims);
        if (scaling == 1) f /= factor;
        else if (scaling == 2) { const double share = std::min(1.0, std::max(0.0, (original * f / two_pi - first) / (second - first))); f = f * share + f / factor * (1.0 - share); }
        else if (scaling == 3) { const double ramp = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001))); f = f / factor * ramp + f * (1.0 - ramp); }
        freqs_out[i] = f;
    }
    *amplitude_out = scaling == 3 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return OA_OK;
}

int oa_k_rotary(const void* x, int64_t ldx, void* out, int64_t ldo, const int32_t* positions, int32_t T, int32_t n_heads, int32_t head_dim, int32_t rot_dims, int32_t layout,
                const double* freqs, float amplitude, int32_t transpose, int32_t f32, void* stream) {
    const char* wrong = rotary_wrong(T, n_heads, head_dim, rot_dims, layout, freqs, amplitude, ldx, ldo);
    if (wrong) return bad(wrong);
    if (T == 0) return OA_OK;
    if (beyond_memory(T, ldx) || beyond_memory(T, ldo)) return bad("rotary: rows further apart than memory reaches");
    const int64_t esz = f32 ? 4 : 2;
    if (!x || !out || !positions) return bad("rotary: null pointer");
    if (((uintptr_t)x | (uintptr_t)out) % esz || (uintptr_t)positions % 4) return bad("rotary: a pointer is not aligned to its elements");
    if (!apart_or_same(x, ldx, out, ldo, T, (int64_t)n_heads * head_dim, esz)) return bad("rotary: out overlaps x without being x");
    OA_ON_DEVICE_OF(x, out, positions);
    RotaryArgs a{};
    a.x = x; a.ldx = ldx; a.out = out; a.ldo = ldo; a.positions = positions; a.T = T; a.n_heads = n_heads; a.head_dim = head_dim;
    rotary_turns(a, freqs, rot_dims, amplitude, transpose != 0);
    return device_rc(launch_rotary(a, layout, f32 != 0, (cudaStream_t)stream));
}

int oa_k_rotary_cache(const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv, void* q_out, int64_t ldqo, void* kv_cache, int32_t num_pages, const int32_t* positions,
                      const int32_t* slots, int32_t T, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t rot_dims, int32_t layout, const double* freqs, float amplitude,
                      int32_t* status, void* stream) {
    const char* wrong = rotary_wrong(T, n_heads, head_dim, rot_dims, layout, freqs, amplitude, ldq, ldqo);
    if (wrong) return bad(wrong);
    if (n_kv < 1 || n_kv > (1 << 14) || num_pages < 1 || ldkv < (int64_t)n_kv * head_dim) return bad("rotary: bad cache, or a row of keys is longer than its pitch");
    if (T == 0) return OA_OK;
    if (!q || !k || !v || !q_out || !kv_cache || !positions || !slots) return bad("rotary: null pointer");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)kv_cache) % 2 || ((uintptr_t)positions | (uintptr_t)slots | (uintptr_t)status) % 4) return bad("rotary: a pointer is not aligned to its elements");
    if (beyond_memory(T, ldq) || beyond_memory(T, ldqo) || beyond_memory(T, ldkv)) return bad("rotary: rows further apart than memory reaches");
    const int64_t cols = (int64_t)n_heads * head_dim, kv_cols = (int64_t)n_kv * head_dim;
    if (!apart_or_same(q, ldq, q_out, ldqo, T, cols, 2)) return bad("rotary: q_out overlaps q without being q");
    if (!apart(k, ldkv, kv_cols, q_out, ldqo, cols, T, 2) || !apart(v, ldkv, kv_cols, q_out, ldqo, cols, T, 2)) return bad("rotary: q_out overlaps the keys or values");
    auto out_of_cache = [&](const void* x, int64_t ld, int64_t w) { return outside_cache(kv_cache, num_pages, n_kv, head_dim, x, ld, w, T); };
    if (!out_of_cache(q, ldq, cols) || !out_of_cache(q_out, ldqo, cols) || !out_of_cache(k, ldkv, kv_cols) || !out_of_cache(v, ldkv, kv_cols)) return bad("rotary: rows overlap the cache");
    OA_ON_DEVICE_OF(q, k, v, q_out, kv_cache, positions, slots, status);
    RotaryArgs a{};
    a.x = q; a.ldx = ldq; a.out = q_out; a.ldo = ldqo; a.positions = positions; a.T = T; a.n_heads = n_heads; a.head_dim = head_dim;
    a.k = k; a.v = v; a.ldkv = ldkv; a.cache = kv_cache; a.slots = slots; a.n_kv = n_kv; a.num_pages = num_pages; a.status = status;
    rotary_turns(a, freqs, rot_dims, amplitude, false);
    return device_rc(launch_rotary(a, layout, false, (cudaStream_t)stream));
}

int oa_host_cache_grow(const oa_page_table* t, int32_t row, int32_t n_tokens) {
    try { return page_rc(table_grow(t, row, n_tokens)); } catch (const std::exception&) { return OA_ERR_INTERNAL; }
}
int oa_host_cache_free(const oa_page_table* t, const int32_t* rows, int32_t n) {
    try { return page_rc(table_free(t, rows, n)); } catch (const std::exception&) { return OA_ERR_INTERNAL; }
}
int oa_host_cache_fork(const oa_page_table* t, int32_t parent, const int32_t* children, int32_t n, oa_page_move* moves_out, int32_t cap, int32_t* n_moves_out) {
    try { return page_rc(table_fork(t, parent, children, n, moves_out, cap, n_moves_out)); } catch (const std::exception&) { return OA_ERR_INTERNAL; }
}
int oa_host_cache_compact(const oa_page_table* t, oa_page_move* moves_out, int32_t cap, int32_t* n_moves_out) {
    try { return page_rc(table_compact(t, moves_out, cap, n_moves_out)); } catch (const std::exception&) { return OA_ERR_INTERNAL; }
}

int oa_k_cache_copy(void* kv_cache, int32_t planes, int32_t num_pages, int32_t n_kv, int32_t head_dim, int32_t elem_bytes, const oa_page_move* moves, int32_t n_moves, void* stream) {
    if (planes < 1 || num_pages < 1 || n_kv < 1 || head_dim < 1 || (elem_bytes != 2 && elem_bytes != 4)) return bad("cache copy: bad cache");
    const int64_t row = (int64_t)head_dim * elem_bytes;
    if (row % 16 || row > 4096 || n_kv > 4096) return bad("cache copy: a row is a multiple of 16 bytes, up to 4096, with up to 4096 heads");
    if (cache_beyond_memory(planes, num_pages, row * n_kv * CACHE_PAGE)) return bad("cache copy: a cache larger than memory reaches");
    try {
        if (const char* wrong = moves_wrong(num_pages, moves, n_moves)) return bad(wrong);
        if (n_moves == 0) return OA_OK;
        if (!kv_cache || (uintptr_t)kv_cache % 16) return bad("cache copy: the cache starts on a 16-byte boundary");
        OA_ON_DEVICE_OF(kv_cache);
        return device_rc(launch_cache_copy(kv_cache, planes, num_pages, n_kv, (int)row, reinterpret_cast<const PageMove*>(moves), n_moves, (cudaStream_t)stream));
    } catch (const std::exception&) { return OA_ERR_INTERNAL; }
}

int oa_k_prefix_attention(const void* q, int64_t ldq, void* out, int64_t ldo, const void* kv_cache, int32_t num_pages, const int32_t* prefix_tables, int32_t max_prefix_pages,
                          const int32_t* prefix_lens, const int32_t* prefix_rows, int32_t n_prefixes, const int32_t* own_tables, int32_t max_own_pages, const int32_t* own_lens, int32_t n_seqs,
                          int32_t n_heads, int32_t n_kv, int32_t head_dim, float scale, int32_t* status, void* stream) {
    if (head_dim != 64 && head_dim != 128) return bad("prefix attention: heads of 64 or 128");
    if (n_kv < 1 || n_kv > 1024 || n_heads < 1 || n_heads % n_kv || n_heads / n_kv > PREFIX_MAX_GROUP) return bad("prefix attention: up to 16 query heads of a key/value head");
    if (n_seqs < 0 || n_seqs > (1 << 20) || max_own_pages < 1 || max_own_pages > (1 << 24)) return bad("prefix attention: bad number of sequences or of their pages");
    if (n_prefixes < 0 || n_prefixes > PREFIX_MAX || (n_prefixes > 0 && (max_prefix_pages < 1 || max_prefix_pages > (1 << 24)))) return bad("prefix attention: up to 32 prefixes, each with a page or more of room");
    if (num_pages < 1 || (int64_t)num_pages * n_kv * 2 * CACHE_PAGE > INT32_MAX) return bad("prefix attention: the cache's rows are counted in 31 bits");
    const float scale_log2e = (scale > 0 ? scale : 1.0f / std::sqrt((float)head_dim)) * 1.4426950408889634f;
    if (!std::isfinite(scale_log2e) || !(scale >= 0)) return bad("prefix attention: the scale is positive, and finite times log2(e), or 0 for 1 / sqrt(head_dim)");
    const int64_t width = (int64_t)n_heads * head_dim;
    if (ldq < width || ldo < width || ldq % 8 || ldo % 8) return bad("prefix attention: pitches hold a row and are multiples of 16 bytes");
    if (n_seqs == 0) return OA_OK;
    if (!q || !out || !kv_cache || !own_tables || !own_lens || (n_prefixes > 0 && (!prefix_tables || !prefix_lens || !prefix_rows))) return bad("prefix attention: null pointer");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kv_cache) % 16 || ((uintptr_t)own_tables | (uintptr_t)own_lens | (uintptr_t)status) % 4 ||
        (n_prefixes > 0 && ((uintptr_t)prefix_tables | (uintptr_t)prefix_lens | (uintptr_t)prefix_rows) % 4)) return bad("prefix attention: a pointer is not aligned");
    if (beyond_memory(n_seqs, ldq) || beyond_memory(n_seqs, ldo)) return bad("prefix attention: rows further apart than memory reaches");
    if (n_seqs == 1) ldq = ldo = width;                      // a single row has no pitch, and a tensor map takes none of 2^40 bytes
    if (!apart_or_same(q, ldq, out, ldo, n_seqs, width, 2)) return bad("prefix attention: out overlaps q without being q");
    if (!outside_cache(kv_cache, num_pages, n_kv, head_dim, out, ldo, width, n_seqs)) return bad("prefix attention: out overlaps the cache");
    if (n_prefixes == 0) { prefix_tables = prefix_lens = prefix_rows = nullptr; max_prefix_pages = 0; }
    OA_ON_DEVICE_OF(kv_cache, q, out, prefix_tables, prefix_lens, prefix_rows, own_tables, own_lens, status);
    CUtensorMap tm_q, tm_page;
    const int group = n_heads / n_kv;
    if (make_tmap_bf16_heads(&tm_q, q, (uint64_t)n_seqs, (uint64_t)n_heads, (uint64_t)head_dim, (uint64_t)ldq, 128 / group, group) != 0) return call_failed(OA_ERR_INTERNAL, "prefix attention: no tensor map of the queries");
    const uint64_t rows = 2ull * num_pages * n_kv * CACHE_PAGE;
    if (make_tmap_bf16_2d(&tm_page, kv_cache, rows, head_dim, head_dim, 64, 64) != 0) return call_failed(OA_ERR_INTERNAL, "prefix attention: no tensor map of the cache");
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return device_rc(e);
    const PrefixAttnPlan plan = prefix_attn_plan(n_seqs, n_heads, n_kv, head_dim, n_prefixes, max_prefix_pages, max_own_pages, sms);
    DevBuf scratch(plan.bytes, (cudaStream_t)stream);
    if (!scratch.p) return call_failed(OA_ERR_INTERNAL, "prefix attention: no scratch memory");
    char* base = (char*)scratch.p;
    PrefixAttnArgs a{};
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo; a.prefix_tables = prefix_tables; a.prefix_lens = prefix_lens; a.prefix_rows = prefix_rows; a.n_prefixes = n_prefixes;
    a.max_prefix_pages = max_prefix_pages; a.own_tables = own_tables; a.own_lens = own_lens; a.max_own_pages = max_own_pages;
    a.n_seqs = n_seqs; a.n_heads = n_heads; a.n_kv = n_kv; a.num_pages = num_pages; a.status = status;
    a.scale_log2e = scale_log2e;
    a.pre_o = (float*)(base + plan.pre_o); a.pre_ml = (float*)(base + plan.pre_ml); a.own_o = (float*)(base + plan.own_o); a.own_ml = (float*)(base + plan.own_ml);
    a.more_o = (float*)(base + plan.more_o); a.more_ml = (float*)(base + plan.more_ml); a.own_parts = (int2*)(base + plan.own_parts); a.pre_ctas = plan.pre_ctas; a.own_ctas = plan.own_ctas; a.key_tile = plan.key_tile; a.sms = sms;
    return device_rc(launch_prefix_attention(&tm_q, &tm_page, head_dim, plan.long_prefix, a, (cudaStream_t)stream));
}

int oa_k_cache8_write(const void* k, const void* v, int64_t ldkv, void* kv_cache, int32_t num_pages, const int32_t* slots, int32_t T, int32_t n_kv, int32_t head_dim, int32_t format,
                      int32_t* status, void* stream) {
    if (const char* wrong = rows8_wrong(k, v, ldkv, kv_cache, num_pages, slots, T, n_kv, head_dim, format, status)) return bad(wrong);
    if (T == 0) return OA_OK;
    OA_ON_DEVICE_OF(k, v, kv_cache, slots, status);
    Rows8Args a{};
    a.k = k; a.v = v; a.ldkv = ldkv; a.cache = kv_cache; a.slots = slots; a.T = T; a.n_kv = n_kv; a.head_dim = head_dim; a.num_pages = num_pages; a.status = status;
    return device_rc(launch_cache8_write(a, format == CACHE_E4M3, (cudaStream_t)stream));
}

int oa_k_cache8_read(const void* kv_cache, int32_t num_pages, const int32_t* slots, int32_t T, int32_t n_kv, int32_t head_dim, int32_t format, void* k_out, void* v_out, int64_t ldkv,
                     int32_t* status, void* stream) {
    if (const char* wrong = rows8_wrong(k_out, v_out, ldkv, kv_cache, num_pages, slots, T, n_kv, head_dim, format, status)) return bad(wrong);
    if (T == 0) return OA_OK;
    const int64_t cols = (int64_t)n_kv * head_dim;
    if (!apart(k_out, ldkv, cols, v_out, ldkv, cols, T, 2)) return bad("8-bit cache: rows of keys and of values overlap");
    OA_ON_DEVICE_OF(kv_cache, slots, k_out, v_out, status);
    Rows8Args a{};
    a.k_out = k_out; a.v_out = v_out; a.ldkv = ldkv; a.cache = const_cast<void*>(kv_cache); a.slots = slots; a.T = T; a.n_kv = n_kv; a.head_dim = head_dim; a.num_pages = num_pages; a.status = status;
    return device_rc(launch_cache8_read(a, format == CACHE_E4M3, (cudaStream_t)stream));
}

int oa_k_cache8_copy(void* kv_cache, int32_t planes, int32_t num_pages, int32_t n_kv, int32_t head_dim, const oa_page_move* moves, int32_t n_moves, void* stream) {
    if (const char* wrong = cache8_wrong(num_pages, n_kv, head_dim)) return bad(wrong);
    if (planes < 1) return bad("8-bit cache: no planes");
    if (cache_beyond_memory(planes, num_pages, (int64_t)n_kv * CACHE_PAGE * (head_dim + 4))) return bad("8-bit cache: a cache larger than memory reaches");
    try {
        if (const char* wrong = moves_wrong(num_pages, moves, n_moves)) return bad(wrong);
        if (n_moves == 0) return OA_OK;
        if (!kv_cache || (uintptr_t)kv_cache % 16) return bad("8-bit cache: the cache starts on a 16-byte boundary");
        OA_ON_DEVICE_OF(kv_cache);
        return device_rc(launch_cache8_copy(kv_cache, planes, num_pages, n_kv, head_dim, reinterpret_cast<const PageMove*>(moves), n_moves, (cudaStream_t)stream));
    } catch (const std::exception&) { return OA_ERR_INTERNAL; }
}

int oa_k_tree_attention(const void* q, int64_t ldq, void* out, int64_t ldo, const void* kv_cache, int32_t format, int32_t num_pages, const int32_t* block_tables, int32_t max_pages_per_seq,
                        const int32_t* ctx_lens, const int32_t* row_starts, const uint64_t* seen, int32_t n_seqs, int32_t n_rows, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t window,
                        int32_t sinks, float scale, int32_t* status, void* stream) {
    if (head_dim != 64 && head_dim != 128) return bad("tree attention: heads of 64 or 128");
    if (format < CACHE_BF16 || format > CACHE_INT8) return bad("tree attention: format is 0 (bf16), 1 (e4m3) or 2 (int8)");
    if (n_kv < 1 || n_kv > 1024 || n_heads < 1 || n_heads % n_kv || n_heads / n_kv > TREE_MAX_GROUP) return bad("tree attention: up to 16 query heads of a key/value head");
    if (n_seqs < 0 || n_seqs > (1 << 20) || n_rows < 0 || n_rows > (1 << 24) || max_pages_per_seq < 1 || max_pages_per_seq > (1 << 24)) return bad("tree attention: bad number of sequences, rows or pages");
    if (window != 0 && window < TREE_MAX_TOKENS) return bad("tree attention: a window is 0 (none) or at least 64");
    if (sinks < 0 || (sinks > 0 && window == 0)) return bad("tree attention: first tokens that stay visible need a window");
    const int64_t row_bytes = format == CACHE_BF16 ? 2 * head_dim : head_dim + 4, tm_rows = 2ll * num_pages * n_kv * CACHE_PAGE * row_bytes / (format == CACHE_BF16 ? 2 * head_dim : 128);
    if (num_pages < 1 || tm_rows > INT32_MAX) return bad("tree attention: the cache's rows are counted in 31 bits");
    const float scale_log2e = (scale > 0 ? scale : 1.0f / std::sqrt((float)head_dim)) * 1.4426950408889634f;
    if (!std::isfinite(scale_log2e) || !(scale >= 0)) return bad("tree attention: the scale is positive, and finite times log2(e), or 0 for 1 / sqrt(head_dim)");
    const int64_t width = (int64_t)n_heads * head_dim;
    if (ldq < width || ldo < width || ldq % 8 || ldo % 8) return bad("tree attention: pitches hold a row and are multiples of 16 bytes");
    if (n_seqs == 0 || n_rows == 0) return OA_OK;
    if (!q || !out || !kv_cache || !block_tables || !ctx_lens || !row_starts) return bad("tree attention: null pointer");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kv_cache) % 16 || ((uintptr_t)block_tables | (uintptr_t)ctx_lens | (uintptr_t)row_starts | (uintptr_t)status) % 4 || (uintptr_t)seen % 8)
        return bad("tree attention: a pointer is not aligned");
    if (beyond_memory(n_rows, ldq) || beyond_memory(n_rows, ldo)) return bad("tree attention: rows further apart than memory reaches");
    if (!apart_or_same(q, ldq, out, ldo, n_rows, width, 2)) return bad("tree attention: out overlaps q without being q");
    const uintptr_t out_bytes = ((n_rows - 1) * ldo + width) * 2, q_bytes = ((n_rows - 1) * ldq + width) * 2, cache_bytes = 2ull * num_pages * n_kv * CACHE_PAGE * row_bytes;
    const struct { const void* p; uintptr_t bytes; } arrays[] = {{block_tables, 4ull * n_seqs * max_pages_per_seq}, {ctx_lens, 4ull * n_seqs}, {row_starts, 4ull * n_seqs + 4}, {seen, 8ull * n_rows}};
    if (meet(out, out_bytes, kv_cache, cache_bytes)) return bad("tree attention: out overlaps the cache");
    if (meet(out, out_bytes, status, 4)) return bad("tree attention: out overlaps status");
    for (const auto& x : arrays) {
        if (meet(out, out_bytes, x.p, x.bytes)) return bad("tree attention: out overlaps an array that is read");
        if (meet(status, 4, x.p, x.bytes)) return bad("tree attention: status overlaps an array that is read");
    }
    if (meet(status, 4, q, q_bytes) || meet(status, 4, kv_cache, cache_bytes)) return bad("tree attention: status overlaps an array that is read");
    OA_ON_DEVICE_OF(kv_cache, q, out, block_tables, ctx_lens, row_starts, seen, status);
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return device_rc(e);
    const TreeAttnPlan plan = tree_attn_plan(n_seqs, n_rows, n_heads, n_kv, head_dim, format, max_pages_per_seq, sms);
    if (n_rows == 1) ldq = ldo = width;                      // a single row has no pitch, and a tensor map takes none of 2^40 bytes
    CUtensorMap tm_page, tm_q{};
    const int group = n_heads / n_kv;
    if ((format == CACHE_BF16 ? make_tmap_bf16_2d(&tm_page, kv_cache, (uint64_t)tm_rows, head_dim, head_dim, CACHE_PAGE, 64)
                              : make_tmap_bytes_2d(&tm_page, kv_cache, (uint64_t)tm_rows, CACHE_PAGE * head_dim / 128)) != 0) return call_failed(OA_ERR_INTERNAL, "tree attention: no tensor map of the cache");
    DevBuf scratch(plan.bytes, (cudaStream_t)stream);
    if (!scratch.p) return call_failed(OA_ERR_INTERNAL, "tree attention: no scratch memory");
    char* base = (char*)scratch.p;
    const bool bits8 = format != CACHE_BF16;
    if (plan.rows == 128 && make_tmap_bf16_heads(&tm_q, bits8 ? base + plan.q16 : q, (uint64_t)n_rows, (uint64_t)n_heads, (uint64_t)head_dim, (uint64_t)(bits8 ? width : ldq), 128 / group, group) != 0)
        return call_failed(OA_ERR_INTERNAL, "tree attention: no tensor map of the queries");
    TreeAttnArgs a{};
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo; a.cache = kv_cache; a.tables = block_tables; a.ctx_lens = ctx_lens; a.row_starts = row_starts; a.seen = seen;
    a.max_pages = max_pages_per_seq; a.n_seqs = n_seqs; a.n_rows = n_rows; a.n_heads = n_heads; a.n_kv = n_kv; a.num_pages = num_pages; a.window = window; a.sinks = sinks;
    a.scale_log2e = scale_log2e; a.status = status;
    a.part_o = (float*)(base + plan.part_o); a.part_ml = (float*)(base + plan.part_ml); a.joins = (TreeJoin*)(base + plan.joins); a.q16 = (uint32_t*)(base + plan.q16); a.q_factor = (float*)(base + plan.q_factor); a.ctas = plan.ctas; a.rows = plan.rows;
    return device_rc(launch_tree_attention(&tm_q, &tm_page, head_dim, format, a, (cudaStream_t)stream));
}

}  // extern "C"
