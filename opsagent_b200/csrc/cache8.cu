// cache8.cu — keys and values stored in 8 bits: rows quantised as they are written to a paged cache, read back, and copied with their pages.
//
// A head of a page is one block: 64 tokens' values of one byte, [64][head_dim], then their scales, fp32 [64].  A row x of a token's head has one scale,
//   s = max |x| / L,  y = rne(x / s) held to [-L, L],  L = 448 for e4m3, 127 for int8,
// and stands for y s.  The division is IEEE's, as is the rounding, so that bits are defined.  x / s passes L by a rounding at most, but for rows whose s is subnormal in fp32; a row of zeros (or whose s
// underflows) has scale 0 and zeros, a row with an infinity or a NaN keeps nothing: zeros under a scale of NaN.
//
// Bound by memory.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"
#include "work_units.hpp"

namespace oa {

constexpr int ROWS8_THREADS = 256;
constexpr int ROWS8_UNROLL = 2;          // rows in flight per thread

OA_DEVINL uint32_t to_e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | (uint32_t)hi << 16;
}
OA_DEVINL int held_int8(float x) { return min(max(__float2int_rn(x), -127), 127); }
OA_DEVINL uint32_t to_int8x4(float a, float b, float c, float d) {
    return (uint32_t)(held_int8(a) & 255) | (uint32_t)(held_int8(b) & 255) << 8 | (uint32_t)(held_int8(c) & 255) << 16 | (uint32_t)held_int8(d) << 24;
}
template <bool E4M3>
OA_DEVINL void from_8x4(uint32_t w, float (&x)[4]) {
    if (E4M3) {
        uint32_t lo, hi;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
    }
}

// A row's place: rows run over tokens, then planes, then heads
struct RowAt { int64_t block; int place; int head, plane, token; };
OA_DEVINL bool row_at(const Rows8Args& a, int64_t r, RowAt& at) {
    at.token = (int)quotient(r, 2 * a.n_kv);
    const int rem = (int)(r - (int64_t)at.token * (2 * a.n_kv));
    at.plane = rem >= a.n_kv; at.head = rem - at.plane * a.n_kv;
    const int slot = __ldcg(a.slots + at.token);
    if (slot < 0) return false;
    const int page = slot / CACHE_PAGE;
    if (page >= a.num_pages) { if (a.status) *a.status = 400; return false; }
    at.place = slot % CACHE_PAGE;
    at.block = ((int64_t)at.plane * a.num_pages + page) * a.n_kv + at.head;
    return true;
}

// LANES of eight channels each take a row; those behind its end go along
template <int LANES, bool E4M3, bool WHOLE>
__global__ void __launch_bounds__(ROWS8_THREADS) cache8_write_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int ROWS = ROWS8_THREADS / LANES;
    griddep_launch();
    const int lane = threadIdx.x % LANES, c = lane * 8;
    const bool in = c < a.head_dim;
    const int64_t rows = (int64_t)a.T * 2 * a.n_kv, block_bytes = (int64_t)CACHE_PAGE * (a.head_dim + 4);
    griddep_wait();
    for (int64_t r0 = (int64_t)blockIdx.x * (ROWS * ROWS8_UNROLL); r0 < rows; r0 += (int64_t)gridDim.x * (ROWS * ROWS8_UNROLL)) {
        RowAt at[ROWS8_UNROLL]; bool live[ROWS8_UNROLL]; uint4 raw[ROWS8_UNROLL];
#pragma unroll
        for (int j = 0; j < ROWS8_UNROLL; ++j) {
            const int64_t r = r0 + j * ROWS + threadIdx.x / LANES;
            live[j] = r < rows && row_at(a, r, at[j]);
            raw[j] = make_uint4(0u, 0u, 0u, 0u);
            if (live[j] && in) {
                const uint16_t* src = reinterpret_cast<const uint16_t*>(at[j].plane ? a.v : a.k) + (int64_t)at[j].token * a.ldkv + (int64_t)at[j].head * a.head_dim + c;
                if (WHOLE) raw[j] = ld_once_16(src);
                else {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldcg(src + 2 * i) | (uint32_t)__ldcg(src + 2 * i + 1) << 16;
                    raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < ROWS8_UNROLL; ++j) {
            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
            uint32_t top = 0;                                    // magnitudes order as their bits do, infinities and NaN above all others
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, max(w[i] << 16 & 0x7fffffffu, w[i] & 0x7fff0000u));
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (!live[j]) continue;
            const bool bad = top >= 0x7f800000u;
            const float scale = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(top), E4M3 ? 448.f : 127.f);
            const bool some = scale > 0.f;
            uint32_t y[2] = {0u, 0u};
            if (some)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x0 = __fdiv_rn(bf16lo(w[2 * i]), scale), x1 = __fdiv_rn(bf16hi(w[2 * i]), scale), x2 = __fdiv_rn(bf16lo(w[2 * i + 1]), scale), x3 = __fdiv_rn(bf16hi(w[2 * i + 1]), scale);
                    y[i] = E4M3 ? to_e4m3x4(x0, x1, x2, x3) : to_int8x4(x0, x1, x2, x3);
                }
            uint8_t* block = reinterpret_cast<uint8_t*>(a.cache) + at[j].block * block_bytes;
            if (in) *reinterpret_cast<uint2*>(block + at[j].place * a.head_dim + c) = make_uint2(y[0], y[1]);
            if (lane == 0) reinterpret_cast<float*>(block + CACHE_PAGE * a.head_dim)[at[j].place] = scale;
        }
    }
}

// sixteen channels a lane
template <int LANES, bool E4M3, bool WHOLE>
__global__ void __launch_bounds__(ROWS8_THREADS) cache8_read_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int ROWS = ROWS8_THREADS / LANES;
    griddep_launch();
    const int lane = threadIdx.x % LANES, c = lane * 16;
    const bool in = c < a.head_dim;
    const int64_t rows = (int64_t)a.T * 2 * a.n_kv, block_bytes = (int64_t)CACHE_PAGE * (a.head_dim + 4);
    griddep_wait();
    for (int64_t r0 = (int64_t)blockIdx.x * (ROWS * ROWS8_UNROLL); r0 < rows; r0 += (int64_t)gridDim.x * (ROWS * ROWS8_UNROLL)) {
        RowAt at[ROWS8_UNROLL]; bool live[ROWS8_UNROLL]; uint4 raw[ROWS8_UNROLL]; float scale[ROWS8_UNROLL];
#pragma unroll
        for (int j = 0; j < ROWS8_UNROLL; ++j) {
            const int64_t r = r0 + j * ROWS + threadIdx.x / LANES;
            live[j] = in && r < rows && row_at(a, r, at[j]);
            if (!live[j]) continue;
            const uint8_t* block = reinterpret_cast<const uint8_t*>(a.cache) + at[j].block * block_bytes;
            raw[j] = ld_once_16(block + at[j].place * a.head_dim + c);
            scale[j] = __ldcg(reinterpret_cast<const float*>(block + CACHE_PAGE * a.head_dim) + at[j].place);
        }
#pragma unroll
        for (int j = 0; j < ROWS8_UNROLL; ++j) {
            if (!live[j]) continue;
            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[4];
                from_8x4<E4M3>(w[i], x);
                o[2 * i] = pack_bf16x2(x[0] * scale[j], x[1] * scale[j]); o[2 * i + 1] = pack_bf16x2(x[2] * scale[j], x[3] * scale[j]);
            }
            uint16_t* dst = reinterpret_cast<uint16_t*>(at[j].plane ? a.v_out : a.k_out) + (int64_t)at[j].token * a.ldkv + (int64_t)at[j].head * a.head_dim + c;
            if (WHOLE) {
                reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
                reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
            } else
#pragma unroll
                for (int i = 0; i < 16; ++i) dst[i] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
        }
    }
}

template <typename K>
static cudaError_t launch_rows(K kern, int lanes, const Rows8Args& a, cudaStream_t s) {
    const int64_t each = ROWS8_THREADS / lanes * ROWS8_UNROLL, ctas = ((int64_t)a.T * 2 * a.n_kv + each - 1) / each;
    return launch_k(kern, dim3((unsigned)(ctas < 0x7fffffffll ? ctas : 0x7fffffffll)), dim3(ROWS8_THREADS), 0, s, a);
}
template <bool E4M3, bool WHOLE>
static cudaError_t launch_write(const Rows8Args& a, cudaStream_t s) {
    if (a.head_dim <= 64) return launch_rows(cache8_write_kernel<8, E4M3, WHOLE>, 8, a, s);
    if (a.head_dim <= 128) return launch_rows(cache8_write_kernel<16, E4M3, WHOLE>, 16, a, s);
    return launch_rows(cache8_write_kernel<32, E4M3, WHOLE>, 32, a, s);
}
template <bool E4M3, bool WHOLE>
static cudaError_t launch_read(const Rows8Args& a, cudaStream_t s) {
    if (a.head_dim <= 64) return launch_rows(cache8_read_kernel<4, E4M3, WHOLE>, 4, a, s);
    if (a.head_dim <= 128) return launch_rows(cache8_read_kernel<8, E4M3, WHOLE>, 8, a, s);
    return launch_rows(cache8_read_kernel<16, E4M3, WHOLE>, 16, a, s);
}
// rows of whole 16-byte pieces where every row starts on such a boundary
static bool whole_rows(const void* k, const void* v, int64_t ld) { return (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ld % 8 == 0; }
cudaError_t launch_cache8_write(const Rows8Args& a, bool e4m3, cudaStream_t s) {
    if (whole_rows(a.k, a.v, a.ldkv)) return e4m3 ? launch_write<true, true>(a, s) : launch_write<false, true>(a, s);
    return e4m3 ? launch_write<true, false>(a, s) : launch_write<false, false>(a, s);
}
cudaError_t launch_cache8_read(const Rows8Args& a, bool e4m3, cudaStream_t s) {
    if (whole_rows(a.k_out, a.v_out, a.ldkv)) return e4m3 ? launch_read<true, true>(a, s) : launch_read<false, true>(a, s);
    return e4m3 ? launch_read<true, false>(a, s) : launch_read<false, false>(a, s);
}

// ---- copies --------------------------------------------------------------------------------------
// As for caches of wider values: moves in the launch's own parameters, a CTA for a plane's blocks of a page (or a part of them).  A block's first tokens are two runs, of values and of scales.
constexpr int COPY8_THREADS = 128, COPY8_UNROLL = 8, COPY8_CHUNKS = COPY8_THREADS * COPY8_UNROLL;
template <int CAP>
struct Copy8Args { uint8_t* cache; int32_t planes, num_pages, n_kv, head_dim, parts; PageMove moves[CAP]; };

template <int CAP>
__global__ void __launch_bounds__(COPY8_THREADS) cache8_copy_kernel(const __grid_constant__ Copy8Args<CAP> a) {
    griddep_launch();
    const unsigned unit = blockIdx.x / (unsigned)a.parts, part = blockIdx.x - unit * (unsigned)a.parts;
    const unsigned move = unit / (unsigned)a.planes, plane = unit - move * (unsigned)a.planes;
    const PageMove m = a.moves[move];
    const unsigned block16 = CACHE_PAGE * (a.head_dim + 4) / 16, values = m.tokens * a.head_dim / 16, piece = values + (m.tokens + 3) / 4, chunks = a.n_kv * piece;
    const unsigned each = (chunks + a.parts - 1) / (unsigned)a.parts, first = part * each, stop = min(first + each, chunks);
    uint4* base = reinterpret_cast<uint4*>(a.cache) + (int64_t)plane * a.num_pages * a.n_kv * block16;
    const uint4* src = base + (int64_t)m.src * a.n_kv * block16;
    uint4* dst = base + (int64_t)m.dst * a.n_kv * block16;
    uint4 v[COPY8_UNROLL]; unsigned at[COPY8_UNROLL]; int words[COPY8_UNROLL];
    griddep_wait();
#pragma unroll
    for (int i = 0; i < COPY8_UNROLL; ++i) {
        const unsigned c = first + i * COPY8_THREADS + threadIdx.x;
        words[i] = 0;
        if (c >= stop) continue;
        const unsigned head = c / piece, x = c - head * piece;
        at[i] = head * block16 + (x < values ? x : CACHE_PAGE * a.head_dim / 16 + (x - values));
        words[i] = x < values ? 4 : min(4, m.tokens - 4 * (int)(x - values));
        v[i] = ld_once_16(src + at[i]);
    }
#pragma unroll
    for (int i = 0; i < COPY8_UNROLL; ++i) {
        if (words[i] == 4) __stcs(dst + at[i], v[i]);
        else if (words[i] > 0) {                                 // the last scales of a page that is not copied whole
            uint32_t* w = reinterpret_cast<uint32_t*>(dst + at[i]);
            w[0] = v[i].x;
            if (words[i] > 1) w[1] = v[i].y;
            if (words[i] > 2) w[2] = v[i].z;
        }
    }
}

template <int CAP>
static cudaError_t launch_copy8(void* cache, int planes, int num_pages, int n_kv, int head_dim, const PageMove* moves, int n, cudaStream_t s) {
    Copy8Args<CAP> a;
    a.cache = reinterpret_cast<uint8_t*>(cache); a.planes = planes; a.num_pages = num_pages; a.n_kv = n_kv; a.head_dim = head_dim;
    int most = 0;
    for (int i = 0; i < n; ++i) { a.moves[i] = moves[i]; if (moves[i].tokens > most) most = moves[i].tokens; }
    if (most == 0) return cudaSuccess;
    a.parts = (n_kv * (most * head_dim / 16 + (most + 3) / 4) + COPY8_CHUNKS - 1) / COPY8_CHUNKS;
    return launch_k(cache8_copy_kernel<CAP>, dim3((unsigned)((int64_t)n * planes * a.parts)), dim3(COPY8_THREADS), 0, s, a);
}
cudaError_t launch_cache8_copy(void* cache, int planes, int num_pages, int n_kv, int head_dim, const PageMove* moves, int n_moves, cudaStream_t s) {
    constexpr int FEW = 64, MANY = 2560;
    const int64_t ctas = (int64_t)planes * (((int64_t)n_kv * (CACHE_PAGE * (head_dim + 4) / 16) + COPY8_CHUNKS - 1) / COPY8_CHUNKS), cap = 0x7fffffffll / ctas;      // CTAs of a launch are counted in 31 bits
    if (cap < 1) return cudaErrorInvalidValue;
    const int many = cap < MANY ? (int)cap : MANY;
    for (int i = 0; i < n_moves;) {
        const int n = n_moves - i < many ? n_moves - i : many;
        const cudaError_t e = n <= FEW ? launch_copy8<FEW>(cache, planes, num_pages, n_kv, head_dim, moves + i, n, s) : launch_copy8<MANY>(cache, planes, num_pages, n_kv, head_dim, moves + i, n, s);
        if (e != cudaSuccess) return e;
        i += n;
    }
    return cudaSuccess;
}

}  // namespace oa
