// cache8.cu — keys and values stored in 8 bits: rows quantised as they are written to a paged cache, read back, and copied with their pages.
//
// A head of a page is one block: 64 tokens' values of one byte, [64][head_dim], then their scales, fp32 [64].  A row x of a token's head has one scale,
//   s = max |x| / L,  y = rne(x / s) held to [-L, L],  L = 448 for e4m3, 127 for int8,
// and stands for y s.  The division is IEEE's, as is the rounding, so that bits are defined.  x / s passes L by a rounding at most, but for rows whose s is subnormal in fp32; a row of zeros (or whose s
// underflows) has scale 0 and zeros, a row with an infinity or a NaN keeps nothing: zeros under a scale of NaN.
//
// Bound by memory and close to it by issue slots: 8192 tokens of 2 x 8 heads of 128, 51 MB, are written in 11.9 us in a graph (2 of them to begin and end; 7.8 at the copy rate), 50001 tokens, 311 MB,
// read back in 52 (47).  A row's place costs a division; with one a row, lanes of 16 consecutive channels and integers converted one by one the latter took 68.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"
#include "work_units.hpp"

namespace oa {

constexpr int ROWS8_THREADS = 128;
constexpr int WRITE8_UNROLL = 2, READ8_UNROLL = 3;       // rows in flight per thread: 32 bytes of one that is written, 16 of one that is read

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
// of values that pass 127 by a rounding at most: the low byte of 1.5 2^23 + x is x to the nearest, ties to even
OA_DEVINL uint32_t near_int8x4(float a, float b, float c, float d) {
    constexpr float M = 12582912.f;
    return __byte_perm(__byte_perm(__float_as_uint(M + a), __float_as_uint(M + b), 0x0040), __byte_perm(__float_as_uint(M + c), __float_as_uint(M + d), 0x0040), 0x5410);
}
OA_DEVINL uint64_t mul_f32x2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
template <bool E4M3>
OA_DEVINL void from_8x4(uint32_t w, float (&x)[4]) {
    if (E4M3) {
        uint32_t lo, hi;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    } else {                                                     // 2^23 + 128 + x has x in its low byte (an integer's conversion runs at a quarter of the rate)
        w ^= 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 + i)) - 8388736.f;
    }
}

// Rows run over tokens, then planes, then heads
struct RowOf { int token, plane, head; };
struct RowWalk {                                                 // a thread's rows, a.step_tokens tokens and a.step_rows rows apart
    int token, rem;
    OA_DEVINL RowWalk(const Rows8Args& a, int64_t r) { token = (int)quotient(r, 2 * a.n_kv); rem = (int)(r - (int64_t)token * (2 * a.n_kv)); }
    OA_DEVINL RowOf next(const Rows8Args& a) {
        RowOf x; x.token = token; x.plane = rem >= a.n_kv; x.head = rem - x.plane * a.n_kv;
        token += a.step_tokens; rem += a.step_rows;
        if (rem >= 2 * a.n_kv) { rem -= 2 * a.n_kv; ++token; }
        return x;
    }
};
// where a row lies in the cache: its block, and its place there; null where its token is passed over
OA_DEVINL uint8_t* block_of(const Rows8Args& a, const RowOf& x, int slot, int& place) {
    if (slot < 0) return nullptr;
    const uint32_t page = (uint32_t)slot / CACHE_PAGE;
    if (page >= (uint32_t)a.num_pages) { if (a.status) *a.status = 400; return nullptr; }
    place = slot & (CACHE_PAGE - 1);
    const uint64_t block = (uint64_t)((uint32_t)x.plane * (uint32_t)a.num_pages + page) * (uint32_t)a.n_kv + (uint32_t)x.head;
    return reinterpret_cast<uint8_t*>(a.cache) + block * (uint32_t)(CACHE_PAGE * (a.head_dim + 4));
}

// LANES take a row, eight channels of either half of it each (their loads and stores lie next to each other so); those behind its end go along.  x / s is IEEE's quotient by Markstein's correction: with r the correctly rounded 1 / s and q = rn(x r), the remainder
// x - q s is exact in a fused operation and rn(q + r (x - q s)) is rn(x / s), as long as nothing underflows: for scales from 2^-64 on a quotient that the rounding to 8 bits does not take to 0 has no
// such remainder.  Smaller ones are divided (divisions throughout: 15.7 us for 8192 tokens of 2 x 8 heads of 128 instead of 11.7).
template <int LANES, bool E4M3, bool WHOLE>
__global__ void __launch_bounds__(ROWS8_THREADS) cache8_write_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int ROWS = ROWS8_THREADS / LANES, UNROLL = WRITE8_UNROLL;
    griddep_launch();
    const int lane = threadIdx.x % LANES, c = lane * 8, half = a.head_dim / 2;
    const bool in = c < half;
    const int64_t rows = (int64_t)a.T * 2 * a.n_kv;
    griddep_wait();
    for (int64_t r0 = (int64_t)blockIdx.x * (ROWS * UNROLL); r0 < rows; r0 += (int64_t)gridDim.x * (ROWS * UNROLL)) {
        RowOf x[UNROLL]; int slot[UNROLL]; uint4 raw[UNROLL][2];
        RowWalk walk(a, r0 + threadIdx.x / LANES);
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const int64_t r = r0 + j * ROWS + threadIdx.x / LANES;
            slot[j] = -1;
            raw[j][0] = raw[j][1] = make_uint4(0u, 0u, 0u, 0u);
            if (r >= rows) continue;
            x[j] = walk.next(a);
            slot[j] = __ldcg(a.slots + x[j].token);
            if (!in) continue;
            const uint16_t* src = reinterpret_cast<const uint16_t*>(x[j].plane ? a.v : a.k) + (int64_t)x[j].token * a.ldkv + (int64_t)x[j].head * a.head_dim + c;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (WHOLE) raw[j][h] = ld_once_16(src + half * h);
                else {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldcg(src + half * h + 2 * i) | (uint32_t)__ldcg(src + half * h + 2 * i + 1) << 16;
                    raw[j][h] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const uint32_t w[8] = {raw[j][0].x, raw[j][0].y, raw[j][0].z, raw[j][0].w, raw[j][1].x, raw[j][1].y, raw[j][1].z, raw[j][1].w};
            uint32_t top = w[0] & 0x7fff7fffu;                   // magnitudes order as their bits do, infinities and NaN above all others
#pragma unroll
            for (int i = 1; i < 7; i += 2) top = __vimax3_u16x2(top, w[i] & 0x7fff7fffu, w[i + 1] & 0x7fff7fffu);
            top = __vmaxu2(top, w[7] & 0x7fff7fffu);
            top = max(top << 16, top & 0xffff0000u);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            int place = 0;
            uint8_t* block = slot[j] >= 0 ? block_of(a, x[j], slot[j], place) : nullptr;
            if (!block) continue;
            const bool bad = top >= 0x7f800000u;
            const float scale = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(top), E4M3 ? 448.f : 127.f);
            uint32_t y[4] = {0u, 0u, 0u, 0u};
            if (scale >= 5.4e-20f) {                             // 2^-64
                const float inv = -__frcp_rn(scale);
                const uint64_t inv2 = pack_f32x2(inv, inv), scale2 = pack_f32x2(scale, scale);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float z[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {                // the quotient's negative: zeros keep their sign so
                        const uint64_t v = pack_f32x2(bf16lo(w[2 * i + e]), bf16hi(w[2 * i + e])), q = mul_f32x2(v, inv2);
                        unpack_f32x2(fma_f32x2(fma_f32x2(q, scale2, v), inv2, q), z[2 * e], z[2 * e + 1]);
                    }
                    y[i] = E4M3 ? to_e4m3x4(-z[0], -z[1], -z[2], -z[3]) : near_int8x4(-z[0], -z[1], -z[2], -z[3]);
                }
            } else if (scale > 0.f) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float z0 = __fdiv_rn(bf16lo(w[2 * i]), scale), z1 = __fdiv_rn(bf16hi(w[2 * i]), scale), z2 = __fdiv_rn(bf16lo(w[2 * i + 1]), scale), z3 = __fdiv_rn(bf16hi(w[2 * i + 1]), scale);
                    y[i] = E4M3 ? to_e4m3x4(z0, z1, z2, z3) : to_int8x4(z0, z1, z2, z3);
                }
            }
            if (in) {
                uint8_t* dst = block + place * a.head_dim + c;
                *reinterpret_cast<uint2*>(dst) = make_uint2(y[0], y[1]); *reinterpret_cast<uint2*>(dst + half) = make_uint2(y[2], y[3]);
            }
            if (lane == 0) reinterpret_cast<float*>(block + CACHE_PAGE * a.head_dim)[place] = scale;
        }
    }
}

template <int LANES, bool E4M3, bool WHOLE>
__global__ void __launch_bounds__(ROWS8_THREADS) cache8_read_kernel(const __grid_constant__ Rows8Args a) {
    constexpr int ROWS = ROWS8_THREADS / LANES, UNROLL = READ8_UNROLL;
    griddep_launch();
    const int lane = threadIdx.x % LANES, c = lane * 8, half = a.head_dim / 2;
    const bool in = c < half;
    const int64_t rows = (int64_t)a.T * 2 * a.n_kv;
    griddep_wait();
    for (int64_t r0 = (int64_t)blockIdx.x * (ROWS * UNROLL); r0 < rows; r0 += (int64_t)gridDim.x * (ROWS * UNROLL)) {
        RowOf x[UNROLL]; int slot[UNROLL]; uint2 raw[UNROLL][2]; float scale[UNROLL];
        RowWalk walk(a, r0 + threadIdx.x / LANES);
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const int64_t r = r0 + j * ROWS + threadIdx.x / LANES;
            slot[j] = -1;
            if (r >= rows || !in) continue;
            x[j] = walk.next(a);
            slot[j] = __ldcg(a.slots + x[j].token);
        }
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            int place = 0;
            const uint8_t* block = slot[j] >= 0 ? block_of(a, x[j], slot[j], place) : nullptr;
            if (!block) { slot[j] = -1; continue; }
            const uint8_t* src = block + place * a.head_dim + c;
#pragma unroll
            for (int h = 0; h < 2; ++h) raw[j][h] = __ldcg(reinterpret_cast<const uint2*>(src + half * h));
            scale[j] = __ldcg(reinterpret_cast<const float*>(block + CACHE_PAGE * a.head_dim) + place);
        }
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            if (slot[j] < 0) continue;
            uint16_t* dst = reinterpret_cast<uint16_t*>(x[j].plane ? a.v_out : a.k_out) + (int64_t)x[j].token * a.ldkv + (int64_t)x[j].head * a.head_dim + c;
#pragma unroll
            for (int h = 0; h < 2; ++h, dst += half) {
                float v[2][4];
                from_8x4<E4M3>(raw[j][h].x, v[0]); from_8x4<E4M3>(raw[j][h].y, v[1]);
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(v[i >> 1][2 * (i & 1)] * scale[j], v[i >> 1][2 * (i & 1) + 1] * scale[j]);
                if (WHOLE) __stcs(reinterpret_cast<uint4*>(dst), make_uint4(o[0], o[1], o[2], o[3]));
                else
#pragma unroll
                    for (int i = 0; i < 8; ++i) dst[i] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
            }
        }
    }
}

template <typename K>
static cudaError_t launch_rows(K kern, int lanes, int unroll, Rows8Args a, cudaStream_t s) {
    a.step_tokens = ROWS8_THREADS / lanes / (2 * a.n_kv); a.step_rows = ROWS8_THREADS / lanes % (2 * a.n_kv);
    const int64_t each = ROWS8_THREADS / lanes * unroll, ctas = ((int64_t)a.T * 2 * a.n_kv + each - 1) / each;
    return launch_k(kern, dim3((unsigned)(ctas < 0x7fffffffll ? ctas : 0x7fffffffll)), dim3(ROWS8_THREADS), 0, s, a);
}
template <bool E4M3, bool WHOLE>
static cudaError_t launch_write(const Rows8Args& a, cudaStream_t s) {
    if (a.head_dim <= 64) return launch_rows(cache8_write_kernel<4, E4M3, WHOLE>, 4, WRITE8_UNROLL, a, s);
    if (a.head_dim <= 128) return launch_rows(cache8_write_kernel<8, E4M3, WHOLE>, 8, WRITE8_UNROLL, a, s);
    return launch_rows(cache8_write_kernel<16, E4M3, WHOLE>, 16, WRITE8_UNROLL, a, s);
}
template <bool E4M3, bool WHOLE>
static cudaError_t launch_read(const Rows8Args& a, cudaStream_t s) {
    if (a.head_dim <= 64) return launch_rows(cache8_read_kernel<4, E4M3, WHOLE>, 4, READ8_UNROLL, a, s);
    if (a.head_dim <= 128) return launch_rows(cache8_read_kernel<8, E4M3, WHOLE>, 8, READ8_UNROLL, a, s);
    return launch_rows(cache8_read_kernel<16, E4M3, WHOLE>, 16, READ8_UNROLL, a, s);
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
