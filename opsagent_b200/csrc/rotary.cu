// rotary.cu — rotary positions on rows of heads, alone or together with the write of new keys and values to a paged cache.
//
// Pair i of a head, (a, b), turns by the angle p f_i of its token's position p:  (a, b) -> s (a cos - b sin, a sin + b cos), s an amplitude (1 but for
// YaRN's).  Pairs lie half the rotated part apart or next to each other; channels behind the rotated part are copied.  The transposed map, a gradient's, is
// the same with -f_i.
//
// The angle is taken in 64 bits, in turns: p (f_i / 2 pi) less its nearest whole number is below 1/2 with an error of 2^-22 turns for positions of 31 bits (a
// product in 32 bits would be whole turns off), and only then rounded to fp32.  cos and sin of it, times s, in fp32; products and sums in fp32; one rounding
// at the end.
//
// Bound by memory: a CTA carries one token, whose cos and sin its threads take once for all its heads (64 of them under the loads of the first channels), a
// thread two pieces of 16 bytes of a head at a time, the pairs' a and b, and several of those in flight.
#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"

namespace oa {

constexpr int ROT_THREADS = 128;
constexpr int ROT_UNROLL = 4;            // units of two pieces in flight per thread

OA_DEVINL void rot_read(const float* p, float (&v)[4]) { const float4 x = *reinterpret_cast<const float4*>(p); v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
OA_DEVINL void rot_read(const float* p, float (&v)[1]) { v[0] = *p; }
OA_DEVINL void rot_read(const uint16_t* p, float (&v)[8]) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    v[0] = bf16lo(x.x); v[1] = bf16hi(x.x); v[2] = bf16lo(x.y); v[3] = bf16hi(x.y); v[4] = bf16lo(x.z); v[5] = bf16hi(x.z); v[6] = bf16lo(x.w); v[7] = bf16hi(x.w);
}
OA_DEVINL void rot_read(const uint16_t* p, float (&v)[1]) { v[0] = bf16_bits_to_f32(*p); }
OA_DEVINL void rot_write(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
OA_DEVINL void rot_write(float* p, const float (&v)[1]) { *p = v[0]; }
OA_DEVINL void rot_write(uint16_t* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
OA_DEVINL void rot_write(uint16_t* p, const float (&v)[1]) { *p = (uint16_t)(pack_bf16x2(v[0], 0.f) & 0xffffu); }

// E: uint16_t (bf16 bits) or float; VEC: elements of a piece, 16 bytes or 1 where rows, heads or halves are not aligned to pieces.  A unit is two pieces:
// the a and the b of VEC pairs (HALVES: pairs apart; else 2 VEC channels side by side), or 2 VEC channels that are copied.
template <typename E, int VEC, bool HALVES, bool CACHE>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const __grid_constant__ RotaryArgs a) {
    __shared__ float2 cs[ROTARY_MAX_PAIRS];
    const int t = blockIdx.x;
    const int D = a.head_dim, pairs = a.pairs;
    const int per_head = D / (2 * VEC), turned = pairs / VEC;
    const int heads = a.n_heads + (CACHE ? 2 * a.n_kv : 0), units = heads * per_head;
    griddep_launch();
    griddep_wait();
    const double p = (double)a.positions[t];
    int64_t page_row = -1;                                      // the token's row of head 0 in a plane of the cache
    if (CACHE) {
        const int slot = a.slots[t];
        if (slot >= 0 && slot / CACHE_PAGE < a.num_pages) page_row = (int64_t)(slot / CACHE_PAGE) * a.n_kv * CACHE_PAGE + slot % CACHE_PAGE;
        else if (slot >= 0 && a.status && threadIdx.x == 0) *a.status = 400;
    }
    bool first = true;
    const int stride = gridDim.y * ROT_THREADS;
    for (int u0 = blockIdx.y * ROT_THREADS; u0 < units; u0 += stride * ROT_UNROLL) {
        float lo[ROT_UNROLL][VEC], hi[ROT_UNROLL][VEC];
        E* dst[ROT_UNROLL]; int step[ROT_UNROLL], angle[ROT_UNROLL];
#pragma unroll
        for (int k = 0; k < ROT_UNROLL; ++k) {
            const int u = u0 + k * stride + threadIdx.x;
            dst[k] = nullptr;
            if (u >= units) continue;
            const int head = u / per_head, r = u - head * per_head;
            const E* src; E* to;
            bool turn = r < turned;
            if (!CACHE || head < a.n_heads) {
                src = reinterpret_cast<const E*>(a.x) + (int64_t)t * a.ldx + (int64_t)head * D;
                to = reinterpret_cast<E*>(a.out) + (int64_t)t * a.ldo + (int64_t)head * D;
            } else {
                const int kv = (head - a.n_heads) % a.n_kv;
                const bool value = head >= a.n_heads + a.n_kv;
                if (page_row < 0) continue;
                src = reinterpret_cast<const E*>(value ? a.v : a.k) + (int64_t)t * a.ldkv + (int64_t)kv * D;
                to = reinterpret_cast<E*>(a.cache) + (page_row + (int64_t)kv * CACHE_PAGE + (value ? (int64_t)a.num_pages * a.n_kv * CACHE_PAGE : 0)) * D;
                turn = turn && !value;
            }
            const bool apart = HALVES && r < turned;            // values too: their pieces only have to be all of the head's
            const int at = apart ? r * VEC : r * 2 * VEC;
            step[k] = apart ? pairs : VEC; angle[k] = turn ? r * VEC : -1;
            dst[k] = to + at;
            rot_read(src + at, lo[k]); rot_read(src + at + step[k], hi[k]);
        }
        if (first) {
            for (int i = threadIdx.x; i < pairs; i += ROT_THREADS) {
                const double turns = p * a.turns[i];
                float sn, cn;
                sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cn);
                cs[i] = make_float2(cn * a.amplitude, sn * a.amplitude);
            }
            __syncthreads();
            first = false;
        }
#pragma unroll
        for (int k = 0; k < ROT_UNROLL; ++k) {
            if (!dst[k]) continue;
            if (angle[k] >= 0) {
                if (HALVES) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float2 c = cs[angle[k] + i]; const float x = lo[k][i], y = hi[k][i];
                        lo[k][i] = x * c.x - y * c.y; hi[k][i] = x * c.y + y * c.x;
                    }
                } else if constexpr (VEC == 1) {
                    const float2 c = cs[angle[k]]; const float x = lo[k][0], y = hi[k][0];
                    lo[k][0] = x * c.x - y * c.y; hi[k][0] = x * c.y + y * c.x;
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; i += 2) {
                        const float2 c = cs[angle[k] + i / 2], d = cs[angle[k] + VEC / 2 + i / 2];
                        const float x = lo[k][i], y = lo[k][i + 1], z = hi[k][i], w = hi[k][i + 1];
                        lo[k][i] = x * c.x - y * c.y; lo[k][i + 1] = x * c.y + y * c.x;
                        hi[k][i] = z * d.x - w * d.y; hi[k][i + 1] = z * d.y + w * d.x;
                    }
                }
            }
            rot_write(dst[k], lo[k]); rot_write(dst[k] + step[k], hi[k]);
        }
    }
}

template <typename E, int VEC>
static cudaError_t launch_rotary_e(const RotaryArgs& a, bool halves, cudaStream_t s) {
    const bool cache = a.cache != nullptr;
    auto kern = halves ? rotary_kernel<E, VEC, true, false> : rotary_kernel<E, VEC, false, false>;
    if constexpr (sizeof(E) == 2) if (cache) kern = halves ? rotary_kernel<E, VEC, true, true> : rotary_kernel<E, VEC, false, true>;      // a cache of pages is bf16
    const int64_t units = (int64_t)(a.n_heads + (cache ? 2 * a.n_kv : 0)) * (a.head_dim / (2 * VEC));
    // few tokens: a token's heads over several CTAs, so that each thread has one unit or two
    const int64_t parts = a.T >= 148 ? 1 : (units + ROT_THREADS - 1) / ROT_THREADS;
    return launch_k(kern, dim3(a.T, (unsigned)(parts < 1 ? 1 : parts > 64 ? 64 : parts)), dim3(ROT_THREADS), 0, s, a);
}

cudaError_t launch_rotary(const RotaryArgs& a, int layout, bool f32, cudaStream_t s) {
    if (a.T <= 0) return cudaSuccess;
    const int esz = f32 ? 4 : 2, vec = 16 / esz;
    auto aligned = [&](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % vec == 0; };
    bool pieces = a.head_dim % (2 * vec) == 0 && a.pairs % vec == 0 && (2 * a.pairs) % (2 * vec) == 0 && aligned(a.x, a.ldx) && aligned(a.out, a.ldo);
    if (a.cache) pieces = pieces && aligned(a.k, a.ldkv) && aligned(a.v, a.ldkv) && aligned(a.cache, 0);
    const bool halves = layout == 1;
    if (f32) return pieces ? launch_rotary_e<float, 4>(a, halves, s) : launch_rotary_e<float, 1>(a, halves, s);
    return pieces ? launch_rotary_e<uint16_t, 8>(a, halves, s) : launch_rotary_e<uint16_t, 1>(a, halves, s);
}

}  // namespace oa
