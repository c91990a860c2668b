// rotary.cu — rotary positions on rows of heads, alone or together with the write of new keys and values to a paged cache.
//
// Pair i of a head, (a, b), turns by the angle p f_i of its token's position p:  (a, b) -> s (a cos - b sin, a sin + b cos), s an amplitude (1 but for
// YaRN's).  Pairs lie half the rotated part apart or next to each other; channels behind the rotated part are copied.  The transposed map, a gradient's, is
// the same with -f_i.
//
// The angle is taken in 64 bits, in turns: p (f_i / 2 pi) less its nearest whole number is below 1/2 with an error of 2^-22 turns for positions of 31 bits (a
// product in 32 bits would be whole turns off), and only then rounded to fp32; what that rounding leaves (up to 1e-7, more than a result's own) turns cos and
// sin of it by its first order.  These, times s, in fp32; products and sums in fp32; one rounding at the end.
//
// Bound by memory.  A CTA walks over tokens (where one does not fill it) with ROT_CTAS of them on an SM: a thread holds its pair's frequency throughout, takes the pair's cos and sin of the
// token under the loads of its first units, and reads those of its place in a head once a token; the next token's position comes a token ahead.  Pieces stay packed
// until they turn: 80 registers a thread, four units of 32 bytes in flight each.  8192 tokens of 32 + 2 x 8 heads of 128 channels, 201 MB, take 33 us (6.1 TB/s; a
// CTA for each token, with its cos and sin in shared memory and unpacked pieces, 70 us), 1337 tokens of 40 + 2 x 8 heads 7.7 us with
// one set of inputs, which L2 holds (10.3 us), 8.7 over three.
#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"

namespace oa {

constexpr int ROT_THREADS = 128;         // at least ROTARY_MAX_PAIRS: a pair's angle a thread
constexpr int ROT_UNROLL = 4;            // units of two pieces in flight per thread
constexpr int ROT_CTAS = 6;              // of an SM: 80 registers a thread
static_assert(ROT_THREADS >= ROTARY_MAX_PAIRS);

template <typename E, int VEC> struct RotPiece { E v; };
template <> struct RotPiece<uint16_t, 8> { uint4 v; };
template <> struct RotPiece<float, 4> { float4 v; };

OA_DEVINL void rot_unpack(const RotPiece<float, 4>& p, float (&v)[4]) { v[0] = p.v.x; v[1] = p.v.y; v[2] = p.v.z; v[3] = p.v.w; }
OA_DEVINL void rot_unpack(const RotPiece<float, 1>& p, float (&v)[1]) { v[0] = p.v; }
OA_DEVINL void rot_unpack(const RotPiece<uint16_t, 8>& p, float (&v)[8]) {
    v[0] = bf16lo(p.v.x); v[1] = bf16hi(p.v.x); v[2] = bf16lo(p.v.y); v[3] = bf16hi(p.v.y); v[4] = bf16lo(p.v.z); v[5] = bf16hi(p.v.z); v[6] = bf16lo(p.v.w); v[7] = bf16hi(p.v.w);
}
OA_DEVINL void rot_unpack(const RotPiece<uint16_t, 1>& p, float (&v)[1]) { v[0] = bf16_bits_to_f32(p.v); }
OA_DEVINL void rot_pack(RotPiece<float, 4>& p, const float (&v)[4]) { p.v = make_float4(v[0], v[1], v[2], v[3]); }
OA_DEVINL void rot_pack(RotPiece<float, 1>& p, const float (&v)[1]) { p.v = v[0]; }
OA_DEVINL void rot_pack(RotPiece<uint16_t, 8>& p, const float (&v)[8]) { p.v = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])); }
OA_DEVINL void rot_pack(RotPiece<uint16_t, 1>& p, const float (&v)[1]) { p.v = (uint16_t)(pack_bf16x2(v[0], 0.f) & 0xffffu); }

template <int VEC>
OA_DEVINL void rot_angles(const float* from, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = *from;
    else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) { const float4 x = *reinterpret_cast<const float4*>(from + i); v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w; }
    }
}

// E: uint16_t (bf16 bits) or float; VEC: elements of a piece, 16 bytes or 1 where rows, heads or halves are not aligned to pieces.  A unit is two pieces:
// the a and the b of VEC pairs (HALVES: pairs apart; else 2 VEC channels side by side), or 2 VEC channels that are copied.  A thread keeps its place in a head
// and walks over heads, so that it reads its cos and sin once a token.
template <typename E, int VEC, bool HALVES, bool CACHE>
__global__ void __launch_bounds__(ROT_THREADS, ROT_CTAS) rotary_kernel(const __grid_constant__ RotaryArgs a) {
    using Piece = RotPiece<E, VEC>;
    __shared__ __align__(16) float cosines[2][ROTARY_MAX_PAIRS], sines[2][ROTARY_MAX_PAIRS];
    const int D = a.head_dim, pairs = a.pairs;
    const int per_head = D / (2 * VEC), turned = pairs / VEC;
    const int heads = a.n_heads + (CACHE ? 2 * a.n_kv : 0);
    const int across = per_head < ROT_THREADS ? per_head : ROT_THREADS, down = ROT_THREADS / across;     // threads on a head, heads at a time
    const int r0 = threadIdx.x % across, row = threadIdx.x / across;
    const int head0 = row < down ? blockIdx.y * down + row : heads, head_step = gridDim.y * down;
    const double turns = threadIdx.x < pairs ? a.turns[threadIdx.x] : 0.0;
    griddep_launch();
    griddep_wait();
    int position = a.positions[blockIdx.x], slot = CACHE ? a.slots[blockIdx.x] : -1;
    int phase = 0;
    for (unsigned t = blockIdx.x; t < (unsigned)a.T; t += gridDim.x, phase ^= 1) {
        const int64_t plane = CACHE ? (int64_t)a.num_pages * a.n_kv * CACHE_PAGE : 0;
        int64_t page_row = -1;                                  // the token's row of head 0 in a plane of the cache
        if (CACHE) {
            if (slot >= 0 && slot / CACHE_PAGE < a.num_pages) page_row = (int64_t)(slot / CACHE_PAGE) * a.n_kv * CACHE_PAGE + slot % CACHE_PAGE;
            else if (slot >= 0 && a.status && threadIdx.x == 0) *a.status = 400;
        }
        const double p = (double)position;
        if (t + gridDim.x < (unsigned)a.T) { position = a.positions[t + gridDim.x]; if (CACHE) slot = a.slots[t + gridDim.x]; }
        const E* x = reinterpret_cast<const E*>(a.x) + (int64_t)t * a.ldx;
        E* out = reinterpret_cast<E*>(a.out) + (int64_t)t * a.ldo;
        // head h's source and place, nullptr where it is not written; values are neither turned nor in out
        auto source = [&](int h) -> const E* {
            if (!CACHE || h < a.n_heads) return x + (int64_t)h * D;
            const bool value = h >= a.n_heads + a.n_kv;
            return reinterpret_cast<const E*>(value ? a.v : a.k) + (int64_t)t * a.ldkv + (int64_t)(h - a.n_heads - (value ? a.n_kv : 0)) * D;
        };
        auto place = [&](int h) -> E* {
            if (!CACHE || h < a.n_heads) return out + (int64_t)h * D;
            const bool value = h >= a.n_heads + a.n_kv;
            return reinterpret_cast<E*>(a.cache) + (page_row + (int64_t)(h - a.n_heads - (value ? a.n_kv : 0)) * CACHE_PAGE + (value ? plane : 0)) * D;
        };
        const int last = CACHE && page_row < 0 ? a.n_heads : heads;
        bool angles = false;
        for (int r = r0; r < per_head; r += across) {
            const bool apart = HALVES && r < turned;            // values too: their pieces only have to be all of the head's
            const int at = apart ? r * VEC : r * 2 * VEC, step = apart ? pairs : VEC;
            float cn[VEC], sn[VEC];
            int h = head0;
            do {
                Piece lo[ROT_UNROLL], hi[ROT_UNROLL];
#pragma unroll
                for (int k = 0; k < ROT_UNROLL; ++k) {
                    const int hk = h + k * head_step;
                    if (hk < last) { const E* src = source(hk) + at; lo[k] = *reinterpret_cast<const Piece*>(src); hi[k] = *reinterpret_cast<const Piece*>(src + step); }
                }
                if (!angles) {
                    if (threadIdx.x < pairs) {
                        const double full = p * turns, half = 2.0 * (full - rint(full));
                        const float near = (float)half, rest = (float)(half - (double)near) * 3.14159265f;
                        float s, c;
                        sincospif(near, &s, &c);
                        cosines[phase][threadIdx.x] = (c - s * rest) * a.amplitude; sines[phase][threadIdx.x] = (s + c * rest) * a.amplitude;
                    }
                    __syncthreads();                            // of the other phase's readers too: they are through with the token before
                    angles = true;
                }
                if (h == head0 && r < turned) { rot_angles<VEC>(&cosines[phase][r * VEC], cn); rot_angles<VEC>(&sines[phase][r * VEC], sn); }
#pragma unroll
                for (int k = 0; k < ROT_UNROLL; ++k) {
                    const int hk = h + k * head_step;
                    if (hk >= last) continue;
                    if (r < turned && (!CACHE || hk < a.n_heads + a.n_kv)) {
                        float u[VEC], w[VEC];
                        rot_unpack(lo[k], u); rot_unpack(hi[k], w);
                        if constexpr (HALVES || VEC == 1) {
#pragma unroll
                            for (int i = 0; i < VEC; ++i) { const float m = u[i], n = w[i]; u[i] = m * cn[i] - n * sn[i]; w[i] = m * sn[i] + n * cn[i]; }
                        } else {
#pragma unroll
                            for (int i = 0; i < VEC; i += 2) {
                                const int j = i / 2, l = VEC / 2 + j;
                                const float m = u[i], n = u[i + 1], o = w[i], q = w[i + 1];
                                u[i] = m * cn[j] - n * sn[j]; u[i + 1] = m * sn[j] + n * cn[j];
                                w[i] = o * cn[l] - q * sn[l]; w[i + 1] = o * sn[l] + q * cn[l];
                            }
                        }
                        rot_pack(lo[k], u); rot_pack(hi[k], w);
                    }
                    E* dst = place(hk) + at;
                    *reinterpret_cast<Piece*>(dst) = lo[k]; *reinterpret_cast<Piece*>(dst + step) = hi[k];
                }
                h += ROT_UNROLL * head_step;
            } while (h < last);
        }
    }
}

template <typename E, int VEC>
static cudaError_t launch_rotary_e(const RotaryArgs& a, bool halves, cudaStream_t s) {
    const bool cache = a.cache != nullptr;
    auto kern = halves ? rotary_kernel<E, VEC, true, false> : rotary_kernel<E, VEC, false, false>;
    if constexpr (sizeof(E) == 2) if (cache) kern = halves ? rotary_kernel<E, VEC, true, true> : rotary_kernel<E, VEC, false, true>;      // a cache of pages is bf16
    const int per_head = a.head_dim / (2 * VEC), down = ROT_THREADS / (per_head < ROT_THREADS ? per_head : ROT_THREADS);
    const int heads = a.n_heads + (cache ? 2 * a.n_kv : 0);
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    // Few tokens: a token's heads over several CTAs, a unit a thread (us with one CTA a token / several, 48 heads of 128: 6 tokens 2.1 / 1.8, 100 2.3 / 2.2, 300 3.1 / 3.5).
    const int parts = a.T >= sms ? 1 : (heads + down - 1) / down;
    // CTAs walk over tokens that do not fill their threads' loads in flight: 8192 tokens of 32 + 2 x 8 heads of 128 in bf16 33.3 us (a CTA a token 36.8), of 32 heads 23.3 (26.7), of 8 heads in
    // fp32 15.4 (19.8).  Tokens that do have a CTA each, as many as registers allow: 32 heads in fp32 40.3 (walking 44.9), 64 heads in bf16 41.3 (47.5), 64 + 2 x 8 56
    const bool walk = (int64_t)heads * per_head < ROT_THREADS * ROT_UNROLL;
    return launch_k(kern, dim3(walk && a.T > ROT_CTAS * sms ? ROT_CTAS * sms : a.T, parts > 64 ? 64 : parts), dim3(ROT_THREADS), 0, s, a);
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
