// cache_copy.cu — copies of pages (or of a page's first places) of a paged cache, in all its planes and heads, by one launch.
//
// The pairs of pages travel in the launch's own parameters: no copy to the device ahead of the kernel, nothing to keep alive behind the call, and a captured
// call holds its own.  Up to 64 pairs go with 0.8 KB of parameters, up to 2560 with 30 KB; beyond that another launch.
//
// Bound by memory.  The places of a head of a page are one piece of up to 16 KB in each plane; a CTA copies 16 KB of a (pair, plane), eight loads of 16 bytes in
// flight per thread, whose heads lie next to each other where whole pages are copied and a stride apart otherwise.
#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"

namespace oa {

constexpr int COPY_THREADS = 128, COPY_UNROLL = 8, COPY_CHUNKS = COPY_THREADS * COPY_UNROLL;

template <int CAP>
struct CopyArgs {
    uint4* cache; int32_t planes, num_pages, n_kv, row16, parts, n;       // row16: 16-byte chunks of a row; parts: CTAs of a (pair, plane)
    PageMove moves[CAP];
};

template <int CAP>
__global__ void __launch_bounds__(COPY_THREADS) cache_copy_kernel(const __grid_constant__ CopyArgs<CAP> a) {
    griddep_launch();
    const unsigned unit = blockIdx.x / (unsigned)a.parts, part = blockIdx.x - unit * (unsigned)a.parts;
    const unsigned move = unit / (unsigned)a.planes, plane = unit - move * (unsigned)a.planes;
    const PageMove m = a.moves[move];
    const unsigned page16 = CACHE_PAGE * a.row16, piece = m.tokens * a.row16, chunks = a.n_kv * piece;
    const uint4* src = a.cache + ((int64_t)plane * a.num_pages + m.src) * a.n_kv * page16;
    uint4* dst = a.cache + ((int64_t)plane * a.num_pages + m.dst) * a.n_kv * page16;
    griddep_wait();
    uint4 v[COPY_UNROLL]; unsigned at[COPY_UNROLL];
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i) {
        const unsigned c = part * COPY_CHUNKS + i * COPY_THREADS + threadIdx.x;
        const unsigned head = m.tokens == CACHE_PAGE ? 0 : c / piece;
        at[i] = c + head * (page16 - piece);
        if (c < chunks) v[i] = ld_nc_16(src + at[i]);
    }
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i)
        if (part * COPY_CHUNKS + i * COPY_THREADS + threadIdx.x < chunks) dst[at[i]] = v[i];
}

template <int CAP>
static cudaError_t launch_copy(void* cache, int planes, int num_pages, int n_kv, int row_bytes, const PageMove* moves, int n, cudaStream_t s) {
    CopyArgs<CAP> a;
    a.cache = reinterpret_cast<uint4*>(cache); a.planes = planes; a.num_pages = num_pages; a.n_kv = n_kv; a.row16 = row_bytes / 16; a.n = n;
    int most = 0;
    for (int i = 0; i < n; ++i) { a.moves[i] = moves[i]; if (moves[i].tokens > most) most = moves[i].tokens; }
    a.parts = (n_kv * most * a.row16 + COPY_CHUNKS - 1) / COPY_CHUNKS;
    return launch_k(cache_copy_kernel<CAP>, dim3((unsigned)((int64_t)n * planes * a.parts)), dim3(COPY_THREADS), 0, s, a);
}

cudaError_t launch_cache_copy(void* cache, int planes, int num_pages, int n_kv, int row_bytes, const PageMove* moves, int n_moves, cudaStream_t s) {
    constexpr int FEW = 64, MANY = 2560;
    // CTAs of a launch are counted in 31 bits
    const int64_t ctas = (int64_t)planes * (((int64_t)n_kv * CACHE_PAGE * (row_bytes / 16) + COPY_CHUNKS - 1) / COPY_CHUNKS);
    const int64_t cap = 0x7fffffffll / (ctas > 0 ? ctas : 1);
    if (cap < 1) return cudaErrorInvalidValue;
    const int many = cap < MANY ? (int)cap : MANY;
    for (int i = 0; i < n_moves;) {
        const int n = n_moves - i < many ? n_moves - i : many;
        const cudaError_t e = n <= FEW ? launch_copy<FEW>(cache, planes, num_pages, n_kv, row_bytes, moves + i, n, s) : launch_copy<MANY>(cache, planes, num_pages, n_kv, row_bytes, moves + i, n, s);
        if (e != cudaSuccess) return e;
        i += n;
    }
    return cudaSuccess;
}

}  // namespace oa
