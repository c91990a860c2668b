// cache_copy.cu — copies of pages (or of a page's first places) of a paged cache, in all its planes and heads, by one launch.
//
// The pairs of pages travel in the launch's own parameters: no copy to the device ahead of the kernel, nothing to keep alive behind the call, and a captured
// call holds its own.  Up to 64 pairs go with 0.8 KB of parameters (a call takes the host 3.9 us; with 30 KB 5.9 us), up to
// 2560 with 30 KB; beyond that another launch.
//
// Bound by memory.  The places of a head of a page are one piece of up to 16 KB in each plane; a CTA copies up to 16 KB of a plane of a page, eight loads of 16
// bytes in flight per thread, whose heads lie next to each other where whole pages are copied and a stride apart otherwise.  515 MB of whole pages (257 MB read, as
// many written) take 83.3 us over three sets of inputs, 6.2 TB/s (78 with one, whose last pages L2 still holds).
//
// A fork writes one page to many.  A CTA then keeps what it has read in registers and writes it to several pages: as many as leave every SM the CTAs that it runs at
// once (9 at 56 registers), where at least every other pair's source is that of the pair before.  The bytes that come out of L2 are what it saves.  us for a page of 49 places in 64 planes
// of 8 x 128 channels written to 64 / 32 / 16 / 8 pages, a CTA for each pair: 103 / 53 / 25.6 / 10.3, by this rule (24, 12, 6, 3) 69 / 36 / 18.1 / 9.5, fewer (up to
// 16, 12 CTAs an SM) 73 / 39 / 20.0 / 9.4, more (6 CTAs) 77 / 39 / 19.5 / 10.7; floors 64 / 32 / 17 / 9.  A CTA's
// pairs are rounded down and the groups of pairs up: each of these four launches has 1344 CTAs, where 1332 run at once, and its last group may have fewer pairs.
#include "common.cuh"
#include "kernels.hpp"
#include "cache_ops.hpp"

namespace oa {

constexpr int COPY_THREADS = 128, COPY_UNROLL = 8, COPY_CHUNKS = COPY_THREADS * COPY_UNROLL;
constexpr int COPY_SHARE_CTAS = 8 * 148;                      // eight of an SM's nine: rounded up to groups, about as many as run at once

template <int CAP>
struct CopyArgs {
    uint4* cache; int32_t planes, num_pages, n_kv, row16, parts, share, n;      // row16: 16-byte chunks of a row; parts: CTAs of a plane of a page; share: moves of a CTA
    PageMove moves[CAP];
};

template <int CAP>
__global__ void __launch_bounds__(COPY_THREADS) cache_copy_kernel(const __grid_constant__ CopyArgs<CAP> a) {
    griddep_launch();
    const unsigned unit = blockIdx.x / (unsigned)a.parts, part = blockIdx.x - unit * (unsigned)a.parts;
    const unsigned group = unit / (unsigned)a.planes, plane = unit - group * (unsigned)a.planes;
    const unsigned page16 = CACHE_PAGE * a.row16;
    uint4* base = a.cache + (int64_t)plane * a.num_pages * a.n_kv * page16;
    uint4 v[COPY_UNROLL]; unsigned at[COPY_UNROLL];
    int read = -1, tokens = 0;                                   // what v holds
    unsigned mine = 0;
    griddep_wait();
    for (int k = group * a.share, end = min(k + a.share, a.n); k < end; ++k) {
        const PageMove m = a.moves[k];
        if (m.src != read || m.tokens != tokens) {
            read = m.src; tokens = m.tokens;
            const unsigned piece = tokens * a.row16, chunks = a.n_kv * piece;
            const unsigned each = (chunks + a.parts - 1) / (unsigned)a.parts, first = part * each, stop = min(first + each, chunks);
            const uint4* src = base + (int64_t)read * a.n_kv * page16;
            mine = 0;
#pragma unroll
            for (int i = 0; i < COPY_UNROLL; ++i) {
                const unsigned c = first + i * COPY_THREADS + threadIdx.x;
                const unsigned head = tokens == CACHE_PAGE ? 0 : c / piece;
                at[i] = c + head * (page16 - piece);
                if (c < stop) { mine |= 1u << i; v[i] = ld_once_16(src + at[i]); }
            }
        }
        uint4* dst = base + (int64_t)m.dst * a.n_kv * page16;
        // what is copied leaves L2 first: 69.0 us instead of 70.6 for the 64 pages above, 83.3 instead of 84.3 for 515 MB of whole pages over three sets of inputs
#pragma unroll
        for (int i = 0; i < COPY_UNROLL; ++i)
            if (mine >> i & 1) __stcs(dst + at[i], v[i]);
    }
}

template <int CAP>
static cudaError_t launch_copy(void* cache, int planes, int num_pages, int n_kv, int row_bytes, const PageMove* moves, int n, cudaStream_t s) {
    CopyArgs<CAP> a;
    a.cache = reinterpret_cast<uint4*>(cache); a.planes = planes; a.num_pages = num_pages; a.n_kv = n_kv; a.row16 = row_bytes / 16; a.n = n;
    int most = 0, again = 0;
    for (int i = 0; i < n; ++i) { a.moves[i] = moves[i]; if (moves[i].tokens > most) most = moves[i].tokens; if (i && moves[i].src == moves[i - 1].src) ++again; }
    if (most == 0) return cudaSuccess;
    a.parts = (n_kv * most * a.row16 + COPY_CHUNKS - 1) / COPY_CHUNKS;
    const int64_t ctas = (int64_t)n * planes * a.parts;
    const int64_t share = again * 2 >= n ? ctas / COPY_SHARE_CTAS : 1;
    a.share = share < 1 ? 1 : (int)share;
    return launch_k(cache_copy_kernel<CAP>, dim3((unsigned)((n + a.share - 1) / a.share * (int64_t)planes * a.parts)), dim3(COPY_THREADS), 0, s, a);
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
