// work_units.hpp — units of work dealt out contiguously over a grid's CTAs: `total` units over `busy` CTAs, the same number to each but for one.  Host and device: the kernels that
// deal themselves such units use it, and a host program can compute it for sizes that no GPU has to run.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define OA_UNITS_FN __host__ __device__ __forceinline__
#else
#define OA_UNITS_FN inline
#endif

namespace oa {

// of a grid's CTAs the first min(grid, total) have units, each at least one: an item's parts are those of consecutive CTAs
OA_UNITS_FN int64_t busy_ctas(int64_t grid, int64_t total) { return total < grid ? (total > 0 ? total : 1) : grid; }
OA_UNITS_FN int64_t quotient(int64_t a, int64_t b) { return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }      // a >= 0, b > 0; in 32 bits where both fit: a 64-bit division takes several times as long
OA_UNITS_FN int64_t first_unit(int64_t cta, int64_t busy, int64_t total) { return cta < busy ? quotient(total * cta, busy) : total; }
OA_UNITS_FN int cta_of(int64_t unit, int64_t busy, int64_t total) { return (int)quotient((unit + 1) * busy - 1, total); }

}  // namespace oa
