// tma.cpp — CUtensorMap construction.  cuTensorMapEncodeTiled is resolved through the CUDA runtime
// (cudaGetDriverEntryPoint) so the library has no link-time dependency on libcuda.so and loads on a
// GPU-less build box.
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "kernels.hpp"

namespace oa {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn resolve_encode() {
    static std::atomic<EncodeTiledFn> fn{nullptr};
    if (EncodeTiledFn f = fn.load()) return f;
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qres;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !p) return nullptr;
    fn = reinterpret_cast<EncodeTiledFn>(p);
    return fn.load();
}

// Encodes with the driver's own function, which wants a context on the calling thread: a thread whose first call this is has none until the runtime binds the current device's to it.
static int encode(CUtensorMap* out, CUtensorMapDataType type, uint32_t rank, const void* base, const cuuint64_t* gdim, const cuuint64_t* gstride, const cuuint32_t* box) {
    EncodeTiledFn enc = resolve_encode();
    if (!enc) return -1;
    const cuuint32_t estr[3] = {1, 1, 1};
    auto call = [&] {
        return enc(out, type, rank, const_cast<void*>(base), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = call();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = call();
    }
    return r == CUDA_SUCCESS ? 0 : (int)r;
}

int make_tmap_bf16_2d(CUtensorMap* out, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch_elems,
                      uint32_t box_rows, uint32_t box_cols) {
    if (box_cols * 2 > 128 || box_rows > 256 || (pitch_elems * 2) % 16 != 0 || (reinterpret_cast<uintptr_t>(base) & 15)) return -2;
    cuuint64_t gdim[2] = {cols, rows};
    cuuint64_t gstride[1] = {pitch_elems * 2};
    cuuint32_t box[2] = {box_cols, box_rows};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, gdim, gstride, box);
}

int make_tmap_bytes_2d(CUtensorMap* out, const void* base, uint64_t rows, uint32_t box_rows) {
    if (box_rows > 256 || (reinterpret_cast<uintptr_t>(base) & 15)) return -2;
    cuuint64_t gdim[2] = {128, rows};
    cuuint64_t gstride[1] = {128};
    cuuint32_t box[2] = {128, box_rows};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, gdim, gstride, box);
}

int make_tmap_bf16_heads(CUtensorMap* out, const void* base, uint64_t tokens, uint64_t heads, uint64_t head_dim, uint64_t pitch_elems, uint32_t box_tokens, uint32_t box_heads) {
    if (head_dim % 64 != 0 || box_tokens > 256 || box_heads > 256 || (pitch_elems * 2) % 16 != 0 || (reinterpret_cast<uintptr_t>(base) & 15)) return -2;
    cuuint64_t gdim[3] = {head_dim, heads, tokens};
    cuuint64_t gstride[2] = {head_dim * 2, pitch_elems * 2};
    cuuint32_t box[3] = {64, box_heads, box_tokens};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, gdim, gstride, box);
}

static std::atomic<uint64_t> g_launches{0};
uint64_t launches_total() { return g_launches.load(); }
void count_launch() { g_launches.fetch_add(1, std::memory_order_relaxed); }
bool pdl_enabled() {
    static const bool on = [] { const char* e = std::getenv("OA_PDL"); return !(e && e[0] == '0'); }();
    return on;
}

}  // namespace oa
