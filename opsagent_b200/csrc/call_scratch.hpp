// call_scratch.hpp — device scratch of one kernel-level call, and the device a call runs on.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include <initializer_list>
#include <mutex>

namespace oa {

// Making the pool is no work of a stream, and a stream that is being captured, here or on another thread, would refuse it and lose its capture: it is allowed on this thread for as long as
// this lives.
class BesideCaptures {
public:
    BesideCaptures() { if (cudaThreadExchangeStreamCaptureMode(&mode_) != cudaSuccess) known_ = false; }
    BesideCaptures(const BesideCaptures&) = delete;
    ~BesideCaptures() { if (known_) cudaThreadExchangeStreamCaptureMode(&mode_); }

private:
    cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
    bool known_ = true;
};

// Scratch of one call (partials, plans, tables) comes from a stream-ordered pool of this library's own, one per device, made at the first use:
// cudaMalloc and cudaFree stop the whole device and cost 0.1 ms to several ms a call, more than most kernels here (paged attention of 6 x 3000
// tokens: 10 us of kernels in a call of 0.7 ms and more; from the pool 0.05 ms).  An allocation is ordered on the call's stream, so calls on
// several streams and threads never share a block; what the pool keeps between calls is bounded, the rest goes back to the device when a call
// synchronises.
constexpr uint64_t SCRATCH_KEEP_BYTES = 64ull << 20;
inline cudaMemPool_t scratch_pool() {
    static std::mutex mu;
    static cudaMemPool_t pools[64] = {};         // by device; nothing here may throw through the C boundary
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    std::lock_guard<std::mutex> lk(mu);
    cudaMemPool_t& pool = pools[dev];
    if (!pool) {
        const BesideCaptures making_the_pool;
        cudaMemPoolProps props{};
        props.allocType = cudaMemAllocationTypePinned; props.handleTypes = cudaMemHandleTypeNone;
        props.location.type = cudaMemLocationTypeDevice; props.location.id = dev;
        if (cudaMemPoolCreate(&pool, &props) != cudaSuccess) { pool = nullptr; return nullptr; }
        uint64_t keep = SCRATCH_KEEP_BYTES;
        cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
    }
    return pool;
}
// p is null where there is no memory.  The call says so by its code: the runtime's error does not stay behind for whoever asks next, which may be another library's check of its own launch.
struct DevBuf {
    void* p = nullptr;
    cudaStream_t s;
    DevBuf(size_t n, cudaStream_t stream) : s(stream) {
        if (n == 0) return;
        cudaMemPool_t pool = scratch_pool();
        if (!pool || cudaMallocFromPoolAsync(&p, n, pool, s) != cudaSuccess) { p = nullptr; cudaGetLastError(); }
    }
    DevBuf(const DevBuf&) = delete;
    ~DevBuf() { if (p) cudaFreeAsync(p, s); }
};

// The device that holds a call's memory, current for as long as this lives, if foreign() is false and error() is none: then every pointer is device (or managed) memory of that one device.
class CallDevice {
public:
    explicit CallDevice(std::initializer_list<const void*> pointers) {
        int dev = -1;
        for (const void* p : pointers) {
            if (!p) continue;
            cudaPointerAttributes at{};
            const cudaError_t e = cudaPointerGetAttributes(&at, p);
            if (e != cudaSuccess) { cudaGetLastError(); rc_ = e; return; }
            if ((at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) || (dev >= 0 && at.device != dev)) { foreign_ = true; return; }
            dev = at.device;
        }
        if (dev < 0) return;
        if ((rc_ = cudaGetDevice(&before_)) != cudaSuccess) { before_ = -1; return; }
        if (before_ == dev) { before_ = -1; return; }
        rc_ = cudaSetDevice(dev);
    }
    CallDevice(const CallDevice&) = delete;
    ~CallDevice() { if (before_ >= 0) cudaSetDevice(before_); }
    bool foreign() const { return foreign_; }           // a pointer that kernels cannot read, or of another device than the others
    cudaError_t error() const { return rc_; }

private:
    int before_ = -1;
    bool foreign_ = false;
    cudaError_t rc_ = cudaSuccess;
};

int call_failed(int code, const char* why);             // the text of oa_last_error() (engine.cpp); returns code

}  // namespace oa
