// What the files of C ABI entry points share: early return on a failed check, the calling thread's device, the number
// of SMs.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "check.h"
#include "rwkv7_b200.h"

#define RWKV7_TRY(expr)            \
    do {                           \
        if (int st_ = (expr)) return st_; \
    } while (0)

namespace rwkv7 {

// Makes `device` current for the duration of a call and restores the caller's.  A thread's first call sets the device in any
// case: until a thread has done something with its device it has no current context, and a tensor map cannot be encoded.
class DeviceGuard {
   public:
    explicit DeviceGuard(int device) {
        static thread_local int bound = -1;
        err_ = cudaGetDevice(&prev_);
        if (err_ == cudaSuccess && (prev_ != device || bound != device)) {
            err_ = cudaSetDevice(device);
            switched_ = err_ == cudaSuccess && prev_ != device;
            if (err_ == cudaSuccess) bound = device;
        }
    }
    ~DeviceGuard() {
        if (switched_) cudaSetDevice(prev_);
    }
    cudaError_t error() const { return err_; }

   private:
    int prev_ = 0;
    bool switched_ = false;
    cudaError_t err_ = cudaSuccess;
};

inline int cuda_fail(const char *what, int err) {
    return fail(RWKV7_ERR_CUDA, "CudaError: %s: %s", what, cudaGetErrorString((cudaError_t)err));
}

inline int num_sms(int device, int *out) {
    constexpr int kMaxDevices = 64;
    static std::atomic<int> known[kMaxDevices] = {};
    if (device < 0 || device >= kMaxDevices)
        return fail(RWKV7_ERR_BAD_ARGUMENT, "BadArgument: device ordinal %d out of range", device);
    int v = known[device].load(std::memory_order_relaxed);
    if (v == 0) {
        cudaError_t e = cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return cuda_fail("cudaDeviceGetAttribute", (int)e);
        known[device].store(v, std::memory_order_relaxed);
    }
    *out = v;
    return RWKV7_OK;
}

inline bool float_dtype_supported(int32_t dtype) { return dtype == RWKV7_F32 || dtype == RWKV7_BF16; }

}  // namespace rwkv7
