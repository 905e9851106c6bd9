// What the translation units of the layer operators need of a context.  Not
// part of the public ABI.
#pragma once
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

#include "bm_sampler.h"

enum { BM_WORK_SCAN = 0, BM_WORK_FP8 = 1, BM_WORK_KINDS = 2 };

// The largest workspace of bm_ssm_prefill: 2^26 rows times heads, the last part
// of 16 rows of each of up to 2^16 heads filled up, 16.5 bytes each.
constexpr size_t BM_WORK_SCAN_MOST = (((size_t)1 << 26) + ((size_t)1 << 20)) * 33 / 2;

// The library's error channel: sets bm_last_error's text, returns code.
int bm_detail_fail(int code, const char *msg);

// The context's device (returned), SM count, device error word and stream.
int bm_detail_ctx(bm_ctx_t *c, int *sms, int **d_err, cudaStream_t *stream);

// The context's workspace of a kind, at least `bytes` long, zeroed when it was
// allocated and never freed before the context.  Growing it allocates and
// synchronises the device, so it fails under stream capture.  It grows to twice
// its size, so that all that were outgrown are together less than twice the
// last of them, but not past the largest that its kind asks for, and to no more
// than is asked for where twice cannot be had.
int bm_detail_work(bm_ctx_t *c, int kind, size_t bytes, void **out);

namespace bmc {

// Reports a failed call, and clears the error that it leaves in the thread: a
// later call that succeeds would report it.
inline int cuda_fail(cudaError_t e, const char *what) {
    cudaGetLastError();
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
    return bm_detail_fail(e == cudaErrorMemoryAllocation ? BM_ERR_OOM : BM_ERR_CUDA, buf);
}

// The size that a workspace of `cap` bytes grows to when `bytes` are asked for,
// and no call asks for more than `most`.
inline size_t grown(size_t cap, size_t bytes, size_t most) {
    size_t n = cap <= most / 2 ? 2 * cap : most;
    if (n < bytes) n = bytes;
    return (n + 255) & ~(size_t)255;
}

// Makes a context's device current, and the caller's again at the end.
struct DeviceGuard {
    int before = -1, now;
    cudaError_t error;
    explicit DeviceGuard(int device) : now(device) {
        error = cudaGetDevice(&before);
        if (error == cudaSuccess && before != now) error = cudaSetDevice(now);
    }
    ~DeviceGuard() {
        if (before >= 0 && before != now) cudaSetDevice(before);
    }
};

// Lets a kernel take `bytes` of dynamic shared memory on a device: always the
// same number for a kernel, so that calls of several threads agree, and set
// once a device (the call costs as much as a launch).
struct SharedMemory {
    std::atomic<uint64_t> done{0};  // a bit per device, the first 64
    cudaError_t allow(const void *kernel, int bytes, int device) {
        const uint64_t bit = device < 64 ? 1ull << device : 0;
        if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
        const cudaError_t e =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
        return e;
    }
};

// A launch whose result is its own (what cudaGetLastError gives behind a launch
// may be an earlier call's, and states would be taken for unchanged).
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t shared, cudaStream_t s, A &&...args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = shared;
    c.stream = s;
    return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

}  // namespace bmc

#define BMC_CK(call)                                                     \
    do {                                                                 \
        cudaError_t e_ = (call);                                         \
        if (e_ != cudaSuccess) return bmc::cuda_fail(e_, #call);         \
    } while (0)
