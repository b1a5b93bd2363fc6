// host.hpp -- what the library's translation units share on the host: the
// error text of the calling thread, the device the library was initialised
// on, and a launch with programmatic stream serialisation.
#pragma once

#include <cuda_runtime.h>

#include <utility>

#include "../../include/mvllm_moe.h"

namespace mvb {

// Records the text mvllm_moe_last_error returns and passes `code` through.
int host_fail(int code, const char *fmt, ...);
// The initialised device and its SM count; MVLLM_ERR_NOT_INIT before
// mvllm_moe_init.
int host_device(int *device, int *sms);

#define MVB_TRY(expr)                                                                           \
    do {                                                                                        \
        cudaError_t e_ = (expr);                                                                \
        if (e_ != cudaSuccess)                                                                  \
            return ::mvb::host_fail(MVLLM_ERR_CUDA, "%s failed: %s", #expr,                     \
                                    cudaGetErrorString(e_));                                    \
    } while (0)

// Makes the library's device current for one call and puts the caller's back.
struct DeviceScope {
    int saved = -1, device = -1, sms = 0;
    int enter() {
        int cur = -1;
        if (int rc = host_device(&device, &sms))
            return rc;
        MVB_TRY(cudaGetDevice(&cur));
        if (cur != device) {
            MVB_TRY(cudaSetDevice(device));
            saved = cur;
        }
        return MVLLM_OK;
    }
    ~DeviceScope() {
        if (saved >= 0)
            cudaSetDevice(saved);
    }
};

// A launch that may begin while the previous kernel of the stream finishes;
// the kernel calls pdl_wait() before it touches global memory.
template <typename... KArgs, typename... Args>
cudaError_t launch_serial(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                          cudaStream_t st, Args &&...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

} // namespace mvb
