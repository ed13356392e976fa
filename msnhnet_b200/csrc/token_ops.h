// What the entry points of the token operators (rms_norm.cu, w4_linear.cu, attn_decode.cu, kv_cache.cu) share on the host.
#pragma once
#include "plan_internal.h"

namespace msnh {

inline size_t dtype_size(int dtype) { return dtype == MSNH_B200_F32 ? 4 : dtype == MSNH_B200_E4M3 ? 1 : 2; }
inline bool is_float_type(int dtype) { return dtype == MSNH_B200_F32 || dtype == MSNH_B200_F16 || dtype == MSNH_B200_BF16; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The context's device is the current one for the length of a call; the caller's own is put back.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        status = cudaGetDevice(&before_);
        if (status == cudaSuccess && before_ != device) { status = cudaSetDevice(device); moved_ = status == cudaSuccess; }
    }
    ~DeviceScope() { if (moved_) cudaSetDevice(before_); }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    cudaError_t status;
private:
    int before_ = 0;
    bool moved_ = false;
};

// One launch; `dependent`: it may be scheduled while the kernel before it in the stream still runs (it waits for that one's end
// itself before it touches memory). The launch's own status is returned, whatever an earlier call left behind.
template <typename... Params, typename... Args>
cudaError_t launch_token_kernel(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, void *stream, bool dependent, Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    if (dependent) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        config.attrs = attr;
        config.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

}  // namespace msnh
