// Host-side helpers of the entries that take device arrays with strides.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

struct sddmm_handle_s;

namespace sddmm {

// Makes a device current and gives the caller's back.
class DeviceGuard {
    int before = -1, device;

  public:
    explicit DeviceGuard(int d) : device(d)
    {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before != device) cudaSetDevice(device);
    }
    ~DeviceGuard()
    {
        if (before >= 0 && before != device) cudaSetDevice(before);
    }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;
};

// Whether p is memory of this device (its own, or managed).
inline bool on_device(const void *p, int device)
{
    if (!p) return false;
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return false;
    }
    return a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == device);
}

// Whether n_a x n_b pieces of `width` elements, a_stride and b_stride elements apart, never overlap.
inline bool strides_apart(int64_t a_stride, int64_t n_a, int64_t b_stride, int64_t n_b, int64_t width)
{
    if (n_a <= 1 && n_b <= 1) return true;
    if (n_a <= 1) return b_stride >= width;
    if (n_b <= 1) return a_stride >= width;
    return (a_stride >= width && b_stride >= (n_a - 1) * a_stride + width) || (b_stride >= width && a_stride >= (n_b - 1) * b_stride + width);
}

// Status of the handle's device status word, which it clears (the stream has been waited for).
int device_status(sddmm_handle_s *h);

}  // namespace sddmm
