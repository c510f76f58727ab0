// What the readout operators share: element types, index loads, the device of a call.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "gtm_host.cuh"

namespace gtm_readout {

constexpr int64_t kMostRows = (int64_t)1 << 31;     // rows, ids, labels: below 2^31, so that they fit the 32-bit indices of the kernels

// The device of a call, for its duration: the caller's current device is set back.
struct DeviceGuard {
    int before = -1, status = GTM_OK;
    explicit DeviceGuard(int device) { status = enter(device); }
    int enter(int device)
    {
        int now = 0;
        GTM_CU(cudaGetDevice(&now));
        if (now == device) return GTM_OK;
        GTM_CU(cudaSetDevice(device));
        before = now;
        return GTM_OK;
    }
    ~DeviceGuard()
    {
        if (before >= 0) cudaSetDevice(before);
    }
};

inline size_t type_bytes(int type)
{
    switch (type) {
    case GTM_F32: return 4;
    case GTM_BF16: case GTM_F16: return 2;
    default: return 0;
    }
}

inline bool aligned(const void *p, int64_t row_bytes, unsigned to)
{
    return ((uintptr_t)p | (uint64_t)row_bytes) % to == 0;
}

inline uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Element `i` of an array of int32 or int64.  Not by the read-only path: the kernels begin while the one before them still writes, and what that path
// loads must not change as long as a kernel lives.
__device__ __forceinline__ long long index_at(const void *p, int wide, long long i)
{
    return wide ? ((const long long *)p)[i] : (long long)((const int *)p)[i];
}

// The kernel behind this one may be set up while this one ends, and waits for its end before it reads what others have written.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A launch that may be set up while the kernel before it on the stream ends; its kernel begins with `wait_for_previous`.
template <class... Params, class... Given>
inline int launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream, Given &&...given)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = grid, config.blockDim = block, config.dynamicSmemBytes = shared, config.stream = stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization, attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute, config.numAttrs = 1;
    GTM_CU(cudaLaunchKernelEx(&config, kernel, static_cast<Params>(given)...));
    return GTM_OK;
}

template <class T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

}  // namespace gtm_readout
