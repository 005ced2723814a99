// operators.cuh -- what the language-model operators (embed_bags.cu, token_logprobs.cu) share:
// element types, vector loads that convert to f32, and the guard of their C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <stdexcept>
#include <string>

#include "common.cuh"
#include "hanns_gpu.h"
#include "ivf_usq_gpu.h"

namespace hanns {

void set_last_error(const std::string& msg);

// Runs f and maps what it throws to the CError codes of the C ABI.
template <class F>
int32_t operator_entry(F&& f) {
    try {
        f();
        return HANNS_OK;
    } catch (const std::invalid_argument& e) {
        set_last_error(e.what());
        return HANNS_INVALID_ARG;
    } catch (const CudaError& e) {
        set_last_error(e.what());
        return e.code == cudaErrorMemoryAllocation ? HANNS_OUT_OF_MEMORY : HANNS_INTERNAL;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return HANNS_INTERNAL;
    } catch (...) {
        set_last_error("unknown error");
        return HANNS_INTERNAL;
    }
}

inline void require(bool ok, const char* what) {
    if (!ok) throw std::invalid_argument(what);
}

// A pointer that the kernels may read or write as elements of `bytes` bytes (null is another check's).
inline bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }

// Kernels are started while the one before them in the stream comes to its end, and wait here for it
// to have finished before they read or write anything.  (Every kernel waits, so that waiting for one
// is waiting for all before it.)  The gradient of 150,001 tokens takes 121 us for 142 this way.
// Letting the next kernel's blocks onto the SMs earlier, from a kernel's start, does not pay: they
// wait where the last blocks of this one could run (143).
__device__ __forceinline__ void wait_for_previous() {
    cudaGridDependencySynchronize();
}
template <class... Params, class... Args>
void launch_early(void (*kernel)(Params...), unsigned grid, unsigned block, size_t shared, cudaStream_t s,
                  Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    HANNS_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
}

inline int dtype_bytes(int32_t dtype) { return dtype == HANNS_DTYPE_F32 ? 4 : 2; }
inline bool dtype_known(int32_t dtype) {
    return dtype == HANNS_DTYPE_F32 || dtype == HANNS_DTYPE_F16 || dtype == HANNS_DTYPE_BF16;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// One rounding to nearest even, the only one between the f32 sums and a 16-bit result.
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// N elements of T moved by one access (N * sizeof(T) is 16, 8, 4 or 2 bytes).
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, N>*>(p);
}

// Two 16-bit elements in a word, as f32.
template <class T> __device__ __forceinline__ float2 pair_f32(uint32_t w);
template <> __device__ __forceinline__ float2 pair_f32<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 pair_f32<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
}

// A pack's elements as f32 pairs (one element: in the first lane).
template <class T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float2 (&x)[(N + 1) / 2]) {
    if constexpr (N == 1) {
        x[0] = make_float2(to_f32(p.v[0]), 0.0f);
    } else if constexpr (sizeof(T) == 2) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&p);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) x[i] = pair_f32<T>(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) x[i] = make_float2(to_f32(p.v[2 * i]), to_f32(p.v[2 * i + 1]));
    }
}

}  // namespace hanns
