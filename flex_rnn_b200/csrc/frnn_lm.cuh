// What the kernels around the scans (frnn_embedding.cu, frnn_layer_norm.cu, frnn_logprobs.cu) share: element types,
// conversions, reductions, and the error reporting of the C ABI.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/frnn.h"

// defined in frnn_shim.cu: records the message that frnn_last_error returns, gives `code` back
int frnn_fail(int code, const char* fmt, ...);

namespace frnn_lm {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// Results are rounded once, to nearest, when they are stored.
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

inline size_t dtype_bytes(int dtype) { return dtype == FRNN_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == FRNN_F32 || dtype == FRNN_BF16 || dtype == FRNN_F16; }

// Calls f(T()) with the element type that `dtype` names.
template <class F> int with_dtype(int dtype, F f) {
    switch (dtype) {
        case FRNN_F32: return f(float());
        case FRNN_BF16: return f(__nv_bfloat16());
        default: return f(__half());
    }
}

inline bool on_boundary(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

inline int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? FRNN_OK : frnn_fail(FRNN_E_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
}

// Token i of int32 or int64 tokens.
__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t i) {
    return bytes == 8 ? ((const int64_t*)tokens)[i] : (int64_t)((const int32_t*)tokens)[i];
}

enum { CODE_TOKEN = 96 };      // error word: a token outside the vocabulary

}  // namespace frnn_lm
