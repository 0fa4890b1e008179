// What the kernels around the scans (frnn_embedding.cu, frnn_layer_norm.cu, frnn_logprobs.cu) share: element types,
// conversions, reductions, and the error reporting of the C ABI.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <cstring>
#include <mutex>

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

// E consecutive elements as one access of 16 bytes (E = 16 / size), or a single element (E = 1).
template <class T, int E> struct Pack;
template <class T> struct Pack<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    __device__ __forceinline__ void zero() { v = from_float<T>(0.f); }
    __device__ __forceinline__ void set(int, T x) { v = x; }
    __device__ __forceinline__ T get(int) const { return v; }
    __device__ __forceinline__ void to(float* f) const { f[0] = to_float(v); }
    __device__ __forceinline__ void from(const float* f) { v = from_float<T>(f[0]); }
};
template <> struct Pack<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *(const float4*)p; }
    __device__ __forceinline__ void store(float* p) const { *(float4*)p = v; }
    __device__ __forceinline__ void zero() { v = make_float4(0, 0, 0, 0); }
    __device__ __forceinline__ void set(int i, float x) { (&v.x)[i] = x; }
    __device__ __forceinline__ float get(int i) const { return (&v.x)[i]; }
    __device__ __forceinline__ void to(float* f) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
    __device__ __forceinline__ void from(const float* f) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <class T> struct Pack<T, 8> {           // 16-bit elements: the lower half of a word comes first
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = *(const uint4*)p; }
    __device__ __forceinline__ void store(T* p) const { *(uint4*)p = v; }
    __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void set(int i, T x) {
        unsigned short b;
        memcpy(&b, &x, 2);
        unsigned& w = (&v.x)[i / 2];
        w = i & 1 ? (w & 0xFFFFu) | (unsigned)b << 16 : (w & 0xFFFF0000u) | b;
    }
    __device__ __forceinline__ T get(int i) const {
        const unsigned short b = (unsigned short)((&v.x)[i / 2] >> (i & 1 ? 16 : 0));
        T x;
        memcpy(&x, &b, 2);
        return x;
    }
    __device__ __forceinline__ void to(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; i++) pair((&v.x)[i], f + 2 * i, T());
    }
    __device__ __forceinline__ void from(const float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) (&v.x)[i] = join(f[2 * i], f[2 * i + 1], T());
    }
    static __device__ __forceinline__ void pair(unsigned w, float* f, __nv_bfloat16) { f[0] = __uint_as_float(w << 16); f[1] = __uint_as_float(w & 0xFFFF0000u); }
    static __device__ __forceinline__ void pair(unsigned w, float* f, __half) {
        __half2 h;
        memcpy(&h, &w, 4);
        const float2 r = __half22float2(h);
        f[0] = r.x;
        f[1] = r.y;
    }
    static __device__ __forceinline__ unsigned join(float a, float b, __nv_bfloat16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        unsigned w;
        memcpy(&w, &h, 4);
        return w;
    }
    static __device__ __forceinline__ unsigned join(float a, float b, __half) {
        const __half2 h = __floats2half2_rn(a, b);
        unsigned w;
        memcpy(&w, &h, 4);
        return w;
    }
};
template <class T> constexpr int WIDE = 16 / (int)sizeof(T);

// Two 32-bit numbers at a time (add, mul, fma.rn.f32x2): half the instructions, the roundings of the single ones.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Stores of the E elements at p + at those with 0 <= at + e < n.
template <class T, int E> __device__ __forceinline__ void store_part(const Pack<T, E>& v, T* p, int at, int n) {
    if (at >= 0 && at + E <= n) {
        v.store(p + at);
    } else {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (at + e >= 0 && at + e < n) p[at + e] = v.get(e);
    }
}

// E elements out of 32 aligned bytes, from the one numbered `off` on.
template <class T, int E> __device__ __forceinline__ void shift_out(Pack<T, E>& v, const uint4& low, const uint4& high, unsigned off) {
    const unsigned words = off * (unsigned)sizeof(T) / 4, bits = sizeof(T) == 2 ? (off & 1) * 16 : 0;
    unsigned w[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
#pragma unroll
    for (int i = 0; i < 6; i++) w[i] = words & 2 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = words & 1 ? w[i + 1] : w[i];
    const uint4 r = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
    memcpy(&v.v, &r, 16);
}

// E elements from p, which may lie anywhere between 16-byte boundaries, by two accesses of 16 bytes and shifts.  These may
// hold other elements of the tensor [begin, end), but nothing outside of it: there, one element at a time.
template <class T, int E> __device__ __forceinline__ void load_anywhere(Pack<T, E>& v, const T* p, const T* begin, const T* end) {
    const unsigned off = (unsigned)((uintptr_t)p & 15) / (unsigned)sizeof(T);
    if (off == 0) {
        v.load(p);
    } else if (p - off >= begin && p - off + 2 * E <= end) {
        shift_out(v, *(const uint4*)(p - off), *(const uint4*)(p - off + E), off);
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) v.set(e, p[e]);
    }
}

// Launches a kernel; `early`: it may start while the one before it in the stream still runs, and itself waits where it needs
// that one's results (cudaGridDependencySynchronize).  `cluster` > 1: blocks of a cluster.
template <class... P, class... A> inline int launch(const char* what, void (*kernel)(P...), dim3 grid, unsigned threads, size_t shared, cudaStream_t stream, bool early, int cluster, A... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attrs[2];
    config.attrs = attrs;
    if (early) {
        attrs[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attrs[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[config.numAttrs].val.clusterDim.x = cluster;
        attrs[config.numAttrs].val.clusterDim.y = attrs[config.numAttrs].val.clusterDim.z = 1;
        config.numAttrs++;
    }
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, P(args)...);
    cudaGetLastError();
    return e == cudaSuccess ? (int)FRNN_OK : frnn_fail(FRNN_E_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
}

// Streaming multiprocessors of the current device (148 where there is none to ask).
inline int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return 148; }
    int n = known[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) { cudaGetLastError(); n = 148; }
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Shared memory beyond 48 KB has to be allowed for a kernel, once a device.  Sizes differ from launch to launch: the lock
// keeps a thread that asks for less from setting the attribute back after one that asks for more.
template <auto KERNEL> inline bool allow_shared(size_t bytes) {
    static std::atomic<size_t> allowed[64];
    static std::mutex setting;
    int dev = 0;
    if (bytes <= 40 * 1024) return true;             // (with what the kernel has besides)
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (allowed[dev].load(std::memory_order_acquire) >= bytes) return true;
    std::lock_guard<std::mutex> lock(setting);
    if (allowed[dev].load(std::memory_order_relaxed) >= bytes) return true;
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return false;
    allowed[dev].store(bytes, std::memory_order_release);
    return true;
}

// Token i of int32 or int64 tokens.
__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t i) {
    return bytes == 8 ? ((const int64_t*)tokens)[i] : (int64_t)((const int32_t*)tokens)[i];
}

enum { CODE_TOKEN = 96 };      // error word: a token outside the vocabulary

}  // namespace frnn_lm
