// Layer norm over the last dimension, forward and backward, with weights for each column or for each head and column.
#include "frnn_lm.cuh"

using namespace frnn_lm;

namespace {

// A row's place in a tensor: row r of `frnn_rows` is (r / (n1 n2), r / n2 mod n1, r mod n2).
__device__ __forceinline__ int64_t place(const frnn_rows& s, const int64_t* stride, int64_t r) {
    const int64_t i2 = r % s.n2, q = r / s.n2;
    return (q / s.n1) * stride[0] + (q % s.n1) * stride[1] + i2 * stride[2];
}

__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[32];
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    float s = 0;
    for (int i = 0; i < blockDim.x / 32; i++) s += part[i];
    return s;
}

// y = (x - mean) rstd w + b, one block a row; the variance is that of the centred values, so a large mean costs no digits.
template <class T, class P>
__global__ void layer_norm_fw(frnn_rows s, const T* __restrict__ x, const P* __restrict__ w, const P* __restrict__ b, float eps, T* __restrict__ y, float2* stats) {
    const int64_t rows = s.n0 * s.n1 * s.n2;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + place(s, s.x, r);
        const int64_t par = s.heads > 1 ? (r % s.n2) * s.width : 0;
        float sum = 0;
        for (int64_t d = threadIdx.x; d < s.width; d += blockDim.x) sum += to_float(xr[d]);
        const float mean = block_sum(sum) / (float)s.width;
        float sq = 0;
        for (int64_t d = threadIdx.x; d < s.width; d += blockDim.x) {
            const float c = to_float(xr[d]) - mean;
            sq += c * c;
        }
        const float rstd = rsqrtf(block_sum(sq) / (float)s.width + eps);
        if (stats && threadIdx.x == 0) stats[r] = make_float2(mean, rstd);
        for (int64_t d = threadIdx.x; d < s.width; d += blockDim.x) {
            float v = (to_float(xr[d]) - mean) * rstd;
            if (w) v *= to_float(w[par + d]);
            if (b) v += to_float(b[par + d]);
            y[r * s.width + d] = from_float<T>(v);
        }
    }
}

// dx = rstd (g - mean(g) - xh mean(g xh)) with g = dy w, xh = (x - mean) rstd.
template <class T, class P>
__global__ void layer_norm_dx(frnn_rows s, const T* __restrict__ dy, const T* __restrict__ x, const P* __restrict__ w, const float2* __restrict__ stats, T* __restrict__ dx) {
    const int64_t rows = s.n0 * s.n1 * s.n2;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + place(s, s.x, r), *gr = dy + place(s, s.dy, r);
        T* dr = dx + place(s, s.dx, r);
        const int64_t par = s.heads > 1 ? (r % s.n2) * s.width : 0;
        const float2 st = stats[r];
        float a = 0, c = 0;
        for (int64_t d = threadIdx.x; d < s.width; d += blockDim.x) {
            const float g = to_float(gr[d]) * (w ? to_float(w[par + d]) : 1.f), xh = (to_float(xr[d]) - st.x) * st.y;
            a += g;
            c += g * xh;
        }
        a = block_sum(a) / (float)s.width;
        c = block_sum(c) / (float)s.width;
        for (int64_t d = threadIdx.x; d < s.width; d += blockDim.x) {
            const float g = to_float(gr[d]) * (w ? to_float(w[par + d]) : 1.f), xh = (to_float(xr[d]) - st.x) * st.y;
            dr[d] = from_float<T>(st.y * (g - a - xh * c));
        }
    }
}

// Sums over a slab of the rows of one head: part[slab][0|1][heads * width].
template <class T>
__global__ void layer_norm_dw(frnn_rows s, const T* __restrict__ dy, const T* __restrict__ x, const float2* __restrict__ stats, float* __restrict__ part, int slabs) {
    const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (d >= s.width) return;
    const int64_t head = blockIdx.y, rows = s.n0 * s.n1 * s.n2 / s.heads;
    float dw = 0, db = 0;
    for (int64_t i = blockIdx.z; i < rows; i += slabs) {
        const int64_t r = i * s.heads + head;
        const float2 st = stats[r];
        const float g = to_float(dy[place(s, s.dy, r) + d]);
        dw += g * ((to_float(x[place(s, s.x, r) + d]) - st.x) * st.y);
        db += g;
    }
    const int64_t all = s.heads * s.width;
    part[(blockIdx.z * 2) * all + head * s.width + d] = dw;
    part[(blockIdx.z * 2 + 1) * all + head * s.width + d] = db;
}

template <class P>
__global__ void layer_norm_join(const float* __restrict__ part, int slabs, int64_t all, P* __restrict__ dw, P* __restrict__ db) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= all) return;
    float a = 0, c = 0;
    for (int k = 0; k < slabs; k++) {
        a += part[(2ll * k) * all + i];
        c += part[(2ll * k + 1) * all + i];
    }
    if (dw) dw[i] = from_float<P>(a);
    if (db) db[i] = from_float<P>(c);
}

int slabs_of(const frnn_rows& s) {
    const int64_t rows = s.n0 * s.n1 * s.n2 / s.heads;
    return (int)(rows < 64 ? (rows ? rows : 1) : 64);
}

int bad_shape(const char* what, const frnn_rows* s, int dtype, int param_dtype) {
    if (!s || !dtype_known(dtype) || !dtype_known(param_dtype)) return frnn_fail(FRNN_E_ARG, "%s: bad argument or unknown data type", what);
    if (param_dtype != dtype && param_dtype != FRNN_F32) return frnn_fail(FRNN_E_ARG, "%s: weights have the type of x or are fp32", what);
    if (s->n0 < 0 || s->n1 < 0 || s->n2 < 0 || s->width < 0 || s->heads < 1 || (s->heads > 1 && s->heads != s->n2)) return frnn_fail(FRNN_E_ARG, "%s: bad sizes", what);
    if ((s->n0 && s->n1 && s->n2) && (double)s->n0 * s->n1 * s->n2 >= 2147483648.0) return frnn_fail(FRNN_E_ARG, "%s: 2^31 rows or more", what);
    if (s->width >= (1ll << 31) || s->heads > 65535) return frnn_fail(FRNN_E_ARG, "%s: width has to be below 2^31, heads below 2^16", what);
    return FRNN_OK;
}

// Calls f(T(), P()) with the element type of x and that of the weights (the same, or fp32).
template <class F> int with_types(int dtype, int param_dtype, F f) {
    return with_dtype(dtype, [&](auto t) {
        if (param_dtype == FRNN_F32) return f(t, float());
        return f(t, t);
    });
}

}  // namespace

extern "C" {

int frnn_layer_norm_forward(const frnn_rows* s, int dtype, const void* x, int param_dtype, const void* weight, const void* bias, float eps, void* y, float* stats,
                            void* stream) {
    if (int rc = bad_shape("frnn_layer_norm_forward", s, dtype, param_dtype)) return rc;
    const int64_t rows = s->n0 * s->n1 * s->n2;
    if (rows == 0 || s->width == 0) return FRNN_OK;
    if (!x || !y) return frnn_fail(FRNN_E_ARG, "frnn_layer_norm_forward: bad argument");
    if (!on_boundary(x, dtype_bytes(dtype)) || !on_boundary(y, dtype_bytes(dtype)) || !on_boundary(weight, dtype_bytes(param_dtype)) ||
        !on_boundary(bias, dtype_bytes(param_dtype)) || !on_boundary(stats, 8))
        return frnn_fail(FRNN_E_ARG, "frnn_layer_norm_forward: a pointer is not on a boundary of its elements (the statistics: of 8 bytes)");
    return with_types(dtype, param_dtype, [&](auto t, auto p) {
        typedef decltype(t) T;
        typedef decltype(p) P;
        layer_norm_fw<T, P><<<(unsigned)rows, 256, 0, (cudaStream_t)stream>>>(*s, (const T*)x, (const P*)weight, (const P*)bias, eps, (T*)y, (float2*)stats);
        return launched("frnn_layer_norm_forward");
    });
}

size_t frnn_layer_norm_backward_workspace(const frnn_rows* s) {
    return s && s->heads >= 1 && s->width > 0 ? (size_t)slabs_of(*s) * 2 * s->heads * s->width * 4 : 0;
}

int frnn_layer_norm_backward(const frnn_rows* s, int dtype, const void* dy, const void* x, int param_dtype, const void* weight, const float* stats, void* dx,
                             void* dweight, void* dbias, void* workspace, void* stream) {
    if (int rc = bad_shape("frnn_layer_norm_backward", s, dtype, param_dtype)) return rc;
    const int64_t rows = s->n0 * s->n1 * s->n2;
    if (s->width == 0) return FRNN_OK;
    if ((rows && (!dy || !x || !stats)) || ((dweight || dbias) && !workspace)) return frnn_fail(FRNN_E_ARG, "frnn_layer_norm_backward: bad argument");
    if (!on_boundary(x, dtype_bytes(dtype)) || !on_boundary(dy, dtype_bytes(dtype)) || !on_boundary(dx, dtype_bytes(dtype)) || !on_boundary(weight, dtype_bytes(param_dtype)) ||
        !on_boundary(dweight, dtype_bytes(param_dtype)) || !on_boundary(dbias, dtype_bytes(param_dtype)) || !on_boundary(stats, 8) || !on_boundary(workspace, 16))
        return frnn_fail(FRNN_E_ARG, "frnn_layer_norm_backward: a pointer is not on a boundary of its elements (the statistics: of 8, the workspace: of 16 bytes)");
    const cudaStream_t st = (cudaStream_t)stream;
    return with_types(dtype, param_dtype, [&](auto t, auto p) {
        typedef decltype(t) T;
        typedef decltype(p) P;
        if (dx && rows) {
            layer_norm_dx<T, P><<<(unsigned)rows, 256, 0, st>>>(*s, (const T*)dy, (const T*)x, (const P*)weight, (const float2*)stats, (T*)dx);
            if (int rc = launched("frnn_layer_norm_backward")) return rc;
        }
        if (!dweight && !dbias) return (int)FRNN_OK;
        const int slabs = slabs_of(*s);
        const int64_t all = s->heads * s->width;
        layer_norm_dw<T><<<dim3((unsigned)((s->width + 127) / 128), (unsigned)s->heads, slabs), 128, 0, st>>>(*s, (const T*)dy, (const T*)x, (const float2*)stats, (float*)workspace, slabs);
        if (int rc = launched("frnn_layer_norm_backward")) return rc;
        layer_norm_join<P><<<(unsigned)((all + 127) / 128), 128, 0, st>>>((const float*)workspace, slabs, all, (P*)dweight, (P*)dbias);
        return launched("frnn_layer_norm_backward");
    });
}

}  // extern "C"
