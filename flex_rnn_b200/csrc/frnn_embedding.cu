// Embedding lookup with scaling, and its gradient by sorted tokens.
#include "frnn_lm.cuh"

using namespace frnn_lm;

namespace {

// y_i = scale * W[t_i]; a zero row where t_i is ignored or (reported) outside the vocabulary.
template <class T>
__global__ void embedding_fw(const T* __restrict__ w, int64_t rows, int64_t width, int64_t row_stride, int64_t col_stride, const void* __restrict__ tokens,
                             int token_bytes, int64_t n, float scale, int64_t ignore, T* __restrict__ out, int* err) {
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int64_t t = token_at(tokens, token_bytes, i);
        const bool there = t != ignore && t >= 0 && t < rows;
        if (t != ignore && !there && threadIdx.x == 0) *err = CODE_TOKEN;
        for (int64_t d = threadIdx.x; d < width; d += blockDim.x)
            out[i * width + d] = from_float<T>(there ? scale * to_float(w[t * row_stride + d * col_stride]) : 0.f);
    }
}

// Tokens that take no part (ignored, outside the vocabulary) get the key `rows`, behind all others.
__device__ __forceinline__ unsigned key_of(const void* tokens, int bytes, int64_t i, int64_t rows, int64_t ignore) {
    const int64_t t = token_at(tokens, bytes, i);
    return t != ignore && t >= 0 && t < rows ? (unsigned)t : (unsigned)rows;
}

enum { SORT_THREADS = 1024, DIGIT_BITS = 8, DIGITS = 1 << DIGIT_BITS };

// Stable radix sort of (token, place) by token, one block: places of equal tokens stay in order, so the sums below do
// not depend on how threads are scheduled.  Each warp takes a contiguous part of the places in rounds of 32.
__global__ void __launch_bounds__(SORT_THREADS) embedding_sort(const void* __restrict__ tokens, int token_bytes, int n, int64_t rows, int64_t ignore, int passes,
                                                               unsigned* key_a, unsigned* key_b, int* at_a, int* at_b) {
    extern __shared__ unsigned count[];                        // [warps][DIGITS]
    __shared__ unsigned total[DIGITS];
    const int warps = SORT_THREADS / 32, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int part = (int)(((int64_t)n + warps - 1) / warps + 31) / 32 * 32;
    const int lo = min((int64_t)n, (int64_t)warp * part), hi = min((int64_t)n, (int64_t)lo + part);
    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * DIGIT_BITS;
        const unsigned *from = (pass & 1) ? key_b : key_a;
        const int* from_at = (pass & 1) ? at_b : at_a;
        unsigned* to = (pass & 1) ? key_a : key_b;
        int* to_at = (pass & 1) ? at_a : at_b;
        for (int i = threadIdx.x; i < warps * DIGITS; i += SORT_THREADS) count[i] = 0;
        __syncthreads();
        for (int i = lo + lane; i < hi; i += 32)
            atomicAdd(&count[warp * DIGITS + (((pass ? from[i] : key_of(tokens, token_bytes, i, rows, ignore)) >> shift) & (DIGITS - 1))], 1u);
        __syncthreads();
        for (int d = threadIdx.x; d < DIGITS; d += SORT_THREADS) {
            unsigned sum = 0;
            for (int k = 0; k < warps; k++) { const unsigned c = count[k * DIGITS + d]; count[k * DIGITS + d] = sum; sum += c; }
            total[d] = sum;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned sum = 0;
            for (int d = 0; d < DIGITS; d++) { const unsigned c = total[d]; total[d] = sum; sum += c; }
        }
        __syncthreads();
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const int i = i0 + lane;
            const bool in = i < hi;
            const unsigned key = !in ? 0 : pass ? from[i] : key_of(tokens, token_bytes, i, rows, ignore);
            const unsigned digit = in ? (key >> shift) & (DIGITS - 1) : DIGITS;
            const unsigned same = __match_any_sync(~0u, digit);
            if (in) {
                const unsigned before = __popc(same & ((1u << lane) - 1));
                const unsigned base = count[warp * DIGITS + digit];
                to[total[digit] + base + before] = key;
                to_at[total[digit] + base + before] = pass ? from_at[i] : i;
            }
            __syncwarp();
            if (in && (same & ((1u << lane) - 1)) == 0) count[warp * DIGITS + digit] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
    }
}

__device__ __forceinline__ int lower_bound(const unsigned* keys, int n, unsigned key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (keys[mid] < key) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// dW_v = scale * sum of the upstream rows at the places of token v, in the order of the places, in 32 bits.
template <class T>
__global__ void embedding_bw(const T* __restrict__ dy, const unsigned* __restrict__ keys, const int* __restrict__ at, int n, int64_t rows, int64_t width,
                             float scale, T* __restrict__ dw) {
    for (int64_t v = blockIdx.x; v < rows; v += gridDim.x) {
        const int lo = lower_bound(keys, n, (unsigned)v), hi = lower_bound(keys, n, (unsigned)v + 1);
        for (int64_t d = threadIdx.x; d < width; d += blockDim.x) {
            float sum = 0;
            for (int j = lo; j < hi; j++) sum += to_float(dy[(int64_t)at[j] * width + d]);
            dw[v * width + d] = from_float<T>(scale * sum);
        }
    }
}

int sort_passes(int64_t rows) {
    int bits = 1;
    while ((rows >> bits) != 0) bits++;          // the keys are 0 .. rows
    return (bits + DIGIT_BITS - 1) / DIGIT_BITS;
}

int bad_shape(const char* what, int dtype, int64_t rows, int64_t width, int token_bytes, int64_t n) {
    if (!dtype_known(dtype) || (token_bytes != 4 && token_bytes != 8)) return frnn_fail(FRNN_E_ARG, "%s: unknown data type", what);
    if (rows < 0 || width < 0 || n < 0 || rows >= (1ll << 31) || width >= (1ll << 31) || n >= (1ll << 31))
        return frnn_fail(FRNN_E_ARG, "%s: sizes have to be below 2^31", what);
    return FRNN_OK;
}

}  // namespace

extern "C" {

int frnn_embedding_forward(int dtype, const void* weight, int64_t rows, int64_t width, int64_t row_stride, int64_t col_stride, const void* tokens, int token_bytes,
                           int64_t n, float scale, int64_t ignore_index, void* out, int* err_word, void* stream) {
    if (int rc = bad_shape("frnn_embedding_forward", dtype, rows, width, token_bytes, n)) return rc;
    if (n == 0 || width == 0) return FRNN_OK;
    if ((!weight && rows) || !tokens || !out || !err_word) return frnn_fail(FRNN_E_ARG, "frnn_embedding_forward: bad argument");
    if (!on_boundary(weight, dtype_bytes(dtype)) || !on_boundary(out, dtype_bytes(dtype)) || !on_boundary(tokens, token_bytes) || !on_boundary(err_word, 4))
        return frnn_fail(FRNN_E_ARG, "frnn_embedding_forward: a pointer is not on a boundary of its elements");
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        embedding_fw<T><<<(unsigned)(n < 65535 ? n : 65535), 256, 0, (cudaStream_t)stream>>>((const T*)weight, rows, width, row_stride, col_stride, tokens, token_bytes, n,
                                                                                          scale, ignore_index, (T*)out, err_word);
        return launched("frnn_embedding_forward");
    });
}

size_t frnn_embedding_backward_workspace(int dtype, int64_t rows, int64_t width, int64_t n) {
    (void)dtype; (void)rows; (void)width;
    return n <= 0 ? 0 : (size_t)n * 16;
}

int frnn_embedding_backward(int dtype, const void* dout, const void* tokens, int token_bytes, int64_t n, int64_t rows, int64_t width, float scale,
                            int64_t ignore_index, void* dweight, void* workspace, void* stream) {
    if (int rc = bad_shape("frnn_embedding_backward", dtype, rows, width, token_bytes, n)) return rc;
    if (rows == 0 || width == 0) return FRNN_OK;
    if (!dweight || (n && (!dout || !tokens || !workspace))) return frnn_fail(FRNN_E_ARG, "frnn_embedding_backward: bad argument");
    if (!on_boundary(dout, dtype_bytes(dtype)) || !on_boundary(dweight, dtype_bytes(dtype)) || !on_boundary(tokens, token_bytes) || !on_boundary(workspace, 16))
        return frnn_fail(FRNN_E_ARG, "frnn_embedding_backward: a pointer is not on a boundary of its elements (the workspace: of 16 bytes)");
    unsigned* key = (unsigned*)workspace;
    int* at = (int*)(key + 2 * n);
    const int passes = sort_passes(rows);
    if (n) {
        embedding_sort<<<1, SORT_THREADS, SORT_THREADS / 32 * DIGITS * 4, (cudaStream_t)stream>>>(tokens, token_bytes, (int)n, rows, ignore_index, passes, key, key + n, at, at + n);
        if (int rc = launched("frnn_embedding_backward")) return rc;
    }
    const int side = passes & 1;
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        embedding_bw<T><<<(unsigned)(rows < 65535 ? rows : 65535), 256, 0, (cudaStream_t)stream>>>((const T*)dout, key + side * n, at + side * n, (int)n, rows, width,
                                                                                             scale, (T*)dweight);
        return launched("frnn_embedding_backward");
    });
}

}  // extern "C"
