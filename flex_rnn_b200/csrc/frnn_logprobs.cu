// Log probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
#include "frnn_lm.cuh"

using namespace frnn_lm;

namespace {

enum { THREADS = 256 };
constexpr float NIL = -512.f;      // 2^NIL is 0 in 32 bits; finite, so that 0 * log 0 is 0
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float max_nan(float a, float b) {       // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Orders floats as unsigned numbers; every NaN above +infinity, -0 with +0.
__device__ __forceinline__ unsigned ordered(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <class Op> __device__ __forceinline__ float block_all(float v, Op op) {
    __shared__ float part[32];
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    float s = part[0];
    for (int i = 1; i < THREADS / 32; i++) s = op(s, part[i]);
    return s;
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long v) {
    __shared__ unsigned long long part[32];
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    unsigned long long s = part[0];
    for (int i = 1; i < THREADS / 32; i++) s = max(s, part[i]);
    return s;
}

// One block a row.  In units of log 2, with m = max x, c = log2(e) / temperature, u_j = (x_j - m) c:
// s = sum 2^u, log2 p_j = u_j - log2 s, entropy = ln 2 (log2 s - sum 2^u u / s).
template <class T>
__global__ void __launch_bounds__(THREADS) logprobs_fw(const T* __restrict__ logits, int64_t vocab, int64_t row_stride, const void* __restrict__ tokens, int token_bytes,
                                                       float inv_t, int64_t ignore, int top, float* logprob, float* entropy, float* top_logprob, int64_t* top_token,
                                                       float* stats, int* err) {
    const int64_t row = blockIdx.x;
    const float c = LOG2E * inv_t;
    const T* x = logits + row * row_stride;
    float m = -INFINITY;
    for (int64_t j = threadIdx.x; j < vocab; j += THREADS) m = max_nan(m, to_float(x[j]));
    m = block_all(m, [](float a, float b) { return max_nan(a, b); });
    const bool empty = m == -INFINITY;                     // nothing may follow here
    const float m0 = empty ? 0.f : m;
    float s = 0, t = 0;
    for (int64_t j = threadIdx.x; j < vocab; j += THREADS) {
        const float u = max_nan((to_float(x[j]) - m0) * c, NIL), e = exp2f(u);
        s += e;
        t += e * u;                                        // 0 * NIL = -0 where a mask took the token out
    }
    s = block_all(s, [](float a, float b) { return a + b; });
    t = block_all(t, [](float a, float b) { return a + b; });
    const float l2s = log2f(s), h = empty ? 0.f : LN2 * (l2s - t / s);
    auto logp = [&](float v) { return empty ? -INFINITY : (v - m) * inv_t - LN2 * l2s; };
    if (threadIdx.x == 0) {
        const int64_t tok = token_at(tokens, token_bytes, row);
        float lp = 0;
        if (tok != ignore) {
            const bool in = tok >= 0 && tok < vocab;
            if (!in) *err = CODE_TOKEN;
            lp = in ? logp(to_float(x[tok])) : NAN;
        }
        logprob[row] = lp;
        entropy[row] = h;
        if (stats) { stats[3 * row] = m; stats[3 * row + 1] = l2s; stats[3 * row + 2] = h; }
    }
    // the k-th alternative is the largest (value, lowest token first) below the one before it
    unsigned long long last = ~0ull;
    for (int k = 0; k < top; k++) {
        unsigned long long best = 0;
        for (int64_t j = threadIdx.x; j < vocab; j += THREADS) {
            const unsigned long long key = (unsigned long long)ordered(to_float(x[j])) << 32 | (0xFFFFFFFFu - (unsigned)j);
            if (key < last && key > best) best = key;
        }
        last = block_max(best);
        if (threadIdx.x == 0) {
            const int64_t j = 0xFFFFFFFFu - (unsigned)last;
            top_token[row * top + k] = j;
            top_logprob[row * top + k] = logp(to_float(x[j]));
        }
    }
}

// d logits_j = 1/T [ g (1[j = token] - p_j) - h p_j (ln p_j + H) ], g and h the upstream gradients of log probability and entropy.
template <class T>
__global__ void __launch_bounds__(THREADS) logprobs_bw(const T* __restrict__ logits, int64_t vocab, int64_t row_stride, const void* __restrict__ tokens, int token_bytes,
                                                       float inv_t, int64_t ignore, const float* __restrict__ glp, const float* __restrict__ gent,
                                                       const float* __restrict__ stats, T* __restrict__ dlogits) {
    const int64_t row = blockIdx.x, tok = token_at(tokens, token_bytes, row);
    const T* x = logits + row * row_stride;
    const float m = stats[3 * row], l2s = stats[3 * row + 1], H = stats[3 * row + 2];
    const float c = LOG2E * inv_t, g = glp && tok != ignore ? glp[row] : 0.f, h = gent ? gent[row] : 0.f;
    for (int64_t j = threadIdx.x; j < vocab; j += THREADS) {
        float d = 0;
        if (m != -INFINITY) {
            const float lp2 = max_nan((to_float(x[j]) - m) * c - l2s, NIL), p = exp2f(lp2);
            d = -p * (g + h * (LN2 * lp2 + H));
            if (j == tok) d += g;
            d *= inv_t;
        }
        dlogits[row * vocab + j] = from_float<T>(d);
    }
}

int bad_shape(const char* what, int dtype, int64_t n, int64_t vocab, int token_bytes, float temperature) {
    if (!dtype_known(dtype) || (token_bytes != 4 && token_bytes != 8)) return frnn_fail(FRNN_E_ARG, "%s: unknown data type", what);
    if (n < 0 || vocab < 1 || n >= (1ll << 31) || vocab >= (1ll << 31)) return frnn_fail(FRNN_E_ARG, "%s: sizes have to be below 2^31, and the vocabulary not empty", what);
    if (!(temperature >= 1e-30f) || !(temperature <= 1e30f)) return frnn_fail(FRNN_E_ARG, "%s: the temperature has to be positive, from 1e-30 to 1e30", what);
    return FRNN_OK;
}

}  // namespace

extern "C" {

int frnn_token_logprobs_forward(int dtype, const void* logits, int64_t n, int64_t vocab, int64_t row_stride, const void* tokens, int token_bytes, int top, float temperature,
                                int64_t ignore_index, float* logprob, float* entropy, float* top_logprob, int64_t* top_token, float* stats, int* err_word, void* stream) {
    if (int rc = bad_shape("frnn_token_logprobs_forward", dtype, n, vocab, token_bytes, temperature)) return rc;
    if (top < 0 || top > FRNN_MAX_TOP || top > vocab) return frnn_fail(FRNN_E_ARG, "frnn_token_logprobs_forward: top has to be 0 to %d, and at most the vocabulary", FRNN_MAX_TOP);
    if (n == 0) return FRNN_OK;
    if (!logits || !tokens || !logprob || !entropy || !err_word || (top && (!top_logprob || !top_token)))
        return frnn_fail(FRNN_E_ARG, "frnn_token_logprobs_forward: bad argument");
    if (!on_boundary(logits, dtype_bytes(dtype)) || !on_boundary(tokens, token_bytes) || !on_boundary(logprob, 4) || !on_boundary(entropy, 4) || !on_boundary(top_logprob, 4) ||
        !on_boundary(top_token, 8) || !on_boundary(stats, 4) || !on_boundary(err_word, 4))
        return frnn_fail(FRNN_E_ARG, "frnn_token_logprobs_forward: a pointer is not on a boundary of its elements");
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        logprobs_fw<T><<<(unsigned)n, THREADS, 0, (cudaStream_t)stream>>>((const T*)logits, vocab, row_stride, tokens, token_bytes, 1.f / temperature, ignore_index, top,
                                                                           logprob, entropy, top_logprob, top_token, stats, err_word);
        return launched("frnn_token_logprobs_forward");
    });
}

int frnn_token_logprobs_backward(int dtype, const void* logits, int64_t n, int64_t vocab, int64_t row_stride, const void* tokens, int token_bytes, float temperature,
                                 int64_t ignore_index, const float* dlogprob, const float* dentropy, const float* stats, void* dlogits, void* stream) {
    if (int rc = bad_shape("frnn_token_logprobs_backward", dtype, n, vocab, token_bytes, temperature)) return rc;
    if (n == 0) return FRNN_OK;
    if (!logits || !tokens || !stats || !dlogits) return frnn_fail(FRNN_E_ARG, "frnn_token_logprobs_backward: bad argument");
    if (!on_boundary(logits, dtype_bytes(dtype)) || !on_boundary(dlogits, dtype_bytes(dtype)) || !on_boundary(tokens, token_bytes) || !on_boundary(dlogprob, 4) ||
        !on_boundary(dentropy, 4) || !on_boundary(stats, 4))
        return frnn_fail(FRNN_E_ARG, "frnn_token_logprobs_backward: a pointer is not on a boundary of its elements");
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        logprobs_bw<T><<<(unsigned)n, THREADS, 0, (cudaStream_t)stream>>>((const T*)logits, vocab, row_stride, tokens, token_bytes, 1.f / temperature, ignore_index, dlogprob,
                                                                           dentropy, stats, (T*)dlogits);
        return launched("frnn_token_logprobs_backward");
    });
}

}  // extern "C"
