// Log probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
//
// Forward: one pass over the row.  In units of log 2, with c = log2(e) / temperature and u_j = (x_j - m) c for the largest
// logit m: s = sum 2^u, t = sum 2^u u, log2 p_j = u_j - log2 s, entropy = ln 2 (log2 s - t / s).  Each thread keeps its own
// m, s and t and rescales them when a batch brings a larger logit; threads, warps and the blocks of a cluster join theirs
// in a fixed order.  A cluster of up to 8 blocks shares a row where rows are few.
// Alternatives: the k-th largest of 64 groups' maxima bounds the k-th largest logit from below; the threads that have
// seen something as large look at their logits again (a few dozen of the row pass) and the candidates are ranked by
// counting.  The order is total, (logit, lowest token first), so the result does not depend on the threads.
// Backward: one pass, one read and one write a logit, with m, log2 s and the entropy from the forward.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "frnn_lm.cuh"

using namespace frnn_lm;
namespace cg = cooperative_groups;

namespace {

enum { THREADS = 256, WARPS = THREADS / 32, LOADS = 4, GROUPS = 64, MOST_CANDIDATES = 1024, MOST_CLUSTER = 8 };
constexpr float NIL = -512.f;      // 2^NIL is 0 in 32 bits; finite, so that 0 * log 0 is 0
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

typedef unsigned long long Key;

__device__ __forceinline__ float max_nan(float a, float b) {       // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {              // 2 units in the last place; below 2^-126: 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float exp2_small(float x) {             // the same, down to the smallest numbers
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Orders floats as unsigned numbers; every NaN above +infinity, -0 with +0.
__device__ __forceinline__ unsigned ordered(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ Key key_of(float x, int64_t token) { return (Key)ordered(x) << 32 | (0xFFFFFFFFu - (unsigned)token); }
__device__ __forceinline__ int64_t token_of(Key k) { return 0xFFFFFFFFu - (unsigned)k; }

// A row as accesses of E logits from the 16-byte boundary at or before its first one; the part of a block of the cluster.
template <class T, int E> struct Row {
    const T* x;
    int vocab, shift, first, end;           // accesses [first, end) are this block's
    __device__ __forceinline__ Row(const T* x, int vocab, int rank, int blocks) : x(x), vocab(vocab) {
        shift = E == 1 ? 0 : (int)((uintptr_t)x & 15) / (int)sizeof(T);
        const int all = (int)(((int64_t)vocab + shift + E - 1) / E), each = (all + blocks - 1) / blocks;
        first = min(all, rank * each);
        end = min(all, first + each);
    }
    __device__ __forceinline__ int at(int access) const { return access * E - shift; }
    __device__ __forceinline__ bool whole(int access) const { return at(access) >= 0 && at(access) <= vocab - E; }
    __device__ __forceinline__ bool there(int access, int e) const { return at(access) + e >= 0 && at(access) + e < vocab; }
    // logits of an access; -inf, which adds nothing, where there are none
    __device__ __forceinline__ void get(int access, float* f) const {
        if (access < end && whole(access)) {
            Pack<T, E> v;
            v.load(x + at(access));
            v.to(f);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) f[e] = access < end && there(access, e) ? to_float(x[at(access) + e]) : -INFINITY;
        }
    }
};

// m, s, t of a part of a row.  Without any finite logit: m = -inf, s = t = 0.
struct Part {
    float m, s, t;
};

// s and t of a part for a larger maximum.
__device__ __forceinline__ Part move_to(Part p, float m, float c) {
    const float d = m == -INFINITY ? 0.f : max_nan((p.m - m) * c, NIL), r = exp2_fast(d);
    return Part{m, p.s * r, (p.t + d * p.s) * r};
}

__device__ __forceinline__ Part block_join(Part p, float c) {
    __shared__ float largest[WARPS];
    __shared__ float2 sums[WARPS];
    float m = p.m;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; i++) m = max_nan(m, largest[i]);
    p = move_to(p, m, c);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        p.s += __shfl_xor_sync(~0u, p.s, o);
        p.t += __shfl_xor_sync(~0u, p.t, o);
    }
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x / 32] = make_float2(p.s, p.t);
    __syncthreads();
    p.s = p.t = 0;
#pragma unroll
    for (int i = 0; i < WARPS; i++) {
        p.s += sums[i].x;
        p.t += sums[i].y;
    }
    return p;
}

// ---- alternatives ----------------------------------------------------------------------------------------------------------

struct Candidates {
    Key key[MOST_CANDIDATES];
    int count;
};

// Adds the keys of the lanes that have one, as long as there is room; counts all of them.
__device__ __forceinline__ void push(Candidates& c, bool has, Key key, unsigned lanes) {
    const unsigned who = __ballot_sync(lanes, has);
    if (!who) return;
    const int lane = threadIdx.x & 31, leader = __ffs(who) - 1;
    int base = 0;
    if (lane == leader) base = atomicAdd(&c.count, __popc(who));
    base = __shfl_sync(lanes, base, leader);
    const int slot = base + __popc(who & ((1u << lane) - 1));
    if (has && slot < MOST_CANDIDATES) c.key[slot] = key;
}

// Candidates of the logits that are at least (strictly: above) `bound`, from the threads whose largest logit is.
template <class T, int E> __device__ void collect(const Row<T, E>& row, Candidates& c, unsigned largest, unsigned bound, bool strictly) {
    __syncthreads();                                       // (everyone has read the last count)
    if (threadIdx.x == 0) c.count = 0;
    __syncthreads();
    const bool mine = strictly ? largest > bound : largest >= bound;
    if (__any_sync(~0u, mine)) {
        for (int a0 = row.first + (threadIdx.x & ~31); a0 < row.end; a0 += LOADS * THREADS) {
            float f[LOADS][E];
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const int a = a0 + (threadIdx.x & 31) + u * THREADS;
                if (mine && a < row.end) row.get(a, f[u]);
            }
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const int a = a0 + (threadIdx.x & 31) + u * THREADS;
                unsigned hits = 0;
                if (mine && a < row.end)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const unsigned o = ordered(f[u][e]);
                        if (row.there(a, e) && (strictly ? o > bound : o >= bound)) hits |= 1u << e;
                    }
                if (!__any_sync(~0u, hits)) continue;
#pragma unroll
                for (int e = 0; e < E; e++) push(c, hits >> e & 1, key_of(f[u][e], row.at(a) + e), ~0u);
            }
        }
    }
    __syncthreads();
}

// The first `want` candidates by (logit, lowest token) of `n` in best[0 ...]; zeros behind them.
__device__ void rank(const Key* key, int n, int want, Key* best) {
    for (int i = threadIdx.x; i < FRNN_MAX_TOP; i += THREADS) best[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const Key k = key[i];
        int before = 0;
        for (int j = 0; j < n; j++) before += key[j] > k;
        if (before < want) best[before] = k;
    }
    __syncthreads();
}

// The `top` best logits of a block's part of the row, in best[]; `largest`: the largest logit that this thread has seen.
template <class T, int E> __device__ void block_top(const Row<T, E>& row, float largest, int top, Candidates& c, Key* best) {
    __shared__ unsigned group[GROUPS];
    __shared__ unsigned found;
    __shared__ int before[WARPS];
    __shared__ Key leader[WARPS];
    constexpr int EACH = THREADS / GROUPS;
    const unsigned mine = ordered(largest);
    unsigned g = mine;
#pragma unroll
    for (int o = 1; o < EACH; o *= 2) g = max(g, __shfl_xor_sync(~0u, g, o));
    if (threadIdx.x % EACH == 0) group[threadIdx.x / EACH] = g;
    __syncthreads();
    if (threadIdx.x < GROUPS) {
        const unsigned v = group[threadIdx.x];
        int larger = 0;
        for (int i = 0; i < GROUPS; i++) larger += group[i] > v || (group[i] == v && i < threadIdx.x);
        if (larger == top - 1) found = v;
    }
    __syncthreads();
    const unsigned bound = found;
    // a bound of -inf says that fewer than `top` groups hold any token that may follow: all of those, then the first others
    bool many = bound <= ordered(-INFINITY) && (int64_t)(row.end - row.first) * E > MOST_CANDIDATES;
    if (!many) {
        collect(row, c, mine, bound, false);
        many = c.count > MOST_CANDIDATES;
    }
    if (many) {                            // many logits equal to the bound: those above it, then the equal ones in order
        collect(row, c, mine, bound, true);
        const int above = c.count;
        __syncthreads();
        if (above <= MOST_CANDIDATES - FRNN_MAX_TOP) {
            int have = 0;
            for (int a0 = row.first; a0 < row.end && have < top; a0 += THREADS) {
                const int a = a0 + threadIdx.x;
                float f[E];
                row.get(a, f);
                unsigned hits = 0;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (a < row.end && row.there(a, e) && ordered(f[e]) == bound) hits |= 1u << e;
                int upto = __popc(hits);
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int v = __shfl_up_sync(~0u, upto, o);
                    if ((threadIdx.x & 31) >= o) upto += v;
                }
                if ((threadIdx.x & 31) == 31) before[threadIdx.x / 32] = upto;
                __syncthreads();
                int at = have + upto - __popc(hits), all = 0;
                for (int w = 0; w < WARPS; w++) {
                    if (w < threadIdx.x / 32) at += before[w];
                    all += before[w];
                }
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (hits >> e & 1) {
                        if (at < top) c.key[above + at] = key_of(f[e], row.at(a) + e);
                        at++;
                    }
                have = min(top, have + all);
            }
            if (threadIdx.x == 0) c.count = above + have;
            __syncthreads();
        } else {                           // more than the buffer holds: one alternative after the other
            Key last = ~0ull;
            if (threadIdx.x < FRNN_MAX_TOP) best[threadIdx.x] = 0;
            for (int k = 0; k < top; k++) {
                Key b = 0;
                for (int a = row.first + threadIdx.x; a < row.end; a += THREADS) {
                    float f[E];
                    row.get(a, f);
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const Key key = key_of(f[e], row.at(a) + e);
                        if (row.there(a, e) && key < last && key > b) b = key;
                    }
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) b = max(b, __shfl_xor_sync(~0u, b, o));
                __syncthreads();
                if ((threadIdx.x & 31) == 0) leader[threadIdx.x / 32] = b;
                __syncthreads();
                for (int w = 0; w < WARPS; w++) b = max(b, leader[w]);
                if (threadIdx.x == 0) best[k] = b;
                last = b;
            }
            __syncthreads();
            return;
        }
    }
    rank(c.key, c.count, top, best);
}

// ---- forward -----------------------------------------------------------------------------------------------------------------

// What the blocks of a cluster tell each other.
struct Share {
    Part part;
    Key best[FRNN_MAX_TOP];
};

template <class T, int E>
__global__ void __launch_bounds__(THREADS, 4) logprobs_fw(const T* __restrict__ logits, int vocab, int64_t row_stride, const void* __restrict__ tokens, int token_bytes, float inv_t,
                                                          int64_t ignore, int top, int blocks, float* logprob, float* entropy, float* top_logprob, int64_t* top_token, float* stats,
                                                          int* err) {
    __shared__ Share share;
    __shared__ Candidates candidates;
    const int rank_ = blockIdx.x % blocks;
    const int64_t row = blockIdx.x / blocks;
    const T* x = logits + row * row_stride;
    const float c = LOG2E * inv_t;
    const Row<T, E> part(x, vocab, rank_, blocks);
    float m = -INFINITY, m0 = 0;                          // m0: m, but 0 before there is any finite logit
    float2 s = both(0.f), t = both(0.f);
    const float2 c2 = both(c);
    for (int a = part.first + threadIdx.x; a < part.end; a += LOADS * THREADS) {
        constexpr int N = LOADS * E;
        float2 f[(N + 1) / 2];
        float* f1 = &f[0].x;
#pragma unroll
        for (int u = 0; u < LOADS; u++) part.get(a + u * THREADS, f1 + u * E);
        float b = f1[0];
#pragma unroll
        for (int i = 1; i < N; i++) b = max_nan(b, f1[i]);
        if (!(b <= m)) {
            const float d = max_nan((m - b) * c, NIL), r = exp2_fast(d);
            t = mul2(fma2(s, both(d), t), both(r));
            s = mul2(s, both(r));
            m = b;
            m0 = b == -INFINITY ? 0.f : b;
        }
        const float2 from = both(-m0);
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            float2 u = mul2(add2(f[i], from), c2);
            u.x = max_nan(u.x, NIL);
            u.y = max_nan(u.y, NIL);
            const float2 e = make_float2(exp2_fast(u.x), exp2_fast(u.y));
            s = add2(s, e);
            t = fma2(e, u, t);
        }
    }
    Part all = block_join(Part{m, s.x + s.y, t.x + t.y}, c);
    if (top) block_top(part, m, top, candidates, share.best);
    if (blocks > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) share.part = all;
        cluster.sync();
        if (rank_ == 0) {
            float most = -INFINITY;
            for (int k = 0; k < blocks; k++) most = max_nan(most, cluster.map_shared_rank(&share, k)->part.m);
            all = Part{most, 0, 0};
            for (int k = 0; k < blocks; k++) {
                const Part p = move_to(cluster.map_shared_rank(&share, k)->part, most, c);
                all.s += p.s;
                all.t += p.t;
            }
            if (top)
                for (int i = threadIdx.x; i < blocks * top; i += THREADS) candidates.key[i] = cluster.map_shared_rank(&share, i / top)->best[i % top];
        }
        cluster.sync();                                    // the others' shared memory has been read
        if (rank_) return;
        if (top) rank(candidates.key, blocks * top, top, share.best);
    }
    const bool empty = all.m == -INFINITY;                 // nothing may follow here
    const float l2s = log2f(all.s), h = empty ? 0.f : LN2 * (l2s - all.t / all.s);
    auto logp = [&](float v) { return empty ? -INFINITY : (v - all.m) * inv_t - LN2 * l2s; };
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
        if (stats) {
            stats[3 * row] = all.m;
            stats[3 * row + 1] = l2s;
            stats[3 * row + 2] = h;
        }
    }
    if (threadIdx.x < top) {
        const int64_t j = token_of(share.best[threadIdx.x]);
        top_token[row * top + threadIdx.x] = j;
        top_logprob[row * top + threadIdx.x] = logp(to_float(x[j]));
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------

// d logits_j = 1/T [ g (1[j = token] - p_j) - h p_j (ln p_j + H) ], g and h the upstream gradients of log probability and
// entropy: p_j times a linear function of log2 p_j, and the token's own term.  A block has LOADS * THREADS accesses of a row.
template <class T, int E>
__global__ void __launch_bounds__(THREADS) logprobs_bw(const T* __restrict__ logits, int vocab, int64_t row_stride, const void* __restrict__ tokens, int token_bytes, float inv_t,
                                                       int64_t ignore, const float* __restrict__ glp, const float* __restrict__ gent, const float* __restrict__ stats,
                                                       T* __restrict__ dlogits, unsigned tiles) {
    const unsigned row = blockIdx.x / tiles, tile = blockIdx.x - row * tiles;
    const Row<T, E> part(logits + row * row_stride, vocab, 0, 1);
    T* d = dlogits + (int64_t)row * vocab;
    const int first = (int)(tile * (LOADS * THREADS) + threadIdx.x);
    float f[LOADS][E];
#pragma unroll
    for (int u = 0; u < LOADS; u++) part.get(first + u * THREADS, f[u]);
    const float m = stats[3ll * row], l2s = stats[3ll * row + 1], H = stats[3ll * row + 2], c = LOG2E * inv_t;
    const int64_t tok = token_at(tokens, token_bytes, row);
    const float g = glp && tok != ignore ? glp[row] : 0.f, h = gent ? gent[row] : 0.f;
    const bool empty = m == -INFINITY;
    const float slope = empty ? 0.f : -inv_t * LN2 * h, level = empty ? 0.f : -inv_t * fmaf(h, H, g), own = empty ? 0.f : inv_t * g;
    const float m0 = empty ? 0.f : m, l0 = empty ? 0.f : l2s;
#pragma unroll
    for (int u = 0; u < LOADS; u++) {
        const int a = first + u * THREADS;
        if (a >= part.end) return;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float l = max_nan(fmaf(f[u][e] - m0, c, -l0), NIL);
            f[u][e] = exp2_small(l) * fmaf(l, slope, level);      // (a gradient is p times some tens: it may be seen where p is not)
        }
        const int64_t k = tok - part.at(a);
        if (k >= 0 && k < E)
#pragma unroll
            for (int e = 0; e < E; e++)
                if (k == e) f[u][e] += own;
        if (part.whole(a)) {
            Pack<T, E> v;
            v.from(f[u]);
            v.store(d + part.at(a));
        } else {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (part.there(a, e)) d[part.at(a) + e] = from_float<T>(f[u][e]);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------

int bad_shape(const char* what, int dtype, int64_t n, int64_t vocab, int token_bytes, float temperature) {
    if (!dtype_known(dtype) || (token_bytes != 4 && token_bytes != 8)) return frnn_fail(FRNN_E_ARG, "%s: unknown data type", what);
    if (n < 0 || vocab < 1 || n >= (1ll << 31) || vocab >= (1ll << 30)) return frnn_fail(FRNN_E_ARG, "%s: rows have to be below 2^31, and the vocabulary 1 to 2^30", what);
    if (!(temperature >= 1e-30f) || !(temperature <= 1e30f)) return frnn_fail(FRNN_E_ARG, "%s: the temperature has to be positive, from 1e-30 to 1e30", what);
    return FRNN_OK;
}

// Blocks that share a row: as many as it takes for two on each SM, as long as each thread has one round of loads.
int blocks_of(int64_t n, int64_t vocab, size_t size) {
    int blocks = 1;
    while (blocks < MOST_CLUSTER && n * blocks < 2 * sm_count() && vocab * (int64_t)size >= 2 * blocks * THREADS * LOADS * 16) blocks *= 2;
    return blocks;
}

// Calls f(T(), integral_constant E): accesses of 16 bytes, or of one element.
template <class F> int with_access(int dtype, bool wide, F f) {
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        if (wide) return f(t, std::integral_constant<int, WIDE<T>>());
        return f(t, std::integral_constant<int, 1>());
    });
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
    int blocks = blocks_of(n, vocab, dtype_bytes(dtype));
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)(n * blocks));
        config.blockDim = dim3(THREADS);
        config.stream = (cudaStream_t)stream;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = blocks;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.attrs = &cluster;
        config.numAttrs = blocks > 1;
        cudaLaunchKernelEx(&config, logprobs_fw<T, WIDE<T>>, (const T*)logits, (int)vocab, row_stride, tokens, token_bytes, 1.f / temperature, ignore_index, top, blocks, logprob, entropy,
                           top_logprob, top_token, stats, err_word);
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
    // rows of logits and of their gradient at the same distance behind 16-byte boundaries
    const int64_t size = (int64_t)dtype_bytes(dtype);
    const bool wide = (((uintptr_t)logits ^ (uintptr_t)dlogits) & 15) == 0 && (n == 1 || (row_stride - vocab) * size % 16 == 0);
    return with_access(dtype, wide, [&](auto t, auto e) {
        typedef decltype(t) T;
        const int64_t each = LOADS * THREADS * e.value, tiles = (vocab + e.value - 1 + each - 1) / each;
        if (n * tiles >= (1ll << 31)) return frnn_fail(FRNN_E_ARG, "frnn_token_logprobs_backward: too many logits");
        logprobs_bw<T, e.value><<<(unsigned)(n * tiles), THREADS, 0, (cudaStream_t)stream>>>((const T*)logits, (int)vocab, row_stride, tokens, token_bytes, 1.f / temperature, ignore_index,
                                                                                             dlogprob, dentropy, stats, (T*)dlogits, (unsigned)tiles);
        return launched("frnn_token_logprobs_backward");
    });
}

}  // extern "C"
