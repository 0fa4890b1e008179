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

enum { LOADS = 4, MOST_CLUSTER = 8 };
// A row, or a cluster block's part of it, belongs to a block of 256 threads, or of 32 where rows are short.
template <int N> struct Block {
    static constexpr int WARPS = N / 32, GROUPS = N < 64 ? N : 64, MOST = N < 256 ? 512 : 1024;      // MOST: candidates
};
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

// The largest of several accesses' logits, NaN if one is: in pairs for 16-bit types.
template <int N> __device__ __forceinline__ float largest(const Pack<float, 4> (&v)[N]) {
    float m = v[0].v.x;
#pragma unroll
    for (int i = 0; i < N; i++) m = max_nan(max_nan(max_nan(m, v[i].v.x), max_nan(v[i].v.y, v[i].v.z)), v[i].v.w);
    return m;
}
template <class T, int N> __device__ __forceinline__ float largest(const Pack<T, 8> (&v)[N]) {
    typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
    auto two = [](unsigned w) {
        T2 r;
        memcpy(&r, &w, 4);
        return r;
    };
    T2 m = two(v[0].v.x);
#pragma unroll
    for (int i = 0; i < N; i++) m = __hmax2_nan(__hmax2_nan(__hmax2_nan(m, two(v[i].v.x)), __hmax2_nan(two(v[i].v.y), two(v[i].v.z))), two(v[i].v.w));
    return max_nan(to_float(m.x), to_float(m.y));
}

// Orders floats as unsigned numbers; every NaN above +infinity, -0 with +0.
__device__ __forceinline__ unsigned ordered(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
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
    __device__ __forceinline__ void get(int access, Pack<T, E>& v) const {
        if (access < end && whole(access)) {
            v.load(x + at(access));
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) v.set(e, access < end && there(access, e) ? x[at(access) + e] : from_float<T>(-INFINITY));
        }
    }
    // LOADS accesses, `step` apart: the checks of all of them at once where none is at an end
    __device__ __forceinline__ void get_round(int access, int step, Pack<T, E> (&v)[LOADS]) const {
        if (access + (LOADS - 1) * step < end && at(access) >= 0 && at(access + (LOADS - 1) * step) <= vocab - E) {
            const T* from = x + at(access);
#pragma unroll
            for (int u = 0; u < LOADS; u++) v[u].load(from + u * step * E);
        } else {
#pragma unroll
            for (int u = 0; u < LOADS; u++) get(access + u * step, v[u]);
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

template <int N> __device__ __forceinline__ Part block_join(Part p, float c) {
    constexpr int WARPS = Block<N>::WARPS;
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

enum { SLOTS = 16 };
template <int N> struct Candidates {
    Key key[Block<N>::MOST];
    unsigned short where[Block<N>::MOST];     // slots to look into: slot * N + thread
    int count, places;
    float seen[SLOTS][N];          // the largest logit of a thread in each `rounds` rounds of its loads
    int rounds;
};

// Candidates among the logits that are at least (strictly: above) `bound`.  The slots that have one are listed first, then
// their loads are dealt out to all threads, so that they wait for memory once.  More than there is room for: the count says
// so, and what is kept is of no use.
template <class T, int E, int N> __device__ void collect(const Row<T, E>& row, Candidates<N>& c, float bound, bool strictly) {
    constexpr int MOST = Block<N>::MOST;
    __syncthreads();                                       // (everyone has read the last count)
    if (threadIdx.x == 0) c.count = c.places = 0;
    __syncthreads();
    const unsigned least = ordered(bound);
    const int each = LOADS * c.rounds;
    for (int slot = 0; row.first + (int)threadIdx.x + slot * each * N < row.end; slot++) {
        const float seen = c.seen[slot][threadIdx.x];
        if (strictly ? seen <= bound : seen < bound) continue;      // (a NaN is not)
        const int i = atomicAdd(&c.places, 1);
        if (i < MOST) c.where[i] = (unsigned short)(slot * N + threadIdx.x);
    }
    __syncthreads();
    const int places = c.places;
    for (int i = threadIdx.x; i < min(places, MOST) * each; i += N) {
        const int where = c.where[i / each], a = row.first + where % N + (where / N * each + i % each) * N;
        if (a >= row.end) continue;
        Pack<T, E> v[1];
        row.get(a, v[0]);
        if (largest(v) < bound) continue;
        float f[E];
        v[0].to(f);
#pragma unroll
        for (int e = 0; e < E; e++) {
            const unsigned o = ordered(f[e]);
            if (!row.there(a, e) || (strictly ? o <= least : o < least)) continue;
            const int at = atomicAdd(&c.count, 1);
            if (at < MOST) c.key[at] = key_of(f[e], row.at(a) + e);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && places > MOST) c.count = MOST + 1;
    __syncthreads();
}

// The first `want` of `n` keys in best[0 ...], zeros behind them: a key's place is the number of larger ones.
template <int N> __device__ void rank(const Key* key, int n, int want, Key* best) {
    for (int i = threadIdx.x; i < FRNN_MAX_TOP; i += N) best[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += N) {
        const Key k = key[i];
        int before = 0;
        for (int j = 0; j < n; j++) before += key[j] > k;
        if (before < want) best[before] = k;
    }
    __syncthreads();
}

// The `top` best logits of a block's part of the row, in best[]; `seen`: the largest logit that this thread has seen.
template <class T, int E, int N> __device__ void block_top(const Row<T, E>& row, float seen, int top, Candidates<N>& c, Key* best) {
    constexpr int WARPS = Block<N>::WARPS, GROUPS = Block<N>::GROUPS, EACH = N / GROUPS, MOST = Block<N>::MOST;
    __shared__ unsigned group[GROUPS], found;
    __shared__ int before[WARPS];
    __shared__ Key leader[WARPS];
    float g = seen;
#pragma unroll
    for (int o = 1; o < EACH; o *= 2) g = max_nan(g, __shfl_xor_sync(~0u, g, o));
    if (threadIdx.x % EACH == 0) group[threadIdx.x / EACH] = ordered(g);
    __syncthreads();
    if (threadIdx.x < GROUPS) {
        const unsigned o = group[threadIdx.x];
        int larger = 0;
#pragma unroll 8
        for (int i = 0; i < GROUPS; i++) larger += group[i] > o || (group[i] == o && i < threadIdx.x);
        if (larger == top - 1) found = o;
    }
    __syncthreads();
    // a bound of -inf says that fewer than `top` groups hold a token that may follow: all of those, then the first others
    const float bound = value_of(found);
    bool many = bound == -INFINITY && (int64_t)(row.end - row.first) * E > MOST;
    if (!many) {
        collect<T, E, N>(row, c, bound, false);
        many = c.count > MOST;
    }
    if (many) {                            // many logits equal to the bound: those above it, then the equal ones in order
        collect<T, E, N>(row, c, bound, true);
        const int above = c.count;
        __syncthreads();
        if (above <= MOST - FRNN_MAX_TOP) {
            int have = 0;
            for (int a0 = row.first; a0 < row.end && have < top; a0 += N) {
                const int a = a0 + threadIdx.x;
                Pack<T, E> v;
                float f[E];
                row.get(a, v);
                v.to(f);
                unsigned hits = 0;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (a < row.end && row.there(a, e) && ordered(f[e]) == ordered(bound)) hits |= 1u << e;
                int upto = __popc(hits);
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int w = __shfl_up_sync(~0u, upto, o);
                    if ((threadIdx.x & 31) >= o) upto += w;
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
        } else {                           // more than there is room for: one alternative after the other
            Key last = 0;                  // (none before the first: a NaN of token 0 has the largest key that there is)
            for (int i = threadIdx.x; i < FRNN_MAX_TOP; i += N) best[i] = 0;
            for (int k = 0; k < top; k++) {
                Key b = 0;
                for (int a = row.first + threadIdx.x; a < row.end; a += N) {
                    Pack<T, E> v;
                    float f[E];
                    row.get(a, v);
                    v.to(f);
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const Key key = key_of(f[e], row.at(a) + e);
                        if (row.there(a, e) && (k == 0 || key < last) && key > b) b = key;
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
    rank<N>(c.key, c.count, top, best);
}

// ---- forward -----------------------------------------------------------------------------------------------------------------

// 8192 x 65536 bf16: 173 us, 6.2 TB/s of the copy's 6.5 (the exponentials' unit is two thirds busy, issue slots three
// quarters); with 5 alternatives 223 us, with 20 236; 2000 x 50003 fp32: 70 and with 5 alternatives 87.  One row: 6 us, of
// which the launch is most.  The next round's loads go out before this round's arithmetic (without that 325 us), and a round
// is checked for the row's ends once (each access by itself: 189 us).

// What the blocks of a cluster tell each other.
struct Share {
    Part part;
    Key best[FRNN_MAX_TOP];
};

template <class T, int E, int N>
__global__ void __launch_bounds__(N, N < 256 ? 32 : 4) logprobs_fw(const T* __restrict__ logits, int vocab, int64_t row_stride, const void* __restrict__ tokens, int token_bytes,
                                                                   float inv_t, int64_t ignore, int top, int blocks, float* logprob, float* entropy, float* top_logprob,
                                                                   int64_t* top_token, float* stats, int* err) {
    __shared__ Share share;
    __shared__ Candidates<N> candidates;
    const int rank_ = blockIdx.x % blocks;
    const int64_t row = blockIdx.x / blocks;
    const T* x = logits + row * row_stride;
    const float c = LOG2E * inv_t;
    const Row<T, E> part(x, vocab, rank_, blocks);
    float m = -INFINITY, m0 = 0;                          // m0: m, but 0 before there is any finite logit
    float2 s = both(0.f), t = both(0.f);
    const float2 c2 = both(c);
    Pack<T, E> next[LOADS];
    const int64_t tok = token_at(tokens, token_bytes, row);
    const int rounds = (part.end - part.first + SLOTS * LOADS * N - 1) / (SLOTS * LOADS * N);      // of a slot
    float slot_max = -INFINITY;
    int slot = 0, left = rounds;
    int a = part.first + threadIdx.x;
    part.get_round(a, N, next);
    // the token's logit is on its way behind the first round's
    const bool in = tok >= 0 && tok < vocab;
    const float own = rank_ == 0 && threadIdx.x == 0 && tok != ignore && in ? to_float(x[tok]) : 0.f;
    while (a < part.end) {
        Pack<T, E> v[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; u++) v[u] = next[u];
        a += LOADS * N;
        if (a < part.end) part.get_round(a, N, next);      // the next round's loads are under way during this one
        const float b = largest(v);
        if (top) {
            slot_max = max_nan(slot_max, b);
            candidates.seen[slot][threadIdx.x] = slot_max;
            if (--left == 0) {
                slot++;
                left = rounds;
                slot_max = -INFINITY;
            }
        }
        if (!(b <= m)) {
            const float d = max_nan((m - b) * c, NIL), r = exp2_fast(d);
            t = mul2(fma2(s, both(d), t), both(r));
            s = mul2(s, both(r));
            m = max_nan(m, b);                             // (a NaN stays, whatever comes after it)
            m0 = m == -INFINITY ? 0.f : m;
        }
        const float2 from = both(-m0);
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            float2 f[E / 2];
            v[u].to(&f[0].x);
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                float2 w = mul2(add2(f[i], from), c2);
                w.x = max_nan(w.x, NIL);
                w.y = max_nan(w.y, NIL);
                const float2 e = make_float2(exp2_fast(w.x), exp2_fast(w.y));
                s = add2(s, e);
                t = fma2(e, w, t);
            }
        }
    }
    Part all = block_join<N>(Part{m, s.x + s.y, t.x + t.y}, c);
    if (top && threadIdx.x == 0) candidates.rounds = rounds;
    if (top) block_top<T, E, N>(part, m, top, candidates, share.best);
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
                for (int i = threadIdx.x; i < blocks * top; i += N) candidates.key[i] = cluster.map_shared_rank(&share, i / top)->best[i % top];
        }
        cluster.sync();                                    // the others' shared memory has been read
        if (rank_) return;
        if (top) rank<N>(candidates.key, blocks * top, top, share.best);
    }
    const bool empty = all.m == -INFINITY;                 // nothing may follow here
    const float l2s = log2f(all.s), h = empty ? 0.f : LN2 * (l2s - all.t / all.s);
    auto logp = [&](float v) { return empty ? -INFINITY : (v - all.m) * inv_t - LN2 * l2s; };
    if (threadIdx.x == 0) {
        if (tok != ignore && !in) *err = CODE_TOKEN;
        logprob[row] = tok == ignore ? 0.f : in ? logp(own) : NAN;
        entropy[row] = h;
        if (stats) {
            stats[3 * row] = all.m;
            stats[3 * row + 1] = l2s;
            stats[3 * row + 2] = h;
        }
    }
    for (int k = threadIdx.x; k < top; k += N) {
        top_token[row * top + k] = token_of(share.best[k]);
        top_logprob[row * top + k] = logp(value_of((unsigned)(share.best[k] >> 32)));
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------

// d logits_j = 1/T [ g (1[j = token] - p_j) - h p_j (ln p_j + H) ], g and h the upstream gradients of log probability and
// entropy: p_j times a linear function of log2 p_j, and the token's own term.  p is the square of 2^(log2 p / 2): a gradient
// is p times some tens and may be seen where p itself is below the smallest number that the exponential gives.
// 8192 x 65536 bf16: 326 us for 2 GB, 2000 x 50003 fp32: 122 us, both a copy's rate.
// `lanes` threads have `tiles` tiles of a row, of LOADS * lanes accesses each.
template <class T, int E>
__global__ void __launch_bounds__(256) logprobs_bw(const T* __restrict__ logits, unsigned n, int vocab, int64_t row_stride, const void* __restrict__ tokens, int token_bytes,
                                                   float inv_t, int64_t ignore, const float* __restrict__ glp, const float* __restrict__ gent, const float* __restrict__ stats,
                                                   T* __restrict__ dlogits, unsigned spans, int tiles, int lanes) {
    const unsigned unit = blockIdx.x * (256u / lanes) + threadIdx.x / lanes, row = unit / spans, span = unit - row * spans;
    if (row >= n) return;
    const Row<T, E> part(logits + row * row_stride, vocab, 0, 1);
    T* d = dlogits + (int64_t)row * vocab;
    int a = (int)(span * (tiles * LOADS * lanes) + threadIdx.x % lanes);
    Pack<T, E> v[LOADS];
    part.get_round(a, lanes, v);
    const float m = stats[3ll * row], l2s = stats[3ll * row + 1], H = stats[3ll * row + 2];
    const int64_t tok = token_at(tokens, token_bytes, row);
    const float g = glp && tok != ignore ? glp[row] : 0.f, h = gent ? gent[row] : 0.f;
    const bool empty = m == -INFINITY;
    const float half_c = 0.5f * LOG2E * inv_t;
    const float2 by = both(half_c), from = both(empty ? 0.f : -m), less = both(empty ? 0.f : -0.5f * l2s);
    const float2 slope = both(empty ? 0.f : -2.f * inv_t * LN2 * h), level = both(empty ? 0.f : -inv_t * fmaf(h, H, g));
    const float own = empty ? 0.f : inv_t * g;
    const int hit = tok >= 0 && tok < vocab ? (int)tok : -E;             // (-E: in no access that is written)
    for (int tile = 0; tile < tiles && a < part.end; tile++) {
        if (tile) part.get_round(a, lanes, v);
        const bool inner = part.at(a) >= 0 && part.at(a + (LOADS - 1) * lanes) <= vocab - E;
#pragma unroll
        for (int u = 0; u < LOADS; u++) {
            if (!inner && a + u * lanes >= part.end) break;
            const int at = part.at(a + u * lanes);
            float2 f[(E + 1) / 2];
            float* f1 = &f[0].x;
            if (E == 1) f1[1] = 0;
            v[u].to(f1);
#pragma unroll
            for (int i = 0; i < (E + 1) / 2; i++) {
                float2 l = fma2(add2(f[i], from), by, less);       // log2 p / 2
                l.x = max_nan(l.x, NIL);
                l.y = max_nan(l.y, NIL);
                const float2 q = make_float2(exp2_fast(l.x), exp2_fast(l.y));
                f[i] = mul2(mul2(fma2(l, slope, level), q), q);
            }
            if ((unsigned)(hit - at) < (unsigned)E)
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (hit - at == e) f1[e] += own;
            v[u].from(f1);
            if (inner) v[u].store(d + at);
        }
        if (!inner)
#pragma unroll
            for (int u = 0; u < LOADS; u++) {
                const int access = a + u * lanes, at = part.at(access);
                if (access < part.end) store_part(v[u], d, at, vocab);
            }
        a += LOADS * lanes;
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------

int bad_shape(const char* what, int dtype, int64_t n, int64_t vocab, int token_bytes, float temperature) {
    if (!dtype_known(dtype) || (token_bytes != 4 && token_bytes != 8)) return frnn_fail(FRNN_E_ARG, "%s: unknown data type", what);
    if (n < 0 || vocab < 1 || n >= (1ll << 31) || vocab >= (1ll << 30)) return frnn_fail(FRNN_E_ARG, "%s: rows have to be below 2^31, and the vocabulary 1 to 2^30", what);
    if (!(temperature >= 1e-30f) || !(temperature <= 1e30f)) return frnn_fail(FRNN_E_ARG, "%s: the temperature has to be positive, from 1e-30 to 1e30", what);
    return FRNN_OK;
}

enum { SHORT_ROW = 8192 };       // bytes of a row that a block of one warp takes, where there are rows enough for eight of them on each SM

// Blocks that share a row: as many as it takes for two on each SM, as long as each thread has one round of loads.
int blocks_of(int64_t n, int64_t vocab, size_t size) {
    int blocks = 1;
    while (blocks < MOST_CLUSTER && n * blocks < 2 * sm_count() && vocab * (int64_t)size >= 2 * blocks * 256 * LOADS * 16) blocks *= 2;
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
    const int blocks = blocks_of(n, vocab, dtype_bytes(dtype));
    const bool is_short = vocab * (int64_t)dtype_bytes(dtype) <= SHORT_ROW && n > 8 * sm_count();
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)(n * blocks));
        config.blockDim = dim3(is_short ? 32 : 256);
        config.stream = (cudaStream_t)stream;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = blocks;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.attrs = &cluster;
        config.numAttrs = blocks > 1;
        cudaLaunchKernelEx(&config, is_short ? logprobs_fw<T, WIDE<T>, 32> : logprobs_fw<T, WIDE<T>, 256>, (const T*)logits, (int)vocab, row_stride, tokens, token_bytes,
                           1.f / temperature, ignore_index, top, blocks, logprob, entropy, top_logprob, top_token, stats, err_word);
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
        const int64_t accesses = (vocab + e.value - 1 + e.value - 1) / e.value;      // with up to E - 1 elements before a row's first
        int lanes = 32;                                    // as few as cover a short row, a block for others
        while (lanes < 256 && lanes * LOADS < accesses) lanes *= 2;
        // four tiles for what a thread needs besides (8192 x 65536 bf16: 326 us, one 367, eight 340), but rather one each for eight blocks an SM
        const int tiles = n * ((accesses + 4 * LOADS * lanes - 1) / (4 * LOADS * lanes)) >= 8 * sm_count() ? 4 : 1;
        const int64_t spans = (accesses + tiles * LOADS * lanes - 1) / (tiles * LOADS * lanes), units = n * spans;
        if (units >= (1ll << 31)) return frnn_fail(FRNN_E_ARG, "frnn_token_logprobs_backward: too many logits");
        const int in_block = 256 / lanes;
        logprobs_bw<T, e.value><<<(unsigned)((units + in_block - 1) / in_block), 256, 0, (cudaStream_t)stream>>>((const T*)logits, (unsigned)n, (int)vocab, row_stride, tokens, token_bytes,
                                                                                                               1.f / temperature, ignore_index, dlogprob, dentropy, stats, (T*)dlogits,
                                                                                                               (unsigned)spans, tiles, lanes);
        return launched("frnn_token_logprobs_backward");
    });
}

}  // extern "C"
