// Layer norm over the last dimension, forward and backward, with weights for each column or for each head and column.
//
// Both directions are bound by memory: a pass over x (and dy) that keeps a row in registers between its reductions and its
// results, so each element is read and written once.  A row belongs to a group of lanes, 16 elements a lane: 2 to 32
// lanes of a warp up to 512 columns, a block of up to 512 threads up to 8192; longer rows are read again (``*_long``).
// A group walks over rows of one head, so its weights and the sums of its weight gradients stay in registers; the sums go
// to the workspace once and `layer_norm_join` adds them in a fixed order.
#include <algorithm>
#include <numeric>
#include <type_traits>

#include "frnn_lm.cuh"

using namespace frnn_lm;

namespace {

enum { PER_LANE = 16, BLOCK = 256, MOST_THREADS = 512 };

// A row's place in a tensor: row r of `frnn_rows` is (r / (n1 n2), r / n2 mod n1, r mod n2).
__device__ __forceinline__ int64_t place(const frnn_rows& s, const int64_t* stride, unsigned r) {
    const unsigned n1 = (unsigned)s.n1, n2 = (unsigned)s.n2;
    if (n1 == 1 && n2 == 1) return r * stride[0];
    const unsigned q = r / n2, i2 = r - q * n2;
    if (n1 == 1) return q * stride[0] + i2 * stride[2];
    const unsigned i0 = q / n1, i1 = q - i0 * n1;
    return i0 * stride[0] + i1 * stride[1] + i2 * stride[2];
}

// How rows are dealt out: `groups` groups in all, group g takes rows g, g + groups, ... ; groups is a multiple of the number
// of heads (a group's rows have one head) and of 8 (its rows lie alike to 16-byte boundaries whatever the width).
struct Deal {
    unsigned rows, groups, rounds;
};

// Sums over the lanes of a group: L lanes of a warp, or (L = 0) all threads of the block, by way of shared memory.  Two
// buffers by turns: one barrier a sum.
template <int L> struct Sums {
    float2 (*buffer)[MOST_THREADS / 32];
    int turn = 0;
    __device__ __forceinline__ float2 all(float2 v) {
#pragma unroll
        for (int o = L ? L / 2 : 16; o; o >>= 1) {
            v.x += __shfl_xor_sync(~0u, v.x, o);
            v.y += __shfl_xor_sync(~0u, v.y, o);
        }
        if (L) return v;
        if ((threadIdx.x & 31) == 0) buffer[turn][threadIdx.x / 32] = v;
        __syncthreads();
        float2 s = make_float2(0, 0);
        for (int i = 0; i < blockDim.x / 32; i++) {
            s.x += buffer[turn][i].x;
            s.y += buffer[turn][i].y;
        }
        turn ^= 1;
        return s;
    }
};

// Weights of the 16 columns of a lane, as 32-bit numbers.
template <class P, int E, int NV> __device__ __forceinline__ void load_params(const P* p, const int* at, int width, float none, float (&out)[NV * E]) {
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = at[j] + e;
            out[j * E + e] = p && c >= 0 && c < width ? to_float(p[c]) : none;
        }
}

// y = (x - mean) rstd w + b.  The variance is that of the centred values, so that a large mean costs no digits.
template <class T, class P, int L, int E>
__global__ void __launch_bounds__(L ? BLOCK : MOST_THREADS) layer_norm_fw(frnn_rows s, Deal deal, const T* __restrict__ x, const P* __restrict__ w, const P* __restrict__ b, float eps,
                                                                         T* __restrict__ y, float2* __restrict__ stats) {
    constexpr int NV = PER_LANE / E;
    __shared__ float2 buffer[2][MOST_THREADS / 32];
    const int width = (int)s.width, lanes = L ? L : blockDim.x, lane = L ? threadIdx.x % (L ? L : 1) : threadIdx.x;
    const unsigned g = L ? blockIdx.x * (BLOCK / (L ? L : 1)) + threadIdx.x / (L ? L : 1) : blockIdx.x;
    const unsigned head = s.heads > 1 ? g % (unsigned)s.heads : 0;
    Sums<L> sums{buffer};
    const int shift = E == 1 ? 0 : (int)((uintptr_t)(x + (g < deal.rows ? place(s, s.x, g) : 0)) & 15) / (int)sizeof(T);
    int at[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) at[j] = (j * lanes + lane) * E - shift;
    float wf[PER_LANE], bf[PER_LANE];
    load_params<P, E, NV>(w ? w + (int64_t)head * width : w, at, width, 1.f, wf);
    load_params<P, E, NV>(b ? b + (int64_t)head * width : b, at, width, 0.f, bf);
    Pack<T, E> v[NV], next[NV];
    auto fetch = [&](Pack<T, E>* to, unsigned r) {
        const T* from = x + place(s, s.x, r);
#pragma unroll
        for (int j = 0; j < NV; j++) load_part(to[j], from, at[j], width);
    };
    if (g < deal.rows) fetch(next, g);
    for (unsigned i = 0; i < deal.rounds; i++) {
        const unsigned r = i * deal.groups + g;
        const bool there = r < deal.rows;
#pragma unroll
        for (int j = 0; j < NV; j++) v[j] = next[j];
        if (there && deal.rows - r > deal.groups) fetch(next, r + deal.groups);
        float sum = 0, sq = 0;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float f[E];
            v[j].to(f);
#pragma unroll
            for (int e = 0; e < E; e++) sum += f[e];
        }
        const float mean = sums.all(make_float2(sum, 0)).x / (float)width;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float f[E];
            v[j].to(f);
            const bool whole = at[j] >= 0 && at[j] + E <= width;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float c = f[e] - mean;
                if (whole || (at[j] + e >= 0 && at[j] + e < width)) sq += c * c;
            }
        }
        const float rstd = rsqrtf(sums.all(make_float2(sq, 0)).x / (float)width + eps);
        if (!there) continue;
        if (stats && lane == 0) stats[r] = make_float2(mean, rstd);
        T* to = y + (int64_t)r * width;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float f[E];
            v[j].to(f);
#pragma unroll
            for (int e = 0; e < E; e++) f[e] = fmaf((f[e] - mean) * rstd, wf[j * E + e], bf[j * E + e]);
            Pack<T, E> out;
            out.from(f);
            store_part(out, to, at[j], width);
        }
    }
}

// dx = rstd (g - mean(g) - xh mean(g xh)) with g = dy w, xh = (x - mean) rstd; sums over the group's rows of dy xh and dy.
// part: [partials][2][width], one for each group, or (merge) for each warp; may be NULL, and so may dx.
template <class T, class P, int L, int E>
__global__ void __launch_bounds__(L ? BLOCK : MOST_THREADS) layer_norm_bw(frnn_rows s, Deal deal, const T* __restrict__ dy, const T* __restrict__ x, const P* __restrict__ w,
                                                                         const float2* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, bool merge) {
    constexpr int NV = PER_LANE / E;
    __shared__ float2 buffer[2][MOST_THREADS / 32];
    const int width = (int)s.width, lanes = L ? L : blockDim.x, lane = L ? threadIdx.x % (L ? L : 1) : threadIdx.x;
    const unsigned g = L ? blockIdx.x * (BLOCK / (L ? L : 1)) + threadIdx.x / (L ? L : 1) : blockIdx.x;
    const unsigned head = s.heads > 1 ? g % (unsigned)s.heads : 0;
    Sums<L> sums{buffer};
    const int shift = E == 1 ? 0 : (int)((uintptr_t)(x + (g < deal.rows ? place(s, s.x, g) : 0)) & 15) / (int)sizeof(T);
    int at[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) at[j] = (j * lanes + lane) * E - shift;
    float wf[PER_LANE], dw[PER_LANE], db[PER_LANE];
    load_params<P, E, NV>(w ? w + (int64_t)head * width : w, at, width, 1.f, wf);
#pragma unroll
    for (int i = 0; i < PER_LANE; i++) dw[i] = db[i] = 0;
    Pack<T, E> xv[NV], gv[NV], xn[NV], gn[NV];
    float2 st, sn = make_float2(0, 0);
    auto fetch = [&](unsigned r) {
        const T *px = x + place(s, s.x, r), *pg = dy + place(s, s.dy, r);
        sn = stats[r];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            load_part(xn[j], px, at[j], width);
            load_part(gn[j], pg, at[j], width);
        }
    };
#pragma unroll
    for (int j = 0; j < NV; j++) { xn[j].zero(); gn[j].zero(); }
    if (g < deal.rows) fetch(g);
    for (unsigned i = 0; i < deal.rounds; i++) {
        const unsigned r = i * deal.groups + g;
        const bool there = r < deal.rows;
        st = sn;
#pragma unroll
        for (int j = 0; j < NV; j++) { xv[j] = xn[j]; gv[j] = gn[j]; }
        if (there && deal.rows - r > deal.groups) fetch(r + deal.groups);
        float2 a = make_float2(0, 0);
        if (there) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                float f[E], u[E];
                xv[j].to(f);
                gv[j].to(u);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float xh = (f[e] - st.x) * st.y, gw = u[e] * wf[j * E + e];      // u = 0 where there is no column
                    a.x += gw;
                    a.y += gw * xh;
                    dw[j * E + e] += u[e] * xh;
                    db[j * E + e] += u[e];
                }
            }
        }
        if (dx) {
            a = sums.all(a);
            a.x /= (float)width;
            a.y /= (float)width;
            if (there) {
                T* to = dx + place(s, s.dx, r);
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    float f[E], u[E];
                    xv[j].to(f);
                    gv[j].to(u);
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float xh = (f[e] - st.x) * st.y;
                        f[e] = st.y * (u[e] * wf[j * E + e] - a.x - xh * a.y);
                    }
                    Pack<T, E> out;
                    out.from(f);
                    store_part(out, to, at[j], width);
                }
            }
        }
    }
    if (!part) return;
    unsigned p = g;
    if (L && L < 32 && merge) {           // the groups of a warp hold the same columns of the same head
#pragma unroll
        for (int o = L ? L : 32; o < 32; o *= 2)
#pragma unroll
            for (int i = 0; i < PER_LANE; i++) {
                dw[i] += __shfl_xor_sync(~0u, dw[i], o);
                db[i] += __shfl_xor_sync(~0u, db[i], o);
            }
        p = g * (L ? L : 1) / 32;
        if (threadIdx.x % 32 >= (L ? L : 1)) return;
    }
    float* to = part + 2ll * p * width;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = at[j] + e;
            if (c >= 0 && c < width) {
                to[c] = dw[j * E + e];
                to[width + c] = db[j * E + e];
            }
        }
}

// ---- rows that no block keeps in registers: read again for each step ---------------------------------------------------

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

template <class T, class P>
__global__ void layer_norm_fw_long(frnn_rows s, const T* __restrict__ x, const P* __restrict__ w, const P* __restrict__ b, float eps, T* __restrict__ y, float2* stats) {
    const unsigned r = blockIdx.x;
    const T* xr = x + place(s, s.x, r);
    const int64_t par = s.heads > 1 ? (r % s.n2) * s.width : 0;
    float sum = 0, sq = 0;
    for (int64_t d = threadIdx.x; d < s.width; d += blockDim.x) sum += to_float(xr[d]);
    const float mean = block_sum(sum) / (float)s.width;
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

template <class T, class P>
__global__ void layer_norm_dx_long(frnn_rows s, const T* __restrict__ dy, const T* __restrict__ x, const P* __restrict__ w, const float2* __restrict__ stats, T* __restrict__ dx) {
    const unsigned r = blockIdx.x;
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

// A thread sums a column of a head over the rows of a slab.
template <class T>
__global__ void layer_norm_dw_long(frnn_rows s, const T* __restrict__ dy, const T* __restrict__ x, const float2* __restrict__ stats, float* __restrict__ part, int slabs) {
    const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (d >= s.width) return;
    const unsigned head = blockIdx.y, heads = (unsigned)s.heads, rows = (unsigned)(s.n0 * s.n1 * s.n2);
    float dw = 0, db = 0;
    for (int64_t r = (int64_t)blockIdx.z * heads + head; r < rows; r += (int64_t)slabs * heads) {
        const float2 st = stats[r];
        const float g = to_float(dy[place(s, s.dy, (unsigned)r) + d]);
        dw += g * ((to_float(x[place(s, s.x, (unsigned)r) + d]) - st.x) * st.y);
        db += g;
    }
    float* to = part + 2 * ((int64_t)blockIdx.z * heads + head) * s.width;
    to[d] = dw;
    to[s.width + d] = db;
}

// Sum of the partial sums of a head: partials head, head + heads, ..., a warp takes every eighth of them.
template <class P>
__global__ void __launch_bounds__(BLOCK) layer_norm_join(const float* __restrict__ part, int partials, int heads, int width, P* __restrict__ dw, P* __restrict__ db) {
    __shared__ float share[BLOCK / 32][32];
    const int c = blockIdx.x * 32 + threadIdx.x % 32, slice = threadIdx.x / 32, head = blockIdx.y;
    P* to = blockIdx.z ? db : dw;
    if (!to) return;
    float sum = 0;
    if (c < width)
#pragma unroll 8
        for (int64_t p = head + (int64_t)slice * heads; p < partials; p += (int64_t)heads * (BLOCK / 32)) sum += part[(2 * p + blockIdx.z) * width + c];
    share[slice][threadIdx.x % 32] = sum;
    __syncthreads();
    if (slice || c >= width) return;
    for (int i = 1; i < BLOCK / 32; i++) sum += share[i][threadIdx.x];
    to[(int64_t)head * width + c] = from_float<P>(sum);
}

// ---- host ------------------------------------------------------------------------------------------------------------------

// Lanes of a group and how the rows are dealt out; nothing here depends on addresses, so the workspace's size can be asked
// for without them.  Rows that are no multiple of 16 bytes wide start up to 7 elements behind a boundary.
struct Plan {
    int lanes = 0, threads = 0, grid = 0;
    bool is_long = false;
    Deal deal{};
};

Plan plan_of(const frnn_rows& s, int threads_per_sm) {
    Plan p;
    const int64_t rows = s.n0 * s.n1 * s.n2, need = s.width % 8 ? s.width + 7 : s.width;
    if (need > PER_LANE * MOST_THREADS) {
        p.is_long = true;
        const int64_t each = rows / s.heads, slabs = each < 64 ? std::max<int64_t>(1, each) : 64;
        p.grid = (int)slabs;
        p.deal.groups = (unsigned)(slabs * s.heads);
        return p;
    }
    for (p.lanes = 2; p.lanes <= 32 && p.lanes * PER_LANE < need; p.lanes *= 2) {}
    if (p.lanes > 32) p.lanes = 0;
    p.threads = p.lanes ? BLOCK : (int)((need + PER_LANE * 32 - 1) / (PER_LANE * 32) * 32);
    const int64_t in_block = p.lanes ? BLOCK / p.lanes : 1, unit = std::lcm<int64_t>(s.heads, 8);
    const int64_t step = unit / std::gcd(unit, in_block);                 // blocks by which the number of groups stays a multiple of `unit`
    const int64_t full = (int64_t)sm_count() * std::max(1, threads_per_sm / p.threads), want = std::max<int64_t>(1, std::min((rows + in_block - 1) / in_block, full));
    const int64_t down = want / step * step;
    p.grid = (int)(down && (rows + in_block - 1) / in_block > full ? down : (want + step - 1) / step * step);
    p.deal.rows = (unsigned)rows;
    p.deal.groups = (unsigned)(p.grid * in_block);
    p.deal.rounds = (unsigned)((rows + p.deal.groups - 1) / p.deal.groups);
    return p;
}

// How a tensor's rows lie to 16-byte boundaries.
struct Lie {
    unsigned base, unit;          // address of the first row, distance from row to row, modulo 16 bytes
    bool even, same;              // one distance from row to row; all distances multiples of 16 bytes
};

Lie lie_of(const frnn_rows& s, const void* p, const int64_t* stride, size_t size) {
    const int64_t n[3] = {s.n0, s.n1, s.n2};
    int64_t run = 1, unit = 0;
    Lie l{(unsigned)((uintptr_t)p & 15), 0, true, true};
    for (int k = 2; k >= 0; k--) {
        if (n[k] == 1) continue;
        if (run == 1) unit = stride[k];
        else if (stride[k] != unit * run) l.even = false;
        if (stride[k] * (int64_t)size & 15) l.same = false;
        run *= n[k];
    }
    l.unit = (unsigned)(unit * (int64_t)size & 15);
    return l;
}

enum Access { ELEMENTS, WIDE_ALIKE, WIDE_APART };

// 16-byte accesses need rows of all tensors at the same distance behind a boundary.  WIDE_ALIKE: all rows at a boundary;
// WIDE_APART: evenly spaced rows, each group's at one distance (groups are dealt out in multiples of 8 rows).
Access access_of(const frnn_rows& s, const Lie* l, int count) {
    bool alike = s.width % 8 == 0, apart = s.width % 8 != 0;
    for (int i = 0; i < count; i++) {
        alike = alike && l[i].same && l[i].base == 0;
        apart = apart && l[i].even && l[i].base == l[0].base && l[i].unit == l[0].unit;
    }
    return alike ? WIDE_ALIKE : apart ? WIDE_APART : ELEMENTS;
}

int bad_shape(const char* what, const frnn_rows* s, int dtype, int param_dtype) {
    if (!s || !dtype_known(dtype) || !dtype_known(param_dtype)) return frnn_fail(FRNN_E_ARG, "%s: bad argument or unknown data type", what);
    if (param_dtype != dtype && param_dtype != FRNN_F32) return frnn_fail(FRNN_E_ARG, "%s: weights have the type of x or are fp32", what);
    if (s->n0 < 0 || s->n1 < 0 || s->n2 < 0 || s->width < 0 || s->heads < 1 || (s->heads > 1 && s->heads != s->n2)) return frnn_fail(FRNN_E_ARG, "%s: bad sizes", what);
    if ((s->n0 && s->n1 && s->n2) && (double)s->n0 * s->n1 * s->n2 >= 2147483648.0) return frnn_fail(FRNN_E_ARG, "%s: 2^31 rows or more", what);
    if (s->width >= (1ll << 30) || s->heads > 65535) return frnn_fail(FRNN_E_ARG, "%s: width has to be below 2^30, heads below 2^16", what);
    return FRNN_OK;
}

// Calls f(T(), P()) with the element type of x and that of the weights (the same, or fp32).
template <class F> int with_types(int dtype, int param_dtype, F f) {
    return with_dtype(dtype, [&](auto t) {
        if (param_dtype == FRNN_F32) return f(t, float());
        return f(t, t);
    });
}

// Calls f(integral_constant L, integral_constant E).
template <class T, class F> int with_lanes(int lanes, Access access, F f) {
    auto pick = [&](auto l) {
        if (access == ELEMENTS) return f(l, std::integral_constant<int, 1>());
        return f(l, std::integral_constant<int, WIDE<T>>());
    };
    switch (lanes) {
        case 2: return pick(std::integral_constant<int, 2>());
        case 4: return pick(std::integral_constant<int, 4>());
        case 8: return pick(std::integral_constant<int, 8>());
        case 16: return pick(std::integral_constant<int, 16>());
        case 32: return pick(std::integral_constant<int, 32>());
        default: return pick(std::integral_constant<int, 0>());
    }
}

enum { FW_THREADS_PER_SM = 1536, BW_THREADS_PER_SM = 768 };

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
    const cudaStream_t st = (cudaStream_t)stream;
    const Plan plan = plan_of(*s, FW_THREADS_PER_SM);
    const int64_t dense[3] = {s->n1 * s->n2 * s->width, s->n2 * s->width, s->width};
    const Lie lies[2] = {lie_of(*s, x, s->x, dtype_bytes(dtype)), lie_of(*s, y, dense, dtype_bytes(dtype))};
    return with_types(dtype, param_dtype, [&](auto t, auto p) {
        typedef decltype(t) T;
        typedef decltype(p) P;
        if (plan.is_long) {
            layer_norm_fw_long<T, P><<<(unsigned)rows, BLOCK, 0, st>>>(*s, (const T*)x, (const P*)weight, (const P*)bias, eps, (T*)y, (float2*)stats);
            return launched("frnn_layer_norm_forward");
        }
        return with_lanes<T>(plan.lanes, access_of(*s, lies, 2), [&](auto l, auto e) {
            layer_norm_fw<T, P, l.value, e.value><<<plan.grid, plan.threads, 0, st>>>(*s, plan.deal, (const T*)x, (const P*)weight, (const P*)bias, eps, (T*)y, (float2*)stats);
            return launched("frnn_layer_norm_forward");
        });
    });
}

size_t frnn_layer_norm_backward_workspace(const frnn_rows* s) {
    return s && s->heads >= 1 && s->width > 0 ? (size_t)plan_of(*s, BW_THREADS_PER_SM).deal.groups * 2 * s->width * 4 : 0;
}

int frnn_layer_norm_backward(const frnn_rows* s, int dtype, const void* dy, const void* x, int param_dtype, const void* weight, const float* stats, void* dx,
                             void* dweight, void* dbias, void* workspace, void* stream) {
    if (int rc = bad_shape("frnn_layer_norm_backward", s, dtype, param_dtype)) return rc;
    const int64_t rows = s->n0 * s->n1 * s->n2;
    if (s->width == 0) return FRNN_OK;
    const bool sums = dweight || dbias;
    if ((rows && (!dy || !x || !stats)) || (sums && !workspace)) return frnn_fail(FRNN_E_ARG, "frnn_layer_norm_backward: bad argument");
    if (!on_boundary(x, dtype_bytes(dtype)) || !on_boundary(dy, dtype_bytes(dtype)) || !on_boundary(dx, dtype_bytes(dtype)) || !on_boundary(weight, dtype_bytes(param_dtype)) ||
        !on_boundary(dweight, dtype_bytes(param_dtype)) || !on_boundary(dbias, dtype_bytes(param_dtype)) || !on_boundary(stats, 8) || !on_boundary(workspace, 16))
        return frnn_fail(FRNN_E_ARG, "frnn_layer_norm_backward: a pointer is not on a boundary of its elements (the statistics: of 8, the workspace: of 16 bytes)");
    const cudaStream_t st = (cudaStream_t)stream;
    const Plan plan = plan_of(*s, BW_THREADS_PER_SM);
    const size_t size = dtype_bytes(dtype);
    const Lie lies[3] = {lie_of(*s, x, s->x, size), lie_of(*s, dy, s->dy, size), lie_of(*s, dx, s->dx, size)};
    const Access access = access_of(*s, lies, dx ? 3 : 2);
    const bool merge = s->heads == 1 && access != WIDE_APART && plan.lanes && plan.lanes < 32;
    const int partials = (int)(rows == 0 ? 0 : merge ? plan.deal.groups * plan.lanes / 32 : plan.deal.groups);
    return with_types(dtype, param_dtype, [&](auto t, auto p) {
        typedef decltype(t) T;
        typedef decltype(p) P;
        int rc = FRNN_OK;
        if (rows && plan.is_long) {
            if (dx) {
                layer_norm_dx_long<T, P><<<(unsigned)rows, BLOCK, 0, st>>>(*s, (const T*)dy, (const T*)x, (const P*)weight, (const float2*)stats, (T*)dx);
                rc = launched("frnn_layer_norm_backward");
            }
            if (sums && !rc) {
                layer_norm_dw_long<T><<<dim3((unsigned)((s->width + 127) / 128), (unsigned)s->heads, plan.grid), 128, 0, st>>>(*s, (const T*)dy, (const T*)x, (const float2*)stats,
                                                                                                                              (float*)workspace, plan.grid);
                rc = launched("frnn_layer_norm_backward");
            }
        } else if (rows && (dx || sums)) {
            rc = with_lanes<T>(plan.lanes, access, [&](auto l, auto e) {
                layer_norm_bw<T, P, l.value, e.value><<<plan.grid, plan.threads, 0, st>>>(*s, plan.deal, (const T*)dy, (const T*)x, (const P*)weight, (const float2*)stats, (T*)dx,
                                                                                          sums ? (float*)workspace : nullptr, merge);
                return launched("frnn_layer_norm_backward");
            });
        }
        if (rc || !sums) return rc;
        layer_norm_join<P><<<dim3((unsigned)((s->width + 31) / 32), (unsigned)s->heads, 2), BLOCK, 0, st>>>((const float*)workspace, partials, (int)s->heads, (int)s->width, (P*)dweight,
                                                                                                          (P*)dbias);
        return launched("frnn_layer_norm_backward");
    });
}

}  // extern "C"
