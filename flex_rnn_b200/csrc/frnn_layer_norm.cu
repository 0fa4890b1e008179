// Layer norm over the last dimension, forward and backward, with weights for each column or for each head and column.
//
// Both directions are bound by memory: a pass over x (and dy) that keeps a row in registers between its reductions and its
// results, so each element is read and written once.  A row belongs to a group of lanes, 16 elements a lane: 2 to 256
// lanes up to 4096 columns, or a block of up to 512 threads up to 8192; longer rows are read again (``*_long``).
// A group walks over rows of one head, so its weights and the sums of its weight gradients stay in registers.  At the end
// each block (with weights for each head: each group) writes one partial sum to the workspace, and `layer_norm_join` adds
// those, all in a fixed order.  (Clusters that add theirs first through each other's shared memory gained nothing with 2
// blocks, 8192 x 4096 bf16 backward 55 us, and with 4 not all of them ran at once: 75 us.)
#include <algorithm>
#include <numeric>
#include <type_traits>

#include "frnn_lm.cuh"

using namespace frnn_lm;

namespace {

enum { PER_LANE = 16, BLOCK = 256, MOST_THREADS = 512 };
template <class T> constexpr int STAGES = sizeof(T) == 4 ? 3 : 4;      // rows under way in a ring: two blocks of 256 threads share an SM in the backward

// A row's place in a tensor: row r of `frnn_rows` is (r / (n1 n2), r / n2 mod n1, r mod n2).
__device__ __forceinline__ int64_t place(const frnn_rows& s, const int64_t* stride, unsigned r) {
    const unsigned n1 = (unsigned)s.n1, n2 = (unsigned)s.n2;
    if (n1 == 1 && n2 == 1) return r * stride[0];
    const unsigned q = r / n2, i2 = r - q * n2;
    if (n1 == 1) return q * stride[0] + i2 * stride[2];
    const unsigned i0 = q / n1, i1 = q - i0 * n1;
    return i0 * stride[0] + i1 * stride[1] + i2 * stride[2];
}

// How rows are dealt out: `groups` groups in all, group g takes rows g, g + groups, ... ; where that is more than one row,
// groups is a multiple of the number of heads (a group's rows have one head) and of 8 (its rows lie alike to 16-byte
// boundaries whatever the width), and, if that is not too many, of n2: a group's rows then are a fixed step apart.
struct Deal {
    unsigned rows, groups, rounds;
    int64_t x, dy, dx;          // steps
    bool even;                  // the steps hold
};

// The rows of a group in a tensor, one after the other: by steps for groups of lanes, for which a place's two divisions are dear
// (8192 x 4096 bf16: backward 53.7 us, by steps 43.3); groups that are whole blocks, whose registers are short, work each
// place out.
template <class T, bool STEPS> struct Walk {
    T *base, *now;
    __device__ __forceinline__ Walk(T* base, const frnn_rows& s, const int64_t* stride, unsigned r, unsigned rows) : base(base) {
        if (STEPS) now = base + (r < rows ? place(s, stride, r) : 0);
    }
    __device__ __forceinline__ T* at(const frnn_rows& s, const int64_t* stride, unsigned r) const { return STEPS ? now : base + place(s, stride, r); }
    // on to row r
    __device__ __forceinline__ void next(const frnn_rows& s, const int64_t* stride, const Deal& d, int64_t step, unsigned r) {
        if (!STEPS) return;
        if (d.even) now += step;
        else if (r < d.rows) now = base + place(s, stride, r);
    }
};

// How the rows of a call's tensors lie to 16-byte boundaries, and so how they are accessed.  WIDE_ALIKE: all rows at a
// boundary, in accesses of 16 bytes.  WIDE_APART: evenly spaced rows, those of a group at one distance behind a boundary
// in all tensors: accesses of 16 bytes but at the ends.  ELEMENTS: one element at a time.
enum Access { ELEMENTS, WIDE_ALIKE, WIDE_APART };

// The 16 columns of a lane: access j has E consecutive ones from at[j], of which those from 0 to width are there.
template <class T, Access A> struct Columns {
    static constexpr int E = A == ELEMENTS ? 1 : WIDE<T>, NV = PER_LANE / E;
    int at[NV], width;

    __device__ __forceinline__ Columns(int width, int lanes, int lane, int shift) : width(width) {
#pragma unroll
        for (int j = 0; j < NV; j++) at[j] = (j * lanes + lane) * E - shift;
    }
    // the whole of access j is there
    __device__ __forceinline__ bool whole(int j) const { return A == WIDE_APART ? at[j] >= 0 && at[j] + E <= width : at[j] < width; }
    __device__ __forceinline__ bool there(int j, int e) const { return A == WIDE_APART ? at[j] + e >= 0 && at[j] + e < width : at[j] < width; }
    // (single elements: nothing else is loaded without a ring)
    __device__ __forceinline__ void load(Pack<T, E>* v, const T* row) const {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (whole(j)) v[j].load(row + at[j]);
            else v[j].zero();
        }
    }
    // Row's accesses on their way; `begin`: the tensor's first element.  An access that begins before its row begins in the
    // row before (or the gap between them), one that ends behind it stops there; what is not the row's is cleared later.
    template <class R> __device__ __forceinline__ void copy(const R& ring, int first, const T* row, const T* begin) const {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (whole(j)) {
                ring.copy(first + j, row + at[j], 16);
            } else if (A == WIDE_APART && at[j] < width && at[j] > -E) {
                const int upto = min(E, width - at[j]);
                if (row + at[j] >= begin) ring.copy(first + j, row + at[j], upto * (int)sizeof(T));
                else
                    for (int e = max(0, -at[j]); e < upto; e++) ring.put(first + j, e, row[at[j] + e]);
            }
        }
    }
    template <class R> __device__ __forceinline__ void take(const R& ring, int first, float2* f) const {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            Pack<T, E> v;
            if (whole(j) || A == WIDE_APART) ring.take(first + j, v);
            else v.zero();
            v.to(&f[0].x + j * E);
        }
        if (A == WIDE_APART) clear(f);
    }
    __device__ __forceinline__ void store(T* row, const float2* f) const {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (A != WIDE_APART && !whole(j)) continue;
            Pack<T, E> v;
            v.from(&f[0].x + j * E);
            if (whole(j)) v.store(row + at[j]);
            else store_part(v, row, at[j], width);
        }
    }
    static __device__ __forceinline__ void unpack(const Pack<T, E>* v, float2* f) {
#pragma unroll
        for (int j = 0; j < NV; j++) v[j].to(&f[0].x + j * E);
    }
    // zeros where there is no column
    __device__ __forceinline__ void clear(float2* f) const {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (!whole(j))
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (!there(j, e)) (&f[0].x)[j * E + e] = 0;
    }
    template <class P> __device__ __forceinline__ void params(const P* p, float none, float2* f) const {
        constexpr int EP = WIDE<P> < E ? WIDE<P> : E;         // weights in 16-byte accesses where they are on a boundary, too
        const bool even = A == WIDE_ALIKE && p && ((uintptr_t)p & 15) == 0;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (even && whole(j)) {
#pragma unroll
                for (int k = 0; k < E; k += EP) {
                    Pack<P, EP> v;
                    v.load(p + at[j] + k);
                    v.to(&f[0].x + j * E + k);
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) (&f[0].x)[j * E + e] = p && there(j, e) ? to_float(p[at[j] + e]) : none;
            }
        }
    }
    __device__ __forceinline__ int count() const {
        int n = 0;
#pragma unroll
        for (int j = 0; j < NV; j++) n += max(0, min(at[j] + E, width) - max(at[j], 0));
        return n;
    }
};

// A lane's place: its group and its place in it.
template <int L> struct Seat {
    int lanes, lane, place;      // place: of the group in its block
    unsigned group, head;
    __device__ __forceinline__ Seat(const frnn_rows& s) {
        lanes = L ? L : blockDim.x;
        place = L ? threadIdx.x / (L ? L : 1) : 0;
        lane = L ? threadIdx.x % (L ? L : 1) : threadIdx.x;
        group = blockIdx.x * (L ? BLOCK / (L ? L : 1) : 1) + place;
        head = s.heads > 1 ? group % (unsigned)s.heads : 0;
    }
};

// Rows on their way to a thread, a few rounds ahead: each thread has slots of its own in shared memory for its accesses,
// filled by asynchronous copies, so no registers and no barriers are spent on them.  (With the next row in registers 32 KB
// an SM were under way, and the warps waited for loads 3.9 cycles an instruction; with the ring 0.4.)
template <class T, int N, int ROUNDS> struct Ring {
    static constexpr int E = WIDE<T>;
    char* slot;                  // this thread's first 16 bytes; its next ones follow at distances of 16 bytes a thread
    int stage = 0;
    __device__ __forceinline__ Ring(char* shared) : slot(shared + 16 * threadIdx.x) {}
    __device__ __forceinline__ char* place(int i) const { return slot + 16 * (stage * N + i) * blockDim.x; }
    // the first `bytes` of 16, and zeros behind them
    __device__ __forceinline__ void copy(int i, const T* from, int bytes) const {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(place(i))), "l"(from), "r"(bytes) : "memory");
    }
    __device__ __forceinline__ void put(int i, int e, T x) const { ((T*)place(i))[e] = x; }
    __device__ __forceinline__ void commit() {
        asm volatile("cp.async.commit_group;" ::: "memory");
        stage = stage + 1 == ROUNDS ? 0 : stage + 1;
    }
    // the oldest round is there
    __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(ROUNDS - 1) : "memory"); }
    __device__ __forceinline__ void take(int i, Pack<T, E>& v) const { v.load((const T*)place(i)); }
};

template <int L> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = L && L < 32 ? L / 2 : 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// A float2 of each warp of a group of several warps (a block, L = 0, or L lanes), seen by all its threads; two buffers by
// turns, so one barrier of the group each time is enough.
template <int L> struct Exchange {
    float2 (*buffer)[MOST_THREADS / 32];
    int turn = 0;
    static __device__ __forceinline__ int first() { return L ? threadIdx.x / (L ? L : 1) * (L / 32) : 0; }      // the group's first warp
    template <class F> __device__ __forceinline__ void operator()(float2 mine, F each) {
        if ((threadIdx.x & 31) == 0) buffer[turn][threadIdx.x / 32] = mine;
        if (L) asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.x / (L ? L : 1)), "n"(L ? L : 32) : "memory");
        else __syncthreads();
        turn ^= 1;
        again(each);
    }
    // the last ones once more
    template <class F> __device__ __forceinline__ void again(F each) const {
        const float4* all = (const float4*)(buffer[turn ^ 1] + first());
        const int warps = L ? L / 32 : blockDim.x / 32;
#pragma unroll
        for (int i = 0; i < (L ? L : MOST_THREADS) / 64; i++) {
            if (2 * i >= warps) break;
            const float4 v = all[i];
            each(2 * i, make_float2(v.x, v.y));
            if (2 * i + 1 < warps) each(2 * i + 1, make_float2(v.z, v.w));
        }
    }
};

// y = (x - mean) rstd w + b.  The variance is that of the centred values, so that a large mean costs no digits; warps of a
// block each centre theirs and join: sum of squares = sum over warps of theirs + count (their mean - mean)^2.
// 8192 x 4096 bf16: 31 us (4.4 TB/s; the floor is 21), 262144 x 128: 25 us.  It is bound by its instructions, 12 to 18 an
// element (the issue slots are 60 % busy): conversions, the two passes over a row, and what a row costs a thread whatever
// its elements (shuffles, addresses, the exchange).  A warp for each row of 4096 had half the instructions and eight
// warps an SM: 37 us; 32 elements a lane, weights from the L1 cache: 41.
template <class T, class P, int L, Access A>
__global__ void __launch_bounds__(L ? BLOCK : MOST_THREADS, L ? 2 : 1) layer_norm_fw(frnn_rows s, Deal deal, const T* __restrict__ x, const P* __restrict__ w, const P* __restrict__ b, float eps,
                                                                         T* __restrict__ y, float2* __restrict__ stats) {
    typedef Columns<T, A> C;
    __shared__ __align__(16) float2 buffer[2][MOST_THREADS / 32];
    __shared__ float counts[MOST_THREADS / 32];
    const Seat<L> seat(s);
    const unsigned g = seat.group;
    const int width = (int)s.width;
    const int shift = A == WIDE_APART ? (int)((uintptr_t)(x + (g < deal.rows ? place(s, s.x, g) : 0)) & 15) / (int)sizeof(T) : 0;
    const C cols(width, seat.lanes, seat.lane, shift);
    Exchange<L> exchange{buffer};
    constexpr bool CROSS = L == 0 || L > 32;               // a group is several warps
    float2 wf[PER_LANE / 2], bf[PER_LANE / 2], f[PER_LANE / 2];
    cols.params(w ? w + (int64_t)seat.head * width : w, 1.f, wf);
    cols.params(b ? b + (int64_t)seat.head * width : b, 0.f, bf);
    const float per_row = 1.f / (float)width;
    float per_warp = 0;
    if (CROSS) {
        const float mine = lanes_sum<0>((float)cols.count());
        per_warp = mine > 0 ? 1.f / mine : 0.f;
        if (seat.lane % 32 == 0) counts[threadIdx.x / 32] = mine;      // (seen by the group after the first exchange's barrier)
    }
    constexpr bool RING = A != ELEMENTS;
    extern __shared__ __align__(16) char shared[];
    Pack<T, C::E> next[C::NV];
    Ring<T, RING ? C::NV : 0, RING ? STAGES<T> : 1> ring(shared);
    // rows are on their way AHEAD rounds before they are used
    Walk<const T, (L > 0)> wx(x, s, s.x, g, deal.rows);
    unsigned left = g < deal.rows ? (deal.rows - g + deal.groups - 1) / deal.groups : 0;      // rows that are still to be fetched
    auto fetch = [&](unsigned r) {
        if (left) {
            const T* px = wx.at(s, s.x, r);
            if constexpr (RING) cols.copy(ring, 0, px, x);
            else cols.load(next, px);
            left--;
            wx.next(s, s.x, deal, deal.x, r + deal.groups);
        }
        if constexpr (RING) ring.commit();
    };
    constexpr int AHEAD = RING ? STAGES<T> : 1;
#pragma unroll
    for (int i = 0; i < AHEAD; i++) fetch(g + i * deal.groups);
    for (unsigned i = 0; i < deal.rounds; i++) {
        const unsigned r = i * deal.groups + g;
        const bool there = r < deal.rows;
        if constexpr (RING) {
            ring.wait();
            cols.take(ring, 0, f);
        } else {
            C::unpack(next, f);
        }
        fetch(r + AHEAD * deal.groups);
        float2 t = f[0];
#pragma unroll
        for (int k = 1; k < PER_LANE / 2; k++) t = add2(t, f[k]);
        const float sum = lanes_sum<L>(t.x + t.y);
        float mean = sum * (CROSS ? per_warp : per_row);
#pragma unroll
        for (int k = 0; k < PER_LANE / 2; k++) f[k] = add2(f[k], both(-mean));
        cols.clear(f);
        t = mul2(f[0], f[0]);
#pragma unroll
        for (int k = 1; k < PER_LANE / 2; k++) t = fma2(f[k], f[k], t);
        float sq = lanes_sum<L>(t.x + t.y);
        if (CROSS) {
            const float own = mean;
            float2 t = both(0.f);
            exchange(make_float2(own, sq), [&](int k, float2 v) { t = fma2(v, make_float2(counts[exchange.first() + k], 1.f), t); });
            mean = t.x * per_row;
            sq = t.y;
            exchange.again([&](int k, float2 v) {
                const float d = v.x - mean;
                sq = fmaf(counts[exchange.first() + k] * d, d, sq);
            });
            const float2 move = both(own - mean);
#pragma unroll
            for (int k = 0; k < PER_LANE / 2; k++) f[k] = add2(f[k], move);
        }
        const float rstd = rsqrtf(sq * per_row + eps);
        if (!there) continue;
        if (stats && seat.lane == 0) stats[r] = make_float2(mean, rstd);
#pragma unroll
        for (int k = 0; k < PER_LANE / 2; k++) f[k] = fma2(mul2(f[k], both(rstd)), wf[k], bf[k]);
        cols.store(y + (int64_t)r * width, f);
    }
}

// dx = rstd (g - mean(g) - xh mean(g xh)) with g = dy w, xh = (x - mean) rstd; sums over the group's rows of dy xh and dy.
// 8192 x 4096 bf16: 42 us with the weights' gradients, 37 without (5.4 TB/s; the floor is 31); 262144 x 128 with weights for
// each of 32 heads: 45 and 37.  16 warps an SM, whose registers hold weights and both sums; bound by instructions as above.
// part: [blocks][2][pitch] where blocks have several groups of one head, else [groups][2][pitch], pitch the next multiple
// of 4 of the width; may be NULL, and so may dx.
template <class T, class P, int L, Access A>
__global__ void __launch_bounds__(L ? BLOCK : MOST_THREADS, L ? 2 : 1) layer_norm_bw(frnn_rows s, Deal deal, const T* __restrict__ dy, const T* __restrict__ x, const P* __restrict__ w,
                                                                         const float2* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part) {
    typedef Columns<T, A> C;
    __shared__ __align__(16) float2 buffer[2][MOST_THREADS / 32];
    const Seat<L> seat(s);
    const unsigned g = seat.group;
    const int width = (int)s.width;
    const int shift = A == WIDE_APART ? (int)((uintptr_t)(x + (g < deal.rows ? place(s, s.x, g) : 0)) & 15) / (int)sizeof(T) : 0;
    const C cols(width, seat.lanes, seat.lane, shift);
    Exchange<L> exchange{buffer};
    constexpr bool CROSS = L == 0 || L > 32;               // a group is several warps
    cudaTriggerProgrammaticLaunchCompletion();
    float2 wf[PER_LANE / 2], dw[PER_LANE / 2], db[PER_LANE / 2], f[PER_LANE / 2], u[PER_LANE / 2];
    cols.params(w ? w + (int64_t)seat.head * width : w, 1.f, wf);
    const float per_row = 1.f / (float)width;
#pragma unroll
    for (int k = 0; k < PER_LANE / 2; k++) dw[k] = db[k] = both(0.f);
    constexpr bool RING = A != ELEMENTS;
    extern __shared__ __align__(16) char shared[];
    Pack<T, C::E> xn[C::NV], gn[C::NV];
    Ring<T, RING ? 2 * C::NV : 0, RING ? STAGES<T> : 1> ring(shared);
    float2 sn = both(0.f);
#pragma unroll
    for (int j = 0; j < C::NV; j++) { xn[j].zero(); gn[j].zero(); }
    Walk<const T, (L > 0)> wx(x, s, s.x, g, deal.rows), wg(dy, s, s.dy, g, deal.rows);
    Walk<T, (L > 0)> wd(dx, s, s.dx, g, deal.rows);
    unsigned left = g < deal.rows ? (deal.rows - g + deal.groups - 1) / deal.groups : 0;      // rows that are still to be fetched
    auto fetch = [&](unsigned r) {
        if (left) {
            const T *px = wx.at(s, s.x, r), *pg = wg.at(s, s.dy, r);
            if constexpr (RING) {
                cols.copy(ring, 0, px, x);
                cols.copy(ring, C::NV, pg, dy);
            } else {
                cols.load(xn, px);
                cols.load(gn, pg);
            }
            left--;
            wx.next(s, s.x, deal, deal.x, r + deal.groups);
            wg.next(s, s.dy, deal, deal.dy, r + deal.groups);
        }
        if constexpr (RING) ring.commit();
    };
    constexpr int AHEAD = RING ? STAGES<T> : 1;
    if (g < deal.rows) sn = stats[g];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) fetch(g + i * deal.groups);
    for (unsigned i = 0; i < deal.rounds; i++) {
        const unsigned r = i * deal.groups + g;
        const bool there = r < deal.rows;
        const float2 st = sn;
        if constexpr (RING) {
            ring.wait();
            cols.take(ring, 0, f);
            cols.take(ring, C::NV, u);
        } else {
            C::unpack(xn, f);
            C::unpack(gn, u);
        }
        if (there && deal.rows - r > deal.groups) sn = stats[r + deal.groups];
        fetch(r + AHEAD * deal.groups);
        float2 a = both(0.f), c = both(0.f);
        if (there) {
#pragma unroll
            for (int k = 0; k < PER_LANE / 2; k++) {
                f[k] = mul2(add2(f[k], both(-st.x)), both(st.y));
                dw[k] = fma2(u[k], f[k], dw[k]);           // u = 0 where there is no column
                db[k] = add2(db[k], u[k]);
                u[k] = mul2(u[k], wf[k]);
                a = add2(a, u[k]);
                c = fma2(u[k], f[k], c);
            }
        }
        if (!dx) continue;
        float ma = lanes_sum<L>(a.x + a.y), mc = lanes_sum<L>(c.x + c.y);
        if (CROSS) {
            float2 t = both(0.f);
            exchange(make_float2(ma, mc), [&](int, float2 v) { t = add2(t, v); });
            ma = t.x;
            mc = t.y;
        }
        if (!there) continue;
        const float2 off = both(-st.y * (ma * per_row)), by = both(-st.y * (mc * per_row));
#pragma unroll
        for (int k = 0; k < PER_LANE / 2; k++) f[k] = fma2(f[k], by, fma2(u[k], both(st.y), off));
        cols.store(wd.at(s, s.dx, r), f);
        wd.next(s, s.dx, deal, deal.dx, r + deal.groups);
    }
    if (!part) return;
    const int pitch = (width + 3) & ~3;
    // by way of shared memory where groups of a block have one head (their sums are added there), and where columns are not
    // in runs of 16 bytes (single ones would be written 32 bytes apart)
    int places = L ? BLOCK / (L ? L : 1) : 1;
    const bool merged = L && s.heads == 1;
    const bool staged = merged || A != WIDE_ALIKE;
    float* to = part + 2ll * g * pitch;
    bool write = true;
    if (staged) {
        int place = seat.place;
        if constexpr (L && L < 32 && A != WIDE_APART) {
            if (merged) {                                  // the groups of a warp hold the same columns
#pragma unroll
                for (int o = L; o < 32; o *= 2)
#pragma unroll
                    for (int k = 0; k < PER_LANE / 2; k++) {
                        dw[k] = add2(dw[k], make_float2(__shfl_xor_sync(~0u, dw[k].x, o), __shfl_xor_sync(~0u, dw[k].y, o)));
                        db[k] = add2(db[k], make_float2(__shfl_xor_sync(~0u, db[k].x, o), __shfl_xor_sync(~0u, db[k].y, o)));
                    }
                place = threadIdx.x / 32;
                places = BLOCK / 32;
                write = threadIdx.x % 32 < L;
            }
        }
        __syncthreads();                                   // the rows' shared memory takes the sums
        to = (float*)shared + 2 * place * pitch;
    }
    if (write)
#pragma unroll
        for (int j = 0; j < C::NV; j++) {
            const float *pw = &dw[0].x + j * C::E, *pb = &db[0].x + j * C::E;
            if constexpr (A == WIDE_ALIKE) {               // (widths of multiples of 8)
                if (cols.whole(j))
#pragma unroll
                    for (int e = 0; e < C::E; e += 4) {
                        *(float4*)(to + cols.at[j] + e) = make_float4(pw[e], pw[e + 1], pw[e + 2], pw[e + 3]);
                        *(float4*)(to + pitch + cols.at[j] + e) = make_float4(pb[e], pb[e + 1], pb[e + 2], pb[e + 3]);
                    }
            } else {
#pragma unroll
                for (int e = 0; e < C::E; e++)
                    if (cols.there(j, e)) {
                        to[cols.at[j] + e] = pw[e];
                        to[pitch + cols.at[j] + e] = pb[e];
                    }
            }
        }
    if (!staged) return;
    __syncthreads();
    if (merged) {
        for (int i = threadIdx.x; i < 2 * pitch; i += blockDim.x) {
            float sum = 0;
#pragma unroll 8
            for (int k = 0; k < places; k++) sum += ((const float*)shared)[2 * k * pitch + i];
            part[2ll * blockIdx.x * pitch + i] = sum;
        }
    } else {
        float4* out = (float4*)(part + 2ll * blockIdx.x * places * pitch);
        for (int i = threadIdx.x; i < places * pitch / 2; i += blockDim.x) out[i] = ((const float4*)shared)[i];
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
    const int64_t pitch = (s.width + 3) & ~3ll;
    float* to = part + 2 * ((int64_t)blockIdx.z * heads + head) * pitch;
    to[d] = dw;
    to[pitch + d] = db;
}

// Sum of the partial sums of a head (partials head, head + heads, ...): 8 lanes have 4 columns each, 32 slices of the
// partials are summed side by side, so that few loads wait for one another: 3 to 4 us behind the backward, 10 MB of partials.
template <class P>
__global__ void __launch_bounds__(BLOCK) layer_norm_join(const float* __restrict__ part, int partials, int heads, int width, P* __restrict__ dw, P* __restrict__ db) {
    constexpr int LANES = 8, SLICES = BLOCK / LANES;
    __shared__ float4 share[SLICES][LANES];
    const int lane = threadIdx.x % LANES, slice = threadIdx.x / LANES, head = blockIdx.y, c = (blockIdx.x * LANES + lane) * 4, pitch = (width + 3) & ~3;
    P* to = blockIdx.z ? db : dw;
    cudaGridDependencySynchronize();
    if (!to) return;
    float4 sum = make_float4(0, 0, 0, 0);
    if (c < width)
#pragma unroll 8
        for (int64_t p = head + (int64_t)slice * heads; p < partials; p += (int64_t)heads * SLICES) {
            const float4 v = *(const float4*)(part + (2 * p + blockIdx.z) * pitch + c);      // (columns behind the width are read and dropped)
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
    share[slice][lane] = sum;
    __syncthreads();
    const int i = threadIdx.x, col = blockIdx.x * LANES * 4 + i;
    if (i >= LANES * 4 || col >= width) return;
    float total = 0;
#pragma unroll
    for (int k = 0; k < SLICES; k++) total += ((const float*)share[k])[i];
    to[(int64_t)head * width + col] = from_float<P>(total);
}

// ---- host ------------------------------------------------------------------------------------------------------------------

// Lanes of a group and how the rows are dealt out; nothing here depends on addresses, so the workspace's size can be asked
// for without them.  Rows that are no multiple of 16 bytes wide start up to 7 elements behind a boundary.
struct Plan {
    int lanes = 0, threads = 0, grid = 0;
    bool is_long = false;
    bool merged = false;       // partial sums of weight gradients: one for a block, or one for a group
    Deal deal{};
    int64_t partials() const { return merged ? grid : deal.groups; }
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
    for (p.lanes = 2; p.lanes <= BLOCK && p.lanes * PER_LANE < need; p.lanes *= 2) {}
    // a block of just the threads that a wide row needs where a group of a power of two would leave many without columns
    if (p.lanes > BLOCK || (p.lanes > 64 && 5 * need < 4 * p.lanes * PER_LANE)) p.lanes = 0;
    p.threads = p.lanes ? BLOCK : (int)((need + PER_LANE * 32 - 1) / (PER_LANE * 32) * 32);
    const int64_t in_block = p.lanes ? BLOCK / p.lanes : 1;
    const int64_t blocks = (rows + in_block - 1) / in_block, full = (int64_t)sm_count() * std::max(1, threads_per_sm / p.threads);
    auto blocks_by = [&](int64_t unit) { return unit / std::gcd(unit, in_block); };      // by which the number of groups stays a multiple of `unit`
    const int64_t unit = std::lcm<int64_t>(s.heads, 8), with_n2 = blocks_by(std::lcm<int64_t>(unit, std::max<int64_t>(1, s.n2)));
    const int64_t by = p.lanes && s.n2 <= 128 && with_n2 <= full ? with_n2 : blocks_by(unit);
    p.merged = p.lanes && s.heads == 1;
    // A group for each row where they all fit: any number of groups does then.  (Rounded up to `by`, n2 = 127 rows of 4096 had
    // 1016 groups and 33 MB of partial sums: their backward took 21 us, it takes 7.)
    p.grid = (int)(blocks <= std::max(full, by) ? std::max<int64_t>(1, blocks) : std::max(full / by, (int64_t)1) * by);
    p.deal.rows = (unsigned)rows;
    p.deal.groups = (unsigned)(p.grid * in_block);
    p.deal.rounds = (unsigned)((rows + p.deal.groups - 1) / p.deal.groups);
    // rows (i0, i1, i2) and `groups` rows on: the same i2, and i1 further on by a fixed number as long as there is no i0
    const int64_t down1 = p.deal.groups / std::max<int64_t>(1, s.n2);
    p.deal.even = s.n1 * s.n2 == 1 || (s.n0 == 1 && p.deal.groups % std::max<int64_t>(1, s.n2) == 0);
    auto step = [&](const int64_t* stride) { return s.n1 * s.n2 == 1 ? p.deal.groups * stride[0] : down1 * stride[1]; };
    p.deal.x = step(s.x);
    p.deal.dy = step(s.dy);
    p.deal.dx = step(s.dx);
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

// Calls f(integral_constant L, integral_constant A).
template <class F> int with_lanes(int lanes, Access access, F f) {
    auto pick = [&](auto l) {
        if (access == ELEMENTS) return f(l, std::integral_constant<Access, ELEMENTS>());
        if (access == WIDE_ALIKE) return f(l, std::integral_constant<Access, WIDE_ALIKE>());
        return f(l, std::integral_constant<Access, WIDE_APART>());
    };
    switch (lanes) {
        case 2: return pick(std::integral_constant<int, 2>());
        case 4: return pick(std::integral_constant<int, 4>());
        case 8: return pick(std::integral_constant<int, 8>());
        case 16: return pick(std::integral_constant<int, 16>());
        case 32: return pick(std::integral_constant<int, 32>());
        case 64: return pick(std::integral_constant<int, 64>());
        case 128: return pick(std::integral_constant<int, 128>());
        case 256: return pick(std::integral_constant<int, 256>());
        default: return pick(std::integral_constant<int, 0>());
    }
}

enum { FW_THREADS_PER_SM = 512, BW_THREADS_PER_SM = 512 };

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
        const Access access = access_of(*s, lies, 2);
        return with_lanes(plan.lanes, access, [&](auto l, auto a) {
            const size_t shared = a.value != ELEMENTS ? (size_t)plan.threads * (PER_LANE / WIDE<T>) * STAGES<T> * 16 : 0;
            if (!allow_shared<layer_norm_fw<T, P, l.value, a.value>>(shared)) return launched("frnn_layer_norm_forward");
            return launch("frnn_layer_norm_forward", layer_norm_fw<T, P, l.value, a.value>, dim3(plan.grid), plan.threads, shared, st, false, 1, *s, plan.deal, (const T*)x,
                          (const P*)weight, (const P*)bias, eps, (T*)y, (float2*)stats);
        });
    });
}

size_t frnn_layer_norm_backward_workspace(const frnn_rows* s) {
    return s && s->heads >= 1 && s->width > 0 ? (size_t)plan_of(*s, BW_THREADS_PER_SM).partials() * 2 * ((s->width + 3) & ~3ll) * 4 : 0;
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
    const int partials = rows ? (int)plan.partials() : 0;
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
            rc = with_lanes(plan.lanes, access, [&](auto l, auto a) {
                const size_t ring = a.value != ELEMENTS ? (size_t)plan.threads * 2 * (PER_LANE / WIDE<T>) * STAGES<T> * 16 : 0;
                const size_t shared = std::max(ring, sums && (plan.merged || a.value != WIDE_ALIKE) ? (size_t)plan.threads * (PER_LANE + 2) * 2 * 4 : 0);      // (pitch: up to 3 floats more than a group's columns)
                if (!allow_shared<layer_norm_bw<T, P, l.value, a.value>>(shared)) return launched("frnn_layer_norm_backward");
                return launch("frnn_layer_norm_backward", layer_norm_bw<T, P, l.value, a.value>, dim3(plan.grid), plan.threads, shared, st, false, 1, *s, plan.deal, (const T*)dy,
                              (const T*)x, (const P*)weight, (const float2*)stats, (T*)dx, sums ? (float*)workspace : (float*)nullptr);
            });
        }
        if (rc || !sums) return rc;
        return launch("frnn_layer_norm_backward", layer_norm_join<P>, dim3((unsigned)((s->width + 31) / 32), (unsigned)s->heads, 2), BLOCK, 0, st, rows > 0, 1, (const float*)workspace, partials,
                      (int)s->heads, (int)s->width, (P*)dweight, (P*)dbias);
    });
}

}  // extern "C"
