// Rotary positions: pairs (u, w) of each head's first 2 * pairs values turned by position * frequency, the rest copied.
//
//   u' = scale (u cos - w sin),  w' = scale (u sin + w cos);   the gradient is the turn back, scaled the same
//
// Bound by memory: x once, y once.  A warp has a place (of a batch and a position) and some or all of its heads.  Its lanes compute
// the place's sines and cosines once, each a few, into a table in shared memory; a lane then keeps those of its E pairs in
// registers for all heads that it passes, U of them at a time, whose loads are under way together and before the table is made.
// Angles: position * frequency in 64 bits, taken modulo a turn there (a position of 10^6 at frequency 1 is 1.6 10^5 turns: in 32 bits
// 2 % of a turn would be lost), then sine and cosine of the rest in 32 bits, corrected by what its rounding took off: fp32 results are within 4.5e-8 of
// 64 bits in norm, without the correction 5.7e-8.  (Sines and cosines in 64 bits: 8 % less, but 1.3 % slower where a place has few heads' pairs to hide them.)
#include <algorithm>

#include "frnn_lm.cuh"

using namespace frnn_lm;

namespace {

struct RotaryArgs {
    const void *x, *positions, *frequencies;
    void* y;
    int64_t length, heads, width, pairs, start;
    int64_t x_stride[3], y_stride[3], p_stride[2];
    int64_t warps, per_place, heads_each;      // warps in all, warps to a place, heads to a warp
    int position_bytes, frequency_bytes, lanes;      // lanes: of a head, a power of two
    float scale, direction;
};

template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef unsigned type; };
template <> struct Raw<2> { typedef unsigned short type; };

template <class T, int E> __device__ __forceinline__ void load_few(const T* p, T* v) {
    const typename Raw<E * (int)sizeof(T)>::type r = *(const typename Raw<E * (int)sizeof(T)>::type*)p;
    memcpy(v, &r, sizeof r);
}
template <class T, int E> __device__ __forceinline__ void store_few(T* p, const T* v) {
    typename Raw<E * (int)sizeof(T)>::type r;
    memcpy(&r, v, sizeof r);
    *(typename Raw<E * (int)sizeof(T)>::type*)p = r;
}

__device__ __forceinline__ void turn(double position, double frequency, float scale, float direction, float& c, float& s) {
    const double angle = position * frequency, whole = rint(angle * 0.15915494309189535);
    // (1 / (2 pi) as the sum of two numbers of 64 bits)
    const double rest = fma(angle, -9.839338337591243e-18, fma(angle, 0.15915494309189535, -whole));
    const float near = (float)rest, off = 6.2831853f * (float)(rest - near);
    float c0, s0;
    sincospif(2.f * near, &s0, &c0);
    c = fmaf(-off, s0, c0) * scale;
    s = fmaf(off, c0, s0) * (scale * direction);
}

template <class T, int E, bool INTERLEAVED> __global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    constexpr int U = E >= 4 ? 4 : 8;
    __shared__ float2 tables[8][32 * E];
    const int lane = threadIdx.x % 32, in_head = lane % a.lanes, heads_at_once = 32 / a.lanes;
    const int64_t warp = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
    if (warp >= a.warps) return;
    float2* const table = tables[threadIdx.x / 32];
    const int64_t place = warp / a.per_place, b = place / a.length, t = place % a.length;
    const int64_t first = warp % a.per_place * a.heads_each, last = min(a.heads, first + a.heads_each);
    const T* const x = (const T*)a.x + b * a.x_stride[0] + t * a.x_stride[1];
    T* const y = (T*)a.y + b * a.y_stride[0] + t * a.y_stride[1];
    const double position = a.positions ? (double)token_at(a.positions, a.position_bytes, b * a.p_stride[0] + t * a.p_stride[1]) : (double)(a.start + t);
    const int items = (int)(a.pairs / E);
    for (int i0 = 0; i0 < items; i0 += a.lanes) {
        const int i = i0 + in_head;
        const bool mine = i < items;
        const int64_t u = INTERLEAVED ? 2 * E * i : E * i, w = INTERLEAVED ? 2 * E * i + E : a.pairs + E * i;
        T p[U][E], q[U][E];
        auto fetch = [&](int64_t h) {
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int64_t at = h + k * heads_at_once;
                if (mine && at < last) {
                    load_few<T, E>(x + at * a.x_stride[2] + u, p[k]);
                    load_few<T, E>(x + at * a.x_stride[2] + w, q[k]);
                }
            }
        };
        int64_t h = first + lane / a.lanes;
        fetch(h);
        __syncwarp();                     // (the table of the pairs before these has been read)
        for (int k = lane; k < min(a.lanes, items - i0) * E; k += 32) {
            const int pair = i0 * E + k;
            turn(position, a.frequency_bytes == 8 ? ((const double*)a.frequencies)[pair] : (double)((const float*)a.frequencies)[pair], a.scale, a.direction, table[k].x, table[k].y);
        }
        __syncwarp();
        float c[E], s[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float2 z = mine ? table[in_head * E + e] : make_float2(0.f, 0.f);
            c[e] = z.x;
            s[e] = z.y;
        }
        while (h < last) {
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int64_t at = h + k * heads_at_once;
                if (!mine || at >= last) continue;
                auto rotate = [&](T& p0, T& q0, float c0, float s0) {
                    const float f = to_float(p0), g = to_float(q0);
                    p0 = from_float<T>(f * c0 - g * s0);
                    q0 = from_float<T>(f * s0 + g * c0);
                };
                if constexpr (INTERLEAVED && E > 1) {      // E pairs lie in a row, half of them in p
#pragma unroll
                    for (int e = 0; e < E / 2; e++) {
                        rotate(p[k][2 * e], p[k][2 * e + 1], c[e], s[e]);
                        rotate(q[k][2 * e], q[k][2 * e + 1], c[E / 2 + e], s[E / 2 + e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++) rotate(p[k][e], q[k][e], c[e], s[e]);
                }
                store_few<T, E>(y + at * a.y_stride[2] + u, p[k]);
                store_few<T, E>(y + at * a.y_stride[2] + w, q[k]);
            }
            h += U * heads_at_once;
            if (h < last) fetch(h);
        }
    }
    const int rest = (int)((a.width - 2 * a.pairs) / E);
    for (int i = in_head; i < rest; i += a.lanes)
        for (int64_t h = first + lane / a.lanes; h < last; h += U * heads_at_once) {
            T p[U][E];
#pragma unroll
            for (int k = 0; k < U; k++)
                if (h + k * heads_at_once < last) load_few<T, E>(x + (h + k * heads_at_once) * a.x_stride[2] + 2 * a.pairs + E * i, p[k]);
#pragma unroll
            for (int k = 0; k < U; k++)
                if (h + k * heads_at_once < last) store_few<T, E>(y + (h + k * heads_at_once) * a.y_stride[2] + 2 * a.pairs + E * i, p[k]);
        }
}

template <class T, int E> int run(const RotaryArgs& a, bool interleaved, cudaStream_t stream) {
    const int64_t blocks = (a.warps + 7) / 8;
    if (interleaved) rotary_kernel<T, E, true><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else rotary_kernel<T, E, false><<<(unsigned)blocks, 256, 0, stream>>>(a);
    return launched("rotary");
}

}  // namespace

extern "C" int frnn_rotary(const frnn_rotary_call* c, const void* x, const void* positions, const void* frequencies, void* y, void* stream) {
    if (!c || !dtype_known(c->dtype) || (positions && c->position_bytes != 4 && c->position_bytes != 8) || (c->frequency_bytes != 4 && c->frequency_bytes != 8))
        return frnn_fail(FRNN_E_ARG, "rotary: bad argument");
    const int64_t most = 1ll << 31;
    if (c->batch < 0 || c->length < 0 || c->heads < 0 || c->width < 0 || c->pairs < 0 || c->batch >= most || c->length >= most || c->heads >= most || c->width >= most || 2 * c->pairs > c->width)
        return frnn_fail(FRNN_E_ARG, "rotary: bad sizes");
    if (!c->batch || !c->length || !c->heads || !c->width) return FRNN_OK;
    const size_t e = dtype_bytes(c->dtype);
    if (!x || !y || (c->pairs && !frequencies) || !on_boundary(x, e) || !on_boundary(y, e) || (positions && !on_boundary(positions, c->position_bytes)) || !on_boundary(frequencies, c->frequency_bytes))
        return frnn_fail(FRNN_E_ARG, "rotary: bad pointer");
    RotaryArgs a = {};
    a.x = x;
    a.y = y;
    a.positions = positions;
    a.frequencies = frequencies;
    a.length = c->length;
    a.heads = c->heads;
    a.width = c->width;
    a.pairs = c->pairs;
    a.start = c->start;
    a.position_bytes = c->position_bytes;
    a.frequency_bytes = c->frequency_bytes;
    a.scale = c->scale;
    a.direction = c->inverse ? -1.f : 1.f;
    // the widest access that everything it has to divide allows
    int64_t odd = c->pairs | c->width | (int64_t)((uintptr_t)x / e) | (int64_t)((uintptr_t)y / e);
    for (int i = 0; i < 3; i++) {
        a.x_stride[i] = c->x_stride[i];
        a.y_stride[i] = c->y_stride[i];
        odd |= c->x_stride[i] | c->y_stride[i];
        if (i < 2) a.p_stride[i] = c->position_stride[i];
    }
    const int widest = 16 / (int)e, each = (int)std::min<int64_t>(widest, odd & -odd);
    const int64_t items = std::max<int64_t>(1, c->pairs / each);
    a.lanes = 1;
    while (a.lanes < 32 && a.lanes < items) a.lanes *= 2;
    // Heads to a warp: all of a place's, so that each angle is computed once, unless that leaves multiprocessors idle.
    const int64_t places = c->batch * c->length, at_once = 32 / a.lanes, rounds = (c->heads + at_once - 1) / at_once, enough = (int64_t)sm_count() * 32;
    a.per_place = std::max<int64_t>(1, std::min(rounds, enough / places));
    a.heads_each = (rounds + a.per_place - 1) / a.per_place * at_once;
    a.per_place = (c->heads + a.heads_each - 1) / a.heads_each;
    a.warps = places * a.per_place;
    if (a.warps >= (1ll << 33)) return frnn_fail(FRNN_E_ARG, "rotary: too many places");
    cudaStream_t s = (cudaStream_t)stream;
    return with_dtype(c->dtype, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2) {
            if (each == 8) return run<T, 8>(a, c->interleaved, s);
        }
        switch (each) {
            case 4: return run<T, 4>(a, c->interleaved, s);
            case 2: return run<T, 2>(a, c->interleaved, s);
            default: return run<T, 1>(a, c->interleaved, s);
        }
    });
}
