// Matrix products on the tensor cores (tcgen05) with what follows them done on the tile that leaves Tensor Memory: the products
// of frnn_gated_mlp.cu and frnn_linear_logprobs.cu.
//
//   C[m, n] = sum over pairs g and k of A_g[m, k] B_g[n, k]          (a second pair: da Wg + db Wu)
//
// Operands are 16-bit (bf16 or fp16), accumulators 32-bit.  fp32 operands are three bf16 planes hi + mid + lo (each the rest of
// the one before, rounded to nearest: 24 bits, exactly), and a product of them six, the terms above 2^-24: lo hi, hi lo, mid mid,
// mid hi, hi mid, hi hi.  A step copies the three planes of both once for all six.
//
// Layout.  A block computes 128 rows.  Operands come by TMA, 64 values of k a stage, swizzled over 128 bytes.  An operand whose
// rows run along k lies in shared memory as rows of 128 bytes (8 rows and 1024 bytes an atom); one that runs along m or n as
// 64 rows of k, each 64 values of m, in parts of 8 KB: the tensor cores take both, nothing is transposed.  Beyond a matrix'
// edges TMA fills in zeros, so that sizes need not be multiples of anything; rows have to start on 16-byte boundaries.
//
// Roles: one thread issues copies (6 stages of 32 KB under way), one the products, 8 warps take finished accumulators out of
// Tensor Memory (which holds two sets, so that the next tile's products run meanwhile).  Blocks stay for several tiles.  Three forms:
//   PAIR   256 x 256 by a pair of blocks, each with half of B's rows, so that a byte of B in shared memory serves 256 rows
//   ALONE  128 x 128 by a block: small products spread over more multiprocessors
//   SPLIT  128 x 128 by a cluster of 2, 4 or 8 blocks, each with a part of k.  Each block then owns a part of the tile's columns:
//          the others send it their sums of these (into its shared memory), it adds them in the order of the blocks and has the
//          epilogue to itself.  (5 stages, and 64 KB for what arrives, where the epilogue turns its rows over afterwards.)
// THIN (ALONE or SPLIT, up to 32 rows, as in generation): only 32 of A's rows are copied, so that 10 stages of B are under way, 160 KB a
// multiprocessor: such products are as fast as their weights come.  The tensor cores read 128 rows all the same: what they find
// behind the 32 ends in rows of the result that nobody looks at.
#pragma once
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "frnn_lm.cuh"

#include "frnn_device.cuh"
#include "frnn_chunk.cuh"

// defined in frnn_shim.cu: a tensor map of a [planes][rows][cols] matrix of 16-bit elements, swizzled over 128 bytes
int frnn_tensor_map_swizzled(void* out_map, const void* base, uint64_t cols, uint64_t rows, uint64_t planes, uint64_t row_bytes, uint64_t plane_bytes, uint32_t box_cols, uint32_t box_rows);

namespace frnn_lm {

enum Form { PAIR, ALONE, SPLIT };
enum { BK = 64, STAGE_BYTES = 32768, THIN_ROWS = 32, EPILOGUE_WARPS = 8, PRODUCT_THREADS = 384, STAGING_BYTES = 4096 };
// Registers of the warps that copy and issue, and of the epilogue's: 128 x 56 + 256 x 224 = 384 x 168, what a block starts with.
enum { CONTROL_REGISTERS = 56, EPILOGUE_REGISTERS = 224, START_REGISTERS = 168 };
enum { PRODUCT_SHARED = 6 * STAGE_BYTES + EPILOGUE_WARPS * STAGING_BYTES + 1024 };      // (6 stages; 5 and 64 KB for what arrives; 10 thin ones, 16 KB and less staging)
enum { CODE_PRODUCT = 97 };       // error word: a wait inside a matrix product ran out

// What becomes of a tile.
enum { STORE = 0, GLU_FORWARD = 1, GLU_BACKWARD = 2, LOGPROB_STATS = 3, LOGPROB_GRAD = 4 };

// A 16-bit operand of a later product as an epilogue writes it: bf16 or fp16, or for fp32 three bf16 planes.
struct Planes {
    void* p;
    int64_t ld, plane;          // elements between rows, between planes
};

struct alignas(64) ProductArgs {
    CUtensorMap a, b[2];
    int M, N;                   // rows and columns of the result (N: of each of the two products where dual)
    int flush;                  // steps along k of a part
    int pairs;                  // products that are added up
    int ksteps, segments;       // steps of 64 along k in a segment; segments: pairs, where fp32 takes one product a step six times as many
    int tiles_m, tiles_n, group, slices;      // slices of k, each with a result of its own (STORE)
    int stacked;                // two products with the same B: the second's A is this many planes further on, its result at out2 (0: one)
    void* out2;
    int b_ready;                // the kernel before this one writes nothing of B: its copies begin before that one ends
    int dual;                   // a tile's columns are half of B0's rows and half of B1's
    unsigned idesc;
    int* err;
    // STORE
    void* out;
    int64_t out_ld, out_slice;  // out_slice: elements between two slices' results
    int out_dtype, out_wide;    // wide: rows start on 16-byte boundaries
    const float* add;           // fp32 [M][add_ld] to add, or NULL
    int64_t add_ld;
    const float* alpha;         // a factor on the device, or NULL
    // GLU_*
    int io, activation;
    float *by_gate, *by_up;     // b act'(a) and act(a), [M][by_ld]; written forward (NULL: not), read backward
    int64_t by_ld;
    Planes h, da, db;
    // LOGPROB_*
    float c2;                   // log2(e) / temperature
    float inv_t;
    const void* tokens;
    int token_bytes;
    int64_t ignore_index, first;      // first: token of column 0
    float* partial;             // STATS: [columns / stats_columns][max, sum, sum of products][M]
    float* target;              // STATS: [M] of u at the row's token
    const float *stats, *dlogprob, *dentropy;      // GRAD: [M][2] log2 of the sum, entropy
    const float* scale;         // GRAD: a power of two that brings fp16 gradients into range, or NULL
    Planes grad;
    int rest;                   // 16 bits: what rounding takes off the gradient is a second plane
};

// ---- instructions -----------------------------------------------------------------------------------------------------------

__device__ __forceinline__ u32 cluster_rank() {
    u32 r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ u32 cluster_blocks() {
    u32 r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
// the address of the same variable in block `rank` of the cluster
__device__ __forceinline__ u32 in_block(const void* p, u32 rank) {
    u32 r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(frnn_smem_addr(p)), "r"(rank));
    return r;
}
template <int CG> __device__ __forceinline__ void tma_load(u32 dst, const CUtensorMap* map, int x, int y, int z, u32 bar) {
    if constexpr (CG == 2)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"((u64)map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"((u64)map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// 16 bytes to another block's shared memory.  (st.async, which counts each of them on an mbarrier, took 5 us for a block's 64 KB.)
__device__ __forceinline__ void send(u32 dst, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// an arrival that says that what this warp has done in shared memory, its own block's or another's, is done
__device__ __forceinline__ void arrive_after_sending(u32 bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void arrive_at(u32 bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// A bounded wait (as frnn_mbar_wait) on a barrier given by its address; CLUSTER: for what other blocks of the cluster have written.
template <bool CLUSTER = false> __device__ __forceinline__ bool wait_at(u32 bar, u32 parity, int* err) {
    auto there = [&] {
        u32 ok;
        if constexpr (CLUSTER)
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        return ok != 0;
    };
    if (there()) return true;
    const u64 from = frnn_now_ns();
#pragma unroll 1
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; i++)
            if (there()) return true;
        if (frnn_now_ns() - from > FRNN_WAIT_LIMIT_NS) {
            frnn_report(err, CODE_PRODUCT);
            return false;
        }
    }
}
__device__ __forceinline__ void expect_bytes(u32 bar, u32 bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
template <int CG> __device__ __forceinline__ void mma_f16(u32 d, u64 a, u64 b, u32 idesc, u32 accumulate) {
    if constexpr (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// An arrival on `bar` (of both blocks of a pair) when the products issued so far are done.
template <int CG> __device__ __forceinline__ void mma_commit(u32 bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int CG> __device__ __forceinline__ void tmem_alloc(u32* at, u32 columns) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(frnn_smem_addr(at)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        frnn_tmem_alloc(at, columns);
    }
}
template <int CG> __device__ __forceinline__ void tmem_free(u32 at, u32 columns) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
    else frnn_tmem_dealloc(at, columns);
}
// Shared-memory operand swizzled over 128 bytes: 1024 bytes between groups of 8 rows; `parts` bytes between parts of 64 values
// of m or n (only where rows run along m or n).
__device__ __forceinline__ u64 operand_desc(u32 smem, u32 parts) {
    return (u64)((smem & 0x3ffffu) >> 4) | ((u64)(parts >> 4) << 16) | ((u64)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ---- rows of 32 values --------------------------------------------------------------------------------------------------------

// Each lane has 32 consecutive values of its row; they go to dst (rows ld elements apart) by way of shared memory, so that
// neighbouring lanes write neighbouring bytes.  Of the warp's 32 rows `rows` exist, of the 32 columns `cols`.  `wide`: rows of dst begin on 16-byte
// boundaries; `padded`: what lies behind a row's end up to such a boundary is nobody's.
template <class T> __device__ __forceinline__ void put_rows(unsigned char* staging, int lane, const float* v, T* dst, int64_t ld, int rows, int cols, bool wide, bool padded) {
    constexpr int W = WIDE<T>, CHUNKS = 32 / W, ROW = 32 * (int)sizeof(T);       // 4 chunks of 8, or 8 of 4
    auto slot = [](int r, int c) { return r * ROW + ((c ^ (sizeof(T) == 2 ? (r >> 1) & 3 : r & 7)) * 16); };
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
        Pack<T, W> x;
        x.from(v + c * W);
        x.store((T*)(staging + slot(lane, c)));
    }
    __syncwarp();
    if (wide && (padded || cols % W == 0)) {
        constexpr int AT_ONCE = 32 / CHUNKS;      // rows
        const int c = lane % CHUNKS;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
            const int r = r0 + lane / CHUNKS;
            Pack<T, W> x;
            x.load((const T*)(staging + slot(r, c)));
            if (r < rows && c * W < cols) x.store(dst + r * ld + c * W);
        }
    } else if (lane < cols) {
        for (int r = 0; r < rows; r++) dst[r * ld + lane] = *(const T*)(staging + slot(r, lane / W) + lane % W * sizeof(T));
    }
    __syncwarp();
}
__device__ __forceinline__ void put_rows_as(int dtype, unsigned char* staging, int lane, const float* v, void* dst, int64_t at, int64_t ld, int rows, int cols, bool wide, bool padded) {
    if (dtype == FRNN_F32) put_rows(staging, lane, v, (float*)dst + at, ld, rows, cols, wide, padded);
    else if (dtype == FRNN_BF16) put_rows(staging, lane, v, (__nv_bfloat16*)dst + at, ld, rows, cols, wide, padded);
    else put_rows(staging, lane, v, (__half*)dst + at, ld, rows, cols, wide, padded);
}
// x = hi + mid + lo in bf16, exactly (values above the largest bf16 are cut off first; what is not finite stays in hi alone).
__device__ __forceinline__ void split3(float x, float& hi, float& mid, float& lo) {
    hi = __bfloat162float(__float2bfloat16_rn(x));
    if (fabsf(hi) == INFINITY && fabsf(x) != INFINITY) hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    const float rest = x - hi;
    const bool whole = fabsf(hi) < INFINITY;
    mid = whole ? __bfloat162float(__float2bfloat16_rn(rest)) : 0.f;
    lo = whole ? rest - mid : 0.f;
}
template <bool FP32> __device__ __forceinline__ void put_planes(int io, unsigned char* staging, int lane, float* v, const Planes& to, int64_t row, int col, int rows, int cols) {
    const int64_t at = row * to.ld + col;
    if constexpr (FP32) {
#pragma unroll 1
        for (int plane = 0; plane < 3; plane++) {          // each round leaves the rest of the one before
            float part[32];
#pragma unroll
            for (int j = 0; j < 32; j++) {
                float mid, lo;
                split3(v[j], part[j], mid, lo);
                v[j] = fabsf(part[j]) < INFINITY ? v[j] - part[j] : 0.f;
            }
            put_rows(staging, lane, part, (__nv_bfloat16*)to.p + plane * to.plane + at, to.ld, rows, cols, true, true);
        }
    } else if (io == FRNN_F16) {
        put_rows(staging, lane, v, (__half*)to.p + at, to.ld, rows, cols, true, true);
    } else {
        put_rows(staging, lane, v, (__nv_bfloat16*)to.p + at, to.ld, rows, cols, true, true);
    }
}

// The way back: 32 values of each lane's row out of 32 rows, read by neighbouring lanes (aligned rows; undefined beyond rows and cols).
// Asked for first, turned over by way of shared memory later.
template <class T> struct Rows {
    static constexpr int W = WIDE<T>, CHUNKS = 32 / W, AT_ONCE = 32 / CHUNKS;
    Pack<T, W> x[CHUNKS];
    __device__ __forceinline__ void ask(int lane, const T* src, int64_t ld, int rows, int cols) {
        const int c = lane % CHUNKS;
#pragma unroll
        for (int k = 0; k < CHUNKS; k++) {
            const int r = k * AT_ONCE + lane / CHUNKS;
            if (r < rows && c * W < cols) x[k].load(src + r * ld + c * W);      // (rows are padded to whole accesses)
        }
    }
    __device__ __forceinline__ void get(unsigned char* staging, int lane, float* v) const {
        constexpr int ROW = 32 * (int)sizeof(T);
        auto slot = [](int r, int c) { return r * ROW + ((c ^ (sizeof(T) == 2 ? (r >> 1) & 3 : r & 7)) * 16); };
#pragma unroll
        for (int k = 0; k < CHUNKS; k++) x[k].store((T*)(staging + slot(k * AT_ONCE + lane / CHUNKS, lane % CHUNKS)));
        __syncwarp();
#pragma unroll
        for (int k = 0; k < CHUNKS; k++) {
            Pack<T, W> y;
            y.load((const T*)(staging + slot(lane, k)));
            y.to(v + k * W);
        }
        __syncwarp();
    }
};

// ---- activations -----------------------------------------------------------------------------------------------------------

// h = act(a) b of N values, and where asked for its derivatives by a and b, in their place.  (One choice for all of them:
// chosen for each value, the code of all four no longer fit the instruction cache, and a tile took five times as long.)
// gelu: a Phi(a), Phi(-t) = exp(-t^2 / 2) R(t) with R(t) = erfcx(t / sqrt 2) / 2, which is smooth: s = 1 / (1 + 0.26 t) times a polynomial
// in s, fitted over 0 <= t <= 14.5 (beyond, Phi(-t) is 0) for the least relative error by reweighted least squares: 2.8e-8, in 32 bits 4e-7 and
// t^2 2^-23.  (8192 x 1024 to 4096 in bf16, us without and with derivatives: silu 84 and 118, gelu 102 and 129, gelu with erfcf 123 and 166.)
template <int KIND> __device__ __forceinline__ void activate(float a, float& act, float& slope) {
    if constexpr (KIND == FRNN_SILU || KIND == FRNN_SIGMOID) {
        const float s = __fdividef(1.f, 1.f + __expf(-a));
        act = KIND == FRNN_SILU ? a * s : s;
        slope = KIND == FRNN_SILU ? fmaf(act, 1.f - s, s) : s * (1.f - s);
    } else if constexpr (KIND == FRNN_GELU) {
        const float t = fminf(fabsf(a), 14.5f), s = __fdividef(1.f, fmaf(0.26f, t, 1.f)), e = exp2_fast(-0.72134752044448170f * (t * t));
        float r = 3.023032099e-02f;
        r = fmaf(r, s, -1.514945477e-01f);
        r = fmaf(r, s, 2.487334311e-01f);
        r = fmaf(r, s, -1.477895379e-01f);
        r = fmaf(r, s, 1.587588638e-01f);
        r = fmaf(r, s, 5.196479708e-02f);
        r = fmaf(r, s, 1.027886793e-01f);
        r = fmaf(r, s, 1.030509695e-01f);
        r = fmaf(r, s, 1.037570164e-01f);
        const float low = e * (r * s), share = a > 0.f ? 1.f - low : low;
        act = a * share;
        slope = fmaf(a, 0.39894228040143268f * e, share);
    } else {
        act = a > 0.f || a != a ? a : 0.f;
        slope = a > 0.f ? 1.f : 0.f;
    }
}
template <int KIND, int N> __device__ __forceinline__ void glu_of(float* a, float* b, float* h, bool derivatives) {
#pragma unroll
    for (int j = 0; j < N; j++) {
        float act, slope;
        activate<KIND>(a[j], act, slope);
        h[j] = act * b[j];
        if (derivatives) {
            a[j] = b[j] * slope;
            b[j] = act;
        }
    }
}
template <int N> __device__ __forceinline__ void glu(int kind, float* a, float* b, float* h, bool derivatives) {
    switch (kind) {
        case FRNN_SILU: return glu_of<FRNN_SILU, N>(a, b, h, derivatives);
        case FRNN_GELU: return glu_of<FRNN_GELU, N>(a, b, h, derivatives);
        case FRNN_RELU: return glu_of<FRNN_RELU, N>(a, b, h, derivatives);
        default: return glu_of<FRNN_SIGMOID, N>(a, b, h, derivatives);
    }
}

// ---- epilogues ---------------------------------------------------------------------------------------------------------------

// The tensor cores add to an accumulator with truncation, not rounding: a sum over k loses up to two units of its last bit for each 16
// values, all in one direction (measured against 64 bits, 2-norm: 7e-6 at k = 4096 in 16 bits, 2e-5 at 8192 in fp32, where 32-bit sums
// rounded to nearest lose some 9e-7).  So sums along k come in parts of `flush` steps, which the epilogue's warps add up in registers, half
// of a tile's columns a warp; the sums go back to where the last part was, and the epilogue is the same for all.  (One that took them from
// registers had its loops unrolled, and its code did not fit the instruction cache.)
//   results in 16 bits: parts of 64 steps, so that no length of k loses more than 7e-6 (2.4e-5 of positive terms) beside the results'
//     rounding, 2e-4 in fp16; a k of 100000 in one part leaned by 2e-4.  No cost that shows (mlp_train, in turn: 6.29 and 6.33 ms).
//   log probabilities of 16-bit operands: parts of 16, 4e-7 (of 4: loss_train a sixth slower).  Up to 128 rows, which wait for weights and not
//     for the epilogue, of 4: 16 rows of 4096 against 65536 tokens 6.3e-7 -> 9e-8 for 104 -> 107 us.  The same in their backward (2 % of
//     loss_train), because a probability is an exponential of the difference between its logits and the forward's log of the sum: of
//     tokens with p = 0.999 at logits of 40, gradients from sums in one part were wrong altogether.
//   fp32 where a step is six products: parts of one, whose small products come first, while the accumulator is small: 3e-7 (of two steps
//     1.6e-6 and 4 % faster); in SPLIT: parts of 4, 6e-7.

// 32 columns of accumulators, of the lane's row.  (Waited for apart: the next ones are under way while these are worked on.)
__device__ __forceinline__ void ask(u32 taddr, float* v) { frnn_tmem_ld<32>(taddr, v); }
template <int N> __device__ __forceinline__ void wait_for(float* v) {
    frnn_tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < N; j++) asm volatile("" : "+f"(v[j]));      // (nothing that uses them moves up)
}

// da = dh (b act'(a)), db = dh act(a), 32 columns at a time; the next ones' factors are on their way meanwhile.
template <bool FP32>
__device__ __forceinline__ void glu_backward(const ProductArgs& p, u32 acc, int64_t row0, int first, int count, int rows, int lane, unsigned char* staging) {
    Rows<float> gate, up;
    auto fetch = [&](Rows<float>& to, const float* from, int i) {
        const int col = first + i;
        if (i < count) to.ask(lane, from + row0 * p.by_ld + col, p.by_ld, rows, min(32, min(count - i, p.N - col)));
    };
    if (p.da.p) fetch(gate, p.by_gate, 0);
    if (p.db.p) fetch(up, p.by_up, 0);
#pragma unroll 1
    for (int i = 0; i < count; i += 32) {
        float d[32], f[32];
        ask(acc + i, d);
        wait_for<32>(d);
        const int col = first + i, cols = min(32, min(count - i, p.N - col));
        if (rows <= 0 || cols <= 0) break;
        if (p.da.p) {
            gate.get(staging, lane, f);
            fetch(gate, p.by_gate, i + 32);
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] *= d[j];
            put_planes<FP32>(p.io, staging, lane, f, p.da, row0, col, rows, cols);
        }
        if (p.db.p) {
            up.get(staging, lane, f);
            fetch(up, p.by_up, i + 32);
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] *= d[j];
            put_planes<FP32>(p.io, staging, lane, f, p.db, row0, col, rows, cols);
        }
    }
}

// What the epilogues of log probabilities know of a lane's row, asked for before the accumulators are there.
struct RowData {
    int64_t token;
    float lse2, entropy, g, h;
};
template <int EPI> __device__ __forceinline__ RowData row_data(const ProductArgs& p, int64_t row) {
    RowData d = {-1, 0.f, 0.f, 0.f, 0.f};
    if constexpr (EPI == LOGPROB_STATS || EPI == LOGPROB_GRAD) {
        if (row < p.M) {
            d.token = token_at(p.tokens, p.token_bytes, row);
            if constexpr (EPI == LOGPROB_GRAD) {
                d.lse2 = p.stats[2 * row];
                d.entropy = p.stats[2 * row + 1];
                if (p.dlogprob) d.g = p.dlogprob[row];
                if (p.dentropy) d.h = p.dentropy[row];
            }
        }
    }
    return d;
}

struct Tile { int tm, tn, slice, from, to; bool second; };      // from, to: steps along k of a block

// `count` columns from the one numbered `first` on, whose accumulators lie at `acc` (of GLU_FORWARD's second product at `acc2`), of the 32
// rows from row0 on.
template <int EPI, bool FP32>
__device__ __forceinline__ void epilogue(const ProductArgs& p, const RowData& data, u32 acc, u32 acc2, int64_t row0, int first, int count, const Tile& w, int lane, unsigned char* staging) {
    // body(col, cols, v) for each 32 columns
    auto each = [&](auto body) {
        float v[32], next[32];
        ask(acc, v);
#pragma unroll 1
        for (int i = 0; i < count; i += 32) {
            wait_for<32>(v);
            if (i + 32 < count) ask(acc + i + 32, next);
            body(first + i, min(32, min(count - i, p.N - first - i)), v);
            if (i + 32 < count) {
                wait_for<32>(next);
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = next[j];
            }
        }
    };
    const int rows = (int)min((int64_t)32, max((int64_t)0, p.M - row0));
    const int64_t row = row0 + lane;
    if constexpr (EPI == STORE) {
        const float alpha = p.alpha ? *p.alpha : 1.f;
        each([&](int col, int cols, float* v) {
            if (rows <= 0 || cols <= 0) return;
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] *= alpha;
            if (p.add) {
                float o[32];
                Rows<float> sum;
                sum.ask(lane, p.add + row0 * p.add_ld + col, p.add_ld, rows, cols);
                sum.get(staging, lane, o);
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] += o[j];
            }
            put_rows_as(p.out_dtype, staging, lane, v, w.second ? p.out2 : p.out, w.slice * p.out_slice + row0 * p.out_ld + col, p.out_ld, rows, cols, p.out_wide, false);
        });
    } else if constexpr (EPI == GLU_FORWARD) {
#pragma unroll 1
        for (int i = 0; i < count; i += 32) {
            float a[32], b[32], h[32];
            ask(acc + i, a);
            ask(acc2 + i, b);
            wait_for<32>(a);
            wait_for<32>(b);
            const int col = first + i, cols = min(32, min(count - i, p.N - col));
            if (rows <= 0 || cols <= 0) continue;
            glu<32>(p.activation, a, b, h, p.by_gate);
            if (p.by_gate) {
                const int64_t at = row0 * p.by_ld + col;
                put_rows(staging, lane, a, p.by_gate + at, p.by_ld, rows, cols, true, true);
                put_rows(staging, lane, b, p.by_up + at, p.by_ld, rows, cols, true, true);
            }
            put_planes<FP32>(p.io, staging, lane, h, p.h, row0, col, rows, cols);
        }
    } else if constexpr (EPI == GLU_BACKWARD) {
        glu_backward<FP32>(p, acc, row0, first, count, rows, lane, staging);
    } else if constexpr (EPI == LOGPROB_STATS) {
        const int64_t token = data.token;
        float m = -3.4028235e38f, s = 0.f, t = 0.f;
        each([&](int col, int cols, float* v) {
            if (cols <= 0) return;
            const int64_t hit = token - p.first - col;
            float tops[4] = {m, m, m, m};
            if (cols == 32) {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] *= p.c2;
            } else {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = j < cols ? v[j] * p.c2 : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 32; j++) tops[j % 4] = fmaxf(tops[j % 4], v[j]);
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            if (__any_sync(0xffffffffu, hit >= 0 && hit < cols)) {          // (one chunk of thousands)
                float x = 0.f;          // (a choice of one becomes an index into registers, which then all live in memory)
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (hit == j) x += v[j];
                if (hit >= 0 && hit < cols && lane < rows) p.target[row] = x;
            }
            const float down = exp2_fast(m - top);
            t = s == 0.f ? 0.f : down * (t + s * (m - top));
            s *= down;
            float s4[4] = {}, t4[4] = {};
#pragma unroll
            for (int j = 0; j < 32; j++) {
                const float u = v[j] - top, e = exp2_fast(u);
                s4[j % 4] += e;
                t4[j % 4] = fmaf(e, fmaxf(u, -1e30f), t4[j % 4]);
            }
            s += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            t += (t4[0] + t4[1]) + (t4[2] + t4[3]);
            m = top;
        });
        if (lane < rows) {
            float* to = p.partial + (int64_t)(first / count) * 3 * p.M + row;
            to[0] = m;
            to[p.M] = s;
            to[2 * (int64_t)p.M] = t;
        }
    } else {
        const int64_t token = data.token;
        const float lse2 = data.lse2, entropy = data.entropy, g = token != p.ignore_index ? data.g : 0.f, h = data.h;
        const bool empty = lse2 == -INFINITY;
        const float scale = p.scale ? *p.scale : 1.f, gk = -g * p.inv_t * scale, hk = -h * p.inv_t * scale;      // (g first: 1 / T alone times the factor may pass 2^128)
        each([&](int col, int cols, float* v) {
            if (rows <= 0 || cols <= 0) return;
            const int64_t hit = token - p.first - col;
#pragma unroll
            for (int j = 0; j < 32; j++) {
                const float u = fmaf(v[j], p.c2, -lse2), e = exp2_fast(u);
                v[j] = e * fmaf(hk, fmaf(fmaxf(u, -1e30f), 0.69314718055994531f, entropy), gk);
            }
            if (__any_sync(0xffffffffu, hit >= 0 && hit < cols)) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (hit == j) v[j] -= gk;
            }
            if (__any_sync(0xffffffffu, empty)) {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = empty ? 0.f : v[j];
            }
            put_planes<FP32>(p.io, staging, lane, v, p.grad, row0, col, rows, cols);
            if (!FP32 && p.rest) {
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    const float near = p.io == FRNN_F16 ? __half2float(__float2half_rn(v[j])) : __bfloat162float(__float2bfloat16_rn(v[j]));
                    v[j] = fabsf(near) < INFINITY ? v[j] - near : 0.f;
                }
                put_planes<FP32>(p.io, staging, lane, v, p.grad, row0 + p.M, col, rows, cols);      // (its rows follow the first plane's)
            }
        });
    }
}

// ---- the kernel ---------------------------------------------------------------------------------------------------------------

// Part `part` of `parts` of a tile's (a slice's) steps along k.
__device__ __forceinline__ void steps_of(const ProductArgs& p, Tile& w, u32 part, u32 parts) {
    const int steps = p.ksteps * p.segments;
    if (p.slices * parts == 1) {                   // (64-bit divisions take as long as a small tile's products)
        w.from = 0;
        w.to = steps;
    } else {
        const int64_t all = (int64_t)p.slices * parts, at = (int64_t)w.slice * parts + part;
        w.from = (int)(steps * at / all);
        w.to = (int)(steps * (at + 1) / all);
    }
}
// Tiles in groups of `group` rows of tiles, column after column: A's rows of a group stay in L2 while B passes by once.
__device__ __forceinline__ Tile tile_of(const ProductArgs& p, int u, u32 part, u32 parts) {
    Tile w;
    const int tiles = p.tiles_m * p.tiles_n;
    w.slice = p.slices > 1 ? u / tiles : 0;
    const int in_slice = u - w.slice * tiles, a_group = p.group * p.tiles_n, g = in_slice / a_group, in = in_slice - g * a_group, high = min(p.group, p.tiles_m - g * p.group);
    w.tn = in / high;
    w.tm = g * p.group + in - w.tn * high;
    w.second = p.stacked && w.tm >= p.tiles_m / 2;
    if (w.second) w.tm -= p.tiles_m / 2;
    steps_of(p, w, part, parts);
    return w;
}

// AT, BT: the operand's rows run along m (n) instead of k.
template <Form FORM, bool THIN, bool AT, bool BT, int EPI, bool FP32> __global__ void __launch_bounds__(PRODUCT_THREADS, 1) product_kernel(const __grid_constant__ ProductArgs p) {
    // fp32: a step copies three planes of each operand and multiplies them six times; in SPLIT, whose stages hold no two such steps, it is one
    // product of two planes, and the six follow one another over all of k
    constexpr bool FUSED = FP32 && (FORM != SPLIT || THIN);
    constexpr int PLANES = FUSED ? 3 : 1;
    constexpr int CG = FORM == PAIR ? 2 : 1, BN = FORM == PAIR ? 256 : 128, STAGES = THIN ? 10 : FORM == SPLIT ? 5 : 6;
    constexpr int NB = BN / CG;                        // B's rows in this block
    constexpr int ROWS = THIN ? (int)THIN_ROWS : 128;  // of A, that are copied and that have a result
    constexpr u32 A_BYTES = ROWS * BK * 2, B_BYTES = NB * BK * 2, STAGE = A_BYTES + B_BYTES, COLUMNS = FORM == SPLIT ? 512 : 2 * BN;
    constexpr u32 EXCHANGE = FORM == SPLIT ? ROWS * BN * 4 : 0;
    constexpr bool SHARE = FORM == SPLIT && !THIN;     // staging lies where the sums arrived
    static_assert(STAGES * STAGE + EXCHANGE + (SHARE ? 0 : ROWS / 32 * 2 * STAGING_BYTES) + 1024 <= PRODUCT_SHARED && COLUMNS <= 512, "shared memory or Tensor Memory is too small");
    static_assert(!THIN || (!AT && CG == 1), "only rows along k can be left out");
    extern __shared__ unsigned char raw[];
    __shared__ u64 full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], arrived, taken, summed, halves[4];
    __shared__ u32 tmem;
    unsigned char* const smem = raw + (1024 - (frnn_smem_addr(raw) & 1023)) % 1024;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const u32 rank = FORM == ALONE ? 0 : cluster_rank(), blocks = FORM == ALONE ? 1 : cluster_blocks();
    const u32 half_m = CG == 2 ? rank : 0;        // which 128 of a tile's rows
    const int tiles = p.tiles_m * p.tiles_n * p.slices, first = blockIdx.x / blocks, stride = gridDim.x / blocks;
    const u32 part = FORM == SPLIT ? rank : 0, parts = FORM == SPLIT ? blocks : 1;       // of a tile's steps along k

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            frnn_mbar_init(&full[s], 1);
            frnn_mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            frnn_mbar_init(&acc_full[b], 1);
            frnn_mbar_init(&acc_empty[b], EPILOGUE_WARPS * CG);
        }
        if (FORM == SPLIT) {
            frnn_mbar_init(&arrived, EPILOGUE_WARPS * blocks);
            frnn_mbar_init(&taken, EPILOGUE_WARPS * blocks);
            frnn_mbar_init(&summed, EPILOGUE_WARPS);
        }
        for (int q = 0; q < 4; q++) frnn_mbar_init(&halves[q], 2);
        frnn_mbar_init_fence();
    }
    if (warp == 1 && lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"((u64)(lane ? &p.b[lane - 1] : &p.a)) : "memory");
    __syncwarp();
    if (warp == 2) tmem_alloc<CG>(&tmem, COLUMNS);
    frnn_tmem_fence_before_sync();
    if constexpr (FORM != ALONE) cluster_sync();
    __syncthreads();
    frnn_tmem_fence_after_sync();
    // Up to here nothing has been read that a kernel before this one may still be writing; the next one may come as far.  (That one finds
    // everything written that was before this kernel's own predecessor ended.)
    if (warp != 0) {
        cudaGridDependencySynchronize();
        cudaTriggerProgrammaticLaunchCompletion();
    }

    if (warp < 4) {
        frnn_regs_release<CONTROL_REGISTERS>();
        if (warp == 0) {
            // (One thread each copies and issues: of few instructions a step, because a step of 128 x 128 is done in 256 cycles.)
            if (frnn_elect()) {
                const u32 base = frnn_smem_addr(smem), empty0 = frnn_smem_addr(&empty[0]), full0 = frnn_smem_addr(&full[0]), full_lead = CG == 2 ? in_block(&full[0], 0) : full0;
                u32 s = 0, phase = 1, issued = 0;
                bool ok = true;
                auto load_b = [&](u32 s, const CUtensorMap* map, int n, int plane, int k) {
                    const u32 bar = full_lead + s * 8, at = base + s * STAGE + A_BYTES;
                    if (CG == 1 || half_m == 0) expect_bytes(full0 + s * 8, STAGE * CG);      // (a's bytes too)
                    if constexpr (BT) {
#pragma unroll
                        for (int part = 0; part < NB / 64; part++) tma_load<CG>(at + part * 8192, map, n + part * 64, k, plane, bar);
                    } else {
                        tma_load<CG>(at, map, k, n, plane, bar);
                        if (CG == 1 && p.dual) tma_load<CG>(at + B_BYTES / 2, &p.b[1], k, n, plane, bar);      // (copies of 64 rows)
                    }
                };
                auto load_a = [&](u32 s, int m, int plane, int k) {
                    const u32 bar = full_lead + s * 8, at = base + s * STAGE;
                    if constexpr (AT) {
                        tma_load<CG>(at, &p.a, m, k, plane, bar);
                        tma_load<CG>(at + A_BYTES / 2, &p.a, m + 64, k, plane, bar);
                    } else {
                        tma_load<CG>(at, &p.a, k, m, plane, bar);
                    }
                };
                auto column = [&](const Tile& w) { return p.dual ? w.tn * (BN / 2) : w.tn * BN + (int)half_m * NB; };
                // (of two B a pair's blocks have one each)
                auto map_of = [&](int g) { return &p.b[p.dual ? (CG == 2 ? (int)half_m : 0) : FP32 && !FUSED ? g % p.pairs : g]; };
                // planes of a and b in segment g (fp32 in SPLIT: small terms first)
                auto plane_a = [&](int g) {
                    if (!FP32 || FUSED) return g * PLANES;
                    const int t = g / p.pairs;
                    return (t == 0 ? 2 : t == 2 || t == 3 ? 1 : 0) + g % p.pairs * 3;
                };
                auto plane_b = [&](int g) {
                    if (!FP32 || FUSED) return 0;
                    const int t = g / p.pairs;
                    return t == 1 ? 2 : t == 2 || t == 4 ? 1 : 0;
                };
                u32 early = 0;
                if (p.b_ready && first < tiles) {
                    const Tile w = tile_of(p, first, part, parts);
                    early = min(STAGES, min(STAGES, w.to - w.from) * PLANES);
                    for (u32 i = 0; i < early; i++) {
                        const int step = w.from + (int)i / PLANES, g = step / p.ksteps;
                        load_b(i, map_of(g), column(w), plane_b(g) + (int)i % PLANES, (step - g * p.ksteps) * BK);
                    }
                }
                cudaGridDependencySynchronize();
                for (int u = first; ok && u < tiles; u += stride) {
                    const Tile w = tile_of(p, u, part, parts);
                    const int m = (w.tm * CG + (int)half_m) * 128, n = column(w), further = w.second ? p.stacked : 0;
                    int g = w.from / p.ksteps, at = w.from - g * p.ksteps, left = w.to - w.from;      // (in steps: all segments together may pass 2^31 values)
                    for (; ok && left > 0; g++, at = 0) {
                        const CUtensorMap* const map = map_of(g);
                        const int pa = plane_a(g) + further, pb = plane_b(g), some = min(p.ksteps - at, left);
                        left -= some;
                        int k = at * BK;
                        const int end = k + some * BK;
#pragma unroll 1
                        for (; ok && k < end; k += BK) {
#pragma unroll
                            for (int plane = 0; plane < PLANES; plane++) {
                                if (issued >= early) {
                                    if (!(ok = wait_at(empty0 + s * 8, phase, p.err))) break;
                                    load_b(s, map, n, pb + plane, k);
                                }
                                load_a(s, m, pa + plane, k);
                                issued++;
                                if (++s == STAGES) {
                                    s = 0;
                                    phase ^= 1;
                                }
                            }
                        }
                    }
                }
                // every copy has been used, and every arrival has come, before the block leaves
                for (u32 i = issued > STAGES ? issued - STAGES : 0; i < issued; i++)
                    if (!wait_at(empty0 + i % STAGES * 8, i / STAGES & 1, p.err)) break;
            }
            __syncwarp();
        } else if (warp == 1) {
            if (half_m == 0 && frnn_elect()) {
                const u32 full0 = frnn_smem_addr(&full[0]), empty0 = frnn_smem_addr(&empty[0]);
                const u64 a0 = operand_desc(frnn_smem_addr(smem), 8192), b0 = operand_desc(frnn_smem_addr(smem) + A_BYTES, 8192);
                u32 s = 0, phase = 0, t = 0;
                bool ok = true;
                for (int u = first; ok && u < tiles; u += stride) {
                    const Tile w = tile_of(p, u, part, parts);
                    for (int from = w.from; ok && from < w.to; t++) {
                        const int to = min(from + p.flush, w.to);
                        const u32 buf = t & 1, d = tmem + buf * BN;
                        if (!(ok = wait_at(frnn_smem_addr(&acc_empty[buf]), (t / 2 & 1) ^ 1, p.err))) break;
                        frnn_tmem_fence_after_sync();
                        u32 more = 0;                      // (the first product of a part overwrites what was there)
#pragma unroll 1
                        for (int i = from; i < to; i++) {
                            u32 at[PLANES];                // the stages of a step's planes
#pragma unroll
                            for (int plane = 0; plane < PLANES; plane++) {
                                at[plane] = s;
                                if (ok) ok = wait_at(full0 + s * 8, phase, p.err);
                                if (++s == STAGES) {
                                    s = 0;
                                    phase ^= 1;
                                }
                            }
                            if (!ok) break;
                            frnn_tmem_fence_after_sync();
                            // of three planes the products above 2^-24 of the largest, the small ones first, while the accumulators are small
                            constexpr int PRODUCTS = FUSED ? 6 : 1;
#pragma unroll
                            for (int q = 0; q < PRODUCTS; q++) {
                                const int of_a = !FUSED ? 0 : q == 0 ? 2 : q == 2 || q == 3 ? 1 : 0, of_b = !FUSED ? 0 : q == 1 ? 2 : q == 2 || q == 4 ? 1 : 0;
                                const u64 a = a0 + at[of_a] * (STAGE / 16), b = b0 + at[of_b] * (STAGE / 16);
#pragma unroll
                                for (int k = 0; k < BK / 16; k++) {      // 16 values of k: 32 bytes of a row, or 16 rows
                                    mma_f16<CG>(d, a + k * (AT ? 2048 / 16 : 32 / 16), b + k * (BT ? 2048 / 16 : 32 / 16), p.idesc, more);
                                    more = 1;
                                }
                            }
#pragma unroll
                            for (int plane = 0; plane < PLANES; plane++) mma_commit<CG>(empty0 + at[plane] * 8);
                        }
                        mma_commit<CG>(frnn_smem_addr(&acc_full[buf]));
                        from = to;
                    }
                }
            }
            __syncwarp();
        }
    } else {
        frnn_regs_acquire<EPILOGUE_REGISTERS>();
        const int quarter = warp % 4, half = (warp - 4) / 4;
        const bool idle = quarter * 32 >= ROWS;                               // none of this warp's rows has a result
        unsigned char* const staging = smem + STAGES * STAGE + (SHARE ? 0 : EXCHANGE) + (half * (ROWS / 32) + (idle ? 0 : quarter)) * STAGING_BYTES;
        float4* const exchange = (float4*)(smem + STAGES * STAGE);            // SPLIT: [block][own columns / 4][rows]
        u32 t = 0, round = 0;
        bool ok = true;
        auto filled = [&] {            // waits for accumulators; their address
            ok = __all_sync(0xffffffffu, wait_at(frnn_smem_addr(&acc_full[t & 1]), t / 2 & 1, p.err));
            frnn_tmem_fence_after_sync();
            return tmem + (t & 1) * BN + frnn_tmem_lane_base(quarter);
        };
        auto emptied = [&] {           // this warp has taken what it needs
            frnn_tmem_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) arrive_at(in_block(&acc_empty[t & 1], 0));
                else frnn_mbar_arrive(&acc_empty[t & 1]);
            }
            t++;
        };
        auto row_of = [&](const Tile& w) { return (int64_t)(w.tm * CG + (int)half_m) * 128 + quarter * 32; };
        Tile next = {};
        RowData next_data = {};
        if (first < tiles) {
            next = tile_of(p, first, part, parts);
            next_data = row_data<EPI>(p, row_of(next) + lane);
        }
        // waits for other warps of this block, once a round (with a limit, as all waits: a warp that gave up does not come)
        auto met = [&](u64* bar) {
            __syncwarp();
            if (lane == 0) frnn_mbar_arrive(bar);
            ok = __all_sync(0xffffffffu, wait_at(frnn_smem_addr(bar), round & 1, p.err));
        };
        for (int u = first; ok && u < tiles; u += stride, round++) {
            const Tile w = next;
            const RowData data = next_data;
            const int64_t row0 = row_of(w);
            if (u + stride < tiles) {          // (its data is on its way while this one leaves)
                next = tile_of(p, u + stride, part, parts);
                next_data = row_data<EPI>(p, row_of(next) + lane);
            }
            u32 acc = filled();
            if (!ok) break;
            if (FORM == SPLIT || w.from + p.flush < w.to) {
                float sum[BN / 2];
#pragma unroll
                for (int i = 0; i < BN / 2; i += 32) ask(acc + half * (BN / 2) + i, sum + i);
                wait_for<BN / 2>(sum);
                for (int from = w.from + p.flush; from < w.to; from += p.flush) {
                    emptied();
                    acc = filled();
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < BN / 2; i += 32) {
                        float v[32];
                        ask(acc + half * (BN / 2) + i, v);
                        wait_for<32>(v);
#pragma unroll
                        for (int j = 0; j < 32; j++) sum[i + j] += v[j];
                    }
                }
                if (!ok) break;
                if constexpr (FORM == SPLIT) {
                    emptied();
                    // to the owners: of every block's columns those that this warp has, four at a time
                    const int own = BN / (int)blocks, row = quarter * 32 + lane;      // (own: a power of two)
                    ok = __all_sync(0xffffffffu, wait_at<true>(frnn_smem_addr(&taken), (round & 1) ^ 1, p.err));
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < BN / 2 && !idle; i += 4) {
                        const int c = half * (BN / 2) + i;
                        int owner, at;
                        if (EPI == GLU_FORWARD) {      // (an owner has the same columns of both products)
                            owner = i >> (__ffs(own) - 2);
                            at = (i & (own / 2 - 1)) + half * (own / 2);
                        } else {
                            owner = c >> (__ffs(own) - 1);
                            at = c & (own - 1);
                        }
                        send(in_block(&exchange[((int)rank * own + at) / 4 * ROWS + row], owner), sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
                    }
                    __syncwarp();
                    if (lane < (int)blocks) arrive_after_sending(in_block(&arrived, lane));
                    ok = __all_sync(0xffffffffu, wait_at<true>(frnn_smem_addr(&arrived), round & 1, p.err));
                    if (!ok) break;
                    // the owner's columns: half of them each, but whole accesses of 8 (both products' of GLU_FORWARD)
                    const int width = EPI == GLU_FORWARD ? own / 2 : own, count = max(8, width / 2), from = half * count;
                    const u32 place = tmem + 2 * BN + frnn_tmem_lane_base(quarter) + half * 64;
                    const bool works = from < width && !idle && row0 < p.M;
                    if (works) {
                        const int values = (EPI == GLU_FORWARD ? 2 : 1) * count;
                        float v[32] = {};
                        for (u32 b = 0; b < blocks; b++) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                if (i >= values) continue;
                                const int at = i < count ? from + i : own / 2 + from + i - count;
                                const float4 x = exchange[((int)b * own + at) / 4 * ROWS + row];
                                v[i] += x.x; v[i + 1] += x.y; v[i + 2] += x.z; v[i + 3] += x.w;
                            }
                        }
                        frnn_tmem_st<32>(place, v);
                        frnn_tmem_wait_st();
                    }
                    // The others may write here again, what has been read and (SHARE) staged here lies before that: a release to the cluster, which their
                    // wait acquires.  It waits for this warp's stores of the tile, so it comes only where another round does.
                    auto done_with = [&] {
                        if (u + stride >= tiles) return;
                        __syncwarp();
                        if (lane < (int)blocks) arrive_after_sending(in_block(&taken, lane));
                    };
                    if constexpr (SHARE) {
                        met(&summed);
                        if (!ok) break;
                    } else {
                        done_with();
                    }
                    if (works) {
                        const int tile_col = w.tn * (EPI == GLU_FORWARD ? BN / 2 : BN) + (int)rank * width;
                        epilogue<EPI, FP32>(p, data, place, place + count, row0, tile_col + from, count, w, lane, staging);
                    }
                    if constexpr (SHARE) done_with();
                    continue;
                } else {
#pragma unroll
                    for (int i = 0; i < BN / 2; i += 32) frnn_tmem_st<32>(acc + half * (BN / 2) + i, sum + i);
                    frnn_tmem_wait_st();
                    if constexpr (EPI == GLU_FORWARD) {      // (a warp's columns of the two products lie in both warps' halves)
                        frnn_tmem_fence_before_sync();
                        met(&halves[quarter]);
                        frnn_tmem_fence_after_sync();
                        if (!ok) break;
                    }
                }
            }
            constexpr int COUNT = EPI == GLU_FORWARD ? BN / 4 : BN / 2;
            if (!idle && row0 < p.M) epilogue<EPI, FP32>(p, data, acc + half * COUNT, acc + half * COUNT + BN / 2, row0, w.tn * 2 * COUNT + half * COUNT, COUNT, w, lane, staging);
            emptied();
        }
    }
    frnn_tmem_fence_before_sync();
    __syncthreads();
    if constexpr (FORM != ALONE) cluster_sync();
    frnn_tmem_fence_after_sync();
    if (warp == 2) tmem_free<CG>(tmem, COLUMNS);
}

// The results of `slices` slices of k, fp32 [slices][M][ld] at p.out, added in their order.
static __global__ void __launch_bounds__(256) join_slices(const __grid_constant__ ProductArgs p, void* to, int to_dtype, int64_t to_ld) {
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const int64_t quads = (p.N + 3) / 4;
    const float alpha = p.alpha ? *p.alpha : 1.f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.M * quads; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / quads, col = i % quads * 4;
        const float* const from = (const float*)p.out + row * p.out_ld + col;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < p.slices; s++) {
            const float4 x = *(const float4*)(from + s * p.out_slice);
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (col + e >= p.N) break;
            float x = (&v.x)[e] * alpha;
            if (p.add) x += p.add[row * p.add_ld + col + e];
            const int64_t at = row * to_ld + col + e;
            if (to_dtype == FRNN_F32) ((float*)to)[at] = x;
            else if (to_dtype == FRNN_BF16) ((__nv_bfloat16*)to)[at] = from_float<__nv_bfloat16>(x);
            else ((__half*)to)[at] = from_float<__half>(x);
        }
    }
}

// ---- operands -------------------------------------------------------------------------------------------------------------------

// Rows of any type and stride as 16-bit operands: rows on 16-byte boundaries, fp32 as three planes.  A thread takes 8 columns;
// blockIdx.y is the matrix.
enum { MAX_PACKS = 5 };
struct PackJob {
    const void* x;
    int64_t rows, cols, stride;
    Planes to;
    int wide;                   // rows of x start on 16-byte boundaries
};
struct Packs {
    PackJob each[MAX_PACKS];
    int count;
};
template <class T> __global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packs packs) {
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const PackJob& m = packs.each[blockIdx.y];
    const int64_t eights = (m.cols + 7) / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < m.rows * eights; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / eights, col = i % eights * 8;
        const T* const from = (const T*)m.x + row * m.stride + col;
        float v[8];
        if (m.wide && col + 8 <= m.cols) {
            constexpr int W = WIDE<T>;
#pragma unroll
            for (int c = 0; c < 8; c += W) {
                Pack<T, W> q;
                q.load(from + c);
                q.to(v + c);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = col + e < m.cols ? to_float(from[e]) : 0.f;
        }
        if constexpr (sizeof(T) == 2) {
            Pack<T, 8> q;
            q.from(v);
            q.store((T*)m.to.p + row * m.to.ld + col);
        } else {
            float part[3][8];
#pragma unroll
            for (int e = 0; e < 8; e++) split3(v[e], part[0][e], part[1][e], part[2][e]);
#pragma unroll
            for (int k = 0; k < 3; k++) {
                Pack<__nv_bfloat16, 8> q;
                q.from(part[k]);
                q.store((__nv_bfloat16*)m.to.p + k * m.to.plane + row * m.to.ld + col);
            }
        }
    }
}

// Scratch handed out piece by piece; `used` may be set back when what came after is no longer needed.  Without memory behind it,
// `most` is what is asked for.
struct Scratch {
    char* base;
    size_t used = 0, most = 0;
    void* take(size_t bytes) {
        void* const p = base ? base + used : nullptr;
        used += (bytes + 255) / 256 * 256;
        most = std::max(most, used);
        return p;
    }
};

// Rows of 16-bit operands begin on whole lines: a box' rows of 128 bytes that straddle two cost two requests each.
inline int64_t padded(int64_t n) { return (n + 63) / 64 * 64; }
inline int planes_of(int dtype) { return dtype == FRNN_F32 ? 3 : 1; }

struct Operand {                  // a [rows][cols] matrix in 16 bits
    const void* p = nullptr;
    int64_t rows = 0, cols = 0, ld = 0, plane = 0;
    int planes = 1;
    Planes writable() const { return {const_cast<void*>(p), ld, plane}; }
    Operand from_row(int64_t r, int64_t n) const {
        Operand o = *this;
        o.p = (const char*)p + r * ld * 2;
        o.rows = n;
        return o;
    }
};
inline Operand new_operand(Scratch& s, int dtype, int64_t rows, int64_t cols, int copies = 1) {
    Operand o;
    o.rows = rows;
    o.cols = cols;
    o.ld = padded(cols);
    o.plane = o.ld * rows;
    o.planes = planes_of(dtype) * copies;
    o.p = s.take((size_t)o.plane * o.planes * 2);
    return o;
}
// The caller's matrix itself where the tensor cores can read it as it is, else a copy, which `packs` has to make.
inline Operand as_operand(Scratch& s, Packs& packs, int dtype, const void* x, int64_t rows, int64_t cols, int64_t stride) {
    if (rows == 1) stride = padded(cols);
    Operand o;
    if (dtype != FRNN_F32 && on_boundary(x, 16) && stride % 8 == 0 && stride >= cols) {
        o.p = x;
        o.rows = rows;
        o.cols = cols;
        o.ld = stride;
        o.plane = rows * stride;
        o.planes = 1;
        return o;
    }
    o = new_operand(s, dtype, rows, cols);
    packs.each[packs.count++] = {x, rows, cols, stride, o.writable(), on_boundary(x, 16) && stride * dtype_bytes(dtype) % 16 == 0};
    return o;
}
inline int pack(const Packs& packs, int dtype, cudaStream_t stream) {
    if (!packs.count) return FRNN_OK;
    int64_t most = 0;
    for (int i = 0; i < packs.count; i++) most = std::max(most, packs.each[i].rows * ((packs.each[i].cols + 7) / 8));
    const dim3 grid((unsigned)std::min<int64_t>((most + 255) / 256, (int64_t)sm_count() * 16), packs.count);
    return with_dtype(dtype, [&](auto t) { return launch("matrix product: operands", pack_kernel<decltype(t)>, grid, 256, 0, stream, true, 1, packs); });
}

// ---- products --------------------------------------------------------------------------------------------------------------------

struct Product {
    ProductArgs args = {};
    int dtype;                                    // of the operands: FRNN_F32 means planes
    Operand a, b[2];
    int64_t m, n, k;
    int pairs = 1;                                // products that are added up: of a's planes (groups of them) with b[0], b[1]
    bool few = false;                             // log probabilities of a call of up to 128 rows (forward and backward cut a call into different pieces)
    void* out = nullptr;                          // STORE
    int out_dtype = 0;
    int64_t out_ld = 0;
};

struct ProductPlan {
    Form form;
    int blocks, slices;                           // of a cluster; of k beyond that
    int64_t tiles_m, tiles_n;
    size_t scratch;                               // the slices' results
    int columns() const { return form == PAIR ? 128 : form == SPLIT ? 64 / blocks : 64; }      // that a warp of the epilogue has in a row
};

// Clusters of 1, 2, 4 or 8 blocks that run at once, one block to a multiprocessor.
template <auto KERNEL> inline int clusters_at_once(int blocks) {
    static std::atomic<int> known[64][9];
    if (blocks == 1) return sm_count();
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return sm_count() / blocks; }
    int n = known[dev][blocks].load(std::memory_order_relaxed);
    if (!n) {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(blocks * sm_count());
        config.blockDim = dim3(PRODUCT_THREADS);
        config.dynamicSmemBytes = PRODUCT_SHARED;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = blocks;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        config.attrs = &attr;
        config.numAttrs = 1;
        if (!allow_shared<KERNEL>(PRODUCT_SHARED) || cudaOccupancyMaxActiveClusters(&n, KERNEL, &config) != cudaSuccess || n <= 0) n = sm_count() / blocks;
        cudaGetLastError();
        known[dev][blocks].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Which form: the one that is done first, by what was measured (ns, on a B200; 16-bit operands, then fp32, whose steps but for SPLIT are six products).  A step of 64 along k takes 285 in PAIR (for 128 x 256 in
// each block; the tensor cores' own time is 270), 215 in ALONE and 225 in SPLIT (for 128 x 128; 135, but the 32 KB that are copied for it are 78
// bytes a cycle, about what a multiprocessor takes in; 256 x 128 by a pair, 24 KB each, took 180 and was ahead by 5 % at a few sizes: left out).
// A tile leaves in `leave` (STORE, GLU_FORWARD, GLU_BACKWARD, LOGPROB_STATS, LOGPROB_GRAD), while the next one is computed; in SPLIT that
// has the exchange in it.
// Products of up to 128 rows read 16 KB of weights a step that nobody else reads: 372 when all multiprocessors do (6.5 TB/s).  THIN takes 225
// at least (the tensor cores read 128 rows of A whatever is in them).
// Measured, us: 256 x 512 of K = 2048 PAIR 14.9, ALONE 9.7, SPLIT 9.9, 8.8 and 8.8 (2, 4 and 8 blocks); K = 16384 ALONE 55, SPLIT in 4 23.
// A block of 16 rows, 4096 wide, 12288 hidden (both products): ALONE and 4 63, 2 and 4 58, 4 and 4 66; 2048 wide, 8192 hidden: ALONE and 4 29, 2 and 4 32.
// Log probabilities of 16 rows, 65536 tokens, 4096 wide: ALONE 105, SPLIT in 2 115.
inline bool is_thin(const Product& q, bool at, Form form) { return !at && (form == ALONE || form == SPLIT) && q.m <= THIN_ROWS; }
template <int EPI, bool AT, bool BT> inline ProductPlan plan_product(const Product& q) {
    static const int leave[2][3][5] = {{{3100, 5800, 10900, 4500, 5900}, {1600, 3400, 6000, 2500, 3000}, {4000, 6000, 7000, 4500, 5000}},
                                       {{5000, 20000, 26000, 4500, 12000}, {2500, 12500, 16000, 2500, 6000}, {5000, 9000, 12000, 4500, 7000}}}, step[2][3] = {{285, 215, 225}, {1650, 1150, 225}};
    const int64_t steps = (q.k + BK - 1) / BK * q.pairs, width = q.args.dual ? 2 : 1;
    const bool few = !AT && q.m <= 128, fp32 = q.dtype == FRNN_F32;
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    auto cost = [&](Form form, int blocks, int64_t tiles, int slices) {
        const int64_t at_once = clusters_at_once<product_kernel<SPLIT, false, AT, BT, EPI, true>>(blocks), rounds = up(tiles, at_once), out = leave[fp32][form][EPI];
        auto k_time = [&](int64_t tiles) {
            const bool apart = fp32 && form == SPLIT && !is_thin(q, AT, form);      // (six steps of one product)
            return up(steps * (apart ? 6 : 1), form == SPLIT ? blocks * slices : slices) * std::max<int64_t>(is_thin(q, AT, form) ? (fp32 ? 900 : 225) : step[fp32][form], few ? (!fp32 ? 1 : apart ? 2 : 3) * 372 * tiles * blocks / sm_count() : 0);
        };
        const int64_t last = k_time(tiles - (rounds - 1) * at_once), start = (form == ALONE ? 1000 : 2000) + (form == SPLIT ? 1000 * rounds : 0);      // (its blocks wait for one another)
        return rounds == 1 ? start + last + out : start + k_time(at_once) + (rounds - 2) * std::max(k_time(at_once), out) + std::max(last, out) + out;
    };
    const int64_t stack = q.args.stacked ? 2 : 1;
    ProductPlan best = {PAIR, 2, 1, up(q.m, 256) * stack, up(q.n * width, 256), 0};
    int64_t least = cost(PAIR, 2, best.tiles_m * best.tiles_n, 1);
    const int64_t tm = up(q.m, 128) * stack, tn = up(q.n * width, 128);
    for (int blocks = 1; blocks <= 8 && blocks <= steps; blocks *= 2) {
        const Form form = blocks > 1 ? SPLIT : ALONE;
        // a long sum for few tiles: slices of at least 32 steps a block, whose results (up to 32 MB) a second kernel adds up
        for (int slices = 1; slices <= (EPI == STORE && !q.args.stacked ? 32 : 1); slices *= 2) {
            const size_t scratch = slices > 1 ? (size_t)slices * q.m * padded(q.n) * 4 : 0;
            if (slices > 1 && (steps < (fp32 ? 8ll : 32ll) * blocks * slices || scratch > (32u << 20))) break;
            const int64_t c = cost(form, blocks, tm * tn * slices, slices) + (slices > 1 ? 8000 + (int64_t)(scratch >> 12) : 0);
            if (c < least) {
                least = c;
                best = {form, blocks, slices, tm, tn, scratch};
            }
        }
    }
    return best;
}

template <Form FORM, bool THIN, bool AT, bool BT, int EPI, bool FP32> inline int launch_product(const char* what, const ProductArgs& p, int blocks, cudaStream_t stream) {
    constexpr auto kernel = product_kernel<FORM, THIN, AT, BT, EPI, FP32>;
    // (the warps would wait for registers that the block does not have)
    static const bool enough = [] {
        cudaFuncAttributes a = {};
        const bool ok = cudaFuncGetAttributes(&a, kernel) == cudaSuccess && a.numRegs >= START_REGISTERS;
        cudaGetLastError();
        return ok;
    }();
    if (!enough) return frnn_fail(FRNN_E_LAUNCH, "%s: the kernel was not built for %d registers a thread, or there is no GPU to run it", what, (int)START_REGISTERS);
    if (!allow_shared<kernel>(PRODUCT_SHARED)) { cudaGetLastError(); return frnn_fail(FRNN_E_LAUNCH, "%s: no room in shared memory", what); }
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.slices, clusters = std::min<int64_t>(tiles, clusters_at_once<product_kernel<SPLIT, false, AT, BT, EPI, true>>(blocks));
    return launch(what, kernel, dim3((unsigned)(clusters * blocks)), PRODUCT_THREADS, PRODUCT_SHARED, stream, true, blocks, p);
}

// One product.  Without memory behind `s` only its scratch is counted.
template <int EPI, bool AT, bool BT> inline int run_product(const char* what, Product& q, Scratch& s, cudaStream_t stream) {
    ProductArgs& p = q.args;
    const ProductPlan plan = plan_product<EPI, AT, BT>(q);
    void* const sliced = plan.slices > 1 ? s.take(plan.scratch) : nullptr;
    if (!s.base) return FRNN_OK;
    if (plan.tiles_m * plan.tiles_n * plan.slices >= (1ll << 31)) return frnn_fail(FRNN_E_ARG, "%s: too many tiles", what);
    p.M = (int)q.m;
    p.N = (int)q.n;
    p.ksteps = (int)((q.k + BK - 1) / BK);
    p.tiles_m = (int)plan.tiles_m;
    p.tiles_n = (int)plan.tiles_n;
    p.group = plan.form == PAIR ? 16 : 32;
    p.slices = plan.slices;
    const unsigned type = q.dtype == FRNN_F16 ? 0 : 1, side = plan.form == PAIR ? 256 : 128;
    p.idesc = (1u << 4) | (type << 7) | (type << 10) | ((unsigned)AT << 15) | ((unsigned)BT << 16) | ((side >> 3) << 17) | ((side >> 4) << 24);
    const bool thin = is_thin(q, AT, plan.form), fp32 = q.dtype == FRNN_F32, fused = fp32 && (plan.form != SPLIT || thin);
    p.pairs = q.pairs;
    p.segments = q.pairs * (fp32 && !fused ? 6 : 1);
    p.flush = fused ? 1 : fp32 ? 4 : EPI != LOGPROB_STATS && EPI != LOGPROB_GRAD ? 64 : q.few ? 4 : 16;
    if ((int64_t)p.ksteps * p.segments >= (1ll << 31) - 64) return frnn_fail(FRNN_E_ARG, "%s: too long", what);
    auto encode = [&](CUtensorMap& map, const Operand& o, bool across, unsigned high) {
        return frnn_tensor_map_swizzled(&map, o.p, o.cols, o.rows, o.planes, (uint64_t)o.ld * 2, (uint64_t)o.plane * 2, 64, across ? 64 : high);
    };
    int rc = encode(p.a, q.a, AT, thin ? THIN_ROWS : 128);
    for (int i = 0; i < 2 && rc == FRNN_OK; i++) {
        if (i && !q.b[1].p) p.b[1] = p.b[0];
        else rc = encode(p.b[i], q.b[i], BT, p.dual && plan.form != PAIR ? 64 : 128);
    }
    if (rc != FRNN_OK) return rc;
    p.out = q.out;
    p.out_dtype = q.out_dtype;
    p.out_ld = q.out_ld;
    const float *const add = p.add, *const alpha = p.alpha;
    if (sliced) {
        p.out = sliced;
        p.out_dtype = FRNN_F32;
        p.out_ld = padded(q.n);
        p.out_slice = q.m * p.out_ld;
        p.add = p.alpha = nullptr;
    }
    p.out_wide = on_boundary(p.out, 16) && on_boundary(p.out2, 16) && p.out_ld * (int64_t)dtype_bytes(p.out_dtype) % 16 == 0;
    auto run = [&](auto form, auto rows) {
        constexpr Form FORM = decltype(form)::value;
        constexpr bool THIN = decltype(rows)::value;
        return q.dtype == FRNN_F32 ? launch_product<FORM, THIN, AT, BT, EPI, true>(what, p, plan.blocks, stream) : launch_product<FORM, THIN, AT, BT, EPI, false>(what, p, plan.blocks, stream);
    };
    const std::false_type all;
    const std::true_type few;
    if (plan.form == PAIR) rc = run(std::integral_constant<Form, PAIR>(), all);
    else if (!thin) rc = plan.form == ALONE ? run(std::integral_constant<Form, ALONE>(), all) : run(std::integral_constant<Form, SPLIT>(), all);
    else if constexpr (!AT) rc = plan.form == ALONE ? run(std::integral_constant<Form, ALONE>(), few) : run(std::integral_constant<Form, SPLIT>(), few);
    if (rc != FRNN_OK || !sliced) return rc;
    p.add = add;
    p.alpha = alpha;
    const int64_t blocks = std::min<int64_t>((q.m * ((q.n + 3) / 4) + 255) / 256, (int64_t)sm_count() * 8);
    return launch(what, join_slices, dim3((unsigned)blocks), 256, 0, stream, true, 1, p, q.out, q.out_dtype, q.out_ld);
}

}  // namespace frnn_lm
