// Embedding lookup with scaling, and its gradient by sorted tokens.
//
// The lookup moves rows and is bound by memory.  The gradient is dense: most of its bytes are the rows of tokens that do
// not occur.  Two kernels run side by side, therefore: in `embedding_sort` one cluster of blocks sorts the tokens (places
// of equal tokens stay in order), and `embedding_fill` writes the zero rows, for which it only has to know which tokens
// occur.  `embedding_sums` then walks over the sorted places in chunks of one length, whatever the frequencies of the tokens (a
// text's most frequent token has hundreds of times its average share): runs of equal tokens inside a chunk are finished
// there, those that cross its ends leave a partial sum each, which `embedding_join` adds.  The order of a sum follows from
// where its token stands and from the chunks' length (sizes, number of SMs), never from how threads are scheduled.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "frnn_lm.cuh"

using namespace frnn_lm;
namespace cg = cooperative_groups;

namespace {

enum { BLOCK = 256, UNROLL = 8 };

// How rows are accessed.  ALIKE: all of them at 16-byte boundaries, in accesses of 16 bytes.  APART: rows at any distances
// behind boundaries; a thread's columns follow the boundaries of the row that is written, the row that is read comes in
// two accesses and shifts.  ELEMENTS: one element at a time (columns that are not consecutive).
enum Access { ALIKE, APART, ELEMENTS };

template <class T, Access A> constexpr int EACH = A == ELEMENTS ? 1 : WIDE<T>;

// How a block's threads stand to rows: `lanes` threads (a power of two, all of the block for wide rows) have E columns
// each, blockIdx.y counts the parts of rows wider than that.
struct Shape {
    int lanes, groups;         // threads of a group, groups of a block
    unsigned parts;            // blocks side by side over a row's columns
};

template <class T, Access A> Shape shape_of(int64_t width) {
    constexpr int E = EACH<T, A>;
    const int64_t vectors = (width + (A == APART ? E - 1 : 0) + E - 1) / E;
    Shape s{1, 1, 1};
    while (s.lanes < BLOCK && s.lanes < vectors) s.lanes *= 2;
    s.groups = BLOCK / s.lanes;
    s.parts = (unsigned)((vectors + s.lanes - 1) / s.lanes);
    return s;
}

// First of a thread's columns of a row that is written at `row`, thread `t` along the row.
template <class T, Access A> __device__ __forceinline__ int column(const T* row, unsigned t) {
    return (int)t * EACH<T, A> - (A == APART ? (int)((uintptr_t)row & 15) / (int)sizeof(T) : 0);
}

template <class T, Access A> __device__ __forceinline__ void write_columns(const Pack<T, EACH<T, A>>& v, T* row, int c, int width) {
    if (A != APART) {
        if (c < width) v.store(row + c);
    } else {
        store_part(v, row, c, width);
    }
}

// y_i = scale * W[t_i]; a zero row where t_i is ignored or (reported) outside the vocabulary.  A group takes UNROLL / 2
// rows, whose loads are all under way before the first is used.  Bound by memory: 8192 rows of 4096 bf16 in 18.7 us, 64 MB
// written and about 20 MB of distinct rows read (4.5 TB/s); 16384 of 1001 in 21 us (one element at a time: 33).
template <class T, Access A>
__global__ void __launch_bounds__(BLOCK) embedding_fw(const T* __restrict__ w, int64_t rows, int width, int64_t row_stride, int64_t col_stride, const void* __restrict__ tokens,
                                                      int token_bytes, int n, float scale, int64_t ignore, T* __restrict__ out, int* err, Shape shape) {
    constexpr int ROWS = UNROLL / 2, E = EACH<T, A>;
    const unsigned t = blockIdx.y * shape.lanes + threadIdx.x % shape.lanes;
    const int first = (blockIdx.x * shape.groups + threadIdx.x / shape.lanes) * ROWS;
    const T* end = w + (rows - 1) * row_stride + width;
    Pack<T, E> v[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        v[u].zero();
        if (first + u >= n) continue;
        const int64_t k = token_at(tokens, token_bytes, first + u);
        const bool there = k != ignore && k >= 0 && k < rows;
        if (k != ignore && !there && t == 0) *err = CODE_TOKEN;
        if (!there) continue;
        const T* row = w + k * row_stride;
        const int c = column<T, A>(out + (int64_t)(first + u) * width, t);
        if constexpr (A == APART) {
            if (c >= 0 && c + E <= width) load_anywhere(v[u], row + c, w, end);
            else
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (c + e >= 0 && c + e < width) v[u].set(e, row[c + e]);
        } else if (c < width) {
            v[u].load(row + (A == ELEMENTS ? c * col_stride : c));
        }
    }
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
        if (first + u >= n) return;
        float f[E];
        v[u].to(f);
#pragma unroll
        for (int e = 0; e < E; e++) f[e] *= scale;
        v[u].from(f);
        T* to = out + (int64_t)(first + u) * width;
        write_columns<T, A>(v[u], to, column<T, A>(to, t), width);
    }
}

// Tokens that take no part (ignored, outside the vocabulary) get the key `rows`, behind all others.
__device__ __forceinline__ unsigned key_of(const void* tokens, int bytes, int64_t i, int64_t rows, int64_t ignore) {
    const int64_t t = token_at(tokens, bytes, i);
    return t != ignore && t >= 0 && t < rows ? (unsigned)t : (unsigned)rows;
}

enum { CLUSTER = 8, SORT_THREADS = 1024, WARPS = SORT_THREADS / 32, MOST_BITS = 9, DIGITS = 1 << MOST_BITS, ROUNDS = 4, FLAGS = 32768 };

// Zeros into the bytes [lo, hi) of p, by the lanes of a warp; lo, hi and p are on boundaries of elements of `size` bytes.
__device__ __forceinline__ void fill_zero(char* p, int64_t lo, int64_t hi, int size) {
    const int lane = threadIdx.x & 31;
    const int64_t head = min(hi, lo + (int64_t)(-(uintptr_t)(p + lo) & 15)), tail = max(head, hi - (int64_t)((uintptr_t)(p + hi) & 15));
    for (int64_t i = head + 16 * lane; i < tail; i += 512) *(uint4*)(p + i) = make_uint4(0, 0, 0, 0);
    if (size == 4) {
        if (lo + 4 * lane < head) *(unsigned*)(p + lo + 4 * lane) = 0;
        if (tail + 4 * lane < hi) *(unsigned*)(p + tail + 4 * lane) = 0;
    } else {
        if (lo + 2 * lane < head) *(unsigned short*)(p + lo + 2 * lane) = 0;
        if (tail + 2 * lane < hi) *(unsigned short*)(p + tail + 2 * lane) = 0;
    }
}

// Zero rows for the tokens that do not occur: each block has a range of rows and looks through all tokens for it, so it
// waits for no sort.  Bound by writes: 0.5 GB in 77 to 81 us, 6.6 TB/s.
__global__ void __launch_bounds__(SORT_THREADS, 1)
embedding_fill(const void* __restrict__ tokens, int token_bytes, int n, int64_t rows, int64_t ignore, char* dw, int64_t row_bytes, int size) {
    extern __shared__ unsigned char occurs[];                  // of FLAGS rows
    const int warp = threadIdx.x / 32;
    cudaTriggerProgrammaticLaunchCompletion();
    const int64_t each = (rows + gridDim.x - 1) / gridDim.x, from = blockIdx.x * each, to = min(rows, from + each);
    for (int64_t lo = from; lo < to; lo += FLAGS) {
        const int here = (int)min((int64_t)FLAGS, to - lo);
        __syncthreads();
        for (int i = threadIdx.x; i < here; i += SORT_THREADS) occurs[i] = 0;
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += SORT_THREADS) {
            const int64_t t = token_at(tokens, token_bytes, i);
            if (t >= lo && t < lo + here && t != ignore) occurs[t - lo] = 1;
        }
        __syncthreads();
        // a warp takes 32 rows and fills each run of them in one go
        for (int i = 32 * warp; i < here; i += 32 * WARPS) {
            const int lane = threadIdx.x & 31;
            unsigned absent = __ballot_sync(~0u, i + lane < here && !occurs[i + lane]);
            while (absent) {
                const int first = __ffs(absent) - 1, ones = __ffs(~(absent >> first)) - 1, last = ones < 0 ? 32 : first + ones;      // (ones: 32 of them have no end)
                fill_zero(dw, (lo + i + first) * row_bytes, (lo + i + last) * row_bytes, size);
                absent = last >= 32 ? 0 : absent & (~0u << last);
            }
        }
    }
    cudaGridDependencySynchronize();                           // not done before the sort is: the next kernel waits for this one
}

// One cluster: stable radix sort of (token, place) by token, `bits` bits a pass.  Each warp takes a contiguous part of the
// places, 32 a round; a place's rank is what comes before it in its round, its warp, its block, its cluster and among the
// smaller digits.  Bound by latency (barriers of the cluster, scattered stores of 8 bytes): 10 us for 16 tokens, 15 us for
// 16384 in two passes; behind the zero rows of a large vocabulary it costs nothing.
__global__ void __launch_bounds__(SORT_THREADS, 1)
embedding_sort(const void* __restrict__ tokens, int token_bytes, int n, int64_t rows, int64_t ignore, int passes, int bits, uint2* a, uint2* b) {
    extern __shared__ unsigned count[];                        // [WARPS][DIGITS]
    __shared__ unsigned total[DIGITS], carry[WARPS];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    cudaTriggerProgrammaticLaunchCompletion();                 // `embedding_fill` needs nothing from here
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = blockIdx.x, mask = (1u << bits) - 1, digits = 1u << bits;
    const int64_t part = (((int64_t)n + CLUSTER * WARPS - 1) / (CLUSTER * WARPS) + 31) / 32 * 32;
    const int lo = (int)min((int64_t)n, (int64_t)(rank * WARPS + warp) * part), hi = (int)min((int64_t)n, lo + part);
    unsigned* mine = count + warp * DIGITS;
    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * bits;
        const uint2* from = pass & 1 ? b : a;
        uint2* to = pass & 1 ? a : b;                          // a token and its place together: one scattered store, not two
        // the buffers were written by other SMs: read past this one's L1
        auto pair = [&](int i) { return pass ? __ldcg(from + i) : make_uint2(key_of(tokens, token_bytes, i, rows, ignore), (unsigned)i); };
        for (int i = lane; i < digits; i += 32) mine[i] = 0;
        __syncwarp();
        for (int i0 = lo + lane; i0 < hi; i0 += 32 * ROUNDS) {
            unsigned k[ROUNDS];
#pragma unroll
            for (int u = 0; u < ROUNDS; u++) k[u] = i0 + 32 * u < hi ? pair(i0 + 32 * u).x : 0;
#pragma unroll
            for (int u = 0; u < ROUNDS; u++)
                if (i0 + 32 * u < hi) atomicAdd(&mine[(k[u] >> shift) & mask], 1u);
        }
        __syncthreads();
        unsigned all = 0, below = 0;
        const int d = threadIdx.x;
        if (d < digits) {
            unsigned sum = 0;
#pragma unroll 8
            for (int k = 0; k < WARPS; k++) { const unsigned c = count[k * DIGITS + d]; count[k * DIGITS + d] = sum; sum += c; }
            total[d] = sum;
        }
        cluster.sync();
        if (d < digits)
#pragma unroll
            for (int k = 0; k < CLUSTER; k++) {
                const unsigned c = cluster.map_shared_rank(total, k)[d];
                if (k < rank) below += c;
                all += c;
            }
        cluster.sync();                                        // everyone has read `total`; it takes the digits' bases next
        unsigned scan = all;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const unsigned v = __shfl_up_sync(~0u, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) carry[warp] = scan;
        __syncthreads();
        unsigned before = 0;
#pragma unroll
        for (int k = 0; k < DIGITS / 32; k++) before += k < warp ? carry[k] : 0;
        if (d < digits) total[d] = before + scan - all + below;
        __syncthreads();
        for (int i0 = lo + lane; i0 < hi + lane; i0 += 32 * ROUNDS) {
            uint2 k[ROUNDS];
#pragma unroll
            for (int u = 0; u < ROUNDS; u++) k[u] = i0 + 32 * u < hi ? pair(i0 + 32 * u) : make_uint2(0, 0);
#pragma unroll
            for (int u = 0; u < ROUNDS; u++) {
                if (i0 - lane + 32 * u >= hi) break;
                const bool in = i0 + 32 * u < hi;
                const unsigned digit = in ? (k[u].x >> shift) & mask : digits;
                const unsigned same = __match_any_sync(~0u, digit), earlier = same & ((1u << lane) - 1);
                if (in) to[total[digit] + mine[digit] + __popc(earlier)] = k[u];
                __syncwarp();
                if (in && !earlier) mine[digit] += __popc(same);
                __syncwarp();
            }
        }
        cluster.sync();
    }
}

enum : unsigned { NO_KEY = 0xFFFFFFFFu };

// The E columns from c on of a row of `width`, zeros where there are none: `fetch` starts the loads, `get` waits for them,
// so that those of several rows are under way at once.  [begin, end): the tensor.  APART reads the 32 aligned bytes around
// its columns, which may hold other rows' elements but nothing outside of the tensor: there, one element at a time.
template <class T, Access A> struct Reader {
    static constexpr int E = EACH<T, A>;
    Pack<T, E> v;
    __device__ __forceinline__ void fetch(const T* row, int c, int width, const T*, const T*, bool there) {
        v.zero();
        if (there && c < width) v.load(row + c);
    }
    __device__ __forceinline__ void get(Pack<T, E>& to) const { to = v; }
};
template <class T> struct Reader<T, APART> {
    static constexpr int E = WIDE<T>;
    uint4 low, high;
    const T* row;
    int c, width;             // width: 0 where there is no row
    bool wide;
    __device__ __forceinline__ void fetch(const T* row_, int c_, int width_, const T* begin, const T* end, bool there) {
        row = row_;
        c = c_;
        width = there ? width_ : 0;
        const T* from = row + c - ((uintptr_t)(row + c) & 15) / sizeof(T);
        wide = there && c < width && from >= begin && from + 2 * E <= end;
        if (wide) {
            low = *(const uint4*)from;
            high = *(const uint4*)(from + E);
        }
    }
    __device__ __forceinline__ void get(Pack<T, E>& to) const {
        if (!wide) {
#pragma unroll
            for (int e = 0; e < E; e++) to.set(e, c + e >= 0 && c + e < width ? row[c + e] : from_float<T>(0.f));
            return;
        }
        shift_out(to, low, high, (unsigned)((uintptr_t)(row + c) & 15) / (unsigned)sizeof(T));
        if (c < 0 || c + E > width)
#pragma unroll
            for (int e = 0; e < E; e++)
                if (c + e < 0 || c + e >= width) to.set(e, from_float<T>(0.f));
    }
};
// A group sums a chunk of the sorted places, with 8 rows under way (4 where each takes two accesses).  8192 rows of 4096 bf16
// in 27 us behind 0.5 GB of zeros that still drain from the L2 cache, 16384 of 1000 in 17 us (33 MB, 1.9 TB/s): places and
// then rows are two loads in a row of which each thread has one or two rounds.  part: [chunks][2][pitch] (pitch: the width's next multiple of 4), sums of the
// run that came in over the chunk's start and of the one that goes on over its end.
template <class T, Access A>
__global__ void __launch_bounds__(BLOCK) embedding_sums(const T* __restrict__ dy, const uint2* __restrict__ sorted, int n, unsigned rows, int width,
                                                        int chunk, float scale, T* __restrict__ dw, float* __restrict__ part, Shape shape) {
    constexpr int E = EACH<T, A>;
    const unsigned t = blockIdx.y * shape.lanes + threadIdx.x % shape.lanes;
    const int64_t mine = (int64_t)blockIdx.x * shape.groups + threadIdx.x / shape.lanes, from = mine * chunk;
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    if (from >= n || (int)t * E >= width + (A == APART ? E - 1 : 0)) return;
    const int lo = (int)from, hi = (int)min((int64_t)n, from + chunk), pitch = (width + 3) & ~3;
    const T* end = dy + (int64_t)n * width;
    unsigned run = sorted[lo].x;
    bool came_in = lo > 0 && sorted[lo - 1].x == run;
    const unsigned after = hi < n ? sorted[hi].x : NO_KEY;
    float sum[E] = {};
    auto finish = [&](bool goes_on) {
        T* row = dw + (int64_t)run * width;
        const int c = column<T, A>(row, t);
        if (came_in || goes_on) {
            float* to = part + (2 * mine + !came_in) * pitch;
            if (A == ALIKE) {
#pragma unroll
                for (int e = 0; e < E; e += 4) *(float4*)(to + c + e) = make_float4(sum[e], sum[e + 1], sum[e + 2], sum[e + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (c + e >= 0 && c + e < width) to[c + e] = sum[e];
            }
            return;
        }
        float f[E];
#pragma unroll
        for (int e = 0; e < E; e++) f[e] = scale * sum[e];
        Pack<T, E> v;
        v.from(f);
        write_columns<T, A>(v, row, c, width);
    };
    constexpr int ROUND = A == APART ? UNROLL / 2 : UNROLL;       // rows under way at once
    uint2 next[ROUND];
    auto look = [&](int j) {
#pragma unroll
        for (int u = 0; u < ROUND; u++) next[u] = j + u < hi ? sorted[j + u] : make_uint2(NO_KEY, 0);
    };
    look(lo);
    for (int j = lo; j < hi && run < rows; j += ROUND) {
        unsigned k[ROUND];
        Reader<T, A> in[ROUND];
#pragma unroll
        for (int u = 0; u < ROUND; u++) {
            k[u] = next[u].x;
            const bool there = k[u] < rows;
            in[u].fetch(dy + (int64_t)next[u].y * width, column<T, A>(dw + (int64_t)(there ? k[u] : 0) * width, t), width, dy, end, there);
        }
        look(j + ROUND);                                  // the next round's places, while these rows are on their way
#pragma unroll
        for (int u = 0; u < ROUND; u++) {
            if (j + u < hi && k[u] != run) {
                if (run < rows) finish(false);
                run = k[u];
                came_in = false;
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] = 0;
            }
            Pack<T, E> v;
            float f[E];
            in[u].get(v);
            v.to(f);
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] += f[e];
        }
    }
    if (run < rows) finish(after == run);
}

// Sums of the runs that cross ends of chunks.  A block looks at JOINED chunks for runs that start there and go on.  A run of
// few partial sums is added in their order by one warp, several runs side by side; a longer one by the block, 64 threads with
// 4 columns each and 4 slices of the partial sums (every fourth one), which are added last.  Bound by latency: 10 us for 512 chunks of
// 4096 columns, most of it three loads that wait for one another.
enum { JOINED = BLOCK / 32, FEW = 16 };
template <class T>
__global__ void __launch_bounds__(BLOCK) embedding_join(const uint2* __restrict__ sorted, int n, unsigned rows, int width, int chunk, float scale, T* __restrict__ dw,
                                                        const float* __restrict__ part) {
    constexpr int LANES = 64, SLICES = BLOCK / LANES;
    __shared__ float4 share[SLICES][LANES];
    __shared__ unsigned runs[JOINED];
    __shared__ int64_t ends[JOINED];                      // the last chunk that the run reaches
    cudaGridDependencySynchronize();
    {
        const int r = threadIdx.x / 32, lane = threadIdx.x & 31;
        const int64_t q = (int64_t)blockIdx.x * JOINED + r, lo = q * chunk, hi = lo + chunk;
        unsigned run = NO_KEY;
        if (hi < n) {
            const unsigned over = sorted[hi].x, last = sorted[hi - 1].x, before = lo > 0 ? sorted[lo - 1].x : NO_KEY;
            if (over < rows && last == over && before != over) run = over;
        }
        int64_t last = q;
        while (run != NO_KEY) {
            const int64_t next = last + 1 + lane;
            const int more = __popc(__ballot_sync(~0u, next * chunk < n && sorted[next * chunk].x == run));      // sorted: the first `more` of them
            last += more;
            if (more < 32) break;
        }
        const bool few = run != NO_KEY && last - q < FEW;
        if (lane == 0) {
            runs[r] = few ? NO_KEY : run;
            ends[r] = last;
        }
        if (few)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int c = (int)(blockIdx.y * 64 + half * 32 + lane) * 4, pitch = (width + 3) & ~3;
                if (c >= width) continue;
                float4 sum = *(const float4*)(part + (2 * q + 1) * pitch + c);      // (columns behind the width are read and dropped)
#pragma unroll 8
                for (int64_t k = q + 1; k <= last; k++) {
                    const float4 v = *(const float4*)(part + 2 * k * pitch + c);
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                T* to = dw + (int64_t)run * width + c;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (c + e < width) to[e] = from_float<T>(scale * (&sum.x)[e]);
            }
    }
    __syncthreads();
    for (int r = 0; r < JOINED; r++) {
        const unsigned run = runs[r];
        if (run == NO_KEY) continue;
        const int64_t mine = (int64_t)blockIdx.x * JOINED + r, last = ends[r];
        const int lane = threadIdx.x % LANES, slice = threadIdx.x / LANES, c = (int)(blockIdx.y * LANES + lane) * 4, pitch = (width + 3) & ~3;
        float4 sum = make_float4(0, 0, 0, 0);
        if (c < width)
#pragma unroll 8
            for (int64_t q = mine + slice; q <= last; q += SLICES) {
                const float4 v = *(const float4*)(part + (2 * q + (q == mine)) * pitch + c);      // (columns behind the width are read and dropped)
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
        share[slice][lane] = sum;
        __syncthreads();
        const int col = blockIdx.y * LANES * 4 + threadIdx.x;
        if (col < width) {
            float total = 0;
#pragma unroll
            for (int k = 0; k < SLICES; k++) total += ((const float*)share[k])[threadIdx.x];
            dw[(int64_t)run * width + col] = from_float<T>(scale * total);
        }
        __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------

struct Plan {
    int passes, bits;          // of the sort
    int chunk;                 // places of a chunk: 8 to 128, so that about eight blocks an SM have one
    int64_t chunks;
    size_t at_parts, bytes;    // of the workspace: where the partial sums are, all of it
};

Plan plan_of(int dtype, int64_t rows, int64_t width, int64_t n) {
    Plan p;
    int all = 1;
    while ((rows >> all) != 0) all++;          // the keys are 0 .. rows
    p.passes = (all + MOST_BITS - 1) / MOST_BITS;
    p.bits = (all + p.passes - 1) / p.passes;
    const double blocks = (double)n * width * dtype_bytes(dtype) / (16 * BLOCK);       // blocks' worth of places, with 16 bytes a thread
    for (p.chunk = 8; p.chunk < 128 && blocks / p.chunk > 8.0 * sm_count(); p.chunk *= 2) {}
    p.chunks = (n + p.chunk - 1) / p.chunk;
    p.at_parts = ((size_t)n * 16 + 255) / 256 * 256;
    p.bytes = p.at_parts + (size_t)p.chunks * 2 * ((width + 3) & ~3ll) * 4;
    return p;
}

int bad_shape(const char* what, int dtype, int64_t rows, int64_t width, int token_bytes, int64_t n) {
    if (!dtype_known(dtype) || (token_bytes != 4 && token_bytes != 8)) return frnn_fail(FRNN_E_ARG, "%s: unknown data type", what);
    if (rows < 0 || width < 0 || n < 0 || rows >= (1ll << 31) || width >= (1ll << 21) || n >= (1ll << 30))
        return frnn_fail(FRNN_E_ARG, "%s: the vocabulary has to be below 2^31, the width below 2^21, the number of tokens below 2^30", what);
    return FRNN_OK;
}

enum { SORT_SHARED = WARPS * DIGITS * 4, FILL_BLOCKS = 128 };

// Calls f(T(), integral_constant A).
template <class F> int with_access(int dtype, Access access, F f) {
    return with_dtype(dtype, [&](auto t) {
        switch (access) {
            case ALIKE: return f(t, std::integral_constant<Access, ALIKE>());
            case APART: return f(t, std::integral_constant<Access, APART>());
            default: return f(t, std::integral_constant<Access, ELEMENTS>());
        }
    });
}

}  // namespace

extern "C" {

int frnn_embedding_forward(int dtype, const void* weight, int64_t rows, int64_t width, int64_t row_stride, int64_t col_stride, const void* tokens, int token_bytes,
                           int64_t n, float scale, int64_t ignore_index, void* out, int* err_word, void* stream) {
    if (int rc = bad_shape("frnn_embedding_forward", dtype, rows, width, token_bytes, n)) return rc;
    if (n == 0 || width == 0) return FRNN_OK;
    if ((!weight && rows) || !tokens || !out || !err_word) return frnn_fail(FRNN_E_ARG, "frnn_embedding_forward: bad argument");
    const size_t size = dtype_bytes(dtype);
    if (!on_boundary(weight, size) || !on_boundary(out, size) || !on_boundary(tokens, token_bytes) || !on_boundary(err_word, 4))
        return frnn_fail(FRNN_E_ARG, "frnn_embedding_forward: a pointer is not on a boundary of its elements");
    const bool alike = width * size % 16 == 0 && row_stride * (int64_t)size % 16 == 0 && on_boundary(weight, 16) && on_boundary(out, 16);
    return with_access(dtype, col_stride != 1 ? ELEMENTS : alike ? ALIKE : APART, [&](auto t, auto a) {
        typedef decltype(t) T;
        const Shape shape = shape_of<T, a.value>(width);
        const int64_t each = shape.groups * (UNROLL / 2);
        embedding_fw<T, a.value><<<dim3((unsigned)((n + each - 1) / each), shape.parts), BLOCK, 0, (cudaStream_t)stream>>>(
            (const T*)weight, rows, (int)width, row_stride, col_stride, tokens, token_bytes, (int)n, scale, ignore_index, (T*)out, err_word, shape);
        return launched("frnn_embedding_forward");
    });
}

size_t frnn_embedding_backward_workspace(int dtype, int64_t rows, int64_t width, int64_t n) {
    return n <= 0 || rows <= 0 || width <= 0 || bad_shape("frnn_embedding_backward_workspace", dtype, rows, width, 8, n) ? 0 : plan_of(dtype, rows, width, n).bytes;
}

int frnn_embedding_backward(int dtype, const void* dout, const void* tokens, int token_bytes, int64_t n, int64_t rows, int64_t width, float scale,
                            int64_t ignore_index, void* dweight, void* workspace, void* stream) {
    if (int rc = bad_shape("frnn_embedding_backward", dtype, rows, width, token_bytes, n)) return rc;
    if (rows == 0 || width == 0) return FRNN_OK;
    if (!dweight || (n && (!dout || !tokens || !workspace))) return frnn_fail(FRNN_E_ARG, "frnn_embedding_backward: bad argument");
    const size_t size = dtype_bytes(dtype);
    if (!on_boundary(dout, size) || !on_boundary(dweight, size) || !on_boundary(tokens, token_bytes) || !on_boundary(workspace, 16))
        return frnn_fail(FRNN_E_ARG, "frnn_embedding_backward: a pointer is not on a boundary of its elements (the workspace: of 16 bytes)");
    const cudaStream_t st = (cudaStream_t)stream;
    const Plan plan = plan_of(dtype, rows, width, n);
    uint2* pairs = (uint2*)workspace;
    float* part = n ? (float*)((char*)workspace + plan.at_parts) : nullptr;
    if (n) {
        // 8 blocks: 16 sort 32768 tokens 5 us faster, but then fewer blocks fill (0.5 GB of zeros and 8192 tokens: 116 us, with 16 blocks 128)
        if (!allow_shared<embedding_sort>(SORT_SHARED)) return launched("frnn_embedding_backward");
        if (int rc = launch("frnn_embedding_backward", embedding_sort, dim3(CLUSTER), SORT_THREADS, SORT_SHARED, st, false, CLUSTER, tokens, token_bytes, (int)n, rows, ignore_index,
                            plan.passes, plan.bits, pairs, pairs + n))
            return rc;
    }
    // 64 KB of zeros for each block, and at most 128 blocks: with more, the same bytes took longer (0.5 GB: 78 us, with 136 to 296 blocks 89)
    const int64_t fill = rows * width * (int64_t)size / (1 << 16) + 1;
    if (int rc = launch("frnn_embedding_backward", embedding_fill, dim3((unsigned)std::min<int64_t>(fill, FILL_BLOCKS)), SORT_THREADS, FLAGS, st, n > 0, 1, tokens, token_bytes, (int)n,
                        rows, ignore_index, (char*)dweight, width * (int64_t)size, (int)size))
        return rc;
    if (n == 0) return FRNN_OK;
    const uint2* sorted = pairs + (plan.passes & 1) * n;
    const bool alike = width * size % 16 == 0 && on_boundary(dout, 16) && on_boundary(dweight, 16);
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        auto run = [&](auto a) {
            const Shape shape = shape_of<T, a.value>(width);
            if (int rc = launch("frnn_embedding_backward", embedding_sums<T, a.value>, dim3((unsigned)((plan.chunks + shape.groups - 1) / shape.groups), shape.parts), BLOCK, 0, st, true, 1,
                                (const T*)dout, sorted, (int)n, (unsigned)rows, (int)width, plan.chunk, scale, (T*)dweight, part, shape))
                return rc;
            if (plan.chunks < 2) return (int)FRNN_OK;
            return launch("frnn_embedding_backward", embedding_join<T>, dim3((unsigned)((plan.chunks + JOINED - 1) / JOINED), (unsigned)((width + 255) / 256)), BLOCK, 0, st, true, 1, sorted,
                          (int)n, (unsigned)rows, (int)width, plan.chunk, scale, (T*)dweight, (const float*)part);
        };
        return alike ? run(std::integral_constant<Access, ALIKE>()) : run(std::integral_constant<Access, APART>());
    });
}

}  // extern "C"
