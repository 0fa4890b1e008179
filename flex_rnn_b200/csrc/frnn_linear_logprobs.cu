// Log probabilities of tokens and entropies of softmax(x W^T / T), without keeping the logits (frnn_product.cuh).
//
// With u = log2(e) / T x W^T, of each row in blocks of columns: m = max u, s = sum 2^(u - m), t = sum 2^(u - m) (u - m), from
// the tile that leaves Tensor Memory; a second kernel joins the blocks:
//   log p[token] = ln 2 ((u[token] - m) - log2 s),   H = ln 2 (log2 s - t / s)
// Backward, a piece of the vocabulary at a time: the logits again, their gradient
//   G = (g (1[v = token] - p) - h p (ln p + H)) / T
// as a 16-bit operand (in one rounding; up to 128 rows in two planes, see there; fp32 in three), dx += G W, dW of the piece = G^T x.  2 n V D operations forward, 6 n V D backward (2 of them for the
// logits that were not kept).
#include "frnn_product.cuh"

using namespace frnn_lm;

namespace {

// Rows of partial results [blocks][3][n] joined: SLICES threads a row take every SLICES-th block, four at a time so that their
// loads are under way together, then their results in order.  32 rows a block where there are many (whole lines of the
// partial results), 8 and more threads to each where there are few.
template <int JOIN_ROWS, int JOIN_SLICES>
__global__ void __launch_bounds__(JOIN_ROWS* JOIN_SLICES) join_kernel(const float* partial, const float* target, int64_t blocks, int64_t n, const void* tokens, int token_bytes, int64_t vocab,
                                                                      int64_t ignore_index, float* logprob, float* entropy, float* stats, int* err) {
    __shared__ float part[3][JOIN_SLICES][JOIN_ROWS];
    cudaGridDependencySynchronize();
    const int r = threadIdx.x % JOIN_ROWS, slice = threadIdx.x / JOIN_ROWS;
    const int64_t row = (int64_t)blockIdx.x * JOIN_ROWS + r;
    const float lowest = -3.4028235e38f;
    float m = lowest, s = 0.f, t = 0.f;
    auto add = [&](float m2, float s2, float t2) {
        const float top = fmaxf(m, m2), d1 = exp2_fast(m - top), d2 = exp2_fast(m2 - top);
        t = (s == 0.f ? 0.f : d1 * (t + s * (m - top))) + (s2 == 0.f ? 0.f : d2 * (t2 + s2 * (m2 - top)));
        s = d1 * s + d2 * s2;
        m = top;
    };
    if (row < n)
        for (int64_t b = slice; b < blocks; b += 4 * JOIN_SLICES) {
            float v[4][3];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool there = b + k * JOIN_SLICES < blocks;
                const float* p = partial + (b + k * JOIN_SLICES) * 3 * n + row;
                v[k][0] = there ? p[0] : lowest;
                v[k][1] = there ? p[n] : 0.f;
                v[k][2] = there ? p[2 * n] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; k++) add(v[k][0], v[k][1], v[k][2]);
        }
    part[0][slice][r] = m;
    part[1][slice][r] = s;
    part[2][slice][r] = t;
    for (int half = JOIN_SLICES / 2; half; half /= 2) {
        __syncthreads();
        if (slice < half) {
            add(part[0][slice + half][r], part[1][slice + half][r], part[2][slice + half][r]);
            part[0][slice][r] = m;
            part[1][slice][r] = s;
            part[2][slice][r] = t;
        }
    }
    if (slice || row >= n) return;
    const bool empty = s == 0.f;
    const float lse2 = empty ? -INFINITY : m + log2f(s), h = empty ? 0.f : 0.69314718055994531f * (log2f(s) - t / s);
    const int64_t token = token_at(tokens, token_bytes, row);
    float lp = 0.f;
    if (token != ignore_index) {
        const bool inside = token >= 0 && token < vocab;
        // (u - m first: of the likeliest token it is 0, and what is left as exact as s, whatever m; from lse2, at m of some tens, 2^-19 is lost)
        lp = inside ? (empty ? -INFINITY : 0.69314718055994531f * ((target[row] - m) - log2f(s))) : NAN;
        if (!inside) frnn_report(err, CODE_TOKEN);
    }
    logprob[row] = lp;
    entropy[row] = h;
    if (stats) {
        stats[2 * row] = lse2;
        stats[2 * row + 1] = h;
    }
}

// A power of two that brings the logits' gradient, at most (|g| + (ln V + 1) |h|) / T, up to 2^13, and its inverse: fp16 has
// normal numbers from 2^-14 to 2^16, and most of the gradient lies many powers below its largest values.  Counted is what reaches
// the logits: g only where the token is not ignored (whatever stands there, it is no gradient), and no row whose gradients are not
// finite (its own results are lost at any scale, the other rows' are not).
__global__ void __launch_bounds__(1024) range_kernel(const float* g, const float* h, const void* tokens, int token_bytes, int64_t ignore_index, int64_t n, float inv_t, float* out) {
    __shared__ float part[32];
    float most = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        const float a = g && token_at(tokens, token_bytes, i) != ignore_index ? fabsf(g[i]) : 0.f, b = (a + 23.f * (h ? fabsf(h[i]) : 0.f)) * inv_t;
        if (b < INFINITY) most = fmaxf(most, b);
    }
    for (int d = 16; d; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = most;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < 32; i++) most = fmaxf(most, part[i]);
    int e = 0;
    if (most > 0.f) e = max(-100, min(100, 13 - ilogbf(most)));
    out[0] = ldexpf(1.f, e);
    out[1] = ldexpf(1.f, -e);
}

int check(const char* what, const frnn_linear_logprobs_call* c) {
    if (!c || !dtype_known(c->dtype) || (c->token_bytes != 4 && c->token_bytes != 8) || !c->x || !c->weight || !c->tokens || !on_boundary(c->tokens, c->token_bytes))
        return frnn_fail(FRNN_E_ARG, "%s: bad argument", what);
    if (c->n < 1 || c->vocab < 1 || c->width < 1 || c->n >= (1ll << 30) || c->vocab >= (1ll << 30) || c->width >= (1ll << 30)) return frnn_fail(FRNN_E_ARG, "%s: sizes have to be 1 to 2^30 - 1", what);
    if (!(c->temperature >= 1e-30f && c->temperature <= 1e30f)) return frnn_fail(FRNN_E_ARG, "%s: the temperature has to be positive", what);
    const size_t e = dtype_bytes(c->dtype);
    if (!on_boundary(c->x, e) || !on_boundary(c->weight, e) || (c->n > 1 && (c->x_stride < 0 || c->x_stride >= (1ll << 36))) || (c->vocab > 1 && (c->weight_stride < 0 || c->weight_stride >= (1ll << 36))))
        return frnn_fail(FRNN_E_ARG, "%s: bad operand", what);
    return FRNN_OK;
}

Product logits(const frnn_linear_logprobs_call* c, const Operand& x, const Operand& w, int64_t first, bool few, int* err) {
    Product q;
    q.dtype = c->dtype;
    q.m = c->n;
    q.n = w.rows;
    q.k = c->width;
    q.a = x;
    q.b[0] = w;
    q.few = few;
    q.args.err = err;
    q.args.io = c->dtype;
    q.args.c2 = (float)(1.4426950408889634 / c->temperature);
    q.args.inv_t = (float)(1.0 / c->temperature);
    q.args.tokens = c->tokens;
    q.args.token_bytes = c->token_bytes;
    q.args.ignore_index = c->ignore_index;
    q.args.first = first;
    return q;
}

int forward(const frnn_linear_logprobs_call* c, float* logprob, float* entropy, float* stats, Scratch& s, int* err, cudaStream_t stream) {
    const char* what = "linear_logprobs";
    Packs packs = {};
    const Operand x = as_operand(s, packs, c->dtype, c->x, c->n, c->width, c->x_stride), w = as_operand(s, packs, c->dtype, c->weight, c->vocab, c->width, c->weight_stride);
    // pieces of rows whose partial results, 12 bytes for each row and 64 columns, take 256 MB (of large tiles, for each 128 columns, 128 MB), but 256 rows
    const int64_t most = std::max<int64_t>(256, (1ll << 28) / (24 * ((c->vocab + 127) / 128)) / 256 * 256), pieces = (c->n + most - 1) / most;
    const int64_t piece = pieces == 1 ? c->n : ((c->n + pieces - 1) / pieces + 255) / 256 * 256;
    int rc = s.base ? pack(packs, c->dtype, stream) : (int)FRNN_OK;
    const size_t kept = s.used;
    for (int64_t r = 0; r < c->n && rc == FRNN_OK; r += piece) {
        s.used = kept;
        frnn_linear_logprobs_call some = *c;
        some.n = std::min(piece, c->n - r);
        some.tokens = (const char*)c->tokens + r * c->token_bytes;
        Product q = logits(&some, x.from_row(r, some.n), w, 0, c->n <= 128, err);
        const ProductPlan plan = plan_product<LOGPROB_STATS, false, false>(q);
        const int64_t blocks = plan.tiles_n * (plan.form == PAIR ? 256 : 128) / plan.columns();
        q.args.partial = (float*)s.take((size_t)blocks * 3 * some.n * 4);
        q.args.target = (float*)s.take((size_t)some.n * 4);
        if (!s.base) continue;
        rc = run_product<LOGPROB_STATS, false, false>(what, q, s, stream);
        if (rc != FRNN_OK) return rc;
        auto join = [&](auto kernel, int rows, int slices) {
            return launch(what, kernel, dim3((unsigned)((some.n + rows - 1) / rows)), rows * slices, 0, stream, true, 1, q.args.partial, q.args.target, blocks, some.n, some.tokens, c->token_bytes, c->vocab,
                          c->ignore_index, logprob + r, entropy + r, stats ? stats + 2 * r : nullptr, err);
        };
        rc = some.n >= 2048 ? join(join_kernel<32, 16>, 32, 16) : join(join_kernel<8, 128>, 8, 128);
    }
    return rc;
}

int backward(const frnn_linear_logprobs_call* c, const float* dlogprob, const float* dentropy, const float* stats, void* dx, void* dweight, Scratch& s, int* err, cudaStream_t stream) {
    const char* what = "linear_logprobs_backward";
    const bool count = !s.base, want_x = count || dx, want_w = count || dweight;
    Packs packs = {};
    const Operand x = as_operand(s, packs, c->dtype, c->x, c->n, c->width, c->x_stride), w = as_operand(s, packs, c->dtype, c->weight, c->vocab, c->width, c->weight_stride);
    // pieces of up to 2^28 elements of the logits' gradient (512 MB; half as many in three planes), whole tiles of 256 columns
    const int64_t most = std::max<int64_t>(256, ((c->dtype == FRNN_F32 ? 1ll << 27 : 1ll << 28) / c->n) / 256 * 256), pieces = (c->vocab + most - 1) / most;
    const int64_t piece = pieces == 1 ? c->vocab : std::min(most, ((c->vocab + pieces - 1) / pieces + 255) / 256 * 256);
    // Up to 128 rows the gradient is two 16-bit planes, what rounding leaves is the second: few rows' gradients at their own tokens are nearly
    // all of a result, and their rounding did not average out (9 rows, half of them ignored, bf16: 2.7e-3 against 64 bits, where the result's own
    // rounding is 1.6e-3).  The limit is one of cost: products of so few rows wait for the weights' copies, and the second plane takes 13 % (3 rows of
    // 107200 tokens, 6848 wide, 1306 -> 1480 us); of more rows it would take half as long again (12 operations for 8).  So rows that are ignored count,
    // and a row among 129 has one rounding more than among 128, of at most half a unit of the last place of each gradient.
    const int planes = c->dtype != FRNN_F32 && c->n <= 128 ? 2 : 1;
    const Operand grad = new_operand(s, c->dtype, c->n, piece, planes);
    float* const sum = pieces > 1 ? (float*)s.take((size_t)c->n * padded(c->width) * 4) : nullptr;
    float* const range = c->dtype == FRNN_F16 ? (float*)s.take(8) : nullptr;
    int rc = count ? (int)FRNN_OK : pack(packs, c->dtype, stream);
    if (rc != FRNN_OK) return rc;
    if (range && !count) {
        range_kernel<<<1, 1024, 0, stream>>>(dlogprob, dentropy, c->tokens, c->token_bytes, c->ignore_index, c->n, (float)(1.0 / c->temperature), range);
        rc = launched(what);
        if (rc != FRNN_OK) return rc;
    }
    const size_t kept = s.used;
    for (int64_t v = 0; v < c->vocab; v += piece) {
        s.used = kept;                             // (what slices of the piece before left has been added up)
        const int64_t cols = std::min(piece, c->vocab - v);
        const bool first = v == 0, last = v + cols == c->vocab;
        const Operand part = w.from_row(v, cols);
        Operand g = grad;
        g.cols = cols;
        {
            Product q = logits(c, x, part, v, c->n <= 128, err);
            q.args.dlogprob = dlogprob;
            q.args.dentropy = dentropy;
            q.args.stats = stats;
            q.args.scale = range;
            q.args.grad = g.writable();
            q.args.rest = planes == 2;
            rc = run_product<LOGPROB_GRAD, false, false>(what, q, s, stream);
            if (rc != FRNN_OK) return rc;
        }
        if (want_x) {
            Product q;
            q.dtype = c->dtype;
            q.m = c->n;
            q.n = c->width;
            q.k = cols;
            q.a = g;
            q.b[0] = q.b[1] = part;
            q.pairs = planes;
            q.args.b_ready = 1;
            q.args.err = err;
            q.args.alpha = range ? range + 1 : nullptr;
            q.args.add = first ? nullptr : sum;
            q.args.add_ld = padded(c->width);
            q.out = last ? dx : sum;
            q.out_dtype = last ? c->dtype : (int)FRNN_F32;
            q.out_ld = last ? c->width : padded(c->width);
            rc = run_product<STORE, false, true>(what, q, s, stream);
            if (rc != FRNN_OK) return rc;
        }
        if (want_w) {
            Product q;
            q.dtype = c->dtype;
            q.m = cols;
            q.n = c->width;
            q.k = c->n;
            q.a = g;
            q.b[0] = q.b[1] = x;
            q.pairs = planes;
            q.args.b_ready = 1;
            q.args.err = err;
            q.args.alpha = range ? range + 1 : nullptr;
            q.out = count ? nullptr : (char*)dweight + v * c->width * dtype_bytes(c->dtype);
            q.out_dtype = c->dtype;
            q.out_ld = c->width;
            rc = run_product<STORE, true, true>(what, q, s, stream);
            if (rc != FRNN_OK) return rc;
        }
    }
    return FRNN_OK;
}

}  // namespace

extern "C" {

size_t frnn_linear_logprobs_forward_workspace(const frnn_linear_logprobs_call* c) {
    if (check("linear_logprobs", c) != FRNN_OK) return 0;
    Scratch s = {nullptr};
    forward(c, nullptr, nullptr, nullptr, s, nullptr, nullptr);
    return s.most;
}

int frnn_linear_logprobs_forward(const frnn_linear_logprobs_call* c, float* logprob, float* entropy, float* stats, void* workspace, int* err, void* stream) {
    const int rc = check("linear_logprobs", c);
    if (rc != FRNN_OK) return rc;
    if (!logprob || !entropy || !workspace || !err || !on_boundary(workspace, 16) || !on_boundary(logprob, 4) || !on_boundary(entropy, 4) || !on_boundary(stats, 4))
        return frnn_fail(FRNN_E_ARG, "linear_logprobs: bad argument");
    Scratch s = {(char*)workspace};
    return forward(c, logprob, entropy, stats, s, err, (cudaStream_t)stream);
}

size_t frnn_linear_logprobs_backward_workspace(const frnn_linear_logprobs_call* c) {
    if (check("linear_logprobs_backward", c) != FRNN_OK) return 0;
    Scratch s = {nullptr};
    backward(c, nullptr, nullptr, nullptr, nullptr, nullptr, s, nullptr, nullptr);
    return s.most;
}

int frnn_linear_logprobs_backward(const frnn_linear_logprobs_call* c, const float* dlogprob, const float* dentropy, const float* stats, void* dx, void* dweight, void* workspace, int* err, void* stream) {
    const int rc = check("linear_logprobs_backward", c);
    if (rc != FRNN_OK) return rc;
    const size_t e = dtype_bytes(c->dtype);
    if (!stats || !workspace || !err || !on_boundary(workspace, 16) || !on_boundary(stats, 4) || !on_boundary(dlogprob, 4) || !on_boundary(dentropy, 4) || !on_boundary(dx, e) || !on_boundary(dweight, e))
        return frnn_fail(FRNN_E_ARG, "linear_logprobs_backward: bad argument");
    if (!dx && !dweight) return FRNN_OK;
    Scratch s = {(char*)workspace};
    return backward(c, dlogprob, dentropy, stats, dx, dweight, s, err, (cudaStream_t)stream);
}

}  // extern "C"
