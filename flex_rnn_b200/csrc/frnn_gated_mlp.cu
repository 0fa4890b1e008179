// The gated feed-forward block and its backward pass as products on the tensor cores (frnn_product.cuh):
//
//   a = x Wg^T, b = x Wu^T          one product, a tile holds columns of both; its epilogue makes h = act(a) b
//   y = h Wd^T
//   dh = dy Wd                      its epilogue makes da = dh (b act'(a)), db = dh act(a)
//   dWd = dy^T h, dWg = da^T x, dWu = db^T x, dx = da Wg + db Wu (one product of twice the length)
//
// n D F (D = width = out_width): 6 operations a value forward, 12 backward.
//
// Of 16-bit operands h, da and db are rounded to 16 bits, once each, because the tensor cores read them so.  That is one rounding beside the result's
// own: errors against 64 bits are 2.35e-3 in bf16 and 2.9e-4 in fp16, where the result's rounding alone makes 1.66e-3 and 2.1e-4.  (h, da and db as
// sums of two 16-bit numbers would take 30 operations for 18 in training.)  In fp16 what passes 65504 there is infinite, as a result is.
// The forward keeps h, as it is multiplied, and its two derivatives b act'(a) and act(a) in 32 bits: 10 bytes a hidden value (fp32: 14), 1 GB for 8192
// rows of 12288.  (Gradients in bf16: 2.35e-3 so, 2.9e-3 with derivatives in 16 bits, 3.5e-3 with a and b kept in 16 bits instead, which the
// backward's epilogue took through the activation again.)
#include "frnn_product.cuh"

using namespace frnn_lm;

namespace {

int check(const char* what, const frnn_gated_mlp_call* c) {
    if (!c || !dtype_known(c->dtype)) return frnn_fail(FRNN_E_ARG, "%s: bad argument", what);
    if (c->activation < FRNN_SILU || c->activation > FRNN_SIGMOID) return frnn_fail(FRNN_E_ARG, "%s: unknown activation %d", what, (int)c->activation);
    const int64_t most = (1ll << 31) - 1024;
    if (c->n < 1 || c->width < 1 || c->hidden < 1 || c->out_width < 1 || c->n > most || c->width > most || c->hidden > most || c->out_width > most)
        return frnn_fail(FRNN_E_ARG, "%s: sizes have to be 1 to 2^31 - 1024", what);
    const size_t e = dtype_bytes(c->dtype);
    const void* const p[4] = {c->x, c->gate, c->up, c->down};
    const int64_t rows[4] = {c->n, c->hidden, c->hidden, c->out_width}, strides[4] = {c->x_stride, c->gate_stride, c->up_stride, c->down_stride};
    for (int i = 0; i < 4; i++)
        if (!p[i] || !on_boundary(p[i], e) || (rows[i] > 1 && (strides[i] < 0 || strides[i] >= (1ll << 36)))) return frnn_fail(FRNN_E_ARG, "%s: bad operand", what);
    return FRNN_OK;
}

Product product(const frnn_gated_mlp_call* c, int64_t m, int64_t n, int64_t k) {
    Product q;
    q.dtype = c->dtype;
    q.m = m;
    q.n = n;
    q.k = k;
    q.args.io = c->dtype;
    q.args.activation = c->activation;
    return q;
}

// The hidden vectors as the forward keeps them.
Operand kept(const frnn_gated_mlp_call* c, const void* hidden) {
    Scratch none = {nullptr};
    Operand h = new_operand(none, c->dtype, c->n, c->hidden);
    h.p = hidden;
    return h;
}

int forward(const frnn_gated_mlp_call* c, void* y, float* by_gate, float* by_up, void* hidden, Scratch& s, int* err, cudaStream_t stream) {
    const char* what = "gated_mlp";
    Packs packs = {};
    const Operand x = as_operand(s, packs, c->dtype, c->x, c->n, c->width, c->x_stride), gate = as_operand(s, packs, c->dtype, c->gate, c->hidden, c->width, c->gate_stride);
    const Operand up = as_operand(s, packs, c->dtype, c->up, c->hidden, c->width, c->up_stride), down = as_operand(s, packs, c->dtype, c->down, c->out_width, c->hidden, c->down_stride);
    const Operand h = hidden ? kept(c, hidden) : new_operand(s, c->dtype, c->n, c->hidden);
    int rc = s.base ? pack(packs, c->dtype, stream) : (int)FRNN_OK;
    if (rc != FRNN_OK) return rc;
    {
        Product q = product(c, c->n, c->hidden, c->width);
        q.a = x;
        q.b[0] = gate;
        q.b[1] = up;
        q.args.dual = 1;
        q.args.err = err;
        q.args.by_gate = by_gate;
        q.args.by_up = by_up;
        q.args.by_ld = padded(c->hidden);
        q.args.h = h.writable();
        rc = run_product<GLU_FORWARD, false, false>(what, q, s, stream);
        if (rc != FRNN_OK) return rc;
    }
    Product q = product(c, c->n, c->out_width, c->hidden);
    q.a = h;
    q.b[0] = down;
    q.args.b_ready = 1;
    q.args.err = err;
    q.out = y;
    q.out_dtype = c->dtype;
    q.out_ld = c->out_width;
    return run_product<STORE, false, false>(what, q, s, stream);
}

int backward(const frnn_gated_mlp_call* c, const void* dy, int64_t dy_stride, const float* by_gate, const float* by_up, const void* hidden, void* dx, void* dgate, void* dup, void* ddown, Scratch& s, int* err, cudaStream_t stream) {
    const char* what = "gated_mlp_backward";
    const bool count = !s.base, want_x = count || dx, want_gate = count || dgate, want_up = count || dup, want_down = count || ddown, want_hidden = want_x || want_gate || want_up;
    Packs packs = {};
    Operand x, gate, up, down;
    const Operand g = as_operand(s, packs, c->dtype, dy, c->n, c->out_width, dy_stride);
    if (want_gate || want_up) x = as_operand(s, packs, c->dtype, c->x, c->n, c->width, c->x_stride);
    if (want_x) gate = as_operand(s, packs, c->dtype, c->gate, c->hidden, c->width, c->gate_stride);
    if (want_x) up = as_operand(s, packs, c->dtype, c->up, c->hidden, c->width, c->up_stride);
    if (want_hidden) down = as_operand(s, packs, c->dtype, c->down, c->out_width, c->hidden, c->down_stride);
    const int planes = planes_of(c->dtype);
    const Operand both = new_operand(s, c->dtype, c->n, c->hidden, 2);      // da, db
    Operand da = both, db = both;
    da.planes = db.planes = planes;
    db.p = (const char*)both.p + both.plane * planes * 2;
    int rc = count ? (int)FRNN_OK : pack(packs, c->dtype, stream);
    if (rc != FRNN_OK) return rc;
    auto store = [&](Product& q, void* out, int64_t ld) {
        q.args.b_ready = 1;                // (the hidden gradients, which the first product writes, are always A)
        q.args.err = err;
        q.out = out;
        q.out_dtype = c->dtype;
        q.out_ld = ld;
    };
    if (want_hidden) {
        Product q = product(c, c->n, c->hidden, c->out_width);
        q.a = g;
        q.b[0] = down;
        q.args.err = err;
        q.args.by_gate = const_cast<float*>(by_gate);
        q.args.by_up = const_cast<float*>(by_up);
        q.args.by_ld = padded(c->hidden);
        if (want_x || want_gate) q.args.da = da.writable();
        if (want_x || want_up) q.args.db = db.writable();
        rc = run_product<GLU_BACKWARD, false, true>(what, q, s, stream);
        if (rc != FRNN_OK) return rc;
    }
    if (want_down) {
        Product q = product(c, c->out_width, c->hidden, c->n);
        q.a = g;
        q.b[0] = kept(c, hidden);
        store(q, ddown, c->hidden);
        q.args.b_ready = want_hidden;      // (else it is the first: what is before it is not known)
        rc = run_product<STORE, true, true>(what, q, s, stream);
        if (rc != FRNN_OK) return rc;
    }
    // both in one, because half of a small product would leave multiprocessors idle (counted is what one of them alone asks for: more)
    if (want_gate || want_up) {
        const bool two = want_gate && want_up && !count;
        Product q = product(c, c->hidden, c->width, c->n);
        q.a = want_gate ? both : db;
        q.b[0] = x;
        q.args.stacked = two ? planes : 0;
        q.args.out2 = two ? dup : nullptr;
        store(q, want_gate ? dgate : dup, c->width);
        rc = run_product<STORE, true, true>(what, q, s, stream);
        if (rc != FRNN_OK) return rc;
    }
    if (want_x) {
        Product q = product(c, c->n, c->width, c->hidden);
        q.a = both;
        q.b[0] = gate;
        q.b[1] = up;
        q.pairs = 2;
        store(q, dx, c->width);
        rc = run_product<STORE, false, true>(what, q, s, stream);
    }
    return rc;
}

}  // namespace

extern "C" {

size_t frnn_gated_mlp_forward_workspace(const frnn_gated_mlp_call* c) {
    if (check("gated_mlp", c) != FRNN_OK) return 0;
    Scratch s = {nullptr};
    forward(c, nullptr, nullptr, nullptr, nullptr, s, nullptr, nullptr);
    return s.most;
}

int frnn_gated_mlp_forward(const frnn_gated_mlp_call* c, void* y, float* by_gate, float* by_up, void* hidden, void* workspace, int* err, void* stream) {
    const int rc = check("gated_mlp", c);
    if (rc != FRNN_OK) return rc;
    if (!y || !err || !workspace || !on_boundary(workspace, 16) || !on_boundary(y, dtype_bytes(c->dtype)) || !by_gate != !by_up || !by_gate != !hidden || !on_boundary(by_gate, 16) || !on_boundary(by_up, 16) ||
        !on_boundary(hidden, 16))
        return frnn_fail(FRNN_E_ARG, "gated_mlp: bad argument");
    Scratch s = {(char*)workspace};
    return forward(c, y, by_gate, by_up, hidden, s, err, (cudaStream_t)stream);
}

size_t frnn_gated_mlp_backward_workspace(const frnn_gated_mlp_call* c, const void* dy, int64_t dy_stride) {
    if (check("gated_mlp_backward", c) != FRNN_OK) return 0;
    Scratch s = {nullptr};
    backward(c, dy, dy_stride, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, s, nullptr, nullptr);
    return s.most;
}

int frnn_gated_mlp_backward(const frnn_gated_mlp_call* c, const void* dy, int64_t dy_stride, const float* by_gate, const float* by_up, const void* hidden, void* dx, void* dgate, void* dup,
                            void* ddown, void* workspace, int* err, void* stream) {
    const int rc = check("gated_mlp_backward", c);
    if (rc != FRNN_OK) return rc;
    const size_t e = dtype_bytes(c->dtype);
    if (!dy || !on_boundary(dy, e) || (c->n > 1 && (dy_stride < 0 || dy_stride >= (1ll << 36))) || !by_gate || !by_up || !hidden || !on_boundary(by_gate, 16) ||
        !on_boundary(by_up, 16) || !on_boundary(hidden, 16) || !err || !workspace ||
        !on_boundary(workspace, 16) || !on_boundary(dx, e) || !on_boundary(dgate, e) || !on_boundary(dup, e) || !on_boundary(ddown, e))
        return frnn_fail(FRNN_E_ARG, "gated_mlp_backward: bad argument");
    if (!dx && !dgate && !dup && !ddown) return FRNN_OK;
    Scratch s = {(char*)workspace};
    return backward(c, dy, dy_stride, by_gate, by_up, hidden, dx, dgate, dup, ddown, s, err, (cudaStream_t)stream);
}

}  // extern "C"
