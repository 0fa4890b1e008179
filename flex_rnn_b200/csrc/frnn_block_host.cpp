// The matrix products and rotations around the scans as PyTorch operators (flex_rnn_b200::gated_mlp, linear_logprobs, rotary and
// their backward), in the manner of frnn_lm_host.cpp.
#include "frnn_lm_host.h"

using namespace frnn_ops;

namespace {

decltype(&frnn_gated_mlp_forward) g_gated_mlp_forward = nullptr;
decltype(&frnn_gated_mlp_forward_workspace) g_gated_mlp_forward_workspace = nullptr;
decltype(&frnn_gated_mlp_backward) g_gated_mlp_backward = nullptr;
decltype(&frnn_gated_mlp_backward_workspace) g_gated_mlp_backward_workspace = nullptr;
decltype(&frnn_linear_logprobs_forward) g_linear_logprobs_forward = nullptr;
decltype(&frnn_linear_logprobs_forward_workspace) g_linear_logprobs_forward_workspace = nullptr;
decltype(&frnn_linear_logprobs_backward) g_linear_logprobs_backward = nullptr;
decltype(&frnn_linear_logprobs_backward_workspace) g_linear_logprobs_backward_workspace = nullptr;
decltype(&frnn_rotary) g_rotary = nullptr;

// A weight [rows, columns] with consecutive columns, else a contiguous copy.
Tensor as_weight(const Tensor& t) { return t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous(); }

void check_weight(const char* op, const char* what, const Tensor& t, const Tensor& x) {
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), "flex_rnn_b200: ", op, ": ", what, " has to have the type of x, got ", t.scalar_type(), " for x in ", x.scalar_type());
    TORCH_CHECK(t.dim() == 2 && t.size(0) >= 1 && t.size(1) >= 1, "flex_rnn_b200: ", op, ": ", what, " has to be a matrix that is not empty, got ", t.sizes());
    check_one(op, what, t, x);
}

Tensor nothing(const Tensor& like) { return make("nothing", {0}, like.scalar_type(), like); }

// ---- gated feed-forward block ---------------------------------------------------------------------------------------------

struct GatedMlp {
    frnn_gated_mlp_call c;
    Tensor x, gate, up, down;
};

GatedMlp gated_mlp_call(const char* op, const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int64_t activation) {
    GatedMlp m;
    m.c.dtype = dtype_of(op, "x", x);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "flex_rnn_b200: ", op, ": x has to be [..., width] with a width that is not 0, got ", x.sizes());
    check_one(op, "x", x, x);
    check_weight(op, "gate", gate, x);
    check_weight(op, "up", up, x);
    check_weight(op, "down", down, x);
    TORCH_CHECK(gate.size(1) == x.size(-1) && up.sizes() == gate.sizes() && down.size(1) == gate.size(0), "flex_rnn_b200: ", op,
                ": gate and up have to be [hidden, width] and down [out, hidden], got ", gate.sizes(), ", ", up.sizes(), " and ", down.sizes(), " for x ", x.sizes());
    TORCH_CHECK(activation >= FRNN_SILU && activation <= FRNN_SIGMOID, "flex_rnn_b200: ", op, ": unknown activation ", activation);
    m.c.activation = (int32_t)activation;
    m.c.n = x.numel() / x.size(-1);
    m.c.width = x.size(-1);
    m.c.hidden = gate.size(0);
    m.c.out_width = down.size(0);
    if (m.c.n) m.x = as_rows(x);
    m.gate = as_weight(gate);
    m.up = as_weight(up);
    m.down = as_weight(down);
    m.c.x = ptr(m.x);
    m.c.gate = m.gate.data_ptr();
    m.c.up = m.up.data_ptr();
    m.c.down = m.down.data_ptr();
    m.c.x_stride = m.c.n ? m.x.stride(0) : 0;
    m.c.gate_stride = m.gate.stride(0);
    m.c.up_stride = m.up.stride(0);
    m.c.down_stride = m.down.stride(0);
    return m;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_mlp_cuda(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int64_t activation, bool save) {
    c10::cuda::OptionalCUDAGuard guard;
    if (x.is_cuda()) guard.set_device(x.device());
    const GatedMlp m = gated_mlp_call("gated_mlp", x, gate, up, down, activation);
    int* err = error_word(x.device().index());
    auto sizes = x.sizes().vec();
    sizes.back() = m.c.out_width;
    const int64_t n = save ? m.c.n : 0, ld = (m.c.hidden + 63) / 64 * 64;
    const bool wide = x.scalar_type() == at::kFloat;
    Tensor y = make("the output", sizes, x.scalar_type(), x), by_gate = make("the derivatives by gate", {n, ld}, at::kFloat, x), by_up = make("the derivatives by up", {n, ld}, at::kFloat, x);
    Tensor hidden = make("the hidden vectors", {wide ? 3 : 1, n, ld}, wide ? at::kBFloat16 : x.scalar_type(), x);
    if (m.c.n) {
        const Tensor work = workspace(g_gated_mlp_forward_workspace(&m.c), x);
        ran(g_gated_mlp_forward(&m.c, y.data_ptr(), n ? by_gate.data_ptr<float>() : nullptr, n ? by_up.data_ptr<float>() : nullptr, n ? hidden.data_ptr() : nullptr, ptr(work), err, stream_of(x)), x);
    }
    return {y, by_gate, by_up, hidden};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_mlp_backward_cuda(const Tensor& grad, const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, const Tensor& by_gate, const Tensor& by_up, const Tensor& hidden,
                                                                   int64_t activation, bool want_x, bool want_gate, bool want_up, bool want_down) {
    const char* op = "gated_mlp_backward";
    c10::cuda::OptionalCUDAGuard guard;
    if (x.is_cuda()) guard.set_device(x.device());
    const GatedMlp m = gated_mlp_call(op, x, gate, up, down, activation);
    TORCH_CHECK(grad.scalar_type() == x.scalar_type() && grad.dim() == x.dim() && grad.size(-1) == m.c.out_width && grad.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1), "flex_rnn_b200: ", op,
                ": the gradient has to have the shape and type of the output, got ", grad.sizes());
    check_one(op, "the gradient", grad, x);
    const int64_t ld = (m.c.hidden + 63) / 64 * 64;
    const bool wide = x.scalar_type() == at::kFloat;
    for (const Tensor* t : {&by_gate, &by_up, &hidden}) {
        const bool h = t == &hidden;
        TORCH_CHECK(t->dim() == (h ? 3 : 2) && t->size(-2) == m.c.n && t->size(-1) == ld && (!h || t->size(0) == (wide ? 3 : 1)) && t->scalar_type() == (!h ? at::kFloat : wide ? at::kBFloat16 : x.scalar_type()),
                    "flex_rnn_b200: ", op, ": what the forward kept has to be given as it was");
        check_one(op, "what the forward kept", *t, x);
    }
    int* err = error_word(x.device().index());
    auto result = [&](bool want, const char* what, const Tensor& like) { return want ? make(what, like.sizes(), like.scalar_type(), like) : Tensor(); };
    Tensor dx = result(want_x, "x's gradient", x), dgate = result(want_gate, "gate's gradient", gate), dup = result(want_up, "up's gradient", up), ddown = result(want_down, "down's gradient", down);
    if (m.c.n) {
        const Tensor g = as_rows(grad), sa = saved(by_gate), sb = saved(by_up), sh = saved(hidden);
        const Tensor work = workspace(g_gated_mlp_backward_workspace(&m.c, g.data_ptr(), g.stride(0)), x);
        ran(g_gated_mlp_backward(&m.c, g.data_ptr(), g.stride(0), sa.data_ptr<float>(), sb.data_ptr<float>(), sh.data_ptr(), ptr(dx), ptr(dgate), ptr(dup), ptr(ddown), ptr(work), err, stream_of(x)), x);
    } else {
        for (Tensor* t : {&dgate, &dup, &ddown})
            if (t->defined()) t->zero_();
    }
    auto some = [&](const Tensor& t) { return t.defined() ? t : nothing(x); };
    return {some(dx), some(dgate), some(dup), some(ddown)};
}

// ---- log probabilities without logits ---------------------------------------------------------------------------------------

struct LinearLogprobs {
    frnn_linear_logprobs_call c;
    Tensor x, weight, tokens;
};

LinearLogprobs linear_logprobs_call(const char* op, const Tensor& x, const Tensor& weight, const Tensor& tokens, double temperature, int64_t ignore_index) {
    LinearLogprobs l;
    l.c.dtype = dtype_of(op, "x", x);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "flex_rnn_b200: ", op, ": x has to be [..., width] with a width that is not 0, got ", x.sizes());
    check_one(op, "x", x, x);
    check_weight(op, "weight", weight, x);
    TORCH_CHECK(weight.size(1) == x.size(-1), "flex_rnn_b200: ", op, ": weight has to be [vocabulary, width], got ", weight.sizes(), " for x ", x.sizes());
    TORCH_CHECK(x.sizes().slice(0, x.dim() - 1) == tokens.sizes(), "flex_rnn_b200: ", op, ": tokens have to have the shape of x without its last dimension, got ", tokens.sizes(), " for x ", x.sizes());
    TORCH_CHECK(temperature >= 1e-30 && temperature <= 1e30, "flex_rnn_b200: ", op, ": the temperature has to be positive, from 1e-30 to 1e30, got ", temperature);
    l.tokens = check_tokens(op, tokens, x);
    l.c.token_bytes = (int32_t)l.tokens.element_size();
    l.c.tokens = l.tokens.data_ptr();
    l.c.n = tokens.numel();
    l.c.vocab = weight.size(0);
    l.c.width = x.size(-1);
    if (l.c.n) l.x = as_rows(x);
    l.weight = as_weight(weight);
    l.c.x = ptr(l.x);
    l.c.weight = l.weight.data_ptr();
    l.c.x_stride = l.c.n ? l.x.stride(0) : 0;
    l.c.weight_stride = l.weight.stride(0);
    l.c.ignore_index = ignore_index;
    l.c.temperature = (float)temperature;
    return l;
}

std::tuple<Tensor, Tensor, Tensor> linear_logprobs_cuda(const Tensor& x, const Tensor& weight, const Tensor& tokens, double temperature, int64_t ignore_index, bool save) {
    c10::cuda::OptionalCUDAGuard guard;
    if (x.is_cuda()) guard.set_device(x.device());
    const LinearLogprobs l = linear_logprobs_call("linear_logprobs", x, weight, tokens, temperature, ignore_index);
    int* err = error_word(x.device().index());
    Tensor lp = make("the log probabilities", tokens.sizes(), at::kFloat, x), ent = make("the entropies", tokens.sizes(), at::kFloat, x), stats = make("the statistics", {save ? l.c.n : 0, 2}, at::kFloat, x);
    if (l.c.n) {
        const Tensor work = workspace(g_linear_logprobs_forward_workspace(&l.c), x);
        ran(g_linear_logprobs_forward(&l.c, lp.data_ptr<float>(), ent.data_ptr<float>(), save ? stats.data_ptr<float>() : nullptr, ptr(work), err, stream_of(x)), x);
    }
    return {lp, ent, stats};
}

std::tuple<Tensor, Tensor> linear_logprobs_backward_cuda(const optional<Tensor>& dlogprob, const optional<Tensor>& dentropy, const Tensor& x, const Tensor& weight, const Tensor& tokens, const Tensor& stats,
                                                         double temperature, int64_t ignore_index, bool want_x, bool want_weight) {
    const char* op = "linear_logprobs_backward";
    c10::cuda::OptionalCUDAGuard guard;
    if (x.is_cuda()) guard.set_device(x.device());
    const LinearLogprobs l = linear_logprobs_call(op, x, weight, tokens, temperature, ignore_index);
    check_one(op, "the statistics", stats, x);
    TORCH_CHECK(stats.dim() == 2 && stats.size(0) == l.c.n && stats.size(1) == 2 && stats.scalar_type() == at::kFloat, "flex_rnn_b200: ", op, ": the statistics have to be those of the forward");
    auto upstream = [&](const optional<Tensor>& g) {
        if (!g.has_value() || !g->defined()) return Tensor();
        TORCH_CHECK(g->sizes() == tokens.sizes(), "flex_rnn_b200: ", op, ": upstream gradients have to have the shape of tokens");
        check_one(op, "an upstream gradient", *g, x);
        return g->to(at::kFloat).contiguous();
    };
    int* err = error_word(x.device().index());
    const Tensor glp = upstream(dlogprob), gent = upstream(dentropy), st = saved(stats);
    Tensor dx = want_x ? make("x's gradient", x.sizes(), x.scalar_type(), x) : Tensor(), dw = want_weight ? make("weight's gradient", weight.sizes(), x.scalar_type(), x) : Tensor();
    if (l.c.n) {
        const Tensor work = workspace(g_linear_logprobs_backward_workspace(&l.c), x);
        ran(g_linear_logprobs_backward(&l.c, ptr<float>(glp), ptr<float>(gent), st.data_ptr<float>(), ptr(dx), ptr(dw), ptr(work), err, stream_of(x)), x);
    } else if (dw.defined()) {
        dw.zero_();
    }
    return {dx.defined() ? dx : nothing(x), dw.defined() ? dw : nothing(x)};
}

// ---- rotary positions ---------------------------------------------------------------------------------------------------------

// Dimensions between the places and the last one as one dimension of heads, where their strides allow.
bool heads_of(const Tensor& x, int64_t& heads, int64_t& stride) {
    heads = 1;
    stride = 0;
    for (int64_t d = 2; d < x.dim() - 1; d++) {
        if (x.size(d) == 1) continue;
        if (heads != 1 && stride != x.size(d) * x.stride(d)) return false;
        heads *= x.size(d);
        stride = x.stride(d);
    }
    return true;
}

Tensor rotary_cuda(const Tensor& x, const optional<Tensor>& positions, c10::SymInt start, const Tensor& frequencies, bool interleaved, double scale, bool inverse) {
    const char* op = "rotary";
    frnn_rotary_call c = {};
    c.dtype = dtype_of(op, "x", x);
    TORCH_CHECK(x.dim() >= 3, "flex_rnn_b200: rotary: x has to be [batch, length, ..., width], got ", x.sizes());
    check_one(op, "x", x, x);
    TORCH_CHECK(frequencies.dim() == 1 && (frequencies.scalar_type() == at::kFloat || frequencies.scalar_type() == at::kDouble), "flex_rnn_b200: rotary: frequencies have to be a vector in float32 or float64, got ",
                frequencies.sizes(), " in ", frequencies.scalar_type());
    TORCH_CHECK(2 * frequencies.size(0) <= x.size(-1), "flex_rnn_b200: rotary: ", frequencies.size(0), " frequencies turn ", 2 * frequencies.size(0), " values, but a head has ", x.size(-1));
    check_one(op, "frequencies", frequencies, x);
    Tensor where;
    if (positions.has_value() && positions->defined()) {
        const Tensor& p = *positions;
        TORCH_CHECK(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt, "flex_rnn_b200: rotary: positions have to be int64 or int32, got ", p.scalar_type());
        TORCH_CHECK((p.dim() == 1 || (p.dim() == 2 && (p.size(0) == x.size(0) || p.size(0) == 1))) && p.size(-1) == x.size(1), "flex_rnn_b200: rotary: positions have to be [length] or [batch, length], got ", p.sizes(),
                    " for x ", x.sizes());
        check_one(op, "positions", p, x);
        where = p;
        c.position_bytes = (int32_t)p.element_size();
        c.position_stride[0] = p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0;
        c.position_stride[1] = p.size(-1) > 1 ? p.stride(-1) : 0;
    }
    c10::cuda::CUDAGuard guard(x.device());
    error_word(x.device().index());
    Tensor from = x;
    if ((x.size(-1) > 1 && x.stride(-1) != 1) || !heads_of(x, c.heads, c.x_stride[2])) {
        from = x.contiguous();
        heads_of(from, c.heads, c.x_stride[2]);
    }
    const Tensor f = frequencies.contiguous();
    Tensor y = make("the output", x.sizes(), x.scalar_type(), x);
    c.interleaved = interleaved;
    c.inverse = inverse;
    c.frequency_bytes = (int32_t)f.element_size();
    c.scale = (float)scale;
    c.batch = x.size(0);
    c.length = x.size(1);
    c.width = x.size(-1);
    c.pairs = f.size(0);
    c.start = start.expect_int();
    for (int d = 0; d < 2; d++) c.x_stride[d] = x.size(d) > 1 ? from.stride(d) : 0;
    c.y_stride[2] = c.heads > 1 ? c.width : 0;
    c.y_stride[1] = c.length > 1 ? c.heads * c.width : 0;
    c.y_stride[0] = c.batch > 1 ? c.length * c.heads * c.width : 0;
    if (x.numel()) ran(g_rotary(&c, from.data_ptr(), ptr(where), f.data_ptr(), y.data_ptr(), stream_of(x)), x);
    return y;
}

// ---- autograd -------------------------------------------------------------------------------------------------------------------

FRNN_OP(gated_mlp, gated_mlp_cuda)
FRNN_OP(gated_mlp_backward, gated_mlp_backward_cuda)
FRNN_OP(linear_logprobs, linear_logprobs_cuda)
FRNN_OP(linear_logprobs_backward, linear_logprobs_backward_cuda)
FRNN_OP(rotary, rotary_cuda)

struct GatedMlpBackward : Saving {
    using Saving::Saving;
    int64_t activation;
    std::string name() const override { return "GatedMlpBackward"; }
    variable_list apply(variable_list&& up) override {
        bool want[4];
        for (int i = 0; i < 4; i++) want[i] = task_should_compute_output(i);
        if (!up[0].defined() || !(want[0] || want[1] || want[2] || want[3])) return variable_list(4);
        const variable_list k = unpack();
        auto [dx, dgate, dup, ddown] = gated_mlp_backward().call(up[0], k[0], k[1], k[2], k[3], k[4], k[5], k[6], activation, want[0], want[1], want[2], want[3]);
        return {want[0] ? dx : Tensor(), want[1] ? dgate : Tensor(), want[2] ? dup : Tensor(), want[3] ? ddown : Tensor()};
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_mlp_autograd(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int64_t activation, bool save) {
    for (const Tensor* t : {&x, &gate, &up, &down}) no_tangent(*t);
    const bool grad = at::GradMode::is_enabled() && (needs(x) || needs(gate) || needs(up) || needs(down));
    std::tuple<Tensor, Tensor, Tensor, Tensor> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = gated_mlp().call(x, gate, up, down, activation, save || grad);
    }
    if (grad) {
        auto node = make_node<GatedMlpBackward>(x, gate, up, down);
        node->activation = activation;
        for (const Tensor& t : {x, gate, up, down, std::get<1>(r), std::get<2>(r), std::get<3>(r)}) node->save(t);
        torch::autograd::create_gradient_edge(std::get<0>(r), node);
    }
    return r;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_mlp_backward_autograd(const Tensor& grad, const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, const Tensor& by_gate, const Tensor& by_up, const Tensor& hidden,
                                                                       int64_t activation, bool want_x, bool want_gate, bool want_up, bool want_down) {
    for (const Tensor* t : {&grad, &x, &gate, &up, &down}) no_tangent(*t);
    std::tuple<Tensor, Tensor, Tensor, Tensor> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = gated_mlp_backward().call(grad, x, gate, up, down, by_gate, by_up, hidden, activation, want_x, want_gate, want_up, want_down);
    }
    only_once({&std::get<0>(r), &std::get<1>(r), &std::get<2>(r), &std::get<3>(r)}, grad, x, gate, up, down);
    return r;
}

struct LinearLogprobsBackward : Saving {
    using Saving::Saving;
    double temperature;
    int64_t ignore_index;
    std::string name() const override { return "LinearLogprobsBackward"; }
    variable_list apply(variable_list&& up) override {
        const bool wx = task_should_compute_output(0), ww = task_should_compute_output(1);
        if ((!up[0].defined() && !up[1].defined()) || !(wx || ww)) return variable_list(2);
        const variable_list k = unpack();
        auto [dx, dw] = linear_logprobs_backward().call(maybe(up[0]), maybe(up[1]), k[0], k[1], k[2], k[3], temperature, ignore_index, wx, ww);
        return {wx ? dx : Tensor(), ww ? dw : Tensor()};
    }
};

std::tuple<Tensor, Tensor, Tensor> linear_logprobs_autograd(const Tensor& x, const Tensor& weight, const Tensor& tokens, double temperature, int64_t ignore_index, bool save) {
    no_tangent(x);
    no_tangent(weight);
    const bool grad = at::GradMode::is_enabled() && (needs(x) || needs(weight));
    std::tuple<Tensor, Tensor, Tensor> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = linear_logprobs().call(x, weight, tokens, temperature, ignore_index, save || grad);
    }
    if (grad) {
        auto node = make_node<LinearLogprobsBackward>(x, weight);
        node->temperature = temperature;
        node->ignore_index = ignore_index;
        for (const Tensor& t : {x, weight, tokens, std::get<2>(r)}) node->save(t);
        torch::autograd::create_gradient_edge(std::get<0>(r), node);
        torch::autograd::create_gradient_edge(std::get<1>(r), node);
    }
    return r;
}

std::tuple<Tensor, Tensor> linear_logprobs_backward_autograd(const optional<Tensor>& dlogprob, const optional<Tensor>& dentropy, const Tensor& x, const Tensor& weight, const Tensor& tokens,
                                                             const Tensor& stats, double temperature, int64_t ignore_index, bool want_x, bool want_weight) {
    no_tangent(dlogprob);
    no_tangent(dentropy);
    no_tangent(x);
    no_tangent(weight);
    std::tuple<Tensor, Tensor> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = linear_logprobs_backward().call(dlogprob, dentropy, x, weight, tokens, stats, temperature, ignore_index, want_x, want_weight);
    }
    only_once({&std::get<0>(r), &std::get<1>(r)}, dlogprob, dentropy, x, weight);
    return r;
}

// A rotation is linear and its gradient the rotation back: the same operator, differentiable in its turn.  (A compiled program
// may have `start` as a symbol: generation goes on from another position each call.)
struct RotaryBackward : Saving {
    using Saving::Saving;
    c10::SymInt start;
    bool interleaved, inverse, positions;
    double scale;
    std::string name() const override { return "RotaryBackward"; }
    variable_list apply(variable_list&& up) override {
        if (!up[0].defined() || !task_should_compute_output(0)) return {Tensor()};
        const variable_list k = unpack();
        return {rotary().call(up[0], positions ? maybe(k[1]) : optional<Tensor>(), start, k[0], interleaved, scale, !inverse)};
    }
};

Tensor rotary_autograd(const Tensor& x, const optional<Tensor>& positions, c10::SymInt start, const Tensor& frequencies, bool interleaved, double scale, bool inverse) {
    no_tangent(x);
    no_tangent(frequencies);
    TORCH_CHECK(!at::GradMode::is_enabled() || !needs(frequencies), "flex_rnn_b200: rotary: the frequencies carry no gradient");
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = rotary().call(x, positions, start, frequencies, interleaved, scale, inverse);
    }
    if (at::GradMode::is_enabled() && needs(x)) {
        auto node = make_node<RotaryBackward>(x);
        node->start = start;
        node->interleaved = interleaved;
        node->inverse = inverse;
        node->scale = scale;
        node->positions = positions.has_value() && positions->defined();
        node->save(frequencies);
        if (node->positions) node->save(*positions);
        torch::autograd::create_gradient_edge(y, node);
    }
    return y;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(flex_rnn_b200, m) {
    m.def("gated_mlp(Tensor x, Tensor gate, Tensor up, Tensor down, int activation, bool save) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("gated_mlp_backward(Tensor grad, Tensor x, Tensor gate, Tensor up, Tensor down, Tensor by_gate, Tensor by_up, Tensor hidden, int activation, bool want_x, bool want_gate, bool want_up, bool want_down) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("linear_logprobs(Tensor x, Tensor weight, Tensor tokens, float temperature, int ignore_index, bool save) -> (Tensor, Tensor, Tensor)");
    m.def("linear_logprobs_backward(Tensor? dlogprob, Tensor? dentropy, Tensor x, Tensor weight, Tensor tokens, Tensor stats, float temperature, int ignore_index, bool want_x, bool want_weight) -> (Tensor, Tensor)");
    m.def("rotary(Tensor x, Tensor? positions, SymInt start, Tensor frequencies, bool interleaved, float scale, bool inverse) -> Tensor");
}

#define FRNN_ALL(how) \
    m.impl("gated_mlp", how(gated_mlp)); \
    m.impl("gated_mlp_backward", how(gated_mlp_backward)); \
    m.impl("linear_logprobs", how(linear_logprobs)); \
    m.impl("linear_logprobs_backward", how(linear_logprobs_backward)); \
    m.impl("rotary", how(rotary));

TORCH_LIBRARY_IMPL(flex_rnn_b200, CUDA, m) { FRNN_ALL(FRNN_ON_CUDA) }
TORCH_LIBRARY_IMPL(flex_rnn_b200, Autograd, m) { FRNN_ALL(FRNN_ON_AUTOGRAD) }
TORCH_LIBRARY_IMPL(flex_rnn_b200, CPU, m) { FRNN_ALL(FRNN_REFUSED) }

void frnn_bind_block(py::module& m) {
    m.def("bind_block", [](const std::map<std::string, uintptr_t>& at_) {
        auto take = [&](auto& fn, const char* name) { fn = (std::decay_t<decltype(fn)>)at_.at(name); };
        take(g_gated_mlp_forward, "frnn_gated_mlp_forward");
        take(g_gated_mlp_forward_workspace, "frnn_gated_mlp_forward_workspace");
        take(g_gated_mlp_backward, "frnn_gated_mlp_backward");
        take(g_gated_mlp_backward_workspace, "frnn_gated_mlp_backward_workspace");
        take(g_linear_logprobs_forward, "frnn_linear_logprobs_forward");
        take(g_linear_logprobs_forward_workspace, "frnn_linear_logprobs_forward_workspace");
        take(g_linear_logprobs_backward, "frnn_linear_logprobs_backward");
        take(g_linear_logprobs_backward_workspace, "frnn_linear_logprobs_backward_workspace");
        take(g_rotary, "frnn_rotary");
    });
}
