// The operators around the scans as PyTorch operators (flex_rnn_b200::embedding, layer_norm, token_logprobs and their
// backward): checks of arguments, layouts, allocation, autograd.  Kernels are reached through the C ABI of
// libfrnn_b200.so (include/frnn.h), whose entry points are handed over by address, on the current stream.  They are
// dispatcher operators, so torch.compile, fake tensors and dispatch modes see each call as one operator.
#include "frnn_lm_host.h"

using namespace frnn_ops;

namespace {

decltype(&frnn_embedding_forward) g_embedding_forward = nullptr;
decltype(&frnn_embedding_backward) g_embedding_backward = nullptr;
decltype(&frnn_embedding_backward_workspace) g_embedding_backward_workspace = nullptr;
decltype(&frnn_layer_norm_forward) g_layer_norm_forward = nullptr;
decltype(&frnn_layer_norm_backward) g_layer_norm_backward = nullptr;
decltype(&frnn_layer_norm_backward_workspace) g_layer_norm_backward_workspace = nullptr;
decltype(&frnn_token_logprobs_forward) g_token_logprobs_forward = nullptr;
decltype(&frnn_token_logprobs_backward) g_token_logprobs_backward = nullptr;

// ---- embedding ----------------------------------------------------------------------------------------------------------

Tensor embedding_cuda(const Tensor& tokens, const Tensor& weight, double scale, int64_t ignore_index) {
    const char* op = "embedding";
    const int dtype = dtype_of(op, "weight", weight);
    TORCH_CHECK(weight.dim() == 2, "flex_rnn_b200: embedding: weight has to be [vocabulary, width], got ", weight.sizes());
    check_one(op, "weight", weight, weight);
    const Tensor tok = check_tokens(op, tokens, weight);
    c10::cuda::CUDAGuard guard(weight.device());
    int* err = error_word(weight.device().index());
    auto sizes = tokens.sizes().vec();
    sizes.push_back(weight.size(1));
    Tensor out = make("the output", sizes, weight.scalar_type(), weight);
    ran(g_embedding_forward(dtype, weight.data_ptr(), weight.size(0), weight.size(1), weight.stride(0), weight.stride(1), tok.data_ptr(), (int)tok.element_size(),
                            tok.numel(), (float)scale, ignore_index, out.data_ptr(), err, stream_of(weight)), weight);
    return out;
}

Tensor embedding_backward_cuda(const Tensor& grad, const Tensor& tokens, int64_t rows, double scale, int64_t ignore_index) {
    const char* op = "embedding_backward";
    const int dtype = dtype_of(op, "the gradient", grad);
    TORCH_CHECK(grad.dim() >= 1 && grad.sizes().slice(0, grad.dim() - 1) == tokens.sizes() && rows >= 0, "flex_rnn_b200: embedding_backward: the gradient has to be ",
                "[*tokens.shape, width], got ", grad.sizes(), " for tokens ", tokens.sizes());
    check_one(op, "the gradient", grad, grad);
    const Tensor tok = check_tokens(op, tokens, grad);
    c10::cuda::CUDAGuard guard(grad.device());
    error_word(grad.device().index());
    const int64_t width = grad.size(-1), n = tok.numel();
    const Tensor g = grad.contiguous(), work = workspace(g_embedding_backward_workspace(dtype, rows, width, n), grad);
    Tensor dw = make("the weight's gradient", {rows, width}, grad.scalar_type(), grad);
    ran(g_embedding_backward(dtype, g.data_ptr(), tok.data_ptr(), (int)tok.element_size(), n, rows, width, (float)scale, ignore_index, dw.data_ptr(), ptr(work), stream_of(grad)), grad);
    return dw;
}

// ---- layer norm ---------------------------------------------------------------------------------------------------------

// The rows of x and of tensors of its shape: leading dimensions that are one run in all of them become one.  The last
// leading dimension stays on its own where there are weights for each head.  False where that takes more than three.
bool rows_of(const Tensor* const* t, int count, bool heads, frnn_rows& r) {
    const Tensor& x = *t[0];
    std::vector<int64_t> n;
    std::vector<std::vector<int64_t>> s(count);
    const int64_t lead = x.dim() - 1;
    for (int64_t d = 0; d < lead; d++) {
        const bool apart = heads && d == lead - 1;
        if (x.size(d) == 1 && !apart) continue;
        bool joins = !n.empty() && !apart;
        for (int i = 0; i < count && joins; i++) joins = s[i].back() == t[i]->size(d) * t[i]->stride(d);
        if (joins) {
            n.back() *= x.size(d);
            for (int i = 0; i < count; i++) s[i].back() = t[i]->stride(d);
        } else {
            n.push_back(x.size(d));
            for (int i = 0; i < count; i++) s[i].push_back(t[i]->stride(d));
        }
    }
    if (n.size() > 3) return false;
    int64_t* to[3] = {r.x, r.dy, r.dx};
    r.n0 = r.n1 = r.n2 = 1;
    int64_t* size[3] = {&r.n0, &r.n1, &r.n2};
    for (int k = 0; k < 3; k++)
        for (int i = 0; i < 3; i++) to[i][k] = 0;
    const size_t first = n.size() == 1 && !heads ? 0 : 3 - n.size();      // (one run alone is n0: kernels step through it; n2 is for heads)
    for (size_t k = 0; k < n.size(); k++) {
        *size[first + k] = n[k];
        for (int i = 0; i < count; i++) to[i][first + k] = s[i][k];
    }
    r.width = x.size(-1);
    r.heads = heads ? x.size(-2) : 1;
    return true;
}

// Kernels read the elements of a row one after the other; other layouts are copied first.
bool rows_dense(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

int check_params(const char* op, const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, bool& heads) {
    int dtype = FRNN_F32;
    heads = false;
    TORCH_CHECK(x.dim() >= 1, "flex_rnn_b200: ", op, ": x has to have at least one dimension");
    const Tensor* first = nullptr;
    for (const auto* p : {&weight, &bias}) {
        if (!p->has_value() || !(*p)->defined()) continue;
        const Tensor& w = **p;
        const char* what = p == &weight ? "weight" : "bias";
        dtype = dtype_of(op, what, w);
        TORCH_CHECK(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "flex_rnn_b200: ", op, ": ", what, " has to have the type of x or be float32, got ",
                    w.scalar_type(), " for x in ", x.scalar_type());
        const bool vector = w.dim() == 1 && w.size(0) == x.size(-1), each = w.dim() == 2 && x.dim() >= 2 && w.size(0) == x.size(-2) && w.size(1) == x.size(-1);
        TORCH_CHECK(vector || each, "flex_rnn_b200: ", op, ": ", what, " has to be [width] or [heads, width] for x [..., heads, width], got ", w.sizes(), " for x ", x.sizes());
        TORCH_CHECK(!first || (first->sizes() == w.sizes() && first->scalar_type() == w.scalar_type()), "flex_rnn_b200: ", op,
                    ": weight and bias have to have one shape and type");
        check_one(op, what, w, x);
        first = &w;
        heads = each;
    }
    return dtype;
}

optional<Tensor> dense(const optional<Tensor>& t) { return t.has_value() && t->defined() ? optional<Tensor>(t->contiguous()) : optional<Tensor>(); }

std::tuple<Tensor, Tensor> layer_norm_cuda(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps, bool save) {
    const char* op = "layer_norm";
    const int dtype = dtype_of(op, "x", x);
    bool heads;
    const int ptype = check_params(op, x, weight, bias, heads);
    check_one(op, "x", x, x);
    c10::cuda::CUDAGuard guard(x.device());
    error_word(x.device().index());
    frnn_rows r;
    Tensor from = x;
    const Tensor* ts[1] = {&from};
    if (!rows_dense(x) || !rows_of(ts, 1, heads, r)) {
        from = x.contiguous();
        TORCH_INTERNAL_ASSERT(rows_of(ts, 1, heads, r));
    }
    Tensor y = make("the output", x.sizes(), x.scalar_type(), x);
    const int64_t rows = x.numel() ? x.numel() / x.size(-1) : 0;
    Tensor stats = make("the statistics", {save ? rows : 0, 2}, at::kFloat, x);
    const optional<Tensor> w = dense(weight), b = dense(bias);
    if (x.numel()) ran(g_layer_norm_forward(&r, dtype, from.data_ptr(), ptype, ptr(w), ptr(b), (float)eps, y.data_ptr(), save ? stats.data_ptr<float>() : nullptr, stream_of(x)), x);
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_cuda(const Tensor& grad, const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, const Tensor& stats,
                                                            bool want_x, bool want_weight, bool want_bias) {
    const char* op = "layer_norm_backward";
    const int dtype = dtype_of(op, "x", x);
    bool heads;
    const int ptype = check_params(op, x, weight, bias, heads);
    check_one(op, "x", x, x);
    check_one(op, "the gradient", grad, x);
    check_one(op, "the statistics", stats, x);
    const int64_t rows = x.numel() ? x.numel() / x.size(-1) : 0;
    TORCH_CHECK(grad.sizes() == x.sizes() && grad.scalar_type() == x.scalar_type(), "flex_rnn_b200: layer_norm_backward: the gradient has to have the shape and type of x");
    TORCH_CHECK(stats.dim() == 2 && stats.size(0) == rows && stats.size(1) == 2 && stats.scalar_type() == at::kFloat, "flex_rnn_b200: layer_norm_backward: the statistics have to be those of the forward");
    c10::cuda::CUDAGuard guard(x.device());
    error_word(x.device().index());
    Tensor dx = want_x && !t_guard ? at::empty_like(x) : Tensor();
    if (want_x && t_guard) {
        const Tensor shape = at::empty_like(x, x.options().device(at::kMeta));      // (the same layout)
        dx = make_strided("x's gradient", shape.sizes(), shape.strides(), x.scalar_type(), x);
    }
    Tensor from = rows_dense(x) ? x : x.contiguous(), g = rows_dense(grad) ? grad : grad.contiguous(), to = want_x && rows_dense(dx) ? dx : make("x's gradient", x.sizes(), x.scalar_type(), x);
    frnn_rows r;
    const Tensor* ts[3] = {&from, &g, &to};
    if (!rows_of(ts, 3, heads, r)) {
        from = x.contiguous();
        g = grad.contiguous();
        to = make("x's gradient", x.sizes(), x.scalar_type(), x);
        TORCH_INTERNAL_ASSERT(rows_of(ts, 3, heads, r));
    }
    const optional<Tensor> w = dense(weight);
    const Tensor st = saved(stats);
    auto param = [&](bool want, const optional<Tensor>& p) { return want && p.has_value() && p->defined() ? make("a weight's gradient", p->sizes(), p->scalar_type(), x) : Tensor(); };
    Tensor dw = param(want_weight, weight), db = param(want_bias, bias);
    if (x.size(-1) && r.heads) {                           // (without a head the weights have no element either)
        const Tensor work = dw.defined() || db.defined() ? workspace(g_layer_norm_backward_workspace(&r), x) : Tensor();
        ran(g_layer_norm_backward(&r, dtype, g.data_ptr(), from.data_ptr(), ptype, ptr(w), st.data_ptr<float>(), want_x ? to.data_ptr() : nullptr, ptr(dw), ptr(db), ptr(work),
                                  stream_of(x)), x);
    }
    if (want_x && !to.is_same(dx)) dx.copy_(to);
    auto some = [&](const Tensor& t) { return t.defined() ? t : make("nothing", {0}, x.scalar_type(), x); };
    return {some(dx), some(dw), some(db)};
}

// ---- log probabilities of tokens ------------------------------------------------------------------------------------------

void check_logits(const char* op, const Tensor& logits, const Tensor& tokens) {
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, "flex_rnn_b200: ", op, ": logits have to be [..., vocabulary] with a vocabulary that is not empty, got ", logits.sizes());
    TORCH_CHECK(logits.sizes().slice(0, logits.dim() - 1) == tokens.sizes(), "flex_rnn_b200: ", op, ": tokens have to have the shape of logits without its last dimension, got ",
                tokens.sizes(), " for logits ", logits.sizes());
    check_one(op, "logits", logits, logits);
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_cuda(const Tensor& logits, const Tensor& tokens, int64_t top, double temperature, int64_t ignore_index, bool save) {
    const char* op = "token_logprobs";
    const int dtype = dtype_of(op, "logits", logits);
    check_logits(op, logits, tokens);
    const int64_t vocab = logits.size(-1), n = tokens.numel();
    TORCH_CHECK(top >= 0 && top <= FRNN_MAX_TOP && top <= vocab, "flex_rnn_b200: token_logprobs: top has to be 0 to ", (int)FRNN_MAX_TOP, " and at most the vocabulary, got ", top);
    TORCH_CHECK(temperature >= 1e-30 && temperature <= 1e30, "flex_rnn_b200: token_logprobs: the temperature has to be positive, from 1e-30 to 1e30, got ", temperature);
    const Tensor tok = check_tokens(op, tokens, logits);
    c10::cuda::CUDAGuard guard(logits.device());
    int* err = error_word(logits.device().index());
    const Tensor x = n ? as_rows(logits) : logits;
    auto sizes = tokens.sizes().vec();
    Tensor lp = make("the log probabilities", sizes, at::kFloat, logits), ent = make("the entropies", sizes, at::kFloat, logits), stats = make("the statistics", {save ? n : 0, 3}, at::kFloat, logits);
    sizes.push_back(top);
    Tensor top_lp = make("the alternatives' log probabilities", sizes, at::kFloat, logits), top_tok = make("the alternatives", sizes, at::kLong, logits);
    if (n)
        ran(g_token_logprobs_forward(dtype, x.data_ptr(), n, vocab, x.stride(0), tok.data_ptr(), (int)tok.element_size(), (int)top, (float)temperature, ignore_index, lp.data_ptr<float>(),
                                     ent.data_ptr<float>(), top_lp.data_ptr<float>(), top_tok.data_ptr<int64_t>(), save ? stats.data_ptr<float>() : nullptr, err, stream_of(logits)), logits);
    return {lp, ent, top_lp, top_tok, stats};
}

Tensor token_logprobs_backward_cuda(const optional<Tensor>& dlogprob, const optional<Tensor>& dentropy, const Tensor& logits, const Tensor& tokens, const Tensor& stats,
                                    double temperature, int64_t ignore_index) {
    const char* op = "token_logprobs_backward";
    const int dtype = dtype_of(op, "logits", logits);
    check_logits(op, logits, tokens);
    const Tensor tok = check_tokens(op, tokens, logits);
    check_one(op, "the statistics", stats, logits);
    const int64_t vocab = logits.size(-1), n = tokens.numel();
    TORCH_CHECK(stats.dim() == 2 && stats.size(0) == n && stats.size(1) == 3 && stats.scalar_type() == at::kFloat, "flex_rnn_b200: token_logprobs_backward: the statistics have to be those of the forward");
    auto upstream = [&](const optional<Tensor>& g) {
        if (!g.has_value() || !g->defined()) return Tensor();
        TORCH_CHECK(g->sizes() == tokens.sizes(), "flex_rnn_b200: token_logprobs_backward: upstream gradients have to have the shape of tokens");
        check_one(op, "an upstream gradient", *g, logits);
        return g->to(at::kFloat).contiguous();
    };
    c10::cuda::CUDAGuard guard(logits.device());
    error_word(logits.device().index());
    const Tensor glp = upstream(dlogprob), gent = upstream(dentropy), st = saved(stats), x = n ? as_rows(logits) : logits;
    Tensor dx = make("the logits' gradient", logits.sizes(), logits.scalar_type(), logits);
    if (n)
        ran(g_token_logprobs_backward(dtype, x.data_ptr(), n, vocab, x.stride(0), tok.data_ptr(), (int)tok.element_size(), (float)temperature, ignore_index, ptr<float>(glp),
                                      ptr<float>(gent), st.data_ptr<float>(), dx.data_ptr(), stream_of(logits)), logits);
    return dx;
}

// ---- autograd ------------------------------------------------------------------------------------------------------------

FRNN_OP(embedding, embedding_cuda)
FRNN_OP(embedding_backward, embedding_backward_cuda)
FRNN_OP(layer_norm, layer_norm_cuda)
FRNN_OP(layer_norm_backward, layer_norm_backward_cuda)
FRNN_OP(token_logprobs, token_logprobs_cuda)
FRNN_OP(token_logprobs_backward, token_logprobs_backward_cuda)

struct EmbeddingBackward : Saving {
    using Saving::Saving;
    int64_t rows, ignore_index;
    double scale;
    std::string name() const override { return "EmbeddingBackward"; }
    variable_list apply(variable_list&& up) override {
        if (!up[0].defined() || !task_should_compute_output(0)) return {Tensor()};
        return {embedding_backward().call(up[0], unpack()[0], rows, scale, ignore_index)};
    }
};

Tensor embedding_autograd(const Tensor& tokens, const Tensor& weight, double scale, int64_t ignore_index) {
    no_tangent(weight);
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = embedding().call(tokens, weight, scale, ignore_index);
    }
    if (at::GradMode::is_enabled() && needs(weight)) {
        auto node = make_node<EmbeddingBackward>(weight);
        node->rows = weight.size(0);
        node->scale = scale;
        node->ignore_index = ignore_index;
        node->save(tokens);
        torch::autograd::create_gradient_edge(y, node);
    }
    return y;
}

Tensor embedding_backward_autograd(const Tensor& grad, const Tensor& tokens, int64_t rows, double scale, int64_t ignore_index) {
    no_tangent(grad);
    Tensor dw;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        dw = embedding_backward().call(grad, tokens, rows, scale, ignore_index);
    }
    only_once({&dw}, grad);
    return dw;
}

// Bytes of a tensor's first element behind a 16-byte boundary (its storage starts on one; a fake tensor has no address, and
// an offset that is symbolic while a call is traced does not matter: no hook moves what is saved there).
int64_t behind_boundary(const Tensor& t) { return t.sym_storage_offset().maybe_as_int().value_or(0) * (int64_t)t.element_size() & 15; }

struct LayerNormBackward : Saving {
    using Saving::Saving;
    int64_t behind;
    std::string name() const override { return "LayerNormBackward"; }
    variable_list apply(variable_list&& up) override {
        if (!up[0].defined()) return {Tensor(), Tensor(), Tensor()};
        variable_list kept = unpack();          // x, weight, bias (says only whether there is one, and of which shape), statistics
        // a saved-tensor hook may move x off the boundary it was on; the sums have the order of aligned rows all the same
        if (behind_boundary(kept[0]) && !behind) kept[0] = kept[0].clone();
        const bool wx = task_should_compute_output(0), ww = kept[1].defined() && task_should_compute_output(1), wb = kept[2].defined() && task_should_compute_output(2);
        auto [dx, dw, db] = layer_norm_backward().call(up[0], kept[0], maybe(kept[1]), maybe(kept[2]), kept[3], wx, ww, wb);
        return {wx ? dx : Tensor(), ww ? dw : Tensor(), wb ? db : Tensor()};
    }
};

std::tuple<Tensor, Tensor> layer_norm_autograd(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps, bool save) {
    no_tangent(x);
    no_tangent(weight);
    no_tangent(bias);
    const bool grad = at::GradMode::is_enabled() && (needs(x) || needs(weight) || needs(bias));
    std::tuple<Tensor, Tensor> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = layer_norm().call(x, weight, bias, eps, save || grad);
    }
    if (grad) {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
        auto node = make_node<LayerNormBackward>(x, w, b);
        node->behind = behind_boundary(x);
        for (const Tensor& t : {x, w, b, std::get<1>(r)}) node->save(t);
        torch::autograd::create_gradient_edge(std::get<0>(r), node);
    }
    return r;
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_autograd(const Tensor& grad, const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, const Tensor& stats,
                                                                bool want_x, bool want_weight, bool want_bias) {
    no_tangent(grad);
    no_tangent(x);
    no_tangent(weight);
    std::tuple<Tensor, Tensor, Tensor> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = layer_norm_backward().call(grad, x, weight, bias, stats, want_x, want_weight, want_bias);
    }
    only_once({&std::get<0>(r), &std::get<1>(r), &std::get<2>(r)}, grad, x, weight);
    return r;
}

struct TokenLogprobsBackward : Saving {
    using Saving::Saving;
    double temperature;
    int64_t ignore_index;
    std::string name() const override { return "TokenLogprobsBackward"; }
    variable_list apply(variable_list&& up) override {
        if ((!up[0].defined() && !up[1].defined()) || !task_should_compute_output(0)) return {Tensor()};
        const variable_list kept = unpack();
        return {token_logprobs_backward().call(maybe(up[0]), maybe(up[1]), kept[0], kept[1], kept[2], temperature, ignore_index)};
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_autograd(const Tensor& logits, const Tensor& tokens, int64_t top, double temperature, int64_t ignore_index, bool save) {
    no_tangent(logits);
    const bool grad = at::GradMode::is_enabled() && needs(logits);
    std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = token_logprobs().call(logits, tokens, top, temperature, ignore_index, save || grad);
    }
    if (grad) {
        auto node = make_node<TokenLogprobsBackward>(logits);
        node->temperature = temperature;
        node->ignore_index = ignore_index;
        for (const Tensor& t : {logits, tokens, std::get<4>(r)}) node->save(t);
        torch::autograd::create_gradient_edge(std::get<0>(r), node);
        torch::autograd::create_gradient_edge(std::get<1>(r), node);
    }
    return r;
}

Tensor token_logprobs_backward_autograd(const optional<Tensor>& dlogprob, const optional<Tensor>& dentropy, const Tensor& logits, const Tensor& tokens, const Tensor& stats,
                                        double temperature, int64_t ignore_index) {
    no_tangent(dlogprob);
    no_tangent(dentropy);
    no_tangent(logits);
    Tensor dx;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        dx = token_logprobs_backward().call(dlogprob, dentropy, logits, tokens, stats, temperature, ignore_index);
    }
    only_once({&dx}, dlogprob, dentropy, logits);
    return dx;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(flex_rnn_b200, m) {
    m.def("embedding(Tensor tokens, Tensor weight, float scale, int ignore_index) -> Tensor");
    m.def("embedding_backward(Tensor grad, Tensor tokens, int rows, float scale, int ignore_index) -> Tensor");
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool save) -> (Tensor, Tensor)");
    m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, bool want_x, bool want_weight, bool want_bias) -> (Tensor, Tensor, Tensor)");
    m.def("token_logprobs(Tensor logits, Tensor tokens, int top, float temperature, int ignore_index, bool save) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("token_logprobs_backward(Tensor? dlogprob, Tensor? dentropy, Tensor logits, Tensor tokens, Tensor stats, float temperature, int ignore_index) -> Tensor");
}

#define FRNN_ALL(how) \
    m.impl("embedding", how(embedding)); \
    m.impl("embedding_backward", how(embedding_backward)); \
    m.impl("layer_norm", how(layer_norm)); \
    m.impl("layer_norm_backward", how(layer_norm_backward)); \
    m.impl("token_logprobs", how(token_logprobs)); \
    m.impl("token_logprobs_backward", how(token_logprobs_backward));

TORCH_LIBRARY_IMPL(flex_rnn_b200, CUDA, m) { FRNN_ALL(FRNN_ON_CUDA) }
TORCH_LIBRARY_IMPL(flex_rnn_b200, Autograd, m) { FRNN_ALL(FRNN_ON_AUTOGRAD) }
TORCH_LIBRARY_IMPL(flex_rnn_b200, CPU, m) { FRNN_ALL(FRNN_REFUSED) }

void frnn_bind_lm(py::module& m) {
    m.def("bind_lm", [](const std::map<std::string, uintptr_t>& at_, py::object word_of, py::object raise) {
        auto take = [&](auto& fn, const char* name) { fn = (std::decay_t<decltype(fn)>)at_.at(name); };
        take(g_last_error, "frnn_last_error");
        take(g_embedding_forward, "frnn_embedding_forward");
        take(g_embedding_backward, "frnn_embedding_backward");
        take(g_embedding_backward_workspace, "frnn_embedding_backward_workspace");
        take(g_layer_norm_forward, "frnn_layer_norm_forward");
        take(g_layer_norm_backward, "frnn_layer_norm_backward");
        take(g_layer_norm_backward_workspace, "frnn_layer_norm_backward_workspace");
        take(g_token_logprobs_forward, "frnn_token_logprobs_forward");
        take(g_token_logprobs_backward, "frnn_token_logprobs_backward");
        g_word_of = word_of.release().ptr();      // kept until the process ends
        g_raise = raise.release().ptr();
    });
}
