// What the PyTorch operators around the scans (frnn_lm_host.cpp, frnn_block_host.cpp) share: checks of arguments, allocation,
// the debugging switches, and what an autograd node needs.
#pragma once
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <atomic>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

#include "../../include/frnn.h"

namespace py = pybind11;
using at::Tensor;
using std::optional;
using torch::autograd::variable_list;

namespace frnn_ops {

inline decltype(&frnn_last_error) g_last_error = nullptr;

enum { MAX_DEVICES = 64 };
inline std::atomic<int*> g_word[MAX_DEVICES];           // error words in pinned host memory, by device
inline PyObject *g_word_of = nullptr, *g_raise = nullptr;     // Python: (device) -> address of its word; (device) raises what it says

// Run a Python callable from any thread; its exception keeps its type.
template <class F> auto with_python(F f) {
    py::gil_scoped_acquire g;
    try {
        return f();
    } catch (py::error_already_set& e) {
        e.restore();
        python_error err;
        err.persist();
        throw std::move(err);
    }
}

// FRNN_GUARD=1: every buffer that kernels write lies between two bands of a byte pattern, which are looked at after the
// call; FRNN_CHECK=1: each call waits and raises what its kernels reported.  Debugging only: both wait for the GPU.
enum { BAND = 4096, FILL = 0xA5 };
struct Guarded {
    const char* what;
    Tensor raw;
    int64_t bytes;
};
inline thread_local bool t_guard = false, t_check = false;
inline thread_local std::vector<Guarded> t_guarded;

inline bool asked(const char* name) {
    const char* e = getenv(name);
    return e && *e && strcmp(e, "0");
}

// The error word of a device, after raising what kernels of earlier calls left there.  A call begins with it.
inline int* error_word(c10::DeviceIndex device) {
    t_guard = asked("FRNN_GUARD");
    t_check = asked("FRNN_CHECK");
    t_guarded.clear();
    TORCH_CHECK(device >= 0 && device < MAX_DEVICES, "flex_rnn_b200: device index ", (int)device);
    int* w = g_word[device].load(std::memory_order_acquire);
    if (!w) {
        w = with_python([&] { return (int*)py::cast<uintptr_t>(py::reinterpret_borrow<py::object>(g_word_of)((int)device)); });
        g_word[device].store(w, std::memory_order_release);
    }
    if (*(volatile int*)w) with_python([&] { py::reinterpret_borrow<py::object>(g_raise)((int)device); });
    return w;
}

inline void* stream_of(const Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The end of a call: its return code, and what the debugging switches ask for.
inline void ran(int rc, const Tensor& like) {
    TORCH_CHECK(rc == FRNN_OK, "flex_rnn_b200: ", g_last_error());
    if (t_guard || t_check) c10::cuda::getCurrentCUDAStream(like.device().index()).synchronize();
    std::vector<Guarded> guarded;
    guarded.swap(t_guarded);
    for (const Guarded& g : guarded) {
        const int64_t lo = g.raw.narrow(0, 0, BAND).ne(FILL).sum().item<int64_t>(), hi = g.raw.narrow(0, BAND + g.bytes, g.raw.numel() - BAND - g.bytes).ne(FILL).sum().item<int64_t>();
        TORCH_CHECK(!lo && !hi, "flex_rnn_b200: a kernel wrote ", lo + hi, " byte(s) outside ", g.what, " (", lo ? "before" : "after", " the buffer)");
    }
    if (t_check) {
        const bool guard = t_guard;
        error_word(like.device().index());
        t_guard = guard;
    }
}

inline int dtype_of(const char* op, const char* what, const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return FRNN_F32;
        case at::kBFloat16: return FRNN_BF16;
        case at::kHalf: return FRNN_F16;
        default: TORCH_CHECK(false, "flex_rnn_b200: ", op, ": ", what, " has to be float32, bfloat16 or float16, got ", t.scalar_type());
    }
}

inline void check_one(const char* op, const char* what, const Tensor& t, const Tensor& first) {
    TORCH_CHECK(t.layout() == at::kStrided, "flex_rnn_b200: ", op, ": ", what, " has to be a strided tensor");
    TORCH_CHECK(t.is_cuda() && t.device() == first.device(), "flex_rnn_b200: all tensors of a call have to be on one CUDA device, got ", first.device(), " and ", t.device());
    if (t.numel() == 0) return;
    int64_t reach = 1;
    for (int64_t d = 0; d < t.dim(); d++) reach += (t.size(d) - 1) * t.stride(d);
    TORCH_CHECK((size_t)(reach + t.storage_offset()) * t.element_size() <= t.storage().nbytes(), "flex_rnn_b200: ", op, ": the strides of ", what,
                " reach past the end of its storage");
}

inline Tensor check_tokens(const char* op, const Tensor& tokens, const Tensor& first) {
    TORCH_CHECK(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "flex_rnn_b200: ", op, ": tokens have to be int64 or int32, got ", tokens.scalar_type());
    check_one(op, "tokens", tokens, first);
    return tokens.contiguous();
}

inline Tensor make_strided(const char* what, at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type, const Tensor& like) {
    if (!t_guard) return at::detail::empty_strided_cuda(sizes, strides, type, like.device());
    int64_t extent = 1;
    for (size_t d = 0; d < sizes.size(); d++) extent = sizes[d] == 0 ? 0 : extent ? extent + (sizes[d] - 1) * strides[d] : 0;
    const int64_t bytes = extent * (int64_t)c10::elementSize(type);
    Tensor raw = at::detail::empty_strided_cuda({2 * BAND + (bytes + 255) / 256 * 256}, {1}, at::kByte, like.device());
    raw.fill_(FILL);
    t_guarded.push_back({what, raw, bytes});
    return raw.narrow(0, BAND, bytes).view(type).as_strided(sizes, strides);
}

inline Tensor make(const char* what, at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    std::vector<int64_t> strides(sizes.size());
    int64_t s = 1;
    for (size_t d = sizes.size(); d--;) { strides[d] = s; s *= std::max<int64_t>(1, sizes[d]); }
    return make_strided(what, sizes, strides, type, like);
}

// What a forward saved, contiguous and on a 16-byte boundary, whatever a saved-tensor hook made of it.
inline Tensor saved(const Tensor& t) {
    const Tensor c = t.contiguous();
    return (uintptr_t)c.data_ptr() & 15 ? c.clone() : c;
}

// Rows along the last dimension: one stride between rows and consecutive elements, else a contiguous copy.
inline Tensor as_rows(const Tensor& t) {
    const int64_t width = t.size(-1);
    if (t.dim() == 1) return t.stride(0) == 1 || width == 1 ? t.unsqueeze(0) : t.contiguous().unsqueeze(0);
    if (t.stride(-1) != 1 && width > 1) return t.contiguous().reshape({-1, width});
    return t.reshape({-1, width});
}

inline Tensor workspace(size_t bytes, const Tensor& like) { return bytes ? make("the workspace", {(int64_t)bytes}, at::kByte, like) : Tensor(); }
template <class T = void> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
template <class T = void> T* ptr(const optional<Tensor>& t) { return t.has_value() && t->defined() ? (T*)t->data_ptr() : nullptr; }

// ---- autograd ------------------------------------------------------------------------------------------------------------

// Gradients of gradients are refused, but only when they are asked for: create_graph=True alone is no error.
struct OnlyOnce : torch::autograd::Node {
    explicit OnlyOnce(torch::autograd::edge_list&& e) : Node(std::move(e)) {}
    std::string name() const override { return "OnlyOnce"; }
    variable_list apply(variable_list&&) override { TORCH_CHECK(false, "flex_rnn_b200: gradients of this operator are not differentiable through autograd in their turn"); }
};

template <class... A> void only_once(std::initializer_list<Tensor*> results, const A&... inputs) {
    if (!at::GradMode::is_enabled()) return;
    variable_list in;
    auto add = [&](const optional<Tensor>& t) { if (t.has_value() && t->defined()) in.push_back(*t); };
    (add(inputs), ...);
    if (!torch::autograd::any_variable_requires_grad(in)) return;
    for (Tensor* t : results) {
        if (!t->defined()) continue;
        auto node = std::shared_ptr<OnlyOnce>(new OnlyOnce(torch::autograd::collect_next_edges(in)), torch::autograd::deleteNode);
        torch::autograd::create_gradient_edge(*t, node);
    }
}

inline bool needs(const optional<Tensor>& t) { return t.has_value() && t->defined() && t->requires_grad(); }
inline optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); }

// A node of the autograd graph: what a call saved, until it has been used.  (torch::autograd::Function does the same with
// more on the way; a training call of small tensors is all host time.)
struct Saving : torch::autograd::Node {
    std::vector<torch::autograd::SavedVariable> saved;
    bool released = false;
    explicit Saving(torch::autograd::edge_list&& e) : Node(std::move(e)) {}
    void save(const Tensor& t) { saved.emplace_back(t, false); }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto& v : saved) v.reset_data();
        released = true;
    }
    variable_list unpack() {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        variable_list kept;
        kept.reserve(saved.size());
        for (auto& v : saved) kept.push_back(v.unpack(shared_from_this()));
        return kept;
    }
};

template <class N, class... T> std::shared_ptr<N> make_node(const T&... inputs) {
    return std::shared_ptr<N>(new N(torch::autograd::collect_next_edges(inputs...)), torch::autograd::deleteNode);
}

// Forward and backward refuse what would otherwise be dropped without a word: a tangent may come on an upstream gradient alone.
inline void no_tangent(const optional<Tensor>& t) {
    TORCH_CHECK(!t.has_value() || !t->defined() || !t->_fw_grad(0).defined(), "flex_rnn_b200: forward-mode derivatives of this operator are not built");
}

// There is no CPU path: tensors elsewhere are refused by name.
template <class R, class... A> struct Refuse;
template <class R, class... A> struct Refuse<R(A...)> {
    static R run(A...) { TORCH_CHECK(false, "flex_rnn_b200: the operators around the scans run on CUDA tensors; there is no CPU path"); }
};

#define FRNN_OP(name, fn) \
    auto name() -> const c10::TypedOperatorHandle<decltype(fn)>& { \
        static const auto handle = c10::Dispatcher::singleton().findSchemaOrThrow("flex_rnn_b200::" #name, "").typed<decltype(fn)>(); \
        return handle; \
    }
#define FRNN_ON_CUDA(name) TORCH_FN(name##_cuda)
#define FRNN_ON_AUTOGRAD(name) TORCH_FN(name##_autograd)
#define FRNN_REFUSED(name) TORCH_FN(Refuse<decltype(name##_cuda)>::run)

}  // namespace frnn_ops
