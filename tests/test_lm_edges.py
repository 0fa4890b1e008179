"""Calls of the operators around the scans (flex_rnn_b200.lm) at their edges; tolerances are those of test_lm."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as ad

import flex_rnn_b200 as fr
from flex_rnn_b200 import build, lm, runtime
from conftest import ROOT
from test_lm import DTYPES, both, calls, layer_norm_check, logits_of, logprobs_check, params, rand


# ---- log probabilities: NaN --------------------------------------------------------------------------------------------------

def short_row(dtype):
    """The longest row that one warp takes where there are rows enough."""
    return 8192 // torch.finfo(dtype).bits * 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V", [(3, 9001), (3, 70000), (400, 40000), (1300, 0)])
def test_nan_among_masked_logits(n, V, dtype):
    """A NaN makes its row NaN whatever follows it: rows whose other logits are all -inf, or nearly all, with the NaN in the
    first loads of a thread that has more of them.  Rows of nothing but -inf stay what they are."""
    V = V or short_row(dtype) - 3
    x = torch.full((n, V), -math.inf, dtype=dtype, device="cuda")
    t = torch.full((n,), 5, device="cuda")
    at = [3, 0]
    for row in range(n):
        if row % 3 != 2:
            x[row, at[row % 3]] = math.nan
    x[1, 7] = 1.5
    leaf = x.requires_grad_()
    r = fr.token_logprobs(leaf, t, top=4)
    g = torch.autograd.grad((r.logprob, r.entropy), leaf, (torch.ones(n, device="cuda"), torch.ones(n, device="cuda")))[0]
    bad = torch.arange(n, device="cuda") % 3 != 2
    for v in (r.logprob, r.entropy):
        assert torch.equal(v.isnan(), bad)
    assert torch.equal(r.top_logprob.isnan().all(1), bad) and torch.equal(g.isnan().all(1), bad)
    assert (r.logprob[~bad] == -math.inf).all() and not r.entropy[~bad].any() and not g[~bad].any()
    assert r.top_token[0].tolist() == [3, 0, 1, 2] and r.top_token[1].tolist() == [0, 7, 1, 2] and r.top_token[2].tolist() == [0, 1, 2, 3]


def few_threads(n, V, dtype, threads, block, seed=0):
    """Logits of which only the accesses (16 bytes) of a few of a block's threads are large, so that next to no group of
    threads holds a large one and the bound for candidates lets most of theirs through."""
    x, t = logits_of(n, V, dtype, seed=seed)
    access = torch.arange(V, device="cuda") // (128 // torch.finfo(dtype).bits)
    return torch.where(access % block < threads, x + 40.0, x - 40.0).to(dtype), t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_of_few_threads(dtype):
    """More candidates than there is room for, all of them distinct in rank: one block, a cluster, one warp a row."""
    logprobs_check(*few_threads(300, 40000, dtype, 16, 256), top=8)
    logprobs_check(*few_threads(3, 200000, dtype, 16, 256), top=8)
    logprobs_check(*few_threads(1300, short_row(dtype), dtype, 9, 32), top=12)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_of_nan(dtype):
    """NaN comes before every number and by the lowest token, token 0 among them, also where candidates are too many."""
    for (n, V, threads, block, top) in [(300, 40000, 16, 256, 8), (3, 200000, 16, 256, 8), (1300, short_row(dtype), 9, 32, 12), (3, 900, 9, 256, 12)]:
        x, t = few_threads(n, V, dtype, threads, block)
        best = x[0].sort(descending=True, stable=True).indices[:top].tolist()
        x[0, 0] = math.nan
        x[1] = math.nan
        x[2, 5], x[2, V - 2] = math.nan, math.nan
        r = fr.token_logprobs(x, t, top=top)
        assert r.top_token[0].tolist() == ([0] + [i for i in best if i != 0])[:top]
        assert r.top_token[1].tolist() == list(range(top))
        assert r.top_token[2, :2].tolist() == [5, V - 2]
        assert r.top_logprob[:3].isnan().all() and r.top_logprob[3:].isfinite().all()


# ---- layer norm: few rows ------------------------------------------------------------------------------------------------------

def test_layer_norm_workspace_follows_the_rows():
    """Partial sums of weight gradients: no more than one for each row (with weights for each head: for each group of a block
    that has a row), however the rows are divided."""
    L, i64 = runtime.lib(), ctypes.c_int64
    L.frnn_layer_norm_backward_workspace.restype = ctypes.c_size_t

    def partials(n, width, heads):
        rows = (i64 * 14)(*n, width, heads, *[0] * 9)
        return L.frnn_layer_norm_backward_workspace(rows) // (8 * ((width + 3) // 4 * 4))

    for width in (16, 77, 128, 601, 1001, 2047, 4096, 8192):
        for rows in (*range(1, 300, 2), 1000, 3001):
            assert partials((1, 1, rows), width, 1) <= rows and partials((rows, 1, 1), width, 1) <= rows
            for n2 in (3, 32, 101, 127):
                assert partials((1, rows, n2), width, 1) <= rows * n2 and partials((1, rows, n2), width, n2) <= rows * n2 + 127


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,D", [(1, 127, 4096), (3, 101, 4001), (5, 127, 1025), (11, 101, 72), (2, 1, 4096), (77, 1, 4096), (127, 1, 2047), (100, 1, 640), (7, 125, 77)])
def test_layer_norm_of_few_rows(T, H, D, dtype):
    """Fewer rows than groups run at once, or hardly more, and numbers of heads that share no factor with a block's groups."""
    x, dy = (0.3 + rand(T, H, D)).to(dtype), rand(T, H, D, seed=2).to(dtype)
    for kind in ("heads", "vector"):
        layer_norm_check(x, *params(kind, H, D, dtype), dy)
    layer_norm_check(rand(T, 3, H, D, seed=5).to(dtype)[:, 1], *params("vector", H, D, dtype), dy)


@pytest.mark.gpu
def test_layer_norm_rows_that_kernels_get():
    """How rows are handed over: one run of rows as n0, through which kernels step, heads with weights of their own as n2."""
    class Rows(ctypes.Structure):
        _fields_ = [(k, ctypes.c_int64) for k in ("n0", "n1", "n2", "width", "heads")] + [(k, ctypes.c_int64 * 3) for k in ("x", "dy", "dx")]

    seen = []

    def forward(rows, *rest):
        r = rows.contents
        seen.append((r.n0, r.n1, r.n2, r.width, r.heads, *r.x))
        return 0

    vp, ci = ctypes.c_void_p, ctypes.c_int
    callback = ctypes.CFUNCTYPE(ci, ctypes.POINTER(Rows), ci, vp, ci, vp, vp, ctypes.c_float, vp, vp, vp)(forward)
    host, L = runtime.host(), runtime.lib()
    address = lambda f: ctypes.cast(f, vp).value
    entries = {n: address(getattr(L, n)) for n in runtime.SYMBOLS if n.startswith(("frnn_embedding", "frnn_layer_norm", "frnn_token", "frnn_last"))}
    bind = lambda **other: host.bind_lm({**entries, **other}, runtime._status_word, runtime._status_raise)
    x, w, h = rand(4, 30, 64), rand(64), rand(5, 64)
    bind(frnn_layer_norm_forward=address(callback))
    try:
        fr.layer_norm(x, w)
        fr.layer_norm(x[..., 32:])
        fr.layer_norm(h, w)
        fr.layer_norm(h, h)
        fr.layer_norm(x.view(4, 6, 5, 64), h)
        fr.layer_norm(x[:, 3:])
        fr.layer_norm(w, w)
    finally:
        bind()
    assert seen == [(120, 1, 1, 64, 1, 64, 0, 0), (120, 1, 1, 32, 1, 64, 0, 0), (5, 1, 1, 64, 1, 64, 0, 0), (1, 1, 5, 64, 5, 0, 0, 64), (1, 24, 5, 64, 5, 0, 320, 64),
                    (1, 4, 27, 64, 1, 0, 1920, 64), (1, 1, 1, 64, 1, 0, 0, 0)]


# ---- layer norm: no heads --------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("guard", ["0", "1"])
def test_layer_norm_of_no_heads(guard, monkeypatch):
    """x [B,T,0,D] with weights [0,D], forward and backward; FRNN_GUARD=1 looks for writes into buffers of no element."""
    monkeypatch.setenv("FRNN_GUARD", guard)
    x = torch.empty(2, 3, 0, 16, device="cuda", requires_grad=True)
    w, b = (torch.empty(0, 16, device="cuda", requires_grad=True) for _ in range(2))
    y = fr.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == gx.shape == x.shape and gw.shape == gb.shape == w.shape


# ---- forward-mode derivatives ------------------------------------------------------------------------------------------------

def on_meta(name):
    """(function of its leaf, the leaf, shapes of its differentiable results) without a GPU"""
    lm._operators()
    t, x = torch.zeros(3, dtype=torch.int64, device="meta"), torch.empty(3, 8, device="meta")
    return {"embedding": (lambda w: (fr.embedding(t, w),), torch.empty(5, 8, device="meta"), [(3, 8)]), "layer_norm": (lambda x: (fr.layer_norm(x),), x, [(3, 8)]),
            "token_logprobs": (lambda x: fr.token_logprobs(x, t)[:2], x, [(3,), (3,)])}[name]


@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_tangent_on_an_upstream_gradient(name):
    """Refused, not dropped; dual levels and functional transforms without one go through."""
    f, leaf, shapes = on_meta(name)
    for k in range(len(shapes)):
        with ad.dual_level():
            x = leaf.clone().requires_grad_()
            up = [torch.empty(s, device="meta") for s in shapes]
            assert torch.autograd.grad(f(x), x, up)[0].shape == leaf.shape
            up[k] = ad.make_dual(up[k], torch.empty_like(up[k]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(f(x), x, up)
    h = torch.empty(shapes[0], device="meta")
    gradient = lambda h: torch.func.grad(lambda x: (f(x)[0] * h).sum())(leaf)
    assert gradient(h).shape == leaf.shape
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(gradient, (h,), (torch.empty_like(h),))


# ---- torch.compile -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_first_use_is_a_compiled_one(name):
    """A process whose first use of an operator is traced whole gets as far as the operator itself, which refuses the CPU;
    on meta tensors the compiled call gives a result, and again without another compilation."""
    program = f"""
import torch, flex_rnn_b200 as fr
def make(device):
    t, w, x = torch.zeros(2, 3, dtype=torch.int64, device=device), torch.zeros(5, 8, device=device), torch.zeros(2, 3, 8, device=device)
    return dict(embedding=(t, w), layer_norm=(x,), token_logprobs=(x, t))["{name}"]
graphs = []
compiled = torch.compile(lambda *a: fr.{name}(*a), fullgraph=True, backend=lambda g, _: graphs.append(g) or g)
try:
    compiled(*make("cpu"))
except RuntimeError as e:
    print("refused" if "CUDA tensors" in str(e) else e)
graphs.clear()           # (the CPU call's)
for _ in range(2):
    r = compiled(*make("meta"))
print(tuple(r.shape) if torch.is_tensor(r) else tuple(r.logprob.shape), len(graphs))
"""
    r = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, cwd=ROOT, timeout=600)
    shape = {"embedding": (2, 3, 8), "layer_norm": (2, 3, 8), "token_logprobs": (2, 3)}[name]
    assert r.stdout.splitlines() == ["refused", f"{shape} 1"], r.stdout + r.stderr[-2000:]


def of_batch(name, b, device):
    """(function, its leaves, upstream gradients) for a batch of b"""
    t = (torch.arange(7 * b, device=device) * 5 % 11).view(b, 7)
    one = lambda *s: torch.linspace(-2, 3, math.prod(s), device=device).sin().view(s)
    leaf = lambda *s: one(*s).requires_grad_()
    return {"embedding": (lambda w: (fr.embedding(t, w),), [leaf(11, 24)], [one(b, 7, 24)]),
            "layer_norm": (lambda x, w: (fr.layer_norm(x, w),), [leaf(b, 7, 24), leaf(24)], [one(b, 7, 24)]),
            "sliced layer_norm": (lambda x: (fr.layer_norm(x[1:, :, 3:]),), [leaf(b, 7, 24)], [one(b - 1, 7, 21)]),
            "token_logprobs": (lambda x: fr.token_logprobs(x, t, top=2)[:2], [leaf(b, 7, 11)], [one(b, 7), one(b, 7)])}[name]


OF_BATCH = ["embedding", "layer_norm", "sliced layer_norm", "token_logprobs"]


@pytest.mark.parametrize("name", OF_BATCH)
def test_symbolic_sizes(name):
    """Traced with symbolic sizes, with gradients, whole and sliced layouts."""
    lm._operators()
    torch._dynamo.reset()
    compiled = torch.compile(lambda f, a: f(*a), fullgraph=True, backend="aot_eager", dynamic=True)
    for b in (6, 7, 9):
        f, leaves, up = of_batch(name, b, "meta")
        assert [g.shape for g in torch.autograd.grad(compiled(f, leaves), leaves, up)] == [v.shape for v in leaves]


@pytest.mark.gpu
@pytest.mark.parametrize("name", OF_BATCH)
def test_compiled_for_any_batch(name):
    torch._dynamo.reset()
    compiled = torch.compile(lambda f, a: f(*a), fullgraph=True, dynamic=True)
    for b in (6, 7, 9):
        f, leaves, up = of_batch(name, b, "cuda")
        assert all(torch.equal(a, g) for a, g in zip(both(lambda *a: compiled(f, a), leaves, up), both(f, leaves, up)))


# ---- shared memory beyond 48 KB ------------------------------------------------------------------------------------------------

ALLOW_SHARED = r"""
#include <cuda_runtime.h>

#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

static std::atomic<size_t> permitted{0};        // what the kernel's attribute says
static cudaError_t set_attribute(size_t bytes, bool slow) {
    permitted = bytes;
    if (slow) std::this_thread::sleep_for(std::chrono::milliseconds(400));
    return cudaSuccess;
}
#define cudaGetDevice(d) (*(d) = 0, cudaSuccess)
#define cudaFuncSetAttribute(kernel, which, bytes) set_attribute(bytes, (bytes) > 100000)
#include "frnn_lm.cuh"

__global__ void kernel() {}
int frnn_fail(int code, const char*, ...) { return code; }

int main() {
    std::thread large([] { frnn_lm::allow_shared<kernel>(200000); });
    std::this_thread::sleep_for(std::chrono::milliseconds(100));
    std::thread small([] { frnn_lm::allow_shared<kernel>(90000); });
    large.join();
    small.join();
    const bool ok = frnn_lm::allow_shared<kernel>(200000);
    printf("%d %d\n", ok, permitted >= 200000);
}
"""


def test_shared_memory_of_two_threads(tmp_path):
    """A kernel is launched with sizes that differ: a thread that asks for less while another asks for more leaves the kernel
    with what the record says.  The runtime's two calls are stand-ins, so no device is needed."""
    source, program = tmp_path / "allow.cu", tmp_path / "allow"
    source.write_text(ALLOW_SHARED)
    subprocess.run([build.nvcc_path(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "flex_rnn_b200", "csrc"), "-o", str(program), str(source)], check=True)
    assert subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout.split() == ["1", "1"]


# ---- all of them --------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_threads(name):
    """Calls from several threads, each on a stream of its own, give what one thread gives."""
    import threading
    f, leaves, up = calls()[name]
    want = both(f, leaves, up)
    torch.cuda.synchronize()
    wrong = []

    def work():
        try:
            mine, side = [v.detach().clone().requires_grad_() for v in leaves], torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(20):
                    got = both(f, mine, up)
                    side.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        wrong.append("other results")
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_repeated_alternatives_give_the_same_bits():
    """Candidates are listed in whatever order threads come; their ranks, and joins of a cluster, do not show it."""
    for n, V in [(2, 200001), (400, 32003), (1300, 1000)]:
        x, t = logits_of(n, V, torch.bfloat16)
        want = fr.token_logprobs(x, t, top=32)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(fr.token_logprobs(x, t, top=32), want))
