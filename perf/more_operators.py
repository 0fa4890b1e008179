"""The matrix products around a recurrent language model's scans, as performance cases: ``gated_mlp`` (the gated feed-forward
block between scans), ``linear_logprobs`` (log probabilities of given tokens and entropy from hidden vectors, without logits)
and ``rotary`` (positions on the queries and keys of scans such as retention).

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges, ``prepare`` makes a case's tensors from
a seed, ``run`` does one pass: with ``own`` through this package's entry points, without it in elementary torch operations
in 32 bits (angles in 64).  ``exact`` restates the definitions in 64 bits.  A "train" case is a forward and its gradients.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100           # the token of padded places


def _mlp(name, mode, n, D, F, io, activation):
    c = {"op": "gated_mlp", "mode": mode, "n": n, "D": D, "F": F, "io": io, "activation": activation}
    return {"name": name, **c} if name else c


def _logprobs(name, mode, n, V, D, io, pad, temperature):
    c = {"op": "linear_logprobs", "mode": mode, "n": n, "V": V, "D": D, "io": io, "pad": pad, "temperature": temperature}
    return {"name": name, **c} if name else c


def _rotary(name, mode, B, T, H, N, pairs, io, interleaved, layout, start, factor):
    c = {"op": "rotary", "mode": mode, "B": B, "T": T, "H": H, "N": N, "pairs": pairs, "io": io, "interleaved": interleaved, "layout": layout, "start": start, "factor": factor}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token of generation for a batch of 16 sequences, a model of 32 heads of 128: all weights are read once
        _mlp("mlp_decode", "infer", 16, 4096, 12288, "bf16", "silu"),
        # the gradient check of a small model: 8 sequences of 256 tokens
        _mlp("mlp_check_fp32", "train", 2048, 256, 1024, "fp32", "gelu"),
        # fine-tuning on three sequences, sizes that are no multiple of anything
        _mlp("mlp_tune_ragged", "train", 3 * 777, 5 * 97, 1291, "fp16", "silu"),
        # the benchmark's batch: 8 sequences of 1024 tokens
        _mlp("mlp_train", "train", 8 * 1024, 4096, 12288, "bf16", "silu"),
        # how probable a proposed token is for each of 16 sequences
        _logprobs("score_decode", "infer", 16, 65536, 4096, "bf16", 0.0, 0.8),
        # scoring one prompt of 2000 tokens in fp32, an odd vocabulary
        _logprobs("score_prompt_fp32", "infer", 2000, 50003, 1024, "fp32", 0.0, 1.0),
        # a policy gradient with entropy on padded sequences, nothing a multiple of anything
        _logprobs("loss_ragged_fp16", "train", 777, 32003, 5 * 97, "fp16", 0.1, 1.0),
        # the loss of the benchmark's batch
        _logprobs("loss_train", "train", 8 * 1024, 65536, 4096, "bf16", 0.02, 1.0),
        # the next token of 16 sequences that are far along: queries and keys of 32 heads each, one slice of a fused projection
        _rotary("rotary_decode", "infer", 16, 1, 64, 128, 64, "bf16", False, "sliced", 1000000, 1.0),
        # odd lengths, part of the head, neighbours as pairs, head-major rows in fp32
        _rotary("rotary_ragged_fp32", "train", 3, 777, 5, 97, 31, "fp32", True, "transposed", 0, 1.0),
        # the benchmark's batch, queries and keys
        _rotary("rotary_train", "train", 8, 1024, 64, 128, 64, "bf16", False, "plain", 0, 1.0),
        # reading a document of 65536 tokens with stretched positions, half of each head turned
        _rotary("rotary_long_fp16", "infer", 1, 65536, 32, 128, 32, "fp16", True, "plain", 0, 8.0),
    ]


def _cost(c):
    """Operations of a matrix product (those in fp32 take six times as long as others), values of a rotation."""
    train = c["mode"] == "train"
    if c["op"] == "rotary":
        return c["B"] * c["T"] * c["H"] * c["N"] * BYTES[c["io"]] * (2 if train else 1)
    products = 6 * c["D"] * c["F"] if c["op"] == "gated_mlp" else 2 * c["D"] * c["V"]
    return c["n"] * products * (3 if train else 1) * (6 if c["io"] == "fp32" else 1)


LARGEST = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("gated_mlp", "linear_logprobs", "rotary")}


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    """Batches from one token to 65536, widths of 16 to 8192, feed-forward widths to 16384, vocabularies of 100 to 150000
    tokens, heads of 2 to 256 values, positions beyond a million."""
    op = rng.choice(["gated_mlp", "linear_logprobs", "rotary"])
    mode = rng.choice(["infer", "train", "train"])
    io = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = lambda lo, hi, m: min(hi, -(-_log(rng, lo, hi) // m) * m) if rng.random() < 0.6 else _log(rng, lo, hi)      # most sizes in use are multiples of something
    if op == "gated_mlp":
        c = _mlp(None, mode, _log(rng, 1, 16384), size(16, 8192, 64), size(16, 16384, 64), io, rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]))
        small = ("n", "F", "D")
    elif op == "linear_logprobs":
        c = _logprobs(None, mode, _log(rng, 1, 16384), size(100, 150000, 64), size(16, 8192, 64), io, rng.choice([0.0, 0.0, 0.1, 0.5]), rng.choice([1.0, 1.0, 0.7]))
        small = ("n", "V", "D")
    else:
        N = size(2, 256, 16)
        pairs = N // 2 if rng.random() < 0.6 else rng.randint(1, N // 2)
        c = _rotary(None, mode, _log(rng, 1, 16), _log(rng, 1, 65536), _log(rng, 1, 64), N, pairs, io, rng.random() < 0.5, rng.choice(["plain", "plain", "sliced", "transposed"]),
                    rng.choice([0, 0, _log(rng, 1, 2000000)]), rng.choice([1.0, 1.0, 4.0, 32.0]))
        small = ("T", "B", "H")
    for k in small:
        while c[k] > 16 and _cost(c) > LARGEST[op]:
            c[k] //= 2
    return c


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    io, train = DTYPES[c["io"]], c["mode"] == "train"
    leaf = lambda t: t.to(io).requires_grad_(train)
    if c["op"] == "gated_mlp":
        n, D, F = c["n"], c["D"], c["F"]
        return {"c": c, "x": leaf(rand(n, D)), "gate": leaf(rand(F, D).mul_(D ** -0.5)), "up": leaf(rand(F, D).mul_(D ** -0.5)), "down": leaf(rand(D, F).mul_(F ** -0.5)),
                "dy": rand(n, D).to(io) if train else None}
    if c["op"] == "linear_logprobs":
        n, V, D = c["n"], c["V"], c["D"]
        # tokens with the frequencies of text (the v-th most frequent about 1 / v); text is mostly what the model expects
        t = (torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
        w = rand(V, D).mul_(2 * D ** -0.5)
        x = rand(n, D).add_(6 * torch.rand(n, 1, generator=g, device="cuda") / 4 * w[t])
        if c["pad"]:
            t = torch.where(torch.rand(n, generator=g, device="cuda") < c["pad"], IGNORE, t)
        return {"c": c, "x": leaf(x), "weight": leaf(w), "tokens": t, "up": (rand(n), 0.1 * rand(n)) if train else None}
    B, T, H, N = (c[k] for k in "BTHN")
    if c["layout"] == "sliced":                    # queries and keys, without the values behind them
        x = rand(B, T, H + -(-H // 2), N).to(io)[:, :, :H]
    elif c["layout"] == "transposed":              # what a head-major layer gives
        x = rand(B, H, T, N).to(io).transpose(1, 2)
    else:
        x = rand(B, T, H, N).to(io)
    # each sequence is somewhat further along than the one before it; positions stretched by a factor
    positions = c["start"] + 37 * torch.arange(B, device="cuda")[:, None] + torch.arange(T, device="cuda")
    frequencies = 10000.0 ** -(torch.arange(c["pairs"], device="cuda", dtype=torch.float64) / c["pairs"]) / c["factor"]
    return {"c": c, "x": x.requires_grad_(train), "positions": positions, "frequencies": frequencies, "scale": 1.0 if c["factor"] == 1 else 0.1 * math.log(c["factor"]) + 1,
            "dy": rand(B, T, H, N).to(io) if train else None}


# ---- the framework's operators, as a user's program calls them ---------------------------------------------------------

def _run_own(s):
    import flex_rnn_b200 as fr
    c = s["c"]
    train = c["mode"] == "train"
    with torch.set_grad_enabled(train):
        if c["op"] == "gated_mlp":
            y = fr.gated_mlp(s["x"], s["gate"], s["up"], s["down"], activation=c["activation"])
            return {"y": y.detach(), "grads": list(torch.autograd.grad(y, [s["x"], s["gate"], s["up"], s["down"]], s["dy"]))} if train else {"y": y}
        if c["op"] == "linear_logprobs":
            r = fr.linear_logprobs(s["x"], s["weight"], s["tokens"], temperature=c["temperature"], ignore_index=IGNORE)
            out = {"logprob": r.logprob.detach(), "entropy": r.entropy.detach()}
            if train:
                out["grads"] = list(torch.autograd.grad((r.logprob, r.entropy), [s["x"], s["weight"]], s["up"]))
            return out
        y = fr.rotary(s["x"], s["positions"], s["frequencies"], interleaved=c["interleaved"], scale=s["scale"])
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]} if train else {"y": y}


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _plain_activation(a, kind):
    """act(a) and its derivative"""
    if kind == "relu":
        return torch.where(a > 0, a, 0.0), (a > 0).float()
    if kind == "gelu":
        phi = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-a))
    return (s, s * (1 - s)) if kind == "sigmoid" else (a * s, s * (1 + a * (1 - s)))


def _plain_mlp(s):
    io, x, gate, up, down = s["x"].dtype, *(s[k].float() for k in ("x", "gate", "up", "down"))
    a, b = x @ gate.T, x @ up.T
    act, slope = _plain_activation(a, s["c"]["activation"])
    h = act * b
    y = (h @ down.T).to(io)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    dh = dy @ down
    da, db = dh * b * slope, dh * act
    return {"y": y, "grads": [t.to(io) for t in (da @ gate + db @ up, da.T @ x, db.T @ x, dy.T @ h)]}


def _plain_logprobs(s):
    c, io, x, w, t = s["c"], s["x"].dtype, s["x"].float(), s["weight"].float(), s["tokens"]
    z = (x @ w.T).div_(c["temperature"])
    z -= z.amax(-1, True)
    e = torch.exp(z)
    total = e.sum(-1, True)
    logp = z.sub_(torch.log(total))
    p = e.div_(total)
    entropy = -(p * logp).sum(-1, True)
    there = (t != IGNORE)[:, None]
    at = torch.where(there, t[:, None], 0)
    out = {"logprob": torch.where(there, logp.gather(1, at), 0.0)[:, 0], "entropy": entropy[:, 0]}
    if s["up"] is not None:
        glp, gh = torch.where(there, s["up"][0][:, None], 0.0), s["up"][1][:, None]
        d = logp.add_(entropy).mul_(gh).add_(glp).mul_(p).neg_()
        d.scatter_add_(1, at, glp)
        d /= c["temperature"]
        out["grads"] = [(d @ w).to(io), (d.T @ x).to(io)]
    return out


def _plain_rotary(s):
    c, x, P = s["c"], s["x"], s["c"]["pairs"]
    angle = (s["positions"].double()[..., None] * s["frequencies"])[:, :, None]
    cos, sin = (torch.cos(angle) * s["scale"]).float(), (torch.sin(angle) * s["scale"]).float()

    def turn(v, sin):
        f = v.float()
        out = f.clone()
        u, w = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if c["interleaved"] else (slice(0, P), slice(P, 2 * P))
        out[..., u] = f[..., u] * cos - f[..., w] * sin
        out[..., w] = f[..., u] * sin + f[..., w] * cos
        return out.to(v.dtype)

    return {"y": turn(x, sin)} if s["dy"] is None else {"y": turn(x, sin), "dx": turn(s["dy"], -sin)}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"gated_mlp": _plain_mlp, "linear_logprobs": _plain_logprobs, "rotary": _plain_rotary}[state["c"]["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _exact_mlp(s):
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}[s["c"]["activation"]]
    leaves = [s[k].detach().double().requires_grad_(s["dy"] is not None) for k in ("x", "gate", "up", "down")]
    x, gate, up, down = leaves
    linear = torch.nn.functional.linear
    with torch.set_grad_enabled(s["dy"] is not None):
        y = linear(act(linear(x, gate)) * linear(x, up), down)
    if s["dy"] is None:
        return {"y": y}
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, leaves, s["dy"].double()))}


def _exact_logprobs(s):
    T, x, w, tokens = s["c"]["temperature"], s["x"].detach().double(), s["weight"].detach().double(), s["tokens"]
    out, dw = [], torch.zeros_like(w) if s["up"] is not None else None
    rows = max(1, 2 ** 27 // w.shape[0])
    for lo in range(0, x.shape[0], rows):
        t = tokens[lo:lo + rows]
        z = torch.mm(x[lo:lo + rows], w.t()) / T
        logp = torch.log_softmax(z, -1)
        p = torch.softmax(z, -1)
        del z
        h = torch.special.entr(p).sum(-1)
        place = torch.arange(len(t), device=t.device)
        there = t >= 0
        one = {"logprob": torch.where(there, logp[place, t.clamp_min(0)], 0.0), "entropy": h}
        if dw is not None:
            glp = torch.where(there, s["up"][0][lo:lo + rows].double(), 0.0)
            gh = s["up"][1][lo:lo + rows].double()
            d = -p * (glp[:, None] + gh[:, None] * (logp + h[:, None]))
            d[place, t.clamp_min(0)] += glp
            d /= T
            one["dx"] = torch.mm(d, w)
            dw.addmm_(d.t(), x[lo:lo + rows])
        out.append(one)
    r = {k: torch.cat([o[k] for o in out]) for k in out[0]}
    if dw is not None:
        r["grads"] = [r.pop("dx"), dw]
    return r


def _exact_rotary(s):
    c, P = s["c"], s["c"]["pairs"]
    turn = torch.polar(torch.full_like(s["frequencies"], s["scale"]), torch.zeros_like(s["frequencies"])) * torch.exp(1j * s["positions"].double()[:, :, None, None] * s["frequencies"])

    def by(v, z):
        v = v.detach().double()
        head = v[..., :2 * P]
        pairs = head.unflatten(-1, (P, 2)) if c["interleaved"] else head.unflatten(-1, (2, P)).transpose(-1, -2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        head = pairs.flatten(-2) if c["interleaved"] else pairs.transpose(-1, -2).flatten(-2)
        return torch.cat([head, v[..., 2 * P:]], -1)

    return {"y": by(s["x"], turn)} if s["dy"] is None else {"y": by(s["x"], turn), "dx": by(s["dy"], turn.conj())}


def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"gated_mlp": _exact_mlp, "linear_logprobs": _exact_logprobs, "rotary": _exact_rotary}[c["op"]](s)


def work(c):
    """Inputs read once, outputs written once; multiplications and additions of the products (and what is done for each of
    their results), without a second computation of logits."""
    e, train = BYTES[c["io"]], c["mode"] == "train"
    if c["op"] == "gated_mlp":
        n, D, F = c["n"], c["D"], c["F"]
        return {"bytes": e * (2 * n * D + 3 * D * F) * (2 if train else 1), "flops": 6 * n * D * F * (3 if train else 1)}
    if c["op"] == "linear_logprobs":
        n, V, D = c["n"], c["V"], c["D"]
        return {"bytes": e * (n * D + V * D) * (2 if train else 1) + n * (24 if train else 16), "flops": n * V * (2 * D * (3 if train else 1) + (10 if train else 5))}
    x = c["B"] * c["T"] * c["H"] * c["N"]
    return {"bytes": 2 * x * e * (2 if train else 1) + 8 * c["B"] * c["T"], "flops": 3 * x * (2 if train else 1)}
