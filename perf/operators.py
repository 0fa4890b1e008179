"""The operators around a recurrent language model's scans, as performance cases: ``embedding`` (tokens to vectors, with
scaling; its gradient sums by token), ``layer_norm`` (over a model's width, or per head as on a scan's output) and
``token_logprobs`` (log probabilities of given tokens, entropy, top alternatives).

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges, ``prepare`` makes a case's tensors from
a seed, ``run`` does one pass: with ``own`` through this package's entry points, without it in elementary torch operations
in 32 bits.  ``exact`` restates the definitions in 64 bits.  A "train" case is a forward and its gradients.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100           # the token of padded places


def _embedding(name, mode, n, V, D, io, pad):
    c = {"op": "embedding", "mode": mode, "n": n, "V": V, "D": D, "io": io, "pad": pad}
    return {"name": name, **c} if name else c


def _layer_norm(name, mode, B, T, H, D, io, affine, params, layout):
    c = {"op": "layer_norm", "mode": mode, "B": B, "T": T, "H": H, "D": D, "io": io, "affine": affine, "params": params, "layout": layout}
    return {"name": name, **c} if name else c


def _logprobs(name, mode, n, V, io, top, mask, temperature):
    c = {"op": "token_logprobs", "mode": mode, "n": n, "V": V, "io": io, "top": top, "mask": mask, "temperature": temperature}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token of generation for a batch of 16 sequences, a model of 32 heads of 128
        _embedding("embed_decode", "infer", 16, 65536, 4096, "bf16", 0.0),
        # the gradient check of a small model: 8 sequences of 256 tokens, byte-sized vocabulary
        _embedding("embed_check_fp32", "train", 2048, 256, 256, "fp32", 0.0),
        # fine-tuning on three padded sequences, sizes that are no multiple of anything
        _embedding("embed_tune_ragged", "train", 3 * 777, 32003, 5 * 97, "fp16", 0.1),
        # the benchmark's batch: 8 sequences of 1024 tokens
        _embedding("embed_train", "train", 8 * 1024, 65536, 4096, "bf16", 0.02),
        # generation: the norm before a projection, a row for each sequence
        _layer_norm("norm_decode", "infer", 16, 1, 1, 4096, "bf16", "vector", "fp32", "plain"),
        # each head of a scan's output in training, weights for each head
        _layer_norm("norm_heads_train", "train", 8, 1024, 32, 128, "bf16", "heads", "bf16", "plain"),
        # an odd width in fp32, sliced out of one fused projection
        _layer_norm("norm_ragged_fp32", "train", 3, 777, 1, 1001, "fp32", "vector", "fp32", "sliced"),
        # the norm before a projection in training, the benchmark's batch
        _layer_norm("norm_train", "train", 8, 1024, 1, 4096, "bf16", "vector", "fp32", "plain"),
        # generation with a grammar that forbids most tokens: the chosen tokens and 20 alternatives
        _logprobs("score_decode", "infer", 16, 65536, "bf16", 20, "grammar", 0.8),
        # scoring one prompt of 2000 tokens, 5 alternatives, logits in fp32
        _logprobs("score_prompt_fp32", "infer", 2000, 50003, "fp32", 5, "none", 1.0),
        # a policy gradient with entropy on padded sequences, an odd vocabulary, rows that a mask leaves empty
        _logprobs("loss_ragged_fp16", "train", 777, 32003, "fp16", 0, "rows", 1.0),
        # the loss of the benchmark's batch
        _logprobs("loss_train", "train", 8 * 1024, 65536, "bf16", 0, "none", 1.0),
    ]


def _elements(c):
    """Values that a pass reads or writes, roughly."""
    if c["op"] == "embedding":
        return 2 * c["n"] * c["D"] + (c["n"] * c["D"] + c["V"] * c["D"] if c["mode"] == "train" else 0)
    if c["op"] == "layer_norm":
        return c["B"] * c["T"] * c["H"] * c["D"] * (4 if c["mode"] == "train" else 2)
    return c["n"] * c["V"] * (2 if c["mode"] == "train" else 1)


LARGEST = {op: max(_elements(c) * BYTES[c["io"]] for c in listed() if c["op"] == op) for op in ("embedding", "layer_norm", "token_logprobs")}


def _log(rng, lo, hi):
    n = min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))
    return n - 1 if n == 3072 else n


def draw(rng):
    """Batches from one token to 32768, vocabularies of 100 to 200000 tokens, widths of 16 to 8192 (one to 64 heads)."""
    op = rng.choice(["embedding", "layer_norm", "token_logprobs"])
    mode = rng.choice(["infer", "train", "train"])
    io = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    even = lambda n, m: -(-n // m) * m          # most sizes in use are multiples of something
    if op == "embedding":
        D = _log(rng, 16, 8192)
        c = _embedding(None, mode, _log(rng, 1, 32768), _log(rng, 100, 200000), even(D, 64) if rng.random() < 0.6 else D, io, rng.choice([0.0, 0.0, 0.05, 0.5]))
        small = ("n", "V")
    elif op == "layer_norm":
        heads = rng.random() < 0.5
        H = _log(rng, 1, 64) if heads else 1
        D = _log(rng, 16, 256 if heads else 8192)
        affine = rng.choice(["heads", "vector", "none"] if heads else ["vector"])
        c = _layer_norm(None, mode, _log(rng, 1, 16), _log(rng, 1, 2048), H, even(D, 64 if D > 64 else 16) if rng.random() < 0.6 else D, io, affine,
                        rng.choice([io, "fp32"]), rng.choice(["plain", "plain", "sliced", "transposed"]))
        small = ("B", "T")
    else:
        V = _log(rng, 100, 200000)
        top = rng.choice([0, 1, 5, 20, 32]) if mode == "infer" else rng.choice([0, 0, 0, 8])
        c = _logprobs(None, mode, _log(rng, 1, 8192), even(V, 64) if rng.random() < 0.5 else V, io, top, rng.choice(["none", "none", "grammar", "rows"]), rng.choice([1.0, 1.0, 0.7]))
        small = ("n",)
    for k in small:
        while c[k] > 1 and _elements(c) * BYTES[io] > LARGEST[op]:
            c[k] //= 2
    if 3072 in c.values():
        return draw(rng)
    return c


def _tokens(n, V, pad, g):
    """Tokens with the frequencies of text (the v-th most frequent about 1 / v), and padded places."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    t = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
    return torch.where(torch.rand(n, generator=g, device="cuda") < pad, IGNORE, t) if pad else t


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    io, train = DTYPES[c["io"]], c["mode"] == "train"
    if c["op"] == "embedding":
        n, V, D = c["n"], c["V"], c["D"]
        return {"c": c, "tokens": _tokens(n, V, c["pad"], g), "weight": (0.02 * rand(V, D)).to(io).requires_grad_(train), "scale": D ** 0.5,
                "dy": rand(n, D).to(io) if train else None}
    if c["op"] == "layer_norm":
        B, T, H, D = (c[k] for k in "BTHD")
        heads = H > 1 or c["affine"] == "heads"
        shape = (B, T, H, D) if heads else (B, T, D)
        if c["layout"] == "sliced":                # a third of one fused projection's output
            x = rand(B, T, 3, *shape[2:]).add_(0.3).to(io)[:, :, 1]
        elif c["layout"] == "transposed":          # what a head-major layer gives
            x = rand(B, H, T, D).add_(0.3).to(io).transpose(1, 2)
            x = x if heads else x[:, :, 0]
        else:
            x = rand(*shape).add_(0.3).to(io)
        pshape = {"heads": (H, D), "vector": (D,), "none": None}[c["affine"]]
        pt = DTYPES[c["params"]]
        w = (1 + 0.1 * rand(*pshape)).to(pt).requires_grad_(train) if pshape else None
        b = (0.1 * rand(*pshape)).to(pt).requires_grad_(train) if pshape else None
        return {"c": c, "x": x.requires_grad_(train), "weight": w, "bias": b, "eps": 1e-5, "dy": rand(*shape).to(io) if train else None}
    n, V = c["n"], c["V"]
    logits, t = 2.0 * rand(n, V), _tokens(n, V, 0.0, g)
    logits.scatter_add_(1, t[:, None], 6 * torch.rand(n, 1, generator=g, device="cuda"))       # text is mostly what the model expects
    if c["mask"] == "grammar":                     # nine tokens in ten may not follow here
        drop = torch.rand(n, V, generator=g, device="cuda") < 0.9
        logits.masked_fill_(drop.scatter_(1, t[:, None], False), -math.inf)
        del drop
    if c["mask"] == "rows":                        # places that nothing may follow, and padding
        logits.masked_fill_((torch.rand(n, 1, generator=g, device="cuda") < 0.05), -math.inf)
        t = torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, IGNORE, t)
    return {"c": c, "logits": logits.to(io).requires_grad_(train), "tokens": t, "up": (rand(n), 0.1 * rand(n)) if train else None}


# ---- the framework's operators, as a user's program calls them ---------------------------------------------------------

def _run_own(s):
    import flex_rnn_b200 as fr
    c = s["c"]
    train = c["mode"] == "train"
    with torch.set_grad_enabled(train):
        if c["op"] == "embedding":
            y = fr.embedding(s["tokens"], s["weight"], scale=s["scale"], ignore_index=IGNORE)
            return {"y": y.detach(), "dweight": torch.autograd.grad(y, s["weight"], s["dy"])[0]} if train else {"y": y}
        if c["op"] == "layer_norm":
            y = fr.layer_norm(s["x"], s["weight"], s["bias"], eps=s["eps"])
            leaves = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
            return {"y": y.detach(), "grads": list(torch.autograd.grad(y, leaves, s["dy"]))} if train else {"y": y}
        r = fr.token_logprobs(s["logits"], s["tokens"], top=c["top"], temperature=c["temperature"], ignore_index=IGNORE)
        out = {"logprob": r.logprob.detach(), "entropy": r.entropy.detach()}
        if c["top"]:
            out.update(top_logprob=r.top_logprob, top_token=r.top_token)
        if train:
            out["dlogits"] = torch.autograd.grad((r.logprob, r.entropy), s["logits"], s["up"])[0]
        return out


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _plain_embedding(s):
    t, w = s["tokens"], s["weight"]
    there = t != IGNORE
    at = torch.where(there, t, 0)
    y = (w[at].float() * s["scale"] * there[:, None]).to(w.dtype)
    if s["dy"] is None:
        return {"y": y}
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, at, s["dy"].float() * there[:, None])
    return {"y": y, "dweight": (dw * s["scale"]).to(w.dtype)}


def _plain_layer_norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    xf = x.float()
    centred = xf - xf.mean(-1, True)
    rstd = (centred.square().mean(-1, True) + s["eps"]).rsqrt()
    xh = centred * rstd
    y = (xh if w is None else xh * w.float() + b.float()).to(x.dtype)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    gw = dy if w is None else dy * w.float()
    dx = ((gw - gw.mean(-1, True) - xh * (gw * xh).mean(-1, True)) * rstd).to(x.dtype)
    if w is None:
        return {"y": y, "grads": [dx]}
    over = tuple(range(x.dim() - w.dim()))
    return {"y": y, "grads": [dx, (dy * xh).sum(over).to(w.dtype), dy.sum(over).to(b.dtype)]}


def _plain_logprobs(s):
    c, x, t = s["c"], s["logits"], s["tokens"]
    z = x.float() / c["temperature"]
    m = z.amax(-1, True)
    empty = m == -math.inf
    z = z - torch.where(empty, 0.0, m)
    e = torch.exp(z)
    total = e.sum(-1, True)
    logp = z - torch.where(empty, 0.0, torch.log(total))
    del z
    p = e / torch.where(empty, 1.0, total)
    del e
    plogp = torch.where(p == 0, 0.0, p * logp)
    entropy = -plogp.sum(-1, True)
    there = (t != IGNORE)[:, None]
    at = torch.where(there, t[:, None], 0)
    out = {"logprob": torch.where(there, logp.gather(1, at), 0.0)[:, 0], "entropy": entropy[:, 0]}
    if c["top"]:
        # equal values in the order of their tokens: one whole number holds a value's rank and its token
        bits = (x.float() + 0.0).view(torch.int32).long()
        rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        top = ((rank << 32) - torch.arange(x.shape[1], device=x.device)).topk(min(c["top"], x.shape[1]), -1, sorted=True).values
        out["top_token"] = -top & 0xFFFFFFFF
        out["top_logprob"] = logp.gather(1, out["top_token"])
    if s["up"] is not None:
        glp, gh = torch.where(there, s["up"][0][:, None], 0.0), s["up"][1][:, None]
        d = -p * glp - gh * (plogp + p * entropy)
        d.scatter_add_(1, at, glp)
        out["dlogits"] = torch.where(empty, 0.0, d / c["temperature"]).to(x.dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "layer_norm": _plain_layer_norm, "token_logprobs": _plain_logprobs}[state["c"]["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _exact_embedding(s):
    t, w, scale = s["tokens"], s["weight"].double(), s["scale"]
    y = torch.zeros(len(t), w.shape[1], dtype=torch.float64, device=w.device)
    there = (t >= 0).nonzero()[:, 0]
    y[there] = w[t[there]] * scale
    if s["dy"] is None:
        return {"y": y}
    order = there[torch.argsort(t[there], stable=True)]
    sums = torch.cat([torch.zeros_like(y[:1]), s["dy"].double()[order].cumsum(0)])      # differences of running sums over the sorted tokens
    ends = torch.searchsorted(t[order].contiguous(), torch.arange(w.shape[0], device=w.device), right=True)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends[:-1]])
    dw = torch.zeros_like(w)
    some = (ends > starts).nonzero()[:, 0]
    dw[some] = scale * (sums[ends[some]] - sums[starts[some]])
    return {"y": y, "dweight": dw}


def _exact_layer_norm(s):
    x, D = s["x"].double(), s["x"].shape[-1]
    w = None if s["weight"] is None else s["weight"].double()
    mean = x.sum(-1, True) / D
    sd = ((x * x).sum(-1, True) / D - mean * mean + s["eps"]).sqrt()
    n = (x - mean) / sd
    y = n if w is None else n * w + s["bias"].double()
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].double()
    g = dy if w is None else dy * w
    dx = (D * g - g.sum(-1, True) - n * (g * n).sum(-1, True)) / (D * sd)
    if w is None:
        return {"y": y, "grads": [dx]}
    flat = lambda v: v.reshape(-1, *w.shape)
    return {"y": y, "grads": [dx, torch.einsum("n...,n...->...", flat(dy), flat(n)), flat(dy).sum(0)]}


def _exact_logprobs(s):
    c, T, out = s["c"], s["c"]["temperature"], []
    n, V = s["logits"].shape
    rows = max(1, 2 ** 25 // V)
    for lo in range(0, n, rows):
        x, t = s["logits"][lo:lo + rows].double(), s["tokens"][lo:lo + rows]
        z = x / T
        lse = torch.logsumexp(z, -1)
        some = torch.isfinite(lse)
        p = torch.softmax(z, -1)
        p[~some] = 0
        h = torch.where(some, lse, 0.0) - (p * z.clamp_min(-1e30)).sum(-1)
        place = torch.arange(len(t), device=t.device)
        lp = torch.where(some, z[place, t.clamp_min(0)] - lse, -math.inf)
        one = {"logprob": torch.where(t >= 0, lp, 0.0), "entropy": torch.where(some, h, 0.0)}
        if c["top"]:
            best = torch.sort(x, dim=-1, descending=True, stable=True)
            k = min(c["top"], V)
            one["top_token"] = best.indices[:, :k]
            one["top_logprob"] = torch.where(some[:, None], best.values[:, :k] / T - lse[:, None], -math.inf)
        if s["up"] is not None:
            glp = torch.where((t >= 0) & some, s["up"][0][lo:lo + rows].double(), 0.0)
            gh = s["up"][1][lo:lo + rows].double()
            d = -p * glp[:, None] - p * gh[:, None] * ((z - lse[:, None]).clamp_min(-1e30) + h[:, None])
            d[~some] = 0
            d[place, t.clamp_min(0)] += glp
            one["dlogits"] = d / T
        out.append(one)
    return {k: torch.cat([o[k] for o in out]) for k in out[0]}


def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"embedding": _exact_embedding, "layer_norm": _exact_layer_norm, "token_logprobs": _exact_logprobs}[c["op"]](s)


def work(c):
    """Inputs read once, outputs written once: of a table the rows that the tokens name (their expected number), whose
    gradient is written whole.  Operations: multiplications, additions, exponentials."""
    e, train = BYTES[c["io"]], c["mode"] == "train"
    if c["op"] == "embedding":
        n, V, D = c["n"], c["V"], c["D"]
        v = torch.arange(V, dtype=torch.float64)
        share = torch.log1p(1 / (v + 1)) / math.log(V + 1)
        rows = float((1 - (1 - share) ** (n * (1 - c["pad"]))).sum())
        return {"bytes": 8 * n + e * D * (rows + n + (n + V if train else 0)), "flops": n * D * (2 if train else 1) + (V * D if train else 0)}
    if c["op"] == "layer_norm":
        B, T, H, D = (c[k] for k in "BTHD")
        pars = {"heads": 2 * H * D, "vector": 2 * D, "none": 0}[c["affine"]] * BYTES[c["params"]]
        return {"bytes": (2 if train else 1) * (2 * B * T * H * D * e + pars), "flops": B * T * H * D * (20 if train else 7)}
    n, V = c["n"], c["V"]
    return {"bytes": n * V * e * (2 if train else 1) + n * (16 + 12 * c["top"] + (8 if train else 0)), "flops": n * V * (10 if train else 5)}
