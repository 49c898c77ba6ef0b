"""Cases for the feed-forward operators: gated products, products with bias,
activation and residual, and the global gradient norm with clipping.

``run`` computes one pass, in elementary torch operations (``own`` false) or
through the package's entry points (``own`` true), on what ``prepare`` made.
Rows of a bank are sorted by expert; expert e holds rows offsets[e] ..
offsets[e+1]-1, and rows that no expert holds are padding.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # -- gated products: act(x Wg^T) * (x Wu^T)
        # one new token: both projections are read once, latency
        dict(name="gated_one_token", op="gated", tokens=1, top_k=1, experts=0, n=14336, k=4096,
             act="silu", dtype="bf16", skew=0.0, dropped=0, train=False),
        # a decode batch
        dict(name="gated_batch", op="gated", tokens=96, top_k=1, experts=0, n=14336, k=4096,
             act="gelu_tanh", dtype="fp16", skew=0.0, dropped=0, train=False),
        # a decode batch through the experts of a layer, a few rows for each
        dict(name="gated_experts_batch", op="gated", tokens=61, top_k=2, experts=8, n=14336,
             k=4096, act="silu", dtype="bf16", skew=0.5, dropped=0, train=False),
        # a chunk of prompts over many small experts, odd sizes, padding rows at the end
        dict(name="gated_experts_chunk", op="gated", tokens=509, top_k=4, experts=32, n=1031,
             k=1032, act="gelu", dtype="fp16", skew=0.7, dropped=5, train=False),
        # a long prompt
        dict(name="gated_prompt", op="gated", tokens=8192, top_k=1, experts=0, n=14336, k=4096,
             act="silu", dtype="bf16", skew=0.0, dropped=0, train=False),
        # a training step of a large layer
        dict(name="gated_train", op="gated", tokens=4095, top_k=1, experts=0, n=14336, k=4096,
             act="silu", dtype="bf16", skew=0.0, dropped=0, train=True),
        # a training step of many fine experts
        dict(name="gated_experts_train", op="gated", tokens=2047, top_k=4, experts=64, n=1024,
             k=2048, act="silu", dtype="bf16", skew=1.2, dropped=3, train=True),
        # -- products with bias, activation and residual
        # one token through the projection back, added to its residual stream
        dict(name="act_one_token", op="act", tokens=1, n=4096, k=14336, act="none", bias=False,
             residual=True, dtype="bf16", train=False),
        # a batch through an expanding layer with bias
        dict(name="act_batch", op="act", tokens=200, n=16384, k=4096, act="gelu", bias=True,
             residual=False, dtype="fp16", train=False),
        # a training step with everything in the epilogue
        dict(name="act_train", op="act", tokens=8191, n=8192, k=2048, act="gelu_tanh", bias=True,
             residual=True, dtype="bf16", train=True),
        # -- the gradient norm over many tensors, and clipping by it
        # a small model's gradients: latency
        dict(name="clip_small", op="clip", tensors=60, least=64, most=40000, total=400000, step=1,
             wide=0.3, max_norm=0.01, dtype="bf16"),
        # the gradients of a training step of a large layer
        dict(name="clip_large", op="clip", tensors=48, least=4096, most=117440512,
             total=1200000000, step=8, wide=0.1, max_norm=0.1, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    """A multiple of `step`, even over the logarithm."""
    return max(step, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(["gated", "gated", "act", "clip"])
    dtype = rng.choice(["bf16", "fp16"])
    act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
    if op == "clip":
        tensors = _log(rng, 1, 400)
        most = _log(rng, 256, 50000000)
        return dict(op=op, tensors=tensors, least=rng.choice([0, 1, 100]), most=most,
                    total=_log(rng, 1000, min(1000000000, tensors * most + 1000)),
                    step=rng.choice([1, 8, 64]), wide=rng.choice([0.0, 0.3, 1.0]),
                    max_norm=rng.choice([0.001, 0.1, 1e6]), dtype=dtype)
    n = _size(rng, 256, 14336, rng.choice([1, 8, 64, 128]))
    k = _size(rng, 256, 14336, rng.choice([1, 8, 64, 128]))
    if op == "act":
        train = rng.random() < 0.5
        return dict(op=op, tokens=_log(rng, 1, 8192 if n * k <= 2 ** 25 else 2048), n=n, k=k,
                    act=act, bias=rng.random() < 0.6, residual=rng.random() < 0.6, dtype=dtype,
                    train=train)
    train = rng.random() < 0.4
    experts = rng.choice([0, 0, 4, 8, 17, 64])
    top_k = rng.randint(1, 4) if experts else 1
    while max(experts, 1) * n * k > 4 * 14336 * 4096:
        if n > k:
            n = max(256, n // 2)
        else:
            k = max(256, k // 2)
    tokens = _log(rng, 1, min(8192, 8192 * 4096 * 14336 // (n * k * top_k)))
    if train:
        tokens = min(tokens, 4095, 4095 * 4096 * 14336 // (n * k * top_k))
    rows = tokens * top_k
    return dict(op=op, tokens=tokens, top_k=top_k, experts=experts, n=n, k=k, act=act, dtype=dtype,
                skew=rng.choice([0.0, 0.3, 1.0]) if experts else 0.0,
                dropped=rng.choice([0, 0, min(rows, 3)]) if experts else 0, train=train)


def _sizes(case):
    """Elements of each tensor, and which are 32 bits wide: a model's, whatever the
    seed.  Even over the logarithm, about `total` together at the most."""
    r = np.random.default_rng(case["tensors"])
    lo, hi = math.log(max(1, case["least"])), math.log(case["most"])
    n = np.exp(r.uniform(lo, hi, case["tensors"]))
    n = np.minimum(n * min(1.0, case["total"] / n.sum()), case["most"]).astype(np.int64)
    n = np.maximum(n // case["step"] * case["step"], case["least"])
    return n, r.random(case["tensors"]) < case["wide"]


def _counts(case, seed):
    """Rows per expert when every token goes to top_k different experts."""
    e, t, k = case["experts"], case["tokens"], case["top_k"]
    r = np.random.default_rng(seed)
    lean = -case["skew"] * np.log(np.arange(1, e + 1))  # a power law over the experts
    lean = lean[r.permutation(e)]
    score = lean[None, :] + r.gumbel(size=(t, e))
    chosen = np.argpartition(-score, k - 1, axis=1)[:, :k]
    return np.bincount(chosen.reshape(-1), minlength=e)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)

    state = {"case": case}
    if case["op"] == "clip":
        # A trainer's buckets: 16-bit gradients in one, 32-bit ones in another.
        sizes, wide = _sizes(case)
        # (fp16 gradients come with a loss scale that keeps them off its smallest values)
        low = -2 if case["dtype"] == "fp16" else -7
        spread = np.random.default_rng(seed).uniform(low, low + 3, len(sizes))
        grads, buckets = [], []
        for want, dtype in ((False, dt), (True, torch.float32)):
            mine = np.nonzero(wide == want)[0]
            flat = randn(int(sizes[mine].sum()), dtype=dtype)
            buckets.append(flat)
            at = 0
            for i in mine:
                part = flat[at:at + int(sizes[i])]
                part.mul_(10.0 ** spread[i])
                grads.append(part)
                at += int(sizes[i])
        state["grads"], state["buckets"] = grads, buckets
        state["max_norm"] = case["max_norm"]
        return state
    n, k = case["n"], case["k"]
    rows = case["tokens"]
    if case["op"] == "gated":
        bank = ()
        if case["experts"]:
            counts = _counts(case, seed)
            rows = int(counts.sum())
            ends = np.minimum(np.cumsum(counts), rows - case["dropped"])  # the last are padding
            offsets = np.concatenate([[0], ends]).astype(np.int32)
            state["most"] = max(1, int(np.diff(offsets).max()))
            state["offsets"] = torch.from_numpy(offsets).cuda()
            bank = (case["experts"],)
        state["wg"] = randn(*bank, n, k, scale=k ** -0.5)
        state["wu"] = randn(*bank, n, k, scale=k ** -0.5)
        leaves = ("x", "wg", "wu")
    else:
        state["w"] = randn(n, k, scale=k ** -0.5)
        state["b"] = randn(n) if case["bias"] else None
        state["r"] = randn(rows, n) if case["residual"] else None
        leaves = ("x", "w", "b", "r")
    state["x"] = randn(rows, k)
    if case["train"]:
        state["dy"] = randn(rows, n)
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------ plain forms
ROOT_2_PI = math.sqrt(2 / math.pi)


def _act(name, z):
    """act(z) and its derivative, elementwise."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s, s * (1 - s)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-2 * ROOT_2_PI * (z + 0.044715 * z * z * z)))
    return z * s, s + z * s * (1 - s) * 2 * ROOT_2_PI * (1 + 3 * 0.044715 * z * z)


def _spread(offsets, most, rows):
    """index (experts, most) of each expert's rows and which of them are real;
    per row its expert, its place there, and whether an expert owns it."""
    at = torch.arange(most, device=offsets.device)
    index = offsets[:-1, None].long() + at[None, :]
    real = index < offsets[1:, None]
    row = torch.arange(rows, device=offsets.device)
    expert = (row[:, None] >= offsets[None, 1:]).sum(1)
    owned = expert < offsets.numel() - 1
    expert = expert.clamp(max=offsets.numel() - 2)
    return index.clamp(max=rows - 1), real, expert, (row - offsets[expert]).clamp(max=most - 1), owned


def _plain_gated(state):
    case = state["case"]
    dt = state["x"].dtype
    x, wg, wu = (state[v].detach().float() for v in ("x", "wg", "wu"))
    dy = state["dy"].float() if case["train"] else None
    if case["experts"]:
        index, real, expert, place, owned = _spread(state["offsets"], state["most"], x.shape[0])

        def apart(t):  # rows to (experts, most, width)
            return torch.where(real[..., None], t[index], 0)

        def together(t):
            return torch.where(owned[:, None], t[expert, place], 0)
    else:
        apart = together = lambda t: t  # noqa: E731
    x = apart(x)
    g, u = x @ wg.transpose(-1, -2), x @ wu.transpose(-1, -2)
    a, slope = _act(case["act"], g)
    h = together(a * u).to(dt)
    if not case["train"]:
        return h
    dy = apart(dy)
    dg, du = dy * u * slope, dy * a
    dx = together(dg @ wg + du @ wu)
    return {"h": h, "dx": dx.to(dt), "dwg": (dg.transpose(-1, -2) @ x).to(dt),
            "dwu": (du.transpose(-1, -2) @ x).to(dt)}


def _plain_act(state):
    case = state["case"]
    x, w = state["x"].detach(), state["w"].detach()
    dt = x.dtype
    x, w = x.float(), w.float()
    z = x @ w.t()
    if state["b"] is not None:
        z = z + state["b"].detach().float()
    y, slope = _act(case["act"], z)
    if state["r"] is not None:
        y = y + state["r"].detach().float()
    if not case["train"]:
        return y.to(dt)
    dz = state["dy"].float() * slope
    got = {"y": y.to(dt), "dx": (dz @ w).to(dt), "dw": (dz.t() @ x).to(dt)}
    if state["b"] is not None:
        got["db"] = dz.sum(0).to(dt)
    if state["r"] is not None:
        got["dr"] = state["dy"].clone()
    return got


def _plain_clip(state):
    squares = [t.float().square().sum(dtype=torch.float64) for t in state["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    scale = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    _ = [t.copy_(t.float() * scale) for t in state["grads"]]
    return {"norm": norm.float(), "buckets": state["buckets"]}


# ------------------------------------------------------------------------ run
def run(state):
    case = state["case"]
    if not own:
        return {"gated": _plain_gated, "act": _plain_act, "clip": _plain_clip}[case["op"]](state)
    import blackwell_gemm_b200 as bg
    if case["op"] == "clip":
        norm = bg.clip_grads_b200(state["grads"], state["max_norm"])
        return {"norm": norm, "buckets": state["buckets"]}
    if case["op"] == "gated":
        x, wg, wu = state["x"], state["wg"], state["wu"]
        h = bg.matmul_b200_gated(x, wg.transpose(-1, -2), wu.transpose(-1, -2),
                                 state.get("offsets"), activation=case["act"])
        if not case["train"]:
            return h
        dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), state["dy"])
        return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}
    x, w, b, r = (state[v] for v in ("x", "w", "b", "r"))
    y = bg.matmul_b200_act(x, w.t(), b, r, activation=case["act"])
    if not case["train"]:
        return y
    names = ["dx", "dw"] + ["db"] * (b is not None) + ["dr"] * (r is not None)
    leaves = [t for t in (x, w, b, r) if t is not None]
    return {"y": y, **dict(zip(names, torch.autograd.grad(y, leaves, state["dy"])))}


# ----------------------------------------------------------------------- work
def work(case):
    if case["op"] == "clip":
        sizes, wide = _sizes(case)
        elements = float(sizes.sum())
        # read for the norm; read and written again for the scale
        return {"bytes": 3 * float((sizes * np.where(wide, 4, 2)).sum()), "flops": 3 * elements}
    n, k = case["n"], case["k"]
    rows = case["tokens"] * case.get("top_k", 1)
    if case["op"] == "gated":
        e = case["experts"]
        active = e * (1 - (1 - case["top_k"] / e) ** case["tokens"]) if e else 1  # expected
        bytes_ = 2 * (2 * active * n * k + rows * (n + k))
        if not case["train"]:
            return {"bytes": bytes_, "flops": 4 * rows * n * k}
        # dy read; dx and both weights' gradients written
        return {"bytes": bytes_ + 2 * (rows * (n + k) + 2 * max(e, 1) * n * k),
                "flops": 12 * rows * n * k}
    bytes_ = 2 * (n * k + rows * (n + k) + n * case["bias"] + rows * n * case["residual"])
    if not case["train"]:
        return {"bytes": bytes_, "flops": 2 * rows * n * k}
    return {"bytes": bytes_ + 2 * (rows * (n + k) + n * k + n * case["bias"] +
                                   rows * n * case["residual"]), "flops": 6 * rows * n * k}


# ---------------------------------------------------------------------- exact
def _curve(name, z):
    """The activation and its slope in 64 bits, from their definitions."""
    if name == "gelu":
        half = torch.special.erf(z / 2 ** 0.5)
        # Phi from its smaller tail, which 1 + erf would lose
        tail = torch.special.erfc(z.abs() / 2 ** 0.5) / 2
        phi = torch.where(half < 0, tail, 1 - tail)
        return z * phi, phi + z * torch.exp(-z.square() / 2) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return (z * (1 + t) / 2,
                (1 + t) / 2 + z / 2 * (1 - t * t) * c * (1 + 0.134145 * z.square()))
    if name == "relu":
        return torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
    if name == "none":
        return z, torch.ones_like(z)
    p = torch.special.expit(z)
    q = torch.special.expit(-z)
    return (p, p * q) if name == "sigmoid" else (z * p, p + z * p * q)


def exact(case, seed):
    """The definition, expert by expert and tensor by tensor, in 64 bits."""
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    state = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in state.items()}
    if case["op"] == "clip":
        total = math.fsum(float(t.double().norm()) ** 2 for t in state["grads"] if t.numel())
        norm = math.sqrt(total)
        scale = min(1.0, state["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64),
                "buckets": [b.double() * scale for b in state["buckets"]]}
    x = state["x"].double()
    if case["op"] == "act":
        w = state["w"].double()
        z = torch.mm(x, w.t())
        if case["bias"]:
            z += state["b"].double()
        y, slope = _curve(case["act"], z)
        if case["residual"]:
            y = y + state["r"].double()
        if not case["train"]:
            return y
        dy = state["dy"].double()
        dz = dy * slope
        got = {"y": y, "dx": torch.mm(dz, w), "dw": torch.mm(dz.t(), x)}
        if case["bias"]:
            got["db"] = dz.sum(0)
        if case["residual"]:
            got["dr"] = dy
        return got
    spans = [(None, 0, x.shape[0])]
    if case["experts"]:
        o = state["offsets"].tolist()
        spans = [(e, o[e], o[e + 1]) for e in range(case["experts"])]
    h = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
    if case["train"]:
        dx = torch.zeros_like(x)
        dwg = torch.zeros(state["wg"].shape, dtype=torch.float64, device=x.device)
        dwu = torch.zeros_like(dwg)
    for e, a, b in spans:
        if b <= a:
            continue
        wg, wu = ((state[v] if e is None else state[v][e]).double() for v in ("wg", "wu"))
        g, u = torch.mm(x[a:b], wg.t()), torch.mm(x[a:b], wu.t())
        y, slope = _curve(case["act"], g)
        h[a:b] = y * u
        if case["train"]:
            dy = state["dy"][a:b].double()
            dg, du = dy * u * slope, dy * y
            dx[a:b] = torch.mm(dg, wg) + torch.mm(du, wu)
            at = slice(None) if e is None else e
            dwg[at] = torch.mm(dg.t(), x[a:b])
            dwu[at] = torch.mm(du.t(), x[a:b])
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu} if case["train"] else h
