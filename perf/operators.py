"""Cases for the mixture-of-experts operators: routing, grouped products, 4-bit products.

``run`` computes one pass, in elementary torch operations (``own`` false) or
through the package's entry points (``own`` true), on what ``prepare`` made.
Rows are sorted by expert; expert e holds rows offsets[e] .. offsets[e+1]-1.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # -- products grouped by expert, forward (serving) and with gradients (training)
        # one new token through the up projection of two of eight experts
        dict(name="grouped_one_token", op="grouped", tokens=1, top_k=2, experts=8, n=14336, k=4096,
             dtype="bf16", skew=0.0, dropped=0, train=False),
        # a decode batch through the down projection, a few rows per expert
        dict(name="grouped_decode_batch", op="grouped", tokens=61, top_k=2, experts=8, n=4096,
             k=14336, dtype="fp16", skew=0.5, dropped=0, train=False),
        # a chunk of prompts over many small experts, odd sizes, padding rows at the end
        dict(name="grouped_chunk", op="grouped", tokens=509, top_k=4, experts=32, n=2056, k=1032,
             dtype="bf16", skew=0.7, dropped=5, train=False),
        # a long prompt through the up projection
        dict(name="grouped_prompt", op="grouped", tokens=8192, top_k=2, experts=8, n=14336, k=4096,
             dtype="bf16", skew=0.4, dropped=0, train=False),
        # a training step of many fine experts, some of them without a row
        dict(name="grouped_train_fine", op="grouped", tokens=2047, top_k=4, experts=64, n=1024,
             k=2048, dtype="bf16", skew=1.2, dropped=3, train=True),
        # a training step of a large bank
        dict(name="grouped_train_large", op="grouped", tokens=4096, top_k=2, experts=8, n=14336,
             k=4096, dtype="bf16", skew=0.3, dropped=0, train=True),
        # -- 4-bit weights with group scales
        # one token through one square projection: latency
        dict(name="w4_vector", op="w4", tokens=1, top_k=0, experts=1, n=8192, k=8192, group=128,
             zeros=False, dtype="bf16"),
        # a decode batch through a wide projection, with zero points
        dict(name="w4_batch", op="w4", tokens=16, top_k=0, experts=1, n=28672, k=4096, group=64,
             zeros=True, dtype="fp16"),
        # a few tokens through a bank of experts
        dict(name="w4_experts", op="w4", tokens=7, top_k=2, experts=8, n=14336, k=4096, group=128,
             zeros=False, dtype="bf16"),
        # a larger batch, small groups
        dict(name="w4_many_rows", op="w4", tokens=200, top_k=0, experts=1, n=4096, k=14336,
             group=32, zeros=True, dtype="bf16"),
        # -- routing: choice of experts, gather of their rows, weighted sum of their answers
        # a decode batch: latency
        dict(name="route_decode", op="route", tokens=16, top_k=2, experts=8, width=4096,
             normalize=True, masked=0.0, dtype="bf16", train=False),
        # a training step with masked experts and padding tokens
        dict(name="route_train", op="route", tokens=16383, top_k=4, experts=64, width=2048,
             normalize=False, masked=0.2, dtype="bf16", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    """A multiple of `step`, even over the logarithm (one size is left out)."""
    v = max(step, _log(rng, lo, hi) // step * step)
    return v + step if v == 3072 else v


def draw(rng):
    op = rng.choice(["grouped", "grouped", "w4", "route"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "grouped":
        train = rng.random() < 0.4
        experts = rng.choice([4, 8, 16, 17, 32, 64])
        top_k = rng.randint(1, min(4, experts))
        n = _size(rng, 256, 14336, rng.choice([1, 8, 64, 128]))
        k = _size(rng, 256, 14336, rng.choice([1, 8, 64, 128]))
        while experts * n * k > 8 * 14336 * 4096:
            if n > k:
                n = max(256, n // 2)
            else:
                k = max(256, k // 2)
        n, k = (v + 1 if v == 3072 else v for v in (n, k))
        tokens = _log(rng, 1, min(8192, 8192 * 4096 * 14336 // (n * k * top_k)))
        if train:
            tokens = min(tokens, 4096)
        rows = tokens * top_k
        return dict(op=op, tokens=tokens, top_k=top_k, experts=experts, n=n, k=k, dtype=dtype,
                    skew=rng.choice([0.0, 0.3, 1.0]), dropped=rng.choice([0, 0, min(rows, 3)]),
                    train=train)
    if op == "w4":
        experts = rng.choice([1, 1, 8, 16])
        group = rng.choice([32, 64, 128])
        n = _size(rng, 256, 28672, rng.choice([1, 8, 128]))
        k = _size(rng, 512, 14336, group)
        while experts * n * k > 8 * 14336 * 4096:
            n = max(256, n // 2)
        n = n + 1 if n == 3072 else n
        k = k + group if k == 3072 else k
        return dict(op=op, tokens=_log(rng, 1, 200), top_k=0 if experts == 1 else 2,
                    experts=experts, n=n, k=k, group=group, zeros=rng.random() < 0.5, dtype=dtype)
    experts = rng.choice([4, 8, 60, 64, 128, 256])
    width = _size(rng, 256, 8192, 8)
    top_k = rng.randint(1, min(8, experts))
    most = 16383 * 4 * 2048 // (width * top_k)
    return dict(op=op, tokens=_log(rng, 1, min(16384, most)), top_k=top_k, experts=experts,
                width=width, normalize=rng.random() < 0.5, masked=rng.choice([0.0, 0.2]),
                dtype=dtype, train=rng.random() < 0.5)


def _counts(case, seed):
    """Rows per expert when every token goes to top_k different experts."""
    e, t, k = case["experts"], case["tokens"], case["top_k"]
    r = np.random.default_rng(seed)
    lean = -case.get("skew", 0.0) * np.log(np.arange(1, e + 1))  # a power law over the experts
    lean = lean[r.permutation(e)]
    score = lean[None, :] + r.gumbel(size=(t, e))
    chosen = np.argpartition(-score, k - 1, axis=1)[:, :k]
    return np.bincount(chosen.reshape(-1), minlength=e)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _bank(case, seed):
    """offsets (experts + 1) on the device, the largest count, all rows."""
    counts = _counts(case, seed)
    rows = int(counts.sum())
    drop = case.get("dropped", 0)
    ends = np.minimum(np.cumsum(counts), rows - drop)  # the last rows are padding
    offsets = np.concatenate([[0], ends]).astype(np.int32)
    most = max(1, int(np.diff(offsets).max()))
    return torch.from_numpy(offsets).cuda(), most, rows


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt).mul_(scale)

    state = {"case": case}
    if case["op"] == "grouped":
        e, n, k = case["experts"], case["n"], case["k"]
        state["offsets"], state["most"], rows = _bank(case, seed)
        state["x"] = randn(rows, k)
        state["w"] = randn(e, n, k, scale=k ** -0.5)
        if case["train"]:
            state["dy"] = randn(rows, n)
            state["x"].requires_grad_(True)
            state["w"].requires_grad_(True)
    elif case["op"] == "w4":
        e, n, k, group = case["experts"], case["n"], case["k"], case["group"]
        rows = case["tokens"]
        if e > 1:
            state["offsets"], state["most"], rows = _bank(case, seed)
        state["x"] = randn(rows, k)
        q = torch.randint(0, 256, (e, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s = (torch.rand(e, n, k // group, generator=g, device="cuda") + 0.5) * (0.2 * k ** -0.5)
        s = s.to(dt)
        z = None
        if case["zeros"]:
            z = torch.randint(4, 12, (e, n, k // group), generator=g, device="cuda",
                              dtype=torch.uint8)
        if own:  # a server lays its weights out once, when it loads them
            import blackwell_gemm_b200 as bg
            if e == 1:
                q, s, z = q[0], s[0], None if z is None else z[0]
            state["weight"] = bg.pack_w4(q, s, z)
        else:
            state["q"], state["s"], state["z"] = q, s, z
    else:
        t, e, k, width = case["tokens"], case["experts"], case["top_k"], case["width"]
        logits = torch.randn(t, e, generator=g, device="cuda")
        if case["masked"]:
            shut = torch.rand(t, e, generator=g, device="cuda") < case["masked"]
            shut |= torch.rand(t, 1, generator=g, device="cuda") < 0.02  # padding tokens
            logits.masked_fill_(shut, -math.inf)
        state["logits"] = logits
        state["x"] = randn(t, width)
        state["y"] = randn(t * k, width)  # the experts' answers
        if case["train"]:
            state["dout"] = randn(t, width)
            state["dxs"] = randn(t * k, width)
            for name in ("logits", "x", "y"):
                state[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------ plain forms
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
    return index.clamp(max=rows - 1), real, expert, row - offsets[expert], owned


def _plain_product(x, w, offsets, most):
    """The grouped product, and what its gradients need; w (E, N, K) in 32 bits."""
    index, real, expert, place, owned = _spread(offsets, most, x.shape[0])
    xs = x.float()[index] * real[..., None]
    y = torch.bmm(xs, w.transpose(1, 2))
    place = place.clamp(max=most - 1)
    return y[expert, place] * owned[:, None], (xs, index, real, expert, place, owned)


def _plain_grouped(state):
    case = state["case"]
    x, w = state["x"].detach(), state["w"].detach()
    wide = w.float()
    y, kept = _plain_product(x, wide, state["offsets"], state["most"])
    if not case["train"]:
        return y.to(x.dtype)
    xs, index, real, expert, place, owned = kept
    dys = state["dy"].float()[index] * real[..., None]
    dx = torch.bmm(dys, wide)[expert, place] * owned[:, None]
    dw = torch.bmm(dys.transpose(1, 2), xs)
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(x.dtype)}


def _plain_w4(state):
    case = state["case"]
    x, q, s, z = state["x"], state["q"], state["s"], state["z"]
    e, n, k, group = case["experts"], case["n"], case["k"], case["group"]
    w = torch.stack((q & 15, q >> 4), dim=-1).reshape(e, n, k // group, group).float()
    w = w - (8.0 if z is None else z.float()[..., None])
    w = (w * s.float()[..., None]).reshape(e, n, k)
    if e == 1:
        return (x.float() @ w[0].t()).to(x.dtype)
    return _plain_product(x, w, state["offsets"], state["most"])[0].to(x.dtype)


def _plain_route(state):
    case = state["case"]
    logits, x, y = (state[v].detach() for v in ("logits", "x", "y"))
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    top, experts = torch.sort(logits, dim=1, descending=True, stable=True)
    top, experts = top[:, :k], experts[:, :k]
    open_ = top > -math.inf
    base = top[:, :1].clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(logits - base)
    chosen = torch.exp(top - base)
    total = chosen.sum(1, keepdim=True) if case["normalize"] else p.sum(1, keepdim=True)
    total = total.clamp(min=torch.finfo(torch.float32).tiny)
    weights = chosen / total
    flat = torch.where(open_, experts, e).reshape(-1)
    order = torch.argsort(flat, stable=True)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(t * k, device=order.device)
    counts = torch.bincount(flat, minlength=e + 1)[:e]
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=order.device)
    offsets[1:] = counts.cumsum(0)
    owned = torch.arange(t * k, device=order.device) < offsets[-1]
    rows = torch.where(open_, rows.reshape(t, k), -1)
    tokens = torch.where(owned, order // k, -1)
    experts = torch.where(open_, experts, -1)
    xs = torch.where(owned[:, None], x[tokens.clamp(min=0)], 0)
    mine = torch.where(open_[..., None], y[rows.clamp(min=0)].float(), 0)
    out = (weights[..., None] * mine).sum(1)
    got = {"weights": weights, "experts": experts.int(), "rows": rows.int(),
           "tokens": tokens.int(), "offsets": offsets, "xs": xs, "out": out.to(y.dtype)}
    if not case["train"]:
        return got
    dout = state["dout"].float()
    dxs = torch.where(open_[..., None], state["dxs"][rows.clamp(min=0)].float(), 0)
    dweights = (dout[:, None, :] * mine).sum(2)
    inner = (weights * dweights).sum(1, keepdim=True)
    share = p / total
    # an empty slot is written to a column of its own
    column = torch.where(open_, experts, e).long()
    hit = torch.zeros(t, e + 1, device=x.device).scatter_(
        1, column, torch.where(open_, dweights, 0))[:, :e]
    if case["normalize"]:
        took = torch.zeros(t, e + 1, device=x.device).scatter_(1, column, 1.0)[:, :e]
        dlogits = share * took * (hit - inner)
    else:
        dlogits = share * (hit - inner)
    dy = torch.zeros(t * k + 1, y.shape[1], device=x.device)
    dy[torch.where(open_, rows, t * k)] = weights[..., None] * dout[:, None, :]
    return {**got, "dlogits": dlogits, "dx": dxs.sum(1).to(x.dtype), "dy": dy[:-1].to(y.dtype)}


# ------------------------------------------------------------------------ run
def run(state):
    case = state["case"]
    if not own:
        return {"grouped": _plain_grouped, "w4": _plain_w4, "route": _plain_route}[case["op"]](state)
    import blackwell_gemm_b200 as bg
    if case["op"] == "grouped":
        x, w = state["x"], state["w"]
        y = bg.matmul_b200_grouped(x, w.transpose(1, 2), state["offsets"])
        if not case["train"]:
            return y
        dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if case["op"] == "w4":
        return bg.matmul_b200_w4(state["x"], state["weight"], state.get("offsets"))
    routing = bg.route_b200(state["logits"], case["top_k"], normalize=case["normalize"])
    xs = bg.dispatch_b200(state["x"], routing)
    out = bg.combine_b200(state["y"], routing)
    got = {"weights": routing.weights, "experts": routing.experts, "rows": routing.rows,
           "tokens": routing.tokens, "offsets": routing.offsets, "xs": xs, "out": out}
    if not case["train"]:
        return got
    dlogits, dx, dy = torch.autograd.grad((out, xs), (state["logits"], state["x"], state["y"]),
                                          (state["dout"], state["dxs"]))
    return {**got, "dlogits": dlogits, "dx": dx, "dy": dy}


# ----------------------------------------------------------------------- work
def work(case):
    t, e = case["tokens"], case["experts"]
    if case["op"] == "route":
        k, h = case["top_k"], case["width"]
        small = t * e * 4 + t * k * 16 + e * 4
        bytes_ = small + 2 * h * (t + t * k) * 2  # x -> xs, y -> out
        flops = 2 * t * k * h
        if case["train"]:
            # dxs -> dx; dout and y -> dy and the weights' gradients (y is read once in all)
            bytes_ += 2 * h * (t * k + t) + 2 * h * (t + t * k) + t * e * 4
            flops += 5 * t * k * h
        return {"bytes": bytes_, "flops": flops}
    n, k = case["n"], case["k"]
    rows = t * case["top_k"] if case["top_k"] else t
    active = e * (1 - (1 - case["top_k"] / e) ** t) if case["top_k"] else 1  # expected
    if case["op"] == "w4":
        per = 0.5 + (2 + case["zeros"]) / case["group"]
        return {"bytes": active * n * k * per + 2 * rows * (n + k), "flops": 2 * rows * n * k}
    bytes_ = 2 * (active * n * k + rows * (n + k))
    if not case["train"]:
        return {"bytes": bytes_, "flops": 2 * rows * n * k}
    # dy read; dx and dw written
    return {"bytes": bytes_ + 2 * (rows * (n + k) + e * n * k), "flops": 6 * rows * n * k}


# ---------------------------------------------------------------------- exact
def exact(case, seed):
    """The definition, expert by expert and token by token, in 64 bits."""
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    state = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in state.items()}
    if case["op"] == "route":
        return _exact_route(state)
    x = state["x"].double()
    spans = [(0, 0, x.shape[0])]
    if "offsets" in state:
        o = state["offsets"].tolist()
        spans = [(i, o[i], o[i + 1]) for i in range(case["experts"])]

    def matrix(e):
        if case["op"] == "grouped":
            return state["w"][e].double()
        q = state["q"][e]
        w = torch.empty(case["n"], case["k"], dtype=torch.float64, device=q.device)
        w[:, 0::2] = (q % 16).double()
        w[:, 1::2] = (q // 16).double()
        size = case["group"]
        for j in range(case["k"] // size):
            zero = 8.0 if state["z"] is None else state["z"][e, :, j, None].double()
            part = w[:, j * size:(j + 1) * size]
            part.sub_(zero).mul_(state["s"][e, :, j, None].double())
        return w

    y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
    train = case.get("train", False)
    if train:
        dx = torch.zeros_like(x)
        dw = torch.zeros(case["experts"], case["n"], case["k"], dtype=torch.float64,
                         device=x.device)
    for e, a, b in spans:
        if b <= a:
            continue
        w = matrix(e)
        y[a:b] = x[a:b] @ w.t()
        if train:
            dy = state["dy"][a:b].double()
            dx[a:b] = dy @ w
            dw[e] = dy.t() @ x[a:b]
    return {"y": y, "dx": dx, "dw": dw} if train else y


def _exact_route(state):
    case = state["case"]
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = state["logits"].double().cpu().numpy()
    dev = state["x"].device
    weights = np.zeros((t, k))
    experts = np.full((t, k), -1, dtype=np.int32)
    share = np.zeros((t, e))
    for i in range(t):
        order = np.lexsort((np.arange(e), -logits[i]))[:k]
        order = order[logits[i, order] > -np.inf]
        if not order.size:
            continue
        ex = np.exp(logits[i] - logits[i, order[0]])
        if case["normalize"]:
            keep = np.zeros(e)
            keep[order] = 1
            ex = ex * keep
        share[i] = ex / ex.sum()
        weights[i, :order.size] = share[i, order]
        experts[i, :order.size] = order
    rows = np.full((t, k), -1, dtype=np.int32)
    tokens = np.full(t * k, -1, dtype=np.int32)
    offsets = np.zeros(e + 1, dtype=np.int32)
    at = 0
    for j in range(e):
        ti, slot = np.nonzero(experts == j)
        rows[ti, slot] = np.arange(at, at + ti.size)
        tokens[at:at + ti.size] = ti
        at += ti.size
        offsets[j + 1] = at
    y, x = state["y"].double(), state["x"].double()
    xs = torch.zeros(t * k, x.shape[1], dtype=torch.float64, device=dev)
    xs[:at] = x[torch.from_numpy(tokens[:at]).long().to(dev)]
    out = torch.zeros_like(x)
    for j in range(k):
        ok = torch.from_numpy(np.nonzero(rows[:, j] >= 0)[0]).to(dev)
        r = torch.from_numpy(rows[rows[:, j] >= 0, j]).long().to(dev)
        out[ok] += torch.from_numpy(weights[rows[:, j] >= 0, j]).to(dev)[:, None] * y[r]
    got = {"weights": torch.from_numpy(weights).to(dev), "experts": torch.from_numpy(experts),
           "rows": torch.from_numpy(rows), "tokens": torch.from_numpy(tokens),
           "offsets": torch.from_numpy(offsets), "xs": xs, "out": out}
    if not case["train"]:
        return got
    dout, dxs = state["dout"].double(), state["dxs"].double()
    dx, dy = torch.zeros_like(x), torch.zeros_like(y)
    hit = np.zeros((t, e))
    inner = np.zeros((t, 1))
    for j in range(k):
        have = np.nonzero(rows[:, j] >= 0)[0]
        ok = torch.from_numpy(have).to(dev)
        r = torch.from_numpy(rows[have, j]).long().to(dev)
        w = torch.from_numpy(weights[have, j]).to(dev)
        dx[ok] += dxs[r]
        dy[r] = w[:, None] * dout[ok]
        dweight = (dout[ok] * y[r]).sum(1).cpu().numpy()
        hit[have, experts[have, j]] = dweight
        inner[have, 0] += weights[have, j] * dweight
    dlogits = share * (hit - inner)
    return {**got, "dlogits": torch.from_numpy(dlogits).to(dev), "dx": dx, "dy": dy}
