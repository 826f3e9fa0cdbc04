"""Workloads of the operators around the expert layer: norm, balance loss, adapted projection.

Each in its plain form (elementary torch operations in 32 bits, in 64 where a value decides a code,
rounded once at the end) and through the framework's entry points (exfold_b200.ops):

  norm        root-mean-square norm of the sum with the residual stream
  norm_8bit   the same with its output in 8 bits and scales, and reading it back
  norm_grad   the norm in training: its outputs and the gradients of both inputs and the weight
  balance     the balance loss over a router's logits and routes, the experts' counts and the
              logits' gradient
  adapted     a shared projection with the low-rank adapters of many requests
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one sequence before a layer, where the launch is all of the time
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 2048, "dtype": "bf16",
         "weight": "same", "residual": True, "strided": False},
        # a prefill batch of a DeepSeek-style layer (hidden 4096)
        {"name": "norm prefill", "op": "norm", "rows": 32768, "cols": 4096, "dtype": "bf16",
         "weight": "same", "residual": True, "strided": False},
        # the decode batch of the Qwen3 layer, for 8-bit products with a scale per 128 columns
        {"name": "norm_8bit decode", "op": "norm_8bit", "rows": 256, "cols": 2048,
         "dtype": "bf16", "weight": "same", "residual": True, "strided": False, "code": "e4m3",
         "group": 128},
        # a small odd batch in fp16: integer codes with one scale a row
        {"name": "norm_8bit ragged int8", "op": "norm_8bit", "rows": 61, "cols": 1001,
         "dtype": "fp16", "weight": "fp32", "residual": False, "strided": False, "code": "int8",
         "group": 0},
        # a prefill batch in 8 bits
        {"name": "norm_8bit prefill", "op": "norm_8bit", "rows": 8192, "cols": 4096,
         "dtype": "bf16", "weight": "same", "residual": True, "strided": False, "code": "e4m3",
         "group": 128},
        # a small training micro-batch in fp32, no multiple of any vector
        {"name": "norm_grad ragged fp32", "op": "norm_grad", "rows": 777, "cols": 1001,
         "dtype": "fp32", "weight": "same", "residual": True, "strided": False},
        # a training micro-batch of the DeepSeek-style layer
        {"name": "norm_grad batch", "op": "norm_grad", "rows": 8192, "cols": 4096,
         "dtype": "bf16", "weight": "same", "residual": True, "strided": False},
        # one short sequence over few experts
        {"name": "balance short", "op": "balance", "groups": 1, "tokens": 512, "experts": 64,
         "top_k": 8, "dtype": "fp32", "scoring": "softmax", "padding": 0.0},
        # the tokens of one Qwen3 layer, one loss over all of them
        {"name": "balance layer", "op": "balance", "groups": 1, "tokens": 131072,
         "experts": 128, "top_k": 8, "dtype": "fp32", "scoring": "softmax", "padding": 0.0},
        # one loss for each of 16 sequences of differing length, sigmoid scores of 256 experts
        {"name": "balance padded sequences", "op": "balance", "groups": 16, "tokens": 4096,
         "experts": 256, "top_k": 8, "dtype": "bf16", "scoring": "sigmoid", "padding": 0.5},
        # the shared expert's down projection in a decode batch, each token another request
        {"name": "adapted decode mixed", "op": "adapted", "tokens": 64, "inner": 2048,
         "outer": 4096, "adapters": 32, "rank": 16, "dtype": "bf16", "runs": 0},
        # the same projection over a prefill batch of 12 requests
        {"name": "adapted prefill", "op": "adapted", "tokens": 8192, "inner": 2048,
         "outer": 4096, "adapters": 8, "rank": 64, "dtype": "bf16", "runs": 12},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm_8bit", "norm_grad", "balance", "adapted"])
    if op == "balance":
        groups = _log_int(rng, 1, 16)
        experts = rng.choice([64, 128, 256, _log_int(rng, 8, 512)])
        tokens = _log_int(rng, 1, 16_000_000 // (groups * experts))
        return {"op": op, "groups": groups, "tokens": tokens, "experts": experts,
                "top_k": rng.randint(1, 8), "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "scoring": rng.choice(["softmax", "sigmoid"]),
                "padding": rng.choice([0.0, 0.0, 0.1, 0.5])}
    if op == "adapted":
        inner, outer = 8 * _log_int(rng, 8, 512), 8 * _log_int(rng, 8, 512)
        tokens = min(_log_int(rng, 1, 8192), 60_000_000_000 // (inner * outer))
        return {"op": op, "tokens": tokens, "inner": inner, "outer": outer,
                "adapters": _log_int(rng, 1, 64), "rank": 8 * rng.choice([1, 2, 4, 8, 5]),
                "dtype": rng.choice(["bf16", "fp16"]),
                "runs": 0 if tokens <= 256 else rng.randint(1, 32)}
    cols = _log_int(rng, 16, 16384)
    rows = _log_int(rng, 1, min(65536, (32_000_000 if op != "norm" else 128_000_000) // cols))
    case = {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "weight": rng.choice(["same", "fp32"]), "residual": rng.choice([True, True, False]),
            "strided": rng.choice([False, False, True])}
    if op == "norm_8bit":
        case["code"] = rng.choice(["e4m3", "int8"])
        case["group"] = rng.choice([0, 32, 64, 128])
    return case


# ---- inputs -----------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _stream_rows(rows, cols, dtype, g, strided):
    """Rows of a residual stream: a size of their own, a few channels far above the rest.  strided:
    the first columns of a wider matrix."""
    x = torch.randn(rows, cols + (24 if strided else 0), generator=g, device="cuda")
    x *= torch.exp2(4.0 * torch.rand(rows, 1, generator=g, device="cuda") - 2.0)
    far = torch.rand(x.shape[1], generator=g, device="cuda") < 0.002
    x *= torch.where(far, 30.0, 1.0)
    return x.to(dtype)[:, :cols]


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    dtype = DTYPES[case["dtype"]]
    state = {"op": op}
    if op == "balance":
        n, t, e, k = (case[v] for v in ("groups", "tokens", "experts", "top_k"))
        logits = torch.randn(n, t, e, generator=g, device="cuda")
        # (a router that prefers some experts)
        logits += torch.randn(n, 1, e, generator=g, device="cuda")
        logits = (2.0 * logits).to(dtype)
        ids = logits.float().topk(k, -1).indices.int()
        mask = None
        if case["padding"] > 0.0:
            # sequences of differing length; what stands in their padding is not meant to be read
            length = t - (case["padding"] * 2.0 * t * torch.rand(
                n, 1, generator=g, device="cuda")).long().clamp(max=t)
            mask = torch.arange(t, device="cuda") < length
            logits = torch.where(mask.unsqueeze(-1), logits, float("nan"))
            ids = torch.where(mask.unsqueeze(-1), ids, -1)
        # a loss scale that brings the tokens' gradients to the size of their probabilities
        dloss = t * (0.5 + torch.rand(n, generator=g, device="cuda"))
        state.update(logits=logits.requires_grad_(True), ids=ids, mask=mask, dloss=dloss,
                     scoring=case["scoring"])
        return state
    if op == "adapted":
        t, k, n, r, c = (case[v] for v in ("tokens", "inner", "outer", "adapters", "rank"))

        def normal(*shape, size):
            return (size * torch.randn(*shape, generator=g, device="cuda")).to(dtype)

        state.update(x=normal(t, k, size=1.0), w=normal(n, k, size=k ** -0.5),
                     a=normal(r, c, k, size=k ** -0.5), b=normal(r, n, c, size=0.5 * c ** -0.5),
                     scaling=0.5 + 1.5 * torch.rand(r, generator=g, device="cuda"))
        if case["runs"] == 0:  # each token belongs to a request of its own
            ids = torch.randint(-1, r, (t,), generator=g, device="cuda")
        else:  # requests of differing length, one behind the other, some without an adapter
            cuts = torch.randint(0, t, (case["runs"] - 1,), generator=g, device="cuda").sort()[0]
            mine = torch.randint(-1, r, (case["runs"],), generator=g, device="cuda")
            ids = mine[torch.searchsorted(cuts, torch.arange(t, device="cuda"), right=True)]
        state["ids"] = ids.int()
        return state
    rows, cols = case["rows"], case["cols"]
    x = _stream_rows(rows, cols, dtype, g, case["strided"])
    r = _stream_rows(rows, cols, dtype, g, case["strided"]) if case["residual"] else None
    w = 1.0 + 0.3 * torch.randn(cols, generator=g, device="cuda")
    state.update(x=x, residual=r, weight=w if case["weight"] == "fp32" else w.to(dtype))
    if op == "norm_8bit":
        state.update(code=case["code"], group=case["group"])
    if op == "norm_grad":
        state["dy"] = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
        state["ds"] = (None if r is None
                       else torch.randn(rows, cols, generator=g, device="cuda").to(dtype))
        for v in (x, r, state["weight"]):
            if v is not None:
                v.requires_grad_(True)
    return state


# ---- plain forms --------------------------------------------------------------------------------
def _sum_rows(s):
    x, r = s["x"], s["residual"]
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def _inverse_norm(t):
    v = t.float()
    return torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)


def _plain_norm(s):
    t = _sum_rows(s)
    y = (t.float() * _inverse_norm(t) * s["weight"].float()).to(t.dtype)
    return y if s["residual"] is None else (y, t)


def _plain_norm_8bit(s):
    t = _sum_rows(s)
    cols = t.shape[1]
    group = s["group"] or cols
    # in 64 bits: whether a value falls to one code or the next
    p = t.double() * s["weight"].double()
    p = torch.nn.functional.pad(p, (0, -cols % group)).reshape(t.shape[0], -1, group)
    top = p.abs().amax(-1, keepdim=True)
    most = 448.0 if s["code"] == "e4m3" else 127.0
    q = p * most / torch.where(top > 0.0, top, 1.0)
    if s["code"] == "e4m3":
        step = torch.exp2((torch.frexp(q)[1] - 4).clamp(min=-9).double())
        q = torch.round(q / step) * step
    else:
        q = torch.round(q)
    scale = top * _inverse_norm(t).double().unsqueeze(1) / most
    y = (q * scale).reshape(t.shape[0], -1)[:, :cols].to(t.dtype)
    return y if s["residual"] is None else (y, t)


def _plain_norm_grad(s):
    t, w, dy = _sum_rows(s), s["weight"].float(), s["dy"].float()
    v, f = _inverse_norm(t), t.float()
    y = (f * v * w).to(t.dtype)
    wd = w * dy
    dx = v * wd - f * (v * v * v) * (wd * f).mean(-1, keepdim=True)
    dw = (dy * f * v).sum(0).to(s["weight"].dtype)
    if s["residual"] is None:
        return y, dx.to(t.dtype), dw
    dx = (dx + s["ds"].float()).to(t.dtype)
    return y, t, dx, dx, dw


def _plain_balance(s):
    x, ids, mask = s["logits"].float(), s["ids"], s["mask"]
    n, t, e = x.shape
    k = ids.shape[-1]
    valid = torch.ones(n, t, dtype=torch.bool, device=x.device) if mask is None else mask
    x = torch.where(valid.unsqueeze(-1), x, 0.0)
    if s["scoring"] == "softmax":
        u = torch.exp(x - x.amax(-1, keepdim=True))
        slope = 1.0
    else:
        u = 1.0 / (1.0 + torch.exp(-x))
        slope = 1.0 / (1.0 + torch.exp(x))
    p = torch.where(valid.unsqueeze(-1), u / u.sum(-1, keepdim=True), 0.0)
    there = (ids >= 0) & valid.unsqueeze(-1)
    place = torch.where(there, ids.long(), e) + torch.arange(n, device=x.device).view(n, 1, 1) * (
        e + 1)
    counts = torch.bincount(place.reshape(-1), minlength=n * (e + 1)).view(n, e + 1)[:, :e]
    tokens = valid.sum(-1, keepdim=True)
    share = counts.double() * e / (k * tokens.clamp(min=1).double() ** 2)
    loss = (share * p.double().sum(1)).sum(-1).float()
    a = (share * s["dloss"].double().unsqueeze(-1)).float().unsqueeze(1)
    d = p * (a - (p * a).sum(-1, keepdim=True)) * slope
    return loss, counts.int(), d.to(s["logits"].dtype)


def _plain_adapted(s):
    x, ids = s["x"].float(), s["ids"]
    y = x @ s["w"].float().t()
    for i in range(s["a"].shape[0]):
        rows = torch.nonzero(ids == i).squeeze(1)
        if rows.numel() > 0:
            z = s["scaling"][i] * (x[rows] @ s["a"][i].float().t())
            y[rows] += z @ s["b"][i].float().t()
    return y.to(s["x"].dtype)


PLAIN = {"norm": _plain_norm, "norm_8bit": _plain_norm_8bit, "norm_grad": _plain_norm_grad,
         "balance": _plain_balance, "adapted": _plain_adapted}


def run(state):
    op = state["op"]
    if not own:
        with torch.no_grad():
            return PLAIN[op](state)
    import sys

    if "exfold-moe_b200" not in sys.path:
        sys.path.insert(0, "exfold-moe_b200")
    from exfold_b200 import ops

    if op == "balance":
        loss, counts = ops.balance_loss(state["logits"], state["ids"], scoring=state["scoring"],
                                        mask=state["mask"])
        dlogits, = torch.autograd.grad(loss, state["logits"], state["dloss"])
        return loss.detach(), counts, dlogits
    if op == "adapted":
        return ops.adapted_linear(state["x"], state["w"], state["a"], state["b"], state["ids"],
                                  scaling=state["scaling"])
    x, weight, residual = state["x"], state["weight"], state["residual"]
    if op == "norm":
        return ops.rms_norm(x, weight, EPS, residual=residual)
    if op == "norm_8bit":
        code = torch.float8_e4m3fn if state["code"] == "e4m3" else torch.int8
        group = state["group"] or None
        codes, scales, *total = ops.rms_norm_8bit(x, weight, EPS, residual=residual, dtype=code,
                                                  group=group)
        y = ops.dequantize_8bit(codes, scales, group=group, dtype=x.dtype)
        return (y, *total) if total else y
    if residual is None:
        y = ops.rms_norm(x, weight, EPS)
        return (y.detach(), *torch.autograd.grad(y, (x, weight), state["dy"]))
    y, total = ops.rms_norm(x, weight, EPS, residual=residual)
    grads = torch.autograd.grad((y, total), (x, residual, weight), (state["dy"], state["ds"]))
    return (y.detach(), total.detach(), *grads)


# ---- work ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "balance":
        n, t, e, k = (case[v] for v in ("groups", "tokens", "experts", "top_k"))
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": n * (t * (2 * e * size + 4 * k) + 4 * e), "flops": 10 * n * t * e}
    if op == "adapted":
        t, k, n, r, c = (case[v] for v in ("tokens", "inner", "outer", "adapters", "rank"))
        # adapters that are met when each request picks one of them or none
        met = r * (1.0 - (1.0 - 1.0 / (r + 1)) ** (case["runs"] or t))
        share = r / (r + 1.0)
        return {"bytes": int(2 * (t * k + n * k + t * n + met * c * (k + n)) + 4 * t),
                "flops": int(2 * t * k * n + 2 * share * t * c * (k + n))}
    rows, cols = case["rows"], case["cols"]
    size, res = DTYPES[case["dtype"]].itemsize, int(case["residual"])
    w = cols * (4 if case["weight"] == "fp32" else size)
    if op == "norm":
        return {"bytes": rows * cols * size * (2 + 2 * res) + w, "flops": 5 * rows * cols}
    if op == "norm_8bit":
        # codes and scales are written, read and written back as values
        blocks = -(-cols // (case["group"] or cols))
        return {"bytes": rows * cols * (size * (2 + 2 * res) + 2) + 8 * rows * blocks + w,
                "flops": 8 * rows * cols}
    # both inputs and both upstream gradients in, both outputs and one gradient out
    return {"bytes": rows * cols * size * (4 + 3 * res) + 2 * w, "flops": 14 * rows * cols}


# ---- from the definition, in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "balance":
            return _exact_balance(s)
        if case["op"] == "adapted":
            return _exact_adapted(s)
        x, r, w = s["x"], s["residual"], s["weight"].double()
        # (the stream is rounded before it is normed: that is part of the definition)
        t = (x if r is None else (x.double() + r.double()).to(x.dtype)).double()
        v = 1.0 / torch.sqrt(t.square().sum(-1, keepdim=True) / t.shape[1] + EPS)
        if case["op"] == "norm_8bit":
            y = _exact_8bit(t, w, v, s["code"], s["group"])
        else:
            y = t * w * v
        if case["op"] != "norm_grad":
            return y if r is None else (y, t)
        dy = s["dy"].double()
        hat = t * v
        dhat = dy * w
        dt = v * (dhat - hat * (dhat * hat).sum(-1, keepdim=True) / t.shape[1])
        dw = (dy * hat).sum(0)
        if r is None:
            return y, dt, dw
        dt = dt + s["ds"].double()
        return y, t, dt, dt, dw


def _exact_8bit(t, w, v, code, group):
    rows, cols = t.shape
    out = torch.empty_like(t)
    group = group or cols
    for c in range(0, cols, group):
        p = t[:, c:c + group] * w[c:c + group]
        top = p.abs().amax(-1, keepdim=True)
        if code == "int8":
            q = torch.round(127.0 * p / top)
            out[:, c:c + group] = q * (top * v / 127.0)
            continue
        m = (448.0 * p / top).abs()
        # 3 bits behind the leading one, down to multiples of 2^-9
        unit = torch.exp2(torch.floor(torch.log2(m.clamp(min=2.0 ** -6))) - 3.0)
        q = torch.round(m / unit) * unit
        out[:, c:c + group] = torch.copysign(q, p) * (top * v / 448.0)
    return torch.where(t == 0.0, 0.0, out)


def _exact_balance(s):
    logits, ids, mask, dloss = s["logits"], s["ids"], s["mask"], s["dloss"].double()
    n, t, e = logits.shape
    k = ids.shape[-1]
    loss = torch.zeros(n, dtype=torch.float64, device=logits.device)
    counts = torch.zeros(n, e, dtype=torch.int32, device=logits.device)
    grad = torch.zeros(n, t, e, dtype=torch.float64, device=logits.device)
    for i in range(n):
        rows = (torch.arange(t, device=logits.device) if mask is None
                else torch.nonzero(mask[i]).squeeze(1))
        if rows.numel() == 0:
            continue
        x = logits[i, rows].double()
        if s["scoring"] == "softmax":
            p = torch.softmax(x, -1)
        else:
            g = torch.sigmoid(x)
            p = g / g.sum(-1, keepdim=True)
        mine = ids[i, rows]
        counts[i] = (mine.reshape(-1, 1) == torch.arange(e, device=x.device)).sum(
            0) if mine.numel() * e < 1 << 28 else torch.bincount(
                mine[mine >= 0].long(), minlength=e).int()
        share = counts[i].double() / (k * rows.numel())
        loss[i] = e * (share * p.mean(0)).sum()
        d = p * (share - (p @ share).unsqueeze(-1))
        if s["scoring"] == "sigmoid":
            d = d * torch.sigmoid(-x)
        grad[i, rows] = d * (dloss[i] * e / rows.numel())
    return loss, counts, grad


def _exact_adapted(s):
    x, ids = s["x"].double(), s["ids"].long()
    y = x @ s["w"].double().mT
    for i in torch.unique(ids[ids >= 0]).tolist():
        delta = s["b"][i].double() @ s["a"][i].double() * s["scaling"][i].double()
        mine = (ids == i).unsqueeze(-1)
        if 2 * int(mine.sum()) > x.shape[0]:
            y = torch.where(mine, y + x @ delta.mT, y)
        else:
            rows = torch.nonzero(mine.squeeze(-1)).squeeze(1)
            y[rows] += x[rows] @ delta.mT
    return y
