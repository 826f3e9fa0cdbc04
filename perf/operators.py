"""Workloads of the microscaled 4-bit expert layer and the gated feed-forward block.

Four operators, each in its plain form (elementary torch operations in 32 bits, rounded once at
the end) and through the framework's entry points (exfold_b200.ops):

  quantize    MXFP4 quantisation of a matrix and reading it back: blocks of 32 values share a
              power of two, each value is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}
  experts     the SwiGLU expert layer over routed tokens with MXFP4 weights
  gated       the gated feed-forward block act(x Wg^T) * (x Wu^T)
  gated_grad  the same block in training: its output, dx and dW
"""

import math

import torch

own = False

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # activations of a small decode batch, where the launches are all of the time
        {"name": "quantize decode rows", "op": "quantize", "rows": 16, "cols": 2048,
         "dtype": "bf16"},
        # a ragged fp32 matrix: the last block of a row holds 4 values
        {"name": "quantize ragged fp32", "op": "quantize", "rows": 1021, "cols": 4100,
         "dtype": "fp32"},
        # the gate and up projections of one 128-expert layer (128 x 1536 rows), at load time
        {"name": "quantize layer weights", "op": "quantize", "rows": 196608, "cols": 2048,
         "dtype": "bf16"},
        # one token of one sequence: the weights of its 8 experts, nothing else
        {"name": "experts one token", "op": "experts", "tokens": 1, "experts": 128,
         "hidden": 2048, "inter": 768, "top_k": 8, "world": 1, "padding": 0.0},
        # the decode batch of the Qwen3 layer: every expert active, the weight stream bounds it
        {"name": "experts decode", "op": "experts", "tokens": 256, "experts": 128,
         "hidden": 2048, "inter": 768, "top_k": 8, "world": 1, "padding": 0.0},
        # one of 4 expert-parallel ranks of a 256-expert layer: it holds 64 experts, the routes
        # of the other ranks carry the id -1
        {"name": "experts decode rank of 4", "op": "experts", "tokens": 64, "experts": 64,
         "hidden": 4096, "inter": 2048, "top_k": 8, "world": 4, "padding": 0.0},
        # a prefill batch whose last tenth is padding (every route masked)
        {"name": "experts prefill padded", "op": "experts", "tokens": 8192, "experts": 128,
         "hidden": 2048, "inter": 768, "top_k": 8, "world": 1, "padding": 0.1},
        # the shared expert beside the routed ones, one token
        {"name": "gated one token", "op": "gated", "tokens": 1, "hidden": 2048, "inter": 768,
         "dtype": "bf16", "activation": "silu"},
        # odd sizes, no multiple of any tile
        {"name": "gated ragged fp16", "op": "gated", "tokens": 333, "hidden": 1000,
         "inter": 712, "dtype": "fp16", "activation": "gelu_tanh"},
        # the shared expert of a DeepSeek-style layer over a prefill batch
        {"name": "gated prefill", "op": "gated", "tokens": 8192, "hidden": 4096, "inter": 2048,
         "dtype": "bf16", "activation": "silu"},
        # a small ragged training micro-batch
        {"name": "gated_grad ragged fp16", "op": "gated_grad", "tokens": 777, "hidden": 1000,
         "inter": 520, "dtype": "fp16", "activation": "gelu_tanh"},
        # a training micro-batch of the DeepSeek-style block
        {"name": "gated_grad batch", "op": "gated_grad", "tokens": 8192, "hidden": 4096,
         "inter": 2048, "dtype": "bf16", "activation": "silu"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantize", "experts", "gated", "gated_grad"])
    if op == "quantize":
        cols = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(196608, 300_000_000 // cols))
        return {"op": op, "rows": rows, "cols": cols,
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "experts":
        hidden = 256 * rng.randint(1, 16)
        inter = 128 * rng.randint(1, 16)
        most = max(8, min(128, 1_600_000_000 // (3 * hidden * inter)))
        experts = _log_int(rng, 8, most)
        top_k = rng.randint(1, 8)
        tokens = _log_int(rng, 1, max(1, min(8192, 100_000_000_000 // (top_k * hidden * inter))))
        return {"op": op, "tokens": tokens, "experts": experts, "hidden": hidden, "inter": inter,
                "top_k": top_k, "world": rng.choice([1, 1, 2, 4]),
                "padding": rng.choice([0.0, 0.0, 0.1, 0.5])}
    hidden = 8 * _log_int(rng, 8, 512)
    inter = 8 * _log_int(rng, 8, 256)
    return {"op": op, "tokens": _log_int(rng, 1, 8192), "hidden": hidden, "inter": inter,
            "dtype": rng.choice(["bf16", "fp16"]),
            "activation": rng.choice(["silu", "gelu_tanh"])}


# ---- inputs -----------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "quantize":
        # rows of differing size, a few values far above the rest, a tenth of the rows empty
        rows, cols = case["rows"], case["cols"]
        x = torch.empty(rows, cols, dtype=DTYPES[case["dtype"]], device="cuda")
        step = max(1, (1 << 26) // cols)
        for r in range(0, rows, step):
            n = min(step, rows - r)
            v = torch.randn(n, cols, generator=g, device="cuda")
            size = torch.exp2(4.0 * torch.rand(n, 1, generator=g, device="cuda") - 6.0)
            empty = torch.rand(n, 1, generator=g, device="cuda") < 0.1
            far = torch.rand(n, cols, generator=g, device="cuda") < 0.001
            x[r:r + n] = torch.where(empty, 0.0, torch.where(far, 20.0 * v, v) * size)
        return {"op": op, "x": x}
    if op == "experts":
        t, e, h, i, k = (case[n] for n in ("tokens", "experts", "hidden", "inter", "top_k"))
        # the router's choice over the experts of every rank; this rank's are the first
        score = torch.randn(t, e * case["world"], generator=g, device="cuda")
        weight, ids = torch.softmax(score, -1).topk(k, -1)
        weight = weight / weight.sum(-1, keepdim=True)
        ids = torch.where(ids < e, ids, -1)
        ids[t - int(t * case["padding"]):] = -1
        w13, s13 = _packed_weights(e, 2 * i, h, g)
        w2, s2 = _packed_weights(e, h, i, g)
        return {"op": op, "x": torch.randn(t, h, generator=g, device="cuda").bfloat16(),
                "weight": weight.contiguous(), "ids": ids.int().contiguous(),
                "w13": w13, "s13": s13, "w2": w2, "s2": s2,
                # the scales as the framework's loader lays them out once (tile_mxfp4_scales)
                "t13": _tiled(s13), "t2": _tiled(s2)}
    t, h, i = case["tokens"], case["hidden"], case["inter"]
    dtype = DTYPES[case["dtype"]]
    state = {"op": op, "activation": case["activation"],
             "x": torch.randn(t, h, generator=g, device="cuda").to(dtype),
             "w13": (torch.randn(2 * i, h, generator=g, device="cuda") / math.sqrt(h)).to(dtype)}
    if op == "gated_grad":
        state["dh"] = torch.randn(t, i, generator=g, device="cuda").to(dtype)
        state["x"].requires_grad_(True)
        state["w13"].requires_grad_(True)
    return state


def _packed_weights(experts, rows, cols, g):
    """Normally distributed weights of every expert as MXFP4 codes and scales."""
    codes = torch.empty(experts, rows, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(experts, rows, cols // 32, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (rows * cols))
    for e in range(0, experts, step):
        w = torch.randn(min(step, experts - e), rows, cols, generator=g, device="cuda")
        codes[e:e + step], scales[e:e + step] = _encode(w / math.sqrt(cols))
    return codes, scales


def _tiled(scales):
    """[experts, rows, blocks] scales in tiles of 128 rows x 4 blocks: 512 bytes each, row r of
    a tile at byte 16 * (r % 32) + 4 * (r // 32)."""
    e, rows, blocks = scales.shape
    return (scales.view(e, rows // 128, 4, 32, blocks // 4, 4).permute(0, 1, 4, 3, 2, 5)
            .reshape(e, rows // 128, blocks // 4, 512).contiguous())


# ---- plain forms --------------------------------------------------------------------------------
def _power(e):
    """2^e as fp32, e in [-127, 127]."""
    normal = ((e + 127).clamp(min=1) << 23).view(torch.float32)
    return torch.where(e > -127, normal, 0.5 * normal)


def _encode(v):
    """fp32 [..., cols], cols a multiple of 32 -> (codes [..., cols / 2], scales [..., cols / 32]).
    The shared exponent is floor(log2(largest magnitude)) - 2; values round to the nearest
    representable one, ties to the even code, and saturate at 6."""
    b = v.reshape(*v.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = ((top.view(torch.int32) >> 23) - 129).clamp(min=-127)
    a = b.abs() * _power(-e)
    code = (a > 0.25).byte()
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5.0
    code += 8 * (b < 0).byte()
    code = code.reshape(*v.shape[:-1], -1, 2)
    return code[..., 0] + 16 * code[..., 1], (e + 127).byte().squeeze(-1)


def _decode(codes, scales):
    """The fp32 values of codes [..., n / 2] with scales [..., n / 32]."""
    low = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    pairs = torch.stack([low.repeat(16), low.repeat_interleave(16)], -1)
    v = torch.index_select(pairs, 0, codes.reshape(-1).int())
    v = v.reshape(*scales.shape, 32) * _power(scales.int() - 127).unsqueeze(-1)
    return v.reshape(*scales.shape[:-1], -1)


def _activate(g, activation):
    if activation == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _activate_slope(g, activation):
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    t = torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))
    inner = 0.7978845608028654 * (1.0 + 3.0 * 0.044715 * g * g)
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * inner


def _plain_quantize(s):
    x = s["x"]
    cols = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -cols % 32))
    return _decode(*_encode(v))[:, :cols].to(x.dtype)


def _plain_experts(s):
    """Every active expert's tokens padded to one length: three batched products."""
    x, ids = s["x"].float(), s["ids"].reshape(-1)
    tokens, k = s["ids"].shape
    active, place = torch.unique(ids.clamp(min=-1), return_inverse=True)
    order = torch.argsort(place, stable=True)
    count = torch.bincount(place, minlength=active.numel())
    start = torch.cumsum(count, 0) - count
    rank = torch.empty_like(place)
    rank[order] = torch.arange(order.numel(), device=x.device) - start[place[order]]
    first = int(active[0] < 0)  # the masked routes come first: they are left out
    real = torch.nonzero(ids >= 0).squeeze(1)
    y = torch.zeros_like(x)
    if real.numel() > 0:
        active = active[first:].long()
        at = (place[real] - first, rank[real])
        rows = x.new_zeros(active.numel(), int(count[first:].max()), x.shape[1])
        rows[at] = x[real // k]
        both = rows @ _decode(s["w13"][active], s["s13"][active]).transpose(1, 2)
        gate, up = both.chunk(2, -1)
        out = (_activate(gate, "silu") * up) @ _decode(s["w2"][active],
                                                       s["s2"][active]).transpose(1, 2)
        y.index_add_(0, real // k, out[at] * s["weight"].reshape(-1)[real].unsqueeze(1))
    return y.bfloat16()


def _plain_gated(s):
    gate, up = (s["x"].float() @ s["w13"].float().t()).chunk(2, -1)
    return (_activate(gate, s["activation"]) * up).to(s["x"].dtype)


def _plain_gated_grad(s):
    x, w, dh, dtype = s["x"].float(), s["w13"].float(), s["dh"].float(), s["x"].dtype
    gate, up = (x @ w.t()).chunk(2, -1)
    act = _activate(gate, s["activation"])
    both = torch.cat([dh * up * _activate_slope(gate, s["activation"]), dh * act], -1)
    return (act * up).to(dtype), (both @ w).to(dtype), (both.t() @ x).to(dtype)


PLAIN = {"quantize": _plain_quantize, "experts": _plain_experts, "gated": _plain_gated,
         "gated_grad": _plain_gated_grad}


def run(state):
    op = state["op"]
    if not own:
        with torch.no_grad():
            return PLAIN[op](state)
    import sys

    if "exfold-moe_b200" not in sys.path:
        sys.path.insert(0, "exfold-moe_b200")
    from exfold_b200 import ops

    if op == "quantize":
        x = state["x"]
        codes, scales = ops.quantize_mxfp4(x)
        return ops.dequantize_mxfp4(codes, scales, cols=x.shape[-1], dtype=x.dtype)
    if op == "experts":
        return ops.fused_experts_mxfp4(state["x"], state["weight"], state["ids"], state["w13"],
                                       state["t13"], state["w2"], state["t2"])
    if op == "gated":
        return ops.gated_mlp(state["x"], state["w13"], activation=state["activation"])
    x, w13 = state["x"], state["w13"]
    h = ops.gated_mlp(x, w13, activation=state["activation"])
    dx, dw13 = torch.autograd.grad(h, (x, w13), state["dh"])
    return h.detach(), dx, dw13


# ---- work ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        blocks = case["rows"] * -(-case["cols"] // 32)
        size = DTYPES[case["dtype"]].itemsize
        # values read and written back, 17 bytes for each block written and read
        return {"bytes": 2 * n * size + 2 * 17 * blocks, "flops": 2 * n}
    if op == "experts":
        t, h, i, k = (case[n] for n in ("tokens", "hidden", "inter", "top_k"))
        real = (t - int(t * case["padding"])) * k / case["world"]
        # experts that are met at least once when each route picks one of them
        active = case["experts"] * (1.0 - (1.0 - 1.0 / case["experts"]) ** real)
        return {"bytes": int(active * 3 * h * i * 17 / 32 + 4 * t * h + 8 * t * k),
                "flops": int(6 * real * h * i)}
    t, h, i = case["tokens"], case["hidden"], case["inter"]
    if op == "gated":
        return {"bytes": 2 * (t * h + 2 * i * h + t * i), "flops": 4 * t * h * i}
    return {"bytes": 2 * (2 * t * h + 4 * i * h + 2 * t * i), "flops": 12 * t * h * i}


# ---- from the definition, in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "quantize":
            return _exact_quantize(s["x"])
        if case["op"] == "experts":
            return _exact_experts(s)
        x, w = s["x"].double(), s["w13"].double()
        i = w.shape[0] // 2
        g, u = x @ w[:i].mT, x @ w[i:].mT
        if s["activation"] == "silu":
            a = g * torch.sigmoid(g)
            slope = torch.sigmoid(g) + a * torch.sigmoid(-g)
        else:
            c = math.sqrt(2.0 / math.pi)
            z = c * g + c * 0.044715 * g.pow(3)
            a = g * torch.sigmoid(2.0 * z)
            slope = torch.sigmoid(2.0 * z) + g * torch.sigmoid(2.0 * z) * torch.sigmoid(
                -2.0 * z) * 2.0 * (c + 3.0 * c * 0.044715 * g.pow(2))
        if case["op"] == "gated":
            return a * u
        dh = s["dh"].double()
        dg, du = dh * u * slope, dh * a
        return (a * u, dg @ w[:i] + du @ w[i:], torch.cat([dg.mT @ x, du.mT @ x]))


def _exact_quantize(x):
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    step = max(1, (1 << 26) // cols)
    for r in range(0, rows, step):
        v = torch.nn.functional.pad(x[r:r + step].double(), (0, -cols % 32))
        v = v.reshape(v.shape[0], -1, 32)
        _, e = torch.frexp(v.abs().amax(-1, keepdim=True))
        share = torch.exp2((e - 3).clamp(min=-127).double())
        a = (v / share).abs()
        grid = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
        a = (torch.round(a / grid) * grid).clamp(max=6.0) * share
        out[r:r + step] = torch.copysign(a, v).reshape(v.shape[0], -1)[:, :cols]
    return out


def _exact_weights(codes, scales):
    half = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    m = (half & 7).double()
    v = torch.where(m < 4, 0.5 * m, torch.where(m < 6, m - 2.0, 2.0 * m - 8.0))
    v = torch.where(half > 7, -v, v)
    return v * torch.exp2(scales.double() - 127.0).repeat_interleave(32, -1)


def _exact_experts(s):
    x = s["x"].double()
    y = torch.zeros_like(x)
    for e in range(s["w13"].shape[0]):
        token, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel() == 0:
            continue
        w1, w3 = _exact_weights(s["w13"][e], s["s13"][e]).chunk(2, 0)
        g = x[token] @ w1.mT
        h = g * torch.sigmoid(g) * (x[token] @ w3.mT)
        o = h @ _exact_weights(s["w2"][e], s["s2"][e]).mT
        y.index_add_(0, token, o * s["weight"][token, slot].double().unsqueeze(1))
    return y
