"""torch front end of libexfold_b200.so.

Each function allocates its outputs with torch (so CUDA-graph capture uses the graph's memory
pool), passes raw device pointers to the C ABI and launches on the current CUDA stream.  Nothing
here synchronises with the host.  Weights are float32 / bfloat16 / float16 and ids int32 /
int64 natively; other dtypes are converted on the way in and back on the way out.
"""

from __future__ import annotations

import contextlib
import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib as L

_WDT = {torch.float32: L.EXF_F32, torch.bfloat16: L.EXF_BF16, torch.float16: L.EXF_F16}
_IDT = {torch.int32: L.EXF_I32, torch.int64: L.EXF_I64}
_SCORING = {"softmax": L.EXF_SOFTMAX, "sigmoid": L.EXF_SIGMOID, "sqrtsoftplus": L.EXF_SQRTSOFTPLUS}
_ACTIVATION = {"silu": L.EXF_SILU, "gelu_tanh": L.EXF_GELU_TANH}
_VARIANT = {"qwen3": L.EXF_QWEN3, "dsv4": L.EXF_DSV4}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> ctypes.c_void_p:
    # the raw handle: a torch.cuda.Stream object for it would cost 2 us a call
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(device.index))


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """Makes `device` current for a launch (nothing to do, and nothing spent, where it is)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("ExFold B200 ops require CUDA tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("ExFold B200 ops require all tensors on one device")
    return dev


def _f32c(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None:
        return None
    return t.contiguous() if t.dtype == torch.float32 else t.float().contiguous()


def _logits_in(t: torch.Tensor) -> torch.Tensor:
    """Router logits in their own dtype when it is fp32 / bf16 / fp16 (the kernels convert
    16-bit logits exactly), else as fp32; contiguous and 16-byte aligned."""
    t = t if t.dtype in _WDT else t.float()
    return _aligned(t)


def _aligned(t: torch.Tensor, to: int = 16) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % to == 0 else t.clone()


def _weights_in(w: torch.Tensor) -> torch.Tensor:
    return w.contiguous() if w.dtype in _WDT else w.float().contiguous()


def _ids_in(ids: torch.Tensor) -> torch.Tensor:
    return ids.contiguous() if ids.dtype in _IDT else ids.to(torch.int32).contiguous()


# ---- router ---------------------------------------------------------------------------------
def router_topk(logits: torch.Tensor, top_k: int, scoring: str = "softmax",
                bias: torch.Tensor | None = None, renormalize: bool = True,
                scaling: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Top-k routing of [tokens, experts] logits (fp32, bf16 or fp16 natively) -> (weights fp32,
    ids int32) [tokens, top_k]."""
    dev = _require_cuda(logits, bias)
    x = _logits_in(logits)
    tokens, experts = x.shape
    b = None if bias is None else _aligned(_f32c(bias))
    w = torch.empty((tokens, top_k), dtype=torch.float32, device=dev)
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=dev)
    L.check(L.lib().exf_router_topk(x.data_ptr(), _WDT[x.dtype], tokens, experts, top_k,
                                    _SCORING[scoring],
                                    _ptr(b), int(renormalize), float(scaling), w.data_ptr(),
                                    ids.data_ptr(), _stream(dev)))
    return w, ids


def router_hash(logits: torch.Tensor, token_ids: torch.Tensor, table: torch.Tensor,
                scoring: str = "sqrtsoftplus", renormalize: bool = True,
                scaling: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Hash routing: routes table[token_ids] (table [rows, top_k], in table order) weighted by
    the unbiased scores of those experts -> (weights fp32, ids int32) [tokens, top_k]."""
    dev = _require_cuda(logits, token_ids, table)
    x = _logits_in(logits)
    tokens, experts = x.shape
    tid = _ids_in(token_ids.reshape(-1))
    if tid.numel() != tokens:
        raise ValueError(f"token_ids has {tid.numel()} entries for {tokens} tokens")
    tab = table.to(torch.int32).contiguous()
    if tab.dim() != 2:
        raise ValueError("table must be [rows, top_k]")
    top_k = tab.shape[1]
    w = torch.empty((tokens, top_k), dtype=torch.float32, device=dev)
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=dev)
    L.check(L.lib().exf_router_hash(x.data_ptr(), _WDT[x.dtype], tokens, experts, top_k,
                                    _SCORING[scoring],
                                    tid.data_ptr(), _IDT[tid.dtype], tab.data_ptr(), tab.shape[0],
                                    int(renormalize), float(scaling), w.data_ptr(), ids.data_ptr(),
                                    _stream(dev)))
    return w, ids


def router_fold_prefill(logits: torch.Tensor, top_k: int, target_k: int, coeff: torch.Tensor,
                        sel_loss: torch.Tensor, *, scoring: str = "softmax",
                        bias: torch.Tensor | None = None, renormalize: bool = True,
                        scaling: float = 1.0, variant: str = "qwen3", renorm_mode: int = 0,
                        conf_loss: torch.Tensor | None = None,
                        out: tuple[torch.Tensor, torch.Tensor] | None = None,
                        ) -> tuple[torch.Tensor, torch.Tensor]:
    """Router + prefill fold in one pass.

    logits [tokens, E] with tables [E, E], or [layers, tokens, E] with tables [layers, E, E]
    (and bias [layers, E]).  Returns (weights fp32, ids int32) [..., tokens, target_k].
    """
    dev = _require_cuda(logits, coeff, sel_loss, bias, conf_loss)
    x = _logits_in(logits)
    layers = 1 if x.dim() == 2 else x.shape[0]
    tokens, experts = x.shape[-2], x.shape[-1]
    coeff, sel_loss = _f32c(coeff), _f32c(sel_loss)
    conf_loss = _f32c(conf_loss)
    b = None if bias is None else _aligned(_f32c(bias))
    shape = (*x.shape[:-1], target_k)
    if out is None:
        w = torch.empty(shape, dtype=torch.float32, device=dev)
        ids = torch.empty(shape, dtype=torch.int32, device=dev)
    else:
        w, ids = out
    L.check(L.lib().exf_router_fold_prefill(
        x.data_ptr(), _WDT[x.dtype], tokens, layers, experts, top_k, _SCORING[scoring], _ptr(b),
        int(renormalize), float(scaling), target_k, _VARIANT[variant], int(renorm_mode),
        coeff.data_ptr(), sel_loss.data_ptr(), _ptr(conf_loss), w.data_ptr(), ids.data_ptr(),
        _stream(dev)))
    return w, ids


# ---- prefill fold of given routes -------------------------------------------------------------
def router_tile_min_rows(rows: int | None = None) -> int:
    """The launch size (tokens x layers) from which the router calls use the tile kernels
    (exf_router_tile_min_rows): smaller launches take the generic kernel, whose latency is lower
    there; both give identical results.  Sets it when `rows` is given; returns the previous value."""
    return int(L.lib().exf_router_tile_min_rows(-1 if rows is None else int(rows)))


def fold_prefill(weights: torch.Tensor, ids: torch.Tensor, coeff: torch.Tensor,
                 sel_loss: torch.Tensor, target_k: int, *, variant: str = "qwen3",
                 renorm_mode: int = 0, conf_loss: torch.Tensor | None = None,
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    dev = _require_cuda(weights, ids, coeff, sel_loss, conf_loss)
    w_in, i_in = _weights_in(weights), _ids_in(ids)
    tokens, top_k = w_in.shape
    coeff, sel_loss, conf_loss = _f32c(coeff), _f32c(sel_loss), _f32c(conf_loss)
    ow = torch.empty((tokens, target_k), dtype=w_in.dtype, device=dev)
    oi = torch.empty((tokens, target_k), dtype=i_in.dtype, device=dev)
    if tokens > 0:
        L.check(L.lib().exf_fold_prefill(
            w_in.data_ptr(), _WDT[w_in.dtype], i_in.data_ptr(), _IDT[i_in.dtype], tokens, top_k,
            target_k, coeff.shape[0], _VARIANT[variant], int(renorm_mode), coeff.data_ptr(),
            sel_loss.data_ptr(), _ptr(conf_loss), ow.data_ptr(), oi.data_ptr(), _stream(dev)))
    return ow.to(weights.dtype), oi.to(ids.dtype)


# ---- decode ---------------------------------------------------------------------------------
def decode(weights: torch.Tensor, ids: torch.Tensor, norms: torch.Tensor, coeff: torch.Tensor,
           loss: torch.Tensor, budget: int, *, variant: str = "qwen3",
           subset_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Importance, top-`budget` select, target table and apply in one launch."""
    dev = _require_cuda(weights, ids, norms, coeff, loss)
    w_in, i_in = _weights_in(weights), _ids_in(ids)
    batch, top_k = w_in.shape
    norms, coeff, loss = _f32c(norms), _f32c(coeff), _f32c(loss)
    ow, oi = torch.empty_like(w_in), torch.empty_like(i_in)
    L.check(L.lib().exf_decode(
        w_in.data_ptr(), _WDT[w_in.dtype], i_in.data_ptr(), _IDT[i_in.dtype], batch, top_k,
        coeff.shape[0], int(budget), _VARIANT[variant], norms.data_ptr(), coeff.data_ptr(),
        loss.data_ptr(), ow.data_ptr(), oi.data_ptr(), _ptr(subset_out), _stream(dev)))
    return ow.to(weights.dtype), oi.to(ids.dtype)


def decode_importance(weights: torch.Tensor, ids: torch.Tensor, norms: torch.Tensor,
                      importance: torch.Tensor) -> torch.Tensor:
    """Add this shard's fixed-point importance into `importance` (int64 [E], caller-zeroed)."""
    dev = _require_cuda(weights, ids, norms, importance)
    if importance.dtype != torch.int64 or not importance.is_contiguous():
        raise ValueError("importance must be a contiguous int64 vector")
    w_in, i_in = _weights_in(weights), _ids_in(ids)
    norms = _f32c(norms)
    L.check(L.lib().exf_decode_importance(
        w_in.data_ptr(), _WDT[w_in.dtype], i_in.data_ptr(), _IDT[i_in.dtype], w_in.numel(),
        norms.numel(), norms.data_ptr(), importance.data_ptr(), _stream(dev)))
    return importance


def decode_apply(importance: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor,
                 coeff: torch.Tensor, loss: torch.Tensor, budget: int, *, variant: str = "qwen3",
                 subset_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Select / table / apply from an (all-reduced) importance vector."""
    dev = _require_cuda(importance, weights, ids, coeff, loss)
    w_in, i_in = _weights_in(weights), _ids_in(ids)
    batch, top_k = w_in.shape
    coeff, loss = _f32c(coeff), _f32c(loss)
    ow, oi = torch.empty_like(w_in), torch.empty_like(i_in)
    L.check(L.lib().exf_decode_apply(
        importance.data_ptr(), w_in.data_ptr(), _WDT[w_in.dtype], i_in.data_ptr(),
        _IDT[i_in.dtype], batch, top_k, coeff.shape[0], int(budget), _VARIANT[variant],
        coeff.data_ptr(), loss.data_ptr(), ow.data_ptr(), oi.data_ptr(), _ptr(subset_out),
        _stream(dev)))
    return ow.to(weights.dtype), oi.to(ids.dtype)


def decode_sharded(weights: torch.Tensor, ids: torch.Tensor, norms: torch.Tensor,
                   coeff: torch.Tensor, loss: torch.Tensor, budget: int, *, world: int, rank: int,
                   peers: "ctypes.Array", variant: str = "qwen3",
                   status: torch.Tensor | None = None, wait_ns: int = 0,
                   subset_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Decode budget of this rank's shard in one launch, the importance exchanged with the other
    ranks over peer memory (`peers`: every rank's exchange buffer as mapped here, a ctypes array
    of `world` device pointers; see `exfold_b200.parallel.DecodeExchange`)."""
    dev = _require_cuda(weights, ids, norms, coeff, loss, status)
    w_in, i_in = _weights_in(weights), _ids_in(ids)
    batch, top_k = w_in.shape
    norms, coeff, loss = _f32c(norms), _f32c(coeff), _f32c(loss)
    ow, oi = torch.empty_like(w_in), torch.empty_like(i_in)
    L.check(L.lib().exf_decode_sharded(
        w_in.data_ptr(), _WDT[w_in.dtype], i_in.data_ptr(), _IDT[i_in.dtype], batch, top_k,
        coeff.shape[0], int(budget), _VARIANT[variant], norms.data_ptr(), coeff.data_ptr(),
        loss.data_ptr(), int(world), int(rank), peers, int(wait_ns), ow.data_ptr(), oi.data_ptr(),
        _ptr(subset_out), _ptr(status), _stream(dev)))
    return ow.to(weights.dtype), oi.to(ids.dtype)


def reroute_subset(weights: torch.Tensor, ids: torch.Tensor, subset: torch.Tensor,
                   coeff: torch.Tensor, loss: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    dev = _require_cuda(weights, ids, subset, coeff, loss)
    w_in, i_in = _weights_in(weights), _ids_in(ids)
    batch, top_k = w_in.shape
    sub = subset.to(torch.int32).contiguous()
    coeff, loss = _f32c(coeff), _f32c(loss)
    ow, oi = torch.empty_like(w_in), torch.empty_like(i_in)
    L.check(L.lib().exf_reroute_subset(
        w_in.data_ptr(), _WDT[w_in.dtype], i_in.data_ptr(), _IDT[i_in.dtype], batch, top_k,
        coeff.shape[0], sub.data_ptr(), sub.numel(), coeff.data_ptr(), loss.data_ptr(),
        ow.data_ptr(), oi.data_ptr(), _stream(dev)))
    return ow.to(weights.dtype), oi.to(ids.dtype)


def static_table(norms: torch.Tensor, coeff: torch.Tensor, loss: torch.Tensor,
                 budget: int) -> tuple[torch.Tensor, torch.Tensor]:
    dev = _require_cuda(norms, coeff, loss)
    norms, coeff, loss = _f32c(norms), _f32c(coeff), _f32c(loss)
    experts = norms.numel()
    target = torch.empty(experts, dtype=torch.int32, device=dev)
    scale = torch.empty(experts, dtype=torch.float32, device=dev)
    L.check(L.lib().exf_static_table(norms.data_ptr(), coeff.data_ptr(), loss.data_ptr(), experts,
                                     int(budget), target.data_ptr(), scale.data_ptr(),
                                     _stream(dev)))
    return target, scale


def static_remap_(weights: torch.Tensor, ids: torch.Tensor, target: torch.Tensor,
                  scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """In place: ids = target[ids], weights *= scale[ids] (contiguous natively-typed tensors)."""
    dev = _require_cuda(weights, ids, target, scale)
    if weights.dtype not in _WDT or ids.dtype not in _IDT:
        raise TypeError("static_remap_ needs float32/bfloat16/float16 weights and int32/int64 ids")
    if not (weights.is_contiguous() and ids.is_contiguous()):
        raise ValueError("static_remap_ works in place on contiguous tensors")
    t = target.to(torch.int32).contiguous()
    s = _f32c(scale)
    if weights.numel() > 0:
        L.check(L.lib().exf_static_remap(weights.data_ptr(), _WDT[weights.dtype], ids.data_ptr(),
                                         _IDT[ids.dtype], weights.numel(), t.numel(), t.data_ptr(),
                                         s.data_ptr(), _stream(dev)))
    return weights, ids


# ---- moe_align ------------------------------------------------------------------------------
def moe_align_capacity(numel: int, experts: int, block_size: int, pad_sorted: bool = False) -> int:
    return int(L.lib().exf_moe_align_capacity(numel, experts, block_size, int(pad_sorted)))


def moe_align_block_size(topk_ids: torch.Tensor, block_size: int, num_experts: int,
                         pad_sorted_ids: bool = False,
                         ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(sorted_token_ids, expert_ids, num_tokens_post_padded) as vLLM's moe_align_block_size."""
    dev = _require_cuda(topk_ids)
    ids = _ids_in(topk_ids)
    numel = ids.numel()
    cap = moe_align_capacity(numel, num_experts, block_size, pad_sorted_ids)
    sorted_ids = torch.empty(cap, dtype=torch.int32, device=dev)
    expert_ids = torch.empty((cap + block_size - 1) // block_size, dtype=torch.int32, device=dev)
    post = torch.empty(1, dtype=torch.int32, device=dev)
    ws_bytes = int(L.lib().exf_moe_align_workspace_bytes(numel, num_experts))
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    L.check(L.lib().exf_moe_align(ids.data_ptr(), _IDT[ids.dtype], numel, num_experts, block_size,
                                  cap, sorted_ids.data_ptr(), expert_ids.data_ptr(),
                                  post.data_ptr(), ws.data_ptr(), ws_bytes, _stream(dev)))
    return sorted_ids, expert_ids, post


# ---- grouped SwiGLU experts (tcgen05) ------------------------------------------------------------
def decode_fused_experts(x: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor,
                         norms: torch.Tensor, coeff: torch.Tensor, loss: torch.Tensor, budget: int,
                         w13: torch.Tensor, w2: torch.Tensor, *, variant: str = "qwen3",
                         status: torch.Tensor | None = None
                         ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Decode expert budget, then the expert layer over the remapped routes: returns
    (y, w_out, ids_out).

    `decode` followed by `fused_experts`, with moe_align done inside the decode launch and the
    routes of a token that the budget sends to the same expert merged (weights summed, the
    expert computed once).  w_out / ids_out equal `decode`'s outputs bit for bit (fp32 / int32);
    y equals `fused_experts(x, w_out, ids_out, w13, w2)` within bf16 rounding.  At most 256
    experts, top_k <= 8 and 8192 routes.
    """
    dev = _require_cuda(x, weights, ids, norms, coeff, loss, w13, w2)
    if x.dtype != torch.bfloat16 or w13.dtype != torch.bfloat16 or w2.dtype != torch.bfloat16:
        raise TypeError("decode_fused_experts computes in bf16: x, w13 and w2 must be bfloat16")
    x, w13, w2 = x.contiguous(), w13.contiguous(), w2.contiguous()
    w_in = weights.float().contiguous()
    i_in = ids.to(torch.int32).contiguous()
    batch, top_k = w_in.shape
    hidden = x.shape[1]
    experts, two_i, _ = w13.shape
    inter = two_i // 2
    norms, coeff, loss = _f32c(norms), _f32c(coeff), _f32c(loss)
    ow, oi = torch.empty_like(w_in), torch.empty_like(i_in)
    y = torch.empty_like(x)
    ws_bytes = int(L.lib().exf_decode_fused_experts_workspace_bytes(batch, top_k, experts,
                                                                    hidden, inter))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
    L.check(L.lib().exf_decode_fused_experts(
        x.data_ptr(), w_in.data_ptr(), i_in.data_ptr(), batch, top_k, experts, int(budget),
        _VARIANT[variant], norms.data_ptr(), coeff.data_ptr(), loss.data_ptr(), w13.data_ptr(),
        w2.data_ptr(), hidden, inter, ow.data_ptr(), oi.data_ptr(), y.data_ptr(), ws.data_ptr(),
        ws_bytes, _ptr(status), _stream(dev)))
    return y, ow, oi


def fused_experts(x: torch.Tensor, topk_w: torch.Tensor, topk_ids: torch.Tensor,
                  w13: torch.Tensor, w2: torch.Tensor,
                  status: torch.Tensor | None = None) -> torch.Tensor:
    """y = sum_j topk_w[:, j] * W2[e] (silu(W1[e] x) * (W3[e] x)), e = topk_ids[:, j].

    x bf16 [T, H]; w13 bf16 [E, 2I, H] (gate rows then up rows); w2 bf16 [E, H, I].  The layout
    and meaning follow vLLM's fused_experts.  `status` (int32 [1] on the device) is set to 1 if a
    pipeline wait timed out.
    """
    dev = _require_cuda(x, topk_w, topk_ids, w13, w2)
    if x.dtype != torch.bfloat16 or w13.dtype != torch.bfloat16 or w2.dtype != torch.bfloat16:
        raise TypeError("fused_experts computes in bf16: x, w13 and w2 must be bfloat16")
    x, w13, w2 = x.contiguous(), w13.contiguous(), w2.contiguous()
    tokens, hidden = x.shape
    experts, two_i, _ = w13.shape
    inter = two_i // 2
    top_k = topk_ids.shape[1]
    ids = topk_ids.to(torch.int32).contiguous()
    wts = topk_w.float().contiguous()
    y = torch.empty_like(x)
    ws_bytes = int(L.lib().exf_fused_experts_workspace_bytes(tokens, top_k, experts, hidden,
                                                             inter))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
    L.check(L.lib().exf_fused_experts(x.data_ptr(), wts.data_ptr(), ids.data_ptr(), tokens, top_k,
                                      w13.data_ptr(), w2.data_ptr(), experts, hidden, inter,
                                      y.data_ptr(), ws.data_ptr(), ws_bytes, _ptr(status),
                                      _stream(dev)))
    return y


def _status_ptr(status: torch.Tensor | None) -> int | None:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1:
        raise TypeError("status must be an int32 tensor of one element")
    return status.data_ptr()


# ---- microscaled 4-bit floating point -----------------------------------------------------------
def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """MXFP4 form of x [..., cols] (fp32, bf16 or fp16): codes uint8 [..., 16 * blocks] and scales
    uint8 [..., blocks], blocks = ceil(cols / 32).

    A block of 32 values along the last dimension shares the power of two 2^(scale - 127), the
    largest at which its largest magnitude is at least 4; a value is the nearest of +-{0, 0.5, 1,
    1.5, 2, 3, 4, 6} times it (ties to the even code, saturating at 6), two codes a byte, the even
    column in the low half.  A block holding an infinity or a NaN reads back as NaN.
    """
    dev = _require_cuda(x)
    if x.dtype not in _WDT:
        raise TypeError("quantize_mxfp4 needs a float32, bfloat16 or float16 tensor")
    if x.dim() == 0:
        raise ValueError("quantize_mxfp4 needs at least one dimension")
    cols = x.shape[-1]
    blocks = (cols + 31) // 32
    # rows at a constant distance are read where they lie
    if not (x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= cols):
        x = x.contiguous()
    stride = x.stride(0) if x.dim() == 2 and x.shape[0] > 1 else cols
    lead = x.shape[:-1]
    codes = torch.empty(*lead, 16 * blocks, dtype=torch.uint8, device=dev)
    scales = torch.empty(*lead, blocks, dtype=torch.uint8, device=dev)
    n = x.numel()
    if n > 0:
        with _on(dev):
            L.check(L.lib().exf_mxfp4_quantize(x.data_ptr(), _WDT[x.dtype], n // cols, cols,
                                               stride, codes.data_ptr(), scales.data_ptr(),
                                               _stream(dev)))
    return codes, scales


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, cols: int | None = None,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of quantize_mxfp4's codes and scales as dtype [..., cols] (default: every column
    of the blocks)."""
    dev = _require_cuda(codes, scales)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError("dequantize_mxfp4 needs uint8 codes and scales")
    if dtype not in _WDT:
        raise TypeError("dequantize_mxfp4 gives float32, bfloat16 or float16")
    lead, blocks = scales.shape[:-1], scales.shape[-1] if scales.dim() else 0
    if codes.dim() == 0 or codes.shape[:-1] != lead or codes.shape[-1] != 16 * blocks:
        raise ValueError(f"codes {tuple(codes.shape)} do not match scales {tuple(scales.shape)}: "
                         "16 bytes a block")
    cols = 32 * blocks if cols is None else int(cols)
    if cols < 0 or (cols + 31) // 32 != blocks:
        raise ValueError(f"{cols} columns do not take {blocks} blocks of 32")
    codes, scales = _aligned(codes), scales.contiguous()
    out = torch.empty(*lead, cols, dtype=dtype, device=dev)
    n = out.numel()
    if n > 0:
        with _on(dev):
            L.check(L.lib().exf_mxfp4_dequantize(codes.data_ptr(), scales.data_ptr(), n // cols,
                                                 cols, out.data_ptr(), _WDT[dtype],
                                                 _stream(dev)))
    return out


def tile_mxfp4_scales(scales: torch.Tensor) -> torch.Tensor:
    """The scales [experts, rows, blocks] of expert weights in the layout `fused_experts_mxfp4` reads,
    [experts, rows / 128, blocks / 4, 512]: tiles of 128 rows x 4 blocks, row r of a tile at byte
    16 * (r % 32) + 4 * (r // 32).  Done once, when the weights are loaded."""
    if scales.dtype != torch.uint8:
        raise TypeError("tile_mxfp4_scales needs uint8 scales")
    if scales.dim() != 3 or scales.shape[1] % 128 or scales.shape[2] % 4:
        raise ValueError(f"scales {tuple(scales.shape)} must be [experts, rows, blocks], rows a "
                         "multiple of 128 and blocks of 4")
    e, rows, blocks = scales.shape
    return (scales.reshape(e, rows // 128, 4, 32, blocks // 4, 4).permute(0, 1, 4, 3, 2, 5)
            .reshape(e, rows // 128, blocks // 4, 512).contiguous())


def _expert_ids(ids: torch.Tensor, experts: int) -> torch.Tensor:
    """Integer ids of any width as int32; what lies outside [0, experts) stays outside."""
    if ids.dtype is torch.int32:
        return ids
    if ids.is_floating_point() or ids.is_complex() or ids.dtype is torch.bool:
        raise TypeError(f"expert ids must be integers, got {ids.dtype}")
    # (clamped in 64 bits: -1 is 255 in uint8, and experts may not fit the narrow types)
    return ids.to(torch.int64).clamp(-1, experts).to(torch.int32)


def fused_experts_mxfp4(x: torch.Tensor, topk_w: torch.Tensor, topk_ids: torch.Tensor,
                        w13: torch.Tensor, s13: torch.Tensor, w2: torch.Tensor, s2: torch.Tensor,
                        status: torch.Tensor | None = None) -> torch.Tensor:
    """`fused_experts` with MXFP4 weights: y = sum_j topk_w[:, j] * W2[e] (silu(W1[e] x) *
    (W3[e] x)), e = topk_ids[:, j]; ids outside [0, E) contribute nothing.

    x bf16 [T, H].  w13 uint8 [E, 2I, H / 2] (gate rows then up rows) and w2 uint8 [E, H, I / 2] are
    `quantize_mxfp4`'s codes, s13 and s2 its scales after `tile_mxfp4_scales`; topk_ids integers of
    any width.  Activations keep bf16 precision (two 8-bit terms each, or fp16 ones for a few routes);
    sums are fp32.  H is a multiple of 256, I of 128, top_k <= 8.  `status` as in `fused_experts`.
    For inference: like `fused_experts`, the result carries no gradient.
    """
    dev = _require_cuda(x, topk_w, topk_ids, w13, s13, w2, s2, status)
    if x.dtype is not torch.bfloat16:
        raise TypeError("fused_experts_mxfp4 needs bfloat16 activations")
    u8 = torch.uint8
    if not (w13.dtype is u8 and s13.dtype is u8 and w2.dtype is u8 and s2.dtype is u8):
        raise TypeError("fused_experts_mxfp4 needs uint8 codes and scales")
    if x.dim() != 2 or topk_ids.dim() != 2 or w13.dim() != 3:
        raise ValueError("x must be [T, H], topk_ids [T, top_k] and w13 [E, 2I, H / 2]")
    tokens, hidden = x.shape
    experts, two_i, _ = w13.shape
    inter, top_k = two_i // 2, topk_ids.shape[1]
    if topk_ids.shape[0] != tokens or topk_w.shape != topk_ids.shape:
        raise ValueError(f"routes {tuple(topk_w.shape)}, {tuple(topk_ids.shape)} do not match "
                         f"{tokens} tokens")
    if two_i % 2 or hidden % 256 or inter % 128:
        raise NotImplementedError("fused_experts_mxfp4: hidden must be a multiple of 256 and "
                                  "intermediate a multiple of 128")
    if (w13.shape != (experts, two_i, hidden // 2)
            or s13.shape != (experts, two_i // 128, hidden // 128, 512)
            or w2.shape != (experts, hidden, inter // 2)
            or s2.shape != (experts, hidden // 128, inter // 128, 512)):
        raise ValueError(
            f"for {experts} experts, hidden {hidden} and intermediate {inter}, w13, s13, w2 and s2 "
            f"are {tuple(w13.shape)}, {tuple(s13.shape)}, {tuple(w2.shape)}, {tuple(s2.shape)}")
    x, w13, s13 = _aligned(x), _aligned(w13, 32), _aligned(s13)
    w2, s2 = _aligned(w2, 32), _aligned(s2)
    topk_ids = _expert_ids(topk_ids, experts)
    if topk_w.dtype is not torch.float32:
        topk_w = topk_w.float()
    ids, wts = topk_ids.contiguous(), topk_w.contiguous()
    y = torch.empty_like(x)
    if tokens == 0:
        return y
    lib = L.lib()
    ws_bytes = lib.exf_fused_experts_mxfp4_workspace_bytes(tokens, top_k, experts, hidden, inter)
    ws = torch.empty(ws_bytes if ws_bytes > 32 else 32, dtype=u8, device=dev)
    with _on(dev):
        L.check(lib.exf_fused_experts_mxfp4(
            x.data_ptr(), wts.data_ptr(), ids.data_ptr(), tokens, top_k, w13.data_ptr(),
            s13.data_ptr(), w2.data_ptr(), s2.data_ptr(), experts, hidden, inter, y.data_ptr(),
            ws.data_ptr(), ws_bytes, _status_ptr(status), _stream(dev)))
    return y


# ---- gated feed-forward block ---------------------------------------------------------------------
def _gated_forward(x, w13, activation, status, keep):
    """(h, pre): pre fp32 [tokens, 2 * inter] for the backward pass if `keep`, else None."""
    tokens, hidden = x.shape
    inter = w13.shape[0] // 2
    dev = x.device
    h = torch.empty(tokens, inter, dtype=x.dtype, device=dev)
    pre = torch.empty(tokens, 2 * inter, dtype=torch.float32, device=dev) if keep else None
    with _on(dev):
        ws_bytes = L.lib().exf_gated_mlp_workspace_bytes(tokens, hidden, inter)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
        L.check(L.lib().exf_gated_mlp(x.data_ptr(), w13.data_ptr(), _WDT[x.dtype], tokens, hidden,
                                      inter, activation, h.data_ptr(), _ptr(pre), _ptr(ws),
                                      ws_bytes, _status_ptr(status), _stream(dev)))
    return h, pre


def _gated_backward(ctx, dh):
    x, w13, pre = ctx.saved_tensors
    dtype, dev = x.dtype, x.device
    dh = _aligned(dh if dh.dtype is dtype else dh.to(dtype))
    tokens, hidden = x.shape
    inter = w13.shape[0] // 2
    want_x, want_w, _, _ = ctx.needs_input_grad
    dx = torch.empty_like(x) if want_x else None
    dw13 = torch.empty_like(w13) if want_w else None
    lib = L.lib()
    with _on(dev):
        ws_bytes = lib.exf_gated_mlp_backward_workspace_bytes(tokens, hidden, inter)
        ws = torch.empty(ws_bytes if ws_bytes > 32 else 32, dtype=torch.uint8, device=dev)
        L.check(lib.exf_gated_mlp_backward(
            dh.data_ptr(), pre.data_ptr(), x.data_ptr(), w13.data_ptr(), _WDT[dtype], tokens,
            hidden, inter, ctx.activation, _ptr(dx), _ptr(dw13), ws.data_ptr(), ws_bytes,
            _status_ptr(ctx.status), _stream(dev)))
    return dx, dw13, None, None


_gated_backward_once = torch.autograd.function.once_differentiable(_gated_backward)


class _GatedMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, activation, status):
        h, pre = _gated_forward(x, w13, activation, status, True)
        ctx.save_for_backward(x, w13, pre)
        ctx.activation, ctx.status = activation, status
        return h

    @staticmethod
    def backward(ctx, dh):
        # recorded itself (create_graph): its gradients raise when they are differentiated
        return (_gated_backward_once if torch.is_grad_enabled() else _gated_backward)(ctx, dh)


def _has_tangent(*tensors: torch.Tensor) -> bool:
    """Whether one of them is a dual tensor of forward-mode differentiation."""
    return (forward_ad._current_level >= 0
            and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors))


def gated_mlp(x: torch.Tensor, w13: torch.Tensor, activation: str = "silu",
              status: torch.Tensor | None = None) -> torch.Tensor:
    """h = act(x Wg^T) * (x Wu^T): both projections, the activation and the product in one launch.

    x [..., H] and w13 [2I, H] (gate rows, then up rows, as an expert of `fused_experts`) bf16 or
    fp16; h [..., I].  activation "silu" or "gelu_tanh".  H and I are multiples of 8.
    Differentiable in x and w13 (once, in reverse mode; forward mode is refused): a forward pass that
    autograd records keeps both projections in fp32 (8 bytes per token and intermediate feature) for
    the backward pass.
    `status` (int32 [1] on the device) is set to 1 if a pipeline wait timed out.
    """
    _require_cuda(x, w13, status)
    if x.dtype not in (torch.bfloat16, torch.float16) or w13.dtype != x.dtype:
        raise TypeError("gated_mlp needs x and w13 both bfloat16 or both float16")
    if activation not in _ACTIVATION:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATION)}, got {activation!r}")
    if (x.dim() < 1 or w13.dim() != 2 or w13.shape[0] % 2 or w13.shape[1] != x.shape[-1]
            or w13.numel() == 0):
        raise ValueError(f"x {tuple(x.shape)} and w13 {tuple(w13.shape)} must be [..., H] and "
                         "[2I, H]")
    if _has_tangent(x, w13):
        raise NotImplementedError("gated_mlp has no forward-mode derivative")
    flat = x.dim() == 2
    rows, w = _aligned(x if flat else x.reshape(-1, x.shape[-1])), _aligned(w13)
    act = _ACTIVATION[activation]
    if torch.is_grad_enabled() and (x.requires_grad or w13.requires_grad):
        h = _GatedMlp.apply(rows, w, act, status)
    else:
        h, _ = _gated_forward(rows, w, act, status, False)
    return h if flat else h.view(*x.shape[:-1], h.shape[1])
