"""MXFP4 quantisation against its definition in 64 bits: codes, scales and the values read back are
equal, bit for bit (both sides round the same exact quotient once)."""

from __future__ import annotations

import math

import pytest
import torch

from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(x):
    """(values, scale bytes) of x [rows, cols] in 64 bits, on the CPU."""
    x = x.double().cpu()
    rows, cols = x.shape
    v = torch.nn.functional.pad(x, (0, -cols % 32)).reshape(rows, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    _, e = torch.frexp(torch.where(bad, 1.0, top))
    e = torch.where(top == 0, -127, (e - 3).clamp(min=-127))
    a = torch.where(bad, 0.0, v.abs()) * torch.exp2(-e.double())
    grid = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    a = (torch.round(a / grid) * grid).clamp(max=6.0) * torch.exp2(e.double())
    values = torch.where(bad, math.nan, torch.where(v < 0, -a, a))
    scale = torch.where(bad, 255, e + 127).squeeze(-1)
    return values.reshape(rows, -1)[:, :cols], scale


def check(x):
    codes, scales = ops.quantize_mxfp4(x)
    back = ops.dequantize_mxfp4(codes, scales, cols=x.shape[-1], dtype=torch.float32)
    values, want = definition(x.reshape(-1, x.shape[-1]))
    assert codes.shape == (*x.shape[:-1], 16 * ((x.shape[-1] + 31) // 32))
    assert torch.equal(scales.cpu().reshape(want.shape).int(), want.int())
    got = back.cpu().double().reshape(values.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(values))
    assert torch.equal(got.nan_to_num(0.0), values.nan_to_num(0.0))
    return codes, scales, back


def rand(rows, cols, dtype, seed, spread=6.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=DEV)
    size = torch.exp2(spread * (torch.rand(rows, cols, generator=g, device=DEV) - 0.5))
    return (x * size).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 7), (7, 100),
                                       (64, 2048), (129, 1000), (33, 4100), (1, 8192),
                                       (20000, 40)])
def test_equals_definition(rows, cols, dtype):
    check(rand(rows, cols, dtype, seed=rows + cols))


@pytest.mark.parametrize("dtype", DTYPES)
def test_borders_between_codes(dtype):
    """Every tie, and its neighbours a unit in the last place away, at several scales."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], device=DEV).to(dtype)
    eps = torch.finfo(dtype).eps
    near = torch.cat([mids * (1 - eps), mids, mids * (1 + eps)])
    near = torch.cat([near, -near])
    row = torch.zeros(64, 32, dtype=dtype, device=DEV)
    row[:54, 0] = near
    row[:, 1] = 4.0  # fixes the exponent at 0 for what is below 8
    check(torch.cat([row * s for s in (1.0, 2.0 ** -9, 2.0 ** 7)]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_extremes(dtype):
    f = torch.finfo(dtype)
    x = torch.zeros(10, 96, dtype=dtype, device=DEV)
    x[0, 3], x[1, 40], x[2, 70] = math.inf, -math.inf, math.nan
    x[3, 5], x[3, 6] = f.max, -f.max
    x[4, 7], x[4, 8] = f.tiny, -f.tiny / 2  # smallest normal and a subnormal
    x[5, 9] = f.smallest_normal * f.eps     # smallest subnormal
    x[6] = f.max
    x[7] = -0.0
    x[8, :32] = 1.0
    x[8, 31] = math.nan                     # the neighbouring blocks stay as they are
    check(x)


def test_reading_back_rounds_once_and_scale_255_is_nan():
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(16, 1)
    scales = torch.randint(100, 150, (16, 16), device=DEV).to(torch.uint8)
    scales[:, 0], scales[:, 1], scales[:, 2], scales[:, 3] = 0, 254, 255, 1
    codes = codes.reshape(16, 256)
    m = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    n = torch.stack([codes & 15, codes >> 4], -1).reshape(16, 512).long()
    exact = torch.where(n > 7, -1.0, 1.0) * m[n & 7] * torch.exp2(
        scales.double() - 127).repeat_interleave(32, -1)
    for dtype in DTYPES:
        want = exact.to(dtype)
        want[:, 64:96] = math.nan
        got = ops.dequantize_mxfp4(codes, scales, dtype=dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0, 1e30, -1e30) if dtype != torch.float16 else
                           got.nan_to_num(0.0), want.nan_to_num(0.0, 1e30, -1e30)
                           if dtype != torch.float16 else want.nan_to_num(0.0))


def test_strided_rows_offsets_and_dimensions():
    base = rand(40, 200, torch.bfloat16, seed=5)
    for x in (base[:, :64], base[:, 3:131], base[::2, 8:72], base.t()[:64], base[1:2, 1:34],
              base.reshape(4, 10, 200), base[0]):
        check(x)


def test_rows_far_apart_in_memory():
    """Row offsets past 2^31 elements."""
    base = torch.zeros(1, dtype=torch.float16, device=DEV).expand(1)
    big = torch.empty((1 << 31) + 4096, dtype=torch.float16, device=DEV)
    x = big.as_strided((2, 64), ((1 << 31) + 1024, 1))
    x.copy_(rand(2, 64, torch.float16, seed=9))
    check(x)
    del base, big


def test_more_values_than_32_bits_number():
    """2.15e9 values in odd rows: the last rows as on their own."""
    rows, cols = 40000, 53701
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    for r in range(0, rows, 4000):
        x[r:r + 4000] = torch.randn(4000, cols, device=DEV, dtype=torch.bfloat16)
    codes, scales = ops.quantize_mxfp4(x)
    back = ops.dequantize_mxfp4(codes, scales, cols=cols)
    for part in (slice(0, 3), slice(19998, 20003), slice(rows - 3, rows)):
        c, s = ops.quantize_mxfp4(x[part].clone())
        assert torch.equal(codes[part], c) and torch.equal(scales[part], s)
        assert torch.equal(back[part], ops.dequantize_mxfp4(c, s, cols=cols))


def test_empty():
    codes, scales = ops.quantize_mxfp4(torch.empty(0, 64, device=DEV))
    assert codes.shape == (0, 32) and scales.shape == (0, 2)
    assert ops.dequantize_mxfp4(codes, scales).shape == (0, 64)
    codes, scales = ops.quantize_mxfp4(torch.empty(3, 0, device=DEV))
    assert codes.shape == (3, 0) and scales.shape == (3, 0)


def test_captured_and_other_stream():
    x = rand(64, 512, torch.bfloat16, seed=11)
    want = ops.dequantize_mxfp4(*ops.quantize_mxfp4(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.dequantize_mxfp4(*ops.quantize_mxfp4(x))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.dequantize_mxfp4(*ops.quantize_mxfp4(x))
    x.copy_(rand(64, 512, torch.bfloat16, seed=12))
    graph.replay()
    assert torch.equal(out, ops.dequantize_mxfp4(*ops.quantize_mxfp4(x)))
