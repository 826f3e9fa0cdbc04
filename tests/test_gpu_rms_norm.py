"""The root-mean-square norm, its gradients and its 8-bit form against the formulas in 64 bits.

Bounds are derived, element by element.  With u = eps / 2 of the type, e = 2^-24, s the rounded sum
(exact in both), n columns:
  the sum of squares has terms of one sign, added in chains of at most m = max(32, n / 1024 * 8) a
    thread and 10 more over threads: v = 1 / sqrt(...) is off by (m / 2 + 10) e relative (that half,
    the division, the addition and an inverse root of 2 units in the last place) =: ev
  |dy| <= (ev + 3 e + u) |y|
  c = sum w dy s is off by (m + 13) e sum |w dy s|, k = c v^3 / n by (3 ev + 6 e) |k| more
  |d(dx)| <= (ev + 4 e) |v w dy| + |s| dk + 3 e (|v w dy| + |s k| + |ds|) + u |dx|
  dw sums over rows / 128 rows a block and at most 80 sums: (ev + 3 e + (rows / 128 + 100) e) sum
    |dy s v| + u |dw|
A result below the type's smallest normal is off by at most half its smallest subnormal.
8 bits: the codes are those of the definition, the scales within (ev + 4 e).
"""

from __future__ import annotations

import pytest
import torch

from exfold_b200 import _lib as L
from exfold_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24


def inputs(rows, cols, dtype, seed, weight=None, size=1.0, wide=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    x = (size * normal(rows, cols + wide)).to(dtype)[:, :cols]
    r = (size * normal(rows, cols + wide)).to(dtype)[:, :cols]
    w = (1.0 + 0.3 * normal(cols)).to(weight or dtype)
    return x, r, w, normal(rows, cols).to(dtype), normal(rows, cols).to(dtype)


def chain(cols):
    return max(32, cols / 128)


def formulas(s, w, dy, ds, eps):
    """(y, dx, dw) in 64 bits and their bounds."""
    f, fw = torch.finfo(s.dtype), torch.finfo(w.dtype)
    u, tiny = f.eps / 2, f.smallest_normal * f.eps / 2
    s, w = s.double(), w.double()
    rows, n = s.shape
    m = chain(n)
    ev = (m / 2 + 10) * E
    v = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    y = s * v * w
    ey = (ev + 3 * E + u) * y.abs() + tiny
    if dy is None:
        return y, ey
    dy = dy.double()
    ds = torch.zeros_like(s) if ds is None else ds.double()
    a, c = v * w * dy, (w * dy * s).sum(-1, keepdim=True)
    k = c * v ** 3 / n
    dx = a - s * k + ds
    dk = (m + 13) * E * (w * dy * s).abs().sum(-1, keepdim=True) * v ** 3 / n + (
        3 * ev + 6 * E) * k.abs()
    edx = ((ev + 4 * E) * a.abs() + s.abs() * dk + 3 * E * (a.abs() + (s * k).abs() + ds.abs())
           + u * dx.abs() + tiny)
    dw = (dy * s * v).sum(0)
    edw = ((ev + 3 * E + (rows / 128 + 100) * E) * (dy * s * v).abs().sum(0)
           + fw.eps / 2 * dw.abs() + fw.smallest_normal * fw.eps / 2)
    return (y, dx, dw), (ey, edx * (1 + u), edw * (1 + u))


def near(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (
        f"off by {(off / bound).max().item():.3g} bounds; max {off.max().item():.3g}")


SHAPES = [(1, 1), (1, 8), (3, 7), (1, 2048), (5, 64), (300, 16), (299, 40), (1000, 128), (70, 333),
          (700, 333), (64, 2048), (400, 2048), (37, 1001), (513, 1001), (310, 4096), (4, 4100),
          (301, 4100), (303, 5001), (2, 8192), (299, 8200), (3, 16384), (300, 16392), (2, 16385),
          (300, 20000), (297, 33000), (2, 40001)]


@pytest.mark.parametrize("dtype,weight", [(BF16, None), (BF16, F32), (F16, None), (F16, F32),
                                          (F32, None)])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_gradients(rows, cols, dtype, weight):
    x, r, w, dy, ds = inputs(rows, cols, dtype, rows + cols, weight)
    s = (x.float() + r.float()).to(dtype)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, total = ops.rms_norm(x, w, 1e-5, residual=r)
    assert torch.equal(total, s)
    want, bound = formulas(s, w.detach(), dy, ds, 1e-5)
    got = torch.autograd.grad((y, total), (x, r, w), (dy, ds))
    near(y.detach(), want[0], bound[0])
    near(got[0], want[1], bound[1])
    assert torch.equal(got[0], got[1])
    near(got[2], want[2], bound[2])
    # without a residual, and unrecorded
    y = ops.rms_norm(x, w, 1e-5)
    want, bound = formulas(x.detach(), w.detach(), dy, None, 1e-5)
    near(y.detach(), want[0], bound[0])
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    near(dx, want[1], bound[1])
    near(dw, want[2], bound[2])
    with torch.no_grad():
        assert torch.equal(ops.rms_norm(x, w, 1e-5), y.detach())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("cols,wide", [(64, 8), (2048, 24), (1001, 24), (40, 3), (17000, 8)])
def test_rows_at_a_distance(cols, wide, dtype):
    """Columns of a wider matrix, and gradients through them."""
    x, r, w, dy, ds = inputs(310, cols, dtype, cols, wide=wide)
    assert not x.is_contiguous()
    y, s = ops.rms_norm(x, w, residual=r)
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    near(y, *formulas(s, w, None, None, 1e-6))
    whole = torch.zeros(310, cols + wide, dtype=dtype, device=DEV, requires_grad=True)
    y = ops.rms_norm(whole[:, :cols] + x, w)
    want, bound = formulas(x, w, dy, None, 1e-6)
    g, = torch.autograd.grad(y, whole, dy)
    near(g[:, :cols], want[1], bound[1])
    assert not g[:, cols:].any()
    # a recorded call on the strided rows themselves
    x.requires_grad_(True)
    dx, = torch.autograd.grad(ops.rms_norm(x, w), x, dy)
    near(dx, want[1], bound[1])


def test_shapes_strides_and_partial_gradients():
    x, r, w, dy, ds = inputs(24, 256, BF16, 3)
    y2, s2 = ops.rms_norm(x, w, residual=r)
    y, s = ops.rms_norm(x.view(2, 3, 4, 256), w, residual=r.view(2, 3, 4, 256))
    assert y.shape == (2, 3, 4, 256) and torch.equal(y.view(24, 256), y2)
    assert torch.equal(s.view(24, 256), s2)
    one = ops.rms_norm(x[0], w)
    assert one.shape == (256,) and torch.equal(one, ops.rms_norm(x[:1], w)[0])
    # other orders of memory are copied
    t = x.t().contiguous().t()
    assert torch.equal(ops.rms_norm(t, w), ops.rms_norm(x, w))
    e = x[:1].expand(24, 256)
    assert torch.equal(ops.rms_norm(e, w)[7], one)
    # an odd start: a row of 2-byte values off every vector's boundary
    flat = torch.zeros(24 * 256 + 1, dtype=BF16, device=DEV)
    flat[1:] = x.reshape(-1)
    near(ops.rms_norm(flat[1:].view(24, 256), w), *formulas(x, w, None, None, 1e-6))
    # any subset of the gradients
    want, bound = formulas((x.float() + r.float()).to(BF16), w, dy, ds, 1e-6)
    for need in ([True, False, False], [False, True, False], [False, False, True]):
        a = [v.detach().clone().requires_grad_(n) for v, n in zip((x, r, w), need)]
        y, s = ops.rms_norm(a[0], a[2], residual=a[1])
        g, = torch.autograd.grad((y, s), [v for v in a if v.requires_grad], (dy, ds))
        near(g, want[2 if need[2] else 1], bound[2 if need[2] else 1])
    # only one of the outputs is used
    a = x.clone().requires_grad_(True)
    y, s = ops.rms_norm(a, w, residual=r)
    g, = torch.autograd.grad(s, a, ds, retain_graph=True)
    assert torch.equal(g, ds)
    g, = torch.autograd.grad(y, a, dy)
    want, bound = formulas(s.detach(), w, dy, None, 1e-6)
    near(g, want[1], bound[1])
    # memory in other orders, recorded: the gradient has the input's shape
    a = x.view(4, 6, 256).transpose(0, 1).requires_grad_(True)
    y = ops.rms_norm(a, w)
    assert torch.equal(y.detach(), ops.rms_norm(x, w).view(4, 6, 256).transpose(0, 1))
    g, gw = torch.autograd.grad(y, (a, w.requires_grad_(True)), dy.view(4, 6, 256).transpose(0, 1),
                                allow_unused=True)
    w = w.detach()
    assert g.shape == a.shape and gw is None
    want, bound = formulas(x, w, dy, None, 1e-6)
    near(g.transpose(0, 1).reshape(24, 256), want[1], bound[1])
    # an upstream gradient that is one value for all
    a = x.clone().requires_grad_(True)
    ops.rms_norm(a, w).sum().backward()
    want, bound = formulas(x, w, torch.ones_like(x), None, 1e-6)
    near(a.grad, want[1], bound[1])


def test_empty():
    w = torch.ones(64, dtype=BF16, device=DEV, requires_grad=True)
    x = torch.zeros(0, 64, dtype=BF16, device=DEV, requires_grad=True)
    y, s = ops.rms_norm(x, w, residual=x.detach())
    assert y.shape == (0, 64) and s.shape == (0, 64)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and not w.grad.any()
    codes, scales = ops.rms_norm_8bit(x.detach(), w.detach())
    assert codes.shape == (0, 64) and scales.shape == (0, 1)
    assert ops.dequantize_8bit(codes, scales).shape == (0, 64)


@pytest.mark.parametrize("cols", [64, 2048, 1001, 20001])
def test_far_values(cols):
    """Sums of squares outside fp32's range, rows of zeros, infinities and NaN stay in their rows."""
    x, _, w, dy, _ = inputs(6, cols, F32, cols)
    x[0] *= 1e25
    x[1] *= 1e-30
    x[2] = 0.0
    x[3, 1] = float("inf")
    x[4, 5] = float("nan")
    dy[0] *= 1e20
    for eps in (1e-6, 0.0):
        x.requires_grad_(True)
        y = ops.rms_norm(x, w, eps)
        dx, = torch.autograd.grad(y, x, dy)
        x, y = x.detach(), y.detach()
        want, bound = formulas(x, w, dy, None, eps)
        for row in (0, 1, 2, 5):
            if row == 2 and eps == 0.0:
                assert bool(y[2].isnan().all())
                continue
            # (the inverse norm of huge rows lies among fp32's subnormals: steps of 2^-149)
            v = 1.0 / (x[row].double().square().mean() + eps).sqrt()
            sub = 2.0 ** -149 / v if v < 2.0 ** -126 else 0.0
            near(y[row], want[0][row], bound[0][row] + sub * want[0][row].abs())
            near(dx[row], want[1][row],
                 bound[1][row] + 4 * sub * (dy[row] * w).abs().double().amax() * v)
        assert bool(y[3, 1].isnan()) and not y[3, 0].isnan() and float(y[3, 0]) == 0.0
        assert bool(y[4].isnan().all())
    # bf16 rows beside them keep their values
    xb = x.to(BF16)
    yb = ops.rms_norm(xb, w.to(BF16))
    near(yb[5:], *formulas(xb[5:], w.to(BF16), None, None, 1e-6))


def test_differences():
    """The gradients against central differences of the formula in 64 bits."""
    x, r, w, dy, ds = inputs(3, 40, F32, 11)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = ops.rms_norm(x, w, 1e-3, residual=r)
    grads = torch.autograd.grad((y, s), (x, r, w), (dy, ds))

    def value(x, r, w):
        s = x + r
        y = s * w / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-3)
        return (y * dy.double()).sum() + (s * ds.double()).sum()

    at = [t.detach().double() for t in (x, r, w)]
    h = 1e-4
    for i, g in enumerate(grads):
        for j in range(0, at[i].numel(), 7):
            up, down = [t.clone() for t in at], [t.clone() for t in at]
            up[i].view(-1)[j] += h
            down[i].view(-1)[j] -= h
            slope = (value(*up) - value(*down)) / (2 * h)
            # (third derivatives of order 10 here: h^2 / 6 of them, and fp32 sums of order 10)
            assert abs(float(slope) - float(g.view(-1)[j])) < 1e-5 * (1.0 + abs(float(slope)))


# ---- 8 bits -------------------------------------------------------------------------------------
def codes64(s, w, code, group, eps):
    """(codes as values, scales) by the definition, 64 bits."""
    s, w = s.double(), w.double()
    n = s.shape[1]
    most = 448.0 if code is torch.float8_e4m3fn else 127.0
    v = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    p = s * w
    q, scales = torch.zeros_like(p), []
    for c in range(0, n, group or n):
        part = p[:, c:c + (group or n)]
        top = part.abs().amax(-1, keepdim=True)
        t = torch.where(top > 0, part * most / torch.where(top > 0, top, 1.0), 0.0)
        if code is torch.int8:
            t = torch.round(t)
        else:
            unit = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
            t = torch.round(t / unit) * unit
        q[:, c:c + (group or n)] = t
        scales.append(top * v / most)
    return q, torch.cat(scales, 1)


SHAPES_8 = [(1, 8), (1, 1), (2, 33), (5, 128), (300, 40), (301, 160), (256, 2048), (310, 2048),
            (61, 1001), (400, 1001), (310, 4100), (299, 8192), (3, 4096), (2, 20000), (297, 20000),
            (300, 16391), (2, 50001)]


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("group", [None, 32, 64, 128])
@pytest.mark.parametrize("dtype,weight", [(BF16, None), (BF16, F32), (F16, None), (F32, None)])
def test_8bit(dtype, weight, group, code):
    for rows, cols in SHAPES_8:
        x, r, w, *_ = inputs(rows, cols, dtype, rows + cols, weight, wide=8 * (rows % 2))
        codes, scales, s = ops.rms_norm_8bit(x, w, 1e-6, residual=r, dtype=code, group=group)
        assert torch.equal(s, (x.float() + r.float()).to(dtype))
        q, want = codes64(s, w, code, group, 1e-6)
        assert codes.dtype == code and scales.shape == want.shape
        wrong = codes.double() != q
        assert not wrong.any(), (rows, cols, int(wrong.sum()), codes.double()[wrong][:4],
                                 q[wrong][:4])
        near(scales, want, ((chain(cols) / 2 + 14) * E) * want)
        for out in (dtype, F32):
            back = ops.dequantize_8bit(codes, scales, group=group, dtype=out)
            wide = scales.double().repeat_interleave(group or cols, 1)[:, :cols]
            assert torch.equal(back, (codes.double() * wide).float().to(out))
        alone = ops.rms_norm_8bit(s, w, 1e-6, dtype=code, group=group)
        assert torch.equal(alone[0].view(torch.uint8), codes.view(torch.uint8))
        assert torch.equal(alone[1], scales)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_8bit_borders(dtype):
    """Quotients at and beside the borders between codes: rows whose largest value is the largest code,
    so that the others are their own quotients."""
    # every border of e4m3 in this range, and the values of the type to both sides of it
    grid = torch.arange(0, 127, device=DEV).to(torch.uint8).view(torch.float8_e4m3fn).double()
    mids = ((grid[1:] + grid[:-1]) / 2).tolist()
    for code, most, middles in ((torch.float8_e4m3fn, 448.0, mids),
                                (torch.int8, 127.0, [i + 0.5 for i in range(127)])):
        m = torch.tensor(middles, dtype=torch.float64, device=DEV).to(dtype)
        inf = torch.tensor(float("inf"), dtype=dtype, device=DEV)
        row = torch.cat([m, torch.nextafter(m, inf), torch.nextafter(m, -inf),
                         -m, -torch.nextafter(m, inf)])
        row = row[row.abs() < most]
        row = torch.cat([row, torch.tensor([most], dtype=dtype, device=DEV)])
        for scale in (1.0, 0.375, 2.0 ** -7):
            for cols in (row.numel(), row.numel() + 8 - row.numel() % 8):
                x = torch.zeros(3, cols, dtype=dtype, device=DEV)
                x[:, :row.numel()] = row
                w = torch.full((cols,), scale, dtype=dtype, device=DEV)
                codes, scales = ops.rms_norm_8bit(x, w, dtype=code, group=None)
                q, want = codes64(x, w, code, None, 1e-6)
                assert torch.equal(codes.double(), q)


@pytest.mark.parametrize("cols", [256, 250, 40000])
@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_8bit_far_values(cols, code):
    x, _, w, *_ = inputs(4, cols, F32, cols)
    x[0] = 0.0
    x[1, :128] = 0.0
    x[1, 3] = 1e-37
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    codes, scales = ops.rms_norm_8bit(x, w, dtype=code, group=128)
    back = ops.dequantize_8bit(codes, scales, dtype=F32)
    assert not codes[0].float().any() and not scales[0].any() and not back[0].any()
    q, want = codes64(x[1:2], w, code, 128, 1e-6)
    assert torch.equal(codes[1:2].double(), q)
    near(scales[1:2], want, (chain(cols) / 2 + 14) * E * want + 2.0 ** -148)
    assert bool(scales[2].isnan().all()) and bool(back[2].isnan().all())  # the norm is NaN
    # an infinity: its own group is NaN, the inverse norm 0
    assert bool(back[3, :128].isnan().all()) and not back[3, 128:].any()
    # subnormal products
    tiny = torch.full((1, cols), 2.0 ** -140, device=DEV)
    tiny[0, ::3] *= 0.25
    codes, scales = ops.rms_norm_8bit(tiny, torch.ones(cols, device=DEV), 0.0, dtype=code,
                                      group=None)
    assert torch.equal(codes.double(), codes64(tiny, torch.ones(cols, device=DEV), code, None, 0)[0])


@pytest.mark.parametrize("dtype,weight", [(BF16, None), (F16, F32), (F32, None)])
@pytest.mark.parametrize("wide,start", [(0, 0), (1, 0), (2, 1)])
def test_8bit_rows_off_vectors(dtype, weight, wide, start):
    """Rows that begin and end inside a vector, many a block, of one warp and of several."""
    for rows, cols, group in ((5000, 101, 32), (20001, 9, 64), (3000, 33, 32), (1501, 255, 128),
                              (149, 513, None), (701, 4001, 64), (151, 45001, None), (9, 7, 128)):
        x, r, w, *_ = inputs(rows, cols + start, dtype, cols, weight, wide=wide)
        x, r, w = x[:, start:], r[:, start:], w[start:]
        for code in (torch.float8_e4m3fn, torch.int8):
            codes, scales, s = ops.rms_norm_8bit(x, w, 1e-6, residual=r, dtype=code, group=group)
            assert torch.equal(s, (x.float() + r.float()).to(dtype))
            q, want = codes64(s, w, code, group, 1e-6)
            assert torch.equal(codes.double(), q), (rows, cols)
            near(scales, want, ((chain(cols) / 2 + 14) * E) * want)
            alone = ops.rms_norm_8bit(x, w, 1e-6, dtype=code, group=group)
            assert torch.equal(alone[0].double(), codes64(x, w, code, group, 1e-6)[0])


@pytest.mark.parametrize("group", [None, 32])
@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_8bit_values_that_are_not_finite_in_odd_rows(code, group):
    """Infinities and NaN stay in their groups, in rows that begin on even and on odd elements."""
    rows, cols = 12, 99
    x, _, w, *_ = inputs(rows, cols, F16, 3)
    at = [0, 31, 32, 63, 64, 98]
    for i in range(rows):
        x[i, at[i // 2]] = float("inf")
    codes, scales = ops.rms_norm_8bit(x, w, dtype=code, group=group)
    back = ops.dequantize_8bit(codes, scales, group=group, dtype=F32)
    for i in range(rows):  # (the inverse norm is 0)
        mine = at[i // 2] // 32 if group else 0
        for j in range(scales.shape[1]):
            part = back[i, j * (group or cols):(j + 1) * (group or cols)]
            assert bool(part.isnan().all()) if j == mine else not part.any()
    x[3, 5] = float("nan")
    codes, scales = ops.rms_norm_8bit(x, w, dtype=code, group=group)
    assert bool(scales[3].isnan().all())
    if group is None:  # products that round to 0 and to subnormals, beside one far above
        x = torch.full((4, cols), 6e-8, device=DEV, dtype=F16)
        x[:, 40] = 3e-5
        codes, _ = ops.rms_norm_8bit(x, w, 0.0, dtype=code, group=group)
        assert torch.equal(codes.double(), codes64(x, w, code, group, 0.0)[0])


@pytest.mark.parametrize("cols", [256, 101])
def test_8bit_codes_at_any_address(cols):
    """Codes of vectors and of odd rows at each of eight addresses; nothing beside them is written."""
    rows, lib = 37, L.lib()
    for dtype, d in ((BF16, 1), (F32, 0)):
        x, r, w, *_ = inputs(rows, cols, dtype, 8)
        want, scales, s = ops.rms_norm_8bit(x, w, residual=r, group=64)
        for off in range(8):
            flat = torch.full((rows * cols + 16,), 77, dtype=torch.uint8, device=DEV)
            got_s, got_scales = torch.zeros_like(s), torch.zeros_like(scales)
            L.check(lib.exf_rms_norm_8bit(
                x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), d, d, rows, cols, 1e-6, 0, 64,
                got_s.data_ptr(), flat.data_ptr() + off, got_scales.data_ptr(),
                torch.cuda.current_stream().cuda_stream))
            codes = flat[off:off + rows * cols].view(rows, cols)
            assert torch.equal(codes, want.view(torch.uint8))
            assert torch.equal(got_s, s)
            near(got_scales, scales.double(), 4 * (chain(cols) / 2 + 14) * E * scales.double())
            assert bool((flat[:off] == 77).all()) and bool((flat[off + rows * cols:] == 77).all())


def test_dequantize_ragged_starts():
    """Codes and results off every vector's boundary, more than a row a thread."""
    g = torch.Generator(device=DEV).manual_seed(5)
    for rows, cols, group in ((1000, 3, None), (77, 1, None), (50, 129, 128), (9, 33, 32)):
        codes = torch.randint(-127, 128, (rows, cols), generator=g, device=DEV).to(torch.int8)
        groups = 1 if group is None else -(-cols // group)
        scales = torch.rand(rows, groups, generator=g, device=DEV)
        want = (codes.float() * scales.repeat_interleave(group or cols, 1)[:, :cols])
        for dtype in (BF16, F16, F32):
            assert torch.equal(ops.dequantize_8bit(codes, scales, group, dtype), want.to(dtype))
        flat = torch.zeros(codes.numel() + 1, dtype=torch.int8, device=DEV)
        flat[1:] = codes.reshape(-1)
        got = ops.dequantize_8bit(flat[1:].view(rows, cols), scales, group, F32)
        assert torch.equal(got, want)


def test_graph_streams_and_refusals():
    x, r, w, dy, ds = inputs(300, 2048, BF16, 9)
    want = ops.rms_norm(x, w, residual=r)
    want8 = ops.rms_norm_8bit(x, w, residual=r)
    a, b, c = (t.clone().requires_grad_(True) for t in (x, r, w))
    y, s = ops.rms_norm(a, c, residual=b)
    grads = torch.autograd.grad((y, s), (a, b, c), (dy, ds))
    del y, s
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.rms_norm(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rms_norm(x, w, residual=r)
        got8 = ops.rms_norm_8bit(x, w, residual=r)
        y, s = ops.rms_norm(a, c, residual=b)
        again = torch.autograd.grad((y, s), (a, b, c), (dy, ds))
    for t in (*got, *again):
        t.zero_()
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got8, want8))
    assert all(torch.equal(p, q) for p, q in zip(again, grads))

    with pytest.raises(TypeError):
        ops.rms_norm(x.double(), w)
    with pytest.raises(TypeError):
        ops.rms_norm(x, w.half())
    with pytest.raises(TypeError):
        ops.rms_norm(x, w, residual=r.float())
    with pytest.raises(ValueError):
        ops.rms_norm(x, w[:-1])
    with pytest.raises(ValueError):
        ops.rms_norm(x, w, residual=r[:1])
    with pytest.raises(ValueError):
        ops.rms_norm(x, w, -1.0)
    with pytest.raises(TypeError):
        ops.rms_norm_8bit(x, w, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.rms_norm_8bit(x, w, group=16)
    with pytest.raises(RuntimeError):
        ops.rms_norm(x, w.cpu())
    # gradients of gradients are refused, not silently zero
    y = ops.rms_norm(a, c)
    g, = torch.autograd.grad(y, a, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), c)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, dy)
        with pytest.raises(NotImplementedError):
            ops.rms_norm(dual, w)
