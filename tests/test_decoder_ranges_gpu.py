"""The decoder operators where values leave the usual range: saturated
activations with the kept derivative, upstream gradients beyond fp16's range,
scales whose product leaves fp32's.

Tolerances are bounds, derived here before the first run, on top of those of a
rounding (half a step of the type) and of a sum (2**-23 per term and addition).
"""

from __future__ import annotations

import math

import pytest
import torch

from quantem.cuda import _core
from quantem.cuda.core import ml

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
D = torch.float64


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def _half_step(y, t):
    f = torch.finfo(t)
    return torch.maximum(y.abs() * (f.eps / 2), torch.full_like(y, f.smallest_normal * f.eps / 2))


def _within(got, want, bound, what=""):
    assert got.shape == want.shape
    err = (got.to(D) - want).abs()
    worst = (err - bound).nan_to_num(nan=math.inf).max().item()
    assert worst <= 0, f"{what}: beyond its bound by {worst:.3e} (largest error {err.max().item():.3e})"


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(D)
    if act == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * torch.sigmoid(-z))
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


# ── the kept derivative ───────────────────────────────────────────────────


def _kept_derivative(z, act):
    """act'(z) of a large bf16 call whose z is its bf16 bias (zero weights), as
    the bias gradient of one row's unit upstream gradient."""
    rows, k, n = 700, 512, z.numel()
    x, w = torch.ones(rows, k, dtype=BF16, device="cuda"), torch.zeros(n, k, dtype=BF16, device="cuda")
    b = z.to(BF16).requires_grad_()
    assert n % 8 == 0 and _core.decoder_linear_keep(x, w, b, None, act, None) is not NotImplemented
    dy = torch.zeros(rows, n, dtype=BF16, device="cuda")
    dy[600] = 1
    db, = torch.autograd.grad(ml.linear_act(x, w, b, activation=act), [b], dy)
    return db, b.detach().to(D)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_kept_derivative_over_the_whole_range(act):
    """From saturation to saturation, far beyond any polynomial's range: the
    evaluation (2**-19), the kept fp16 (half a step: values in [1, 2) lie 2**-10
    apart, so 2**-11 of the value, and 2**-25 near zero) and the bf16 gradient's
    half step."""
    far = torch.tensor([50.0, 100.0, 300.0, 1e4, 1e6, 1e8, 1e20, 1e38, 0.0, 1e-30, 6.0, 9.0])
    z = torch.cat([torch.linspace(-40, 40, 4000), far, -far]).cuda()
    db, z = _kept_derivative(z, act)
    want = _act_grad(z, act)
    _within(db, want, (want.abs() * 2.0**-11 + 2.0**-25 + 2.0**-19) * 1.01 + _half_step(want, BF16) * (1 + 2.0**-8), act)


def test_small_kept_derivatives_keep_their_digits():
    """SiLU's derivative down to -30 is between 1e-12 and 1e-4: bf16 holds it,
    so the kept one has to, within a bf16 step (its evaluation, 2**-14 of the
    value, its own rounding, 2**-11, or 2**-37, and bf16's half step)."""
    db, z = _kept_derivative(torch.linspace(-30, -12, 1600).cuda(), "silu")
    want = _act_grad(z, "silu")
    _within(db, want, want.abs() * (2.0**-14 + 2.0**-11 + 2.0**-8) + 2.0**-37)


# ── fp32 upstream gradients of fp16 operands ──────────────────────────────


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e-9, 1.0, 3e6, 1e12])
@pytest.mark.parametrize("rows,k,n", [(20000, 64, 48), (700, 203, 77), (40, 136, 520)])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_upstream_gradients_beyond_fp16(size, rows, k, n, act):
    """fp32 upstream gradients of any size with fp16 operands: dz has fp16's
    digits next to the largest gradient, down to 2**-39 of it. The operands are
    sized so that dx, or dweight, lies within fp16's range."""
    g = _gen(rows + k)
    dy = _randn(g, rows, n, scale=size)
    dy[3] = 0
    for small_w in (True, False):
        # one of dx = dz W and dweight = dz^T x is brought near 1, both where size is 1
        a, c = (size**-1, 1.0) if small_w else (1.0, size**-1)
        a, c = min(max(a, 2.0**-10), 2.0**8), min(max(c, 2.0**-10), 2.0**8)
        w = (_randn(g, n, k) * a).to(F16).requires_grad_()
        x = (_randn(g, rows, k) * c).to(F16).requires_grad_()
        b = (_randn(g, n) * a * c).requires_grad_()
        y = ml.linear_act(x, w, b, activation=act, out_dtype=F32)
        dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
        xd, wd, bd, dyd = (t.detach().to(D) for t in (x, w, b, dy))
        z = xd @ wd.T + bd
        ez = (k + 4) * 2.0**-23 * (xd.abs() @ wd.abs().T + bd.abs())
        # relu: a z within its error of 0 may fall on either side
        ed = {"none": torch.zeros_like(z), "relu": (z.abs() <= ez).to(D), "silu": 1.1 * ez + 2.0**-19}[act]
        dz = dyd * _act_grad(z, act)
        edz = dyd.abs() * ed + 2.0**-23 * dz.abs()
        edz16 = (edz + dz.abs() * 2.0**-11 + dyd.abs().max() * 2.0**-39) * (1 + 2.0**-10)
        mag = dz.abs() + edz16
        for got, want, e, mass, terms, t in (
            (dx, dz @ wd, edz16 @ wd.abs(), mag @ wd.abs(), n, F16),
            (dw, dz.T @ xd, edz16.T @ xd.abs(), mag.T @ xd.abs(), rows, F16),
            (db, dz.sum(0), edz.sum(0), (dz.abs() + edz).sum(0), rows, F32),
        ):
            bound = _half_step(want, t) * (1 + 2.0**-10) + (e + (terms + 4) * 2.0**-23 * mass) * 1.01
            fits = want.abs() + bound < 65504 if t is F16 else torch.ones_like(want, dtype=torch.bool)
            _within(torch.where(fits, got.to(D), 0.0), torch.where(fits, want, 0.0), bound, f"{t} {tuple(want.shape)}")
            if t is F16:
                over = want.abs() - bound > 65536
                assert got[over].isinf().all()
    assert _core.device_fault_word(0, True) == 0


@pytest.mark.parametrize("act", ["none", "silu"])
def test_tiny_gradients_are_not_lost(act):
    """A loss averaged over 1e9 values: dweight is far above fp16's smallest step
    although no upstream gradient is."""
    g = _gen(9)
    x = _randn(g, 30000, 64).abs().to(F16)
    w, dy = _randn(g, 40, 64).abs().to(F16).requires_grad_(), torch.full((30000, 40), 1e-9, device="cuda")
    dw, = torch.autograd.grad(ml.linear_act(x * 8, w, activation=act, out_dtype=F32), [w], dy)
    want = (dy.to(D) * _act_grad((x * 8).to(D) @ w.detach().to(D).T, act)).T @ (x * 8).to(D)
    # 2**-10: half a step of dz and of dweight, and the sum of 30000 positive terms
    _within(dw, want, want.abs() * (2.0**-10 + 30004 * 2.0**-23) + 2.0**-25)


@pytest.mark.parametrize("act", ["none", "gelu"])
def test_not_finite_gradients_stay_in_their_rows(act):
    """A NaN or an infinity upstream neither spoils other rows nor their scale."""
    g = _gen(10)
    x, w = _randn(g, 300, 64).to(F16).requires_grad_(), _randn(g, 48, 64, scale=0.1).to(F16)
    dy = _randn(g, 300, 48, scale=1e-3)
    bad = dy.clone()
    bad[7, 5], bad[200, 1], bad[201, 2] = float("nan"), float("inf"), -float("inf")
    y = ml.linear_act(x, w, activation=act, out_dtype=F32)
    dx, = torch.autograd.grad(y, [x], bad, retain_graph=True)
    dy[[7, 200, 201]] = 0
    clean, = torch.autograd.grad(y, [x], dy)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[7, 200, 201]] = False
    _within(dx[keep], clean[keep].to(D), clean[keep].to(D).abs() * 2.0**-9 + 2.0**-24)
    assert not dx[~keep].isfinite().any()
    zero, = torch.autograd.grad(ml.linear_act(x, w, activation=act, out_dtype=F32), [x], torch.zeros_like(dy))
    assert not zero.any()


# ── scales of 8-bit operands ──────────────────────────────────────────────


@pytest.mark.parametrize("rows", [5, 300])
def test_scales_whose_product_leaves_fp32(rows):
    """The product is multiplied by one scale after the other, so neither a
    product of scales below fp32's normal range nor one above it counts."""
    k, n = 64, 40
    x, w = torch.full((rows, k), 448.0, device="cuda").to(E4M3), torch.full((n, k), 448.0, device="cuda").to(E4M3)
    sx, sw = torch.full((rows,), 3e-30, device="cuda"), torch.full((n,), 7e-13, device="cuda")
    y = ml.linear_act_fp8(x, sx, w, sw, out_dtype=F32)
    want = 448.0**2 * k * sx.to(D)[:, None] * sw.to(D)
    _within(y, want, want * 2.0**-20)
    zero = torch.zeros(rows, k, device="cuda").to(E4M3)
    y = ml.linear_act_fp8(zero, torch.full_like(sx, 1e25), w, torch.full_like(sw, 1e20), out_dtype=F32)
    assert not y.any()


@pytest.mark.parametrize("act", ["none", "silu"])
def test_scaled_gradients_in_a_graph(act):
    """The scale is formed on the device: a captured backward follows the
    gradients that it is replayed on. On another stream, too."""
    g = _gen(13)
    x, w = _randn(g, 700, 64).to(F16).requires_grad_(), _randn(g, 48, 64).to(F16).requires_grad_()
    dy = _randn(g, 700, 48)

    def step():
        return torch.autograd.grad(ml.linear_act(x, w, activation=act, out_dtype=F32), [x, w], dy)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for size in (1.0, 2.0**-20, 2.0**14, 2.0**-30):
        dy.copy_(_randn(g, 700, 48, scale=size))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
