"""Every form of the decoder's products that a size can choose, over several
rounds of tiles and with data in every row. ``linear_act_form`` says which form
a size takes, and each test asserts it, so that a change of the rule cannot take
a form out of the tests.

Small integers, whose sums fp32 holds whole: results are equal to the 64-bit
ones rounded once, whatever the order of the additions. Activations that are no
integers go by the bounds of test_decoder_gpu.py (its _linear_bounds).
"""

from __future__ import annotations

import pytest
import torch
from test_decoder_gpu import _act, _act_grad, _gen, _half_step, _ints, _linear_bounds, _randn, _within

from quantem.cuda import _core
from quantem.cuda.core import ml

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
D = torch.float64
CODE = {BF16: _core.BF16, F16: _core.F16, E4M3: _core.E4M3}
FORWARD, DERIVATIVE, DX, DWEIGHT = range(4)
FEW, SINGLE, PAIR = range(3)


def _form(product, rows, n, k, dtype, want, parts=None, rounds=2):
    form, cols, got_parts, got_rounds = _core.linear_act_form(product, rows, n, k, CODE[dtype])
    assert (form, cols) == want
    assert got_rounds >= rounds and (parts is None or got_parts > 1)


def _no_fault():
    torch.cuda.synchronize()
    assert _core.device_fault_word(0, True) == 0


# odd numbers of row tiles, columns past the last slab and past the last tile
FORWARDS = [
    (BF16, 20011, 1024, 2304, (PAIR, 256)), (BF16, 40011, 1032, 200, (PAIR, 256)), (F16, 20011, 1040, 520, (PAIR, 256)),
    (BF16, 90011, 64, 100, (SINGLE, 128)), (BF16, 60011, 64, 200, (SINGLE, 256)), (F16, 60011, 72, 520, (SINGLE, 256)),
    (E4M3, 90011, 128, 100, (SINGLE, 128)), (E4M3, 60011, 144, 200, (SINGLE, 256)),
    (E4M3, 20011, 2048, 1000, (PAIR, 256)), (E4M3, 40011, 2064, 136, (PAIR, 256)),
    (BF16, 50011, 64, 40, (SINGLE, 64)), (E4M3, 50011, 64, 40, (SINGLE, 64)),
]


def _call(x, w, b, r, act, out, g):
    """y and the 64-bit operands that it stands for (8 bits: power-of-two scales)."""
    if x.dtype == E4M3:
        sx = 2.0 ** torch.randint(-2, 3, (x.shape[0],), generator=g, device="cuda").float()
        sw = 2.0 ** torch.randint(-2, 3, (w.shape[0],), generator=g, device="cuda").float()
        return ml.linear_act_fp8(x, sx, w, sw, b, r, act, out), x.to(D) * sx[:, None], w.to(D) * sw[:, None]
    return ml.linear_act(x, w, b, r, act, out), x.to(D), w.to(D)


@pytest.mark.parametrize("dtype,rows,k,n,form", FORWARDS)
def test_forward_forms_on_integers(dtype, rows, k, n, form):
    _form(FORWARD, rows, n, k, dtype, form)
    g = _gen(rows + k + n)
    x, w = _ints(g, rows, k, lo=-1, hi=2).to(dtype), _ints(g, n, k, lo=-1, hi=2).to(dtype)
    half = BF16 if dtype == E4M3 else dtype
    for out, act, use in ((half, "relu", True), (F32, "none", True), (half, "none", False)):
        b = _ints(g, n).to(out) if use else None
        r = _ints(g, rows, n).to(out) if use else None
        y, xd, wd = _call(x, w, b, r, act, out, g)
        want = xd @ wd.T
        if use:
            want = _act(want + b.to(D), act) + r.to(D)
        assert torch.equal(y, want.to(out))
    # a residual whose rows no 16-byte boundary divides comes by plain loads
    wide = _ints(g, rows, n + 1).to(half)
    y, xd, wd = _call(x, w, None, wide[:, 1:], "none", half, g)
    assert torch.equal(y, (xd @ wd.T + wide[:, 1:].to(D)).to(half))
    _no_fault()


@pytest.mark.parametrize("dtype,rows,k,n,form", FORWARDS)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_forward_forms_against_64_bits(dtype, rows, k, n, form, act):
    _form(FORWARD, rows, n, k, dtype, form)
    g = _gen(rows + 3 * k + n)
    x, w = _randn(g, rows, k), _randn(g, n, k, scale=k**-0.5)
    out = BF16 if dtype == E4M3 else dtype
    b, r = _randn(g, n).to(out), _randn(g, rows, n).to(out)
    if dtype == E4M3:
        (x, sx), (w, sw) = ml.quantize_rows_fp8(x), ml.quantize_rows_fp8(w)
        y = ml.linear_act_fp8(x, sx, w, sw, b, r, act, out)
        xd, wd = x.to(D) * sx[:, None], w.to(D) * sw[:, None]
    else:
        x, w = x.to(dtype), w.to(dtype)
        y, xd, wd = ml.linear_act(x, w, b, r, act), x.to(D), w.to(D)
    want, bound, _, _ = _linear_bounds(xd, wd, b.to(D), r.to(D), act, out)
    _within(y, want, bound)
    _no_fault()


@pytest.mark.parametrize("rows,k,n", [(20, 2048, 300), (32, 1000, 256), (50, 2048, 200), (64, 4096, 72), (300, 4096, 264),
                                      (1000, 4096, 264), (9, 2048, 300)])
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F16, F32), (E4M3, BF16), (E4M3, F32)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_few_rows_with_a_split_reduction(rows, k, n, dtype, out, act):
    """Every tile height of the few-row form with its reduction over a cluster."""
    tile = 16 if rows <= 16 else 32 if rows <= 32 else 64 if rows <= 64 else 128
    if (dtype, rows) == (E4M3, 1000):
        rows = 900  # of 8-bit values: 32 stages, so 32 tiles at most
    _form(FORWARD, rows, n, k, dtype, (FEW, tile), parts=2, rounds=1)
    g = _gen(rows + k + n)
    x, w = _ints(g, rows, k, lo=-1, hi=2).to(dtype), _ints(g, n, k, lo=-1, hi=2).to(dtype)
    b, r = _ints(g, n).to(out), _ints(g, rows, n).to(out)
    if act == "none":
        y, xd, wd = _call(x, w, b, r, act, out, g)
        assert torch.equal(y, (xd @ wd.T + b.to(D) + r.to(D)).to(out))
    else:
        x, w = _randn(g, rows, k), _randn(g, n, k, scale=k**-0.5)
        if dtype == E4M3:
            (x, sx), (w, sw) = ml.quantize_rows_fp8(x), ml.quantize_rows_fp8(w)
            y = ml.linear_act_fp8(x, sx, w, sw, b, r, act, out)
            xd, wd = x.to(D) * sx[:, None], w.to(D) * sw[:, None]
        else:
            x, w = x.to(dtype), w.to(dtype)
            y, xd, wd = ml.linear_act(x, w, b, r, act, out), x.to(D), w.to(D)
        want, bound, _, _ = _linear_bounds(xd, wd, b.to(D), r.to(D), act, out)
        _within(y, want, bound)
    _no_fault()


def _check_grads(x, w, b, dy, act, out):
    """dx, dweight, dbias of integers: equal to the 64-bit ones rounded once.
    Where fp16 has no room for a sum, both round to infinity."""
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ml.linear_act(*leaves, activation=act, out_dtype=out)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    xd, wd, dyd = x.detach().to(D), w.detach().to(D), dy.to(D)
    z = xd @ wd.T + b.detach().to(D)
    dz = dyd * _act_grad(z, act)
    assert torch.equal(y, _act(z, act).to(out))
    for got, want in ((dx, dz @ wd), (dw, dz.T @ xd), (db, dz.sum(0))):
        assert torch.equal(got, want.to(got.dtype))
    _no_fault()


DERIVATIVES = [
    # 256 columns on single CTAs: the groups take slabs out of turn
    (BF16, 262144 + 77, 64, 256, (SINGLE, 256)), (F16, 60011, 64, 520, (SINGLE, 256)), (BF16, 60011, 72, 200, (SINGLE, 256)),
    (F16, 20011, 1024, 520, (PAIR, 256)), (F16, 40011, 1032, 200, (PAIR, 256)),
    (BF16, 90011, 64, 100, (SINGLE, 128)), (F16, 50011, 64, 40, (SINGLE, 64)),
]


@pytest.mark.parametrize("dtype,rows,k,n,form", DERIVATIVES)
def test_derivative_pass_forms(dtype, rows, k, n, form):
    """relu, so that dz is an integer; upstream gradients by TMA, by plain loads
    (rows 2 bytes past a boundary) and in fp32."""
    _form(DERIVATIVE, rows, n, k, dtype, form)
    g = _gen(rows + 5 * k + n)
    x, w, b = _ints(g, rows, k, lo=-1, hi=2), _ints(g, n, k, lo=-1, hi=2), _ints(g, n)
    dy = _ints(g, rows, n + 1, lo=-1, hi=2)
    for out, up in ((dtype, dy[:, 1:].contiguous().to(dtype)), (dtype, dy.to(dtype)[:, 1:]), (F32, dy[:, 1:].contiguous()),
                    (F32, dy[:, 1:])):
        _check_grads(x.to(dtype), w.to(dtype), b.clone(), up, "relu", out)


@pytest.mark.parametrize("product,dtype,rows,k,n,form", [
    (DX, BF16, 40011, 200, 1032, (PAIR, 256)), (DX, F16, 60011, 520, 64, (SINGLE, 256)), (DX, BF16, 90011, 100, 64, (SINGLE, 128)),
    (DWEIGHT, BF16, 40011, 200, 1024, (PAIR, 256)), (DWEIGHT, F16, 40011, 200, 1032, (SINGLE, 256)),
    (DWEIGHT, BF16, 200011, 64, 64, (SINGLE, 64)), (DWEIGHT, BF16, 30011, 130, 2000, None),
    (DWEIGHT, BF16, 3000, 2056, 2056, None),
])
def test_gradient_product_forms(product, dtype, rows, k, n, form):
    if form is not None:
        _form(product, rows, n, k, dtype, form, parts=2 if product == DWEIGHT else None, rounds=1 if product == DWEIGHT else 2)
    g = _gen(rows + 7 * k + n)
    x, w, b = _ints(g, rows, k, lo=-1, hi=2), _ints(g, n, k, lo=-1, hi=2), _ints(g, n)
    _check_grads(x.to(dtype), w.to(dtype), b, _ints(g, rows, n, lo=-1, hi=2).to(dtype), "none", dtype)


@pytest.mark.parametrize("rows,k,n,form", [(40011, 512, 200, (SINGLE, 256)), (20011, 576, 520, (SINGLE, 256)),
                                           (40011, 1024, 200, (PAIR, 256)), (20011, 1088, 520, (PAIR, 256))])
@pytest.mark.parametrize("act", ["relu", "gelu"])
def test_keeping_forward_forms(rows, k, n, form, act):
    _form(FORWARD, rows, n, k, BF16, form)
    assert _core.linear_act_kept_bytes(rows, n, k, _core.BF16, _core.BF16, _core.BF16, getattr(_core, f"ACT_{act.upper()}"))
    g = _gen(rows + k + n)
    if act == "relu":
        x, w, b = _ints(g, rows, k, lo=-1, hi=2), _ints(g, n, k, lo=-1, hi=2), _ints(g, n)
        _check_grads(x.to(BF16), w.to(BF16), b.to(BF16), _ints(g, rows, n, lo=-1, hi=2).to(BF16), act, BF16)
        return
    x, w, b = (t.requires_grad_() for t in (_randn(g, rows, k).to(BF16), _randn(g, n, k, scale=k**-0.5).to(BF16),
                                             _randn(g, n).to(BF16)))
    y = ml.linear_act(x, w, b, activation=act)
    with torch.no_grad():
        assert torch.equal(y, ml.linear_act(x, w, b, activation=act))
    dy = _randn(g, rows, n).to(BF16)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    x, w, b, dy = (t.detach().to(D) for t in (x, w, b, dy))
    _, _, z, ez = _linear_bounds(x, w, b, None, act, BF16)
    d = _act_grad(z, act)
    dz = dy * d
    # the kept derivative: its evaluation and its rounding (2**-11 of the value, 2**-37)
    edz = dy.abs() * (1.1 * ez + 2.0**-19 + d.abs() * 2.0**-11 + 2.0**-37) * 1.01 + 2.0**-23 * dz.abs()
    edz16 = edz * (1 + 2.0**-8) + _half_step(dz, BF16) * (1 + 2.0**-10)
    mag = dz.abs() + edz16
    for got, want, e, mass, terms in ((dx, dz @ w, edz16 @ w.abs(), mag @ w.abs(), n),
                                      (dw, dz.T @ x, edz16.T @ x.abs(), mag.T @ x.abs(), rows),
                                      (db, dz.sum(0), edz.sum(0), (dz.abs() + edz).sum(0), rows)):
        _within(got, want, _half_step(want, BF16) * (1 + 2.0**-8) + (e + (terms + 4) * 2.0**-23 * mass) * 1.01)
    _no_fault()


@pytest.mark.parametrize("dtype,rows,k,n", [(BF16, 30011, 256, 256), (F16, 20011, 1024, 520)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_derivative_pass_against_64_bits(dtype, rows, k, n, act):
    """An fp32 bias keeps nothing: z is formed again, with real-valued dz."""
    g = _gen(rows + k + n)
    x, w, b = (t.requires_grad_() for t in (_randn(g, rows, k).to(dtype), _randn(g, n, k, scale=k**-0.5).to(dtype), _randn(g, n)))
    dy = _randn(g, rows, n).to(dtype)
    dx, dw, db = torch.autograd.grad(ml.linear_act(x, w, b, activation=act), [x, w, b], dy)
    x, w, b, dy = (t.detach().to(D) for t in (x, w, b, dy))
    _, _, z, ez = _linear_bounds(x, w, b, None, act, dtype)
    dz = dy * _act_grad(z, act)
    edz = dy.abs() * (1.1 * ez + 2.0**-19) + 2.0**-23 * dz.abs()
    edz16 = edz * 1.01 + _half_step(dz, dtype) * (1 + 2.0**-10)
    mag = dz.abs() + edz16
    for got, want, e, mass, terms, t in ((dx, dz @ w, edz16 @ w.abs(), mag @ w.abs(), n, dtype),
                                         (dw, dz.T @ x, edz16.T @ x.abs(), mag.T @ x.abs(), rows, dtype),
                                         (db, dz.sum(0), edz.sum(0), (dz.abs() + edz).sum(0), rows, F32)):
        _within(got, want, _half_step(want, t) * (1 + 2.0**-8) + (e + (terms + 4) * 2.0**-23 * mass) * 1.01)
    _no_fault()
