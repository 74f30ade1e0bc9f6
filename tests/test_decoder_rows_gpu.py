"""The norms with more rows than the launch has groups: each warp group or block
goes through several rows, loads the next ones ahead and reuses its shared
slots. Against 64 bits, with the bounds of test_decoder_gpu.py; every row is
checked.
"""

from __future__ import annotations

import pytest
import torch
from test_decoder_gpu import _gen, _half_step, _norm_bounds, _randn, _within

from quantem.cuda import _core
from quantem.cuda.core import ml

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
D = torch.float64

# (rows, width): groups of 4, 8, 16 and 32 lanes, of one to eight vectors; odd widths (a group keeps to
# rows of one remainder); blocks of 256 and 512 threads, odd ones; the strided kernel. 148 SMs hold
# 75776 groups of 4 lanes, 9472 warps, 1184 blocks of 256 threads, 296 of the strided kernel.
ROWS = [(200003, 32), (100003, 64), (60001, 128), (60001, 256), (30001, 512), (30001, 1000), (100001, 30), (60001, 77),
        (30001, 999), (5003, 2048), (5003, 4097), (3001, 8192), (2003, 16384), (1501, 16400), (1501, 20001)]


def _inputs(rows, n, x_type):
    g = _gen(rows + n)
    x = (_randn(g, rows, n) * torch.exp(0.5 * _randn(g, rows, 1))).to(x_type)
    return x, _randn(g, rows, n).to(x_type), (1 + _randn(g, n, scale=0.3)).to(x_type), g


@pytest.mark.parametrize("rows,n", ROWS)
@pytest.mark.parametrize("x_type,out", [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F16)])
def test_norm_of_many_rows(rows, n, x_type, out):
    x, res, w, _ = _inputs(rows, n, x_type)
    for r in (None, res):
        got = ml.rms_norm(x, w, 1e-5, out) if r is None else ml.add_rms_norm(x, r, w, 1e-5, out)
        _, _, y, bound = _norm_bounds(x.to(D), None if r is None else r.to(D), w.to(D), 1e-5, out)
        _within(got if r is None else got[0], y, bound)
        if r is not None:
            assert torch.equal(got[1], (x.float() + r.float()).to(x_type))


@pytest.mark.parametrize("rows,n", ROWS)
@pytest.mark.parametrize("x_type", [F32, BF16, F16])
def test_8_bit_rows_of_many_rows(rows, n, x_type):
    x, res, w, _ = _inputs(rows, n, x_type)
    for kind in ("norm", "added", "plain"):
        if kind == "plain":
            (q, s), y, rel = ml.quantize_rows_fp8(x), x.to(D), 0.0
        else:
            r = res if kind == "added" else None
            if r is None:
                q, s = ml.rms_norm_fp8(x, w, 1e-5)
            else:
                q, s, h = ml.add_rms_norm_fp8(x, r, w, 1e-5)
                assert torch.equal(h, (x.float() + r.float()).to(x_type))
            y = _norm_bounds(x.to(D), None if r is None else r.to(D), w.to(D), 1e-5, F32)[2]
            rel = (n + 16) * 2.0**-24
        # the sum h is off by half a step of the larger summand where it cancels: 2**-24 of the row's largest
        slack = 2.0**-19 if kind == "added" else 0.0
        want = (y.abs().amax(-1) / 448).clamp_min(2.0**-126)
        _within(s, want, want * (rel + 2.0**-22 + slack))
        sd = s.to(D)[:, None]
        bound = torch.maximum(2.0**-4 * y.abs(), 2.0**-10 * sd) * (1 + 2.0**-12) + y.abs() * (rel + 2.0**-21)
        _within(q.to(D) * sd, y, bound + sd * 448 * slack)


@pytest.mark.parametrize("rows,n", ROWS)
@pytest.mark.parametrize("x_type,out", [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F16)])
def test_norm_gradients_of_many_rows(rows, n, x_type, out):
    """dweight of a row left out or taken twice would be off by that row's whole
    part. Its sum has, over the rows of a group, a block's groups and the blocks,
    at most rows/296 + 64 + 80 additions in a row (and each term the row's own
    factor, n + 40): 2**-24 of the terms each."""
    x, res, w, g = _inputs(rows, n, x_type)
    x, w = x.requires_grad_(), w.requires_grad_()
    dy, dh = _randn(g, rows, n).to(out), _randn(g, rows, n).to(x_type)
    for added in (False, True):
        if added:
            res.requires_grad_()
            y, h = ml.add_rms_norm(x, res, w, 1e-5, out)
            dx, dr, dw = torch.autograd.grad([y, h], [x, res, w], [dy, dh])
            assert torch.equal(dx, dr)
            h = x.detach().to(D) + res.detach().to(D)
        else:
            dx, dw = torch.autograd.grad(ml.rms_norm(x, w, 1e-5, out), [x, w], dy)
            h = x.detach().to(D)
        wd, dyd = w.detach().to(D), dy.to(D)
        r = 1 / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + 1e-5)
        gd = dyd * wd
        want = r * (gd - h * r * r * (gd * h).mean(-1, keepdim=True))
        size = r * (gd.abs() + h.abs() * r * r * (gd * h).abs().mean(-1, keepdim=True))
        if added:
            want, size = want + dh.to(D), size + dh.to(D).abs()
        _within(dx, want, (3 * n + 40) * 2.0**-24 * size + _half_step(want, x_type) * (1 + 2.0**-10), "dx")
        terms = dyd * h * r
        rel = (n + 40 + rows / 296 + 64 + 80) * 2.0**-24
        want = terms.sum(0)
        _within(dw, want, rel * terms.abs().sum(0) + _half_step(want, x_type) * (1 + 2.0**-10), "dweight")


@pytest.mark.parametrize("rows,n", [(60001, 77), (30001, 999), (60001, 128), (5003, 4097)])
def test_weight_gradients_of_integers_are_exact(rows, n):
    """h of +-2 has r = 1/2 exactly (eps = 0), so dweight is a sum of integers:
    every row counts once."""
    g = _gen(rows)
    x = (4.0 * torch.randint(0, 2, (rows, n), generator=g, device="cuda").float() - 2).requires_grad_()
    w = torch.ones(n, device="cuda", requires_grad=True)
    dy = torch.randint(-3, 4, (rows, n), generator=g, device="cuda").float()
    y = ml.rms_norm(x, w, 0.0)
    assert torch.equal(y, x.detach().sign())
    dw, = torch.autograd.grad(y, [w], dy)
    assert torch.equal(dw.to(D), (dy.to(D) * x.detach().sign().to(D)).sum(0))


def test_no_fault():
    torch.cuda.synchronize()
    assert _core.device_fault_word(0, True) == 0
