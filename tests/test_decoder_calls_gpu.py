"""How the decoder operators may be called on the device: missing tensors are
refused, forward-mode derivatives are refused, recorded graphs hold the
operators."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.func import functionalize
from torch.fx.experimental.proxy_tensor import make_fx

from quantem.cuda.core import ml

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _inputs(rows=40, k=64, n=72):
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w, nw = (torch.randn(s, generator=g, device="cuda").to(BF16) for s in ((rows, k), (n, k), (k,)))
    return x, w, nw


@pytest.mark.parametrize("call", [
    lambda x, w: ml.rms_norm(x, None),
    lambda x, w: ml.add_rms_norm(x, x, None),
    lambda x, w: ml.rms_norm_fp8(x, None),
    lambda x, w: ml.add_rms_norm_fp8(x, x, None),
    lambda x, w: ml.quantize_rows_fp8(None),
    lambda x, w: ml.linear_act(x, None),
    lambda x, w: ml.linear_act(None, w),
    lambda x, w: ml.linear_act_fp8(x, None, w, None),
    lambda x, w: ml.linear_act_fp8(*ml.quantize_rows_fp8(x.detach()), ml.quantize_rows_fp8(w)[0], None),
    lambda x, w: ml.linear_act_fp8(ml.quantize_rows_fp8(x.detach())[0], None, *ml.quantize_rows_fp8(w)),
    lambda x, w: ml.linear_act_fp8(ml.quantize_rows_fp8(x.detach())[0], None, ml.quantize_rows_fp8(w)[0], None),
])
def test_missing_tensors_are_refused(call):
    x, w, _ = _inputs()
    with pytest.raises(TypeError):
        call(x, w)
    with pytest.raises(TypeError):
        call(x.requires_grad_(), w)


def _chain(x, w, nw):
    y, h = ml.add_rms_norm(x, x, nw)
    q, s = ml.rms_norm_fp8(x, nw)
    q8 = ml.linear_act_fp8(q, s, *ml.quantize_rows_fp8(w))
    return ml.linear_act(ml.rms_norm(h, nw), w, residual=q8, activation="gelu") + ml.linear_act(y, w)


def test_forward_mode_derivatives_are_refused():
    """A tangent is neither dropped in a call nor in a backward; without one a
    call inside a forward-mode level gives its usual values."""
    x, w, nw = _inputs()
    want = _chain(x, w, nw)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ml.rms_norm(dual, nw), lambda: ml.add_rms_norm(x, dual, nw), lambda: ml.rms_norm_fp8(dual, nw),
                     lambda: ml.quantize_rows_fp8(dual), lambda: ml.linear_act(dual, w), lambda: ml.linear_act(x, dual),
                     lambda: ml.linear_act(x, w, residual=fwd.make_dual(want, want))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert torch.equal(_chain(x, w, nw), want)
    xs = x.clone().requires_grad_()
    for y in (ml.rms_norm(xs, nw), ml.linear_act(xs, w, activation="silu")):
        want, = torch.autograd.grad(y, [xs], torch.ones_like(y), retain_graph=True)
        with fwd.dual_level():
            dy = torch.ones_like(y)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, [xs], fwd.make_dual(dy, dy), retain_graph=True)
            got, = torch.autograd.grad(y, [xs], dy)
        assert torch.equal(got, want)


@pytest.mark.parametrize("record", [
    lambda f, a: make_fx(f)(*a),
    lambda f, a: make_fx(f, pre_dispatch=True)(*a),
    lambda f, a: torch.jit.trace(f, a),
], ids=["make_fx", "make_fx_pre_dispatch", "jit_trace"])
def test_recorded_calls_hold_the_operators(record):
    """A graph recorded on some inputs gives other inputs' results."""
    a = _inputs()
    graph = record(_chain, a)
    other = tuple(t.flip(0).contiguous() for t in a)
    for args in (a, other):
        assert torch.equal(graph(*args), _chain(*args))

    def step(x, w, nw):
        xs, ws, ns = (t.detach().requires_grad_() for t in (x, w, nw))
        y = ml.linear_act(ml.rms_norm(xs, ns), ws, activation="gelu")
        return torch.autograd.grad(y, [xs, ws, ns], torch.ones_like(y))

    if record.__code__.co_names[0] == "make_fx":
        graph = make_fx(step)(*a)
        for args in (a, other):
            for got, want in zip(graph(*args), step(*args)):
                assert torch.equal(got, want)


def test_backward_recorded_apart_from_its_forward():
    """The eager forward's backward inside make_fx (of a large bf16 call, too,
    which kept the derivative: the recorded one forms it again)."""
    for rows, k in ((40, 64), (600, 512)):
        x, w, nw = _inputs(rows, k)
        w, nw = w.requires_grad_(), nw.requires_grad_()
        y = ml.linear_act(ml.rms_norm(x, nw), w, activation="silu")
        dy = torch.ones_like(y)
        want = torch.autograd.grad(y, [w, nw], dy, retain_graph=True)
        graph = make_fx(lambda d: torch.autograd.grad(y, [w, nw], d, retain_graph=True))(dy)
        assert any("quantem_cuda" in str(n.target) for n in graph.graph.nodes)
        for got, ref in zip(graph(2 * dy), want):
            assert (got.float() - 2 * ref.float()).norm() <= 2.0**-6 * ref.float().norm()


def test_transformed_tensors():
    """torch.func wraps its tensors: their address is null or cannot be asked
    for. None is taken for a missing argument; torch.func's own gradients and vmap
    are refused."""
    x, w, nw = _inputs()
    b, r = w[:, 0].contiguous(), torch.randn(40, 72, device="cuda").to(BF16)
    want = ml.linear_act(x, w, b, r, "silu")
    assert torch.equal(functionalize(lambda t: ml.linear_act(x, w, t, r, "silu"))(b), want)
    assert torch.equal(functionalize(lambda t: ml.linear_act(x, w, b, t, "silu"))(r), want)
    assert torch.equal(functionalize(lambda t: ml.linear_act(t, w, b, r, "silu"))(x), want)
    want = ml.add_rms_norm(x, x, nw)
    for got in (functionalize(lambda t: ml.add_rms_norm(x, t, nw))(x), functionalize(lambda t: ml.add_rms_norm(x, x, t))(nw)):
        assert all(torch.equal(a, c) for a, c in zip(got, want))

    def loss(t):
        return ml.linear_act(ml.rms_norm(t, nw), w, b, activation="gelu", out_dtype=F32).square().sum()

    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.grad(loss)(x)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda t: ml.rms_norm(t, nw))(x)


def test_calls_under_a_function_mode():
    """torch.device as a context is one; the values are the same."""
    a = _inputs()
    want = _chain(*a)
    with torch.device("cuda"):
        assert torch.equal(_chain(*a), want)
