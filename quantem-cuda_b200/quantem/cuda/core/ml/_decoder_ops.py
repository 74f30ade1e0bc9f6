"""Operators of a decoder behind the K-Planes features: the root-mean-square
norm with the residual's addition and the matrix product with bias, activation
and residual in its epilogue, in 16 bits with their backward passes and in 8
bits (e4m3 with scales) for serving.

    quantem_cuda::rms_norm(x, residual?, weight, eps, out_dtype?) -> Tensor[]      [y] or [y, h]
    quantem_cuda::rms_norm_bwd(x, residual?, weight, dy, dh?, eps) -> Tensor[]     [dx, dweight]
    quantem_cuda::rms_norm_fp8(x, residual?, weight, eps) -> Tensor[]              [q, scale] or [q, scale, h]
    quantem_cuda::quantize_rows_fp8(x) -> (q, scale)
    quantem_cuda::linear_act(x, weight, bias?, residual?, activation, out_dtype?) -> Tensor
    quantem_cuda::linear_act_bwd(x, weight, bias?, dy, activation, need) -> Tensor[]
    quantem_cuda::linear_act_fp8(x, x_scale, weight, weight_scale, bias?, residual?, activation, out_dtype) -> Tensor

The features come as fp32 ``[points, T*C]``; the norm's ``out_dtype`` takes
them to the decoder's type. As in the K-Planes layer, the public wrappers call
the implementations directly when they run eagerly, and the registered ops
while a graph is recorded (``torch.compile``, ``make_fx``, ``torch.jit.trace``),
inside ``torch.func`` transforms and for tensor subclasses. Forward-mode derivatives are refused.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from quantem.cuda import _core

_CODE = {torch.float32: _core.F32, torch.bfloat16: _core.BF16, torch.float16: _core.F16,
         torch.float8_e4m3fn: _core.E4M3}
_ACT = {"none": _core.ACT_NONE, "relu": _core.ACT_RELU, "silu": _core.ACT_SILU, "gelu": _core.ACT_GELU}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_HALVES = (torch.bfloat16, torch.float16)
_FP8 = torch.float8_e4m3fn

_dispatch_modes = torch._C._len_torch_dispatch_stack

# The common calls (plain contiguous tensors on the current device, no modes)
# run in the extension from their checks to the launch; they return
# NotImplemented for anything else, which the functions below then check,
# convert or refuse. (_cuda_getCurrentRawStream gives the stream's handle;
# torch.cuda.current_stream builds a stream object first, 2 us of a 10 us call.)
_core.decoder_setup(Tensor, torch.nn.Parameter, (torch.float32, torch.bfloat16, torch.float16, _FP8), torch.uint8,
                    torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream, torch.is_grad_enabled, _ACT,
                    _dispatch_modes, torch._C._len_torch_function_stack, forward_ad)
_is_compiling = torch.compiler.is_compiling
_early_modes = torch._ops._len_torch_dispatch_stack_pre_dispatch
_trace = torch._C._get_tracing_state
_transform = torch._C._functorch.maybe_current_level


def _direct() -> bool:
    """Whether a call may pass torch's dispatcher by. Not while a graph is
    recorded, which would hold the outputs' allocations alone; not inside a
    forward-mode level, whose tangents those allocations would drop; not inside
    a torch.func transform, whose tensors may have no address."""
    return not (_is_compiling() or forward_ad._current_level >= 0 or _dispatch_modes() or _early_modes()
                or _trace() is not None or _transform() is not None)


def _no_forward_mode(fn: str, *tensors: Tensor | None) -> None:
    """Refuses tangents (the registered ops would drop them)."""
    if forward_ad._current_level < 0:
        return
    for x in tensors:
        if isinstance(x, Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise NotImplementedError(f"{fn} has no forward-mode derivative")


def _launch(entry, x: Tensor, *args) -> None:
    """Calls a C entry on x's device and its current stream."""
    device = x.get_device()
    if device == torch._C._cuda_getDevice():
        entry(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            entry(*args, torch._C._cuda_getCurrentRawStream(device))


_PLAIN = {Tensor, torch.nn.Parameter, type(None)}


def _plain(*tensors: Tensor | None) -> bool:
    """True for plain tensors and parameters of a direct call."""
    for x in tensors:
        if type(x) not in _PLAIN:
            return False
    return _direct()


def _wants_grad(*tensors: Tensor | None) -> bool:
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                return True
    return False


def _new(x: Tensor, shape, dtype: torch.dtype) -> Tensor:
    return x.new_empty(shape) if dtype is x.dtype else x.new_empty(shape, dtype=dtype)


def _no_backward(fn: str, *tensors: Tensor | None) -> None:
    if _wants_grad(*tensors):
        raise RuntimeError(f"{fn} has no backward: call it under torch.no_grad() or detach its inputs")


def _given(fn: str, **tensors) -> None:
    for name, x in tensors.items():
        if not isinstance(x, Tensor):
            raise TypeError(f"{fn}: {name} must be a tensor, got {type(x).__name__}")


def _check(fn: str, name: str, x: Tensor, shape: tuple[int, ...], dtypes: tuple[torch.dtype, ...],
           device: torch.device) -> None:
    if x.dtype not in dtypes:
        want = " or ".join(str(d).removeprefix("torch.") for d in dtypes)
        raise TypeError(f"{fn}: {name} must be {want}, got {x.dtype}")
    if x.shape != shape:
        raise ValueError(f"{fn}: {name} must be {list(shape)}, got {list(x.shape)}")
    if x.device != device:
        raise ValueError(f"{fn}: {name} is on {x.device}; all inputs must be on {device} (CUDA)")


def _check_rows(fn: str, name: str, x: Tensor, dtypes: tuple[torch.dtype, ...]) -> None:
    if x.dtype not in dtypes:
        want = ", ".join(str(d).removeprefix("torch.") for d in dtypes)
        raise TypeError(f"{fn}: {name} must be one of {want}, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{fn}: {name} must be [..., n] with n >= 1, got {list(x.shape)}")
    if not x.is_cuda:
        raise ValueError(f"{fn} requires CUDA tensors ({name} on {x.device}).")


def _rows(x: Tensor) -> tuple[Tensor, int, int]:
    """``[..., n]`` as rows of unit inner stride: the tensor that holds them, how
    many they are and how far apart; a view where the leading dimensions have
    one stride."""
    if x.is_contiguous():
        n = x.shape[-1]
        return x, x.numel() // n, n
    n = x.shape[-1]
    r = x if x.ndim == 2 else x.reshape(-1, n)
    if r.stride(1) != 1 and n > 1:
        r = r.contiguous()
    return r, r.shape[0], r.stride(0)


def _matrix(x: Tensor) -> tuple[Tensor, int, int]:
    """Rows that do not overlap, as the matrix product's operands need."""
    r, rows, stride = _rows(x)
    if rows > 1 and stride < x.shape[-1]:
        r = x.contiguous()
        stride = x.shape[-1]
    return r, rows, stride


def _ptr(x: Tensor | None) -> int:
    return 0 if x is None else x.data_ptr()


# ── root-mean-square norm ─────────────────────────────────────────────────


def _check_norm(fn: str, x: Tensor, residual: Tensor | None, weight: Tensor) -> None:
    _given(fn, x=x, weight=weight)
    _check_rows(fn, "x", x, _FLOATS)
    if residual is not None:
        _check(fn, "residual", residual, x.shape, (x.dtype,), x.device)
    _check(fn, "weight", weight, x.shape[-1:], (x.dtype,), x.device)


def _norm_out_dtype(fn: str, x: Tensor, out_dtype: torch.dtype | None) -> torch.dtype:
    out = x.dtype if out_dtype is None else out_dtype
    if out != x.dtype and out != torch.float32 and not (x.dtype == torch.float32 and out in _HALVES):
        raise TypeError(f"{fn}: out_dtype {out} from {x.dtype}: x's own type, float32, or from float32 a 16-bit type")
    return out


def _launch_norm(x: Tensor, residual: Tensor | None, weight: Tensor, y: Tensor, h: Tensor | None,
                 scale: Tensor | None, eps: float) -> None:
    x2, rows, stride = _rows(x)
    r2, _, r_stride = (None, 0, 0) if residual is None else _rows(residual)
    w = weight.contiguous()
    _launch(
        _core.rms_norm_cuda, x, x2.data_ptr(), _ptr(r2), w.data_ptr(), y.data_ptr(), _ptr(h), _ptr(scale), rows,
        x.shape[-1], stride, r_stride, _CODE[x.dtype], _CODE[y.dtype], eps,
    )


def _rms_norm_impl(fn: str, x: Tensor, residual: Tensor | None, weight: Tensor, eps: float,
                   out_dtype: torch.dtype | None) -> list[Tensor]:
    if out_dtype is not _FP8:
        outs = _core.decoder_norm(x, residual, weight, eps, out_dtype, False)
        if outs is not NotImplemented:
            return list(outs)
    _check_norm(fn, x, residual, weight)
    y = _new(x, x.shape, x.dtype if out_dtype is None else _norm_out_dtype(fn, x, out_dtype))
    h = None if residual is None else x.new_empty(x.shape)
    _launch_norm(x, residual, weight, y, h, None, eps)
    return [y] if h is None else [y, h]


def _rms_norm_bwd_impl(x: Tensor, residual: Tensor | None, weight: Tensor, dy: Tensor, dh: Tensor | None, eps: float,
                       need_dx: bool = True, need_dw: bool = True) -> tuple[Tensor | None, Tensor | None]:
    grads = _core.decoder_norm_grad(x, residual, weight, dy, dh, eps, need_dx, need_dw)
    if grads is not NotImplemented:
        return grads
    fn = "rms_norm_bwd"
    _check_norm(fn, x, residual, weight)
    _check(fn, "dy", dy, x.shape, _FLOATS if x.dtype == torch.float32 else (x.dtype, torch.float32), x.device)
    if dh is not None:
        _check(fn, "dh", dh, x.shape, (x.dtype,), x.device)
    x2, rows, stride = _rows(x)
    dy2, _, dy_stride = _rows(dy)
    r2, _, r_stride = (None, 0, 0) if residual is None else _rows(residual)
    dh2, _, dh_stride = (None, 0, 0) if dh is None else _rows(dh)
    w = weight.contiguous()
    n = x.shape[-1]
    dx = x.new_empty(x.shape) if need_dx else None
    dw = x.new_empty(weight.shape) if need_dw else None
    nbytes = _core.rms_norm_grad_workspace_bytes(rows, n) if need_dw else 0
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch(
        _core.rms_norm_grad_cuda, x, x2.data_ptr(), _ptr(r2), w.data_ptr(), dy2.data_ptr(), _ptr(dh2), _ptr(dx),
        _ptr(dw), rows, n, stride, r_stride, dy_stride, dh_stride, _CODE[x.dtype], _CODE[dy.dtype], eps, _ptr(ws),
        nbytes,
    )
    return dx, dw


def _norm_saved(x: Tensor, residual: Tensor | None, outs) -> tuple[Tensor, Tensor | None]:
    """What the backward forms h from: 16-bit rows x and residual again (the
    stored h has lost bits the weight's gradient would miss), fp32 rows h."""
    if residual is not None and x.dtype == torch.float32:
        return outs[1], None
    return x, residual


@torch.library.custom_op("quantem_cuda::rms_norm", mutates_args=())
def _rms_norm(x: Tensor, residual: Tensor | None, weight: Tensor, eps: float,
              out_dtype: torch.dtype | None) -> list[Tensor]:
    return _rms_norm_impl("rms_norm", x, residual, weight, eps, out_dtype)


@_rms_norm.register_fake
def _(x, residual, weight, eps, out_dtype):
    y = x.new_empty(x.shape, dtype=x.dtype if out_dtype is None else out_dtype)
    return [y] if residual is None else [y, x.new_empty(x.shape)]


@torch.library.custom_op("quantem_cuda::rms_norm_bwd", mutates_args=())
def _rms_norm_bwd(x: Tensor, residual: Tensor | None, weight: Tensor, dy: Tensor, dh: Tensor | None,
                  eps: float) -> list[Tensor]:
    return list(_rms_norm_bwd_impl(x, residual, weight, dy, dh, eps))


@_rms_norm_bwd.register_fake
def _(x, residual, weight, dy, dh, eps):
    return [x.new_empty(x.shape), weight.new_empty(weight.shape)]


def _rms_norm_setup(ctx, inputs, output) -> None:
    x, residual, weight, eps, _ = inputs
    ctx.eps, ctx.added = eps, residual is not None
    ctx.y_dtype = output[0].dtype
    ctx.save_for_backward(*_norm_saved(x, residual, output), weight)


def _rms_norm_backward(ctx, grads):
    x, residual, weight = ctx.saved_tensors
    dy = grads[0] if grads[0] is not None else torch.zeros(x.shape, dtype=ctx.y_dtype, device=x.device)
    dx, dw = _rms_norm_bwd(x, residual, weight, dy, grads[1] if ctx.added else None, ctx.eps)
    return dx, (dx if ctx.added else None), dw, None, None


_rms_norm.register_autograd(_rms_norm_backward, setup_context=_rms_norm_setup)


def _once(backward):
    """A backward that cannot be differentiated again. Where no second graph is
    asked for, once_differentiable's wrapping (3 us) is passed by."""
    wrapped = torch.autograd.function.once_differentiable(backward)

    def call(ctx, *grads):
        return (wrapped if torch.is_grad_enabled() else backward)(ctx, *grads)

    return call


class _RmsNorm(torch.autograd.Function):
    """Eager counterpart of the registered op: no torch.library dispatch."""

    @staticmethod
    def forward(ctx, fn: str, x: Tensor, residual: Tensor | None, weight: Tensor, eps: float,
                out_dtype: torch.dtype | None):
        outs = _rms_norm_impl(fn, x, residual, weight, eps, out_dtype)
        ctx.eps, ctx.added = eps, residual is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*_norm_saved(x, residual, outs), weight)
        return tuple(outs)

    @staticmethod
    @_once
    def backward(ctx, *grads):
        x, residual, weight = ctx.saved_tensors
        dy, dh = grads[0], grads[1] if ctx.added else None
        if dy is None and dh is None:
            return (None,) * 6
        _, need_x, need_r, need_w, _, _ = ctx.needs_input_grad
        if dy is None:  # only the sum h took part in the loss: its gradient passes through
            dw = torch.zeros(weight.shape, dtype=weight.dtype, device=weight.device) if need_w else None
            return None, dh if need_x else None, dh if need_r else None, dw, None, None
        if _direct():
            dx, dw = _rms_norm_bwd_impl(x, residual, weight, dy, dh, ctx.eps, need_x or need_r, need_w)
        else:
            _no_forward_mode("rms_norm_bwd", dy, dh)
            dx, dw = _rms_norm_bwd(x, residual, weight, dy, dh, ctx.eps)
        return None, dx if need_x else None, dx if need_r else None, dw, None, None


def _norm_call(fn: str, x: Tensor, residual: Tensor | None, weight: Tensor, eps: float,
               out_dtype: torch.dtype | None):
    eps = float(eps)
    if out_dtype is not _FP8 and not _is_compiling():
        outs = _core.decoder_norm(x, residual, weight, eps, out_dtype, True)
        if outs is None and _direct():  # plain tensors, a gradient is recorded
            return _RmsNorm.apply(fn, x, residual, weight, eps, out_dtype)
        if outs is not NotImplemented and outs is not None:
            return outs
    if not _plain(x, residual, weight):
        _no_forward_mode(fn, x, residual, weight)
        _check_norm(fn, x, residual, weight)
        _norm_out_dtype(fn, x, out_dtype)
        return _rms_norm(x, residual, weight, eps, out_dtype)
    if _wants_grad(x, residual, weight):
        return _RmsNorm.apply(fn, x, residual, weight, eps, out_dtype)
    return _rms_norm_impl(fn, x, residual, weight, eps, out_dtype)


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6, out_dtype: torch.dtype | None = None) -> Tensor:
    """Root-mean-square norm over the last dimension::

        y = x / sqrt(mean(x**2) + eps) * weight

    Differentiable w.r.t. ``x`` and ``weight`` (in reverse mode). Sums are fp32; ``y`` is rounded
    once. Gradients are the same from run to run.

    Args:
        x:         fp32, bf16 or fp16 CUDA tensor ``[..., n]`` (K-Planes
                   features ``[points, T*C]``, for instance); rows may be
                   strided.
        weight:    ``[n]``, of x's type.
        eps:       added to the mean square.
        out_dtype: type of ``y``: x's (default) or fp32; from fp32 also bf16 or
                   fp16.
    """
    return _norm_call("rms_norm", x, None, weight, eps, out_dtype)[0]


def add_rms_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float = 1e-6,
                 out_dtype: torch.dtype | None = None) -> tuple[Tensor, Tensor]:
    """Residual addition and root-mean-square norm in one pass::

        h = x + residual
        y = h / sqrt(mean(h**2) + eps) * weight

    Returns ``(y, h)``; ``h`` has x's type and is the next residual. ``y`` and
    the gradients are formed from the unrounded sum. The gradients of ``x`` and
    ``residual`` are one tensor. ``residual`` has x's shape and type (an expanded
    one is read in place). Otherwise as :func:`rms_norm`.
    """
    if residual is None:
        raise TypeError("add_rms_norm: residual is missing (rms_norm norms x alone)")
    y, h = _norm_call("add_rms_norm", x, residual, weight, eps, out_dtype)
    return y, h


# ── 8-bit rows ────────────────────────────────────────────────────────────


def _rms_norm_fp8_impl(fn: str, x: Tensor, residual: Tensor | None, weight: Tensor, eps: float) -> list[Tensor]:
    outs = _core.decoder_norm(x, residual, weight, eps, _FP8, False)
    if outs is not NotImplemented:
        return list(outs)
    _check_norm(fn, x, residual, weight)
    q = x.new_empty(x.shape, dtype=_FP8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    h = None if residual is None else x.new_empty(x.shape)
    _launch_norm(x, residual, weight, q, h, scale, eps)
    return [q, scale] if h is None else [q, scale, h]


@torch.library.custom_op("quantem_cuda::rms_norm_fp8", mutates_args=())
def _rms_norm_fp8(x: Tensor, residual: Tensor | None, weight: Tensor, eps: float) -> list[Tensor]:
    return _rms_norm_fp8_impl("rms_norm_fp8", x, residual, weight, eps)


@_rms_norm_fp8.register_fake
def _(x, residual, weight, eps):
    got = [x.new_empty(x.shape, dtype=_FP8), x.new_empty(x.shape[:-1], dtype=torch.float32)]
    return got if residual is None else [*got, x.new_empty(x.shape)]


def _quantize_impl(x: Tensor) -> tuple[Tensor, Tensor]:
    _given("quantize_rows_fp8", x=x)
    _check_rows("quantize_rows_fp8", "x", x, _FLOATS)
    x2, rows, stride = _rows(x)
    q = x.new_empty(x.shape, dtype=_FP8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    _launch(_core.quantize_rows_cuda, x, x2.data_ptr(), q.data_ptr(), scale.data_ptr(), rows, x.shape[-1], stride,
            _CODE[x.dtype])
    return q, scale


@torch.library.custom_op("quantem_cuda::quantize_rows_fp8", mutates_args=())
def _quantize_rows_fp8(x: Tensor) -> tuple[Tensor, Tensor]:
    return _quantize_impl(x)


@_quantize_rows_fp8.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=_FP8), x.new_empty(x.shape[:-1], dtype=torch.float32)


def _norm_fp8_call(fn: str, x: Tensor, residual: Tensor | None, weight: Tensor, eps: float):
    if not _is_compiling():
        outs = _core.decoder_norm(x, residual, weight, eps, _FP8, True)
        if outs is not NotImplemented and outs is not None:
            return outs
    _given(fn, x=x, weight=weight)
    _no_backward(fn, x, residual, weight)
    if not _plain(x, residual, weight):
        _no_forward_mode(fn, x, residual, weight)
        _check_norm(fn, x, residual, weight)
        return _rms_norm_fp8(x, residual, weight, eps)
    return _rms_norm_fp8_impl(fn, x, residual, weight, eps)


def rms_norm_fp8(x: Tensor, weight: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """:func:`rms_norm` with 8-bit output for :func:`linear_act_fp8`: returns
    ``(q, scale)`` with ``q`` e4m3 ``[..., n]`` and ``scale`` fp32 ``[...]``::

        scale = max(max|y| / 448, 2**-126)   (per row),   q = e4m3(y / scale)

    A row with a NaN or an infinity stands for NaN. No backward.
    """
    q, scale = _norm_fp8_call("rms_norm_fp8", x, None, weight, float(eps))
    return q, scale


def add_rms_norm_fp8(x: Tensor, residual: Tensor, weight: Tensor,
                     eps: float = 1e-6) -> tuple[Tensor, Tensor, Tensor]:
    """:func:`add_rms_norm` with 8-bit output: ``(q, scale, h)``. No backward."""
    if residual is None:
        raise TypeError("add_rms_norm_fp8: residual is missing (rms_norm_fp8 norms x alone)")
    q, scale, h = _norm_fp8_call("add_rms_norm_fp8", x, residual, weight, float(eps))
    return q, scale, h


def quantize_rows_fp8(x: Tensor) -> tuple[Tensor, Tensor]:
    """Rows of ``x`` (fp32, bf16 or fp16 ``[..., n]``) as e4m3 with one fp32
    scale per row, ``x ≈ q * scale[..., None]``: the weights ``[N, K]`` and
    inputs of :func:`linear_act_fp8`. No backward."""
    if not _is_compiling():
        outs = _core.decoder_quantize(x, True)
        if outs is not NotImplemented and outs is not None:
            return outs
    _no_backward("quantize_rows_fp8", x)
    if _plain(x):
        return _quantize_impl(x)
    _no_forward_mode("quantize_rows_fp8", x)
    return _quantize_rows_fp8(x)


# ── matrix product with epilogue ──────────────────────────────────────────


def _check_linear(fn: str, x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
                  out: torch.dtype, operand: tuple[torch.dtype, ...], outs: tuple[torch.dtype, ...],
                  biases: tuple[torch.dtype, ...]) -> None:
    _check_rows(fn, "x", x, operand)
    if weight.ndim != 2 or weight.shape[0] < 1:
        raise ValueError(f"{fn}: weight must be [N, K] with N >= 1, got {list(weight.shape)}")
    _check(fn, "weight", weight, (weight.shape[0], x.shape[-1]), (x.dtype,), x.device)
    if activation not in _ACT:
        raise ValueError(f"{fn}: activation must be one of {', '.join(_ACT)}, got {activation!r}")
    if out not in outs:
        want = " or ".join(str(d).removeprefix("torch.") for d in outs)
        raise TypeError(f"{fn}: out_dtype must be {want}, got {out}")
    if bias is not None:
        _check(fn, "bias", bias, weight.shape[:1], biases, x.device)
    if residual is not None:
        _check(fn, "residual", residual, (*x.shape[:-1], weight.shape[0]), (out,), x.device)


def _check_linear16(fn: str, x, weight, bias, residual, activation, out_dtype) -> torch.dtype:
    _given(fn, x=x, weight=weight)
    out = x.dtype if out_dtype is None else out_dtype
    _check_linear(fn, x, weight, bias, residual, activation, out, _HALVES, (x.dtype, torch.float32),
                  (x.dtype, torch.float32))
    return out


def _launch_linear(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, y: Tensor,
                   x_scale: Tensor | None, weight_scale: Tensor | None, activation: str) -> None:
    (x2, rows, sx), (w2, n, sw) = _matrix(x), _matrix(weight)
    r2, _, sr = (None, 0, 0) if residual is None else _rows(residual)
    b = None if bias is None else bias.contiguous()
    k = x.shape[-1]
    code = _CODE[x.dtype]
    px, pw = x2.data_ptr(), w2.data_ptr()
    ws, nbytes = None, 0
    if px % 16 or pw % 16 or sx % 16 or sw % 16:  # rows that may need a copy
        nbytes = _core.linear_act_workspace_bytes(px, pw, rows, n, k, sx, sw, code)
        ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch(
        _core.linear_act_cuda, x, px, pw, _ptr(b), _ptr(r2), y.data_ptr(), _ptr(x_scale), _ptr(weight_scale), rows, n,
        k, sx, sw, sr, code, _CODE[y.dtype], 0 if b is None else _CODE[b.dtype], _ACT[activation], _ptr(ws), nbytes,
    )


def _linear_impl(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
                 out_dtype: torch.dtype | None) -> Tensor:
    y = _core.decoder_linear(x, weight, bias, residual, None, None, activation, out_dtype, False)
    if y is not NotImplemented:
        return y
    out = _check_linear16("linear_act", x, weight, bias, residual, activation, out_dtype)
    y = _new(x, (*x.shape[:-1], weight.shape[0]), out)
    _launch_linear(x, weight, bias, residual, y, None, None, activation)
    return y


def _linear_bwd_impl(x: Tensor, weight: Tensor, bias: Tensor | None, dy: Tensor, activation: str,
                     need: tuple[bool, bool, bool]) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    grads = _core.decoder_linear_grad(x, weight, bias, dy, activation, *need)
    if grads is not NotImplemented:
        return grads
    fn = "linear_act_bwd"
    _check_linear16(fn, x, weight, bias, None, activation, None)
    _check(fn, "dy", dy, (*x.shape[:-1], weight.shape[0]), (x.dtype, torch.float32), x.device)
    (x2, rows, sx), (w2, n, sw), (dy2, _, sdy) = _matrix(x), _matrix(weight), _matrix(dy)
    b = None if bias is None else bias.contiguous()
    dx = x.new_empty(x.shape) if need[0] else None
    dw = weight.new_empty(weight.shape) if need[1] else None
    db = bias.new_empty(bias.shape) if need[2] and bias is not None else None
    px, pw, pdy, pdx, pdw, pdb = x2.data_ptr(), w2.data_ptr(), dy2.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db)
    shape = (rows, n, x.shape[-1], sx, sw, sdy, _CODE[x.dtype], _CODE[dy.dtype])
    act = _ACT[activation]
    with_ptrs = (px, pw, pdy, pdx, pdw, pdb, *shape, act)
    nbytes = _core.linear_act_grad_workspace_bytes(*with_ptrs, x.get_device())
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch(_core.linear_act_grad_cuda, x, px, pw, _ptr(b), pdy, pdx, pdw, pdb, *shape,
            0 if b is None else _CODE[b.dtype], act, _ptr(ws), nbytes)
    return dx, dw, db


@torch.library.custom_op("quantem_cuda::linear_act", mutates_args=())
def _linear_act(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
                out_dtype: torch.dtype | None) -> Tensor:
    return _linear_impl(x, weight, bias, residual, activation, out_dtype)


@_linear_act.register_fake
def _(x, weight, bias, residual, activation, out_dtype):
    return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=x.dtype if out_dtype is None else out_dtype)


@torch.library.custom_op("quantem_cuda::linear_act_bwd", mutates_args=())
def _linear_act_bwd(x: Tensor, weight: Tensor, bias: Tensor | None, dy: Tensor, activation: str,
                    need: list[bool]) -> list[Tensor]:
    """The wanted ones of [dx, dweight, dbias], in this order."""
    return [g for g in _linear_bwd_impl(x, weight, bias, dy, activation, tuple(need)) if g is not None]


@_linear_act_bwd.register_fake
def _(x, weight, bias, dy, activation, need):
    return [t.new_empty(t.shape) for t, wanted in zip((x, weight, bias), need) if wanted and t is not None]


def _linear_setup(ctx, inputs, output) -> None:
    x, weight, bias, _, activation, _ = inputs
    ctx.activation = activation
    ctx.save_for_backward(x, weight, bias)


def _linear_backward(ctx, dy):
    return _linear_backward_op(ctx, *ctx.saved_tensors, dy)


def _linear_backward_op(ctx, x, weight, bias, dy):
    nx, nw, nb, nr = ctx.needs_input_grad[:4]
    need = [nx, nw, nb and bias is not None]
    got = iter(_linear_act_bwd(x, weight, bias, dy, ctx.activation, need) if any(need) else [])
    dx, dw, db = (next(got) if wanted else None for wanted in need)
    return dx, dw, db, dy if nr else None, None, None


_linear_act.register_autograd(_linear_backward, setup_context=_linear_setup)


class _LinearAct(torch.autograd.Function):
    """Eager counterpart of the registered op."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, out_dtype):
        ctx.activation = activation
        kept = None
        if any(ctx.needs_input_grad[:3]):
            outs = _core.decoder_linear_keep(x, weight, bias, residual, activation, out_dtype)
            if outs is not NotImplemented:
                y, kept = outs
        ctx.save_for_backward(x, weight, bias, kept)
        return _linear_impl(x, weight, bias, residual, activation, out_dtype) if kept is None else y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, bias, kept = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if not _direct():
            _no_forward_mode("linear_act_bwd", dy)
            return _linear_backward_op(ctx, x, weight, bias, dy)
        if kept is not None and (nx or nw or nb):
            grads = _core.decoder_linear_grad_kept(x, weight, kept, dy, ctx.activation, nx, nw, nb)
            if grads is not NotImplemented:
                return *grads, dy if nr else None, None, None
        if nx or nw or nb:
            dx, dw, db = _linear_bwd_impl(x, weight, bias, dy, ctx.activation, (nx, nw, nb))
        return dx, dw, db, dy if nr else None, None, None


def linear_act(x: Tensor, weight: Tensor, bias: Tensor | None = None, residual: Tensor | None = None,
               activation: str = "none", out_dtype: torch.dtype | None = None) -> Tensor:
    """Matrix product with bias, activation and residual in its epilogue::

        y = activation(x @ weight.T + bias) + residual

    Differentiable w.r.t. ``x``, ``weight``, ``bias`` and ``residual``. The
    backward forms the activation's argument again; large bf16 calls keep its
    derivative instead (2 bytes per output until the backward). It rounds
    dz = dy activation'(z) to x's type before the products with weight and x; fp32
    gradients of fp16 calls are scaled by a power of two for it (dz below 2**-39
    of the largest dy is lost), fp16 ones beyond 57000 may overflow. Its
    workspace holds dz and partial sums of weight's gradient (2 GB for a million
    rows of 4096 by 4096). No forward-mode derivative. Products
    run on the tensor cores with fp32 accumulation, the epilogue is fp32, and
    ``y`` is rounded once. Sums over rows are taken in a fixed order: outputs
    and gradients are the same from run to run.

    Args:
        x:          bf16 or fp16 CUDA tensor ``[..., K]``; rows may be strided.
        weight:     ``[N, K]`` of x's type.
        bias:       ``[N]``, x's type or fp32.
        residual:   ``[..., N]`` of the output's type, added after the activation.
        activation: ``"none"``, ``"relu"``, ``"silu"`` (z·sigmoid(z)) or
                    ``"gelu"`` (z·Φ(z), the exact form).
        out_dtype:  x's type (default) or fp32.

    Widths and addresses that no 16-byte boundary divides are handled by a copy
    of the operand to padded rows; multiples of 8 features avoid it.
    """
    if not _is_compiling():
        y = _core.decoder_linear(x, weight, bias, residual, None, None, activation, out_dtype, True)
        if y is None and _direct():  # plain tensors, a gradient is recorded
            return _LinearAct.apply(x, weight, bias, residual, activation, out_dtype)
        if y is not NotImplemented and y is not None:
            return y
    if not _plain(x, weight, bias, residual):
        _no_forward_mode("linear_act", x, weight, bias, residual)
        _check_linear16("linear_act", x, weight, bias, residual, activation, out_dtype)
        return _linear_act(x, weight, bias, residual, activation, out_dtype)
    if _wants_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, activation, out_dtype)
    return _linear_impl(x, weight, bias, residual, activation, out_dtype)


def _check_linear8(x, x_scale, weight, weight_scale, bias, residual, activation, out_dtype) -> None:
    fn = "linear_act_fp8"
    _given(fn, x=x, x_scale=x_scale, weight=weight, weight_scale=weight_scale)
    _check_linear(fn, x, weight, bias, residual, activation, out_dtype, (_FP8,), _FLOATS, _FLOATS)
    _check(fn, "x_scale", x_scale, x.shape[:-1], (torch.float32,), x.device)
    _check(fn, "weight_scale", weight_scale, weight.shape[:1], (torch.float32,), x.device)


def _linear8_impl(x, x_scale, weight, weight_scale, bias, residual, activation, out_dtype) -> Tensor:
    _check_linear8(x, x_scale, weight, weight_scale, bias, residual, activation, out_dtype)
    y = x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype)
    _launch_linear(x, weight, bias, residual, y, x_scale.contiguous(), weight_scale.contiguous(), activation)
    return y


@torch.library.custom_op("quantem_cuda::linear_act_fp8", mutates_args=())
def _linear_act_fp8(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Tensor | None,
                    residual: Tensor | None, activation: str, out_dtype: torch.dtype) -> Tensor:
    return _linear8_impl(x, x_scale, weight, weight_scale, bias, residual, activation, out_dtype)


@_linear_act_fp8.register_fake
def _(x, x_scale, weight, weight_scale, bias, residual, activation, out_dtype):
    return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype)


def linear_act_fp8(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Tensor | None = None,
                   residual: Tensor | None = None, activation: str = "none",
                   out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """:func:`linear_act` on 8-bit operands with scales, for serving::

        y = activation((x @ weight.T) * x_scale[..., None] * weight_scale + bias) + residual

    Args:
        x, x_scale:           e4m3 ``[..., K]`` and fp32 ``[...]``
                              (:func:`rms_norm_fp8`, :func:`quantize_rows_fp8`).
        weight, weight_scale: e4m3 ``[N, K]`` and fp32 ``[N]``
                              (:func:`quantize_rows_fp8`, once per weight).
        bias:                 ``[N]``, fp32, bf16 or fp16.
        residual:             ``[..., N]`` of the output's type.
        out_dtype:            bf16 (default), fp16 or fp32.

    Accumulation and epilogue are fp32, rounded once. No backward.
    """
    if x_scale is not None and not _is_compiling():  # without scales, the direct call takes 16-bit operands
        y = _core.decoder_linear(x, weight, bias, residual, x_scale, weight_scale, activation, out_dtype, True)
        if y is not NotImplemented and y is not None:
            return y
    _given("linear_act_fp8", x=x, x_scale=x_scale, weight=weight, weight_scale=weight_scale)
    _no_backward("linear_act_fp8", bias, residual, x_scale, weight_scale)
    args = (x, x_scale, weight, weight_scale, bias, residual, activation, out_dtype)
    if _plain(x, x_scale, weight, weight_scale, bias, residual):
        return _linear8_impl(*args)
    _no_forward_mode("linear_act_fp8", x_scale, weight_scale, bias, residual)
    _check_linear8(*args)
    return _linear_act_fp8(*args)
