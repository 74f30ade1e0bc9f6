"""The bounds-checked build (-DQC_DEBUG_BOUNDS) on the decoder operators: every
index that a kernel computes itself is checked against its array (what TMA moves
is bounded by its tensor map), so a zero fault word means that none left it on
these shapes. The results are the release build's up to rounding: compiled
apart, the two contract a * b + c differently, which moves an fp32 intermediate
by 2**-24 of its terms and may move a 16- or 8-bit result by one step. A result is
held to one step (eps) plus 2**-14 (sums of up to 40011 such terms of either
sign, against sums that cancel to their square root: 40011**0.5 * 2**-24 < 2**-16)
of its array's norm.

As in test_debug_bounds_gpu.py the checked library runs in a child process.
"""

from __future__ import annotations

import ctypes
import multiprocessing as mp
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

LIBDIR = Path(__file__).resolve().parents[1] / "quantem-cuda_b200" / "quantem" / "cuda"
F32, BF16, F16, E4M3 = range(4)
TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16, E4M3: torch.float8_e4m3fn}
NONE, RELU, SILU, GELU = range(4)

# rows, width, further values per row (its stride), x's type, y's type, residual
NORMS = [(1, 1, 0, F32, F32, True), (700, 4, 0, BF16, BF16, True), (37, 30, 0, F16, F16, False), (300, 128, 3, F32, BF16, True),
         (20011, 77, 0, BF16, BF16, True), (12000, 256, 0, F32, BF16, False), (11000, 999, 0, F16, F16, True),
         (1500, 1000, 8, BF16, F32, True), (1300, 2048, 0, F32, F32, True), (1300, 4097, 0, F16, F16, True),
         (40, 8200, 1, BF16, BF16, False), (600, 16400, 0, F32, F16, True), (301, 20001, 0, BF16, BF16, True)]
# rows, K, N, further values per row, operand type, output type, bias, residual, activation
LINEARS = [(1, 1, 1, 0, BF16, BF16, True, True, NONE), (17, 1000, 300, 0, F16, F32, True, True, SILU),
           (50, 2048, 200, 3, E4M3, BF16, True, True, GELU), (300, 2056, 264, 0, BF16, BF16, True, True, RELU),
           (129, 203, 77, 0, F16, F16, True, True, SILU), (300, 96, 256, 1, BF16, F32, True, True, GELU),
           (700, 200, 640, 8, E4M3, F32, True, True, NONE), (20011, 1024, 264, 0, BF16, BF16, True, True, GELU),
           (5000, 64, 520, 0, F16, F16, False, False, RELU), (0, 8, 8, 0, BF16, BF16, True, False, NONE)]
# rows, K, N, further values per row, operand type, upstream type, activation
GRADS = [(1, 8, 8, 0, BF16, BF16, SILU), (130, 203, 77, 0, F16, F16, SILU), (130, 203, 77, 1, F16, F32, GELU),
         (2500, 136, 320, 0, BF16, BF16, NONE), (2500, 136, 321, 0, BF16, F32, NONE), (5000, 24, 16, 3, F16, F32, NONE),
         (700, 64, 200, 1, BF16, BF16, RELU), (20011, 64, 520, 0, BF16, BF16, GELU), (20011, 1024, 264, 0, F16, F16, SILU),
         (40011, 200, 1024, 0, BF16, BF16, NONE), (0, 8, 8, 0, BF16, BF16, SILU)]
KEPT = [(513, 512, 8), (700, 520, 72), (20011, 1024, 264)]


def _load(name):
    vp, i, f, sz, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t, ctypes.c_long
    lib = ctypes.CDLL(str(LIBDIR / name))
    lib.rms_norm_cuda.argtypes = [vp] * 6 + [L, i, L, L, i, i, f, vp]
    lib.quantize_rows_cuda.argtypes = [vp] * 3 + [L, i, L, i, vp]
    lib.rms_norm_grad_workspace_bytes.argtypes = [L, i]
    lib.rms_norm_grad_cuda.argtypes = [vp] * 7 + [L, i, L, L, L, L, i, i, f, vp, sz, vp]
    lib.linear_act_workspace_bytes.argtypes = [vp, vp, L, i, i, L, L, i]
    lib.linear_act_cuda.argtypes = [vp] * 7 + [L, i, i, L, L, L, i, i, i, i, vp, sz, vp]
    lib.linear_act_grad_workspace_bytes.argtypes = [vp] * 6 + [L, i, i, L, L, L, i, i, i, i]
    lib.linear_act_grad_cuda.argtypes = [vp] * 7 + [L, i, i, L, L, L, i, i, i, i, vp, sz, vp]
    lib.linear_act_kept_bytes.argtypes = [L, i, i, i, i, i, i]
    lib.linear_act_keep_cuda.argtypes = [vp] * 6 + [L, i, i, L, L, L, i, i, i, vp, sz, vp]
    lib.linear_act_grad_kept_workspace_bytes.argtypes = [vp] * 6 + [L, i, i, L, L, L, i, i, i]
    lib.linear_act_grad_kept_cuda.argtypes = [vp] * 7 + [L, i, i, L, L, L, i, i, vp, sz, vp]
    for n in ("rms_norm_grad", "linear_act", "linear_act_grad", "linear_act_grad_kept"):
        getattr(lib, f"{n}_workspace_bytes").restype = sz
    lib.linear_act_kept_bytes.restype = sz
    lib.quantem_cuda_device_fault_word.argtypes = [i, ctypes.POINTER(ctypes.c_uint), i]
    lib.quantem_cuda_last_error.restype = ctypes.c_char_p
    return lib


class _Runner:
    def __init__(self, name):
        self.lib = _load(name)
        self.stream = torch.cuda.current_stream().cuda_stream
        self.gen = torch.Generator().manual_seed(7)

    def call(self, fn, *args):
        args = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
        assert getattr(self.lib, fn)(*args, self.stream) == 0, (fn, self.lib.quantem_cuda_last_error())

    def values(self, rows, n, kind, extra=0):
        """[rows, n] of the type, its rows n + extra apart."""
        t = (torch.randn((rows, n + extra), generator=self.gen) / 2).to(TORCH[kind]).cuda()
        return t[:, :n]

    def empty(self, *shape, kind):
        return torch.full(shape, 3, dtype=torch.float32).to(TORCH[kind]).cuda()

    def workspace(self, nbytes):
        return torch.zeros(max(nbytes, 1), dtype=torch.uint8, device="cuda"), nbytes

    def norm(self, rows, n, extra, xt, ot, added):
        x, w = self.values(rows, n, xt, extra), self.values(1, n, xt)[0]
        r = self.values(rows, n, xt, extra) if added else None
        y, h = self.empty(rows, n, kind=ot), self.empty(rows, n, kind=xt) if added else None
        s = n + extra
        self.call("rms_norm_cuda", x, r, w, y, h, None, rows, n, s, s, xt, ot, 1e-5)
        q, scale = self.empty(rows, n, kind=E4M3), self.empty(rows, kind=F32)
        self.call("rms_norm_cuda", x, r, w, q, h, scale, rows, n, s, s, xt, E4M3, 1e-5)
        q2, scale2 = torch.clone(q), torch.clone(scale)
        self.call("quantize_rows_cuda", x, q2, scale2, rows, n, s, xt)
        dy, dh = self.values(rows, n, ot, extra), self.values(rows, n, xt, extra) if added else None
        dx, dw = self.empty(rows, n, kind=xt), self.empty(n, kind=xt)
        ws, nbytes = self.workspace(self.lib.rms_norm_grad_workspace_bytes(rows, n))
        self.call("rms_norm_grad_cuda", x, r, w, dy, dh, dx, dw, rows, n, s, s, s, s, xt, ot, 1e-5, ws, nbytes)
        return [t for t in (y, h, q, scale, q2, scale2, dx, dw) if t is not None]

    def linear(self, rows, k, n, extra, t, ot, bias, res, act):
        x, w = self.values(rows, k, t, extra), self.values(n, k, t, extra)
        b, r = self.values(1, n, ot)[0] if bias else None, self.values(rows, n, ot, extra) if res else None
        sx, sw = (self.values(1, m, F32)[0].abs() if t == E4M3 else None for m in (rows, n))
        y, s = self.empty(rows, n, kind=ot), k + extra
        ws, nbytes = self.workspace(self.lib.linear_act_workspace_bytes(x.data_ptr(), w.data_ptr(), rows, n, k, s, s, t))
        self.call("linear_act_cuda", x, w, b, r, y, sx, sw, rows, n, k, s, s, n + extra, t, ot, ot, act, ws, nbytes)
        return [y]

    def grad(self, rows, k, n, extra, t, dyt, act):
        x, w, b = self.values(rows, k, t, extra), self.values(n, k, t, extra), self.values(1, n, F32)[0]
        dy = self.values(rows, n, dyt, extra)
        dx, dw, db = self.empty(rows, k, kind=t), self.empty(n, k, kind=t), self.empty(n, kind=F32)
        shape = (rows, n, k, k + extra, k + extra, n + extra, t, dyt)
        ws, nbytes = self.workspace(self.lib.linear_act_grad_workspace_bytes(
            *[a.data_ptr() for a in (x, w, dy, dx, dw, db)], *shape, act, 0))
        self.call("linear_act_grad_cuda", x, w, b, dy, dx, dw, db, *shape, F32, act, ws, nbytes)
        return [dx, dw, db]

    def kept(self, rows, k, n):
        x, w, b, dy = (self.values(*s, BF16) for s in ((rows, k), (n, k), (1, n), (rows, n)))
        y, dx, dw, db = (self.empty(*s, kind=BF16) for s in ((rows, n), (rows, k), (n, k), (n,)))
        nbytes = self.lib.linear_act_kept_bytes(rows, n, k, BF16, BF16, BF16, SILU)
        assert nbytes
        kept = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
        ws, none = self.workspace(0)
        self.call("linear_act_keep_cuda", x, w, b, None, y, kept, rows, n, k, k, k, n, BF16, BF16, SILU, ws, none)
        ws, nbytes = self.workspace(self.lib.linear_act_grad_kept_workspace_bytes(
            *[a.data_ptr() for a in (x, w, dy, dx, dw, db)], rows, n, k, k, k, n, BF16, SILU, 0))
        self.call("linear_act_grad_kept_cuda", x, w, kept, dy, dx, dw, db, rows, n, k, k, k, n, BF16, SILU, ws, nbytes)
        return [y, dx, dw, db]


def _run_all(name):
    run = _Runner(name)
    word = ctypes.c_uint(0)
    assert run.lib.quantem_cuda_device_fault_word(0, ctypes.byref(word), 1) == 0
    outs = []
    for cases, fn in ((NORMS, run.norm), (LINEARS, run.linear), (GRADS, run.grad), (KEPT, run.kept)):
        for case in cases:
            for t in fn(*case):
                outs.append(((fn.__name__, *case), torch.finfo(t.dtype).eps, t.float().cpu()))
    torch.cuda.synchronize()
    assert run.lib.quantem_cuda_device_fault_word(0, ctypes.byref(word), 1) == 0
    return outs, word.value


def _child(name, path, queue):
    try:
        outs, fault = _run_all(name)
        torch.save([t for _, _, t in outs], path)
        queue.put(("ok", fault))
    except BaseException as e:  # report, do not hang the parent
        queue.put((repr(e), 0))


def test_checked_decoder_is_clean_and_matches_release(tmp_path):
    if not (LIBDIR / "libquantem_cuda_b200_debug.so").exists():
        pytest.fail("libquantem_cuda_b200_debug.so not built (build_ext.build_debug)")
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    p = ctx.Process(target=_child, args=("libquantem_cuda_b200_debug.so", str(tmp_path / "outs.pt"), queue))
    p.start()
    kind, fault = queue.get(timeout=600)
    p.join(timeout=60)
    assert kind == "ok", kind
    assert fault == 0, f"bounds checks fired: fault word {fault:#x}"
    release, fault = _run_all("libquantem_cuda_b200.so")
    assert fault == 0
    for (case, step, ref), got in zip(release, torch.load(tmp_path / "outs.pt"), strict=True):
        assert (got - ref).norm() <= (step + 2.0**-14) * ref.norm(), case
