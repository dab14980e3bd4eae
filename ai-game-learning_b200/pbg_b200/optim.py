"""Device-only flat Adam/AdamW transition (pbg/core/optimization.py:182-233).

The master parameters, gradients and both moments are single flat fp32
buffers (the reference's DenseGradientOwner layout, optimization.py:106-169)
so one fused kernel sequence updates the whole model.

``orthogonalize`` brings every singular value of a matrix to about one by
Newton-Schulz products; ``FlatMuon`` is the transition that updates the
matrices of a flat master by their orthogonalised momentum, all of them
together.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch
from torch import Tensor

from . import checks
from ._native import NativeError, call, entry, lib, ptr, raw_stream, stream

CONTROL_NAMES = ("lr", "beta1", "beta2", "epsilon", "decay", "clip", "scale", "growth", "backoff", "interval")


class FlatAdam:
    def __init__(self, master: Tensor, *, lr=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, decay=0.0, clip=1.0,
                 scale=1.0, decoupled=True, grad: Tensor | None = None) -> None:
        if master.dtype != torch.float32 or master.ndim != 1 or not master.is_cuda:
            raise ValueError("flat masters must be CUDA fp32 [N]")
        self.master = master
        n = master.numel()
        dev = master.device
        if grad is not None and (grad.shape != master.shape or grad.dtype != torch.float32 or grad.device != dev
                                 or not grad.is_contiguous()):
            raise ValueError("the flat gradient must be like the master")
        self.grad = torch.zeros(n, dtype=torch.float32, device=dev) if grad is None else grad
        self.first = torch.zeros(n, dtype=torch.float32, device=dev)
        self.second = torch.zeros(n, dtype=torch.float32, device=dev)
        self.controls = torch.tensor([lr, beta1, beta2, epsilon, decay, clip, scale, 2.0, 0.5, 2000.0],
                                     dtype=torch.float32, device=dev)
        self.step_count = torch.zeros(1, dtype=torch.int64, device=dev)
        self.partials = torch.zeros(int(lib().pbg_adam_partials_size(n)), dtype=torch.float64, device=dev)
        self.report = torch.zeros(8, dtype=torch.float64, device=dev)
        self.decoupled = bool(decoupled)

    def step(self) -> Tensor:
        """Apply one transition from ``self.grad``; returns the device report."""

        call("pbg_adam_step", self.master.numel(), ptr(self.master), ptr(self.grad), ptr(self.first),
             ptr(self.second), ptr(self.controls), ptr(self.step_count), int(self.decoupled), ptr(self.partials),
             ptr(self.report), stream(self.master.device))
        return self.report


COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ERROR: dict[int, Tensor] = {}
checks.watch(_ERROR, {0x7FFFFFFF: "a wait inside an orthogonalisation gave up: its outputs, or masters and momenta, are incomplete"})


def _error_word(device: torch.device) -> Tensor:
    word = _ERROR.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise NativeError("make one call on this device before capturing one into a graph")
        word = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()  # once: calls on other streams use it too
        _ERROR[device.index] = word
    return word


def orthogonalize_error(device=None) -> int:
    """The device's sticky error word of ``orthogonalize`` and ``FlatMuon`` (0 none, else a bounded wait gave
    up and the outputs are incomplete); synchronises."""

    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return int(_error_word(device).item())


def orthogonalize(x: Tensor, *, steps: int = 5, coefficients: tuple[float, float, float] = COEFFICIENTS,
                  epsilon: float = 1e-7, out_dtype: torch.dtype | None = None, out: Tensor | None = None) -> Tensor:
    """Every matrix of ``x`` ``[..., rows, cols]`` (fp32, bf16 or fp16) orthogonalised by ``steps`` Newton-Schulz
    steps: ``X / (|X|_F + epsilon)``, then ``X <- a X + (b G + c G^2) X`` with ``G = X X^T`` on the short side.

    The output has ``x``'s shape and ``out_dtype`` (``x``'s by default), or goes to ``out`` (contiguous; it
    may be ``x`` itself).  Products carry fp32 accuracy whatever the types; the result is rounded
    once.  A matrix of zeros gives zeros, one with a NaN or an infinity gives NaN.  The result is not part
    of an autograd graph, whatever ``x`` is."""

    if x.ndim < 2 or x.dtype not in _TYPES:
        raise NativeError("orthogonalize takes float32, bfloat16 or float16 matrices [..., rows, cols]")
    if not x.is_cuda:
        raise NativeError("libpbgb200 operates on CUDA tensors only")
    device = x.device
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype if out_dtype is None else out_dtype, device=device)
    elif out.shape != x.shape or out.device != device or not out.is_contiguous() or (
            out_dtype is not None and out.dtype != out_dtype):
        raise NativeError("orthogonalize: out must be contiguous, of x's shape and device and the output type")
    if out.dtype not in _TYPES:
        raise NativeError("orthogonalize: the output must be float32, bfloat16 or float16")
    x = x.contiguous()
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _orthogonalize(x, steps, coefficients, epsilon, out)
    return _orthogonalize(x, steps, coefficients, epsilon, out)


def _orthogonalize(x, steps, coefficients, epsilon, out):
    device = x.device
    rows, cols = x.shape[-2:]
    batch = math.prod(x.shape[:-2])
    size = int(lib().pbg_orthogonalize_workspace(batch, rows, cols))
    workspace = torch.empty(max(size, 1), dtype=torch.uint8, device=device)
    a, b, c = coefficients
    entry("pbg_orthogonalize")(batch, rows, cols, x.data_ptr(), _TYPES[x.dtype], out.data_ptr(), _TYPES[out.dtype],
                               int(steps), float(a), float(b), float(c), float(epsilon), workspace.data_ptr(), size,
                               _error_word(device).data_ptr(), raw_stream(device.index))
    return out


MUON_CONTROL_NAMES = ("lr", "momentum", "decay", "scale")


def _shape_adjust(rows: int, cols: int) -> float:
    return math.sqrt(max(1.0, rows / cols))


def _rms_adjust(rows: int, cols: int) -> float:
    return 0.2 * math.sqrt(max(rows, cols))


ADJUST = {"shape": _shape_adjust, "rms": _rms_adjust}


class FlatMuon:
    """The transition of the matrices of a flat fp32 master by their orthogonalised momentum.

    ``matrices`` lists ``(offset, rows, cols)`` of each into ``master``; other elements of the flat buffers
    are left alone (``FlatAdam`` on its own slice serves vectors and tables).  Per matrix

        m <- mu m + (1 - mu) g / scale;   u = mu m + (1 - mu) g / scale  (``nesterov``) or m
        w <- w (1 - lr decay) - lr s orthogonalize(u)

    with ``s = sqrt(max(1, rows / cols))`` (``adjust="shape"``) or ``0.2 sqrt(max(rows, cols))``
    (``"rms"``: updates as large as AdamW's usual ones).  ``controls`` (device fp32: lr, momentum, decay,
    scale) may be rewritten between steps, also under a captured graph.  A step launches the squares of
    all directions, then the conversion and the products of all matrices whose short side is over 128 (of as
    many at a time as 1 GB of tiles holds), then all others' teams.  A direction that is not finite leaves masters
    and momenta untouched, clears the matrices' gradients and sets ``skipped`` to 1 for that step."""

    def __init__(self, master: Tensor, matrices, *, lr=0.02, momentum=0.95, decay=0.0, scale=1.0, nesterov=True,
                 adjust="shape", steps=5, coefficients=COEFFICIENTS, epsilon=1e-7, grad: Tensor | None = None) -> None:
        if master.dtype != torch.float32 or master.ndim != 1 or not master.is_cuda or not master.is_contiguous():
            raise ValueError("flat masters must be CUDA fp32 [N]")
        if adjust not in ADJUST:
            raise ValueError("adjust must be 'shape' or 'rms'")
        if not 0.0 <= momentum < 1.0:
            raise ValueError("momentum must be in [0, 1)")
        n, dev = master.numel(), master.device
        table = np.array([tuple(map(int, m)) for m in matrices], dtype=np.int64).reshape(-1, 3)
        ends = table[:, 0] + table[:, 1] * table[:, 2]
        if len(table) == 0 or (table[:, 0] < 0).any() or (table[:, 1:] < 1).any() or (ends > n).any():
            raise ValueError("matrices must be (offset, rows, cols) inside the flat master")
        order = np.argsort(table[:, 0], kind="stable")
        if (table[order][1:, 0] < ends[order][:-1]).any():
            raise ValueError("matrices must not overlap")
        if grad is not None and (grad.shape != master.shape or grad.dtype != torch.float32 or grad.device != dev
                                 or not grad.is_contiguous()):
            raise ValueError("the flat gradient must be like the master")
        self.master = master
        self.grad = torch.zeros(n, dtype=torch.float32, device=dev) if grad is None else grad
        self.momentum = torch.zeros(n, dtype=torch.float32, device=dev)
        self.controls = torch.tensor([lr, momentum, decay, scale], dtype=torch.float32, device=dev)
        self.skipped = torch.zeros(1, dtype=torch.int32, device=dev)
        self.nesterov, self.steps, self.coefficients, self.epsilon = bool(nesterov), int(steps), tuple(coefficients), float(epsilon)
        self.matrices = [tuple(int(v) for v in m) for m in table]
        L = lib()
        count = len(table)
        offset, rows, cols = (np.ascontiguousarray(table[:, i]) for i in range(3))
        factor = np.array([ADJUST[adjust](r, c) for _, r, c in self.matrices], dtype=np.float32)
        descriptors = np.zeros(count * int(L.pbg_muon_descriptor_bytes()), dtype=np.uint8)
        self._plan = np.zeros(int(L.pbg_muon_plan_words(count)), dtype=np.int64)
        call("pbg_muon_plan", count, *(a.ctypes.data_as(ctypes.c_void_p) for a in
                                       (offset, rows, cols, factor, descriptors, self._plan)))
        self._descriptors = torch.from_numpy(descriptors).to(dev)
        self._workspace = torch.empty(int(self._plan[0]), dtype=torch.uint8, device=dev)
        _error_word(dev)

    def step(self) -> Tensor:
        """Apply one transition from ``self.grad``; returns the device's ``skipped`` word (int32 [1])."""

        dev = self.master.device
        if dev.index != torch._C._cuda_getDevice():
            with torch.cuda.device(dev):
                return self._step(dev)
        return self._step(dev)

    def _step(self, dev) -> Tensor:
        a, b, c = self.coefficients
        entry("pbg_muon_step")(len(self.matrices), self._descriptors.data_ptr(), self._plan.ctypes.data,
                               self.grad.data_ptr(), self.momentum.data_ptr(), self.master.data_ptr(),
                               self.controls.data_ptr(), int(self.nesterov), self.steps, float(a), float(b), float(c),
                               self.epsilon, self._workspace.data_ptr(), self._workspace.numel(),
                               self.skipped.data_ptr(), _error_word(dev).data_ptr(), raw_stream(dev.index))
        return self.skipped


__all__ = ["FlatAdam", "FlatMuon", "orthogonalize", "orthogonalize_error"]
