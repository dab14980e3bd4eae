"""Embedding rows by index, times a scale, and the gradient of that lookup.

The policy/value network's token assembly adds rows of small tables (token
types, seats, streets, actions, positions, classes, ranks and suits;
pbg/games/poker/model/preflop.py:206-233, shared.py:36-72).  ``embedding``
looks rows up and scales them in one pass; ``embedding_backward`` sums the
incoming rows of each index after sorting the tokens by index, without
floating-point atomics: the same inputs, laid out and aligned alike, give the
same bits in every run on a device.
``pbg_b200.model_train.embedding_train`` is the two as one autograd function.

An index outside the table gives a row of zeros and no gradient, and sets the
device's sticky error word, which ``index_error`` reads and
``checks.raise_input_errors`` reports (no launch waits for it).  Calls run on the current stream of their tensors' device and can be
captured into graphs once one call has been made on the device.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import checks
from ._native import NativeError, entry, lib, raw_stream

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ERROR: dict[int, Tensor] = {}
checks.watch(_ERROR, {1: "an embedding index is outside its table",
                      2: "a wait inside an embedding gradient gave up: the gradient is incomplete"})


def _error_word(device: torch.device) -> Tensor:
    word = _ERROR.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise NativeError("make one embedding call on this device before capturing one into a graph")
        word = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()  # once: calls on other streams use it too
        _ERROR[device.index] = word
    return word


def index_error(device=None) -> int:
    """The device's sticky error word: 0 none, bit 0 an index outside a table, bit 1 a grid barrier that gave
    up (the gradient of that call is incomplete); synchronises."""

    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return int(_error_word(device).item())


def _rows_matrix(t: Tensor, width: int) -> Tensor:
    """t [..., width] as a matrix of rows with contiguous columns, without a copy where its strides allow."""

    m = t if t.ndim == 2 else t[None] if t.ndim == 1 else t.flatten(0, -2)
    if m.numel() and ((width > 1 and m.stride(1) != 1) or (m.shape[0] > 1 and m.stride(0) < width)):
        m = m.contiguous()
    return m


def _stride(m: Tensor) -> int:
    return m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _check_index(index: Tensor, device: torch.device) -> Tensor:
    if index.dtype not in (torch.int64, torch.int32):
        raise NativeError("embedding: the index must be int64 or int32")
    if index.device != device:
        raise NativeError("embedding: index and rows must be on one CUDA device")
    return index.contiguous()


def embedding(table: Tensor, index: Tensor, scale: float = 1.0, *, out_dtype: torch.dtype | None = None,
              out: Tensor | None = None) -> Tensor:
    """``scale * table[index]``: fp32, bf16 or fp16 rows ``[rows, width]`` (columns contiguous, any row
    stride), ``index`` int64 or int32 of any shape; the product is taken in fp32 and rounded once to
    ``out_dtype`` (the table's by default) or to ``out``'s type (contiguous ``[*index.shape, width]``).
    The result is not part of an autograd graph: ``model_train.embedding_train`` is the differentiable lookup."""

    if table.ndim != 2 or table.dtype not in TYPES:
        raise NativeError("embedding: the table must be a float32, bfloat16 or float16 matrix")
    if not table.is_cuda:
        raise NativeError("libpbgb200 operates on CUDA tensors only")
    device = table.device
    index = _check_index(index, device)
    rows, width = table.shape
    table = _rows_matrix(table, width)
    shape = (*index.shape, width)
    if out is None:
        out = torch.empty(shape, dtype=table.dtype if out_dtype is None else out_dtype, device=device)
    elif out.shape != shape or out.device != device or not out.is_contiguous() or (
            out_dtype is not None and out.dtype != out_dtype):
        raise NativeError("embedding: out must be contiguous [*index.shape, width] of the output type, on the table's device")
    if out.dtype not in TYPES:
        raise NativeError("embedding: the output must be float32, bfloat16 or float16")
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _forward(table, index, scale, out, rows, width)
    return _forward(table, index, scale, out, rows, width)


def _forward(table, index, scale, out, rows, width):
    device = table.device
    entry("pbg_embedding")(index.numel(), rows, width, index.data_ptr(), int(index.dtype == torch.int64), table.data_ptr(),
                           TYPES[table.dtype], _stride(table), float(scale), out.data_ptr(), TYPES[out.dtype],
                           _error_word(device).data_ptr(), raw_stream(device.index))
    return out


def embedding_backward(grad: Tensor, index: Tensor, rows: int, scale: float = 1.0, *, padding_index: int | None = None,
                       out: Tensor | None = None, accumulate: bool = False,
                       out_dtype: torch.dtype = torch.float32) -> Tensor:
    """The table's gradient ``[rows, width]`` of ``embedding``: row v is ``scale`` times the sum of the
    rows of ``grad`` ``[*index.shape, width]`` whose index is v, zeros where there is none.

    Sums are kept in fp32 and rounded once to ``out_dtype`` or ``out``'s type.  With ``accumulate`` the
    sums are added to what ``out`` holds (for example a table's slice of a flat gradient) and rows
    without tokens are neither read nor written.  ``padding_index`` tokens give no gradient.  ``out``
    has contiguous columns and any row stride."""

    if grad.dtype not in TYPES or grad.ndim < 1:
        raise NativeError("embedding_backward: the gradient must be float32, bfloat16 or float16")
    if not grad.is_cuda:
        raise NativeError("libpbgb200 operates on CUDA tensors only")
    device = grad.device
    index = _check_index(index, device)
    if grad.shape[:-1] != index.shape:
        raise NativeError("embedding_backward: grad must be [*index.shape, width]")
    width = grad.shape[-1]
    rows = int(rows)
    if rows < 0:
        raise NativeError("embedding_backward: rows must not be negative")
    if padding_index is None:
        padding_index = -1
    elif not 0 <= padding_index < rows:
        raise NativeError("embedding_backward: the padding index must be a row of the table")
    if out is None:
        if accumulate:
            raise NativeError("embedding_backward: accumulate needs the gradient to add to (out)")
        out = torch.empty((rows, width), dtype=out_dtype, device=device)
    elif out.shape != (rows, width) or out.device != device or (out.numel() and (
            (width > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < width))):
        raise NativeError("embedding_backward: out must be [rows, width] with contiguous columns, on the gradient's device")
    if out.dtype not in TYPES:
        raise NativeError("embedding_backward: the output must be float32, bfloat16 or float16")
    grad = _rows_matrix(grad, width)
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _backward(grad, index, rows, width, scale, padding_index, out, accumulate)
    return _backward(grad, index, rows, width, scale, padding_index, out, accumulate)


def _backward(grad, index, rows, width, scale, padding_index, out, accumulate):
    device = grad.device
    tokens = index.numel()
    size = lib().pbg_embedding_backward_workspace(tokens, width)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    entry("pbg_embedding_backward")(tokens, rows, width, grad.data_ptr(), TYPES[grad.dtype], _stride(grad),
                                    index.data_ptr(), int(index.dtype == torch.int64), padding_index, float(scale),
                                    out.data_ptr(), TYPES[out.dtype], _stride(out), int(bool(accumulate)),
                                    workspace.data_ptr(), size, _error_word(device).data_ptr(), raw_stream(device.index))
    return out


__all__ = ["embedding", "embedding_backward", "index_error"]
