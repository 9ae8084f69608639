"""Orthogonalised updates of matrices (``hivt_orthogonalize``), what ``optim.Muon`` steps along."""
from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence

import torch

from . import _lib
from ._opsbase import _need_gpu, _on_device, _p, _stream, _unsupported, _workspace
from .ops_relative import _DTYPES

_MAX_SIDE = 65536


def matrix_list(ins: Sequence[torch.Tensor], outs: Sequence[torch.Tensor]):
    """The ``hivt_matrix`` array of contiguous matrices."""
    flat = []
    for x, y in zip(ins, outs):
        flat += (x.data_ptr(), y.data_ptr(), x.shape[0], x.shape[1])
    return (ctypes.c_int64 * max(1, len(flat)))(*flat)


def _outputs(matrices: Sequence[torch.Tensor]) -> List[torch.Tensor]:
    """A tensor like each matrix; those of one shape are slices of one allocation (a call of the allocator costs as much
    as launching a kernel)."""
    by_shape = {}
    for i, x in enumerate(matrices):
        by_shape.setdefault(x.shape, []).append(i)
    out: List[Optional[torch.Tensor]] = [None] * len(matrices)
    for shape, at in by_shape.items():
        x = matrices[at[0]]
        for i, y in zip(at, torch.empty((len(at), *shape), dtype=x.dtype, device=x.device).unbind(0)):
            out[i] = y
    return out


def _refuse_overlaps(ins: Sequence[torch.Tensor], outs: Sequence[torch.Tensor]) -> None:
    """An output may be its own matrix and nothing else: matrices of different sizes are worked on one after the other."""
    spans = []
    for i, (x, y) in enumerate(zip(ins, outs)):
        if y.numel():
            size = y.numel() * y.element_size()
            spans.append((y.data_ptr(), y.data_ptr() + size, i, True))
            if x.data_ptr() != y.data_ptr():
                spans.append((x.data_ptr(), x.data_ptr() + size, i, False))
    written = read = 0  # the furthest ends so far
    for begin, end, i, is_out in sorted(spans):
        if begin < written or (is_out and begin < read):
            raise ValueError(f"output or matrix {i} shares memory with another output")
        if is_out:
            written = max(written, end)
        else:
            read = max(read, end)


def _run(ins: Sequence[torch.Tensor], out: List[torch.Tensor], steps: int, eps: float) -> List[torch.Tensor]:
    with _on_device(ins[0]):
        ins = [x.contiguous() for x in ins]
        array = matrix_list(ins, out)
        need = _lib.value("hivt_orthogonalize_workspace_bytes", array, len(ins))
        ws = _workspace(need, ins[0].device)
        _lib.call("hivt_orthogonalize", array, len(ins), _DTYPES[ins[0].dtype], int(steps), float(eps), _p(ws), ws.numel(),
                  _stream(ins[0]))
    return out


@torch.no_grad()
def orthogonalize(matrices: Sequence[torch.Tensor], steps: int = 5, eps: float = 1e-7,
                  out: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
    """Each matrix [rows, cols] of the list, its singular values brought near 1: ``x / (|x| + eps)`` (Frobenius norm), then
    ``steps`` times ``x <- a x + (b g + c g^2) x`` with g = x x^T (of the shorter side) and a, b, c = 3.4445, -4.7750,
    2.0315.  One type for the list, float32, bfloat16 or float16; any shapes up to 65536 a side.  The arithmetic is that of
    fp32 whatever the type, rounded once at the end; equal calls give equal bits, and what else is in the list moves a
    result by the rounding of fp32 sums at most.  ``out``: contiguous tensors to write to (each may be its own matrix, and
    shares no memory with any other one or output); without it, results of one shape are slices of one allocation.  Not
    differentiable."""
    matrices = list(matrices)
    if not matrices:
        return []
    dtype, device = matrices[0].dtype, matrices[0].device
    for x in matrices:
        if x.dtype not in _DTYPES or x.dtype != dtype:
            raise TypeError(f"the matrices must share one of float32, bfloat16, float16, got {x.dtype}")
        if x.dim() != 2:
            raise ValueError(f"expected matrices, got shape {tuple(x.shape)}")
        if max(x.shape) > _MAX_SIDE:
            raise _unsupported(f"orthogonalising a matrix of {tuple(x.shape)} (at most {_MAX_SIDE} a side)")
        if x.device != device:
            raise ValueError(f"matrices on {device} and {x.device}")
    if not 1 <= int(steps) <= 16:
        raise ValueError(f"steps must be 1 to 16, got {steps}")
    if not eps > 0.0:
        raise ValueError(f"eps must be positive, got {eps}")
    _need_gpu(*matrices)
    if out is None:
        return _run(matrices, _outputs(matrices), steps, eps)
    out = list(out)
    if len(out) != len(matrices):
        raise ValueError(f"{len(matrices)} matrices, {len(out)} outputs")
    for x, y in zip(matrices, out):
        if y.shape != x.shape or y.dtype != dtype or y.device != device or not y.is_contiguous():
            raise ValueError(f"an output must be contiguous {dtype} {tuple(x.shape)} on {device}")
    matrices = [x.contiguous() for x in matrices]
    _refuse_overlaps(matrices, out)
    torch.autograd.graph.increment_version([y for y in out if not y.is_inference()])
    return _run(matrices, out, steps, eps)
