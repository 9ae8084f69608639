"""Norm of queries and keys for each head together with their rotation by position (``hivt_qk_norm_rotary_*``)."""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._opsbase import _need_gpu, _on_device, _p, _stream, _unsupported, _workspace
from .ops_relative import _DTYPES, _heads_last, _recorded, _tensor

_Block = ctypes.c_int64 * 48  # hivt_qk_norm_rotary: 64-bit members only


@functools.lru_cache(maxsize=64)
def _rates(rotary_dim: int, theta: float):
    n = rotary_dim // 2
    return (ctypes.c_double * max(1, n))(*[theta ** (-2.0 * i / rotary_dim) for i in range(n)])


def _block(q, k, wq, wk, positions, rotary_dim, interleaved, out=(None, None), d_out=(None, None), dx=(None, None),
           dw=(None, None)):
    b, s, h, d = q.shape
    if positions is None:
        pos = (0, 0, 0, 0)
    else:
        sb, ss = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
        pos = (positions.data_ptr(), sb, ss, positions.element_size())
    return _Block(_DTYPES[q.dtype], b, s, h, k.shape[2], d, rotary_dim, interleaved, *_tensor(q), *_tensor(k), wq.data_ptr(),
                  wk.data_ptr(), *pos, *_tensor(out[0]), *_tensor(out[1]), *_tensor(d_out[0]), *_tensor(d_out[1]),
                  *_tensor(dx[0]), *_tensor(dx[1]), 0 if dw[0] is None else dw[0].data_ptr(),
                  0 if dw[1] is None else dw[1].data_ptr())


def _forward(q, k, wq, wk, positions, rotary_dim, theta, interleaved, eps):
    out = (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device))
    wq32, wk32 = wq.float().contiguous(), wk.float().contiguous()
    with _on_device(q):
        _lib.call("hivt_qk_norm_rotary_fwd", _block(q, k, wq32, wk32, positions, rotary_dim, interleaved, out),
                  _rates(rotary_dim, theta), eps, _stream(q))
    return out


class _QKNormRotary(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, rotary_dim, theta, interleaved, eps):
        out = _forward(q, k, wq, wk, positions, rotary_dim, theta, interleaved, eps)
        ctx.save_for_backward(q, k, wq, wk, positions)
        ctx.cfg = (rotary_dim, theta, interleaved, eps)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_q, d_k):
        q, k, wq, wk, positions = ctx.saved_tensors
        rotary_dim, theta, interleaved, eps = ctx.cfg
        dx = (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device))
        wq32, wk32 = wq.float().contiguous(), wk.float().contiguous()
        dw = (torch.empty_like(wq32), torch.empty_like(wk32))
        if q.numel() == 0:
            dw[0].zero_(), dw[1].zero_()
        else:
            with _on_device(q):
                need = _lib.query("hivt_qk_norm_rotary_bwd_workspace_bytes", q.shape[3])
                ws = _workspace(need, q.device)
                _lib.call("hivt_qk_norm_rotary_bwd",
                          _block(q, k, wq32, wk32, positions, rotary_dim, interleaved, d_out=(_heads_last(d_q), _heads_last(d_k)),
                                 dx=dx, dw=dw), _rates(rotary_dim, theta), eps, _p(ws), ws.numel(), _stream(q))
        grads = (dx[0], dx[1], dw[0].to(wq.dtype), dw[1].to(wk.dtype))
        return (*[g if need else None for g, need in zip(grads, ctx.needs_input_grad)], None, None, None, None, None)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                   positions: Optional[torch.Tensor] = None, rotary_dim: Optional[int] = None, theta: float = 10000.0,
                   interleaved: bool = False, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(R(pos) (q_weight * q / rms(q)), R(pos) (k_weight * k / rms(k)))``, contiguous, differentiable in all four.

    q [B, S, H, d], k [B, S, G, d] in float32, bfloat16 or float16 (any strides; slices of a fused projection need no
    copy), d even and at most 256; the weights [d] in float32 or the tensors' type.  rms(x) = sqrt(mean over d of x^2 +
    eps).  Pair i of the first ``rotary_dim`` components (default all; 0: no rotation) turns by position *
    theta ** (-2 i / rotary_dim); its members are i and i + rotary_dim / 2, or 2 i and 2 i + 1 with ``interleaved``.
    ``positions``: int32 or int64 [S] or [B, S], default 0 .. S - 1.  Sums and angles are fp32 and 64-bit; one rounding
    to the tensors' type at the end."""
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise TypeError(f"queries and keys must share one of float32, bfloat16, float16, got {q.dtype}, {k.dtype}")
    if q.dim() != 4 or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3] or not q.shape[2] or not k.shape[2]:
        raise ValueError(f"expected q [B, S, H, d] and k [B, S, G, d], got {tuple(q.shape)}, {tuple(k.shape)}")
    b, s, _, d = q.shape
    if d < 2 or d > 256 or d % 2:
        raise _unsupported(f"norm and rotation of heads of {d} (even, at most 256)")
    if b >= 2 ** 31 or s >= 2 ** 31 or q.shape[2] >= 65536 or k.shape[2] >= 65536:
        raise _unsupported(f"norm and rotation of {tuple(q.shape)}")
    for w in (q_weight, k_weight):
        if w.shape != (d,) or w.dtype not in (torch.float32, q.dtype):
            raise ValueError(f"the weights must be [{d}] in float32 or {q.dtype}, got {w.dtype} {tuple(w.shape)}")
    rotary_dim = d if rotary_dim is None else int(rotary_dim)
    if rotary_dim < 0 or rotary_dim > d or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be even and at most {d}")
    if not (theta > 0.0 and math.isfinite(theta)) or not eps > 0.0:
        raise ValueError(f"theta {theta} and eps {eps} must be positive")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in ((s,), (b, s)):
            raise ValueError(f"positions must be int32 or int64 [{s}] or [{b}, {s}], got {positions.dtype} "
                             f"{tuple(positions.shape)}")
    _need_gpu(q, k, q_weight, k_weight, positions)
    for t in (k, q_weight, k_weight, positions):
        if t is not None and t.device != q.device:
            raise ValueError(f"tensors on {q.device} and {t.device}")
    args = (_heads_last(q), _heads_last(k), q_weight, k_weight, positions, rotary_dim, float(theta), int(bool(interleaved)),
            float(eps))
    return _QKNormRotary.apply(*args) if _recorded(*args[:4]) else _forward(*args)
