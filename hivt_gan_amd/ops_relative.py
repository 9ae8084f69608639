"""Attention over positions whose distance is felt through a learned bias (``hivt_relative_attn_*``).

Beside ``ops.temporal_attention`` (causal, at most 32 steps, fp32): any lengths, grouped key heads, a mask of keys,
fp32 / bfloat16 / float16, and the gradient of the bias table."""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._opsbase import _need_gpu, _on_device, _p, _stream, _unsupported, _workspace

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_BORDER = 4096
_Block = ctypes.c_int64 * 50  # hivt_relative_attn: 64-bit members only


@functools.lru_cache(maxsize=256)
def relative_buckets(num_buckets: int, max_distance: int, bidirectional: bool) -> Tuple[int, Tuple[int, ...]]:
    """``(exact, borders)``: distances below ``exact`` have a bucket each, a wider bucket starts at ``exact`` and at
    every border.  The borders are spaced by the logarithm, the t-th of L - 1 being the least n with
    n >= exact * (max_distance / exact) ** (t / L), decided in whole numbers so that no rounding moves a border.  With
    ``bidirectional`` the second half of the buckets is for keys behind the query."""
    if num_buckets < 2 or (bidirectional and (num_buckets % 2 or num_buckets < 4)):
        raise ValueError(f"{num_buckets} buckets: at least 2, and an even number of at least 4 for both directions")
    side = num_buckets // 2 if bidirectional else num_buckets
    exact = side // 2
    wide = side - exact
    if max_distance <= exact:
        raise ValueError(f"max_distance {max_distance} must exceed the {exact} distances with a bucket of their own")
    if wide - 1 > 127:
        raise _unsupported(f"{num_buckets} relative-position buckets")
    borders = []
    for t in range(1, wide):
        low, high, goal = exact, max_distance, exact ** (wide - t) * max_distance ** t
        while low < high:
            mid = (low + high) // 2
            if mid ** wide >= goal:
                high = mid
            else:
                low = mid + 1
        borders.append(low)
    if (borders[-1] if borders else exact) > _MAX_BORDER:
        raise _unsupported(f"relative positions told apart beyond a distance of {_MAX_BORDER}")
    return exact, tuple(borders)


@functools.lru_cache(maxsize=256)
def _borders(num_buckets: int, max_distance: int, bidirectional: bool):
    exact, borders = relative_buckets(num_buckets, max_distance, bidirectional)
    return exact, len(borders), (ctypes.c_int32 * max(1, len(borders)))(*borders)


def _heads_last(t: torch.Tensor) -> torch.Tensor:
    """A view whose last dimension is contiguous (the other strides are free)."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _recorded(*tensors: torch.Tensor) -> bool:
    """Whether a call on them needs a node for its backward (one costs a single-token call half its time)."""
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def _tensor(t: Optional[torch.Tensor]):
    return (0, 0, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _block(cfg, q, k, v, table, mask, out=None, stats=None, d_out=None, dq=None, dk=None, dv=None, d_table=None):
    causal, bidirectional, offset, exact, starts = cfg
    b, m, h, d = q.shape
    return _Block(_DTYPES[q.dtype], b, m, k.shape[1], h, k.shape[2], d, causal, bidirectional, offset, table.shape[0],
                  exact, starts, *_tensor(q), *_tensor(k), *_tensor(v), table.data_ptr(),
                  0 if mask is None else mask.data_ptr(), 0 if mask is None else mask.stride(0), *_tensor(out),
                  0 if stats is None else stats.data_ptr(), *_tensor(d_out), *_tensor(dq), *_tensor(dk), *_tensor(dv),
                  0 if d_table is None else d_table.data_ptr())


def _forward(q, k, v, table, mask, cfg, borders, scale, want_stats):
    b, m, h, d = q.shape
    out = torch.empty(b, m, h, d, dtype=q.dtype, device=q.device)
    stats = torch.empty(b * h, m, 2, dtype=torch.float32, device=q.device) if want_stats else None
    with _on_device(q):
        args = _block(cfg, q, k, v, table, mask, out, stats)
        need = _lib.value("hivt_relative_attn_fwd_workspace_bytes", args, borders)
        ws = _workspace(need, q.device) if need else None
        _lib.call("hivt_relative_attn_fwd", args, borders, scale, _p(ws), need, _stream(q))
    return out, stats


def _backward(d_out, q, k, v, table, mask, out, stats, cfg, borders, scale, dq, dk, dv, want_table):
    if q.shape[0] == 0 or q.shape[1] == 0 or q.shape[2] == 0:
        for g in (dq, dk, dv):
            g.zero_()
        return torch.zeros_like(table) if want_table else None
    d_out = _heads_last(d_out)
    d_table = torch.empty_like(table) if want_table else None
    with _on_device(q):
        args = _block(cfg, q, k, v, table, mask, out, stats, d_out, dq, dk, dv, d_table)
        need = _lib.value("hivt_relative_attn_bwd_workspace_bytes", args, borders)
        ws = _workspace(need, q.device)
        _lib.call("hivt_relative_attn_bwd", args, borders, scale, _p(ws), ws.numel(), _stream(q))
    return d_table


class _RelativeAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, table, mask, cfg, borders, scale):
        out, stats = _forward(q, k, v, table, mask, cfg, borders, scale, True)
        ctx.save_for_backward(q, k, v, table, mask, out, stats)
        ctx.cfg = (cfg, borders, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        q, k, v, table, mask, out, stats = ctx.saved_tensors
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)]
        d_table = _backward(d_out, q, k, v, table, mask, out, stats, *ctx.cfg, *grads, ctx.needs_input_grad[3])
        return (*[g if need else None for g, need in zip(grads, ctx.needs_input_grad)], d_table, None, None, None, None)


def _self_forward(qkv, table, heads, mask, cfg, borders, scale, want_stats):
    s, n, three_d = qkv.shape
    q, k, v = qkv.view(s, n, 3, heads, three_d // (3 * heads)).transpose(0, 1).unbind(2)
    out = torch.empty(s, n, heads, q.shape[-1], dtype=qkv.dtype, device=qkv.device)
    stats = torch.empty(n * heads, s, 2, dtype=torch.float32, device=qkv.device) if want_stats else None
    with _on_device(qkv):
        args = _block(cfg, q, k, v, table, mask, out.transpose(0, 1), stats)
        need = _lib.value("hivt_relative_attn_fwd_workspace_bytes", args, borders)
        ws = _workspace(need, qkv.device) if need else None
        _lib.call("hivt_relative_attn_fwd", args, borders, scale, _p(ws), need, _stream(qkv))
    return out, stats


class _RelativeSelfAttention(torch.autograd.Function):
    """The same on the fused projection [S, N, 3 D]: the three gradients are written where the projection's products
    read them."""

    @staticmethod
    def forward(ctx, qkv, table, heads, mask, cfg, borders, scale):
        out, stats = _self_forward(qkv, table, heads, mask, cfg, borders, scale, True)
        ctx.save_for_backward(qkv, table, mask, out, stats)
        ctx.cfg = (heads, cfg, borders, scale)
        return out.flatten(2)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        qkv, table, mask, out, stats = ctx.saved_tensors
        heads, cfg, borders, scale = ctx.cfg
        s, n, three_d = qkv.shape
        width = three_d // (3 * heads)
        split = lambda t: t.view(s, n, 3, heads, width).transpose(0, 1).unbind(2)  # noqa: E731
        d_qkv = torch.empty_like(qkv)
        d_out = d_out.reshape(s, n, heads, width).transpose(0, 1)
        d_table = _backward(d_out, *split(qkv), table, mask, out.transpose(0, 1), stats, cfg, borders, scale,
                            *split(d_qkv), ctx.needs_input_grad[1])
        return d_qkv, d_table, None, None, None, None, None


def _check(q, k, v, table, key_mask, causal, max_distance, bidirectional, scale, query_offset):
    """The argument checks of both entry points; (mask, cfg, borders, scale)."""
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"queries, keys and values must share one of float32, bfloat16, float16, got {q.dtype}, {k.dtype}, "
                        f"{v.dtype}")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"expected q [B, M, H, d], k and v [B, N, G, d], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    b, m, h, d = q.shape
    n, g = k.shape[1], k.shape[2]
    if h < 1 or g < 1 or h % g:
        raise ValueError(f"{h} query heads are no multiple of {g} key heads")
    if table.dtype != torch.float32 or table.dim() != 2 or table.shape[1] != h:
        raise ValueError(f"the bias table must be float32 [buckets, {h}], got {table.dtype} {tuple(table.shape)}")
    if not 1 <= d <= 128:
        raise _unsupported(f"relative-position attention with heads of {d} (1 to 128)")
    if m >= 2 ** 24 or n >= 2 ** 30 or b * h >= 2 ** 31:
        raise _unsupported(f"relative-position attention over {b} x {h} heads, {m} queries, {n} keys")
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != (b, n):
            raise ValueError(f"key_mask must be bool or uint8 [{b}, {n}] (nonzero: left out), got {key_mask.dtype} "
                             f"{tuple(key_mask.shape)}")
        if n > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
        if key_mask.requires_grad:
            raise ValueError("key_mask takes no gradient")
    _need_gpu(q, k, v, table, key_mask)
    for t in (k, v, table, key_mask):
        if t is not None and t.device != q.device:
            raise ValueError(f"tensors on {q.device} and {t.device}")
    bidirectional = (not causal) if bidirectional is None else bool(bidirectional)
    offset = n - m if query_offset is None else int(query_offset)
    if not -2 ** 29 < offset < 2 ** 29:
        raise ValueError(f"query_offset {offset} out of range")
    exact, starts, borders = _borders(int(table.shape[0]), int(max_distance), bidirectional)
    scale = d ** -0.5 if scale is None else float(scale)
    return key_mask, (int(bool(causal)), int(bidirectional), offset, exact, starts), borders, scale


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, causal: bool = False,
                       max_distance: int = 128, key_mask: Optional[torch.Tensor] = None,
                       bidirectional: Optional[bool] = None, scale: Optional[float] = None,
                       query_offset: Optional[int] = None) -> torch.Tensor:
    """``softmax(scale q k^T + table[bucket(key - query position)]) v`` -> [B, M, H, d], differentiable in q, k, v, table.

    q [B, M, H, d]; k, v [B, N, G, d] with H a multiple of G (query head h reads key head h // (H // G)); any strides.
    ``table`` float32 [buckets, H] (see ``relative_buckets``; ``bidirectional`` defaults to ``not causal``).  Query i
    stands at position i + ``query_offset``, by default N - M, so that the queries are the last of the keys: with M = 1
    the call is one step of a sequence.  ``key_mask`` [B, N]: True leaves a key out, whatever it and its value hold; a
    query without any key gives zeros and passes no gradient.  With ``causal``, keys behind the last query are not read (the
    unwritten end of a cache).  (Between the queries of one call the causal rule alone does not shield a row from a NaN or an
    infinity in a later value: weights of zero are multiplied with it.)  Deterministic; scores, weights and sums are
    fp32, weights enter the product with v and score gradients the products with q and k in the tensors' type."""
    mask, cfg, borders, scale = _check(q, k, v, table, key_mask, causal, max_distance, bidirectional, scale, query_offset)
    q, k, v, table = _heads_last(q), _heads_last(k), _heads_last(v), table.contiguous()
    if _recorded(q, k, v, table):
        return _RelativeAttention.apply(q, k, v, table, mask, cfg, borders, scale)
    return _forward(q, k, v, table, mask, cfg, borders, scale, False)[0]


def relative_self_attention(qkv: torch.Tensor, table: torch.Tensor, num_heads: int, causal: bool = True,
                            max_distance: int = 128, key_mask: Optional[torch.Tensor] = None,
                            bidirectional: Optional[bool] = None) -> torch.Tensor:
    """``relative_attention`` over dim 0 of the fused projection ``qkv`` [S, N, 3 D] -> [S, N, D] (the layout of
    ``temporal_attention``); ``key_mask`` [N, S]."""
    if qkv.dim() != 3 or num_heads < 1 or qkv.shape[2] % (3 * num_heads):
        raise ValueError(f"expected qkv [S, N, 3 D] with D a multiple of {num_heads} heads, got {tuple(qkv.shape)}")
    qkv = qkv.contiguous()
    s, n, three_d = qkv.shape
    q, k, v = qkv.view(s, n, 3, num_heads, three_d // (3 * num_heads)).transpose(0, 1).unbind(2)
    mask, cfg, borders, scale = _check(q, k, v, table, key_mask, causal, max_distance, bidirectional, None, None)
    table = table.contiguous()
    if _recorded(qkv, table):
        return _RelativeSelfAttention.apply(qkv, table, int(num_heads), mask, cfg, borders, scale)
    return _self_forward(qkv, table, int(num_heads), mask, cfg, borders, scale, False)[0].flatten(2)
