"""CPU-only checks of the relative-position attention's host side."""
import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_relative_buckets_are_decided_in_whole_numbers():
    from fractions import Fraction
    from hivt_gan_amd import ops
    for buckets, distance, both in ((32, 128, True), (32, 128, False), (8, 16, True), (6, 1000, False), (64, 4096, True),
                                    (3, 40, False), (2, 2, False), (4, 2, True)):
        exact, borders = ops.relative_buckets(buckets, distance, both)
        side = buckets // 2 if both else buckets
        assert exact == side // 2 and len(borders) == side - exact - 1
        for t, n in enumerate(borders, start=1):  # n is the least with (n / exact)^L >= (distance / exact)^t
            reach = Fraction(distance, exact) ** t
            assert Fraction(n, exact) ** (side - exact) >= reach
            assert n == exact or Fraction(n - 1, exact) ** (side - exact) < reach
        assert list(borders) == sorted(borders)
    for bad in ((1, 8, False), (2, 8, True), (7, 8, True), (32, 8, True)):
        with pytest.raises(ValueError):
            ops.relative_buckets(*bad)
    with pytest.raises(ops.UnsupportedShapeError):
        ops.relative_buckets(512, 1000, False)
    with pytest.raises(ops.UnsupportedShapeError):
        ops.relative_buckets(32, 100000, True)


def test_relative_attention_argument_block_matches_the_header():
    header = open(os.path.join(ROOT, "include", "hivt_mi355.h")).read()
    from hivt_gan_amd import ops_relative
    body = re.search(r"typedef struct \{((?:(?!typedef struct).)*?)\} hivt_relative_attn;", header, re.S).group(1)
    members = 0
    for decl in re.findall(r"int64_t ([^;]*);", re.sub(r"/\*.*?\*/", "", body, flags=re.S)):
        for name in decl.split(","):
            size = re.search(r"\[(\d+)\]", name)
            members += int(size.group(1)) if size else 1
    assert ctypes.sizeof(ops_relative._Block) == 8 * members


def test_rotary_argument_block_matches_the_header():
    header = open(os.path.join(ROOT, "include", "hivt_mi355.h")).read()
    from hivt_gan_amd import ops_rotary
    body = re.search(r"typedef struct \{((?:(?!typedef struct).)*?)\} hivt_qk_norm_rotary;", header, re.S).group(1)
    members = 0
    for decl in re.findall(r"int64_t ([^;]*);", re.sub(r"/\*.*?\*/", "", body, flags=re.S)):
        for name in decl.split(","):
            size = re.search(r"\[(\d+)\]", name)
            members += int(size.group(1)) if size else 1
    assert ctypes.sizeof(ops_rotary._Block) == 8 * members


def _cpu(*shape, dtype=None):
    import torch
    return torch.zeros(*shape, dtype=dtype or torch.float32)


def test_relative_attention_refuses_on_the_host():
    import torch
    from hivt_gan_amd import ops
    q, k, table = _cpu(2, 5, 4, 16), _cpu(2, 7, 2, 16), _cpu(32, 4)
    for args, kwargs, error in (
            ((q.double(), k.double(), k.double(), table), {}, TypeError),
            ((q, k.half(), k, table), {}, TypeError),
            ((q[0], k, k, table), {}, ValueError),
            ((q, k, k[:, :6], table), {}, ValueError),
            ((q, k[:1], k[:1], table), {}, ValueError),
            ((q, _cpu(2, 7, 3, 16), _cpu(2, 7, 3, 16), table), {}, ValueError),
            ((q, k, k, table[:, :3]), {}, ValueError),
            ((q, k, k, table.half()), {}, ValueError),
            ((_cpu(2, 5, 4, 130), _cpu(2, 7, 2, 130), _cpu(2, 7, 2, 130), table), {}, ops.UnsupportedShapeError),
            ((_cpu(2, 5, 4, 0), _cpu(2, 7, 2, 0), _cpu(2, 7, 2, 0), table), {}, ops.UnsupportedShapeError),
            ((q, k, k, table), dict(key_mask=_cpu(2, 7)), ValueError),
            ((q, k, k, table), dict(key_mask=_cpu(2, 6, dtype=torch.bool)), ValueError),
            ((q, k, k, table), {}, RuntimeError)):  # on the CPU
        with pytest.raises(error):
            ops.relative_attention(*args, **kwargs)
    with pytest.raises(ValueError):
        ops.relative_self_attention(_cpu(5, 2, 50), table, 4)
    with pytest.raises(ValueError):
        ops.relative_self_attention(_cpu(5, 2, 48), table, 0)


def test_norm_and_rotation_refuse_on_the_host():
    import torch
    from hivt_gan_amd import ops
    q, k, w = _cpu(2, 5, 4, 16), _cpu(2, 5, 2, 16), _cpu(16)
    for args, kwargs, error in (
            ((q.double(), k.double(), w, w), {}, TypeError),
            ((q, k.half(), w, w), {}, TypeError),
            ((q, k[:, :4], w, w), {}, ValueError),
            ((q[..., :15], k[..., :15], w[:15], w[:15]), {}, ops.UnsupportedShapeError),
            ((_cpu(1, 1, 1, 258), _cpu(1, 1, 1, 258), _cpu(258), _cpu(258)), {}, ops.UnsupportedShapeError),
            ((q, k, w[:8], w), {}, ValueError),
            ((q, k, w.half(), w), {}, ValueError),
            ((q, k, w, w), dict(rotary_dim=18), ValueError),
            ((q, k, w, w), dict(rotary_dim=5), ValueError),
            ((q, k, w, w), dict(theta=0.0), ValueError),
            ((q, k, w, w), dict(theta=float("nan")), ValueError),
            ((q, k, w, w), dict(eps=0.0), ValueError),
            ((q, k, w, w), dict(positions=_cpu(5)), ValueError),
            ((q, k, w, w), dict(positions=_cpu(4, dtype=torch.int64)), ValueError),
            ((q, k, w, w), {}, RuntimeError)):
        with pytest.raises(error):
            ops.qk_norm_rotary(*args, **kwargs)


def test_orthogonalize_refuses_on_the_host():
    import torch
    from hivt_gan_amd import ops, ops_orthogonal
    x = _cpu(4, 6)
    assert ops.orthogonalize([]) == []
    for args, kwargs, error in (
            (([x.double()],), {}, TypeError),
            (([x, x.half()],), {}, TypeError),
            (([x[0]],), {}, ValueError),
            (([x],), dict(steps=0), ValueError),
            (([x],), dict(steps=17), ValueError),
            (([x],), dict(eps=0.0), ValueError),
            (([x],), {}, RuntimeError)):
        with pytest.raises(error):
            ops.orthogonalize(*args, **kwargs)
    # an output may be its own matrix, and no other's memory
    store = _cpu(12, 6)
    a, b, c = store[:4], store[4:8], store[8:]
    for ins, outs in (([a, b], [a, b]), ([a, a], [b, c]), ([a], [b]), ([a, b], [c, b]), ([a, store[:0]], [a, store[:0]])):
        ops_orthogonal._refuse_overlaps(ins, outs)
    for ins, outs in (([a, b], [b, a]), ([a, b], [c, c]), ([a, b], [b, c]), ([a], [store[1:5]]), ([a, a], [a, c]),
                      ([store[0:6], c], [store[0:6], store[5:9]]), ([store, a], [torch.empty_like(store), b])):
        with pytest.raises(ValueError):
            ops_orthogonal._refuse_overlaps(ins, outs)
