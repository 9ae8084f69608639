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
