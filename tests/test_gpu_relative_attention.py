"""Attention with a learned bias for each bucket of relative positions: forward and gradients against the formulas in 64
bits, at the sizes, masks, strides and types where it can go wrong.

Tolerances are bounds from rounding, computed element by element beside the reference: with u = eps / 2 of the tensors'
type and w = 2^-24 of fp32,
  scores     off by at most w (d + 8) (scale sum |q k| + |bias|): the weights by that, relatively, twice over (their own
             exponential and the sum they are divided by), and by w (N + 16) for the sum itself;
  out        u |out| for its rounding, u sum p |v| for the weights' rounding in the product, and the weights' own error;
  ds         (weights' error) (p |do| |v| + p |delta|), plus p times the error of delta;
  gradients  u of the result, u of what is rounded for the product (ds, p), and ds's own error."""
import math

import pytest
import torch

from hivt_gan_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
W = 2.0 ** -24


def bucket_matrix(m, n, offset, buckets, max_distance, bidirectional):
    exact, borders = ops.relative_buckets(buckets, max_distance, bidirectional)
    rel = torch.arange(n)[None, :] - (torch.arange(m)[:, None] + offset)
    dist = rel.abs() if bidirectional else (-rel).clamp(min=0)
    wide = exact + (dist[..., None] >= torch.tensor(borders + (2 ** 40,))).sum(-1)
    b = torch.where(dist < exact, dist, wide)
    return (b + buckets // 2 * (rel > 0) if bidirectional else b), rel


def reference(q, k, v, table, d_out, causal, max_distance, mask, bidirectional, scale, offset):
    """Values and bounds, in 64 bits on the CPU: {name: (value, bound)}."""
    u = torch.finfo(q.dtype).eps / 2
    q, k, v, table, d_out = (t.detach().cpu().double() for t in (q, k, v, table, d_out))
    mask = None if mask is None else mask.cpu().bool()
    B, M, H, d = q.shape
    N, G = k.shape[1], k.shape[2]
    bucket, rel = bucket_matrix(M, N, offset, table.shape[0], max_distance, bidirectional)
    ok = torch.ones(B, 1, M, N, dtype=torch.bool)
    if causal:
        ok = ok & (rel <= 0)
    if mask is not None:
        ok = ok & ~mask[:, None, None, :]
        k, v = (t.masked_fill(mask[:, :, None, None], 0.0) for t in (k, v))  # whatever they hold
    qh, oh = q.transpose(1, 2), d_out.transpose(1, 2)
    kh, vh = (t.transpose(1, 2).repeat_interleave(H // G, dim=1) for t in (k, v))
    bias = table[bucket].permute(2, 0, 1)
    s = scale * qh @ kh.transpose(2, 3) + bias
    mag = abs(scale) * qh.abs() @ kh.abs().transpose(2, 3) + bias.abs()
    s = s.masked_fill(~ok, -math.inf)
    top = s.amax(-1, keepdim=True) if N else s.new_zeros(B, H, M, 1)
    p = torch.exp(s - top.clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    p = p.masked_fill(~ok, 0.0)
    out = p @ vh
    e_s = W * (d + 8) * mag.masked_fill(~ok, 0.0) * 1.5
    e_p = e_s + (e_s.amax(-1, keepdim=True) if N else 0.0) + W * (N + 16)  # relative
    t_out = u * out.abs() + (p * (u + e_p)) @ vh.abs() * (1 + u)
    dp, dp_mag = oh @ vh.transpose(2, 3), oh.abs() @ vh.abs().transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = W * (d + 8)
    # delta for dq comes from the rounded output; the passes behind it use the corrected one
    t_delta_q = (oh.abs() * t_out).sum(-1, keepdim=True) + W * (d + 8) * (oh.abs() * out.abs()).sum(-1, keepdim=True)
    t_ds_one = e_p * p * (dp - delta).abs() + p * (e_dp * dp_mag + 4 * W * (dp.abs() + delta.abs()))
    t_delta = t_ds_one.sum(-1, keepdim=True) + W * (N + 16) * (ds.abs().sum(-1, keepdim=True)) + \
        e_p.amax(-1, keepdim=True) * t_delta_q if N else delta
    t_ds_q, t_ds = t_ds_one + p * t_delta_q, t_ds_one + p * t_delta
    group = lambda t: t.view(B, G, H // G, N, d).sum(2)  # noqa: E731
    dq = scale * ds @ kh
    t_dq = u * dq.abs() + abs(scale) * (t_ds_q * (1 + u) + (u + W * (N + 8)) * ds.abs()) @ kh.abs()
    dk = group(scale * ds.transpose(2, 3) @ qh)
    t_dk = u * dk.abs() + group(abs(scale) * (t_ds * (1 + u) + (u + W * (M * H // G + 8)) * ds.abs()).transpose(2, 3) @ qh.abs())
    dv = group(p.transpose(2, 3) @ oh)
    t_dv = u * dv.abs() + group((p * (e_p * (1 + u) + u + W * (M * H // G + 8))).transpose(2, 3) @ oh.abs())
    d_table, t_table = torch.zeros_like(table), torch.zeros_like(table)
    for b in range(table.shape[0]):
        at = (bucket == b)
        d_table[b] = (ds * at).sum((0, 2, 3))
        t_table[b] = ((t_ds + 64 * W * ds.abs()) * at).sum((0, 2, 3))
    t_table += W * d_table.abs()
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    return {"out": (back(out), back(t_out)), "dq": (back(dq), back(t_dq)), "dk": (back(dk), back(t_dk)),
            "dv": (back(dv), back(t_dv)), "d_table": (d_table, t_table)}


def close(name, got, value, bound):
    got = got.detach().cpu().double()
    assert got.shape == value.shape
    assert bool(torch.isfinite(got).all()), f"{name} holds values that are not finite"
    tiny = {torch.float16: 2.0 ** -25}.get(got.dtype, 0.0)
    over = (got - value).abs() - bound * 1.0 - 1e-30 - tiny
    assert float(over.max() if over.numel() else -1.0) <= 0.0, \
        f"{name}: off by {float((got - value).abs().max()):.3e}, allowed there {float(bound.flatten()[over.argmax()]):.3e}"


def inputs(B, M, N, H, G, d, dtype, buckets, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k, v, o = r(B, M, H, d).to(dtype), r(B, N, G, d).to(dtype), r(B, N, G, d).to(dtype), r(B, M, H, d).to(dtype)
    return [t.to(DEV) for t in (q, k, v, r(buckets, H), o)]


def check(q, k, v, table, d_out, causal, max_distance=16, mask=None, bidirectional=None, scale=None, offset=None):
    bidirectional = (not causal) if bidirectional is None else bidirectional
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    out = ops.relative_attention(*leaves, causal=causal, max_distance=max_distance, key_mask=mask, bidirectional=bidirectional,
                                 scale=scale, query_offset=offset)
    grads = torch.autograd.grad(out, leaves, d_out)
    ref = reference(q, k, v, table, d_out, causal, max_distance, mask, bidirectional,
                    q.shape[-1] ** -0.5 if scale is None else scale, k.shape[1] - q.shape[1] if offset is None else offset)
    for name, got in zip(("out", "dq", "dk", "dv", "d_table"), (out, *grads)):
        assert got.dtype == (torch.float32 if name == "d_table" else q.dtype)
        tiny = 2.0 ** -25 if q.dtype == torch.float16 and name != "d_table" else 0.0  # fp16's subnormal step
        value, bound = ref[name]
        close(name, got, value, bound + tiny)
    return out, grads


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,M,N,H,G,d", [
    (3, 21, 21, 8, 8, 16), (2, 1, 37, 4, 2, 8), (1, 1, 1, 1, 1, 4), (2, 65, 65, 2, 1, 32), (1, 130, 257, 6, 2, 80),
    (2, 40, 200, 3, 3, 128), (1, 17, 64, 2, 2, 5), (1, 300, 300, 2, 1, 64), (2, 33, 31, 4, 4, 96), (1, 64, 129, 4, 1, 20),
    (1, 2, 500, 8, 2, 24), (1, 5, 3, 1, 1, 1)])
def test_forward_and_gradients(dtype, causal, B, M, N, H, G, d):
    check(*inputs(B, M, N, H, G, d, dtype, 8), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("M", [1, 19, 150])
def test_masked_keys_may_hold_anything(dtype, causal, M):
    """Empty rows, whole tiles without a key, lone keys, and NaN / infinity / the lowest value behind the mask."""
    B, N, H, G, d = 6, 200, 4, 2, 16
    q, k, v, table, o = inputs(B, M, N, H, G, d, dtype, 8)
    mask = torch.zeros(B, N, dtype=torch.bool)
    mask[0, :] = True                 # nothing left
    mask[1, :130] = True              # late start: tiles without a key, and causal rows without one
    mask[2, 7:] = True                # early end
    mask[3, :] = True
    mask[3, 131] = False              # one key
    mask[4] = torch.rand(N, generator=torch.Generator().manual_seed(1)) < 0.5
    mask = mask.to(DEV)
    for t, fill in ((k, math.nan), (v, math.inf)):
        t[:, :, 0][mask] = fill
        t[:, :, 1][mask] = torch.finfo(dtype).min
    out, grads = check(q, k, v, table, o, causal, mask=mask)
    assert float(out[0].abs().max()) == 0.0 and all(float(g[0].abs().max()) == 0.0 for g in grads[:3])
    assert float(grads[1][mask].abs().max()) == 0.0 and float(grads[2][mask].abs().max()) == 0.0


@pytest.mark.parametrize("buckets,distance,causal,bidirectional", [
    (4, 3, False, True), (2, 2, True, False), (3, 40, True, False), (32, 128, False, True), (32, 100, True, True),
    (6, 1000, False, False), (64, 4096, False, True), (16, 9, True, False)])
def test_buckets(buckets, distance, causal, bidirectional):
    check(*inputs(2, 150, 190, 2, 1, 16, torch.float32, buckets), causal=causal, max_distance=distance,
          bidirectional=bidirectional)


@pytest.mark.parametrize("offset", [-7, 0, 3, 500, -300])
@pytest.mark.parametrize("causal", [False, True])
def test_query_offsets(offset, causal):
    check(*inputs(1, 70, 150, 2, 2, 16, torch.float32, 8), causal=causal, offset=offset)


def test_scale_and_lowest_biases():
    q, k, v, table, o = inputs(1, 40, 90, 2, 2, 16, torch.float32, 8)
    check(q, k, v, table, o, False, scale=0.0)
    check(q, k, v, table, o, True, scale=-0.7)
    table[3, 0] = torch.finfo(torch.float32).min  # a bias that shuts a bucket out
    check(q, k, v, table, o, False)
    low = torch.full_like(table, torch.finfo(torch.float32).min)  # every bias the lowest value: equal weights
    out = ops.relative_attention(q, k, v, low, max_distance=16)
    assert torch.allclose(out, v.mean(1, keepdim=True).expand_as(out), atol=1e-6)
    shut = torch.full_like(table, -math.inf)
    assert float(ops.relative_attention(q, k, v, shut, max_distance=16).abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    """Slices of a fused projection, transposed layouts, odd row strides, an address that is not aligned: equal bits."""
    B, M, H, d = 2, 70, 4, 16
    q, k, v, table, o = inputs(B, M, M, H, H, d, dtype, 8)
    plain = check(q, k, v, table, o, False)
    fused = torch.empty(M, B, 3, H, d, dtype=dtype, device=DEV)
    for i, t in enumerate((q, k, v)):
        fused[:, :, i] = t.transpose(0, 1)
    odd = torch.empty(B, M, H, d + 3, dtype=dtype, device=DEV)[..., 1:d + 1]
    odd.copy_(k)
    spaced = torch.empty(B, H, M, d, dtype=dtype, device=DEV).transpose(1, 2)
    spaced.copy_(v)
    last = torch.empty(B, M, d, H, dtype=dtype, device=DEV).transpose(2, 3)  # head width not contiguous: copied
    last.copy_(q)
    for qq, kk, vv in ((fused[:, :, 0].transpose(0, 1), fused[:, :, 1].transpose(0, 1), fused[:, :, 2].transpose(0, 1)),
                       (last, odd, spaced)):
        got = check(qq, kk, vv, table, o, False)
        assert torch.equal(got[0], plain[0]) and all(torch.equal(a, b) for a, b in zip(got[1], plain[1]))
    wide = torch.zeros(B, 2 * M, dtype=torch.uint8, device=DEV)[:, ::2]
    wide[:, :9] = 1
    check(q, k, v, table, o.transpose(0, 1).contiguous().transpose(0, 1), True, mask=wide)


def test_long_axis_is_split_and_joined():
    for dtype, H, G, M in ((torch.bfloat16, 8, 2, 1), (torch.float32, 4, 4, 1), (torch.float16, 4, 1, 3)):
        q, k, v, table, o = inputs(2, M, 5003, H, G, 64, dtype, 32)
        mask = torch.zeros(2, 5003, dtype=torch.bool, device=DEV)
        mask[1, 40:4900] = True
        check(q, k, v, table, o, True, 128, mask)
        check(q, k, v, table, o, False, 128)


def test_many_sequences_with_shared_heads():
    """Enough key tiles that a workgroup takes all heads of a group, instead of one with the shares added later."""
    for causal in (False, True):
        check(*inputs(520, 40, 70, 4, 2, 8, torch.float32, 8), causal=causal)


def test_equal_calls_give_equal_bits():
    q, k, v, table, o = inputs(4, 200, 200, 8, 2, 32, torch.bfloat16, 32)
    first = check(q, k, v, table, o, True, 64)
    for _ in range(3):
        again = check(q, k, v, table, o, True, 64)
        assert torch.equal(first[0], again[0]) and all(torch.equal(a, b) for a, b in zip(first[1], again[1]))


def test_gradients_against_differences():
    q, k, v, table, o = inputs(1, 9, 13, 2, 1, 4, torch.float32, 8)
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    grads = torch.autograd.grad(ops.relative_attention(*leaves, max_distance=8), leaves, o)

    def value(args):  # the formula in 64 bits
        return (reference(*args, o, False, 8, None, True, 0.5, 4)["out"][0] * o.cpu().double()).sum()

    gen = torch.Generator().manual_seed(3)
    for i, g in enumerate(grads):
        step = torch.randn(leaves[i].shape, generator=gen).double()
        ends = []
        for sign in (1, -1):
            args = [t.detach().cpu().double() for t in leaves]
            args[i] = args[i] + sign * 1e-5 * step
            ends.append(value(args))
        numeric = float(ends[0] - ends[1]) / 2e-5
        # central differences: third derivatives of order one times h^2; fp32 gradients summed over fewer than 60 entries
        assert abs(numeric - float((g.cpu().double() * step).sum())) < 1e-5 * max(1.0, abs(numeric))


def test_partial_gradients_and_none():
    q, k, v, table, o = inputs(1, 30, 30, 2, 2, 16, torch.float32, 8)
    whole = check(q, k, v, table, o, False)
    for i, name in enumerate("qkvt"):
        args = [t.detach() for t in (q, k, v, table)]
        args[i].requires_grad_(True)
        (g,) = torch.autograd.grad(ops.relative_attention(*args, max_distance=16), (args[i],), o)
        assert torch.equal(g, whole[1][i]), name
    with torch.no_grad():
        assert torch.equal(ops.relative_attention(q, k, v, table, max_distance=16), whole[0])


@pytest.mark.parametrize("B,M,N", [(0, 5, 5), (2, 0, 5), (2, 5, 0)])
def test_empty(B, M, N):
    q, k, v, table, o = (t.requires_grad_(True) for t in inputs(B, M, N, 2, 2, 16, torch.float32, 8))
    out = ops.relative_attention(q, k, v, table, max_distance=16)
    grads = torch.autograd.grad(out, (q, k, v, table), o.detach())
    assert out.shape == q.shape and all(g.shape == t.shape for g, t in zip(grads, (q, k, v, table)))
    assert all(t.numel() == 0 or float(t.abs().max()) == 0.0 for t in (out, *grads))


@pytest.mark.parametrize("S,N,H,d,causal", [(21, 50, 8, 16, True), (100, 3, 2, 32, False), (1, 4, 2, 8, True)])
def test_fused_projection_form(S, N, H, d, causal):
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(S, N, 3 * H * d, generator=gen).to(DEV).requires_grad_(True)
    table = torch.randn(8, H, generator=gen).to(DEV).requires_grad_(True)
    o = torch.randn(S, N, H * d, generator=gen).to(DEV)
    mask = torch.zeros(N, S, dtype=torch.bool, device=DEV)
    mask[0, : S // 2] = True
    out = ops.relative_self_attention(qkv, table, H, causal=causal, max_distance=16, key_mask=mask)
    g_qkv, g_table = torch.autograd.grad(out, (qkv, table), o)
    q, k, v = (t.transpose(0, 1).contiguous() for t in qkv.detach().view(S, N, 3, H, d).unbind(2))
    want = check(q, k, v, table.detach(), o.view(S, N, H, d).transpose(0, 1).contiguous(), causal, 16, mask)
    assert torch.equal(out.view(S, N, H, d).transpose(0, 1), want[0])
    for got, ref in zip(g_qkv.view(S, N, 3, H, d).unbind(2), want[1]):
        assert torch.equal(got.transpose(0, 1), ref)
    assert torch.equal(g_table, want[1][3])


def test_captured_and_replayed():
    """Two captured passes whose workspaces live at once, replayed in turn with eager work between, against the eager."""
    cases = []
    for seed, M in ((1, 50), (2, 1)):
        q, k, v, table, o = inputs(2, M, 600, 4, 2, 32, torch.bfloat16, 32, seed)
        leaves = [t.requires_grad_(True) for t in (q, k, v, table)]

        def step(leaves=leaves, o=o):
            out = ops.relative_attention(*leaves, causal=True)
            return (out.detach(), *torch.autograd.grad(out, leaves, o))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        cases.append((graph, got, leaves, step))
    for round_ in range(3):
        for graph, got, leaves, step in cases:
            with torch.no_grad():
                for t in leaves:
                    t.mul_(0.9).add_(0.01 * round_)
            graph.replay()
            torch.cuda.synchronize()
            seen = [t.clone() for t in got]
            want = step()
            assert all(torch.equal(a, b) for a, b in zip(seen, want))


def test_on_a_side_stream():
    q, k, v, table, o = inputs(2, 100, 100, 4, 4, 16, torch.float32, 8)
    want = ops.relative_attention(q, k, v, table, max_distance=16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.relative_attention(q, k, v, table, max_distance=16)
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits():
    """Rows of a buffer that are further apart than 2^31 elements."""
    stride = 2 ** 31 + 64
    if torch.cuda.mem_get_info()[0] < 3 * stride * 2 + (1 << 30):
        pytest.skip("not enough free memory")
    buf = torch.zeros(stride + 4096, dtype=torch.bfloat16, device=DEV)
    far = buf.as_strided((2, 33, 1, 16), (stride, 16, 16, 1))
    q, k, v, table, o = inputs(2, 33, 33, 1, 1, 16, torch.bfloat16, 8)
    far.copy_(k)
    check(q, far, far, table, o, False)
    far.copy_(q)
    check(far, k, v, table, o, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,first", [(1, 40, 22), (3, 32, 10), (1, 700, 300), (19, 300, 100), (90, 300, 130), (70, 200, -30),
                                       (5, 64, -5)])
def test_unwritten_end_of_a_cache(dtype, M, N, first):
    """Causal, behind the last query's position the keys and values are not numbers; nothing sees them."""
    H, G, d = 4, 2, 24
    q, k, v, table, o = inputs(2, M, N, H, G, d, dtype, 8)
    written = max(0, M + first)
    for clean in (k, v):
        clean[:, written:] = 0.0
    want, want_grads = check(q, k, v, table, o, True, offset=first)
    k[:, written:], v[:, written:] = math.nan, math.inf
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    out = ops.relative_attention(*leaves, causal=True, max_distance=16, query_offset=first)
    grads = torch.autograd.grad(out, leaves, o)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))
    assert not bool(grads[1][:, written:].any()) and not bool(grads[2][:, written:].any())


def test_without_gradients_equal_bits():
    q, k, v, table, o = inputs(2, 70, 90, 4, 2, 16, torch.bfloat16, 8)
    want = ops.relative_attention(q, k, v, table.requires_grad_(True), causal=True, max_distance=16)
    assert want.requires_grad
    with torch.no_grad():
        got = ops.relative_attention(q, k, v, table, causal=True, max_distance=16)
    assert not got.requires_grad and torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,H,G,d,buckets,distance,causal", [
    (200, 333, 4, 2, 128, 32, 4096, True), (131, 131, 2, 1, 97, 32, 20, False), (70, 700, 3, 3, 100, 16, 300, False),
    (257, 190, 2, 2, 127, 8, 16, True), (1, 500, 16, 1, 128, 32, 4096, True), (33, 65, 8, 1, 81, 32, 4096, False)])
def test_wide_heads(dtype, M, N, H, G, d, buckets, distance, causal):
    """Heads from 81 on, masked in runs (whole tiles too) and one by one, with the longest tables and odd strides."""
    q, k, v, table, o = inputs(2, M, N, H, G, d, dtype, buckets)
    mask = torch.rand(2, N, generator=torch.Generator().manual_seed(3)) < 0.3
    mask[0, 64:192] = True
    mask[1, :70] = True
    check(q, k, v, table, o, causal, max_distance=distance, mask=mask.to(DEV))
    wide = torch.zeros(2, N, G, 2 * d + 3, dtype=dtype, device=DEV)
    wide[..., 1:d + 1], wide[..., d + 2:2 * d + 2] = k, v
    check(q, wide[..., 1:d + 1], wide[..., d + 2:2 * d + 2], table, o[:, :, :1].expand(2, M, H, d), causal,
          max_distance=distance)


def test_broadcast_inputs():
    """Tensors whose strides are zero: one sequence of keys for the batch, one query row, one gradient."""
    q, k, v, table, o = inputs(3, 80, 90, 4, 2, 16, torch.float32, 8)
    check(q[:1, :1].expand(3, 80, 4, 16), k[:1].expand(3, 90, 2, 16), v[:, :1].expand(3, 90, 2, 16), table,
          o[:1, :1, :1, :1].expand(3, 80, 4, 16), True)


def test_refusals():
    q, k, v, table, o = inputs(1, 8, 8, 4, 2, 16, torch.float32, 8)
    call = ops.relative_attention
    with pytest.raises(TypeError):
        call(q.double(), k.double(), v.double(), table)
    with pytest.raises(TypeError):
        call(q, k.half(), v, table)
    with pytest.raises(ValueError):
        call(q, k[:, :, :1].expand(1, 8, 3, 16), v[:, :, :1].expand(1, 8, 3, 16), table)
    with pytest.raises(ValueError):
        call(q, k, v[:, :7], table)
    with pytest.raises(ValueError):
        call(q, k, v, table[:, :3])
    with pytest.raises(ValueError):
        call(q, k, v, table.half())
    with pytest.raises(ValueError):
        call(q, k, v, table, key_mask=torch.zeros(1, 7, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError):
        call(q, k, v, table, key_mask=torch.zeros(1, 8, device=DEV))
    with pytest.raises(ops.UnsupportedShapeError):
        big = torch.zeros(1, 4, 2, 129, device=DEV)
        call(big, big, big, table[:, :2])
    with pytest.raises(RuntimeError, match="GPU only"):
        call(q, k.cpu(), v, table)
    with pytest.raises(ValueError):
        ops.relative_self_attention(torch.zeros(4, 2, 50, device=DEV), table, 4)
