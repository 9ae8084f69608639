"""Norm and rotation of queries and keys: forward and gradients against the formulas in 64 bits.

Bounds, with u = eps / 2 of the tensors' type and w = 2^-24: the result's rounding u |y|, and for the fp32 arithmetic
behind it w times the number of roundings on the way (sums of d squares: d / 2 + 8 relative, halved by the root; sine and
cosine: 4 each of their scale) times the sum of the magnitudes that are added.  An angle is position * rate in 64 bits
on both sides: the rate, its division by the whole turn, the whole turn itself and the product each round by 2^-53 of
the angle there, the rate and the product here, so the two angles differ by up to 6 * 2^-53 of the angle, and a turned
pair by that times its magnitude (1e-3 at position 10^13; below 2^31 it is under 2e-6)."""
import math

import pytest
import torch

from hivt_gan_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
W = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def turn(x, angle, rotary, interleaved, magnitude=False):
    """x [.., d] turned by angle [B, S, rotary / 2]; with ``magnitude`` the sum of the parts' magnitudes."""
    if rotary == 0:
        return x.abs() if magnitude else x
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    first = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    second = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    a, b, y = x[..., first], x[..., second], x.clone()
    if magnitude:
        y = x.abs().clone()
        y[..., first] = y[..., second] = a.abs() + b.abs()
    else:
        y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def reference(x, w, dy, positions, rotary, theta, interleaved, eps):
    u = torch.finfo(x.dtype).eps / 2
    x, w, dy = (t.detach().cpu().double() for t in (x, w, dy))
    B, S, H, d = x.shape
    pos = torch.arange(S)[None].expand(B, S) if positions is None else positions.cpu().expand(B, S)
    angle = pos.double()[..., None] * theta ** (-2.0 * torch.arange(rotary // 2).double() / max(1, rotary))
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    n = x * r
    k = W * (d / 4 + 16)  # relative error of a normalised component, and of a turned one beside its magnitude
    e_angle = torch.zeros(*angle.shape[:2], 1, d).double()
    if rotary:
        pairs = 6 * 2.0 ** -53 * angle.abs()[:, :, None]
        e_angle[..., :rotary] = torch.stack((pairs, pairs), -1).flatten(-2) if interleaved else torch.cat((pairs, pairs), -1)
    y = turn(n * w, angle, rotary, interleaved)
    t_y = u * y.abs() + (k + 8 * W + e_angle) * turn(n * w, angle, rotary, interleaved, True) * (1 + u)
    b = turn(dy, -angle, rotary, interleaved)
    e_b = (8 * W + e_angle) * turn(dy, -angle, rotary, interleaved, True)
    g = w * b
    mean, mean_mag = (g * n).mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    e_mean = (2 * k + W * (d + 8)) * mean_mag + (e_b * (w * n).abs()).mean(-1, keepdim=True)
    dx = r * (g - n * mean)
    t_dx = u * dx.abs() + r * (1 + u) * (e_b * w.abs() + 2 * k * (g.abs() + n.abs() * mean.abs()) + n.abs() * e_mean)
    dw = (b * n).sum((0, 1, 2))
    rows = B * S * H
    t_dw = ((e_b + (2 * k + W * (rows + 16)) * b.abs()) * n.abs()).sum((0, 1, 2))
    return (y, t_y), (dx, t_dx), (dw, t_dw)


def close(name, got, value, bound, dtype):
    got = got.detach().cpu().double()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    assert got.shape == value.shape and bool(torch.isfinite(got).all()), name
    over = (got - value).abs() - bound - tiny
    assert float(over.max()) <= 0.0, f"{name}: off by {float((got - value).abs().max()):.3e}"


def check(q, k, wq, wk, dq, dk, positions=None, rotary=None, theta=10000.0, interleaved=False, eps=1e-6):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    out = ops.qk_norm_rotary(*leaves, positions=positions, rotary_dim=rotary, theta=theta, interleaved=interleaved, eps=eps)
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    rotary = q.shape[-1] if rotary is None else rotary
    for i, (x, w, dy) in enumerate(((q, wq, dq), (k, wk, dk))):
        ref = reference(x, w, dy, positions, rotary, theta, interleaved, eps)
        assert out[i].dtype == x.dtype and grads[2 + i].dtype == w.dtype
        close(f"out[{i}]", out[i], *ref[0], x.dtype)
        close(f"dx[{i}]", grads[i], *ref[1], x.dtype)
        value, bound = ref[2]
        close(f"dw[{i}]", grads[2 + i], value, bound + torch.finfo(w.dtype).eps / 2 * value.abs(), w.dtype)
    return out, grads


def inputs(B, S, H, G, d, dtype, seed=0, wtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = [2 * r(B, S, H, d), 0.5 * r(B, S, G, d)]
    w = [1 + 0.2 * r(d), 1 + 0.2 * r(d)]
    g = [r(B, S, H, d), r(B, S, G, d)]
    return [x.to(dtype).to(DEV) for x in t] + [x.to(wtype).to(DEV) for x in w] + [x.to(dtype).to(DEV) for x in g]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,G,d,rotary", [
    (2, 21, 8, 8, 16, 16), (1, 1, 1, 1, 2, 2), (3, 5, 4, 2, 80, 80), (1, 100, 3, 1, 64, 32), (2, 7, 5, 5, 6, 4),
    (1, 33, 2, 2, 256, 256), (1, 9, 2, 1, 130, 66), (2, 3, 32, 8, 128, 128), (1, 40, 2, 2, 20, 10), (2, 6, 2, 1, 254, 2),
    (1, 11, 3, 3, 32, 0)])
def test_forward_and_gradients(dtype, interleaved, B, S, H, G, d, rotary):
    check(*inputs(B, S, H, G, d, dtype), rotary=rotary, interleaved=interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions(dtype, kind):
    args = inputs(2, 50, 4, 2, 64, dtype)
    far = torch.tensor([0, -5, 1, 2 ** 31 - 1, 10 ** 6, 131071] + list(range(44)), dtype=kind, device=DEV)
    check(*args, positions=far)
    both = torch.stack((far, far.flip(0)))
    check(*args, positions=both, theta=5e5)
    check(*args, positions=both.t().contiguous().t(), theta=1.0, eps=0.1)
    if kind == torch.int64:
        check(*args, positions=far * 2 ** 12)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_alignment_and_weights_of_the_tensors_type(dtype):
    B, S, H, d = 2, 30, 4, 32
    q, k, wq, wk, dq, dk = inputs(B, S, H, H, d, dtype, wtype=dtype)
    plain = check(q, k, wq, wk, dq, dk)
    fused = torch.stack((q, k), dim=2).transpose(0, 1).contiguous().transpose(0, 1)  # [B, S, 2, H, d], positions first
    odd = torch.empty(B, S, H, d + 1, dtype=dtype, device=DEV)[..., 1:]
    odd.copy_(k)
    swapped = q.transpose(2, 3).contiguous().transpose(2, 3)
    for qq, kk in ((fused[:, :, 0], fused[:, :, 1]), (swapped, odd)):
        got = check(qq, kk, wq, wk, dq.transpose(0, 1).contiguous().transpose(0, 1), dk)
        for a, b in zip(got[0], plain[0]):
            assert torch.equal(a, b) or float((a.double() - b.double()).abs().max()) <= 2 * torch.finfo(dtype).eps * 8


def test_zero_rows_large_and_tiny_values():
    q, k, wq, wk, dq, dk = inputs(2, 9, 2, 2, 16, torch.float32)
    q[0, 0] = 0.0
    q[0, 1] *= 1e15
    q[0, 2] *= 1e-15
    out, grads = check(q, k, wq, wk, dq, dk)
    assert float(out[0][0, 0].detach().abs().max()) == 0.0


def test_many_rows_and_equal_bits():
    args = inputs(600, 21, 8, 8, 16, torch.float32)
    first = check(*args)
    again = check(*args)
    for a, b in zip((*first[0], *first[1]), (*again[0], *again[1])):
        assert torch.equal(a, b)


def test_gradients_against_differences():
    args = inputs(1, 3, 2, 1, 8, torch.float32)
    _, grads = check(*args, rotary=4)
    gen = torch.Generator().manual_seed(1)

    def value(q, k, wq, wk):
        total = 0.0
        for x, w, dy in ((q, wq, args[4]), (k, wk, args[5])):
            total += float((reference(x, w, dy, None, 4, 10000.0, False, 1e-6)[0][0] * dy.cpu().double()).sum())
        return total

    for i, g in enumerate(grads):
        step = torch.randn(args[i].shape, generator=gen).double()
        ends = []
        for sign in (1, -1):
            at = [t.cpu().double() for t in args[:4]]
            at[i] = at[i] + sign * 1e-5 * step
            ends.append(value(*at))
        numeric = (ends[0] - ends[1]) / 2e-5
        assert abs(numeric - float((g.cpu().double() * step).sum())) < 1e-5 * max(1.0, abs(numeric))


def test_one_gradient_of_two():
    q, k, wq, wk, dq, dk = inputs(1, 6, 2, 2, 16, torch.float32)
    whole = check(q, k, wq, wk, dq, torch.zeros_like(dk))
    q.requires_grad_(True)
    out, _ = ops.qk_norm_rotary(q, k, wq, wk)
    (g,) = torch.autograd.grad(out, (q,), dq)  # the keys' output is not used
    assert torch.equal(g, whole[1][0])
    with torch.no_grad():
        assert torch.equal(ops.qk_norm_rotary(q, k, wq, wk)[0], whole[0][0])


@pytest.mark.parametrize("B,S", [(0, 4), (3, 0)])
def test_empty(B, S):
    args = [t.requires_grad_(True) for t in inputs(B, S, 2, 2, 16, torch.float32)[:4]]
    out = ops.qk_norm_rotary(*args)
    grads = torch.autograd.grad(out, args, (torch.zeros_like(out[0]), torch.zeros_like(out[1])))
    assert out[0].shape == (B, S, 2, 16) and float(grads[2].abs().max()) == 0.0 == float(grads[3].abs().max())


def test_captured_and_replayed():
    args = inputs(3, 40, 4, 2, 32, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in args[:4]]

    def step():
        out = ops.qk_norm_rotary(*leaves)
        return (*[o.detach() for o in out], *torch.autograd.grad(out, leaves, args[4:]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            for t in leaves:
                t.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(seen, step()))


def test_refusals():
    q, k, wq, wk, _, _ = inputs(1, 4, 2, 2, 16, torch.float32)
    call = ops.qk_norm_rotary
    with pytest.raises(TypeError):
        call(q.double(), k.double(), wq, wk)
    with pytest.raises(TypeError):
        call(q, k.half(), wq, wk)
    with pytest.raises(ValueError):
        call(q, k[:, :3], wq, wk)
    with pytest.raises(ValueError):
        call(q, k, wq[:8], wk)
    with pytest.raises(ValueError):
        call(q, k, wq.half(), wk)
    for bad in (-2, 3, 18):
        with pytest.raises(ValueError):
            call(q, k, wq, wk, rotary_dim=bad)
    with pytest.raises(ValueError):
        call(q, k, wq, wk, eps=0.0)
    with pytest.raises(ValueError):
        call(q, k, wq, wk, theta=math.inf)
    with pytest.raises(ValueError):
        call(q, k, wq, wk, positions=torch.zeros(4, device=DEV))
    with pytest.raises(ValueError):
        call(q, k, wq, wk, positions=torch.zeros(5, dtype=torch.int64, device=DEV))
    with pytest.raises(ops.UnsupportedShapeError):
        odd = torch.zeros(1, 4, 2, 15, device=DEV)
        call(odd, odd, wq[:15], wk[:15])
    with pytest.raises(RuntimeError, match="GPU only"):
        call(q, k.cpu(), wq, wk)
