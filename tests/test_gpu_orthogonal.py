"""Orthogonalised updates against the iteration in 64 bits.

Tolerance.  The iteration is a^5 = 485 times the identity on vanishing singular values.  Rounding every element of X_j
(X after j steps) by 2^-24 of itself changes it by at most 2^-24 |X_j| in the Frobenius norm, and what is left of the
iteration lifts that by at most a^(5 - j); |X_j| <= a^j |X_0| = a^j, so each such rounding is at most 485 * 2^-24 = 2.9e-5
in the result, absolutely.  There are at most 13 of them: one where the norm is divided out, and in each of at most three
phases the planes of X, the planes of the polynomial in front of it, and the sums of the product (fp32 sums of products:
counted twice).  Low rank and graded matrices are held to that, 3.8e-4 absolutely; it takes a matrix whose small singular
values hold rounding noise only to come near.  Matrices with singular values that differ by less than a few hundred are
lifted by that much less and are held to 3e-5 relative to the result, clearly rectangular Gaussian ones (a factor below
ten) to 3e-6.  16-bit results: u = eps / 2 of the type on
top, and phases of up to three steps: a rounding of the Gram matrix by 2^-24 of its largest eigenvalue moves the factor of
a vanishing singular value by its slope there, 1.4 (1 + a^2 + a^4) = 213 times that and, like every rounding above, is
lifted by the rest: 1e-4 covers it for the Gaussian ones."""
import pytest
import torch

from hivt_gan_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def exact(x, steps=5, eps=1e-7):
    x = x.detach().cpu().double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        g = x @ x.t()
        x = 3.4445 * x + (-4.7750 * g + 2.0315 * (g @ g)) @ x
    return x.t() if flip else x


LIFTED = 13 * 485 * 2.0 ** -24


def check(got, x, steps=5, eps=1e-7, tol=3e-6, absolute=0.0):
    assert got.shape == x.shape and got.dtype == x.dtype
    want = exact(x, steps, eps)
    err = (got.cpu().double() - want).norm()
    if x.dtype != torch.float32:
        tol = max(tol, 1e-4) + torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * x.numel() ** 0.5 if x.dtype == torch.float16 else 0.0
    assert float(err) <= tol * float(want.norm()) + tiny + absolute, f"{tuple(x.shape)}: {float(err / want.norm()):.2e}"


def gaussian(rows, cols, dtype=torch.float32, seed=0, scale=1e-3):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=gen) * scale).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 50), (50, 1), (2, 2), (3, 128), (64, 64), (65, 63), (128, 20), (60, 128),
                                       (130, 257), (512, 128), (128, 512), (200, 1000), (333, 334), (700, 100)])
def test_shapes(dtype, rows, cols):
    x = gaussian(rows, cols, dtype, scale=1.0)
    before = x.clone()
    # (square Gaussian matrices have singular values down to 1 / rows of the largest: the lifted error of the docstring)
    check(ops.orthogonalize([x])[0], x, tol=3e-6 if max(rows, cols) >= 1.5 * min(rows, cols) else 3e-5)
    assert torch.equal(x, before)


@pytest.mark.parametrize("dtype", TYPES)
def test_low_rank_and_graded(dtype):
    gen = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    cases = [r(128, 4) @ r(4, 200), r(128, 128) * torch.logspace(0, -4, 128)[:, None],
             r(100, 300) * torch.logspace(0, -3, 300)[None], torch.eye(70), torch.ones(90, 90),
             r(64, 3) @ r(3, 300)]
    cases = [x.to(dtype).to(DEV) for x in cases]
    for x, y in zip(cases, ops.orthogonalize(cases)):
        check(y, x, tol=0.0, absolute=LIFTED)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 9])
def test_steps(steps):
    for dtype in (torch.float32, torch.bfloat16):
        xs = [gaussian(96, 100, dtype), gaussian(300, 70, dtype)]
        for x, y in zip(xs, ops.orthogonalize(xs, steps=steps)):
            check(y, x, steps, tol=6e-5)  # (more steps than five lift more: 3.4445 times each, up to full size)


def test_norms_from_vanishing_to_huge():
    """|x| far below eps (the result is a^5 x / eps), about eps, and where its square leaves the range of fp32."""
    for scale in (0.0, 1e-30, 1e-20, 1e-12, 1e-9, 1e-8, 1e-7, 1e-3, 1e10, 1e25, 1e35):
        x = gaussian(40, 70, scale=scale)
        y = ops.orthogonalize([x])[0]
        if scale == 0.0:
            assert float(y.abs().max()) == 0.0
        else:
            check(y, x, tol=3e-5)
    x = gaussian(40, 70, scale=1e-3)
    check(ops.orthogonalize([x], eps=10.0)[0], x, eps=10.0, tol=3e-5)


def test_list_and_alone_give_equal_bits():
    shapes = [(128, 128)] * 40 + [(512, 128), (128, 512), (3, 128), (0, 5), (256, 60), (400, 400)] * 9
    xs = [gaussian(r, c, seed=i) for i, (r, c) in enumerate(shapes)]
    ys = ops.orthogonalize(xs)
    for i in (0, 39, 40, 41, 42, 43, 44, 45, 93):
        assert torch.equal(ys[i], ops.orthogonalize([xs[i]])[0])
        if xs[i].numel():
            check(ys[i], xs[i], tol=3e-5)
    again = ops.orthogonalize(xs)
    assert all(torch.equal(a, b) for a, b in zip(ys, again))


def test_strides_in_place_and_not_finite():
    x = gaussian(100, 60)
    want = ops.orthogonalize([x])[0]
    assert torch.equal(ops.orthogonalize([x.t().contiguous().t()])[0], want)
    spaced = torch.empty(100, 64, device=DEV)[:, 1:61]
    spaced.copy_(x)
    assert torch.equal(ops.orthogonalize([spaced])[0], want)
    y = x.clone()
    assert ops.orthogonalize([y], out=[y])[0] is y and torch.equal(y, want)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z[3, 4] = bad
        a, b = ops.orthogonalize([z, x])
        assert not bool(torch.isfinite(a).any()) and torch.equal(b, want)


def test_larger_matrices():
    for dtype, rows, cols in ((torch.float32, 1500, 1100), (torch.bfloat16, 1024, 2500)):
        x = gaussian(rows, cols, dtype)
        check(ops.orthogonalize([x])[0], x, tol=1e-5)


def test_captured_and_replayed():
    groups = [[gaussian(128, 130, seed=1), gaussian(300, 60, seed=2)], [gaussian(200, 200, seed=3)]]
    graphs = []
    for xs in groups:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.orthogonalize(xs)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.orthogonalize(xs)
        graphs.append((graph, xs, got))
    for _ in range(3):
        for graph, xs, got in graphs:
            for x in xs:
                x.mul_(0.9).add_(1e-4)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip([t.clone() for t in got], ops.orthogonalize(xs)))


def test_refusals():
    x = gaussian(8, 8)
    assert ops.orthogonalize([]) == []
    with pytest.raises(TypeError):
        ops.orthogonalize([x.double()])
    with pytest.raises(TypeError):
        ops.orthogonalize([x, x.half()])
    with pytest.raises(ValueError):
        ops.orthogonalize([x[None]])
    for steps in (0, 17):
        with pytest.raises(ValueError):
            ops.orthogonalize([x], steps=steps)
    with pytest.raises(ValueError):
        ops.orthogonalize([x], eps=0.0)
    with pytest.raises(ValueError):
        ops.orthogonalize([x], out=[x.t()[:4]])
    with pytest.raises(ValueError):
        ops.orthogonalize([x], out=[])
    with pytest.raises(ops.UnsupportedShapeError):
        ops.orthogonalize([torch.zeros(1, 65537, device=DEV)])
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.orthogonalize([x.cpu()])


def test_outputs_that_share_memory():
    store = torch.randn(12, 70, device=DEV)
    a, b, c = store[:4], store[4:8], store[8:]
    want = ops.orthogonalize([a, b])
    for ins, outs in (([a, b], [b, a]), ([a, b], [c, c]), ([a, b], [c, a]), ([a], [store[1:5]])):
        with pytest.raises(ValueError, match="shares memory"):
            ops.orthogonalize(ins, out=outs)
    version = store._version
    got = ops.orthogonalize([a, b], out=[a, c])
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(a, want[0])
    assert store._version > version


def test_tiles_left_for_a_last_turn():
    """32 lists of 128-row tiles: 528 of them on and below the diagonal, and 12 x 45 of a product with X."""
    for rows, cols in ((4000, 4100), (1500, 5700)):
        x = gaussian(rows, cols)
        check(ops.orthogonalize([x], steps=2)[0], x, steps=2, tol=1e-5)


def test_tiles_left_in_16_bits_and_in_lists():
    x = gaussian(4000, 4100, torch.bfloat16)
    check(ops.orthogonalize([x], steps=1)[0], x, steps=1)
    xs = [gaussian(900, 1000, torch.float16, seed=i, scale=1.0) for i in range(15)]  # 540 tiles, the last 28 in quarters
    ys = ops.orthogonalize(xs, steps=2)
    for i in (0, 13, 14):
        check(ys[i], xs[i], steps=2)
