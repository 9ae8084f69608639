"""The optimizer of orthogonalised momenta, the temporal encoder with relative positions, and both in training steps."""
import copy
import math

import pytest
import torch

import hivt_gan_amd as hv
from hivt_gan_amd import ops
from hivt_gan_amd.graph import GraphedStep
from hivt_gan_amd.optim import FusedAdamW, Muon

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def parameters(seed=0):
    gen = torch.Generator().manual_seed(seed)
    shapes = [(64, 64), (256, 64), (64, 256), (20, 130), (128, 17), (130, 140)]
    mats = [torch.nn.Parameter((torch.randn(*s, generator=gen) * 0.1).to(DEV)) for s in shapes]
    rest = [torch.nn.Parameter(torch.randn(*s, generator=gen).to(DEV)) for s in ((64,), (3, 5, 7), (9, 2))]
    return mats, rest


def gradients(params, step):
    gen = torch.Generator().manual_seed(100 + step)
    for p in params:
        p.grad = (torch.randn(*p.shape, generator=gen) * 1e-2).to(DEV)


def orthogonal64(x, steps=5, eps=1e-7):
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        g = x @ x.t()
        x = 3.4445 * x + (-4.7750 * g + 2.0315 * (g @ g)) @ x
    return x.t() if flip else x


@pytest.mark.parametrize("nesterov", [True, False])
def test_steps_against_the_formula(nesterov):
    """Matrices against the formula in 64 bits, the rest bit for bit against FusedAdamW.  A direction is off by at most
    1e-4 of its 2-norm relative to the formula's (fp32 momenta, and 3e-5 of the iteration, see its own test), each step adds
    lr scale of that, and rounding adds 2^-22 |p|."""
    mats, rest = parameters()
    twin_mats, twin_rest = parameters()
    opt = Muon(mats, rest, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adam_lr=1e-2, adam_weight_decay=0.01)
    adam = FusedAdamW(twin_rest, lr=1e-2, weight_decay=0.01)
    want = [p.detach().cpu().double() for p in twin_mats]
    buffers = [torch.zeros_like(w) for w in want]
    slack = [0.0] * len(want)
    for step in range(4):
        gradients(mats + rest, step)
        for a, b in zip(rest, twin_rest):
            b.grad = a.grad.clone()
        for i, p in enumerate(mats):
            g = p.grad.cpu().double()
            buffers[i] = 0.9 * buffers[i] + g
            o = orthogonal64(g + 0.9 * buffers[i] if nesterov else buffers[i])
            scale = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            want[i] = want[i] * (1 - 0.05 * 0.1) - 0.05 * scale * o
            slack[i] += 0.05 * scale * 1e-4 * float(o.norm()) + 2.0 ** -22 * float(want[i].norm())
        opt.step()
        adam.step()
    for p, w, s in zip(mats, want, slack):
        assert float((p.detach().cpu().double() - w).norm()) <= s
    for a, b in zip(rest, twin_rest):
        assert torch.equal(a, b)


def test_found_inf_missing_gradients_and_state():
    mats, rest = parameters()
    opt = Muon(mats, rest)
    gradients(mats + rest, 0)
    mats[1].grad = None
    opt.step()
    assert "momentum_buffer" not in opt.state[mats[1]]
    before = [p.detach().clone() for p in mats + rest] + [opt.state[mats[0]]["momentum_buffer"].clone()]
    gradients(mats + rest, 1)
    for p in mats:
        p.grad.fill_(float("nan"))
    opt.found_inf = torch.ones((), device=DEV)
    opt.step()
    after = [p.detach() for p in mats + rest] + [opt.state[mats[0]]["momentum_buffer"]]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert float(opt.state[mats[1]]["momentum_buffer"].abs().max()) == 0.0
    # a restored optimizer takes the same step
    opt.found_inf = torch.zeros((), device=DEV)
    saved, values = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in mats + rest]
    gradients(mats + rest, 2)
    opt.step()
    first = [p.detach().clone() for p in mats + rest]
    with torch.no_grad():
        for p, v in zip(mats + rest, values):
            p.copy_(v)
    other = Muon(mats, rest)
    other.load_state_dict(saved)
    gradients(mats + rest, 2)
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(first, [p.detach() for p in mats + rest]))
    sched = torch.optim.lr_scheduler.CosineAnnealingLR(other, T_max=4)
    sched.step()
    assert other.param_groups[-1]["lr"] != 0.02 and other.param_groups[-1]["orthogonal"]


def test_refusals():
    mats, rest = parameters()
    for bad in ([], [rest[0]], [torch.nn.Parameter(torch.zeros(4, 4))], [torch.nn.Parameter(mats[0].detach().half())]):
        with pytest.raises(ValueError):
            Muon(bad, rest)
    for kw in (dict(momentum=1.0), dict(steps=0), dict(eps=0.0)):
        with pytest.raises(ValueError):
            Muon(mats, rest, **kw)
    opt = Muon(mats, rest)
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4, device=DEV))]))
    with pytest.raises(ValueError):
        hv.HiVT(embed_dim=16, num_heads=2, optimizer="sgd")


@pytest.mark.parametrize("steps,dim,heads", [(20, 64, 8), (40, 128, 8), (75, 32, 2), (1, 16, 2)])
def test_relative_temporal_encoder(steps, dim, heads):
    """The whole encoder (norm and rotation, biased attention, single query in the last layer) and every gradient against
    the same module in float64 on the CPU.  Bound 2e-5 of each tensor's norm: the fp32 dense layers around it are held to
    1e-5 by their own tests, and gradients pass two such layers."""
    torch.manual_seed(3)
    ref = hv.TemporalEncoder(steps, dim, heads, num_layers=2, dropout=0.0, relative_positions=True)
    with torch.no_grad():
        for layer in ref.transformer_encoder.layers:
            layer.relative_bias.normal_()
            layer.q_norm.normal_(1.0, 0.2)
            layer.k_norm.normal_(1.0, 0.2)
    got = copy.deepcopy(ref).to(DEV)
    ref = ref.double()
    x = torch.randn(steps, 9, dim)
    mask = torch.rand(9, steps) < 0.3
    grad = torch.randn(9, dim)
    xa = x.double().requires_grad_(True)
    xb = x.to(DEV).requires_grad_(True)
    a = ref(xa, mask)
    b = got(xb, mask.to(DEV))
    a.backward(grad.double())
    b.backward(grad.to(DEV))

    def near(name, u, v):
        assert float((u.cpu().double() - v).norm()) <= 2e-5 * float(v.norm()) + 1e-12, name

    near("out", b.detach(), a.detach())
    near("dx", xb.grad, xa.grad)
    for (name, p), (_, q) in zip(got.named_parameters(), ref.named_parameters()):
        if name.endswith("in_proj_bias"):  # (the keys' third is zero but for rounding)
            d = dim
            near(name, torch.cat((p.grad[:d], p.grad[2 * d:])), torch.cat((q.grad[:d], q.grad[2 * d:])))
        elif q.grad is not None and float(q.grad.norm()) > 1e-9:
            near(name, p.grad, q.grad)


def model_of(seed=11, **kw):
    torch.manual_seed(seed)
    m = hv.HiVT(embed_dim=64, num_heads=8, dropout=0.0, use_gan=True, num_temporal_layers=2, num_global_layers=2,
                relative_positions=True, optimizer="muon", muon_lr=0.01, **kw).to(DEV)
    m.train()
    for critic in m.critics.values():
        for mod in critic.modules():
            if isinstance(mod, torch.nn.Dropout):
                mod.p = 0.0
    return m


def test_training_steps_recorded_and_eager():
    """A step with relative positions and Muon, launched and recorded, with a change of the learning rate between: equal
    parameters."""
    raw = [hv.make_batch(5, first_index=400 + 10 * i).to(DEV) for i in range(2)]
    eager, recorded = model_of(), model_of()
    spec = hv.GanTrainer.calibrate(eager, raw)
    padded = [hv.pad_batch(b, spec) for b in raw]
    trainer = hv.GanTrainer(eager, distributed=False, edge_capacity=spec.edge_capacity)
    other = hv.GanTrainer(recorded, distributed=False, edge_capacity=spec.edge_capacity)
    assert isinstance(trainer.opt_g, Muon)
    start = {k: v.clone() for k, v in recorded.state_dict().items()}
    step = GraphedStep(other, spec, padded[0], warmup=2)
    assert step.nodes.get("memset", 0) == 0
    assert all(torch.equal(v, start[k]) for k, v in recorded.state_dict().items())
    for i in (0, 1, 0):
        trainer.step(padded[i].clone())
        logs = step.run(padded[i])
        torch.cuda.synchronize()
        assert float(logs["skipped"]) == 0.0
        for t in (trainer, other):
            t.opt_g.param_groups[-1]["lr"] *= 0.5
    for (k, a), (_, b) in zip(recorded.state_dict().items(), eager.state_dict().items()):
        assert torch.equal(a, b), k
    moved = recorded.state_dict()["local_encoder.temporal_encoder.transformer_encoder.layers.0.self_attn.in_proj_weight"]
    assert not torch.equal(moved, start["local_encoder.temporal_encoder.transformer_encoder.layers.0.self_attn.in_proj_weight"])
    assert all(bool(torch.isfinite(p).all()) for p in recorded.parameters())


def test_operators_in_a_row():
    """The operators as they are used together, on their own: rotated normalised heads, attention with the bias, the
    gradients' orthogonalised direction; against the formulas in float64."""
    gen = torch.Generator().manual_seed(9)
    B, S, H, G, d = 2, 90, 4, 2, 16
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    leaves = [r(H * d, 48) * 0.2, r(G * d, 48) * 0.2, r(G * d, 48) * 0.2, torch.ones(d), torch.ones(d), r(32, H)]
    x, do = r(B, S, 48), r(B, S, H, d)

    def run(leaves, x, do, own):
        wq, wk, wv, gq, gk, table = leaves
        q, k, v = ((x @ w.t()).view(B, S, -1, d) for w in (wq, wk, wv))
        if own:
            q, k = ops.qk_norm_rotary(q, k, gq, gk)
            o = ops.relative_attention(q, k, v, table, causal=True)
        else:
            angle = torch.arange(S).double()[:, None] * 10000.0 ** (-torch.arange(d // 2).double() / (d // 2))

            def turned(t, g):
                t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * g
                a, b = t[..., :d // 2], t[..., d // 2:]
                c, s = angle.cos()[:, None], angle.sin()[:, None]
                return torch.cat((a * c - b * s, a * s + b * c), -1)

            q, k = turned(q, gq), turned(k, gk)
            k, v = (t.repeat_interleave(H // G, dim=2) for t in (k, v))
            exact, borders = ops.relative_buckets(32, 128, False)
            dist = (torch.arange(S)[:, None] - torch.arange(S)[None])
            n = dist.clamp(min=0)
            bucket = torch.where(n < exact, n, exact + torch.bucketize(n, torch.tensor(borders), right=True))
            z = torch.einsum("bihd,bjhd->bhij", q, k) / d ** 0.5 + table[bucket].permute(2, 0, 1)
            o = torch.einsum("bhij,bjhd->bihd", torch.softmax(z.masked_fill(dist < 0, -math.inf), -1), v)
        return o, torch.autograd.grad(o, leaves, do)

    dev = [t.to(DEV).requires_grad_(True) for t in leaves]
    out, grads = run(dev, x.to(DEV), do.to(DEV), True)
    ref = [t.double().requires_grad_(True) for t in leaves]
    out64, grads64 = run(ref, x.double(), do.double(), False)
    assert float((out.detach().cpu().double() - out64.detach()).norm()) <= 1e-5 * float(out64.norm())
    for a, b in zip(grads, grads64):
        assert float((a.cpu().double() - b).norm()) <= 1e-5 * float(b.norm())
    for direction, g in zip(ops.orthogonalize(list(grads[:3])), grads[:3]):
        want = orthogonal64(g.cpu().double())
        assert float((direction.cpu().double() - want).norm()) <= 3e-5 * float(want.norm())


def test_a_graph_older_than_the_step_is_refused():
    w = torch.randn(8, 8, device=DEV, requires_grad=True)
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    opt = Muon([w])
    old = (x @ w).sum()
    w.grad = torch.randn(8, 8, device=DEV)
    opt.step()
    with pytest.raises(RuntimeError, match="inplace"):
        old.backward()
