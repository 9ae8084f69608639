"""What is measured of the relative-position attention, the query / key normalisation with rotation and the
orthogonalised update: cases, inputs, the plain form in elementary torch operations and the definition in 64 bits.

Every case is a dict of plain values.  ``own`` chooses between the plain form and the library's operators."""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NS = (3.4445, -4.7750, 2.0315)  # the quintic of the orthogonalised update


def _attention(name, dtype, batch, q_len, k_len, heads, kv_heads, dim, causal, masked, train, buckets=32, distance=128):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "q_len": q_len, "k_len": k_len,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal, "masked": masked, "train": train,
            "buckets": buckets, "distance": distance}


def _rotary(name, dtype, batch, length, heads, kv_heads, dim, rotary, interleaved, start, train):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": interleaved, "start": start, "train": train}


def _orthogonal(name, dtype, shapes):
    return {"name": name, "op": "orthogonal", "dtype": dtype, "shapes": shapes}


def listed():
    return [
        # the class token of one scene's agents looks back over its history: latency alone
        _attention("token_scene", "fp32", 20, 1, 21, 8, 8, 16, True, False, False),
        # the temporal encoder of a 128-scene batch: 20 history steps and a class token for every agent
        _attention("history_train", "fp32", 2560, 21, 21, 8, 8, 16, True, False, True),
        # histories of 30 s at 10 Hz, agents unseen at the start (and some never seen) masked
        _attention("long_history_train", "fp32", 64, 301, 301, 8, 8, 16, False, True, True, 32, 64),
        # encoder layer of a language model over padded sequences
        _attention("encoder_train", "bf16", 8, 1024, 1024, 16, 16, 64, False, True, True),
        # decoder layer over long sequences, four query heads to a key head
        _attention("decoder_train", "bf16", 2, 4096, 4096, 16, 4, 128, True, False, True),
        # one new token a sequence against a long context
        _attention("token_long", "bf16", 8, 1, 30001, 32, 8, 128, True, False, False),
        # a chunk of new tokens behind an odd context, padded batch, odd head width
        _attention("chunk_odd", "fp16", 3, 333, 2011, 6, 2, 80, True, True, False),
        # queries and keys of the temporal encoder, 128 scenes
        _rotary("history_rotary_train", "fp32", 2560, 21, 8, 8, 16, 16, False, 0, True),
        # queries and keys of a decoder layer, far positions
        _rotary("decoder_rotary_train", "bf16", 4, 4096, 32, 8, 128, 128, False, 100000, True),
        # the hidden matrices of the 128-wide model (its equal square projections counted to 36)
        _orthogonal("model_update", "fp32", "128x128*36,512x128*9,128x512*9,384x128*4,60x128*1,128x20*1,256x60*1,3x128*1"),
        # a feed-forward matrix of a small language model
        _orthogonal("feed_forward_update", "bf16", "1024x4096*1"),
        # a square projection of a large one
        _orthogonal("square_update", "fp32", "4096x4096*1"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "orthogonal"])
    if op == "attention":
        train = rng.random() < 0.6
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        dim = rng.choice([4, 8, 12, 16, 20, 32, 40, 48, 64, 80, 96, 112, 128])
        causal = rng.random() < 0.5
        # (with a single key the gradients of queries, keys and biases are zero but for rounding: nothing to compare)
        k_len = _log_int(rng, 8, 4096) if train else _log_int(rng, 1, 32768)
        q_len = 1 if not train and rng.random() < 0.4 else k_len if rng.random() < 0.6 else _log_int(rng, 1, k_len)
        q_len = min(q_len, 4096)
        # at most 2e8 scores, 6e7 rows of a head
        most = max(1, int(min(2e8 / (heads * q_len * k_len), 6e7 / (kv_heads * k_len * dim))))
        if q_len * k_len * heads > 2e8:
            q_len = max(1, int(2e8 / (k_len * heads)))
        batch = _log_int(rng, 1, min(most, 2048))
        half = rng.choice([4, 8, 16])
        return _attention("", rng.choice(["fp32", "bf16", "fp16"]), batch, q_len, k_len, heads, kv_heads, dim, causal,
                          rng.random() < 0.5, train, 2 * half, half * _log_int(rng, 2, 32))
    if op == "rotary":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        dim = rng.choice([8, 16, 20, 32, 64, 80, 96, 128, 256])
        length = _log_int(rng, 1, 8192)
        most = max(1, int(8e7 / ((heads + kv_heads) * dim * length)))
        batch = _log_int(rng, 1, min(most, 4096))
        rotary = dim if rng.random() < 0.6 else 2 * rng.randint(0, dim // 2)
        return _rotary("", rng.choice(["fp32", "bf16", "fp16"]), batch, length, heads, kv_heads, dim, rotary,
                       rng.random() < 0.3, rng.choice([0, 0, 17, 131071, 1000000]), rng.random() < 0.6)
    shapes = []
    for _ in range(rng.randint(1, 4)):
        rows, cols = _log_int(rng, 1, 2048), _log_int(rng, 1, 4096)
        small = min(rows, cols)
        most = max(1, int(2e10 / (small * rows * cols)))
        shapes.append("%dx%d*%d" % (rows, cols, _log_int(rng, 1, min(most, 15))))
    return _orthogonal("", rng.choice(["fp32", "bf16"]), ",".join(shapes))


def _shapes(case):
    return [(int(r), int(c), int(k)) for r, c, k in
            (p.replace("*", "x").split("x") for p in case["shapes"].split(","))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(t)

    s = dict(case)
    if case["op"] == "attention":
        B, M, N, H, G, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))
        s["q"], s["k"], s["v"] = normal(B, M, H, d), normal(B, N, G, d), normal(B, N, G, d)
        s["table"] = torch.randn(case["buckets"], H, generator=gen, device="cuda")
        s["mask"] = None
        if case["masked"]:  # True: the key is left out.  Every sequence ends somewhere; some begin late, one in sixteen has no key
            ends = torch.randint(0, N + 1, (B, 1), generator=gen, device="cuda").clamp(min=(N + 1) // 2)
            begins = torch.randint(0, max(1, N // 4), (B, 1), generator=gen, device="cuda")
            at = torch.arange(N, device="cuda")
            s["mask"] = (at >= ends) | (at < begins) | (torch.rand(B, 1, generator=gen, device="cuda") < 1 / 16)
        if case["train"]:
            s["d_out"] = normal(B, M, H, d)
            for key in ("q", "k", "v", "table"):
                s[key].requires_grad_(True)
    elif case["op"] == "rotary":
        B, S, H, G, d = (case[k] for k in ("batch", "length", "heads", "kv_heads", "dim"))
        s["q"], s["k"] = normal(B, S, H, d, scale=2.0), normal(B, S, G, d, scale=2.0)
        s["wq"] = 1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda")
        s["wk"] = 1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda")
        s["positions"] = torch.arange(case["start"], case["start"] + S, device="cuda")
        if case["train"]:
            s["dq"], s["dk"] = normal(B, S, H, d), normal(B, S, G, d)
            for key in ("q", "k", "wq", "wk"):
                s[key].requires_grad_(True)
    else:
        # momenta of gradients: a few strong directions over noise, of the size that gradients have
        s["updates"] = []
        for rows, cols, count in _shapes(case):
            for _ in range(count):
                rank = max(1, min(rows, cols) // 16)
                low = torch.randn(rows, rank, generator=gen, device="cuda") @ torch.randn(rank, cols, generator=gen, device="cuda")
                s["updates"].append(((low / math.sqrt(rank) + torch.randn(rows, cols, generator=gen, device="cuda")) * 1e-3).to(t))
    return s


# ---- attention with a learned bias for each bucket of relative positions ---------------------------------------------
def _bucket_starts(buckets, distance, bidirectional):
    """Distances at which the buckets behind the single ones start: the least n with
    n >= exact * (distance / exact) ** (t / L), decided in whole numbers."""
    side = buckets // 2 if bidirectional else buckets
    exact_, starts = side // 2, []
    spans = side - exact_
    for t in range(1, spans):
        n = exact_
        while n ** spans < exact_ ** (spans - t) * distance ** t:
            n += 1
        starts.append(n)
    return side, exact_, starts


def _buckets(case, device):
    """Bucket of every key position - query position from -(N - 1) to M - 1, in that order."""
    M, N = case["q_len"], case["k_len"]
    bidirectional = not case["causal"]
    side, exact_, starts = _bucket_starts(case["buckets"], case["distance"], bidirectional)
    rel = torch.arange(-(N - 1), M, device=device)  # the queries stand at the end of the keys
    dist = rel.abs() if bidirectional else (-rel).clamp(min=0)
    far = exact_ + torch.searchsorted(torch.tensor(starts, device=device, dtype=torch.long), dist, right=True)
    bucket = torch.where(dist < exact_, dist, far)
    return bucket + side * (rel > 0) if bidirectional else bucket


def _allowed(s):
    M, N = s["q_len"], s["k_len"]
    rel = torch.arange(N, device="cuda")[None, :] - (torch.arange(M, device="cuda") + N - M)[:, None]
    ok = (rel <= 0) if s["causal"] else torch.ones_like(rel, dtype=torch.bool)
    return (ok if s["mask"] is None else ok & ~s["mask"][:, None, None, :]), rel + (N - 1)


def _attention_plain(s):
    B, M, N, H, G, d = (s[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))
    t = s["q"].dtype
    scale = d ** -0.5
    ok, at = _allowed(s)
    bucket = _buckets(s, "cuda")
    q = s["q"].detach().float().transpose(1, 2)                                  # [B, H, M, d]
    k, v = (s[x].detach().float().transpose(1, 2).repeat_interleave(H // G, dim=1) for x in ("k", "v"))
    bias = s["table"].detach()[bucket].t().contiguous()[:, at]                   # [H, M, N]
    p = (q @ k.transpose(2, 3)).mul_(scale).add_(bias).masked_fill_(~ok, float("-inf"))
    del bias
    top = p.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = p.sub_(top).exp_()
    p = p.div_(p.sum(dim=-1, keepdim=True).clamp(min=1e-30))
    out = p @ v                                                                  # [B, H, M, d]
    if not s["train"]:
        return out.transpose(1, 2).to(t)
    do = s["d_out"].float().transpose(1, 2)
    dv = (p.transpose(2, 3) @ do).view(B, G, H // G, N, d).sum(dim=2)
    # (each row of ds sums to nothing, and the bias gradient may hold little but what is left of that: in 64 bits)
    ds = do @ v.transpose(2, 3)
    ds = ds.sub_((p * ds).sum(dim=-1, keepdim=True, dtype=torch.float64).float()).mul_(p)
    del p
    dq = (ds @ k) * scale
    dk = (ds.transpose(2, 3) @ q).view(B, G, H // G, N, d).sum(dim=2) * scale
    # the bias gradient: sums along the diagonals, then over the buckets.  With the rows in reverse and one column
    # less in the view than in memory, a diagonal stands in a column: column c holds key - row = c - (M - 1)
    by_pair = ds.sum(dim=0).flip(1)                                              # [H, M, N]
    del ds
    wide = torch.cat((by_pair, by_pair.new_zeros(H, M, M)), dim=2).view(H, -1)[:, :M * (N + M - 1)]
    diagonal = wide.view(H, M, N + M - 1).sum(dim=1, dtype=torch.float64)
    rel = torch.arange(-(M - 1), N, device="cuda") - (N - M)
    member = (bucket[rel + N - 1][:, None] == torch.arange(s["buckets"], device="cuda")).double()
    d_table = (diagonal @ member).t()
    back = lambda x: x.transpose(1, 2).to(t)  # noqa: E731
    return back(out), back(dq), back(dk), back(dv), d_table.float()


def _attention_own(s):
    from hivt_gan_amd import ops
    out = ops.relative_attention(s["q"], s["k"], s["v"], s["table"], causal=s["causal"], max_distance=s["distance"],
                                 key_mask=s["mask"])
    if not s["train"]:
        return out
    return (out,) + torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["table"]), s["d_out"])


def _attention_exact(s):
    B, M, N, H, G, d = (s[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))
    f8 = torch.float64
    # the bucket of a distance counted from the definition: how many of its whole steps of the logarithm it has passed
    side = s["buckets"] if s["causal"] else s["buckets"] // 2
    near = side // 2
    steps = side - near

    def of(r):
        n = max(-r, 0) if s["causal"] else abs(r)
        b = n
        if n >= near:
            passed = 0
            while passed < steps - 1 and n ** steps >= near ** (steps - passed - 1) * s["distance"] ** (passed + 1):
                passed += 1
            b = near + passed
        return b + (side if r > 0 and not s["causal"] else 0)

    lo, hi = -(N - 1), M - 1
    edge = s["distance"] + 1
    lut = [of(max(-edge, min(edge, r))) for r in range(lo, hi + 1)]
    bucket = torch.tensor(lut, device="cuda")
    keep, at = _allowed(s)
    keep = keep.expand(B, 1, M, N)[:, 0] if keep.dim() == 4 else keep.expand(B, M, N)
    table = s["table"].detach().to(f8)
    out = torch.zeros(B, M, H, d, dtype=f8, device="cuda")
    dq, dk, dv = torch.zeros_like(out), out.new_zeros(B, N, G, d), out.new_zeros(B, N, G, d)
    d_table = torch.zeros(s["buckets"], H, dtype=f8, device="cuda")
    diag = bucket[at]
    one = max(1, int(3e7 // (M * N)))
    for h in range(H):
        g = h // (H // G)
        pair = table[:, h][diag]
        ds_sum = torch.zeros(M, N, dtype=f8, device="cuda")
        for b in range(0, B, one):
            e = min(B, b + one)
            q, k, v = s["q"][b:e, :, h].detach().to(f8), s["k"][b:e, :, g].detach().to(f8), s["v"][b:e, :, g].detach().to(f8)
            z = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d) + pair
            w = torch.where(keep[b:e], z, torch.full_like(z, -1e300))
            w = torch.where(keep[b:e], torch.exp(w - w.max(dim=2, keepdim=True).values), torch.zeros_like(w))
            total = w.sum(dim=2, keepdim=True)
            w = w / torch.where(total > 0, total, torch.ones_like(total))
            out[b:e, :, h] = w @ v
            if s["train"]:
                o = s["d_out"][b:e, :, h].to(f8)
                dw = o @ v.transpose(1, 2).contiguous()
                dz = w * (dw - (w * dw).sum(dim=2, keepdim=True))
                dq[b:e, :, h] = dz @ k / math.sqrt(d)
                dk[b:e, :, g] += dz.transpose(1, 2).contiguous() @ q / math.sqrt(d)
                dv[b:e, :, g] += w.transpose(1, 2).contiguous() @ o
                ds_sum += dz.sum(dim=0)
        if s["train"]:
            for n in sorted(set(lut)):
                d_table[n, h] = ds_sum[diag == n].sum()
    return (out, dq, dk, dv, d_table) if s["train"] else out


# ---- norm of queries and keys for each head, and their rotation --------------------------------------------------------
def _turn(x, cos, sin, rotary, interleaved):
    head, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = head[..., :rotary // 2], head[..., rotary // 2:]
        head = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((head, rest), dim=-1)


def _angles(s):
    rate = 10000.0 ** (-2.0 * torch.arange(s["rotary"] // 2, device="cuda", dtype=torch.float64) / max(1, s["rotary"]))
    return (s["positions"].double()[:, None] * rate)[None, :, None, :]


def _rotary_plain(s):
    angle = _angles(s)
    cos, sin = angle.cos().float(), angle.sin().float()
    answer = []
    for x, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")):
        v, g = s[x].detach().float(), s[w].detach()
        inv = (v.square().mean(dim=-1, keepdim=True) + 1e-6).rsqrt()
        unit = v * inv
        answer.append(_turn(unit * g, cos, sin, s["rotary"], s["interleaved"]).to(s[x].dtype))
        if s["train"]:
            back = _turn(s[dy].float(), cos, -sin, s["rotary"], s["interleaved"])
            d_unit = back * g
            answer.append(((d_unit - unit * (d_unit * unit).mean(dim=-1, keepdim=True)) * inv).to(s[x].dtype))
            answer.append((back * unit).flatten(0, 2).sum(dim=0, dtype=torch.float64).float())
    return tuple(answer)


def _rotary_own(s):
    from hivt_gan_amd import ops
    q, k = ops.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], positions=s["positions"], rotary_dim=s["rotary"],
                              interleaved=s["interleaved"])
    if not s["train"]:
        return q, k
    dq, dwq, dk, dwk = torch.autograd.grad((q, k), (s["q"], s["wq"], s["k"], s["wk"]), (s["dq"], s["dk"]))
    return q, dq, dwq, k, dk, dwk


def _rotary_exact(s):
    R, f8 = s["rotary"], torch.float64
    turns = torch.exp(-math.log(10000.0) * torch.arange(0, R, 2, device="cuda", dtype=f8) / max(1, R))
    phase = torch.outer(s["positions"].to(f8), turns)
    phase = torch.polar(torch.ones_like(phase), phase)[None, :, None, :]

    def rotate(x, z):
        if R == 0:
            return x
        first = x[..., 0:R:2] if s["interleaved"] else x[..., :R // 2]
        second = x[..., 1:R:2] if s["interleaved"] else x[..., R // 2:R]
        c = torch.complex(first.contiguous(), second.contiguous()) * z
        y = x.clone()
        if s["interleaved"]:
            y[..., 0:R:2], y[..., 1:R:2] = c.real, c.imag
        else:
            y[..., :R // 2], y[..., R // 2:R] = c.real, c.imag
        return y

    answer = []
    for x, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")):
        v, g = s[x].detach().to(f8), s[w].detach().to(f8)
        r = 1.0 / torch.sqrt((v * v).sum(dim=-1, keepdim=True) / s["dim"] + 1e-6)
        answer.append(rotate(v * r * g, phase))
        if s["train"]:
            back = rotate(s[dy].to(f8), phase.conj().resolve_conj())
            answer.append(r * back * g - r ** 3 * v * (back * g * v).sum(dim=-1, keepdim=True) / s["dim"])
            answer.append((back * v * r).sum(dim=(0, 1, 2)))
    return tuple(answer)


# ---- orthogonalised update ------------------------------------------------------------------------------------------------
def _iterate(x):
    """x: [count, rows, cols], rows <= cols, any float type."""
    a, b, c = NS
    x = x / (torch.sqrt(x.square().sum(dim=(1, 2), keepdim=True)) + 1e-7)
    for _ in range(5):
        g = x @ x.transpose(1, 2)
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def _orthogonal_plain(s):
    answer, at = [], 0
    for rows, cols, count in _shapes(s):  # equal shapes as one batch
        x = torch.stack(s["updates"][at:at + count]).float()
        y = _iterate(x) if rows <= cols else _iterate(x.transpose(1, 2).contiguous()).transpose(1, 2)
        answer += [u.contiguous() for u in y.to(s["updates"][at].dtype).unbind(0)]
        at += count
    return answer


def _orthogonal_own(s):
    from hivt_gan_amd import ops
    return ops.orthogonalize(s["updates"])


def _orthogonal_exact(s):
    # one matrix at a time, the polynomial of the Gram matrix formed whole before it is applied
    a, b, c = NS
    answer = []
    for u in s["updates"]:
        x = u.double()
        flip = x.shape[0] > x.shape[1]
        x = (x.t() if flip else x).contiguous()
        x = x / (x.norm() + 1e-7)
        for _ in range(5):
            g = x @ x.t().contiguous()
            p = g @ g
            p.mul_(c).add_(g, alpha=b).diagonal().add_(a)
            x = p @ x
        answer.append((x.t() if flip else x).contiguous())
    return answer


def run(state):
    with torch.set_grad_enabled(own and bool(state.get("train"))):
        if state["op"] == "attention":
            return _attention_own(state) if own else _attention_plain(state)
        if state["op"] == "rotary":
            return _rotary_own(state) if own else _rotary_plain(state)
        return _orthogonal_own(state) if own else _orthogonal_plain(state)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attention":
            return _attention_exact(state)
        if case["op"] == "rotary":
            return _rotary_exact(state)
        return _orthogonal_exact(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        B, M, N, H, G, d = (case[k] for k in ("batch", "q_len", "k_len", "heads", "kv_heads", "dim"))
        pairs = M * N - (M * (M - 1) // 2 if case["causal"] else 0)
        rows = B * d * (2 * M * H + 2 * N * G)
        products = 2
        if case["train"]:
            rows += B * d * (2 * M * H + 2 * N * G)  # d_out read; dq, dk, dv written
            products = 7
        return {"bytes": rows * size + case["buckets"] * H * 4 + (B * N if case["masked"] else 0),
                "flops": 2.0 * products * B * H * pairs * d}
    if case["op"] == "rotary":
        rows = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"])
        moved = 5 if case["train"] else 2  # x, y; and dy, x again, dx
        return {"bytes": rows * case["dim"] * moved * size, "flops": rows * case["dim"] * (20.0 if case["train"] else 7.0)}
    nbytes, flops = 0.0, 0.0
    for rows, cols, count in _shapes(case):
        m, n = float(min(rows, cols)), float(max(rows, cols))
        nbytes += count * 2.0 * m * n * size
        # symmetric products at half: five times (x x', g g, p x), or the polynomials carried on the small side
        flops += count * min(5 * (3 * m * m * n + m ** 3), 3 * m * m * n + 17 * m ** 3)
    return {"bytes": nbytes, "flops": flops}
