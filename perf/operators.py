"""Operators between the sharded projections of an attention block, as a program calls them on one worker's heads: the
positions' rotation of queries and keys, their norms for each head with the rotation in the same pass, and attention to keys
of another length than the queries' (an encoder's states, a cache, the sequence itself).

Queries and keys are [batch, tokens, heads, head_dim], as a projection's output is viewed; where they come out of one
projection they are strided views of it.  A case names an operator, its sizes, element type and direction.  ``run`` computes
it in plain torch operations, or calls the framework's operators where ``own`` is true.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def listed():
    return [
        # One token for each of sixteen sequences, far apart in their positions, one worker's heads of eight: what a
        # decode step rotates.  Latency.
        {"name": "rotary_decode", "op": "rotary", "dtype": "bf16", "batch": 16, "tokens": 1, "heads": 8, "kv_heads": 1, "dim": 128,
         "rotated": 128, "interleaved": False, "reach": 1000000, "amplitude": 1.0, "train": False},
        # Training step on the repository's sequences (4 x 2048 tokens of 8192 features, 64 heads), all heads on one worker.
        {"name": "rotary_train", "op": "rotary", "dtype": "bf16", "batch": 4, "tokens": 2048, "heads": 64, "kv_heads": 8, "dim": 128,
         "rotated": 128, "interleaved": True, "reach": 2048, "amplitude": 1.0, "train": True},
        # Training step in the layers' default type: 0.4 of a head of 80 rotates, an odd number of tokens, positions of a
        # long context with the amplitude that its scaling brings.
        {"name": "rotary_partial", "op": "rotary", "dtype": "f32", "batch": 2, "tokens": 1777, "heads": 20, "kv_heads": 20, "dim": 80,
         "rotated": 32, "interleaved": False, "reach": 131072, "amplitude": 1.25, "train": True},
        # The decode step again with the heads' norms.
        {"name": "head_norm_decode", "op": "head_norm", "dtype": "bf16", "batch": 16, "tokens": 1, "heads": 8, "kv_heads": 1, "dim": 128,
         "rotated": 128, "interleaved": False, "reach": 1000000, "amplitude": 1.0, "train": False},
        # The training step again with the heads' norms and their weights' gradients.
        {"name": "head_norm_train", "op": "head_norm", "dtype": "bf16", "batch": 4, "tokens": 2048, "heads": 64, "kv_heads": 8, "dim": 128,
         "rotated": 128, "interleaved": False, "reach": 2048, "amplitude": 1.0, "train": True},
        # Ragged: heads of 96 of which 64 rotate in neighbouring pairs, odd numbers of sequences and tokens.
        {"name": "head_norm_ragged", "op": "head_norm", "dtype": "f16", "batch": 3, "tokens": 1001, "heads": 12, "kv_heads": 4, "dim": 96,
         "rotated": 64, "interleaved": True, "reach": 8192, "amplitude": 1.0, "train": True},
        # A decoder's token for each of 32 sequences against the encoder's states, of which each sequence has its own number.
        {"name": "cross_decode", "op": "attention", "dtype": "bf16", "batch": 32, "tokens": 1, "keys": 1500, "heads": 16, "kv_heads": 16,
         "dim": 64, "ragged": True, "causal": False, "train": False},
        # One token against a long cache, one worker's heads with one key head: the keys' bytes are the cost.
        {"name": "decode_long", "op": "attention", "dtype": "bf16", "batch": 4, "tokens": 1, "keys": 65536, "heads": 8, "kv_heads": 1,
         "dim": 128, "ragged": True, "causal": False, "train": False},
        # Training step of a decoder's cross attention to padded encoder states.
        {"name": "cross_train", "op": "attention", "dtype": "bf16", "batch": 8, "tokens": 448, "keys": 1500, "heads": 16, "kv_heads": 16,
         "dim": 64, "ragged": True, "causal": False, "train": True},
        # Training step of self attention on the repository's sequences: one of eight workers' heads, one key head for all.
        {"name": "self_train", "op": "attention", "dtype": "bf16", "batch": 4, "tokens": 2048, "keys": 2048, "heads": 8, "kv_heads": 1,
         "dim": 128, "ragged": False, "causal": True, "train": True},
        # Prefill of one long sequence.
        {"name": "prefill_long", "op": "attention", "dtype": "f16", "batch": 1, "tokens": 8192, "keys": 8192, "heads": 8, "kv_heads": 2,
         "dim": 128, "ragged": False, "causal": True, "train": False},
        # Training step in the layers' default type, everything odd: heads of 40, 333 queries to at most 77 keys.
        {"name": "cross_train_f32", "op": "attention", "dtype": "f32", "batch": 3, "tokens": 333, "keys": 77, "heads": 8, "kv_heads": 8,
         "dim": 40, "ragged": True, "causal": False, "train": True},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "head_norm", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4, 5, 8])
    train = rng.random() < 0.6
    if op != "attention":
        dim = rng.choice([40, 64, 72, 80, 96, 100, 128, 128, 192, 256])
        rotated = rng.choice([dim, dim, dim // 2 // 2 * 2, 2 * rng.randint(1, dim // 2)])
        batch = _spread(rng, 1, 32)
        most = 4 * 2048 * 72 * 128 * 2 // (batch * (heads + kv) * dim * SIZE[dtype])
        tokens = _spread(rng, 1, max(1, min(16384, most)))
        return {"op": op, "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim, "rotated": rotated,
                "interleaved": rng.random() < 0.5, "reach": _spread(rng, tokens, 2000000), "amplitude": rng.choice([1.0, 1.0, 1.1]),
                "train": train}
    dim = rng.choice([40, 64, 64, 80, 96, 100, 128, 128, 128])
    mode = rng.choice(["cross", "cross", "self", "decode"])
    if mode == "decode":
        batch, tokens, train = _spread(rng, 1, 64), rng.choice([1, 1, 1, 2, 4]), False
        most = 2 ** 27 // (batch * 2 * kv * dim * SIZE[dtype])
        keys = _spread(rng, 16, max(16, min(65536, most)))
        causal = tokens > 1
    else:
        batch = _spread(rng, 1, 12)
        side = int(math.sqrt(2 ** (27 if train else 28) / (batch * heads * (2 if dtype == "f32" else 1))))
        tokens = _spread(rng, 1, max(1, min(4096, side)))
        keys = tokens if mode == "self" else _spread(rng, 1, max(1, min(4096, side)))
        causal = mode == "self"
    return {"op": op, "dtype": dtype, "batch": batch, "tokens": tokens, "keys": keys, "heads": heads, "kv_heads": kv, "dim": dim,
            "ragged": mode != "self" and rng.random() < 0.7, "causal": causal, "train": train}


def _lengths(case):
    """The sequences' numbers of keys, in some order: spread from a third of them to all, one sequence in eight without any."""
    n, b = case["keys"], case["batch"]
    return [0 if i % 8 == 7 else max(1, n - (2 * n // 3) * i // max(1, b - 1)) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    b, t, h, hk, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dt)

    train = case["train"]
    if case["op"] == "attention":
        # Heads after their projections (and norms): of order one, the queries somewhat larger.
        state = {"q": normal(b, t, h, d, scale=1.5), "k": normal(b, case["keys"], hk, d), "v": normal(b, case["keys"], hk, d),
                 "lengths": None, "causal": case["causal"]}
        if case["ragged"]:
            order = torch.randperm(b, generator=g, device="cuda")
            state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        leaves = ["q", "k", "v"]
        if train:
            state["dy"] = normal(b, t, h, d, scale=0.1)
    else:
        # Queries, keys and values come out of one projection; the first two are views of it.
        packed = normal(b, t, (h + 2 * hk) * d)
        start = torch.randint(0, max(1, case["reach"] - t + 1), (b, 1), generator=g, device="cuda")
        half = case["rotated"] // 2
        state = {"q": packed[..., :h * d].view(b, t, h, d), "k": packed[..., h * d:(h + hk) * d].view(b, t, hk, d),
                 "positions": start + torch.arange(t, device="cuda"),
                 "frequencies": 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half),
                 "interleaved": case["interleaved"], "amplitude": case["amplitude"]}
        leaves = ["q", "k"]
        if case["op"] == "head_norm":
            state["q_weight"], state["k_weight"] = (normal(d, scale=0.2) + 1).to(dt), (normal(d, scale=0.2) + 1).to(dt)
            leaves += ["q_weight", "k_weight"]
        if train:
            state["dq"], state["dk"] = normal(b, t, h, d, scale=0.1), normal(b, t, hk, d, scale=0.1)
    if train:
        for name in leaves:
            state[name] = state[name].detach().requires_grad_()
    state.update(op=case["op"], train=train, leaves=leaves)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from distdl_amd import nn
    if s["op"] == "attention":
        out = nn.attention_shard(s["q"], s["k"], s["v"], s["lengths"], causal=s["causal"])
        if not s["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, [s[n] for n in s["leaves"]], s["dy"])
    if s["op"] == "rotary":
        out = nn.rotary_shard(s["q"], s["k"], s["frequencies"], s["positions"], interleaved=s["interleaved"], amplitude=s["amplitude"])
    else:
        out = nn.head_norm_rotary_shard(s["q"], s["k"], s["q_weight"], s["k_weight"], s["frequencies"], s["positions"], eps=EPS,
                                        interleaved=s["interleaved"], amplitude=s["amplitude"])
    if not s["train"]:
        return out
    return tuple(o.detach() for o in out) + torch.autograd.grad(out, [s[n] for n in s["leaves"]], [s["dq"], s["dk"]])


def _run_plain(s):
    with torch.no_grad():
        if s["op"] == "attention":
            return _attention_plain(s)
        turn = _turn_plain(s)
        outs, grads, weight_grads = [], [], []
        for name in ("q", "k"):
            x, w = s[name], s.get(name + "_weight")
            x32 = x.float()
            if w is not None:
                rstd = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
                x32 = x32 * rstd
            outs.append(_rotated(x32 if w is None else x32 * w.float(), *turn, s["interleaved"]).to(x.dtype))
            if s["train"]:
                g = _rotated(s["d" + name].float(), turn[0], -turn[1], s["interleaved"])
                if w is not None:
                    weight_grads.append((g * x32).sum((0, 1, 2)).to(x.dtype))
                    g = g * w.float()
                    g = (g - x32 * (g * x32).mean(-1, keepdim=True)) * rstd
                grads.append(g.to(x.dtype))
        return tuple(outs + grads + weight_grads)


def _turn_plain(s):
    # Far positions need their angles in 64 bits.
    angle = s["positions"].double()[..., None] * s["frequencies"]
    return (torch.cos(angle) * s["amplitude"]).float()[:, :, None], (torch.sin(angle) * s["amplitude"]).float()[:, :, None]


def _rotated(x, cos, sin, interleaved):
    half = cos.shape[-1]
    if interleaved:
        first, second = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        first, second = x[..., :half], x[..., half:2 * half]
    a, b = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _attention_plain(s):
    q, k, v = s["q"], s["k"], s["v"]
    (b, t, h, d), n, hk = q.shape, k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d)

    # The queries of the heads that share a key head, below each other: [batch, key heads, heads each x tokens, head_dim].
    def rows(x):
        return x.float().view(b, t, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)

    def back(x, like):
        return x.view(b, hk, h // hk, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(like.dtype)

    q32, k32, v32 = rows(q), k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()
    key, at = torch.arange(n, device=q.device), torch.arange(t, device=q.device)
    seen = torch.ones(b, 1, t, n, dtype=torch.bool, device=q.device)
    if s["lengths"] is not None:
        seen = seen & (key < s["lengths"][:, None, None, None])
    if s["causal"]:
        seen = seen & (key <= at[:, None] + (n - t))
    scores = torch.matmul(q32 * scale, k32.transpose(2, 3).contiguous())
    scores = torch.where(seen[:, :, None], scores.view(b, hk, h // hk, t, n), -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(b, hk, -1, n)
    del scores
    out = torch.matmul(p, v32)
    if not s["train"]:
        return back(out, q)
    dy = rows(s["dy"])
    dp = torch.matmul(dy, v32.transpose(2, 3).contiguous())
    ds = p * (dp - (dy * out).sum(-1, keepdim=True)) * scale
    del dp
    dk, dv = torch.matmul(ds.transpose(2, 3).contiguous(), q32), torch.matmul(p.transpose(2, 3).contiguous(), dy)
    return back(out, q), back(torch.matmul(ds, k32), q), dk.transpose(1, 2).to(k.dtype), dv.transpose(1, 2).to(v.dtype)


def _pairs(case):
    """Query and key pairs that count: all of the causal triangle's or of the sequences' lengths."""
    t, n = case["tokens"], case["keys"]
    total = 0
    for length in _lengths(case) if case["ragged"] else [n] * case["batch"]:
        if not case["causal"]:
            total += t * length
        else:     # query i sees min(length, i + n - t + 1) keys
            first, last = n - t + 1, n
            low, high = max(1, first), min(last, length - 1)
            total += max(0, last - max(first, length) + 1) * length + (0 if high < low else (low + high) * (high - low + 1) // 2)
    return total


def work(case):
    size, b, t, h, hk, d = (SIZE[case["dtype"]], case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"])
    if case["op"] == "attention":
        keys = sum(_lengths(case)) if case["ragged"] else b * case["keys"]
        queries, cache = b * t * h * d * size, keys * hk * d * size
        pairs = _pairs(case) * h * d
        if not case["train"]:
            return {"bytes": 2 * queries + 2 * cache, "flops": 4 * pairs}
        # q, k, v, dy in; out, dq, dk, dv out; the gradients of keys that no query sees are written too
        return {"bytes": 4 * queries + 2 * cache + 2 * b * case["keys"] * hk * d * size, "flops": 14 * pairs}
    both = b * t * (h + hk) * d
    twice = 2 if case["train"] else 1
    return {"bytes": 2 * twice * both * size + 8 * b * t, "flops": (6 if case["op"] == "head_norm" else 3) * both * twice}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _attention_exact(s)
    leaves = [s[n].detach().double().requires_grad_() for n in s["leaves"]]
    # The rotation as a product of complex numbers.
    turn = torch.polar(torch.full((), s["amplitude"], dtype=torch.float64, device="cuda"),
                       (s["positions"].double()[:, :, None, None] * s["frequencies"]))
    half, outs = turn.shape[-1], []
    for i, x in enumerate(leaves[:2]):
        if case["op"] == "head_norm":
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * leaves[2 + i]
        part = x[..., :2 * half].unflatten(-1, (half, 2)) if s["interleaved"] else x[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
        part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
        part = part if s["interleaved"] else part.transpose(-1, -2)
        outs.append(torch.cat([part.flatten(-2), x[..., 2 * half:]], -1))
    if not s["train"]:
        return tuple(o.detach() for o in outs)
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, leaves, [s["dq"].double(), s["dk"].double()])


def _attention_exact(s):
    """Head by head in 64 bits, the gradients from the product rule of a softmax."""
    q, k, v = s["q"].detach(), s["k"].detach(), s["v"].detach()
    (b, t, h, d), n, hk = q.shape, k.shape[1], k.shape[2]
    lengths = [n] * b if s["lengths"] is None else s["lengths"].tolist()
    out, dq = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    dk, dv = torch.zeros(k.shape, dtype=torch.float64, device="cuda"), torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    for i in range(b):
        m = lengths[i]
        if m == 0:
            continue
        hidden = torch.ones(t, m, dtype=torch.bool, device="cuda").triu(n - t + 1) if s["causal"] else None
        for j in range(h):
            qj, kj, vj = q[i, :, j].double(), k[i, :m, j * hk // h].double(), v[i, :m, j * hk // h].double()
            z = qj @ kj.t() / math.sqrt(d)
            p = torch.softmax(z if hidden is None else z.masked_fill(hidden, -math.inf), -1)
            if hidden is not None:
                p = p.masked_fill(hidden.all(-1, keepdim=True), 0.0)
            out[i, :, j] = p @ vj
            if s["train"]:
                gj = s["dy"][i, :, j].double()
                dv[i, :m, j * hk // h] += p.t() @ gj
                dz = p * (gj @ vj.t())
                dz = (dz - p * dz.sum(-1, keepdim=True)) / math.sqrt(d)
                dq[i, :, j] = dz @ kj
                dk[i, :m, j * hk // h] += dz.t() @ qj
    return (out, dq, dk, dv) if s["train"] else out
