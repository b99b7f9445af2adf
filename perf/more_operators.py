"""Operators of an experts' feed-forward block, as a program calls them on what one worker holds: the root-mean-square norm in front
of it (with the residual's addition, and with rows in 8 bits that carry a scale each), tokens sorted by their experts and brought
back with the router's weights, and the products of the sorted rows with each expert's own weights.

A case names an operator, its sizes, element type and direction.  ``run`` computes it in plain torch operations, or calls the
framework's operators where ``own`` is true.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
EPS = 1e-6
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126


def listed():
    return [
        # One token for each of sixteen sequences of the repository's 8192 features: the norm in front of a product in 8 bits.  Latency.
        {"name": "norm_decode_8bit", "op": "norm", "dtype": "bf16", "rows": 16, "cols": 8192, "residual": True, "eight": True, "train": False},
        # The same for a prompt's 4 x 2048 tokens.
        {"name": "norm_prefill_8bit", "op": "norm", "dtype": "bf16", "rows": 8192, "cols": 8192, "residual": True, "eight": True, "train": False},
        # Training step on the repository's sequences (4 x 2048 tokens of 8192 features).
        {"name": "norm_train", "op": "norm", "dtype": "bf16", "rows": 8192, "cols": 8192, "residual": True, "eight": False, "train": True},
        # Training step in the layers' default type, odd numbers of rows and columns, no residual.
        {"name": "norm_ragged", "op": "norm", "dtype": "f32", "rows": 3001, "cols": 2501, "residual": False, "eight": False, "train": True},
        # One token for each of sixteen sequences to two of eight experts and back.  Latency.
        {"name": "move_decode", "op": "move", "dtype": "bf16", "tokens": 16, "chosen": 2, "experts": 8, "low": 0, "high": 8, "cols": 8192,
         "padded": 0, "train": False},
        # Training step: the repository's sequences to two of eight experts and back, all gradients.
        {"name": "move_train", "op": "move", "dtype": "bf16", "tokens": 8192, "chosen": 2, "experts": 8, "low": 0, "high": 8, "cols": 8192,
         "padded": 0, "train": True},
        # A prompt to eight of 128 small experts, of which this worker holds an eighth; rows travel in 8 bits with their scales.
        {"name": "move_prefill_8bit", "op": "move", "dtype": "e4m3", "tokens": 8192, "chosen": 8, "experts": 128, "low": 32, "high": 48, "cols": 2048,
         "padded": 0, "train": False},
        # Training step with everything odd: padded tokens, a window of experts, rows that are no whole vectors.
        {"name": "move_ragged", "op": "move", "dtype": "f16", "tokens": 4097, "chosen": 3, "experts": 13, "low": 2, "high": 11, "cols": 1001,
         "padded": 130, "train": True},
        # Sixteen tokens at two of eight experts each, one worker's 3584 of their hidden features: the weights' bytes are the cost.
        {"name": "product_decode", "op": "product", "dtype": "bf16", "rows": 32, "experts": 8, "spare": 0, "k": 8192, "n": 3584, "train": False},
        # A prompt's rows in 8 bits.
        {"name": "product_prefill_8bit", "op": "product", "dtype": "e4m3", "rows": 16384, "experts": 8, "spare": 0, "k": 8192, "n": 3584,
         "train": False},
        # Training step: product, gradients of the rows and of every expert's weights.
        {"name": "product_train", "op": "product", "dtype": "bf16", "rows": 16384, "experts": 8, "spare": 0, "k": 4096, "n": 3584, "train": True},
        # Training step in the layers' default type: odd sizes, an expert without rows, rows behind the last expert's.
        {"name": "product_ragged", "op": "product", "dtype": "f32", "rows": 1501, "experts": 5, "spare": 99, "k": 513, "n": 771, "train": True},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "move", "product", "product"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        eight = rng.random() < 0.4
        cols = _spread(rng, 8, 16384)
        cols = cols // 8 * 8 if rng.random() < 0.6 else cols
        rows = _spread(rng, 1, max(1, min(65536, 2 ** 26 // (cols * (2 if dtype == "f32" else 1)))))
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.7, "eight": eight,
                "train": not eight and rng.random() < 0.7}
    experts = _spread(rng, 1, 256 if op == "move" else 64)
    if op == "move":
        chosen = rng.randint(1, min(8, experts))
        dtype = rng.choice([dtype, dtype, "e4m3"])
        cols = _spread(rng, 8, 8192)
        cols = cols // 16 * 16 if rng.random() < 0.6 and cols >= 16 else cols
        tokens = _spread(rng, 1, max(1, min(32768, 2 ** 26 // (cols * chosen))))
        low, high = 0, experts
        if experts > 3 and rng.random() < 0.5:
            low = rng.randint(0, experts - 2)
            high = rng.randint(low + 1, experts)
        return {"op": op, "dtype": dtype, "tokens": tokens, "chosen": chosen, "experts": experts, "low": low, "high": high, "cols": cols,
                "padded": rng.choice([0, tokens // 9]), "train": dtype != "e4m3" and rng.random() < 0.7}
    dtype = rng.choice([dtype, dtype, "e4m3"])
    k, n = _spread(rng, 64, 8192), _spread(rng, 64, 8192)
    if rng.random() < 0.7:
        k, n = k // 32 * 32, n // 32 * 32
    if dtype == "e4m3":
        k = k // 16 * 16
    experts = max(1, min(experts, 2 ** 28 // (k * n)))
    train = dtype != "e4m3" and rng.random() < 0.6
    most = 2 ** 38 // (k * n * (16 if dtype == "f32" else 3 if train else 1))
    rows = _spread(rng, 1, max(1, min(16384, most)))
    return {"op": op, "dtype": dtype, "rows": rows, "experts": experts, "spare": rng.choice([0, 0, rows // 10]), "k": k, "n": n, "train": train}


def _popularity(experts):
    """How often experts are chosen, relative to each other: some three times as often as others, one in eight hardly ever."""
    return [0.02 if e % 8 == 5 else 0.5 + (e * 7 % 11) / 11.0 for e in range(experts)]


def _counts(case):
    """Rows of each expert, in all ``rows``."""
    share = _popularity(case["experts"])
    if case["experts"] >= 5:
        share[4] = 0.0
    total, counts, left = sum(share), [], case["rows"]
    for e, p in enumerate(share):
        got = left if e == case["experts"] - 1 else min(left, int(round(case["rows"] * p / total)))
        counts.append(got)
        left -= got
    return counts


def _to_rows8(y):
    """``(codes, scales)``: a scale for each row, with which its largest element becomes the type's largest."""
    scale = (y.abs().amax(-1, keepdim=True) / E4M3_MAX).clamp(min=SMALLEST_SCALE)
    return (y / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale[..., 0]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    eight = case["dtype"] == "e4m3"
    dt = torch.bfloat16 if eight else DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dt)

    train = case["train"]
    state = {"op": case["op"], "train": train, "leaves": []}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # The stream grows with depth and has a few features far above the others; the branch that is added is smaller.
        loud = torch.ones(cols, device="cuda")
        loud[torch.randint(0, cols, (max(1, cols // 512),), generator=g, device="cuda")] = 20.0
        state.update(x=normal(rows, cols, scale=0.5), weight=(1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dt),
                     residual=(normal(rows, cols, scale=2.0) * loud.to(dt)) if case["residual"] else None, eight=case["eight"])
        if train:
            state.update(dy=normal(rows, cols, scale=0.1), dh=normal(rows, cols, scale=0.1))
            state["leaves"] = ["x", "weight"] + (["residual"] if case["residual"] else [])
    elif case["op"] == "move":
        tokens, chosen, experts, cols = case["tokens"], case["chosen"], case["experts"], case["cols"]
        logits = torch.tensor(_popularity(experts), device="cuda").log() - torch.log(-torch.log(
            torch.rand(tokens, experts, generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
        top = logits.topk(chosen, -1)
        ids = top.indices
        if case["padded"]:
            ids[tokens - case["padded"]:] = -1
        state.update(ids=ids, experts=experts, window=(case["low"], case["high"]), x=normal(tokens, cols), eight=eight)
        if eight:
            state["x"], state["scales"] = _to_rows8(state["x"].float())
        else:
            state.update(y=normal(tokens * chosen, cols), weights=torch.softmax(top.values, -1))
            state["leaves"] = ["x", "y", "weights"] if train else []
            if train:
                state.update(dsorted=normal(tokens * chosen, cols, scale=0.1), dout=normal(tokens, cols, scale=0.1))
    else:
        counts, rows, k, n = _counts(case), case["rows"] + case["spare"], case["k"], case["n"]
        bounds = [0]
        for c in counts:
            bounds.append(bounds[-1] + c)
        state.update(counts=counts, offsets=torch.tensor(bounds, dtype=torch.int32, device="cuda"), x=normal(rows, k),
                     w=normal(case["experts"], n, k, scale=k ** -0.5), eight=eight)
        if eight:
            state["x"], state["x_scales"] = _to_rows8(state["x"].float())
            state["w"], state["w_scales"] = _to_rows8(state["w"].float())
        if train:
            state["dy"] = normal(rows, n, scale=0.1)
            state["leaves"] = ["x", "w"]
    for name in state["leaves"]:
        state[name] = state[name].detach().requires_grad_()
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _values8(codes, scales):
    """What rows in 8 bits stand for, in 16."""
    return (codes.float() * scales[..., None]).to(torch.bfloat16)


def _run_own(s):
    from distdl_amd import nn
    leaves = [s[n] for n in s["leaves"]]
    if s["op"] == "norm":
        if s["eight"]:
            with torch.no_grad():
                out = nn.rms_norm_shard(s["x"], s["weight"], s["residual"], eps=EPS, eight_bit=True)
            return (_values8(out[0], out[1]),) + tuple(out[2:])
        out = nn.rms_norm_shard(s["x"], s["weight"], s["residual"], eps=EPS)
        outs, grads = (out, [s.get("dy"), s.get("dh")]) if s["residual"] is not None else ((out,), [s.get("dy")])
    elif s["op"] == "move":
        plan = nn.expert_plan(s["ids"], s["experts"], window=s["window"])
        if s["eight"]:
            codes, scales = nn.expert_sort(s["x"], plan, scales=s["scales"])
            return _values8(codes, scales), plan.offsets
        moved, out = nn.expert_sort(s["x"], plan), nn.expert_combine(s["y"], plan, s["weights"])
        if not s["train"]:
            return moved, out, plan.offsets
        return (moved.detach(), out.detach(), plan.offsets) + torch.autograd.grad([moved, out], leaves, [s["dsorted"], s["dout"]])
    else:
        if s["eight"]:
            return nn.expert_linear_shard(s["x"], s["w"], s["offsets"], x_scales=s["x_scales"], weight_scales=s["w_scales"])
        outs, grads = (nn.expert_linear_shard(s["x"], s["w"], s["offsets"]),), [s.get("dy")]
    if not s["train"]:
        return outs
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, leaves, grads)


def _run_plain(s):
    with torch.no_grad():
        return {"norm": _norm_plain, "move": _move_plain, "product": _product_plain}[s["op"]](s)


def _norm_plain(s):
    x, r = s["x"], s["residual"]
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    h32, w32 = h.float(), s["weight"].float()
    rstd = torch.rsqrt((h32 * h32).mean(-1, keepdim=True) + EPS)
    xhat = h32 * rstd
    y = xhat * w32
    if s["eight"]:
        return (_values8(*_to_rows8(y)),) + (() if r is None else (h,))
    outs = (y.to(x.dtype),) + (() if r is None else (h,))
    if not s["train"]:
        return outs
    g = s["dy"].float() * w32
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    if r is not None:
        dx = dx + s["dh"].float()
    dw = (s["dy"].float() * xhat).sum(0)
    dx = dx.to(x.dtype)
    return outs + (dx, dw.to(x.dtype)) + (() if r is None else (dx,))


def _plan_plain(s):
    """``(slots in the experts' order, which of them count, offsets, each slot's place)``."""
    low, high = s["window"]
    ids = s["ids"].reshape(-1)
    ids = torch.where((ids >= low) & (ids < high), ids - low, high - low)
    key, source = torch.sort(ids, stable=True)
    counts = (ids[:, None] == torch.arange(high - low, device=ids.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    place = torch.empty_like(source)
    place[source] = torch.arange(len(source), device=ids.device)
    return source, key < high - low, offsets, place


def _move_plain(s):
    source, held, offsets, place = _plan_plain(s)
    tokens, chosen = s["ids"].shape
    token = source // chosen

    def rows_of(t):     # [tokens, ...] in the experts' order, zeros behind the last
        taken = t.float()[token]
        return torch.where(held.view(-1, *[1] * (taken.dim() - 1)), taken, 0.0)

    if s["eight"]:
        return (rows_of(s["x"]) * rows_of(s["scales"])[:, None]).to(torch.bfloat16), offsets
    dt, weights = s["x"].dtype, s["weights"]
    here = held[place].view(tokens, chosen)

    def back(t):        # [slots, cols] to [tokens, chosen, cols], zeros where an expert is not held
        return torch.where(here[..., None], t.float()[place].view(tokens, chosen, -1), 0.0)

    outs = rows_of(s["x"]).to(dt), (back(s["y"]) * weights[..., None]).sum(1).to(dt), offsets
    if not s["train"]:
        return outs
    dx = back(s["dsorted"]).sum(1).to(dt)
    dy = (rows_of(s["dout"]) * torch.where(held, weights.reshape(-1)[source], 0.0)[:, None]).to(dt)
    dweights = (back(s["y"]) * s["dout"].float()[:, None]).sum(-1)
    return outs + (dx, dy, dweights)


def _product_plain(s):
    x, w, counts = s["x"], s["w"], s["counts"]
    x32 = x.float() * s["x_scales"][:, None] if s["eight"] else x.float()
    y = x32.new_zeros(x.shape[0], w.shape[1])
    if s["train"]:
        dy32 = s["dy"].float()
        dx, dw = torch.zeros_like(x32), torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    at = 0
    for e, c in enumerate(counts):
        rows = slice(at, at + c)
        at += c
        if c == 0:
            continue
        w32 = w[e].float() * s["w_scales"][e][:, None] if s["eight"] else w[e].float()
        y[rows] = x32[rows] @ w32.t()
        if s["train"]:
            dx[rows] = dy32[rows] @ w32
            dw[e] = dy32[rows].t() @ x32[rows]
    out = torch.bfloat16 if s["eight"] else x.dtype
    return (y.to(out), dx.to(out), dw.to(out)) if s["train"] else (y.to(out),) if not s["eight"] else y.to(out)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm":
        # x (and the residual) in, y (and their sum) out; for training dy (and the sum's gradient) and the sum in, one gradient out.
        n, both = case["rows"] * case["cols"], 2 if case["residual"] else 1
        total = n * size * (2 * both if not case["eight"] else 2 * both - 1) + (n + 4 * case["rows"] if case["eight"] else 0)
        total += case["cols"] * size
        if case["train"]:
            total += n * size * (both + 2) + case["cols"] * size
        return {"bytes": total, "flops": n * (14 if case["train"] else 5)}
    if case["op"] == "move":
        # The share of choices that the window holds; every row that is moved is written once, and read once where it comes from.
        share = _popularity(case["experts"])
        low, high = case["low"], case["high"]
        slots = case["tokens"] * case["chosen"]
        held = int((case["tokens"] - case["padded"]) * case["chosen"] * sum(share[low:high]) / sum(share))
        row, sources = case["cols"] * size, min(held, case["tokens"])
        if case["dtype"] == "e4m3":
            return {"bytes": 8 * slots + (slots + sources) * (row + 4), "flops": 1}
        total = 8 * slots + (sources + slots) * row + (held + case["tokens"]) * row + 4 * slots
        flops = 2 * held * case["cols"]
        if case["train"]:
            # dx from the sorted rows' gradients; dy, and the weights' gradients from the rows that are there again
            total += (held + case["tokens"]) * row + (case["tokens"] + slots + held) * row + 8 * slots
            flops *= 4
        return {"bytes": total, "flops": flops}
    rows, k, n = case["rows"] + case["spare"], case["k"], case["n"]
    used = sum(1 for c in _counts(case) if c)
    if case["dtype"] == "e4m3":
        return {"bytes": case["rows"] * (k + 4) + used * (k + 4) * n + rows * n * 2, "flops": 2 * case["rows"] * k * n}
    total, flops = size * (case["rows"] * k + used * k * n + rows * n), 2 * case["rows"] * k * n
    if case["train"]:
        total += size * (case["rows"] * n + rows * k + case["experts"] * k * n)
        flops *= 3
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _norm_exact(s)
    if case["op"] == "move":
        return _move_exact(s)
    return _product_exact(s)


def _norm_exact(s):
    # The sum is rounded once to its type: it is a result of its own, and what is normalised.
    x = s["x"].detach()
    h = x if s["residual"] is None else (x.double() + s["residual"].detach().double()).to(x.dtype)
    leaf, w = h.double().requires_grad_(), s["weight"].detach().double().requires_grad_()
    y = leaf / torch.sqrt(leaf.pow(2).sum(-1, keepdim=True) / leaf.shape[-1] + EPS) * w
    extra = () if s["residual"] is None else (h.double(),)
    if s["eight"]:
        y = y.detach()
        scale = (y.abs().max(-1, keepdim=True).values / E4M3_MAX).clamp(min=SMALLEST_SCALE)
        # The nearest values of three mantissa bits, the smallest normal 2^-6, ties to the even one (round does so).
        v = y / scale
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        return ((torch.round(v / step) * step) * scale,) + extra
    if not s["train"]:
        return (y.detach(),) + extra
    dx, dw = torch.autograd.grad(y, [leaf, w], s["dy"].double())
    if s["residual"] is None:
        return y.detach(), dx, dw
    dx = dx + s["dh"].double()
    return y.detach(), h.double(), dx, dw, dx


def _move_exact(s):
    low, high = s["window"]
    ids = s["ids"]
    tokens, chosen = ids.shape
    lists = [torch.nonzero(ids.reshape(-1) == e)[:, 0] for e in range(low, high)]     # in the slots' order
    slots = torch.cat(lists)
    bounds = torch.tensor([0] + [len(x) for x in lists]).cumsum(0).to(torch.int32).cuda()
    token = torch.div(slots, chosen, rounding_mode="floor")
    n, cols = len(slots), s["x"].shape[1]
    rows = torch.zeros(tokens * chosen, cols, dtype=torch.float64, device="cuda")
    if s["eight"]:
        rows[:n] = (s["x"].double() * s["scales"].double()[:, None])[token]
        return rows, bounds
    weights, y = s["weights"].detach().double(), s["y"].detach().double()
    taken = weights.reshape(-1)[slots][:, None]
    rows[:n] = s["x"].detach().double()[token]
    out = torch.zeros(tokens, cols, dtype=torch.float64, device="cuda").index_add_(0, token, y[:n] * taken)
    if not s["train"]:
        return rows, out, bounds
    dx = torch.zeros_like(out).index_add_(0, token, s["dsorted"].double()[:n])
    dout = s["dout"].double()[token]
    dy = torch.zeros_like(rows)
    dy[:n] = dout * taken
    dweights = torch.zeros(tokens * chosen, dtype=torch.float64, device="cuda")
    dweights[slots] = (dout * y[:n]).sum(-1)
    return rows, out, bounds, dx, dy, dweights.view(tokens, chosen)


def _product_exact(s):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    if s["eight"]:
        x, w = x * s["x_scales"].double()[:, None], w * s["w_scales"].double()[..., None]
    y, at = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda"), 0
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for e, c in enumerate(s["counts"]):
        rows = slice(at, at + c)
        y[rows] = torch.mm(x[rows], w[e].t())
        if s["train"]:
            dx[rows] = torch.mm(s["dy"][rows].double(), w[e])
            dw[e] = torch.mm(s["dy"][rows].double().t(), x[rows])
        at += c
    return (y, dx, dw) if s["train"] else y if s["eight"] else (y,)
