"""Attention against its definition in 64 bits, forward and adjoint, in both forms of the forward (whole key ranges for each
row, and keys split over workgroups).

Tolerances.  With u = half a step of the element type (``finfo.eps / 2``; probabilities and their gradients are rounded to it for
the second product, fp32 keeps them) and e = 2^-24:

* a score is a sum of head_dim <= 128 products in 32 bits, off by at most (128 + 2) e sum |q k| scale, which p turns into as large a
  relative error; with the exponential and the running sums (n terms of one sign) p is off by  c = 131 e A + 2^-21 + n e  of itself,
  A = the largest sum |q k| scale of the case (2^-21: exponential, its argument's rounding for scores up to A is in the first term);
* out: u |out| for the result, (u + 2 c) sum p |v| before it (the error of the total is another c), and u |out| more for the total, which is the
  sum of the probabilities as rounded: with p (1 + d), |d| <= u, for p, sum p (1 + d) v / sum p (1 + d) is sum p d (v - out) off to first
  order, at most u sum p |v - out| <= u (sum p |v| + |out|).  (With values of 0 and one of 1 that has little weight the sum is twice
  u sum p |v|, so the second term is needed.)  The adjoint's probabilities come from the unrounded total;
* gradients: dv as out, with sums over queries of p |dy|; dS = p (dP - D), dP and D off by 130 e sum |dy v| each (D: from `out` and
  what its rounding took, rounded, so off by its tolerance without the result's own: (u + u^2) sum |dy out| + (u + 2 c) sum |dy| (p |v|) more, fp32
  u sum |dy out| instead of the first), so dS is off by
  p ((u + 2 c) (|dP| + |D|) + 260 e sum |dy v| + D's), and dq, dk sum that times |k|, |q|; sums of n terms add n e of their magnitude.
The sums of magnitudes are formed in 64 bits with absolute values.  float16 loses 2^-25 next to zero for every rounding (a probability,
a result) on top.
"""

import numpy as np
import pytest
import torch

from oracle import heads as o_heads

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _f64(t):
    return t.detach().double().cpu().numpy()


def _bounds(q, k, v, lengths, causal, scale, u, tiny, dy=None, rounded=True):
    """Tolerances of out (and dq, dk, dv) as derived above; ``rounded``: the second product takes values of the element type."""
    (batch, tokens, heads, dim), keys, kv_heads = q.shape, k.shape[1], k.shape[2]
    e, up = 2.0 ** -24, (u if rounded else 0.0)
    out, dq, dk, dv = np.zeros_like(q), np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for b in range(batch):
        see = o_heads.visible(tokens, keys, keys if lengths is None else lengths[b], causal)
        some, n = see.any(-1), max(1, int(see.sum(-1).max()))
        for h in range(heads):
            j = h * kv_heads // heads
            kb, vb, qb = np.where(see.any(0)[:, None], k[b, :, j], 0), np.where(see.any(0)[:, None], v[b, :, j], 0), q[b, :, h]
            s = np.where(see, scale * qb @ kb.T, -np.inf)
            p = np.exp(s - np.where(some, s.max(-1, initial=-np.inf), 0)[:, None])
            p /= np.where(some, p.sum(-1), 1)[:, None]
            big = np.where(see, scale * np.abs(qb) @ np.abs(kb).T, 0).max(initial=0)
            c = 131 * e * big + 2.0 ** -21 + n * e
            o = p @ vb
            room = p + tiny * see
            out[b, :, h] = (u + up) * np.abs(o) + (up + 2 * c) * (room @ np.abs(vb)) + tiny * (see @ np.abs(vb)) + tiny
            if dy is None:
                continue
            g = dy[b, :, h]
            dp, dd = g @ vb.T, (g * o).sum(-1)[:, None]
            mag, mago, magp = np.abs(g) @ np.abs(vb).T, (np.abs(g) * np.abs(o)).sum(-1)[:, None], (np.abs(g) * (p @ np.abs(vb))).sum(-1)[:, None]
            off = p * ((up + 2 * c) * (np.abs(dp) + np.abs(dd)) + 260 * e * mag + (up + u * u if u > e else u) * mago + tiny * np.abs(g).sum(-1)[:, None] + (up + 2 * c) * magp) + tiny * see
            ds = p * (dp - dd)
            e_sum = (tokens + keys) * e
            dq[b, :, h] = u * np.abs(scale * ds @ kb) + scale * (off + e_sum * np.abs(ds)) @ np.abs(kb) + tiny
            dk[b, :, j] += scale * (off + e_sum * np.abs(ds)).T @ np.abs(qb)
            dv[b, :, j] += ((up + 2 * c + e_sum) * p + tiny * see).T @ np.abs(g)
    # (the results of dk and dv are rounded as well: below 2^-14 a float16 is off by up to half of 2^-24, whatever its value)
    return out, dq, dk + tiny, dv + tiny


def _within(name, got, want, tol, u=0.0):
    got = _f64(got)
    assert got.shape == want.shape, name
    tol = tol + u * np.abs(want) + 1e-30
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} off, worst {np.max(np.where(np.isfinite(got), np.abs(got - want), np.inf) / tol):.3g} of the tolerance"


def _inputs(dt, batch, tokens, keys, heads, kv_heads, dim, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (1.5 * torch.randn(batch, tokens, heads, dim, generator=g)).to(dt).cuda()
    k = torch.randn(batch, keys, kv_heads, dim, generator=g).to(dt).cuda()
    v = torch.randn(batch, keys, kv_heads, dim, generator=g).to(dt).cuda()
    dy = torch.randn(batch, tokens, heads, dim, generator=g).to(dt).cuda()
    return q, k, v, dy


def _check(dt, q, k, v, lengths=None, causal=False, scale=None, dy=None, rounded=None):
    from distdl_amd import nn
    u, tiny = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == torch.float16 else 0.0
    if dy is not None:
        for t in (q, k, v):
            t.requires_grad_()
    out = nn.attention_shard(q, k, v, lengths, causal=causal, scale=scale)
    assert out.is_contiguous() and out.dtype == dt
    n = None if lengths is None else lengths.cpu().numpy().clip(0, k.shape[1])
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    qn, kn, vn = _f64(q), _f64(k), _f64(v)
    want = o_heads.attention(qn, kn, vn, n, causal, sc, None if dy is None else _f64(dy))
    tol = _bounds(qn, kn, vn, n, causal, sc, u, tiny, None if dy is None else _f64(dy), dt != torch.float32 if rounded is None else rounded)
    _within("out", out, want[0], tol[0])
    if dy is not None:
        grads = torch.autograd.grad(out, [q, k, v], dy)
        for name, g, w, t in zip(("dq", "dk", "dv"), grads, want[2:], tol[1:]):
            _within(name, g, w, t, u)
    return out


CASES = [   # batch, tokens, keys, heads, kv_heads, dim, lengths, causal
    (1, 1, 1, 1, 1, 8, None, False), (2, 3, 5, 2, 1, 16, [5, 0], False), (1, 130, 70, 2, 2, 40, None, False), (3, 33, 65, 4, 2, 64, [65, 1, 33], False),
    (1, 200, 200, 2, 1, 128, None, True), (2, 70, 40, 2, 2, 32, None, True), (2, 40, 70, 2, 2, 96, [70, 31], True), (1, 129, 257, 3, 3, 72, None, True),
    (2, 1, 700, 8, 2, 128, [700, 513], False), (5, 1, 97, 4, 4, 64, [97, 0, 1, 32, 33], False), (1, 4, 1100, 8, 1, 80, None, True),
    (1, 2, 1, 4, 1, 24, None, False), (2, 5, 3, 12, 4, 100, [3, 2], True), (1, 64, 64, 1, 1, 33, None, True), (1, 16, 3000, 8, 1, 48, [2999], False),
    (1, 7, 9, 2, 2, 1, None, False), (1, 300, 520, 2, 1, 128, [400], False),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_forward(dt, case):
    batch, tokens, keys, heads, kv_heads, dim, lengths, causal = case
    q, k, v, _ = _inputs(dt, batch, tokens, keys, heads, kv_heads, dim)
    _check(dt, q, k, v, None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda"), causal)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_adjoint(dt, case):
    batch, tokens, keys, heads, kv_heads, dim, lengths, causal = case
    q, k, v, dy = _inputs(dt, batch, tokens, keys, heads, kv_heads, dim, seed=1)
    _check(dt, q, k, v, None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda"), causal, dy=dy)


# Enough rows for every workgroup to take whole ranges of keys (at least 3 blocks of 32 rows for each of 256 CUs, and at most half as many of 128;
# causal ones count by the keys that they see).
MANY = [
    (20, 130, 70, 8, 8, 40, [70, 0, 33, 64, 1], False), (24, 200, 257, 8, 8, 72, [257, 250, 129], True), (50, 100, 33, 4, 4, 128, None, False),
    (12, 300, 300, 8, 2, 64, None, True), (3, 520, 200, 16, 1, 24, [200, 0, 97], True), (26, 257, 64, 4, 2, 96, [64, 63], False), (10, 513, 97, 16, 2, 128, [97, 65, 0, 32, 31], True),
    (16, 129, 1, 16, 16, 16, [1, 0], False),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", MANY)
def test_many_rows(dt, case):
    batch, tokens, keys, heads, kv_heads, dim, lengths, causal = case
    q, k, v, dy = _inputs(dt, batch, tokens, keys, heads, kv_heads, dim, seed=14)
    n = None if lengths is None else torch.tensor((batch * lengths)[:batch], dtype=torch.int32, device="cuda")
    _check(dt, q, k, v, n, causal)
    _check(dt, q, k, v, n, causal, dy=dy)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", [(1, 300, 1000, 4, 2, 128, None, True), (2, 70, 1300, 4, 4, 64, [1300, 70], True), (1, 130, 2100, 2, 2, 32, None, False),
                                  (1, 900, 700, 2, 1, 96, [650], True), (3, 9, 5000, 8, 1, 16, [5000, 0, 513], True)])
def test_splits_of_several_blocks_of_rows(dt, case):
    """The keys of 2 to 20 splits, whose sums are joined; causal ones end inside them."""
    test_forward(dt, case)
    test_adjoint(dt, case)


@pytest.mark.parametrize("layout", ["packed", "heads_first", "shared_sequences", "unaligned", "strided_features"])
@pytest.mark.parametrize("tokens", [1, 50])
def test_layouts(layout, tokens):
    """Views of a projection's output, heads before tokens, one set of keys for all sequences, operands off 16 bytes: as their copies, bit for bit."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(2)
    heads, kv, dim, keys = 4, 2, 32, 90
    if layout == "packed":
        x = torch.randn(2, keys, (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16).cuda()
        q = x[:, :tokens, :heads * dim].unflatten(-1, (heads, dim))
        k, v = (x[..., (heads + i * kv) * dim:(heads + (i + 1) * kv) * dim].unflatten(-1, (kv, dim)) for i in (0, 1))
    elif layout == "heads_first":
        q, k, v = (torch.randn(2, h, n, dim, generator=g).to(torch.bfloat16).cuda().transpose(1, 2) for h, n in ((heads, tokens), (kv, keys), (kv, keys)))
    elif layout == "shared_sequences":
        q = torch.randn(2, tokens, heads, dim, generator=g).to(torch.bfloat16).cuda()
        k, v = (torch.randn(1, keys, kv, dim, generator=g).to(torch.bfloat16).cuda().expand(2, -1, -1, -1) for _ in range(2))
    elif layout == "unaligned":
        q, k, v = (torch.randn(2, n, h, dim + 1, generator=g).to(torch.bfloat16).cuda()[..., 1:] for h, n in ((heads, tokens), (kv, keys), (kv, keys)))
    else:
        q, k, v = (torch.randn(2, n, h, 2 * dim, generator=g).to(torch.bfloat16).cuda()[..., ::2] for h, n in ((heads, tokens), (kv, keys), (kv, keys)))
    dy = torch.randn(2, tokens, heads, dim, generator=g).to(torch.bfloat16).cuda()
    results = []
    for copy in (False, True):
        leaves = [(t.contiguous() if copy else t).detach().requires_grad_() for t in (q, k, v)]
        out = nn.attention_shard(*leaves)
        results.append([out] + list(torch.autograd.grad(out, leaves, dy if copy else dy.transpose(1, 2).contiguous().transpose(1, 2))))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens,keys,times", [(1, 300, 1), (70, 130, 1), (130, 130, 40), (20, 1300, 1)])
def test_what_lies_behind_a_sequence_is_not_looked_at(dt, tokens, keys, times):
    """NaN and infinities in the padding: same bits as zeros there, zero gradients of the padding; a sequence without keys gives zeros."""
    from distdl_amd import nn
    lengths = torch.tensor(times * [keys - 37, 0, 1], dtype=torch.int32, device="cuda")
    results = []
    for filler in (0.0, float("nan"), float("inf"), -torch.finfo(dt).max):
        q, k, v, dy = _inputs(dt, 3 * times, tokens, keys, 4, 2, 40, seed=3)
        for b, n in enumerate(lengths.tolist()):
            k[b, n:], v[b, n:] = filler, filler
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = nn.attention_shard(*leaves, lengths)
        results.append([out.detach()] + list(torch.autograd.grad(out, leaves, dy)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    out, dq, dk, dv = results[0]
    assert not out[1].any() and not dq[1].any() and not dk[1].any() and not dv[1].any()
    assert not dk[0, keys - 37:].any() and not dv[2, 1:].any()


def test_lengths_outside_the_keys_count_as_none_and_all():
    from distdl_amd import nn
    q, k, v, _ = _inputs(torch.float32, 2, 3, 10, 2, 1, 16, seed=4)
    got = nn.attention_shard(q, k, v, torch.tensor([-5, 1000], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, nn.attention_shard(q, k, v, torch.tensor([0, 10], dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("shape", [(0, 3, 4, 2), (2, 0, 4, 2), (2, 3, 0, 2), (2, 3, 4, 0)])
def test_nothing_to_attend(shape):
    from distdl_amd import nn
    batch, tokens, keys, heads = shape
    q, k, v, dy = _inputs(torch.bfloat16, batch, tokens, keys, heads, min(heads, 1), 16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = nn.attention_shard(*leaves)
    assert out.shape == q.shape and not out.any()
    for leaf, grad in zip(leaves, torch.autograd.grad(out, leaves, dy)):
        assert grad.shape == leaf.shape and not grad.any()


def test_key_heads_without_heads():
    from distdl_amd import nn
    k = torch.randn(2, 5, 2, 16, device="cuda", requires_grad=True)
    q = torch.randn(2, 3, 0, 16, device="cuda", requires_grad=True)
    out = nn.attention_shard(q, k, k)
    assert out.shape == q.shape
    assert not torch.autograd.grad(out.sum(), [k])[0].any()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("keys,tokens", [(1, 5), (50, 5), (200, 5), (200, 3000)])
def test_gradients_of_a_single_key(dt, keys, tokens):
    """A probability of one is not rounded, and dS, the difference of two equal sums, is zero but for errors of 32 bits: the bounds without the
    roundings to the element type, all keys in one tile or not."""
    q, k, v, dy = _inputs(dt, 2, tokens, keys, 8, 2, 64, seed=15)
    _check(dt, q, k, v, torch.tensor([1, 0], dtype=torch.int32, device="cuda"), dy=dy, rounded=False)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("slope", [0.02, 0.3, -0.3])
@pytest.mark.parametrize("batch,tokens", [(1, 40), (160, 130)])
def test_maxima_that_rise_and_fall_along_the_keys(dt, slope, batch, tokens):
    """Scores that climb (by less and by more than the running maximum's slack from tile to tile) or fall along 400 keys."""
    q, k, v, dy = _inputs(dt, batch, tokens, 400, 1, 1, 16, seed=5)
    k.zero_()
    k[:, :, 0, 0] = slope * torch.arange(400, device="cuda")
    q[..., 0] = 2.0
    _check(dt, q, k, v, scale=1.0, dy=dy)
    _check(dt, q.detach()[:, :1], k.detach(), v.detach(), scale=1.0)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,tokens", [(1, 33), (160, 130)])
def test_large_scores_and_other_scales(dt, batch, tokens):
    """Scores of some thousands: one key takes all.  In powers of two they stay below 2^13, where the maximum is rounded by up to 2^-11: the
    probability of the best key comes out as 1 within 2^-11, as does the total, whose rounded one is divided by the unrounded one."""
    from distdl_amd import nn
    q, k, v, _ = _inputs(dt, batch, tokens, 70, 1, 1, 64, seed=6)
    out = nn.attention_shard(q, k, v, scale=100.0)
    s = _f64(q)[:, :, 0] @ _f64(k)[:, :, 0].transpose(0, 2, 1)
    best = s.argmax(-1)
    s = np.sort(s, -1)
    clear = (s[..., -1] - s[..., -2] > 1.0) & (s[..., -1] * 100 * np.log2(np.e) < 2 ** 13)      # e^-100 and less for all others
    assert clear.sum() > 20 * batch
    want = np.take_along_axis(_f64(v)[:, :, 0], best[..., None], 1)[clear]
    assert (np.abs(_f64(out)[:, :, 0][clear] - want) <= (torch.finfo(dt).eps / 2 + 2.0 ** -10) * np.abs(want)).all()


@pytest.mark.parametrize("tokens,heads", [(33, 2), (1600, 16)])
def test_strides_beyond_32_bits(tokens, heads):
    """Two sequences 2^31 elements apart."""
    from distdl_amd import nn
    far = 1 << 31
    base = torch.empty(far + 40 * 2 * 64, dtype=torch.bfloat16, device="cuda")
    k, v = (base.as_strided((2, 40, 1, 64), (far, 128, 64, 1), 64 * i) for i in (0, 1))
    q, kk, vv, dy = _inputs(torch.bfloat16, 2, tokens, 40, heads, 1, 64, seed=7)
    k.copy_(kk), v.copy_(vv)
    results = []
    for a, b in ((k, v), (kk, vv)):
        leaves = [t.detach().requires_grad_() for t in (q, a, b)]
        out = nn.attention_shard(*leaves, causal=True)
        results.append([out.detach()] + list(torch.autograd.grad(out, leaves, dy)) + [nn.attention_shard(q[:, :1], a, b)])
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_gradients_that_are_not_asked_for_and_not_of_the_type():
    from distdl_amd import nn
    q, k, v, dy = _inputs(torch.bfloat16, 2, 20, 30, 2, 2, 32, seed=8)
    whole = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(nn.attention_shard(*whole), whole, dy)
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        got, = torch.autograd.grad(nn.attention_shard(*some), [some[i]], dy)
        assert torch.equal(got, want[i])
    q.requires_grad_()
    out = nn.attention_shard(q, k, v)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(out.float().square().sum(), [q], create_graph=True)[0].sum(), [q])


def test_gradients_against_differences():
    """Central differences of the oracle's value, step 2^-14, with scores and values of order one: they and the fp32 gradients agree to 2^-14."""
    from distdl_amd import nn
    q, k, v, dy = _inputs(torch.float32, 1, 3, 4, 2, 1, 4, seed=9)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(nn.attention_shard(*leaves, causal=True), leaves, dy)
    values, h = [_f64(t) for t in leaves], 2.0 ** -14
    for i, grad in enumerate(grads):
        for at in np.ndindex(*values[i].shape):
            ends = []
            for sign in (1, -1):
                moved = [x.copy() for x in values]
                moved[i][at] += sign * h
                ends.append((o_heads.attention(*moved, causal=True)[0] * _f64(dy)).sum())
            assert abs((ends[0] - ends[1]) / (2 * h) - float(grad[at])) <= 2.0 ** -14 * (1 + np.abs(_f64(dy)).max())


@pytest.mark.parametrize("tokens,times", [(1, 1), (96, 1), (300, 6)])
def test_equal_calls_give_equal_bits_and_replay_from_a_graph(tokens, times):
    """Captured together with the adjoint, replayed with eager calls on the same leaves between, against the eager results."""
    from distdl_amd import nn
    q, k, v, dy = _inputs(torch.bfloat16, 2 * times, tokens, 3000, 8, 1, 64, seed=10)
    lengths = torch.tensor(times * [2999, 64], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        out = nn.attention_shard(*leaves, lengths)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, dy)) + [nn.attention_shard(*(t.detach() for t in leaves), lengths)]

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    g = torch.Generator().manual_seed(11)
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
            lengths[0] = 100 * i
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


@pytest.mark.parametrize("causal", [False, True])
def test_block_of_an_attention_layer(causal):
    """The operators in a row, as a worker runs them: projection to its heads, head norms and positions, attention, projection back, in
    float32 with all gradients, against the same in 64 bits.  The loosest of the operators' bounds is the attention's,
    c = 131 2^-24 A + 2^-21 with scores A up to 2^6: 2^-11 of the largest magnitude; 2^-10 for the chain, whose other errors are below 2^-16."""
    from distdl_amd import nn
    from distdl_amd.backends.stub_hip import SimWorld
    from distdl_amd.nn.linear import linear_shard
    P = SimWorld(1).partition(0).create_partition_inclusive([0]).create_cartesian_topology_partition([1, 1, 1, 1])
    g = torch.Generator().manual_seed(12)
    batch, tokens, heads, kv, dim, features, keys = 2, 45, 4, 2, 32, 64, 45 if causal else 77
    x = torch.randn(batch, tokens, features, generator=g).cuda().requires_grad_()
    states = x if causal else torch.randn(batch, keys, features, generator=g).cuda().requires_grad_()
    wq = (0.2 * torch.randn(heads * dim, features, generator=g)).cuda().requires_grad_()
    wkv = (0.2 * torch.randn(2 * kv * dim, features, generator=g)).cuda().requires_grad_()
    wo = (0.2 * torch.randn(features, heads * dim, generator=g)).cuda().requires_grad_()
    lengths = None if causal else torch.tensor([77, 40], dtype=torch.int32, device="cuda")
    norm, attend = nn.DistributedHeadNormRotary(P, dim, rotated=16), nn.DistributedAttention(P, causal=causal)
    dy = torch.randn(batch, tokens, features, generator=g).cuda()

    def framework():
        q = linear_shard(x, wq, None).unflatten(-1, (heads, dim))
        kv_out = linear_shard(states, wkv, None)
        k, v = (kv_out[..., i * kv * dim:(i + 1) * kv * dim].unflatten(-1, (kv, dim)) for i in (0, 1))
        if causal:
            q, k = norm(q, k)
        else:       # queries and keys have numbers of their own
            q, k = norm(q)[0], nn.head_norm_rotary_shard(None, k, None, norm.k_weight, norm._frequencies)[1]
        return linear_shard(attend(q, k, v, lengths).flatten(-2), wo, None)

    leaves = list(dict.fromkeys([x, states, wq, wkv, wo, norm.q_weight, norm.k_weight]))
    got = framework()
    grads = torch.autograd.grad(got, leaves, dy)

    copies = {t: t.detach().double().cpu().requires_grad_() for t in leaves}
    freq = norm._frequencies.cpu()

    def normed(t, w, n):
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + norm.eps) * w
        angle = (torch.arange(n, dtype=torch.float64)[:, None] * freq)[:, None]
        a, b = t[..., :8], t[..., 8:16]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), t[..., 16:]], -1)

    q = (copies[x] @ copies[wq].T).unflatten(-1, (heads, dim))
    k, v = (copies[states] @ copies[wkv].T).unflatten(-1, (2 * kv, dim)).split(kv, 2)
    q, k = normed(q, copies[norm.q_weight], tokens), normed(k, copies[norm.k_weight], keys)
    k, v = (t.repeat_interleave(heads // kv, 2).permute(0, 2, 3, 1) for t in (k, v))
    s = q.transpose(1, 2) @ k * dim ** -0.5
    for b in range(batch):
        hidden = ~torch.from_numpy(o_heads.visible(tokens, keys, keys if lengths is None else int(lengths[b]), causal).copy())
        s = torch.where(hidden & (torch.arange(batch) == b)[:, None, None, None], -torch.inf, s)
    want = (s.softmax(-1) @ v.transpose(2, 3)).transpose(1, 2).flatten(-2) @ copies[wo].T
    for a, b in zip([got] + list(grads), [want] + list(torch.autograd.grad(want, [copies[t] for t in leaves], dy.double().cpu()))):
        a, b = _f64(a), b.detach().numpy()
        assert np.abs(a - b).max() <= 2.0 ** -10 * np.abs(b).max()


def test_layers_over_batch_and_heads_of_four_workers():
    """Head norms with positions and attention on a 2 x 2 partition of batch and heads, every worker a thread: the workers' results are the whole
    tensor's, bit for bit, and the norms' weights, which live on the first worker, get the gradient of all tokens and heads (sums of another order:
    2^-17 of the magnitude that a single worker's would be off by, as for the head norms alone)."""
    from distdl_amd import nn
    from distdl_amd.backends.stub_hip import SimWorld
    g = torch.Generator().manual_seed(13)
    batch, tokens, heads, kv, dim = 4, 21, 4, 2, 32
    q, k, v, dy = (torch.randn(batch, tokens, h, dim, generator=g) for h in (heads, kv, kv, heads))
    lengths = torch.tensor([21, 7, 0, 20], dtype=torch.int32)

    def body(P_world, P_shape):
        P = P_world.create_partition_inclusive(list(range(int(np.prod(P_shape))))).create_cartesian_topology_partition(P_shape)
        if not P.active:
            return None
        norm, attend = nn.DistributedHeadNormRotary(P, dim, rotated=16), nn.DistributedAttention(P, causal=True)

        def own(t):
            for d in (0, 2) if t.dim() == 4 else (0,):
                t = t.chunk(P_shape[d], d)[P.index[d]]
            return t.contiguous().cuda()

        a, b = own(q).requires_grad_(), own(k).requires_grad_()
        y = attend(*norm(a, b), own(v), own(lengths))
        y.backward(own(dy))
        grads = [w.grad for w in (norm.q_weight, norm.k_weight)]
        return tuple(P.index), y.detach().cpu(), a.grad.cpu(), b.grad.cpu(), [None if w is None else w.cpu() for w in grads]

    whole = SimWorld(1).run(lambda P: body(P, [1, 1, 1, 1]))[0]
    parts = SimWorld(4).run(lambda P: body(P, [2, 1, 2, 1]))
    for index, y, dq, dk, _ in parts:
        for mine, all_ in ((y, whole[1]), (dq, whole[2]), (dk, whole[3])):
            assert torch.equal(mine, all_.chunk(2, 0)[index[0]].chunk(2, 2)[index[2]])
    for got, want in zip(parts[0][4], whole[4]):
        assert (got - want).abs().max() <= 2.0 ** -17 * batch * tokens * heads * want.abs().max()


@pytest.mark.parametrize("batch", [3, 64, 65, 130])
def test_sequences_of_many_lengths(batch):
    """Equal ones, none and all among them, more than a wavefront has lanes: every sequence as it comes out alone."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(16)
    q, k, v, dy = _inputs(torch.bfloat16, batch, 260, 100, 4, 2, 32, seed=16)
    lengths = torch.randint(-3, 104, (batch,), generator=g, dtype=torch.int32)
    lengths[0], lengths[1], lengths[2] = 100, 0, 100
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = nn.attention_shard(*leaves, lengths.cuda())
    whole = [out.detach()] + list(torch.autograd.grad(out, leaves, dy))
    u = torch.finfo(torch.bfloat16).eps / 2
    for b in {0, 1, 2, batch // 2, batch - 1}:
        n = int(lengths[b].clip(0, 100))
        one = [t.detach()[b:b + 1] for t in (q, k, v, dy)]
        want = o_heads.attention(*(_f64(t) for t in one[:3]), [n], False, None, _f64(one[3]))
        tol = _bounds(*(_f64(t) for t in one[:3]), [n], False, 32 ** -0.5, u, 0.0, _f64(one[3]))
        for name, got, exact, t, more in zip(("out", "dq", "dk", "dv"), whole, (want[0],) + want[2:], tol, (0, u, u, u)):
            _within(name, got[b:b + 1], exact, t, more)
