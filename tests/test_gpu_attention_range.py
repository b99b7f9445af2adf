"""Attention where a type's range ends: in float16 with probabilities and gradients of which float16 itself would keep little (many keys, one of which has
most of the weight, and gradients far below or above one), and with scores that leave no digits for a difference.

Tolerances: half a step of the type, u = 2^-11 of the value, for the rounding of a result, of a probability and of its gradient; what lies below the
type's normal numbers costs a result 2^-25 as well, but no sum before it.  Scores are sums of one product here, so a probability is off by c = 2^-18 beside
its rounding: of an exponential and a logarithm in 32 bits, 2^-21 each with arguments below 2^5 (2^-24 of them, times 2^5 ln 2), and of totals whose
terms are equal but for one of them (sums of integers up to 2^24, exact; n 2^-24 <= 2^-11 of the rest next to a large one: c = 2^-10 there).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U, TINY, C = 2.0 ** -11, 2.0 ** -25, 2.0 ** -18


@pytest.mark.parametrize("keys", [300, 8192])
@pytest.mark.parametrize("batch,tokens,heads", [(1, 1, 1), (2, 5, 4), (96, 130, 8)])
@pytest.mark.parametrize("below", [14.25, 18.25, 21.25, 23.25])
@pytest.mark.parametrize("dim", [32, 128])
def test_keys_far_below_one_of_large_weight(keys, batch, tokens, heads, below, dim):
    """One key with value 0 has 2^below times the weight of every other, whose values are about one: the result is theirs alone.

    Their probability is rounded by u of itself, the sum of the rounded ones by as much, and so is the result.  (The scores are 0.5 and below + 0.5
    in powers of two: none of the probabilities is a whole one.)"""
    from distdl_amd import nn
    q = torch.zeros(batch, tokens, heads, dim, dtype=torch.float16, device="cuda")
    k, v = (torch.zeros(batch, keys, 1, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    q[..., 0], k[:, keys // 3, :, 0] = 1.0, below
    q[..., 1], k[..., 1] = 0.5, 1.0
    v.copy_(torch.rand(v.shape, generator=torch.Generator().manual_seed(keys)) + 0.5)
    v[:, keys // 3] = 0.0
    out = nn.attention_shard(q, k, v, scale=0.6931471805599453).double()
    weight = 2.0 ** -below
    want = (weight * v.double().sum(1, keepdim=True) / (1 + (keys - 1) * weight)).expand(out.shape)
    tol = 3 * U * want + 2 * 2.0 ** -10 * want + TINY
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / want).max()


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("tokens,keys,heads", [(5, 60, 2), (1, 700, 4), (130, 700, 2), (70, 8192, 2), (700, 3001, 1)])
@pytest.mark.parametrize("gradient,value", [(2.0 ** -14, 1.0), (2.0 ** -8, 2.0 ** -6), (2.0 ** -8, 1.0), (1.0, 1.0), (2.0 ** 14, 2.0 ** 14)])
def test_gradients_far_from_one(gradient, value, tokens, keys, heads, dim):
    """Half of the keys have a value, scores are zero: dS = +- g value / 2 keys for each of them, from 2^-32 to 2^21, and dq and dk are sums of equal signs.

    dS is rounded by u; its p is off by c, and D, the mean of the values times g, by 2^-20 of dP - D (the mean is rounded twice in 32 bits, the rest that is kept
    of it by u^2 of the value); the sums of n terms by n 2^-24; results by u."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(keys + tokens)
    q, dy = (torch.zeros(1, tokens, heads, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    k, v = (torch.zeros(1, keys, 1, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    with_value = (torch.randperm(keys, generator=g) < keys // 2).cuda()
    q[..., 0] = 1.0
    k[:, with_value, :, 1], v[:, with_value, :, 2] = 1.0, value
    dy[..., 2] = gradient * (1 + torch.rand(1, tokens, heads, generator=g).cuda())
    scale = 4 / (gradient * value)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(nn.attention_shard(*leaves, scale=scale), leaves, dy)
    size, share = dy[..., 2].double() * value, (keys // 2) / keys
    want_q = scale * size * share * (1 - share)
    want_k = torch.where(with_value, 1 - share, -share) * scale * size.sum() / keys
    off = 2 * U + C + 2.0 ** -20
    assert ((dq[..., 1].double() - want_q).abs() <= (off + keys * 2.0 ** -24) * want_q).all(), (dq[..., 1].double() / want_q - 1).abs().max()
    assert ((dk[0, :, 0, 0].double() - want_k).abs() <= (off + tokens * heads * 2.0 ** -24) * want_k.abs() + TINY).all(), (dk[0, :, 0, 0].double() / want_k - 1).abs().max()
    dq[..., 1], dk[..., 0] = 0, 0
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("batch,tokens,keys,heads,causal", [(2, 9, 60, 2, False), (1, 150, 900, 2, False), (1, 300, 300, 4, True), (3, 200, 70, 2, True)])
@pytest.mark.parametrize("rise", [-20, 0, 20])
def test_gradients_that_rise_and_fall_along_keys_and_queries(rise, batch, tokens, keys, heads, causal, dim):
    """Values that change by 2^rise along the keys and gradients that do along the queries: bounds of the general test without what float16 loses next to zero,
    but for 2^-34 of the largest dS of a query or key and for 2^-25 of what is kept of the result's rounding, and of a gradient."""
    from distdl_amd import nn
    from oracle import heads as o_heads
    from test_gpu_attention import _bounds
    g = torch.Generator().manual_seed(tokens + keys)

    def normal(n, h, rises, scale=1.0):
        t = torch.randn(batch, n, h, dim, generator=g) * scale
        return (t * 2.0 ** (rises * (torch.arange(n) / n - 0.5))[:, None, None] if rises else t).half().cuda()

    q, k, v, dy = normal(tokens, heads, 0), normal(keys, 1, 0), normal(keys, 1, rise), normal(tokens, heads, rise, 2.0 ** -4)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    scale = dim ** -0.5
    grads = torch.autograd.grad(nn.attention_shard(*leaves, causal=causal), leaves, dy)
    qn, kn, vn, dyn = (t.detach().double().cpu().numpy() for t in (q, k, v, dy))
    want = o_heads.attention(qn, kn, vn, None, causal, scale, dyn)[2:]
    tol = _bounds(qn, kn, vn, None, causal, scale, U, 0.0, dyn)[1:]
    p, ds, lost = _parts(qn, kn, vn, dyn, causal, scale)
    more_q = torch.einsum("bhij,bjd->bihd", lost + 2.0 ** -34 * ds.abs().amax(-1, keepdim=True), torch.from_numpy(abs(kn[:, :, 0])))
    more_k = torch.einsum("bhij,bihd->bjd", lost + 2.0 ** -34 * ds.abs().amax((1, 2), keepdim=True), torch.from_numpy(abs(qn)))[:, :, None]
    for name, got, exact, bound, more in (("dq", grads[0], want[0], tol[0], more_q), ("dk", grads[1], want[1], tol[1], more_k)):
        got, exact = got.double().cpu(), torch.from_numpy(exact)
        bound = torch.from_numpy(bound) + scale * more + U * exact.abs() + TINY
        # (a gradient itself may leave the type: from 65520 on it rounds to infinity, and may do so as far below as it may be off)
        beyond = torch.where(exact.abs() + bound >= 65520, got == exact.sign() * torch.inf, False)
        near = (got - exact).abs() <= bound
        assert (near | beyond).all(), f"{name}: {((got - exact).abs() / bound)[~beyond].max():.3g} of the tolerance"
        assert beyond.sum() < 0.05 * beyond.numel()


def _parts(q, k, v, dy, causal, scale):
    """In 64 bits, [batch, heads, tokens, keys]: probabilities, their gradients dS, and what 2^-25 of every element of the result makes of dS."""
    q, k, v, dy = (torch.from_numpy(t) for t in (q, k, v, dy))
    s = scale * torch.einsum("bihd,bjd->bhij", q, k[:, :, 0])
    hidden = torch.arange(k.shape[1]) > torch.arange(q.shape[1])[:, None] + k.shape[1] - q.shape[1] if causal else torch.zeros(q.shape[1], k.shape[1], dtype=torch.bool)
    p = s.masked_fill(hidden, -torch.inf).softmax(-1).nan_to_num(0.0)
    dp = torch.einsum("bihd,bjd->bhij", dy, v[:, :, 0])
    return p, p * (dp - (p * dp).sum(-1, keepdim=True)), p * TINY * dy.abs().sum(-1).transpose(1, 2)[..., None]


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("tokens,keys", [(3, 1000001), (130, 330011)])
def test_gradients_of_values_of_very_many_keys(tokens, keys, dim):
    """Scores of zero: every probability is 1 / keys, rounded by u, and off by 2^-18 of it (the logarithm's argument and the exponential's, below 2^5, by 2^-19 and
    2^-20 together; the total is a sum of ones, exact).  So dv = sum dy / keys is off by u and 2^-18 of the magnitudes, the sum's
    tokens 2^-24 of them, and u and 2^-25 for the result."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(keys)
    q, dy = (torch.randn(1, tokens, 1, dim, generator=g).half().cuda() for _ in range(2))
    dy = dy * 256
    k, v = (torch.zeros(1, keys, 1, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    v.requires_grad_()
    dv, = torch.autograd.grad(nn.attention_shard(q, k, v), [v], dy)
    want, size = dy.double().sum(1, keepdim=True) / keys, dy.double().abs().sum(1, keepdim=True) / keys
    tol = (U + C + tokens * 2.0 ** -24) * size + U * want.abs() + TINY
    assert ((dv.double() - want).abs() <= tol).all(), ((dv.double() - want).abs() / tol).max()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,tokens,heads,keys", [(1, 1, 1, 40), (1, 70, 2, 1000), (160, 130, 1, 100)])
@pytest.mark.parametrize("power", [18, 24, 26, 27, 28, 32, 36, 60])
def test_huge_scores_of_which_the_largest_takes_all(dt, batch, tokens, heads, keys, power):
    """Scores of about 2^power in powers of two, a sixteenth apart and more: every probability but those of the largest one, which two keys share, is zero.
    Their two products with the values, the sum of them, the quotient and its product are each off by 2^-24 of at most the mean of the magnitudes (a sum by
    twice that): 2^-21 with room for a second unit of the quotient.  The 16-bit types hold the mean itself."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(power)
    q, k, v = (torch.zeros(batch, n, h, 64, dtype=dt, device="cuda") for n, h in ((tokens, heads), (keys, 1), (keys, 1)))
    sign = torch.randint(0, 2, (tokens, heads), generator=g).cuda() * 2 - 1
    q[..., :3] = sign[..., None].to(dt) * torch.tensor([960.0, 37.0, 3.0], dtype=dt, device="cuda")      # (their products have 20 digits, with the scale some 44)
    part = torch.randint(-12, 13, (keys,), generator=g) / 16
    part[keys // 2] = part[keys - 1] = 1.0
    part[3] = part[keys // 3] = -1.0
    k[..., 0, :3] = (part[:, None] * torch.tensor([960.0, 53.0, 5.0])).to(dt).cuda()
    v.copy_(torch.randint(-64, 64, v.shape, generator=g))
    out = nn.attention_shard(q, k, v, scale=2.0 ** (power - 20) * 0.69).float()
    first, second = (torch.where((sign > 0)[None, :, :, None], v[:, i, None].float(), v[:, j, None].float()) for i, j in ((keys // 2, 3), (keys - 1, keys // 3)))
    assert ((out - (first + second) / 2).abs() <= 2.0 ** -21 * (first.abs() + second.abs()) / 2).all()
