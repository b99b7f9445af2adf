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
