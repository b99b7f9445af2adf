"""Attention with scores that leave no digits for a difference."""

import pytest
import torch

pytestmark = pytest.mark.gpu


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
