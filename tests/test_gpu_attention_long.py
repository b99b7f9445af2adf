"""Attention where offsets within one sequence pass 32 bits, and captured with operands that have to be laid out first."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,heads", [(torch.bfloat16, 8), (torch.float32, 16)])
@pytest.mark.parametrize("tokens", [1, 3, 1100])
def test_one_sequence_beyond_32_bits(dt, heads, tokens):
    """More than 2^31 elements (fp32: 2^32) from the first key to the last: scores are zero but for 4 keys at either end, which are what a query sees; their
    mean is exact.  Of gradients, a probability is off by the rounding of scores and sums near 289 (in powers of two; 2^-16 each, ln 2 of it: 2^-15.5 together),
    and so is D, by that of at most 28: dS by 2^-15.5 of (28 + 28) / 8 = 7.  (bf16 rounds both to what they are.)"""
    from distdl_amd import nn
    dim, keys = 128, (1 << 21) + 77
    k, v = (torch.zeros(1, keys, heads, dim, dtype=dt, device="cuda") for _ in range(2))
    assert k.numel() > 1 << 31
    q, dy = (torch.zeros(1, tokens, heads, dim, dtype=dt, device="cuda") for _ in range(2))
    ends = [*range(4), *range(keys - 4, keys)]
    q[..., 5] = 1.0
    k[:, ends, :, 5] = 200.0      # (2^-288 of their weight is left for the others)
    v[:, ends] = torch.arange(8.0, device="cuda").to(dt)[None, :, None, None] * 8
    dy[:, tokens - 1, heads - 1, 7] = 1.0
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = nn.attention_shard(*leaves, scale=1.0)
    assert (out == 28.0).all()
    dq, dk, dv = torch.autograd.grad(out, leaves, dy)
    assert not dv[:, 4:keys - 4].any() and not dk[:, 4:keys - 4].any()
    want = torch.zeros(heads, dim, dtype=dt, device="cuda")
    want[heads - 1, 7] = 0.125
    off = 2.0 ** -15 if dt == torch.float32 else 0.0
    assert ((dv[0, ends] - want).abs() <= off * want).all()
    want[heads - 1, 7], want[heads - 1, 5] = 0, 1
    assert ((dk[0, ends] - torch.arange(-28.0, 29, 8, device="cuda").to(dt)[:, None, None] / 8 * want).abs() <= 7 * off * want).all()
    assert (dq.abs() <= 8 * 200 * 7 * off).all()


@pytest.mark.parametrize("tokens,keys,dim", [(1, 1500, 100), (70, 90, 33)])
def test_heads_that_are_laid_out_first_replay_from_a_graph(tokens, keys, dim):
    """Heads that are no multiple of 16 bytes, lengths with a stride: forward and adjoint captured together, replayed with eager calls between."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(dim)
    q, k, v, dy = (torch.randn(3, n, h, dim, generator=g).to(torch.bfloat16).cuda() for n, h in ((tokens, 4), (keys, 2), (keys, 2), (tokens, 4)))
    every = torch.tensor([keys, 0, 7, 0, keys // 2, 0], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step(lengths):
        out = nn.attention_shard(*leaves, lengths, causal=True, own_ends=True)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, dy))

    packed = every[::2].contiguous()
    assert all(torch.equal(a, b) for a, b in zip(step(packed), step(every[::2])))
    for lengths in (packed, every[::2]):
        step(lengths)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step(lengths)
        for i in range(3):
            with torch.no_grad():
                k.copy_(torch.randn(k.shape, generator=g).to(k.dtype))
                lengths[1] = 3 * i
            want = step(lengths)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, want))
