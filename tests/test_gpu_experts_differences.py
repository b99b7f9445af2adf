"""Gradients of the way to the experts, their products and the way back against differences, token by token and expert by expert.  Results are linear in every operand, so a step
of any width gives the gradient times the step; each difference is held to the terms that it is made of."""

import pytest
import torch

from distdl_amd import nn

pytestmark = pytest.mark.gpu

U, OUT = 2.0 ** -24, 24
CASES = [(1, 1, 1, None, 3), (37, 3, 5, (1, 4), 65), (300, 2, 8, None, 128), (64, 4, 6, (0, 5), 512)]


class Problem:

    def __init__(self, tokens, chosen, experts, window, cols):
        g = torch.Generator().manual_seed(tokens + cols)
        self.ids = torch.randint(0, experts, (tokens, chosen), generator=g).cuda()
        self.plan = nn.expert_plan(self.ids, experts, window=window)
        self.low, self.held = self.plan.window[0], len(self.plan.offsets) - 1
        self.rows = self.plan.offsets.diff().tolist()
        self.x, self.w, self.weights = (torch.randn(*s, generator=g).cuda() for s in ((tokens, cols), (self.held, OUT, cols), (tokens, chosen)))
        self.dout = torch.randn(tokens, OUT, generator=g).cuda()
        self.g, self.depth = g, cols + chosen + 8        # roundings of a result: a product's terms, the choices, and each factor's own
        leaves = [t.clone().requires_grad_() for t in (self.x, self.w, self.weights)]
        self.grads = torch.autograd.grad(self.run(*leaves), leaves, self.dout)

    def run(self, x, w, weights):
        return nn.expert_combine(nn.expert_linear_shard(nn.expert_sort(x, self.plan), w, self.plan.offsets), self.plan, weights)

    def by_token(self, x, w, weights):
        """``sum(out * dout)`` of each token, and the sizes of its terms."""
        out, sizes = self.run(x, w, weights), self.run(x.abs(), w.abs(), weights.abs())
        return (out.double() * self.dout).sum(-1), (sizes.double() * self.dout.abs()).sum(-1)

    def step(self, t, along):
        """``t`` some way on, and the way as the sum was rounded; with ``along`` where the gradient points, so that the difference is large next to its terms: a gradient
        that is off by some hundredths of itself, or lacks an expert's part, shows."""
        way = torch.randn(t.shape, generator=self.g).cuda()
        far = t + (way if along is None else way.abs() * along.sign())
        return far, far.double() - t.double()


def close(change, slope, near, far, grad, results_depth, grad_depth):
    """Two results, each off by its roundings' share of its terms; the gradient as well."""
    assert ((change - slope).abs() <= 2 * U * (results_depth * (near + far) + grad_depth * grad) + 1e-30).all()


@pytest.mark.parametrize("case", CASES, ids=[f"{t}x{c}of{e}-{k}" for t, c, e, _, k in CASES])
@pytest.mark.parametrize("uphill", [False, True], ids=["anywhere", "uphill"])
def test_each_token(case, uphill):
    p = Problem(*case)
    base, near = p.by_token(p.x, p.w, p.weights)
    far_x, moved = p.step(p.x, p.grads[0] if uphill else None)
    value, far = p.by_token(far_x, p.w, p.weights)
    terms = p.by_token(moved.float(), p.w, p.weights)[1]
    close(value - base, (p.grads[0].double() * moved).sum(-1), near, far, terms, p.depth, p.depth + OUT)
    far_weights, moved = p.step(p.weights, p.grads[2] if uphill else None)
    value, far = p.by_token(p.x, p.w, far_weights)
    terms = p.by_token(p.x, p.w, moved.float())[1]
    close(value - base, (p.grads[2].double() * moved).sum(-1), near, far, terms, p.depth, p.depth + OUT)


@pytest.mark.parametrize("case", CASES, ids=[f"{t}x{c}of{e}-{k}" for t, c, e, _, k in CASES])
@pytest.mark.parametrize("uphill", [False, True], ids=["anywhere", "uphill"])
def test_each_expert(case, uphill):
    p = Problem(*case)
    base, near = p.by_token(p.x, p.w, p.weights)
    for e in range(p.held):
        far_w = p.w.clone()
        far_w[e], moved = p.step(p.w[e], p.grads[1][e] if uphill else None)
        value, far = p.by_token(p.x, far_w, p.weights)
        theirs = (p.ids == p.low + e).any(-1)
        assert torch.equal(value[~theirs], base[~theirs])
        alone = torch.zeros_like(p.w)
        alone[e] = moved.float()
        terms = p.by_token(p.x, alone, p.weights)[1].sum()
        change = (value - base).sum()
        close(change, (p.grads[1][e].double() * moved).sum(), near[theirs].sum(), far[theirs].sum(), terms, p.depth, p.depth + p.rows[e])
