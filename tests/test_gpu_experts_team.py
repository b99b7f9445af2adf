"""An experts' block over workers through the framework's own moves: tokens and the router's weights broadcast, each worker's experts, what came of them summed up, and
the gradients through the moves' adjoints.  Whole numbers, so that no order of sums matters: results and gradients are those of one worker, to the bit."""

import pytest
import torch

from distdl_amd import nn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("workers,experts,tokens,chosen", [(3, 7, 70, 3), (2, 16, 300, 2), (4, 3, 9, 1)])
def test_from_tokens_to_tokens(workers, experts, tokens, chosen, dtype):
    from distdl_amd.backends.stub_hip import SimWorld
    from distdl_amd.utilities.torch import zero_volume_tensor
    cols, out = 40, 24
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts, (tokens, chosen), generator=g)
    x, dy, w = (torch.randint(-1, 2, s, generator=g).to(dtype) for s in ((tokens, cols), (tokens, out), (experts, out, cols)))
    weights = torch.randint(1, 3, (tokens, chosen), generator=g).float()

    def body(P_world, count):
        team = P_world.create_partition_inclusive(list(range(count))).create_cartesian_topology_partition([count, 1])
        root = P_world.create_partition_inclusive([0]).create_cartesian_topology_partition([1, 1])
        layer = nn.DistributedExpertLinear(team, experts, cols, out, dtype=dtype)
        with torch.no_grad():
            layer.weight.copy_(w[slice(*layer.window)])

        def held(t):
            return (t.cuda() if root.active else zero_volume_tensor(dtype=t.dtype, device="cuda")).requires_grad_()

        a, share = held(x), held(weights)
        to_all, to_root = nn.Broadcast(root, team, preserve_batch=False), nn.SumReduce(team, root, preserve_batch=False)
        here, weights_here = to_all(a), nn.Broadcast(root, team, preserve_batch=False)(share)
        plan = nn.expert_plan(ids.cuda(), experts, window=layer.window)
        y = to_root(nn.expert_combine(layer(nn.expert_sort(here, plan), plan), plan, weights_here))
        y.backward(dy.cuda() if root.active else zero_volume_tensor(dtype=dtype, device="cuda"))
        torch.cuda.synchronize()
        return [t.detach().cpu() for t in (y, a.grad, share.grad, layer.weight.grad)]

    (whole,) = SimWorld(1).run(lambda P: body(P, 1))
    parts = SimWorld(workers).run(lambda P: body(P, workers))
    held = (ids >= 0).float() * weights
    chosen_w = w.float()[ids.clamp(min=0)]
    want = torch.einsum("tj,tjoc,tc->to", held, chosen_w, x.float())
    assert torch.equal(whole[0].float(), want)
    for i in range(3):
        assert torch.equal(parts[0][i], whole[i])
    assert torch.equal(torch.cat([p[3] for p in parts]), whole[3])
    assert whole[1].any() and whole[2].any() and whole[3].any()
