"""What the experts' operators promise beside their values: native and general paths alike, gradients of any form, streams and threads, passes that torch records,
experts that do not see each other's rows, sequences beyond 32 bits."""

import threading

import numpy as np
import pytest
import torch

from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import experts as o

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _operators(dt=torch.bfloat16):
    """Name: (call of the leaves, leaves, gradients of the results)."""
    g = torch.Generator().manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(dt).cuda()

    ids = torch.randint(-1, 6, (30, 3), generator=g).cuda()
    plan = nn.expert_plan(ids, 6, window=(1, 6))
    weights = torch.rand(30, 3, generator=g).cuda()
    return {
        "norm": (lambda x, w: nn.rms_norm_shard(x, w), [normal(20, 64), normal(64)], [normal(20, 64)]),
        "norm_plain": (lambda x: nn.rms_norm_shard(x), [normal(20, 64)], [normal(20, 64)]),
        "norm_residual": (lambda x, w, r: nn.rms_norm_shard(x, w, r, eps=1e-5), [normal(4, 5, 64), normal(64), normal(4, 5, 64)], [normal(4, 5, 64), normal(4, 5, 64)]),
        "norm_residual_plain": (lambda x, r: nn.rms_norm_shard(x, None, r), [normal(20, 64), normal(20, 64)], [normal(20, 64), normal(20, 64)]),
        "sort": (lambda x: nn.expert_sort(x, plan), [normal(30, 40)], [normal(90, 40)]),
        "combine": (lambda y, w: nn.expert_combine(y, plan, w), [normal(90, 40), weights], [normal(30, 40)]),
        "combine_ones": (lambda y: nn.expert_combine(y, plan), [normal(90, 40)], [normal(30, 40)]),
        "linear": (lambda x, w: nn.expert_linear_shard(x, w, plan.offsets), [normal(90, 48), normal(5, 32, 48)], [normal(90, 32)]),
    }


NAMES = ["norm", "norm_plain", "norm_residual", "norm_residual_plain", "sort", "combine", "combine_ones", "linear"]


def _listed(out):
    return list(out) if isinstance(out, tuple) else [out]


def _passes(name, seed):
    """All results with their gradients; each result alone; one leaf at a time."""
    call, operands, dys = _operators()[name]
    leaves = [t.detach().clone().requires_grad_() for t in operands]
    out = _listed(call(*leaves))
    dys = [seed * dy for dy in dys]
    passes = [[t.detach() for t in out], torch.autograd.grad(out, leaves, dys, retain_graph=True)]
    passes += [torch.autograd.grad([t], leaves, [dy], retain_graph=True, allow_unused=True) for t, dy in zip(out, dys)]
    passes += [torch.autograd.grad(out, [leaf], dys, retain_graph=True) for leaf in leaves]
    torch.autograd.backward(out, dys)
    return passes + [[leaf.grad for leaf in leaves]]


def _same(got, want):
    for x, y in zip(got, want):
        assert len(x) == len(y)
        for s, t in zip(x, y):
            assert (s is None or not s.any()) if t is None else (torch.equal(s, t) if s is not None else not t.any())


@pytest.mark.parametrize("name", NAMES)
def test_native_and_general_paths_agree(name, monkeypatch):
    from distdl_amd import _lib
    want = _passes(name, 1)

    class General:
        def __getattr__(self, _):
            return lambda *a: None

    monkeypatch.setattr(_lib, "front", General)
    _same(_passes(name, 1), want)


@pytest.mark.parametrize("name", NAMES)
def test_compiled_autograd_gives_the_bits_of_an_ordinary_pass(name):
    from torch._dynamo import compiled_autograd
    want = [_passes(name, seed) for seed in (1, 2)]
    with compiled_autograd._enable(lambda graph: graph):
        got = [_passes(name, seed) for seed in (1, 2)]
    for a, b in zip(got, want):
        _same(a, b)


@pytest.mark.parametrize("general", [False, True], ids=["native", "general"])
@pytest.mark.parametrize("name", NAMES)
def test_adjoints_have_no_derivative_and_say_so(name, general, monkeypatch):
    from distdl_amd import _lib
    if general:
        class General:
            def __getattr__(self, _):
                return lambda *a: None
        monkeypatch.setattr(_lib, "front", General)
    call, operands, dys = _operators(torch.float32)[name]
    leaves = [t.detach().clone().requires_grad_() for t in operands]
    grads = torch.autograd.grad(_listed(call(*leaves)), leaves, [d.requires_grad_() for d in dys], create_graph=True)
    for grad in grads:
        with pytest.raises(RuntimeError, match="twice|once_differentiable"):
            grad.float().sum().backward()


@pytest.mark.parametrize("name", NAMES)
def test_gradients_of_any_form(name):
    """Expanded (of a sum), strided, and of a result that was cast."""
    call, operands, _ = _operators()[name]
    leaves = [t.detach().clone().requires_grad_() for t in operands]
    out = _listed(call(*leaves))
    whole = torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out], retain_graph=True)
    expanded = torch.autograd.grad(sum(t.sum() for t in out), leaves, retain_graph=True)
    strided = torch.autograd.grad(out, leaves, [torch.ones(t.shape[:-1] + (2 * t.shape[-1],), dtype=t.dtype, device="cuda")[..., ::2] for t in out], retain_graph=True)
    cast = torch.autograd.grad([t.float() for t in out], leaves, [torch.ones_like(t, dtype=torch.float32) for t in out])
    for other in (expanded, strided, cast):
        assert all(torch.equal(a, b) for a, b in zip(whole, other))


def test_a_changed_operand_is_noticed():
    x, r = torch.randn(4, 64, device="cuda", requires_grad=True), torch.randn(4, 64, device="cuda")
    y, h = nn.rms_norm_shard(x, None, r)
    with torch.no_grad():
        h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_streams_and_threads():
    """Two threads on streams of their own, each with its own operands, give what one gives alone."""
    def work(seed, out):
        g = torch.Generator().manual_seed(seed)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            x = torch.randn(500, 256, generator=g).cuda().requires_grad_()
            w = torch.randn(8, 64, 256, generator=g).cuda().requires_grad_()
            ids, weights = torch.randint(0, 8, (500, 4), generator=g).cuda(), torch.rand(500, 4, generator=g).cuda()
            dy = torch.randn(500, 64, generator=g).cuda()
            for _ in range(5):
                plan = nn.expert_plan(ids, 8)
                h = nn.rms_norm_shard(x)
                y = nn.expert_combine(nn.expert_linear_shard(nn.expert_sort(h, plan), w, plan.offsets), plan, weights)
                grads = torch.autograd.grad(y, [x, w], dy)
            stream.synchronize()
            out[seed] = [y.detach()] + list(grads)

    alone, both = {}, {}
    for seed in (1, 2):
        work(seed, alone)
    threads = [threading.Thread(target=work, args=(seed, both)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(alone[seed], both[seed]))


def test_a_training_step_captured_next_to_eager_ones():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(300, 128, generator=g).to(torch.bfloat16).cuda()
    w = torch.randn(4, 64, 128, generator=g).to(torch.bfloat16).cuda()
    nw = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    ids, weights = torch.randint(0, 4, (300, 2), generator=g).cuda(), torch.rand(300, 2, generator=g).cuda()
    dy = torch.randn(300, 64, generator=g).to(torch.bfloat16).cuda()

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, nw, weights)]
        plan = nn.expert_plan(ids, 4)
        rows = nn.expert_sort(nn.rms_norm_shard(leaves[0], leaves[2]), plan)
        y = nn.expert_combine(nn.expert_linear_shard(rows, leaves[1], plan.offsets), plan, leaves[3])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(4):
        ids.copy_(torch.randint(-1, 4, (300, 2), generator=torch.Generator().manual_seed(seed)))
        x.copy_(torch.randn(300, 128, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step()))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("counts,k,n", [([3, 5, 2], 64, 32), ([3, 5, 2], 65, 33), ([70, 100, 30], 256, 512), ([130, 200, 129], 264, 1032), ([130, 200, 129], 261, 1031),
                                        ([700, 300, 600], 1024, 1024)])
def test_experts_do_not_see_each_others_rows(dt, counts, k, n):
    """One expert's rows, gradients and weights hold no numbers: the others' results and gradients are what they are without."""
    g = torch.Generator().manual_seed(k)
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    x, w, dy = (torch.randn(*s, generator=g).to(dt).cuda() for s in ((sum(counts), k), (3, n, k), (sum(counts), n)))
    clean = [hip_ops.expert_linear(x, w, offsets), *hip_ops.expert_linear_backward(dy, x, w, offsets)]
    mid = slice(counts[0], counts[0] + counts[1])
    x[mid], dy[mid], w[1] = float("nan"), float("inf"), float("nan")
    got = [hip_ops.expert_linear(x, w, offsets), *hip_ops.expert_linear_backward(dy, x, w, offsets)]
    for rows in (slice(0, mid.start), slice(mid.stop, None)):
        assert torch.equal(got[0][rows], clean[0][rows]) and torch.equal(got[1][rows], clean[1][rows])
    assert torch.equal(got[2][0], clean[2][0]) and torch.equal(got[2][2], clean[2][2])
    assert got[0][mid].isnan().all() and got[2][1].isnan().all()


@pytest.mark.parametrize("dt", DTYPES)
def test_no_experts_no_rows_no_columns_held(dt):
    x = torch.ones(5, 16, dtype=dt, device="cuda", requires_grad=True)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.zeros(0, 8, 16, dtype=dt, device="cuda", requires_grad=True)
    y = nn.expert_linear_shard(x, w, none)
    assert y.shape == (5, 8) and (y == 0).all()
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert (dx == 0).all() and dw.shape == w.shape
    w = torch.ones(3, 8, 16, dtype=dt, device="cuda", requires_grad=True)
    y = nn.expert_linear_shard(x[:0], w, torch.zeros(4, dtype=torch.int32, device="cuda"))
    (dw,) = torch.autograd.grad(y, [w], torch.ones_like(y))
    assert y.shape == (0, 8) and (dw == 0).all()
    plan = nn.expert_plan(torch.zeros(5, 2, dtype=torch.int32, device="cuda"), 4, window=(2, 4))
    assert plan.offsets.tolist() == [0, 0, 0] and (nn.expert_sort(x.detach(), plan) == 0).all()
    assert (nn.expert_combine(torch.full((10, 16), float("nan"), dtype=dt, device="cuda"), plan) == 0).all()
    codes = x.detach().to(torch.float8_e4m3fn)
    ones = torch.ones(5, device="cuda")
    y = nn.expert_linear_shard(codes, codes[:0].view(0, 1, 16), none, x_scales=ones, weight_scales=torch.zeros(0, 1, device="cuda"))
    assert (y == 0).all()


def test_plans_of_other_tensors_stay_inside():
    """Places that name no row move nothing: what lies around the result is left as it was."""
    place = torch.tensor([[0, 2 ** 31 - 1], [-5, 3], [2, 1]], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    x = torch.arange(1.0, 4.0, device="cuda")[:, None].expand(3, 8).contiguous()
    room = torch.full((8, 8), 7.0, device="cuda")
    from distdl_amd import _lib
    held = offsets.data_ptr() + 4
    _lib.check(_lib.load().ddl_expert_sort(x.data_ptr(), 4, 3, 2, 8, 8, place.data_ptr(), held, room[1:].data_ptr(), None, None, hip_ops._stream()), "sort")
    assert room[:, 0].tolist() == [7, 1, 3, 3, 2, 7, 7, 7]
    assert nn.expert_combine(torch.ones(6, 8, device="cuda"), nn.ExpertPlan(place, offsets, (0, 1)))[:, 0].tolist() == [1, 1, 2]
    dy, dw = hip_ops.expert_combine_backward(x, torch.ones(6, 8, device="cuda"), place, offsets, torch.ones(3, 2, device="cuda"))
    assert dw.tolist() == [[8, 0], [0, 16], [24, 24]] and dy[:4, 0].tolist() == [1, 3, 3, 2]


@pytest.mark.parametrize("what", ["norm", "sort", "sort8", "linear"])
def test_more_than_32_bits_of_elements(what):
    """Rows beyond 2^32 bytes and 2^31 elements: the last ones are what they are alone."""
    if what == "norm":
        x = torch.zeros(300000, 8192, dtype=torch.bfloat16, device="cuda")
        tail = torch.randn(3, 8192, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
        x[-3:] = tail
        y = nn.rms_norm_shard(x)
        assert torch.equal(y[-3:], nn.rms_norm_shard(tail)) and (y[:-3] == 0).all()
        dx = hip_ops.rms_norm_backward(x, x, want_weight=False)[0]
        assert torch.equal(dx[-3:], hip_ops.rms_norm_backward(tail, tail, want_weight=False)[0])
    elif what.startswith("sort"):
        dt = torch.bfloat16 if what == "sort" else torch.float8_e4m3fn
        ids = torch.arange(8, device="cuda").expand(70000, 8)
        x = torch.randn(70000, 8192, device="cuda").to(dt)
        plan = nn.expert_plan(ids, 8)
        rows = nn.expert_sort(x, plan) if what == "sort" else nn.expert_sort(x, plan, torch.ones(70000, device="cuda"))[0]
        bits = torch.int16 if what == "sort" else torch.uint8
        for e in (0, 3, 7):
            assert torch.equal(rows[70000 * e:70000 * (e + 1)].view(bits), x.view(bits))
        if what == "sort":
            back = nn.expert_combine(rows, plan, torch.full((70000, 8), 0.125, device="cuda"))
            assert torch.equal(back, x)
            dy, dw = hip_ops.expert_combine_backward(x, rows, plan.place, plan.offsets, torch.ones(70000, 8, device="cuda"))
            assert torch.equal(dy[70000 * 7:], x) and torch.equal(dw[:, 0], dw[:, 7])
    else:
        x = torch.randn(280000, 8192, device="cuda").to(torch.bfloat16)
        w = torch.randn(2, 8, 8192, device="cuda").to(torch.bfloat16)
        offsets = torch.tensor([0, 100, 280000], dtype=torch.int32, device="cuda")
        y = nn.expert_linear_shard(x, w, offsets)
        want = o.product(x[-50:].double().cpu().numpy(), w[1:].double().cpu().numpy(), [0, 50])
        np.testing.assert_allclose(y[-50:].double().cpu().numpy(), want, rtol=2 ** -8, atol=2 ** -6)
        dx, dw = hip_ops.expert_linear_backward(y, x, w, offsets)
        want = y[-50:].double() @ w[1].double()
        assert ((dx[-50:].double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -4).all()
        want = y[100:].t().float() @ x[100:].float()
        assert ((dw[1].float() - want).abs() <= 2 ** -6 * want.abs() + 1e-3 * want.abs().max()).all()


@pytest.mark.parametrize("counts,k,n", [([3, 5, 2], 64, 33), ([20, 60, 21], 272, 96), ([130, 200, 129], 1040, 1032), ([700, 300, 600], 2048, 4100), ([1400, 900, 1300], 528, 4096)])
def test_experts_do_not_see_each_others_rows_in_8_bits(counts, k, n):
    """As above, for codes and scales, by the kernel for few rows, the small and the large tiles."""
    g = torch.Generator().manual_seed(k)
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    x, w = (torch.randn(*s, generator=g).to(torch.float8_e4m3fn).cuda() for s in ((sum(counts), k), (3, n, k)))
    xs, ws = torch.rand(sum(counts), generator=g).cuda(), torch.rand(3, n, generator=g).cuda()
    clean = nn.expert_linear_shard(x, w, offsets, x_scales=xs, weight_scales=ws)
    mid = slice(counts[0], counts[0] + counts[1])
    x.view(torch.uint8)[mid], xs[mid], w.view(torch.uint8)[1], ws[1] = 0x7F, float("inf"), 0xFF, float("nan")
    got = nn.expert_linear_shard(x, w, offsets, x_scales=xs, weight_scales=ws)
    assert torch.equal(got[:mid.start], clean[:mid.start]) and torch.equal(got[mid.stop:], clean[mid.stop:]) and got[mid].isnan().all()


def test_rows_in_8_bits_captured_with_other_choices_each_time():
    """A prompt's rows and single tokens, from the norm to the products, replayed for choices that change which experts have rows."""
    g = torch.Generator().manual_seed(8)
    w8, ws = nn.quantize_rows(torch.randn(6, 264, 512, generator=g).to(torch.bfloat16).cuda())
    for tokens in (3, 700):
        x, r = (torch.randn(tokens, 512, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        ids = torch.randint(0, 6, (tokens, 2), generator=g).cuda()

        @torch.no_grad()
        def step():
            codes, scales, h = nn.rms_norm_shard(x, None, r, eight_bit=True)
            plan = nn.expert_plan(ids, 6, window=(0, 6))
            rows, row_scales = nn.expert_sort(codes, plan, scales)
            return h, nn.expert_combine(nn.expert_linear_shard(rows, w8, plan.offsets, x_scales=row_scales, weight_scales=ws), plan)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for low, high in ((0, 6), (2, 3), (-1, 6), (-1, 0), (4, 6)):
            ids.copy_(torch.randint(low, high, (tokens, 2), generator=g))
            x.copy_(torch.randn(tokens, 512, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, step()))
