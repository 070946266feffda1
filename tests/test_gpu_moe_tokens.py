"""Sorting tokens by expert and combining the experts' rows, with gradients,
against their definitions in 64 bits on the CPU.

Tolerances: an fp32 sum of n products is within (n + 1) 2^-24 of the sum of their
magnitudes (two roundings a term at most, fused or not: 2 n 2^-24), to which half a
step of the output's type is added.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def moe():
    from llmcompressor_amd import moe as m
    return m


def plan_def(ids, experts):
    """By the definition: pairs by expert, then choice, then token; the others last."""
    tokens, top = ids.shape
    key = sorted(((int(ids[t, k]) if 0 <= ids[t, k] < experts else experts), k, t)
                 for t in range(tokens) for k in range(top))
    slots = torch.zeros(tokens, top, dtype=torch.int32)
    for i, (_, k, t) in enumerate(key):
        slots[t, k] = i
    offsets = torch.tensor([sum(1 for e, _, _ in key if e < x) for x in range(experts + 1)])
    return torch.tensor([t for _, _, t in key], dtype=torch.int32), slots, offsets


def plan_fast(ids, experts):
    e = torch.where((ids >= 0) & (ids < experts), ids, experts).long().t().reshape(-1)
    order = torch.sort(e, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel())
    counts = torch.bincount(e, minlength=experts + 1)[:experts]
    return ((order % ids.shape[0]).int(), slots.view(ids.shape[1], -1).t().contiguous().int(),
            torch.cat([torch.zeros(1).long(), counts.cumsum(0)]))


def same_plan(got, want):
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)


@pytest.mark.parametrize("tokens,top,experts", [(0, 2, 4), (1, 1, 1), (1, 8, 128), (3, 5, 2), (64, 1, 64), (65, 8, 7),
                                                (40, 6, 300)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_plan_by_definition(tokens, top, experts, dtype):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-2, experts + 2, (tokens, top), generator=g).to(dtype)     # repeated, and of no expert
    same_plan(moe().plan_tokens(ids.cuda(), experts), plan_def(ids, experts))


@pytest.mark.parametrize("tokens,top,experts", [(255, 8, 60), (256, 8, 8), (257, 8, 8), (2048, 1, 1), (4097, 2, 3),
                                                (9001, 8, 128), (1000, 4, 2040), (150001, 8, 257), (700000, 3, 5)])
@pytest.mark.parametrize("skew", [0.0, 3.0])
def test_plan_of_many(tokens, top, experts, skew):
    g = torch.Generator().manual_seed(tokens + top)
    u = torch.rand(tokens, top, generator=g) ** (1 + skew)
    ids = (u * (experts + 1)).long() - 1                     # -1: of no expert
    same_plan(moe().plan_tokens(ids.cuda(), experts), plan_fast(ids, experts))


def test_plan_of_one_expert_and_of_none():
    ids = torch.full((3000, 2), 4).cuda()
    same_plan(moe().plan_tokens(ids, 9), plan_fast(ids.cpu(), 9))
    same_plan(moe().plan_tokens(ids, 3), plan_fast(ids.cpu(), 3))
    wide = torch.arange(40).view(10, 4).cuda()
    same_plan(moe().plan_tokens(wide[:, 1:3], 40), plan_fast(wide[:, 1:3].cpu(), 40))     # a pitch
    same_plan(moe().plan_tokens(wide.t(), 40), plan_fast(wide.t().cpu(), 40))             # columns
    far = torch.tensor([[2 ** 40, 1], [-2 ** 33, 0]]).cuda()                               # ids beyond 32 bits
    same_plan(moe().plan_tokens(far, 2), plan_fast(far.cpu(), 2))


def close(got, want, bound):
    got = got.cpu()
    half = torch.finfo(got.dtype).eps / 2
    limit = bound + half * (want.abs() + bound) + torch.finfo(got.dtype).smallest_normal * half
    err = (got.double() - want).abs()
    assert got.shape == want.shape and bool((err <= limit).all()), float((err / limit).max())


CASES = [(1, 1, 1, 64), (1, 8, 128, 2048), (5, 3, 4, 7), (33, 8, 16, 100), (130, 2, 8, 2001), (700, 8, 60, 96),
         (257, 9, 30, 264), (3, 20, 40, 4100), (64, 1, 5, 1)]


@pytest.mark.parametrize("tokens,top,experts,cols", CASES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dropped", [0.0, 0.25])
def test_sort(tokens, top, experts, cols, dtype, dropped):
    g = torch.Generator().manual_seed(cols + tokens)
    ids = torch.randint(0, experts, (tokens, top), generator=g)
    ids[torch.rand(tokens, top, generator=g) < dropped] = -1
    x = torch.randn(tokens, cols, generator=g).to(dtype)
    d = torch.randn(tokens * top, cols, generator=g).to(dtype)
    rows, slots, offsets = plan_fast(ids, experts)
    end = int(offsets[-1])
    xg = x.cuda().requires_grad_()
    y, plan = moe().sort_tokens(xg, ids.cuda(), experts)
    same_plan(plan, (rows, slots, offsets))
    want = x[rows.long()].clone()
    want[end:] = 0
    assert torch.equal(y.detach().cpu(), want)
    dg = d.clone()
    dg[end:] = float("nan")                                   # takes no part
    (dx,) = torch.autograd.grad(y, xg, dg.cuda())
    t = rows[:end].long()
    zero = torch.zeros(tokens, cols, dtype=torch.float64)
    close(dx, zero.index_add(0, t, d[:end].double()), 2 * top * 2.0 ** -24 * zero.index_add(0, t, d[:end].double().abs()))


@pytest.mark.parametrize("tokens,top,experts,cols", CASES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dropped,w_dtype", [(0.0, F32), (0.25, BF16), (0.25, F16)])
def test_combine(tokens, top, experts, cols, dtype, dropped, w_dtype):
    g = torch.Generator().manual_seed(cols + tokens)
    ids = torch.randint(0, experts, (tokens, top), generator=g)
    ids[torch.rand(tokens, top, generator=g) < dropped] = experts
    rows, slots, offsets = plan_fast(ids, experts)
    end = int(offsets[-1])
    x = torch.randn(tokens * top, cols, generator=g).to(dtype)
    x[end:] = float("nan")                                    # takes no part
    w = torch.randn(tokens, top, generator=g).to(w_dtype)
    d = torch.randn(tokens, cols, generator=g).to(dtype)
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = moe().combine_tokens(xg, wg, moe().TokenPlan(rows.cuda(), slots.cuda(), offsets.cuda()))
    xd, wd, dd = x.double(), w.double(), d.double()
    xd[end:] = 0
    at = xd[slots.long()]                                     # [tokens, top, cols]
    kept = (slots < end)
    wk = torch.where(kept, wd, 0)
    close(y.detach(), (wk[..., None] * at).sum(1), 2 * top * 2.0 ** -24 * (wk[..., None] * at).abs().sum(1))
    dx, dw = torch.autograd.grad(y, (xg, wg), d.cuda())
    want = torch.zeros(tokens * top, cols, dtype=torch.float64)
    want[slots.long().reshape(-1)] = (wk[..., None] * dd[:, None]).reshape(-1, cols)
    close(dx, want, 2.0 ** -24 * want.abs())
    close(dw, (at * dd[:, None]).sum(2), 2 * cols * 2.0 ** -24 * (at * dd[:, None]).abs().sum(2))


def test_gradients_against_differences():
    """Of a whole layer: sort, an expert's product, combine; fp32 steps of 1/16 of a bilinear function."""
    g = torch.Generator().manual_seed(5)
    ids = torch.tensor([[0, 2], [1, 0], [-1, 2], [1, 1]]).cuda()
    x = torch.randn(4, 6, generator=g).cuda().requires_grad_()
    w = torch.rand(4, 2, generator=g).cuda().requires_grad_()
    c = torch.randn(4, 6, generator=g).cuda()
    m = moe()

    def f(x, w):
        rows, plan = m.sort_tokens(x, ids, 3)
        return (m.combine_tokens(rows * rows.detach().new_tensor(2.0), w, plan) * c).sum()

    dx, dw = torch.autograd.grad(f(x, w), (x, w))
    with torch.no_grad():
        for v, d in ((x, dx), (w, dw)):
            for i in range(v.numel()):
                e = torch.zeros_like(v)
                e.view(-1)[i] = 1 / 16
                args = [(a + s * e if a is v else a) for s in (1, -1) for a in (x, w)]
                slope = (f(*args[:2]) - f(*args[2:])) * 8
                # linear in each argument: only the sums' rounding, 2^-24 of some 50 terms' magnitudes (below 10), times 8
                assert abs(float(slope - d.view(-1)[i])) < 50 * 10 * 8 * 2.0 ** -24


def test_views_and_expanded_gradients():
    g = torch.Generator().manual_seed(9)
    ids = torch.randint(0, 4, (6, 2), generator=g).cuda()
    big = torch.randn(6, 40, generator=g).cuda()
    x = big[:, 3:20]                                           # a pitch, off 16 bytes
    m = moe()
    y, plan = m.sort_tokens(x, ids, 4)
    assert torch.equal(y, x[plan.rows.long()])
    xt = big[:, :6].t().contiguous().t().requires_grad_()      # columns
    y, plan = m.sort_tokens(xt, ids, 4)
    assert torch.equal(y, xt[plan.rows.long()])
    y.sum().backward()                                         # a gradient of stride 0
    assert torch.equal(xt.grad, torch.full_like(xt, 2.0))
    o = torch.randn(12, 6, generator=g).cuda().requires_grad_()
    m.combine_tokens(o, torch.ones(1, 1).cuda().expand(6, 2), plan).sum().backward()
    assert torch.equal(o.grad, torch.ones_like(o))


def test_only_the_gradients_asked_for():
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 4, (6, 2), generator=g).cuda()
    m = moe()
    plan = m.plan_tokens(ids, 4)
    o, w = torch.randn(12, 8, generator=g).cuda(), torch.rand(6, 2, generator=g).cuda()
    a = m.combine_tokens(o.requires_grad_(), w, plan)
    a.sum().backward()
    b = m.combine_tokens(o.detach(), w.requires_grad_(), plan)
    b.sum().backward()
    both = torch.autograd.grad(m.combine_tokens(o, w, plan).sum(), (o, w))
    assert torch.equal(o.grad, both[0]) and torch.equal(w.grad, both[1])


def test_places_that_do_not_exist_are_skipped():
    m = moe()
    x = torch.ones(2, 8).cuda()
    slots = torch.tensor([[0, 5], [-3, 1 << 30]], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 1 << 40]).cuda()
    from llmcompressor_amd import ops
    y = ops.moe_sort(x, slots, offsets)
    assert torch.equal(y[0], x[0])
    o = torch.ones(4, 8).cuda()
    assert torch.equal(ops.moe_combine(o, None, slots, offsets), torch.tensor([[1.0], [0.0]]).cuda().expand(2, 8))
    _, dw = ops.moe_combine_backward(x, o, torch.ones(2, 2).cuda(), slots, offsets)
    assert torch.equal(dw, torch.tensor([[8.0, 0], [0, 0]]).cuda())


def test_replayed_graph_follows_new_ids():
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 16, (900, 4), generator=g).cuda()    # several workgroups
    x = torch.randn(900, 64, generator=g).to(BF16).cuda()
    w = torch.rand(900, 4, generator=g).cuda()
    m = moe()

    def step():
        rows, plan = m.sort_tokens(x, ids, 16)
        return m.combine_tokens(rows, w, plan), plan

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, plan = step()
    for i in range(3):
        ids.add_(1).remainder_(17)                              # 16: of no expert
        graph.replay()
        torch.cuda.synchronize()
        again, other = step()
        assert torch.equal(y, again) and all(torch.equal(a, b) for a, b in zip(plan, other)), i


def test_rows_past_four_gigabytes():
    """Experts' rows of more than 2^32 bytes, and more than 2^31 elements."""
    tokens, cols = 300_000, 4096
    ids = torch.stack([torch.arange(tokens) % 3, 3 + torch.arange(tokens) % 2], 1).cuda()
    x = (torch.arange(tokens, device="cuda") % 251).to(BF16)[:, None] + (torch.arange(cols, device="cuda") % 2).to(BF16)
    x = x.requires_grad_()
    m = moe()
    y, plan = m.sort_tokens(x, ids, 5)
    for a in range(0, 2 * tokens, 50_000):
        assert torch.equal(y[a:a + 50_000], x[plan.rows[a:a + 50_000].long()]), a
    w = torch.full((tokens, 2), 0.5, device="cuda", requires_grad=True)
    out = m.combine_tokens(y, w, plan)
    assert torch.equal(out, x)
    (out[:, :2].float() * 2).sum().backward()
    want = torch.zeros_like(out)
    want[:, :2] = 2
    assert torch.equal(x.grad, want)
    assert torch.equal(w.grad, (2 * x[:, :2].float().sum(1, keepdim=True)).expand(-1, 2))


def test_replayed_gradients_follow_their_inputs():
    """Forward and backward in one graph, no eager graph of the leaves alive while it is captured."""
    g = torch.Generator().manual_seed(17)
    ids = torch.randint(0, 6, (70, 3), generator=g).cuda()
    x = torch.randn(70, 96, generator=g).to(BF16).cuda().requires_grad_()
    w = torch.rand(70, 3, generator=g).cuda().requires_grad_()
    d = torch.randn(70, 96, generator=g).to(BF16).cuda()
    m = moe()

    def step():
        rows, plan = m.sort_tokens(x, ids, 6)
        return torch.autograd.grad(m.combine_tokens(rows, w, plan), (x, w), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        ids.add_(1).remainder_(7)                               # 6: of no expert
        with torch.no_grad():
            x.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step())), i
