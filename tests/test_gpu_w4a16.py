"""4-bit weights: products against their definition in 64 bits on the CPU.

Tolerances.  A group's sum is an fp32 sum of exact products, of which the zero
point's part, z sum x, is one: with L = sum over groups of s sum |x| (q + z)
(MXFP4: sum |x| |w|), a result is within c 2^-24 L of the exact one for a chain of
c roundings; the chains (products inside one instruction, a group's instructions,
groups, waves) stay below 64 a wave for the sizes here, so 64 2^-24 L = 2^-18 L
bounds the value before the output's rounding, of which half a step is added.
Gated: silu's slope is below 1.1, so 1.1 (da |b| + da db) + |silu(a)| db, and 2^-20
of the value for the exponential, the quotient and the product in fp32.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def ops():
    from llmcompressor_amd import ops as o
    return o


def gen(*key):
    return torch.Generator().manual_seed(sum(ord(c) * (i + 1) for i, c in enumerate(repr(key))) & 0x7FFFFFFF)


def pack(codes):
    """codes [..., n] 0 .. 15 eight to an int32, lowest first; the last word filled with junk."""
    pad = -codes.shape[-1] % 8
    c = torch.nn.functional.pad(codes.long(), (0, pad), value=13).view(*codes.shape[:-1], -1, 8)
    w = sum(c[..., i] << (4 * i) for i in range(8))
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


class Weight:
    """A random 4-bit weight, its tensors and its exact values."""

    def __init__(self, g, out, cols, kind, group, scale_dtype=BF16, experts=None):
        lead = () if experts is None else (experts,)
        n = 1 if group is None else -(-cols // group)
        wide = cols if group is None else group
        if kind == "mxfp4":
            n, wide = cols // 32, 32
            codes = torch.randint(0, 16, (*lead, out, cols), generator=g)
            e = torch.randint(110, 125, (*lead, out, n), generator=g)
            self.parts = (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8), e.to(torch.uint8), None
            s = torch.exp2(e.double() - 127)
            self.values = E2M1[codes] * s.repeat_interleave(32, -1)
            self.sizes = self.values.abs()
        else:
            codes = torch.randint(0, 16, (*lead, out, cols), generator=g)
            s = (torch.rand(*lead, out, n, generator=g) * 0.02 + 1e-3).to(scale_dtype)
            z = torch.full((*lead, out, n), 8)
            zp = None
            if kind == "int4z":
                z = torch.randint(0, 16, (*lead, out, n), generator=g)
                zp = pack(z.transpose(-1, -2)).transpose(-1, -2).contiguous()
            self.parts = pack(codes), s, zp
            at = lambda t: t.double().repeat_interleave(wide, -1)[..., :cols]     # noqa: E731
            self.values = (codes.double() - at(z)) * at(s)
            self.sizes = (codes.double() + at(z)) * at(s)
        self.group = group

    def cuda(self):
        return [None if p is None else p.cuda() for p in self.parts]


def expected(x, values, sizes, bias=None, gated=False):
    """(exact result, bound of what precedes the rounding)"""
    x = x.double()
    y, tol = x @ values.T, 2.0 ** -18 * (x.abs() @ sizes.T)
    if bias is not None:
        y = y + bias.double()
        tol = tol + 2.0 ** -23 * y.abs()
    if not gated:
        return y, tol
    (a, b), (da, db) = y.chunk(2, 1), tol.chunk(2, 1)
    silu = a * torch.sigmoid(a)
    v = silu * b
    return v, 1.1 * da * (b.abs() + db) + silu.abs() * db + 2.0 ** -20 * v.abs()


def close(got, want, tol):
    got = got.cpu()
    half = torch.finfo(got.dtype).eps / 2
    limit = tol + half * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal * half
    err = (got.double() - want).abs()
    assert bool((err <= limit).all()), f"error {err.max():.3e}, {(err / limit).max():.2f} of the bound"


def check(rows, out, cols, kind="int4", group=128, dtype=BF16, bias=False, gated=False, out_dtype=None,
          scale_dtype=BF16):
    g = gen(rows, out, cols, kind, group, gated)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g))).to(dtype)
    w = Weight(g, out, cols, kind, group, scale_dtype)
    b = torch.randn(out, generator=g).to(dtype) if bias else None
    y = ops().w4a16_matmul(x.cuda(), *w.cuda(), group_size=group, bias=None if b is None else b.cuda(), gated=gated,
                           out_dtype=out_dtype)
    assert y.dtype == (out_dtype or dtype) and y.shape == (rows, out // 2 if gated else out)
    close(y, *expected(x, w.values, w.sizes, b, gated))


# ---------------------------------------------------------------- one weight
@pytest.mark.parametrize("kind,group", [("int4", 128), ("int4", 32), ("int4", 64), ("int4", 256), ("int4", None),
                                        ("int4z", 128), ("int4z", 32), ("int4z", 64), ("int4z", None), ("mxfp4", 32)])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 17, 40, 150])
def test_formats(rows, dtype, kind, group):
    check(rows, 208, 640, kind, group, dtype)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 300])
@pytest.mark.parametrize("out,cols", [(96, 256), (33, 128), (1, 384), (257, 8), (520, 1160)])
def test_rows_and_widths(rows, out, cols):
    check(rows, out, cols)


@pytest.mark.parametrize("cols", [1, 5, 7, 9, 31, 33, 100, 127, 129, 250, 1001, 2003])
@pytest.mark.parametrize("rows", [1, 20, 140])
@pytest.mark.parametrize("kind", ["int4", "int4z"])
def test_odd_widths(rows, cols, kind):
    check(rows, 77, cols, kind, 32 if cols % 2 else 128, F16 if cols % 3 else BF16)


@pytest.mark.parametrize("cols", [32, 96, 160, 2080])
@pytest.mark.parametrize("rows", [1, 20, 140])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
def test_mxfp4_widths(rows, cols, dtype):
    check(rows, 50, cols, "mxfp4", 32, dtype)


@pytest.mark.parametrize("rows", [1, 19, 130])
@pytest.mark.parametrize("kind,group", [("int4", 128), ("int4z", 32), ("mxfp4", 32)])
@pytest.mark.parametrize("out,bias", [(320, True), (86, False), (2, True)])
def test_gated(rows, kind, group, out, bias):
    check(rows, out, 512, kind, group, BF16, bias, True)


@pytest.mark.parametrize("rows", [1, 9, 40, 130])
@pytest.mark.parametrize("size", [30.0, 300.0, 3e4])
def test_gated_far_from_zero(rows, size):
    """Gates of -88 and below, where e^-gate passes fp32's range, and far above."""
    g = gen("far", rows, size)
    x = (torch.randn(rows, 256, generator=g) * size).to(BF16)
    w = Weight(g, 192, 256, "int4", 128)
    want, tol = expected(x, w.values, w.sizes, None, True)
    y = ops().w4a16_matmul(x.cuda(), *w.cuda(), gated=True, out_dtype=F32)
    assert bool((x.double() @ w.values.T)[:, :96].min() < -100) or size < 100
    close(y, want, tol)


@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("scale_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [3, 200])
def test_types(rows, out_dtype, scale_dtype):
    check(rows, 130, 384, "int4z", 64, BF16, True, False, out_dtype, scale_dtype)


@pytest.mark.parametrize("rows,out", [(700, 3000), (1300, 5000), (2700, 5300)], ids=["64x128", "64x256", "128x256"])
@pytest.mark.parametrize("cols,kind,group,dtype", [(256, "int4", 128, BF16), (168, "int4z", 32, F16),
                                                   (300, "int4z", 64, BF16), (160, "mxfp4", 32, BF16),
                                                   (352, "mxfp4", 32, F16), (261, "int4", None, F16)])
def test_larger_tiles(rows, out, cols, kind, group, dtype):
    check(rows, out, cols, kind, group, dtype, bias=True)


@pytest.mark.parametrize("rows,out", [(70, 600), (700, 6000), (1300, 10000), (2700, 10600)])
@pytest.mark.parametrize("cols,kind,group", [(256, "int4", 128), (168, "int4z", 32), (160, "mxfp4", 32)])
def test_larger_gated_tiles(rows, out, cols, kind, group):
    check(rows, out, cols, kind, group, BF16, rows % 2 == 0, True)


@pytest.mark.parametrize("rows,cols", [(80, 6144), (130, 9000), (70, 2304)])
@pytest.mark.parametrize("gated", [False, True])
def test_split_sums_of_many_columns(rows, cols, gated):
    check(rows, 256, cols, "int4z", 128, BF16, True, gated)
    check(rows // 3, 256, cols, "int4", 128, BF16, True, gated)


@pytest.mark.parametrize("rows", [90, 20])
def test_without_a_workspace(rows):
    """The C entry takes calls without one, by the kernel for few rows and without splitting sums."""
    import ctypes as C

    from llmcompressor_amd import _lib as L
    g = gen("ws", rows)
    x = torch.randn(rows, 4096, generator=g).to(BF16)
    w = Weight(g, 64, 4096, "int4", 128)
    p, s, _ = w.cuda()
    xc, y = x.cuda(), torch.empty(rows, 64, dtype=BF16, device="cuda")
    assert L.lib().mi355q_w4a16_matmul_workspace_size(rows, rows, 1, 64, 4096, L.W4_INT4, 128) > 0
    L.check(L.lib().mi355q_w4a16_matmul(xc.data_ptr(), L.BF16, rows, 4096, None, None, 1, p.data_ptr(), L.W4_INT4, 2048, 0,
                                        s.data_ptr(), L.BF16, 32, 0, None, 0, 0, 128, None, 0, 0, y.data_ptr(), L.BF16, 64,
                                        rows, 64, 4096, None, C.c_size_t(0), L.stream_of(xc)))
    close(y, *expected(x, w.values, w.sizes))


def test_no_rows():
    w = Weight(gen(1), 24, 64, "int4", 32)
    assert ops().w4a16_matmul(torch.empty(0, 64, dtype=BF16, device="cuda"), *w.cuda(), group_size=32).shape == (0, 24)


@pytest.mark.parametrize("rows", [2, 70, 260])
def test_views_and_what_lies_around(rows):
    """Operands as views of larger tensors full of NaN and junk; a transposed x and weight."""
    g = gen("views", rows)
    x = torch.randn(rows, 328, generator=g).to(BF16)
    w = Weight(g, 100, 328, "int4z", 32)
    want = expected(x, w.values, w.sizes)
    big = torch.full((rows + 2, 341), float("nan"), dtype=BF16, device="cuda")
    big[1:-1, 3:331] = x.cuda()
    p, s, z = w.cuda()
    pb = torch.full((102, 47), -1, dtype=torch.int32, device="cuda")
    pb[1:-1, 5:46] = p
    sb = torch.full((102, 13), float("nan"), dtype=BF16, device="cuda")
    sb[1:-1, 1:12] = s
    zb = torch.full((15, 12), -1, dtype=torch.int32, device="cuda")
    zb[1:-1, :11] = z
    close(ops().w4a16_matmul(big[1:-1, 3:331], pb[1:-1, 5:46], sb[1:-1, 1:12], zb[1:-1, :11], 32), *want)
    close(ops().w4a16_matmul(x.cuda().t().contiguous().t(), p.t().contiguous().t(), s.t().contiguous().t(), z, 32),
          *want)


def test_one_row_of_nan_leaves_the_others():
    g = gen("nan")
    x = torch.randn(40, 256, generator=g).to(BF16)
    w = Weight(g, 64, 256, "int4", 128)
    want, tol = expected(x, w.values, w.sizes)
    bad = x.clone()
    bad[7, 11] = float("nan")
    y = ops().w4a16_matmul(bad.cuda(), *w.cuda())
    assert bool(torch.isnan(y[7]).all())
    rest = [i for i in range(40) if i != 7]
    close(y[rest], want[rest], tol[rest])


# ---------------------------------------------------------------- experts
def plan(ids, experts):
    e = torch.where((ids >= 0) & (ids < experts), ids, experts).t().reshape(-1)
    order = torch.sort(e, stable=True).indices
    counts = torch.bincount(e, minlength=experts + 1)
    return (order % ids.shape[0]).int(), torch.cat([torch.zeros(1).long(), counts[:experts].cumsum(0)])


def check_experts(tokens, top, experts, out, cols, kind="int4", group=128, dtype=BF16, gated=False, gather=True,
                  spread=1.0, dropped=0.0):
    g = gen(tokens, top, experts, out, cols, kind)
    ids = (torch.randn(tokens, experts, generator=g) + spread * torch.randn(experts, generator=g)).topk(top).indices
    ids[torch.rand(tokens, generator=g) < dropped] = -1
    rows, offsets = plan(ids, experts)
    x = torch.randn(tokens if gather else tokens * top, cols, generator=g).to(dtype)
    w = Weight(g, out, cols, kind, group, experts=experts)
    y = ops().w4a16_experts_matmul(x.cuda(), rows.cuda() if gather else None, offsets.cuda(), *w.cuda(),
                                   group_size=group, gated=gated).cpu()
    xs = x[rows.long()] if gather else x
    for e in range(experts):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if a < b:
            close(y[a:b], *expected(xs[a:b], w.values[e], w.sizes[e], None, gated))
    assert not y[int(offsets[-1]):].any()


@pytest.mark.parametrize("tokens,top,experts", [(1, 1, 1), (1, 8, 128), (7, 2, 5), (40, 4, 33), (100, 3, 3),
                                                (64, 8, 130), (500, 2, 4)])
@pytest.mark.parametrize("gated", [False, True])
def test_experts(tokens, top, experts, gated):
    check_experts(tokens, top, experts, 96, 256, gated=gated)


@pytest.mark.parametrize("kind,group,dtype", [("int4z", 32, BF16), ("int4z", 128, F16), ("mxfp4", 32, BF16),
                                              ("mxfp4", 32, F16), ("int4", None, F16)])
@pytest.mark.parametrize("tokens", [3, 90, 400])
def test_experts_formats(tokens, kind, group, dtype):
    check_experts(tokens, 3, 6, 72, 416, kind, group, dtype, spread=2.0)


@pytest.mark.parametrize("tokens,top,experts", [(200, 2, 2), (700, 3, 3), (100, 3, 3)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind,group", [("int4", 128), ("int4z", 32)])
def test_experts_of_many_rows(tokens, top, experts, gated, kind, group):
    check_experts(tokens, top, experts, 300, 264, kind, group, gated=gated, gather=not gated, dropped=0.1)


# One expert: as many rows as a dense product, whose sums are split over workgroups at these widths.
@pytest.mark.parametrize("tokens", [1, 24, 60, 100, 700])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind,group", [("int4z", 128), ("mxfp4", 32)])
def test_one_expert(tokens, gated, kind, group):
    check_experts(tokens, 1, 1, 96, 2304, kind, group, gated=gated, gather=gated, dropped=0.2)


# Rows that x does not have are zeros, of one expert too.
@pytest.mark.parametrize("tokens", [24, 100])
@pytest.mark.parametrize("gated", [False, True])
def test_one_expert_rows_not_there(tokens, gated):
    g = gen(tokens, gated)
    x = torch.randn(tokens, 2304, generator=g).to(BF16)
    w = Weight(g, 96, 2304, "int4", 128, experts=1)
    rows = torch.arange(tokens, dtype=torch.int32)
    rows[::3] = -1
    rows[1::6] = tokens
    rows[4] = 2**31 - 1
    there = (rows >= 0) & (rows < tokens)
    y = ops().w4a16_experts_matmul(x.cuda(), rows.cuda(), torch.tensor([0, tokens]).cuda(), *w.cuda(), group_size=128,
                                   gated=gated).cpu()
    close(y[there], *expected(x[there], w.values[0], w.sizes[0], None, gated))
    assert not y[~there].any()


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dropped", [0.3, 1.0])
@pytest.mark.parametrize("tokens", [5, 150])
def test_experts_without_some_tokens(tokens, dropped, gather):
    check_experts(tokens, 2, 7, 40, 136, "int4z", 32, gather=gather, dropped=dropped)


def test_experts_of_whom_most_have_no_rows():
    check_experts(30, 1, 200, 32, 128, spread=6.0)


def test_offsets_and_rows_that_do_not_fit_stay_inside():
    """Rows that x does not have count as zeros; offsets are clamped to y's rows."""
    g = gen("bad")
    x = torch.randn(4, 128, generator=g).to(BF16)
    w = Weight(g, 16, 128, "int4", 128, experts=3)
    rows = torch.tensor([0, -1, 3, 4, 1 << 30], dtype=torch.int32)
    offsets = torch.tensor([0, 2, 4, 5])
    y = ops().w4a16_experts_matmul(x.cuda(), rows.cuda(), offsets.cuda(), *w.cuda()).cpu()
    close(y[:1], *expected(x[:1], w.values[0], w.sizes[0]))
    close(y[2:3], *expected(x[3:4], w.values[1], w.sizes[1]))
    assert not y[[1, 3, 4]].any()
    y = ops().w4a16_experts_matmul(x.cuda(), None, torch.tensor([0, 2, 3, 900]).cuda(), *w.cuda()).cpu()
    close(y[3:], *expected(x[3:], w.values[2], w.sizes[2]))


def test_results_do_not_change_from_run_to_run_and_under_graphs():
    g = gen("graph")
    w = Weight(g, 192, 512, "int4", 128, experts=8)
    parts = w.cuda()
    x = torch.randn(24, 512, generator=g).to(BF16).cuda()
    ids = torch.stack([torch.randperm(8, generator=g)[:2] for _ in range(24)]).cuda()
    o = ops()

    def step():
        rows, _, offsets = o.moe_plan(ids, 8)
        return o.w4a16_experts_matmul(x, rows, offsets, *parts, gated=True)

    first = step()
    assert torch.equal(first, step())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for i in range(3):
        ids.copy_((ids + 1) % 8)
        x.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step()), i


def test_rows_past_four_gigabytes():
    """x of more than 2^32 bytes, in order and gathered."""
    g = gen("far")
    rows, cols = 300_000, 8192
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    some = torch.tensor([0, 1, 255_999, 262_143, 262_144, 299_904, 299_999])
    x[some.cuda()] = torch.randn(len(some), cols, generator=g).to(BF16).cuda()
    w = Weight(g, 32, cols, "int4", 128)
    want = expected(x[some.cuda()].cpu(), w.values, w.sizes)
    y = ops().w4a16_matmul(x, *w.cuda())
    close(y[some.cuda()], *want)
    assert not y[2:255_999].any() and not y[262_145:299_904].any()
    several = [p.expand(3, *p.shape) if p is not None else None for p in w.cuda()]         # the same weight thrice
    for n in (1, 40):
        y = ops().w4a16_experts_matmul(x, some.int().cuda().repeat(n), torch.tensor([0, 2 * n, 2 * n, 7 * n]).cuda(),
                                       *several)
        close(y, want[0].repeat(n, 1), want[1].repeat(n, 1))


def test_bytes_off_every_boundary():
    """MXFP4 codes whose rows and experts lie at odd bytes."""
    g = gen("odd")
    w = Weight(g, 24, 96, "mxfp4", 32, experts=3)
    x = torch.randn(60, 96, generator=g).to(BF16)
    offsets = torch.tensor([0, 20, 20, 60])
    p, s, _ = w.cuda()
    for lead, pitch, gap in ((1, 48, 0), (0, 53, 0), (0, 52, 1), (4, 52, 2)):
        flat = torch.zeros(lead + 3 * (24 * pitch + gap), dtype=torch.uint8, device="cuda")
        view = flat.as_strided((3, 24, 48), (24 * pitch + gap, pitch, 1), lead)
        view.copy_(p)
        y = ops().w4a16_experts_matmul(x.cuda(), None, offsets.cuda(), view, s).cpu()
        for e in (0, 2):
            a, b = int(offsets[e]), int(offsets[e + 1])
            close(y[a:b], *expected(x[a:b], w.values[e], w.sizes[e]))


def test_two_calls_at_once():
    """Calls on two streams, whose workspaces are their own."""
    g = gen("streams")
    w = Weight(g, 256, 1024, "int4z", 32)
    parts = w.cuda()
    xs = [torch.randn(r, 1024, generator=g).to(BF16) for r in (200, 333)]
    gs = [x.cuda() for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    ys = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                ys[i].append(ops().w4a16_matmul(gs[i], *parts, group_size=32))
    torch.cuda.synchronize()
    for x, got in zip(xs, ys):
        want = expected(x, w.values, w.sizes)
        for y in got:
            close(y, *want)
