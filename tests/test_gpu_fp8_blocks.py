"""Block-scaled fp8: quantizers, products, gradients and the gated activation
against their definitions in 64 bits on the CPU.

Tolerances.  Sums are fp32 sums of exact products: with L the sum of the
terms' magnitudes, a result is within c 2^-24 L of the exact one for a chain
of c roundings; the kernels' chains (products inside one matrix instruction,
groups of 128, partial sums) stay far below 64 for the sizes here, so 64 2^-24
L = 2^-18 L is the bound before the output's rounding: a result has to lie
between the output type's roundings of the exact value less and plus that.
Codes are compared with the correctly rounded quotient: they may differ
only where the fp32 quotient rounds onto a tie, which is at most one e4m3 step.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

G = 128
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def ops():
    from llmcompressor_amd import ops as o
    return o


def gen(*key):
    return torch.Generator().manual_seed(hash(key) & 0x7FFFFFFF)


def heavy(g, *shape):
    return torch.randn(*shape, generator=g) * torch.exp(torch.randn(shape[-1], generator=g))


# ---------------------------------------------------------------- definitions, 64 bits
def wide(s, rows, n, k):
    return s.double().repeat_interleave(rows, 0)[:n].repeat_interleave(G, 1)[:, :k]


def tops(x, rows):
    n, k = x.shape
    p = torch.zeros(-(-n // rows) * rows, -(-k // G) * G, dtype=torch.float64)
    p[:n, :k] = x.double().abs()
    return p.view(p.shape[0] // rows, rows, p.shape[1] // G, G).amax((1, 3))


def scale_def(top, kind):
    if kind == torch.float32:
        s = (top / 448).float().double()
        s = torch.where(s == 0, torch.full_like(s, 2.0 ** -23), s)
    else:
        e = torch.ceil(torch.log2(torch.where(top == 0, torch.full_like(top, 448.0), top) / 448)).clamp(-126, 127)
        s = torch.exp2(e)
    return torch.where(torch.isfinite(top), s, torch.full_like(s, math.nan))


def e4m3(v):
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def values(codes, scales):
    """64-bit values of an fp8 matrix, on the CPU."""
    codes, scales = codes.cpu(), scales.cpu()
    rows = 1 if scales.shape[0] == codes.shape[0] else G
    return codes.double() * wide(scales, rows, *codes.shape)


def check_codes(codes, scales, x, rows, kind):
    n, k = x.shape
    s = scale_def(tops(x, rows), kind)
    got_s = scales.cpu().double()
    assert torch.equal(torch.isnan(got_s), torch.isnan(s))
    assert torch.equal(got_s[~torch.isnan(s)], s[~torch.isnan(s)])
    w = wide(s, rows, n, k)
    got, bad = codes.cpu().double(), torch.isnan(w)
    assert bool(torch.isnan(got[bad]).all())
    want = e4m3(x.double() / w)
    got, want, q = got[~bad], want[~bad], (x.double() / w)[~bad]
    differ = got != want
    if bool(differ.any()):     # only where the quotient is within fp32 rounding of a tie
        mid = (got[differ] + want[differ]) / 2
        assert bool(((q[differ] - mid).abs() <= 2.0 ** -23 * mid.abs()).all())


def check_sum(got, want, mags, dtype):
    got, tol = got.cpu(), 2.0 ** -18 * mags
    assert got.dtype == dtype and got.shape == want.shape
    ok = (got >= (want - tol).to(dtype)) & (got <= (want + tol).to(dtype))
    assert bool(ok.all()), f"{int((~ok).sum())} outside, worst {float(((got.double() - want).abs() / mags).max()):.3g}"


# ---------------------------------------------------------------- quantizers
SHAPES = [(1, 128), (1, 1), (3, 127), (5, 129), (7, 200), (1, 4096), (33, 776), (257, 384), (2, 1040)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", [torch.float32, E8M0])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_groups(dev, rows, cols, kind, dtype):
    x = heavy(gen(rows, cols), rows, cols).to(dtype)
    x[0, :min(cols, 128)] = 0                                # a group of zeros
    if cols > 130:
        x[-1, 128] = 448.0                                   # on a boundary of the power-of-two rule
        x[-1, 129:256] *= 0
    codes, scales = ops().fp8_quantize_groups(x.to(dev), kind)
    assert codes.dtype == E4M3 and scales.dtype == kind and scales.shape == (rows, -(-cols // G))
    check_codes(codes, scales, x, 1, kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(128, 128), (1, 1), (129, 257), (300, 200), (64, 512), (127, 136)])
def test_quantize_blocks(dev, rows, cols, dtype):
    w = (torch.randn(rows, cols, generator=gen(rows, cols)) * 0.02).to(dtype)
    codes, scales = ops().fp8_quantize_blocks(w.to(dev))
    assert scales.shape == (-(-rows // G), -(-cols // G))
    check_codes(codes, scales, w, G, torch.float32)


@pytest.mark.parametrize("kind", [torch.float32, E8M0])
def test_quantize_groups_every_bf16_value(dev, kind):
    """Each finite bf16 value as the largest of its group, beside values at many fractions of it."""
    top = torch.arange(0, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(top.numel(), G, dtype=torch.bfloat16)
    x[:] = (top.float().unsqueeze(1) * torch.linspace(-1, 1, G)).to(torch.bfloat16)
    x[:, 0] = top
    codes, scales = ops().fp8_quantize_groups(x.to(dev), kind)
    normal = top.double() >= 2.0 ** -110                     # below: the smallest codes are fp32 subnormals
    check_codes(codes[normal.to(dev)], scales[normal.to(dev)], x[normal], 1, kind)
    s = scale_def(tops(x, 1), kind)
    if kind == E8M0:
        assert torch.equal(scales.cpu().double(), s)
    assert not bool(torch.isnan(codes.cpu().float()).any())


@pytest.mark.parametrize("kind", [torch.float32, E8M0])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_non_finite_groups_are_nan_as_a_whole(dev, kind, bad, dtype):
    x = torch.randn(4, 300, generator=gen(1)).to(dtype)
    x[1, 130] = bad
    x[3, 299] = bad
    codes, scales = ops().fp8_quantize_groups(x.to(dev), kind)
    check_codes(codes, scales, x, 1, kind)
    assert torch.isnan(scales.cpu().float()).sum() == 2
    w = x.to(dev)
    codes, scales = ops().fp8_quantize_blocks(w)
    check_codes(codes, scales, x, G, torch.float32)


def test_quantize_strided_and_empty(dev):
    base = torch.randn(40, 600, generator=gen(2)).to(torch.bfloat16)
    d = base.to(dev)
    for view, ref in ((d[:, 8:264], base[:, 8:264]), (d[:, 3:300], base[:, 3:300]), (d.t(), base.t()),
                      (d[::2, :256], base[::2, :256]), (d[:1].expand(5, 600), base[:1].expand(5, 600))):
        codes, scales = ops().fp8_quantize_groups(view, E8M0)
        check_codes(codes, scales, ref, 1, E8M0)
        codes, scales = ops().fp8_quantize_blocks(view)
        check_codes(codes, scales, ref, G, torch.float32)
    codes, scales = ops().fp8_quantize_groups(d[:0])
    assert codes.shape == (0, 600) and scales.shape == (0, 5)


# ---------------------------------------------------------------- products
def fp8_pair(g, rows, out, cols, kind):
    x = heavy(g, rows, cols).to(torch.bfloat16)
    w = (torch.randn(out, cols, generator=g) * 0.02).to(torch.bfloat16)
    o = ops()
    return *o.fp8_quantize_groups(x.cuda(), kind), *o.fp8_quantize_blocks(w.cuda())


PRODUCTS = [(1, 128, 128), (1, 1, 1), (1, 4096, 512), (2, 130, 257), (3, 64, 40), (15, 200, 1040), (16, 256, 272),
            (17, 256, 4096), (31, 129, 129), (33, 384, 384), (64, 512, 640), (65, 72, 2048), (100, 1000, 144),
            (129, 128, 896), (200, 640, 1168), (256, 256, 256), (257, 513, 528), (300, 264, 1), (513, 768, 640),
            (1025, 520, 400)]


@pytest.mark.parametrize("kind", [torch.float32, E8M0])
@pytest.mark.parametrize("rows,out,cols", PRODUCTS)
def test_block_matmul(dev, rows, out, cols, kind):
    g = gen(rows, out, cols)
    x, xs, w, ws = fp8_pair(g, rows, out, cols, kind)
    dtype = [torch.bfloat16, torch.float16, torch.float32][(rows + out + cols) % 3]
    bias = (torch.randn(out, generator=g) * 3).to([torch.float32, torch.bfloat16, torch.float16][(rows + out) % 3])
    a, b = values(x, xs), values(w, ws)
    want, mags = a @ b.T, a.abs() @ b.abs().T
    check_sum(ops().fp8_block_matmul(x, xs, w, ws, out_dtype=dtype), want, mags, dtype)
    check_sum(ops().fp8_block_matmul(x, xs, w, ws, bias=bias.to(dev), out_dtype=dtype), want + bias.double(),
              mags + bias.double().abs(), dtype)


@pytest.mark.parametrize("rows,out,cols", PRODUCTS)
def test_block_grad_input(dev, rows, out, cols):
    g = gen(rows, out, cols, 5)
    w, ws = ops().fp8_quantize_blocks((torch.randn(out, cols, generator=g) * 0.02).to(torch.bfloat16).to(dev))
    dy = heavy(g, rows, out).to(torch.bfloat16)
    b = values(w, ws)
    check_sum(ops().fp8_block_grad_input(dy.to(dev), w, ws), dy.double() @ b, dy.double().abs() @ b.abs(),
              torch.bfloat16)


@pytest.mark.parametrize("rows,out,cols", PRODUCTS)
def test_block_grad_weight(dev, rows, out, cols):
    g = gen(rows, out, cols, 6)
    x, xs = ops().fp8_quantize_groups(heavy(g, rows, cols).to(torch.bfloat16).to(dev), E8M0)
    dy = (heavy(g, rows, out) * torch.exp(torch.randn(rows, 1, generator=g))).to(torch.bfloat16)
    a = values(x, xs)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        check_sum(ops().fp8_block_grad_weight(dy.to(dev), x, xs, out_dtype=dtype), dy.double().T @ a,
                  dy.double().abs().T @ a.abs(), dtype)


# sizes at which the larger tiles run, with ragged edges in every direction
LARGE = [(2500, 2600, 144), (130, 6200, 4096), (1700, 3800, 272)]


def values_gpu(codes, scales):
    rows = 1 if scales.shape[0] == codes.shape[0] else G
    n, k = codes.shape
    return codes.double() * scales.double().repeat_interleave(rows, 0)[:n].repeat_interleave(G, 1)[:, :k]


def check_sum_gpu(got, a, b, dtype):
    """check_sum against a b^T, all on the GPU (64-bit products of torch)."""
    want, tol = a @ b.T.contiguous(), 2.0 ** -18 * (a.abs() @ b.abs().T.contiguous())
    assert got.dtype == dtype and got.shape == want.shape
    assert bool(((got >= (want - tol).to(dtype)) & (got <= (want + tol).to(dtype))).all())


@pytest.mark.parametrize("kind", [torch.float32, E8M0])
@pytest.mark.parametrize("rows,out,cols", LARGE)
def test_large_products(dev, rows, out, cols, kind):
    o, g = ops(), torch.Generator(device=dev).manual_seed(rows)
    x, xs = o.fp8_quantize_groups((torch.randn(rows, cols, generator=g, device=dev) * 3).to(torch.bfloat16), kind)
    w, ws = o.fp8_quantize_blocks((torch.randn(out, cols, generator=g, device=dev) * 0.02).to(torch.bfloat16))
    a, b = values_gpu(x, xs), values_gpu(w, ws)
    for dtype in (torch.bfloat16, torch.float32):
        check_sum_gpu(o.fp8_block_matmul(x, xs, w, ws, out_dtype=dtype), a, b, dtype)
    dy = torch.randn(rows, out, generator=g, device=dev).to(torch.bfloat16)
    check_sum_gpu(o.fp8_block_grad_input(dy, w, ws), dy.double(), b.T, torch.bfloat16)


@pytest.mark.parametrize("rows,out,cols", [(77, 3800, 3616), (2100, 3080, 4112), (33, 4096, 4096)])
def test_large_weight_gradients(dev, rows, out, cols):
    o, g = ops(), torch.Generator(device=dev).manual_seed(rows)
    x, xs = o.fp8_quantize_groups((torch.randn(rows, cols, generator=g, device=dev) * 3).to(torch.bfloat16), E8M0)
    dy = (torch.randn(rows, out, generator=g, device=dev) * 1e-4).to(torch.bfloat16)
    for dtype in (torch.float32, torch.bfloat16):
        check_sum_gpu(o.fp8_block_grad_weight(dy, x, xs, dtype), dy.double().T.contiguous(),
                      values_gpu(x, xs).T.contiguous(), dtype)


ODD = [(100, 131, 257), (70, 1003, 1001), (300, 777, 135), (1, 1001, 333), (20, 50, 4097), (33, 8, 127), (40, 9, 16),
       (513, 260, 24)]


def raw_products(o, x, xs, w, ws, dy, workspace):
    """The three products through the C entry points, with the queried workspace or with none."""
    from llmcompressor_amd import _lib as L
    rows, cols, out, lib = x.shape[0], x.shape[1], w.shape[0], L.lib()
    y, dx, dw = (torch.full(s, float("nan"), device=x.device, dtype=t) for s, t in (
        ((rows, out), torch.float32), ((rows, cols), torch.bfloat16), ((out, cols), torch.float32)))

    def room(query):
        n = query(rows, out, cols) if workspace else 0
        t = torch.empty(n, dtype=torch.uint8, device=x.device)
        return t, t.data_ptr() if n else None, n
    st = L.stream_of(x)
    k, p, n = room(lib.mi355q_fp8_block_matmul_workspace_size)
    L.check(lib.mi355q_fp8_block_matmul(x.data_ptr(), x.stride(0), xs.data_ptr(), L.SCALE_E8M0, xs.stride(0), w.data_ptr(),
                                        w.stride(0), ws.data_ptr(), ws.stride(0), None, 0, y.data_ptr(), L.F32, out, rows,
                                        out, cols, p, n, st))
    k2, p, n = room(lib.mi355q_fp8_block_grad_input_workspace_size)
    L.check(lib.mi355q_fp8_block_grad_input(dy.data_ptr(), dy.stride(0), w.data_ptr(), w.stride(0), ws.data_ptr(),
                                            ws.stride(0), dx.data_ptr(), cols, rows, out, cols, p, n, st))
    k3, p, n = room(lib.mi355q_fp8_block_grad_weight_workspace_size)
    L.check(lib.mi355q_fp8_block_grad_weight(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), xs.data_ptr(),
                                             xs.stride(0), dw.data_ptr(), L.F32, cols, rows, out, cols, p, n, st))
    torch.cuda.synchronize()
    return y, dx, dw


def check_products(x, xs, w, ws, dy, y, dx, dw):
    a, b, d = values(x, xs), values(w, ws), dy.cpu().double()
    check_sum(y, a @ b.T, a.abs() @ b.abs().T, torch.float32)
    check_sum(dx, d @ b, d.abs() @ b.abs(), torch.bfloat16)
    check_sum(dw, d.T @ a, d.abs().T @ a.abs(), torch.float32)


@pytest.mark.parametrize("rows,out,cols", ODD)
def test_products_of_odd_widths(dev, rows, out, cols):
    """Widths that are no whole number of 16-byte chunks: padded copies, element loads, few tokens."""
    o, g = ops(), gen(rows, out, cols, 3)
    x, xs, w, ws = fp8_pair(g, rows, out, cols, E8M0)
    dy = heavy(g, rows, out).to(torch.bfloat16).to(dev)
    check_products(x, xs, w, ws, dy, o.fp8_block_matmul(x, xs, w, ws, out_dtype=torch.float32),
                   o.fp8_block_grad_input(dy, w, ws), o.fp8_block_grad_weight(dy, x, xs, torch.float32))


@pytest.mark.parametrize("rows,out,cols", [(70, 1003, 1001), (300, 777, 135), (200, 384, 2048), (64, 512, 4096),
                                           (700, 256, 512)])
def test_products_without_a_workspace(dev, rows, out, cols):
    """Without room for splits or padded copies the sums run whole and odd operands take element loads."""
    o, g = ops(), gen(rows, out, cols, 4)
    x, xs, w, ws = fp8_pair(g, rows, out, cols, E8M0)
    dy = heavy(g, rows, out).to(torch.bfloat16).to(dev)
    for workspace in (False, True):
        check_products(x, xs, w, ws, dy, *raw_products(o, x, xs, w, ws, dy, workspace))


def test_products_of_badly_placed_rows(dev):
    """Rows of whole chunks that do not begin on 16 bytes, through the C entry points (no copies are queried)."""
    o, g = ops(), gen(17)
    x, xs, w, ws = fp8_pair(g, 50, 64, 256, E8M0)
    dy = heavy(g, 50, 64).to(torch.bfloat16).to(dev)
    bx, bw = (torch.zeros(t.shape[0], 275, device=dev).to(E4M3)[:, 3:259] for t in (x, w))
    by = torch.zeros(50, 77, device=dev, dtype=torch.bfloat16)[:, 5:69]
    bx.copy_(x), bw.copy_(w), by.copy_(dy)
    check_products(x, xs, w, ws, dy, *raw_products(o, bx, xs, bw, ws, by, True))


def test_products_of_strided_operands(dev):
    """Codes and gradients that are views of wider or transposed buffers."""
    o, g = ops(), gen(11)
    for off, cols in ((16, 256), (3, 200)):
        x, xs, w, ws = fp8_pair(g, 70, 150, cols, E8M0)
        dy = torch.randn(70, 150, generator=g).to(torch.bfloat16).to(dev)
        base_x, base_w = torch.zeros(70, cols + 48, device=dev).to(E4M3), torch.zeros(150, cols + 80, device=dev).to(E4M3)
        vx, vw = base_x[:, off:off + cols], base_w[:, off:off + cols]
        vx.copy_(x), vw.copy_(w)
        base_s = torch.zeros(150 // G + 1, 9, device=dev)
        vs = base_s[:, 1:1 + ws.shape[1]]
        vs.copy_(ws)
        vdy = torch.zeros(70, 200, device=dev, dtype=torch.bfloat16)[:, off:off + 150]
        vdy.copy_(dy)
        want = o.fp8_block_matmul(x, xs, w, ws, out_dtype=torch.float32)
        a, b = values(x, xs), values(w, ws)
        for args in ((vx, xs, vw, vs), (x.t().contiguous().t(), xs.t().contiguous().t(), w, ws)):
            check_sum(o.fp8_block_matmul(*args, out_dtype=torch.float32), a @ b.T, a.abs() @ b.abs().T, torch.float32)
        del want
        d = dy.cpu().double()
        check_sum(o.fp8_block_grad_input(vdy, vw, vs), d @ b, d.abs() @ b.abs(), torch.bfloat16)
        check_sum(o.fp8_block_grad_weight(vdy, vx, xs, torch.float32), d.T @ a, d.abs().T @ a.abs(), torch.float32)


def test_products_without_rows(dev):
    o = ops()
    x, xs, w, ws = fp8_pair(gen(3), 4, 136, 256, E8M0)
    assert o.fp8_block_matmul(x[:0], xs[:0], w, ws).shape == (0, 136)
    dy = torch.zeros(0, 136, device=dev, dtype=torch.bfloat16)
    assert o.fp8_block_grad_input(dy, w, ws).shape == (0, 256)
    dw = o.fp8_block_grad_weight(dy, x[:0], xs[:0], torch.float32)
    assert dw.shape == (136, 256) and bool((dw == 0).all())


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_nan_reaches_its_row_and_nothing_else(dev, rows):
    """A NaN group of x spoils its own row of y (and every column it meets in the gradients), no other."""
    o, g = ops(), gen(rows, 9)
    src = torch.randn(rows, 640, generator=g).to(torch.bfloat16)
    src[rows - 1, 300] = math.inf
    w, ws = o.fp8_quantize_blocks((torch.randn(272, 640, generator=g) * 0.02).to(torch.bfloat16).to(dev))
    for kind in (torch.float32, E8M0):
        x, xs = o.fp8_quantize_groups(src.to(dev), kind)
        bad = torch.isnan(o.fp8_block_matmul(x, xs, w, ws)).cpu()
        assert bool(bad[rows - 1].all()) and not bool(bad[:rows - 1].any())
    dy = torch.randn(rows, 272, generator=g).to(torch.bfloat16).to(dev)
    bad = torch.isnan(o.fp8_block_grad_weight(dy, x, xs)).cpu()
    assert bool(bad[:, 256:384].all()) and not bool(bad[:, :256].any()) and not bool(bad[:, 384:].any())
    dy[rows - 1, 5] = math.nan
    bad = torch.isnan(o.fp8_block_grad_input(dy, w, ws)).cpu()
    assert bool(bad[rows - 1].all()) and not bool(bad[:rows - 1].any())


def test_products_are_the_same_every_time(dev):
    """No order of additions depends on timing."""
    o, g = ops(), gen(21)
    for rows, out, cols in ((5, 512, 4096), (200, 384, 2048), (700, 256, 512)):
        x, xs, w, ws = fp8_pair(g, rows, out, cols, E8M0)
        dy = torch.randn(rows, out, generator=g).to(torch.bfloat16).to(dev)
        first = None
        for _ in range(3):
            now = (o.fp8_block_matmul(x, xs, w, ws, out_dtype=torch.float32), o.fp8_block_grad_input(dy, w, ws),
                   o.fp8_block_grad_weight(dy, x, xs, torch.float32))
            first = first or now
            assert all(torch.equal(a, b) for a, b in zip(first, now))


# ---------------------------------------------------------------- gated activation
def glu_inputs(rows, cols, dtype):
    x = (torch.randn(rows, 2 * cols, generator=gen(rows, cols, 7)) * 2).to(dtype)
    x[0, 0], x[0, cols] = 60.0, -3.0
    x[-1, cols - 1] = -60.0
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 128), (1, 1), (3, 200), (5, 129), (65, 384), (33, 1032)])
def test_silu_mul(dev, rows, cols, dtype):
    """h's codes are those of h = silu(gate) up but for h's own relative error, 2^-20: a scale may take
    the other side of its boundary only if the largest |h| is that near, a code the next step."""
    o, x = ops(), glu_inputs(rows, cols, dtype)
    h, hs, kept, ks = o.fp8_silu_mul(x.to(dev))
    gate, up = x[:, :cols].double(), x[:, cols:].double()
    want = gate * torch.sigmoid(gate) * up
    top = tops(want, 1)
    lo, hi = scale_def(top * (1 - 2.0 ** -20), E8M0), scale_def(top * (1 + 2.0 ** -20), E8M0)
    s = hs.cpu().double()
    assert bool(((s == lo) | (s == hi)).all())
    q = want / wide(s, 1, rows, cols)
    # half a code step (2^-4 of the value, 2^-10 among the subnormal codes) and h's error
    assert bool(((h.cpu().double() - q).abs() <= q.abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10).all())
    G2 = -(-cols // G)
    assert kept.shape == (rows, 2 * cols) and ks.shape == (rows, 2 * G2)
    check_codes(kept[:, :cols], ks[:, :G2], x[:, :cols], 1, E8M0)
    check_codes(kept[:, cols:], ks[:, G2:], x[:, cols:], 1, E8M0)
    h2, hs2 = o.fp8_silu_mul(x.to(dev), save=False)
    assert torch.equal(h.view(torch.uint8), h2.view(torch.uint8)) and torch.equal(hs.view(torch.uint8),
                                                                                  hs2.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 128), (1, 1), (3, 200), (5, 129), (65, 384), (33, 1032)])
def test_silu_mul_backward(dev, rows, cols, dtype):
    o, x = ops(), glu_inputs(rows, cols, dtype)
    _, _, kept, ks = o.fp8_silu_mul(x.to(dev))
    dh = torch.randn(rows, cols, generator=gen(rows, cols, 8)).to(dtype)
    groups = -(-cols // G)
    gate, up = values(kept[:, :cols], ks[:, :groups]), values(kept[:, cols:], ks[:, groups:])
    d, s = dh.double(), torch.sigmoid(gate)
    want = torch.cat([d * up * (s + gate * s * (1 - s)), d * gate * s], 1)
    # the factors' magnitudes bound the error of a short chain of fp32 steps, each within a few 2^-24,
    # and of the sigmoid, within 2^-20
    mags = torch.cat([d.abs() * up.abs() * (s + gate.abs() * s), d.abs() * gate.abs() * s], 1)
    check_sum(o.fp8_silu_mul_backward(dh.to(dev), kept, ks), want, mags, dtype)


def test_silu_mul_backward_against_differences(dev):
    """Central differences of silu(gate) up at the kept values, in 64 bits: step 2^-10, error step^2 / 6 times a
    third derivative below 1 of the sigmoid's product (|gate|, |up| < 8), so 2^-20 8 8, beside fp32 rounding."""
    o = ops()
    x = torch.randn(4, 512, generator=gen(12))
    _, _, kept, ks = o.fp8_silu_mul(x.to(dev))
    dh = torch.randn(4, 256, generator=gen(13))
    got = o.fp8_silu_mul_backward(dh.to(dev), kept, ks).cpu().double()
    gate, up = values(kept[:, :256], ks[:, :2]), values(kept[:, 256:], ks[:, 2:])
    e = 2.0 ** -10

    def h(a, b):
        return a * torch.sigmoid(a) * b
    dg = (h(gate + e, up) - h(gate - e, up)) / (2 * e) * dh.double()
    du = (h(gate, up + e) - h(gate, up - e)) / (2 * e) * dh.double()
    assert float((got - torch.cat([dg, du], 1)).abs().max()) <= 2.0 ** -20 * 64 * float(dh.abs().max())


def test_gradients_against_differences(dev):
    """dX and dW of sum(dY * (X W^T)) against differences of the product itself, which is linear in X and in W:
    a unit step of one element changes it by the gradient exactly."""
    o, g = ops(), gen(31)
    x, xs, w, ws = fp8_pair(g, 24, 40, 160, E8M0)
    dy = torch.randn(24, 40, generator=g).to(torch.bfloat16)
    a, b, d = values(x, xs), values(w, ws), dy.double()
    dx = o.fp8_block_grad_input(dy.to(dev), w, ws).cpu().double()
    dw = o.fp8_block_grad_weight(dy.to(dev), x, xs, torch.float32).cpu().double()
    f = lambda p, q: float((d * (p @ q.T)).sum())   # noqa: E731
    for _ in range(20):
        m, n, k = (int(torch.randint(0, v, (1,), generator=g)) for v in (24, 40, 160))
        p, q = a.clone(), b.clone()
        p[m, k] += 1
        q[n, k] += 1
        step, tol = f(p, b) - f(a, b), 2.0 ** -18 * float((d[m].abs() * b[:, k].abs()).sum()) + 1e-9
        lo, hi = torch.tensor([step - tol, step + tol]).to(torch.bfloat16).tolist()
        assert lo <= float(dx[m, k]) <= hi
        assert abs(f(a, q) - f(a, b) - float(dw[n, k])) <= 2.0 ** -18 * float(
            (d[:, n].abs() * a[:, k].abs()).sum()) + 1e-9


# ---------------------------------------------------------------- refusals, streams
def test_refusals(dev):
    o = ops()
    x, xs, w, ws = fp8_pair(gen(4), 8, 136, 256, E8M0)
    dy = torch.zeros(8, 136, device=dev, dtype=torch.bfloat16)
    bf = torch.zeros(8, 256, device=dev, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        o.fp8_quantize_groups(bf.double())
    with pytest.raises(TypeError, match="scale_dtype"):
        o.fp8_quantize_groups(bf, torch.bfloat16)
    with pytest.raises(ValueError, match="2-D"):
        o.fp8_quantize_groups(bf.view(2, 4, 256))
    with pytest.raises(ValueError, match="2-D"):
        o.fp8_quantize_blocks(bf[:, :0])
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        o.fp8_block_matmul(bf, xs, w, ws)
    with pytest.raises(ValueError, match="takes scales"):
        o.fp8_block_matmul(x, xs[:, :1], w, ws)
    with pytest.raises(TypeError, match="w scales"):
        o.fp8_block_matmul(x, xs, w, ws.double())
    with pytest.raises(ValueError, match="does not multiply"):
        o.fp8_block_matmul(x[:, :128], xs[:, :1], w, ws)
    with pytest.raises(TypeError, match="out_dtype"):
        o.fp8_block_matmul(x, xs, w, ws, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="bias"):
        o.fp8_block_matmul(x, xs, w, ws, bias=bf[0])
    with pytest.raises(TypeError, match="bias"):
        o.fp8_block_matmul(x, xs, w, ws, bias=torch.zeros(136, device=dev, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU only"):
        o.fp8_block_matmul(x.cpu(), xs, w, ws)
    with pytest.raises(RuntimeError, match="GPU only"):
        o.fp8_quantize_groups(bf.cpu())
    with pytest.raises(TypeError, match="bf16"):
        o.fp8_block_grad_input(dy.float(), w, ws)
    with pytest.raises(ValueError, match="output gradient"):
        o.fp8_block_grad_input(dy[:, :8], w, ws)
    with pytest.raises(TypeError, match="x scales"):
        o.fp8_block_grad_weight(dy, x, xs.float())
    with pytest.raises(ValueError, match="output gradient"):
        o.fp8_block_grad_weight(dy[:4], x, xs)
    with pytest.raises(ValueError, match="side by side"):
        o.fp8_silu_mul(bf[:, :255])
    _, _, kept, ks = o.fp8_silu_mul(bf)
    with pytest.raises(ValueError, match="saved codes"):
        o.fp8_silu_mul_backward(bf, kept, ks)
    with pytest.raises(TypeError, match="saved codes"):
        o.fp8_silu_mul_backward(bf[:, :128], kept.view(torch.uint8), ks)


def test_the_current_stream_is_used(dev):
    """On a stream of its own, behind work that the default stream does not wait for."""
    o, g = ops(), gen(41)
    src = heavy(g, 64, 512).to(torch.bfloat16).to(dev)
    w, ws = o.fp8_quantize_blocks((torch.randn(256, 512, generator=g) * 0.02).to(torch.bfloat16).to(dev))
    dy = torch.randn(64, 256, generator=g).to(torch.bfloat16).to(dev)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(src)
        big = torch.randn(4096, 4096, device=dev)
        for _ in range(4):
            big = big @ big * 1e-3
        late.copy_(src)
        x, xs = o.fp8_quantize_groups(late, E8M0)
        y, dw = o.fp8_block_matmul(x, xs, w, ws), o.fp8_block_grad_weight(dy, x, xs)
        dx = o.fp8_block_grad_input(dy, w, ws)
        h = o.fp8_silu_mul(late)
    side.synchronize()
    x2, xs2 = o.fp8_quantize_groups(src, E8M0)
    again = (o.fp8_block_matmul(x2, xs2, w, ws), o.fp8_block_grad_weight(dy, x2, xs2),
             o.fp8_block_grad_input(dy, w, ws), *o.fp8_silu_mul(src))
    for a, b in zip((y, dw, dx, *h), again):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_calls_larger_than_the_cache_equal_their_rows(dev):
    """Calls that move over 256 MB store past the caches; rows are independent, so each equals its own call."""
    o = ops()
    x = torch.randn(8192, 2 * 4992, generator=torch.Generator(device=dev).manual_seed(3), device=dev).to(torch.bfloat16)
    pick = [0, 1, 4095, 8191]
    for op in (lambda t: o.fp8_quantize_groups(t), lambda t: o.fp8_quantize_groups(t, E8M0), o.fp8_silu_mul):
        for a, b in zip(op(x), op(x[pick])):
            assert torch.equal(a[pick].view(torch.uint8), b.view(torch.uint8))
    _, _, kept, ks = o.fp8_silu_mul(x)
    dh = x[:, :4992].contiguous()
    a, b = o.fp8_silu_mul_backward(dh, kept, ks), o.fp8_silu_mul_backward(dh[pick], kept[pick], ks[pick])
    assert torch.equal(a[pick], b)
    w = x.view(-1, 4992)
    c, s = o.fp8_quantize_blocks(w)
    c2, s2 = o.fp8_quantize_blocks(w[1280:1536])
    assert torch.equal(c[1280:1536].view(torch.uint8), c2.view(torch.uint8)) and torch.equal(s[10:12], s2)


@pytest.mark.parametrize("rows,out,cols", [(1, 256, 512), (100, 384, 1024), (300, 300, 301)])
def test_replays_of_a_graph_follow_their_inputs(dev, rows, out, cols):
    """A captured step (split sums and padded copies among it) gives the eager results for every input that is
    put into its buffers, with eager work and synchronizations between the replays."""
    o = ops()
    g = gen(61, rows, out, cols)
    x0 = torch.zeros(rows, cols, dtype=torch.bfloat16, device=dev)
    dy0 = torch.zeros(rows, out, dtype=torch.bfloat16, device=dev)
    w, ws = o.fp8_quantize_blocks(heavy(g, out, cols).to(torch.bfloat16).to(dev))

    def step(x, dy):
        c, s = o.fp8_quantize_groups(x, E8M0)
        return (c, s, o.fp8_block_matmul(c, s, w, ws), o.fp8_block_grad_input(dy, w, ws),
                o.fp8_block_grad_weight(dy, c, s, torch.float32))

    step(x0, dy0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(x0, dy0)
    for _ in range(4):
        x = heavy(g, rows, cols).to(torch.bfloat16).to(dev)
        dy = heavy(g, rows, out).to(torch.bfloat16).to(dev)
        eager = step(x, dy)
        x0.copy_(x)
        dy0.copy_(dy)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_single_rows_of_any_pitch(dev):
    """A matrix of one row (or none) may carry any strides: a transposed column is as good as a row."""
    o = ops()
    g = gen(67)
    w, ws = o.fp8_quantize_blocks(heavy(g, 256, 256).to(torch.bfloat16).to(dev))
    x = heavy(g, 1, 256).to(torch.bfloat16).to(dev)
    column = x.reshape(256, 1).clone().t()
    assert column.stride() == (1, 1)
    for kind in (torch.float32, E8M0):
        c, s = o.fp8_quantize_groups(x, kind)
        c2, s2 = o.fp8_quantize_groups(column, kind)
        assert torch.equal(c.view(torch.uint8), c2.view(torch.uint8)) and torch.equal(s.float(), s2.float())
        y = o.fp8_block_matmul(c, s, w, ws)
        as_column = (t.reshape(-1, 1).clone().t() for t in (c, s))
        assert torch.equal(y, o.fp8_block_matmul(*as_column, w, ws))
    wc, wsc = o.fp8_quantize_blocks(column)
    assert torch.equal(wc.float(), o.fp8_quantize_blocks(x)[0].float())
    h, hs, kept, ks = o.fp8_silu_mul(column)
    for a, b in zip(o.fp8_silu_mul(x), (h, hs, kept, ks)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    dh = heavy(g, 1, 128).to(torch.bfloat16).to(dev)
    want = o.fp8_silu_mul_backward(dh, kept, ks)
    got = o.fp8_silu_mul_backward(*(t.reshape(-1, 1).clone().t() for t in (dh, kept, ks)))
    assert torch.equal(want, got)
    none = torch.empty(256, 0, dtype=torch.bfloat16, device=dev).t()
    c, s = o.fp8_quantize_groups(none)
    assert c.shape == (0, 256) and s.shape == (0, 2)
    assert o.fp8_block_grad_input(none, w, ws).shape == (0, 256)


def test_scales_of_a_wide_pitch(dev):
    """Offsets of a tile's scales that pass 32 bits: 130 rows of scales 2^25 + 2^21 apart, 4.6 GB of address range."""
    o = ops()
    g = gen(71)
    rows, pitch = 130, 2 ** 25 + 2 ** 21
    w, ws = o.fp8_quantize_blocks(heavy(g, 128, 256).to(torch.bfloat16).to(dev))
    c, s = o.fp8_quantize_groups((heavy(g, rows, 256) * torch.exp2(torch.arange(rows) % 40.)[:, None]).to(dev), E8M0)
    far = torch.empty(rows * pitch, dtype=torch.uint8, device=dev).view(E8M0).as_strided((rows, 2), (pitch, 1))
    far.copy_(s)
    assert torch.equal(o.fp8_block_matmul(c, s, w, ws, out_dtype=torch.float32).cpu().isnan(),
                       torch.zeros(rows, 128, dtype=torch.bool))
    check_sum(o.fp8_block_matmul(c, far, w, ws, out_dtype=torch.float32).cpu(), values(c, s) @ values(w, ws).T,
              values(c, s).abs() @ values(w, ws).abs().T, torch.float32)
    dy = heavy(g, rows, 128).to(torch.bfloat16).to(dev)
    check_sum(o.fp8_block_grad_weight(dy, c, far, torch.float32).cpu(), dy.cpu().double().T @ values(c, s),
              dy.cpu().double().abs().T @ values(c, s).abs(), torch.float32)
    del far
    torch.cuda.empty_cache()    # later tests that count free memory do not find these gigabytes in the cache


@pytest.mark.parametrize("rows", [16, 256])
def test_every_e8m0_scale(dev, rows):
    """Every byte as a row's scale, in the few-token kernel and in tiles: 2^(b - 127) exactly, 255 NaN."""
    o = ops()
    for first in range(0, 256, rows):
        b = torch.arange(first, first + rows, dtype=torch.uint8)
        x = torch.ones(rows, 128).to(E4M3).to(dev)
        w = torch.zeros(128, 128)
        w[:, 5] = 1
        ws = torch.ones(1, 1, device=dev)
        y = o.fp8_block_matmul(x, b.view(E8M0)[:, None].to(dev), w.to(E4M3).to(dev), ws, out_dtype=torch.float32).cpu()
        want = torch.exp2(b.double() - 127)
        want[b == 255] = math.nan
        assert torch.equal(y.double().nan_to_num(-1.0), want[:, None].expand(-1, 128).nan_to_num(-1.0))


def test_offsets_past_32_bits(dev):
    """Operands and outputs of more than 2^32 elements' bytes: rows that repeat every 1024 give results that do, and a
    weight gradient of rows that are zero but for the last 1024 is theirs (small integers: every sum is exact)."""
    o = ops()
    g = gen(73)
    period, times, wide = 1024, 512, 8320          # 2^19 rows of 8320: 4.4e9 codes, 8.7e9 bytes of bf16
    rows = period * times

    def base(cols):
        return heavy(g, period, cols).to(torch.bfloat16).to(dev)

    def repeats(t, unit):
        t = t.view(torch.uint8).view(-1, unit * t.shape[-1] * t.element_size())
        return all(torch.equal(t[i], t[0]) for i in (1, t.shape[0] // 2, t.shape[0] - 2, t.shape[0] - 1))

    x = base(wide).repeat(times, 1)
    assert x.numel() * 2 > 2 ** 33
    codes, scales = o.fp8_quantize_groups(x, E8M0)
    assert repeats(codes, period) and repeats(scales, period)
    assert all(repeats(t, r) for t, r in zip(o.fp8_quantize_blocks(x), (period, period // G)))
    h, hs, kept, ks = o.fp8_silu_mul(x)
    assert all(repeats(t, period) for t in (h, hs, kept, ks))
    del h, hs
    dh = base(wide // 2).repeat(times, 1)
    assert repeats(o.fp8_silu_mul_backward(dh, kept, ks), period)
    del dh, kept, ks
    narrow, tall = base(128).repeat(times, 1), heavy(g, wide, 128).to(torch.bfloat16).to(dev)
    w, ws = o.fp8_quantize_blocks(tall.t().contiguous())            # [128, wide]
    v, vs = o.fp8_quantize_blocks(tall)                             # [wide, 128]
    assert repeats(o.fp8_block_matmul(codes, scales, w, ws), period)
    assert repeats(o.fp8_block_matmul(*o.fp8_quantize_groups(narrow), v, vs), period)
    assert repeats(o.fp8_block_grad_input(x, v, vs), period)
    assert repeats(o.fp8_block_grad_input(narrow, w, ws), period)
    del x, codes, scales
    one = torch.full((rows, wide // G), 127, dtype=torch.uint8, device=dev).view(E8M0)
    for out, cols in ((128, wide), (wide, 128)):
        dy = torch.zeros(rows, out, dtype=torch.bfloat16, device=dev)
        dy[-period:] = torch.randint(-8, 9, (period, out), generator=g).to(torch.bfloat16).to(dev)
        c = torch.randint(-8, 9, (period, cols), generator=g).to(torch.float32).to(E4M3).to(dev)
        c = c.view(torch.uint8).repeat(times, 1).view(E4M3)
        e = one[:, :cols // G]
        got = o.fp8_block_grad_weight(dy, c, e, torch.float32)
        assert torch.equal(got, o.fp8_block_grad_weight(dy[-period:], c[-period:], e[-period:], torch.float32))
        del dy, c
    del one, narrow, e, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,out,cols", [(1, 136, 256), (20, 300, 400), (33, 128, 128), (100, 264, 1040), (200, 24, 2064),
                                           (517, 384, 48), (70, 131, 133)])
@pytest.mark.parametrize("off", [16, 3])
def test_only_the_views_are_touched(dev, off, rows, out, cols):
    """Operands and outputs are views into larger buffers: NaN all around the operands reaches no result, and what is
    around the outputs stays as it was."""
    from llmcompressor_amd import _lib as L
    o, lib, g = ops(), L.lib(), gen(79, rows, out, cols, off)
    x, xs, w, ws = fp8_pair(g, rows, out, cols, E8M0)
    dy = heavy(g, rows, out).to(torch.bfloat16).to(dev)

    def inside(shape, dtype, fill):
        pitch = (shape[1] + off + 47) // 16 * 16 + (off % 16)
        buf = torch.full((shape[0] + 4, pitch), fill, dtype=torch.float32, device=dev).to(dtype)
        return buf, buf[2:2 + shape[0], off:off + shape[1]]

    def poisoned(t):
        buf, v = inside(t.shape, t.dtype, float("nan"))
        v.copy_(t)
        return v

    def unchanged(buf, v):
        v.fill_(7)
        return bool((buf.float() == 7).all())
    px, pxs, pw, pws, pdy = (poisoned(t) for t in (x, xs, w, ws, dy))
    a, b, d = values(x, xs), values(w, ws), dy.cpu().double()
    st = L.stream_of(x)
    for dtype, code in ((torch.float32, L.F32), (torch.bfloat16, L.BF16), (torch.float16, L.F16)):
        for query, shape, want, mags, call in (
                ("mi355q_fp8_block_matmul", (rows, out), a @ b.T, a.abs() @ b.abs().T,
                 lambda v, p, n: (px.data_ptr(), px.stride(0), pxs.data_ptr(), L.SCALE_E8M0, pxs.stride(0), pw.data_ptr(),
                                  pw.stride(0), pws.data_ptr(), pws.stride(0), None, 0, v.data_ptr(), code, v.stride(0),
                                  rows, out, cols, p, n, st)),
                ("mi355q_fp8_block_grad_input", (rows, cols), d @ b, d.abs() @ b.abs(),
                 lambda v, p, n: (pdy.data_ptr(), pdy.stride(0), pw.data_ptr(), pw.stride(0), pws.data_ptr(),
                                  pws.stride(0), v.data_ptr(), v.stride(0), rows, out, cols, p, n, st)),
                ("mi355q_fp8_block_grad_weight", (out, cols), d.T @ a, d.abs().T @ a.abs(),
                 lambda v, p, n: (pdy.data_ptr(), pdy.stride(0), px.data_ptr(), px.stride(0), pxs.data_ptr(),
                                  pxs.stride(0), v.data_ptr(), code, v.stride(0), rows, out, cols, p, n, st))):
            if query.endswith("grad_input") and dtype != torch.bfloat16:
                continue
            for room in (0, getattr(lib, query + "_workspace_size")(rows, out, cols)):
                scratch = torch.full((room + 256,), 255, dtype=torch.uint8, device=dev)
                buf, v = inside(shape, dtype, 7)
                L.check(getattr(lib, query)(*call(v, scratch.data_ptr() if room else None, room)))
                check_sum(v.contiguous(), want, mags, dtype)
                assert unchanged(buf, v), query
                assert bool((scratch[room:] == 255).all())


@pytest.mark.parametrize("rows,cols", [(1, 128), (3, 300), (130, 392), (17, 16), (5, 7)])
@pytest.mark.parametrize("off", [16, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantizers_touch_only_their_views(dev, rows, cols, off, dtype):
    """The same of the quantizers and the gated activation: NaN around the inputs, a byte pattern around the outputs."""
    from llmcompressor_amd import _lib as L
    o, lib, g = ops(), L.lib(), gen(83, rows, cols, off)
    code, st, groups = L.BF16 if dtype == torch.bfloat16 else L.F32, L.stream_of(torch.zeros(1, device=dev)), -(-cols // G)

    def poisoned(t):
        buf = torch.full((t.shape[0] + 4, t.shape[1] + 2 * off), float("nan"), device=dev).to(t.dtype)
        v = buf[2:-2, off:off + t.shape[1]]
        v.copy_(t)
        return v

    def guarded(r, c, size):
        buf = torch.full((r + 4, (c + 2 * off) * size), 0xA5, dtype=torch.uint8, device=dev)
        return buf, buf[2:-2, off * size:(off + c) * size]

    def check(outs, want):
        for (buf, v), w in zip(outs, want):
            assert torch.equal(v.contiguous(), w.contiguous().view(torch.uint8).reshape(v.shape))
            v.fill_(0xA5)
            assert bool((buf == 0xA5).all())
    x = heavy(g, rows, 2 * cols).to(dtype).to(dev)
    p, half = poisoned(x), x[:, :cols].contiguous()
    q = poisoned(half)
    for kind, num, size in ((torch.float32, L.SCALE_F32, 4), (E8M0, L.SCALE_E8M0, 1)):
        (cb, c), (sb, s) = outs = guarded(rows, cols, 1), guarded(rows, groups, size)
        L.check(lib.mi355q_fp8_quantize_groups(q.data_ptr(), code, rows, cols, q.stride(0), c.data_ptr(), c.stride(0),
                                               s.data_ptr(), num, s.stride(0) // size, st))
        check(outs, o.fp8_quantize_groups(half, kind))
    (cb, c), (sb, s) = outs = guarded(rows, cols, 1), guarded(-(-rows // G), groups, 4)
    L.check(lib.mi355q_fp8_quantize_blocks(q.data_ptr(), code, rows, cols, q.stride(0), c.data_ptr(), c.stride(0),
                                           s.data_ptr(), s.stride(0) // 4, st))
    check(outs, o.fp8_quantize_blocks(half))
    want = o.fp8_silu_mul(x)
    flat = [torch.full((2 + rows * n, 1), 0xA5, dtype=torch.uint8, device=dev) for n in (groups, 2 * groups)]
    outs = guarded(rows, cols, 1), (flat[0], flat[0][1:-1]), guarded(rows, 2 * cols, 1), (flat[1], flat[1][1:-1])
    h, hs, kept, ks = (v for _, v in outs)
    L.check(lib.mi355q_fp8_silu_mul(p.data_ptr(), code, rows, cols, p.stride(0), h.data_ptr(), h.stride(0), hs.data_ptr(),
                                    kept.data_ptr(), kept.stride(0), ks.data_ptr(), st))
    check(outs, want)
    dh = heavy(g, rows, cols).to(dtype).to(dev)
    pd, pk, ps = poisoned(dh), poisoned(want[2]), poisoned(want[3])
    size = dh.element_size()
    (db, d), = outs = guarded(rows, 2 * cols, size),
    L.check(lib.mi355q_fp8_silu_mul_backward(pd.data_ptr(), code, rows, cols, pd.stride(0), pk.data_ptr(), pk.stride(0),
                                             ps.data_ptr(), ps.stride(0), d.data_ptr(), d.stride(0) // size, st))
    check(outs, (o.fp8_silu_mul_backward(dh, want[2], want[3]),))
