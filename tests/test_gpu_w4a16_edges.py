"""4-bit products where the definition says what is easily got wrong: rows of no expert beside a bias, rows before the
first expert's, gates at the ends of fp32's range, every byte that MXFP4's scales can have."""
import ctypes as C

import pytest
import torch

from test_gpu_w4a16 import BF16, E2M1, F16, F32, Weight, close, expected, gen, ops

pytestmark = pytest.mark.gpu


def entry(x, w, fmt, offsets, experts, group, out, gated, y, bias=None, rows_index=None, n_x=None, workspace=True):
    """The C entry, for what the Python functions do not pass."""
    from llmcompressor_amd import _lib as L
    dt = {BF16: L.BF16, F16: L.F16, F32: L.F32}
    p, s, z = w
    cols, rows = x.shape[1], y.shape[0]
    n_x = x.shape[0] if n_x is None else n_x
    need = L.lib().mi355q_w4a16_matmul_workspace_size(n_x, rows, experts, out, cols, fmt, group) if workspace else 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    per = lambda t: 0 if t is None or t.dim() < 3 else t.stride(0)     # noqa: E731
    L.check(L.lib().mi355q_w4a16_matmul(
        x.data_ptr(), dt[x.dtype], n_x, x.stride(0), L.ptr(rows_index), L.ptr(offsets), experts, p.data_ptr(), fmt,
        p.stride(-2) * p.element_size(), per(p) * p.element_size(), s.data_ptr(), dt.get(s.dtype, L.BF16), s.stride(-2),
        per(s), L.ptr(z), 0 if z is None else z.stride(-2), per(z), group, L.ptr(bias),
        dt[bias.dtype] if bias is not None else 0, int(gated), y.data_ptr(), dt[y.dtype], y.stride(0), rows, out, cols,
        L.ptr(ws), C.c_size_t(need), L.stream_of(x)))
    torch.cuda.synchronize()
    return y


# ---------------------------------------------------------------- rows of no expert
# 9, 40: tiles of few rows; 200, 400: of many; 200 without a workspace: few again
@pytest.mark.parametrize("rows,workspace", [(3, True), (9, True), (40, True), (200, True), (200, False), (400, True)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind", ["int4", "int4z", "mxfp4"])
def test_rows_of_no_expert_have_no_bias(rows, workspace, gated, kind):
    from llmcompressor_amd import _lib as L
    g = gen("bias", rows, gated)
    out, cols = 96, 256
    x = torch.randn(rows, cols, generator=g).to(BF16)
    w = Weight(g, out, cols, kind, 32, experts=2)
    b = torch.randn(out, generator=g).to(BF16)
    ends = [0, rows // 3, rows - rows // 3]
    y = torch.full((rows, out // 2 if gated else out), float("nan"), dtype=BF16, device="cuda")
    entry(x.cuda(), w.cuda(), L.W4_MXFP4 if kind == "mxfp4" else L.W4_INT4, torch.tensor(ends).cuda(), 2, 32, out, gated,
          y, b.cuda(), workspace=workspace)
    for e in range(2):
        close(y[ends[e]:ends[e + 1]], *expected(x[ends[e]:ends[e + 1]], w.values[e], w.sizes[e], b, gated))
    assert not y[ends[-1]:].any()


@pytest.mark.parametrize("rows", [3, 40, 200, 400])
@pytest.mark.parametrize("experts", [1, 3, 70])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_before_the_first_expert_are_zeros(rows, experts, gated):
    """Offsets of a part of the experts: others own the rows before them, and the rows behind."""
    from llmcompressor_amd import _lib as L
    g = gen("before", rows, experts)
    out, cols = 64, 256
    x = torch.randn(rows, cols, generator=g).to(BF16)
    w = Weight(g, out, cols, "int4", 128, experts=experts)
    first, last = rows // 2, rows - rows // 4
    ends = sorted(torch.randint(first, last + 1, (experts - 1,), generator=g).tolist())
    ends = [first, *ends, last]
    for n in (1, experts):
        part = torch.tensor(ends[:n] + [last])
        y = torch.full((rows, out // 2 if gated else out), float("nan"), dtype=BF16, device="cuda")
        p = [None if t is None else t[:n] for t in w.cuda()]
        entry(x.cuda(), p, L.W4_INT4, part.cuda(), n, 128, out, gated, y)
        for e in range(n):
            a, b = int(part[e]), int(part[e + 1])
            if a < b:
                close(y[a:b], *expected(x[a:b], w.values[e], w.sizes[e], None, gated))
        assert not y[:first].any() and not y[last:].any(), n


@pytest.mark.parametrize("rows", [1, 20, 700])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_x_without_rows(rows, gated, out_dtype):
    """No row of x is there: every row of y is zeros, whatever the index says, and x is not read."""
    from llmcompressor_amd import _lib as L
    w = Weight(gen("none"), 40, 128, "int4", 128, experts=3)
    x = torch.empty(0, 128, dtype=BF16, device="cuda")
    index = torch.arange(rows, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, rows // 2, rows // 2, rows], device="cuda")
    y = ops().w4a16_experts_matmul(x, index, offsets, *w.cuda(), gated=gated, out_dtype=out_dtype)
    assert y.shape == (rows, 20 if gated else 40) and not y.any()
    wide = torch.full((rows, 50), float("nan"), dtype=out_dtype, device="cuda")      # a pitch, and a bias
    b = torch.ones(40, dtype=BF16, device="cuda")
    entry(x, w.cuda(), L.W4_INT4, offsets, 3, 128, 40, gated, wide[:, :y.shape[1]], b, index)
    assert not wide[:, :y.shape[1]].any() and bool(wide[:, y.shape[1]:].isnan().all())


# ---------------------------------------------------------------- workspaces
@pytest.mark.parametrize("cols,kind", [(512, "int4"), (520, "int4z"), (544, "mxfp4")])
@pytest.mark.parametrize("rows", [130, 700])
def test_workspace_without_a_copy_of_x(rows, cols, kind):
    """Aligned operands: the smaller size is enough, nothing is written behind it, and the result is that of the larger."""
    from llmcompressor_amd import _lib as L
    g = gen("in place", rows, cols)
    x = torch.randn(rows, cols, generator=g).to(BF16)
    w = Weight(g, 300, cols, kind, 32)
    fmt = L.W4_MXFP4 if kind == "mxfp4" else L.W4_INT4
    need = L.lib().mi355q_w4a16_matmul_workspace_size_in_place(rows, rows, 1, 300, cols, fmt, 32)
    xc, (p, s, z) = x.cuda(), w.cuda()

    def run(size, ws):
        y = torch.empty(rows, 300, dtype=BF16, device="cuda")
        L.check(L.lib().mi355q_w4a16_matmul(
            xc.data_ptr(), L.BF16, rows, cols, None, None, 1, p.data_ptr(), fmt, p.stride(0) * p.element_size(), 0,
            s.data_ptr(), L.BF16, s.stride(0), 0, L.ptr(z), 0 if z is None else z.stride(0), 0, 32, None, 0, 0, y.data_ptr(),
            L.BF16, 300, rows, 300, cols, ws.data_ptr(), C.c_size_t(size), L.stream_of(xc)))
        return y

    ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
    y = run(need, ws)
    close(y, *expected(x, w.values, w.sizes))
    assert bool((ws[need:] == 77).all()) and not bool((ws[:need] == 77).all())
    full = L.lib().mi355q_w4a16_matmul_workspace_size(rows, rows, 1, 300, cols, fmt, 32)
    assert torch.equal(y, run(full, torch.empty(full, dtype=torch.uint8, device="cuda")))


def test_ordinary_calls_do_not_take_the_memory_of_a_copy_of_x():
    g = gen("memory")
    x = torch.randn(20000, 4096, device="cuda").to(BF16)
    parts = Weight(g, 64, 4096, "int4", 128).cuda()
    ops().w4a16_matmul(x, *parts)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops().w4a16_matmul(x, *parts)
    assert torch.cuda.max_memory_allocated() - before < x.numel()      # half of x's bytes


# ---------------------------------------------------------------- the ends of the range
def one_gate(dtype, gate, rows):
    """(x, packed, scales): MXFP4, of 32 columns of gate and 32 of up, whose gates are `gate` in every row and whose
    ups are 1."""
    exponent = 0 if dtype == BF16 else 112                       # fp16 activations end at 65504
    x = torch.zeros(rows, 64, dtype=dtype)
    x[:, 0], x[:, 32] = gate * 2.0 ** -exponent, 1
    codes = torch.zeros(2, 64, dtype=torch.uint8)
    codes[0, 0] = codes[1, 32] = 2                               # the code of 1
    s = torch.tensor([[127 + exponent, 127], [127, 127]], dtype=torch.uint8)
    return x, codes[:, 0::2] | (codes[:, 1::2] << 4), s


@pytest.mark.parametrize("rows", [2, 9, 40, 130])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("gate", [3.3e38, 2.4e38, 2.3e38, 1e30, 1e5])
def test_gates_at_the_ends_of_the_range(rows, dtype, gate):
    """silu(gate) is the gate far above zero and 0 far below, up to fp32's largest numbers; the quotient's and the
    product's roundings are within 2^-20 of the value."""
    x, p, s = one_gate(dtype, gate, rows)
    want = x[0, 0].double() * (1.0 if dtype == BF16 else 2.0 ** 112)
    for out_dtype in (F32, BF16):
        y = ops().w4a16_matmul(x.cuda(), p.cuda(), s.cuda(), gated=True, out_dtype=out_dtype).cpu().double()
        bound = 2.0 ** -20 + torch.finfo(out_dtype).eps / 2
        assert bool(((y - want).abs() <= bound * want).all()), y.flatten()[:3]
        y = ops().w4a16_matmul((-x * (torch.arange(64) < 32) + x * (torch.arange(64) >= 32)).cuda(), p.cuda(), s.cuda(),
                               gated=True, out_dtype=out_dtype).cpu()
        assert not y.any(), y.flatten()[:3]


def test_gates_of_infinity():
    """An infinite gate (bf16: the sum passes fp32) stays one; a gate of -infinity is NaN or 0, never something else."""
    x, p, s = one_gate(BF16, 3.3e38, 4)
    s[0, 0] = 129                                                # times 4
    y = ops().w4a16_matmul(x.cuda(), p.cuda(), s.cuda(), gated=True, out_dtype=F32).cpu()
    assert bool((y == float("inf")).all())
    x[:, 0] *= -1
    y = ops().w4a16_matmul(x.cuda(), p.cuda(), s.cuda(), gated=True, out_dtype=F32).cpu()
    assert bool(((y == 0) | y.isnan()).all())


@pytest.mark.parametrize("rows", [1, 8, 40, 130])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
def test_every_scale_of_mxfp4(rows, dtype):
    """Every byte e as 2^(e - 127), a row of w each, with all codes; activations that bring the results back into the
    range (a power of two, by bytes in turn).  With bf16 activations a weight is a bf16 number, so those of 2^128 and
    more (bytes 253 and 254) are infinite there.  255 is NaN."""
    g = gen("bytes", rows)
    codes = torch.stack([torch.randperm(16, generator=g).repeat(2) for _ in range(255)])
    codes[:, 1] = 7                                              # a code of 6
    e = torch.arange(255)
    packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8)
    values = E2M1[codes] * torch.exp2(e.double() - 127)[:, None]
    nan = ops().w4a16_matmul(torch.ones(rows, 32, dtype=dtype).cuda(), packed[:9].cuda(),
                             torch.full((9, 1), 255, dtype=torch.uint8).cuda())
    assert bool(nan.isnan().all())
    mantissas = torch.randint(-127, 128, (rows, 32), generator=g).double()
    top = 15 if dtype == F16 else 127
    for lo in range(0, 255, 16):
        # |sums| between 2^-126 (normal numbers) and 2^127 for bytes lo .. lo + 15, as far as x's type goes
        power = max(-14 if dtype == F16 else -100, min(top - 8, 127 - lo - 8))
        x = (mantissas * 2.0 ** power).to(dtype)
        part = slice(lo, min(lo + 16, 255))
        y = ops().w4a16_matmul(x.cuda(), packed[part].cuda(), e[part, None].to(torch.uint8).cuda(), out_dtype=F32).cpu()
        want = x.double() @ values[part].T
        # 33 roundings at most, and half a step of subnormal numbers at each
        tol = 33 * (2.0 ** -24 * (x.double().abs() @ values[part].abs().T) + 2.0 ** -150)
        over = (E2M1[codes[part]].abs().double() * torch.exp2(e[part].double() - 127)[:, None] >= 2.0 ** 128).any(1)
        if dtype == BF16 and over.any():
            assert e[part][over].tolist() == [253, 254] and not torch.isfinite(y[:, over]).any()
            y, want, tol = y[:, ~over], want[:, ~over], tol[:, ~over]
        fits = (want.abs() + tol < 3.4e38)
        bad = ((y.double() - want).abs() > tol) & fits
        assert not bad.any(), (lo, e[part][bad.any(0)[:16].nonzero().view(-1)].tolist()
                               if bad.shape[1] == 16 else int(bad.sum()))
