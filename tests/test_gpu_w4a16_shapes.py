"""4-bit products at the sizes that take each of the kernels' shapes, with sums long enough that their loops over
whole steps go round: every cut of a call of few rows (rows per tile, column tiles, waves), and experts' row
tiles in bands of several sizes.  Compared with the definition in 64 bits on the same device.

Tolerances.  As for shorter sums, with the chain counted anew: a wave adds up to 12 steps of four instructions, of
eight roundings each, every one scaled and added (one more), then 8 waves and 8 workgroups: 12 * 4 * 9 + 16
is below 512, so a value is within 512 2^-24 L = 2^-15 L of the exact one before it is rounded (half a step), L = sum
|x| s (q + z), MXFP4 sum |x| |w|.  Splits make the chain shorter.  Tiles of many rows: up to 3 steps here.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LEVELS = [0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6]


def ops():
    from llmcompressor_amd import ops as o
    return o


def words(codes, dim):
    """Codes 0 .. 15 packed eight to an int32 along `dim`, lowest first; the last word filled up with junk."""
    codes = codes.movedim(dim, -1)
    codes = torch.nn.functional.pad(codes, (0, -codes.shape[-1] % 8), value=13).unflatten(-1, (-1, 8))
    w = torch.zeros(codes.shape[:-1], dtype=torch.int32, device=codes.device)
    for i in range(8):
        w |= codes[..., i].int() << (4 * i)
    return w.movedim(-1, dim).contiguous()


class Weight:
    """Random 4-bit weights [*lead, out, cols] on the device: the tensors of a checkpoint, and exact values on demand."""

    def __init__(self, seed, lead, out, cols, kind, group, scale_dtype=BF16):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.kind, self.cols, self.group = kind, cols, group
        self.codes = torch.randint(0, 16, (*lead, out, cols), generator=g, device="cuda", dtype=torch.uint8)
        n = cols // 32 if kind == "mxfp4" else -(-cols // (group or cols))
        if kind == "mxfp4":
            self.s = torch.randint(110, 125, (*lead, out, n), generator=g, device="cuda").to(torch.uint8)
            packed, z = self.codes[..., 0::2] | (self.codes[..., 1::2] << 4), None
        else:
            self.s = (torch.rand(*lead, out, n, generator=g, device="cuda") * 0.02 + 1e-3).to(scale_dtype)
            self.z = torch.full_like(self.s, 8, dtype=torch.uint8)
            z = None
            if kind == "int4z":
                self.z = torch.randint(0, 16, self.z.shape, generator=g, device="cuda", dtype=torch.uint8)
                z = words(self.z, -2)
            packed = words(self.codes, -1)
        self.parts = packed, self.s, z

    def exact(self, e=None):
        """(values, sizes) in 64 bits of expert e's weight."""
        codes, s = (self.codes, self.s) if e is None else (self.codes[e], self.s[e])
        wide = 32 if self.kind == "mxfp4" else self.group or self.cols
        spread = lambda t: t.double().repeat_interleave(wide, -1)[..., :self.cols]     # noqa: E731
        if self.kind == "mxfp4":
            v = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")[codes.long()] * torch.exp2(spread(s) - 127)
            return v, v.abs()
        z = spread(self.z if e is None else self.z[e])
        return (codes.double() - z) * spread(s), (codes.double() + z) * spread(s)


def close(got, x, values, sizes, bias=None, gated=False):
    x = x.double()
    y, tol = x @ values.T.contiguous(), 2.0 ** -15 * (x.abs() @ sizes.T.contiguous())
    if bias is not None:
        y = y + bias.double()
        tol = tol + 2.0 ** -23 * y.abs()
    if gated:
        (a, b), (da, db) = y.chunk(2, 1), tol.chunk(2, 1)
        silu = a * torch.sigmoid(a)
        y = silu * b
        tol = 1.1 * da * (b.abs() + db) + silu.abs() * db + 2.0 ** -20 * y.abs()
    half = torch.finfo(got.dtype).eps / 2
    limit = tol + half * (y.abs() + tol) + torch.finfo(got.dtype).smallest_normal * half
    err = (got.double() - y).abs()
    assert got.shape == y.shape and bool((err <= limit).all()), f"{float((err / limit).max()):.2f} of the bound"


FORMATS = [("int4", 128, BF16, BF16), ("int4", 64, F16, F16), ("int4", 32, BF16, F32), ("int4", 256, BF16, BF16),
           ("int4", None, F16, BF16), ("int4z", 32, BF16, BF16), ("int4z", 128, F16, F32), ("mxfp4", 32, BF16, None),
           ("mxfp4", 32, F16, None)]
NAMES = [f"{k}-{g}-{str(t)[6:]}" for k, g, t, _ in FORMATS]

# rows, out, whole steps, gated: what follows is the cut that the call takes (rows per tile, column tiles, waves) and the
# whole steps of a wave, of which `2 D` and a remainder make the loop go round
SHAPES = [
    (1, 16500, 23, False),      # 4 rows, 1, 2: 11 or 12 steps, four in flight
    (4, 16500, 23, False),
    (3, 6200, 46, False),       # 4 rows, 1, 4: 11 or 12
    (2, 600, 45, False),        # 4 rows, 1, 8: 5 or 6, two in flight
    (1, 33000, 23, True),       # 4 rows, 2, 2: 11 or 12
    (4, 12400, 23, True),       # 4 rows, 2, 4: 5 or 6
    (2, 1040, 45, True),        # 4 rows, 2, 8: 5 or 6
    (5, 12400, 23, False),      # 16 rows, 4, 4: 5 or 6
    (16, 12400, 23, True),
    (11, 8300, 23, False),      # 16 rows, 2, 4: 5 or 6
    (7, 530, 23, True),
    (16, 530, 45, False),       # 16 rows, 1, 8: 5 or 6
    (23, 12400, 27, False),     # 32 rows, 4, 8: 3 or 4, one in flight
    (32, 530, 72, False),       # the same, sums over several workgroups
    (64, 12400, 27, True),      # 64 rows, 4, 8: 3 or 4
    (33, 530, 72, True),
]


@pytest.mark.parametrize("rows,out,steps,gated", SHAPES)
@pytest.mark.parametrize("kind,group,dtype,scale_dtype", FORMATS, ids=NAMES)
def test_cuts_of_few_rows(rows, out, steps, gated, kind, group, dtype, scale_dtype):
    cols = 128 * steps + (32 if kind == "mxfp4" else 41)         # a shorter last step
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, cols, generator=g, device="cuda")
         * torch.randn(cols, generator=g, device="cuda").exp()).to(dtype)
    w = Weight(out + rows, (), out, cols, kind, group, scale_dtype)
    b = torch.randn(out, generator=g, device="cuda").to(dtype) if rows % 2 else None
    y = ops().w4a16_matmul(x, *w.parts, group_size=group, bias=b, gated=gated, out_dtype=F32)
    close(y, x, *w.exact(), b, gated)


def check_experts(pairs, experts, out, cols, kind, group, dtype, scale_dtype, gated, gather):
    """`pairs` rows to `experts` experts, a tenth of them to none; of several one has none, one a fifth of all."""
    g = torch.Generator().manual_seed(pairs + out)
    ids = torch.randint(0, experts, (pairs,), generator=g)
    if experts > 2:
        ids[torch.rand(pairs, generator=g) < 0.2] = experts // 2
        ids[ids == experts // 3] = experts
    ids[torch.rand(pairs, generator=g) < 0.1] = experts
    offsets = torch.cat([torch.zeros(1).long(), torch.bincount(ids, minlength=experts + 1)[:experts].cumsum(0)])
    rows = torch.randint(0, max(1, pairs // 3), (pairs,), generator=g).int().cuda()
    n = max(1, pairs // 3) if gather else pairs
    x = torch.randn(n, cols, generator=g).to(dtype).cuda()
    w = Weight(pairs, (experts,), out, cols, kind, group, scale_dtype)
    y = ops().w4a16_experts_matmul(x, rows if gather else None, offsets.cuda(), *w.parts, group_size=group, gated=gated,
                                   out_dtype=F32)
    ends = offsets.tolist()
    for e in range(experts):
        a, b = ends[e], ends[e + 1]
        if a < b:
            close(y[a:b], x[rows[a:b].long()] if gather else x[a:b], *w.exact(e), None, gated)
    assert not y[ends[-1]:].any()


@pytest.mark.parametrize("pairs,experts,out,steps,gated", [
    (8, 128, 1600, 23, True),       # 4 rows, 2, 4
    (32, 128, 640, 23, False),      # 4 rows, 1, 2
    (32, 128, 1040, 23, True),      # 4 rows, 2, 2
    (410, 128, 560, 7, False),      # 16 rows, 2, 1: 7 steps, two in flight
    (410, 128, 560, 7, True),
    (61, 16, 1000, 23, False),      # 16 rows, 4, 4
    (49, 3, 300, 27, False),        # 32 rows, 4, 8
    (50, 1, 300, 27, True),         # 64 rows, 4, 8
])
@pytest.mark.parametrize("kind,group,dtype,scale_dtype",
                         [FORMATS[i] for i in (0, 2, 5, 6, 7, 8)], ids=[NAMES[i] for i in (0, 2, 5, 6, 7, 8)])
def test_cuts_of_few_rows_of_experts(pairs, experts, out, steps, gated, kind, group, dtype, scale_dtype):
    cols = 128 * steps + (32 if kind == "mxfp4" else 41)
    check_experts(pairs, experts, out, cols, kind, group, dtype, scale_dtype, gated, pairs % 2 == 0)


# Row tiles of experts, of 32, 64 and 128 rows, in bands of 3, 5 and 8
@pytest.mark.parametrize("pairs,experts,out", [
    (2500, 128, 600),               # 32 rows, 207 tiles at the most: bands of 3
    (8000, 128, 600),               # 32 rows, 379: bands of 5
    (12600, 128, 600),              # 32 rows, 522: bands of 8
    (26000, 200, 600),              # 64 rows, 607: bands of 8
    (53000, 100, 600),              # 128 rows, 515: bands of 8
])
@pytest.mark.parametrize("kind,group,dtype,gated", [("int4", 128, BF16, True), ("int4z", 32, F16, False),
                                                    ("mxfp4", 32, BF16, False), ("mxfp4", 32, F16, True)])
def test_bands_of_experts_tiles(pairs, experts, out, kind, group, dtype, gated):
    check_experts(pairs, experts, out, 288, kind, group, dtype, BF16, gated, not gated)


# Tiles of many rows: rows, out, gated; the tile's rows and columns
TILES = [
    (200, 1000, False),     # 32 x 128
    (200, 1000, True),      # 32 x 256
    (700, 3000, False),     # 64 x 128
    (1290, 5100, False),    # 64 x 256
    (1290, 5100, True),
    (2050, 6700, False),    # 128 x 256
    (2050, 6700, True),
]


@pytest.mark.parametrize("rows,out,gated", TILES)
@pytest.mark.parametrize("kind,group,dtype,scale_dtype", FORMATS + [("int4", 64, BF16, F32), ("int4z", 32, F16, F16)],
                         ids=NAMES + ["int4-64-bf16-f32", "int4z-32-f16-f16"])
def test_tiles_of_several_steps(rows, out, gated, kind, group, dtype, scale_dtype):
    """Five whole steps and a shorter one: eight instructions a step, of eight roundings, stay below the bound."""
    cols = 640 + (32 if kind == "mxfp4" else 41)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, cols, generator=g, device="cuda")
         * torch.randn(cols, generator=g, device="cuda").exp()).to(dtype)
    w = Weight(out + rows, (), out, cols, kind, group, scale_dtype)
    b = torch.randn(out, generator=g, device="cuda").to(dtype)
    y = ops().w4a16_matmul(x, *w.parts, group_size=group, bias=b, gated=gated, out_dtype=F32)
    close(y, x, *w.exact(), b, gated)


@pytest.mark.parametrize("pairs,experts,out", [(180, 4, 400), (420, 5, 600), (1500, 7, 600), (3300, 5, 600)],
                         ids=["32x128", "32x256", "64x256", "128x256"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind,group,dtype,scale_dtype", FORMATS, ids=NAMES)
def test_tiles_of_experts_of_several_steps(pairs, experts, out, gated, kind, group, dtype, scale_dtype):
    check_experts(pairs, experts, out, 640 + (32 if kind == "mxfp4" else 41), kind, group, dtype, scale_dtype, gated,
                  not gated)
