"""Layers on 4-bit weights from modules that the modifiers quantized, experts run as
they are served, and the experts' list on sorted tokens.

Tolerances.  A product is within 2^-18 of L = sum |x| (|w| + 8 s) of the exact one
(a chain of at most 64 fp32 roundings, the zero point's part included; 15 s where zero
points are stored) plus half a step of its type.  A mixture of experts adds: the
inner activation's half step times the down projection, and the combination's top
roundings.
"""
import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from llmcompressor_amd import GPTQModifier, QuantizationModifier, W4A16Experts, W4A16Linear, moe, save
from llmcompressor_amd.moe import LinearExperts, moe_calibration_context, route_tokens
from oracle import pack as opack

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def half_step(t):
    return torch.finfo(t).eps / 2


def values(module):
    """(exact values, scales spread over the columns) of a quantized Linear, from what a checkpoint would hold."""
    t = {k: v.cpu() for k, v in save.compress_module(module).items()}
    rows, cols = module.weight.shape
    if t["weight_packed"].dtype == torch.uint8:
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
        p = t["weight_packed"].long()
        codes = grid[torch.stack([p & 15, p >> 4], -1).view(rows, cols)]
        s = torch.exp2(t["weight_scale"].double() - 127).repeat_interleave(32, 1)
        return codes * s, s
    q = torch.from_numpy(opack.unpack_from_int32(t["weight_packed"].numpy(), cols, 4).astype(np.float64))
    groups = t["weight_scale"].shape[1]
    idx = t["weight_g_idx"].long() if "weight_g_idx" in t else torch.arange(cols) // (cols // groups)
    s = t["weight_scale"].double()[:, idx]
    if "weight_zero_point" in t:
        z = opack.unpack_from_int32(np.ascontiguousarray(t["weight_zero_point"].numpy().T), rows, 4).T
        q = q - torch.from_numpy(z.astype(np.float64))[:, idx]
    return q * s, s


def product(x, v, s):
    x = x.double()
    return x @ v.T, 2.0 ** -18 * (x.abs() @ (v.abs() + 15 * s).T)


def close(got, want, tol):
    got = got.cpu()
    h = half_step(got.dtype)
    err, limit = (got.double() - want).abs(), tol + h * (want.abs() + tol) + 1e-30
    assert got.shape == want.shape and bool((err <= limit).all()), float((err / limit).max())


class One(torch.nn.Module):
    def __init__(self, out, cols, bias, dtype, seed):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        self.proj = torch.nn.Linear(cols, out, bias=bias)
        with torch.no_grad():
            self.proj.weight.copy_(torch.randn(out, cols, generator=g) * 0.02)
        self.to(dtype).cuda()

    def forward(self, x):
        return self.proj(x)


@pytest.mark.parametrize("scheme", ["W4A16", "W4A16_ASYM", "MXFP4A16"])
@pytest.mark.parametrize("rows", [(1,), (3, 7), (130,)])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_from_a_quantized_module(scheme, rows, bias):
    m = One(200, 512, bias, BF16, 1)
    QuantizationModifier(scheme=scheme).apply(m)
    lin = W4A16Linear.from_module(m.proj)
    x = torch.randn(*rows, 512, generator=torch.Generator().manual_seed(2)).to(BF16)
    want, tol = product(x.reshape(-1, 512), *values(m.proj))
    if bias:
        want = want + m.proj.bias.detach().cpu().double()
        tol = tol + 2.0 ** -23 * want.abs()
    y = lin(x.cuda())
    assert y.shape == (*rows, 200) and y.dtype == BF16
    close(y.reshape(-1, 200), want, tol)
    # from the tensors of a checkpoint; types survive a conversion of the module
    t = save.compress_module(m.proj)
    again = W4A16Linear(t["weight_packed"], t["weight_scale"], t.get("weight_zero_point"),
                        32 if scheme.startswith("MX") else 128, m.proj.bias).to(F16)
    assert again.linear.weight_packed.dtype == t["weight_packed"].dtype
    assert again.linear.weight_scale.dtype == t["weight_scale"].dtype


@pytest.mark.parametrize("rows", [2, 150])
def test_linear_with_activation_ordering_by_groups(rows):
    m = One(96, 512, False, BF16, 3)
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(2048, 512, generator=g) * torch.exp(torch.randn(512, generator=g))).to(BF16)
    GPTQModifier(scheme="W4A16", actorder="group").apply(m, [x.cuda()])
    assert not torch.equal(m.proj.weight_g_idx.cpu().long(), torch.arange(512) // 128)
    close(W4A16Linear.from_module(m.proj)(x[:rows].cuda()), *product(x[:rows], *values(m.proj)))


def quantized_experts(scheme, n, hidden, inter, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = [(torch.randn(*s, generator=g, device="cuda") * 0.05).to(BF16)
         for s in ((n, inter, hidden), (n, inter, hidden), (n, hidden, inter))]
    experts = LinearExperts.from_stacked(*w)
    QuantizationModifier(scheme=scheme).apply(experts)
    return experts


@pytest.mark.parametrize("scheme", ["W4A16", "W4A16_ASYM", "MXFP4A16"])
@pytest.mark.parametrize("tokens,top", [(1, 4), (9, 2), (300, 3)])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
def test_experts_as_they_are_served(scheme, tokens, top, dtype):
    n, hidden, inter = 7, 256, 384
    experts = quantized_experts(scheme, n, hidden, inter)
    served = W4A16Experts.from_experts(experts)
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=g).to(dtype)
    weights, ids = torch.softmax(torch.randn(tokens, n, generator=g), 1).topk(top)
    ids[-1, -1] = -1                                            # padding takes no part
    y = served(x.cuda(), ids.cuda(), weights.cuda())
    want = torch.zeros(tokens, hidden, dtype=torch.float64)
    tol = torch.zeros_like(want)
    h = half_step(dtype)
    for e in range(n):
        t, k = torch.where(ids == e)
        (a, da), (b, db) = (product(x[t], *values(getattr(experts[e], p))) for p in ("gate_proj", "up_proj"))
        s = a * torch.sigmoid(a)
        v = s * b
        dv = 1.1 * da * (b.abs() + db) + s.abs() * db + 2.0 ** -20 * v.abs()
        dv = dv + h * (v.abs() + dv) + 2.0 ** -25                # rounded (fp16's smallest step among them)
        vd, sd = values(experts[e].down_proj)
        o = v @ vd.T
        do = dv @ vd.abs().T + 2.0 ** -18 * ((v.abs() + dv) @ (vd.abs() + 15 * sd).T)
        do = do + h * (o.abs() + do) + 2.0 ** -25
        w = weights[t, k, None].double()
        want.index_add_(0, t, w * o)
        tol.index_add_(0, t, w * do + 2 * top * 2.0 ** -24 * (w * (o.abs() + do)))
    close(y, want, tol + 2.0 ** -25)


def test_experts_in_a_replayed_graph():
    experts = W4A16Experts.from_experts(quantized_experts("W4A16", 6, 256, 128))
    g = torch.Generator().manual_seed(8)
    x = torch.randn(5, 256, generator=g).to(BF16).cuda()
    ids = torch.stack([torch.randperm(6, generator=g)[:2] for _ in range(5)]).cuda()
    w = torch.rand(5, 2, generator=g).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        experts(x, ids, w)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = experts(x, ids, w)
    for i in range(3):
        ids.add_(1).remainder_(6)
        x.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, experts(x, ids, w)), i


def test_layers_refuse_gradients_and_wrong_inputs():
    experts = quantized_experts("W4A16", 3, 256, 128)
    served = W4A16Experts.from_experts(experts)
    lin = W4A16Linear.from_module(experts[0].gate_proj)
    x = torch.randn(4, 256, device="cuda", dtype=BF16)
    ids, w = torch.zeros(4, 1, dtype=torch.int64, device="cuda"), torch.ones(4, 1, device="cuda")
    with pytest.raises(NotImplementedError, match="derivatives"):
        lin(x.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="derivatives"):
        served(x, ids, w.clone().requires_grad_())
    with torch.no_grad():
        lin(x.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="derivatives"):
        lin(torch.autograd.forward_ad.make_dual(x, x))
    with pytest.raises(ValueError, match="256"):
        lin(x[:, :128])
    with pytest.raises(TypeError, match="bf16 or fp16"):
        lin(x.float())
    with pytest.raises(ValueError, match="take x of|plan|rows|weights"):
        served(x, ids, w[:3])
    with pytest.raises(ValueError, match="quantized"):
        W4A16Linear.from_module(torch.nn.Linear(8, 8))
    m = One(64, 256, False, BF16, 1)
    QuantizationModifier(scheme="W8A16").apply(m)
    with pytest.raises(NotImplementedError, match="int4 or MXFP4"):
        W4A16Linear.from_module(m.proj)


# ---------------------------------------------------------------- refusals of the functions
def test_functions_refuse_what_they_cannot_take():
    from llmcompressor_amd import ops as o
    x = torch.randn(4, 256, device="cuda", dtype=BF16)
    w, s = torch.zeros(16, 32, dtype=torch.int32, device="cuda"), torch.ones(16, 2, dtype=BF16, device="cuda")
    z = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="group_size"):
        o.w4a16_matmul(x, w, s, group_size=48)
    with pytest.raises(ValueError, match="weight_scale must be"):
        o.w4a16_matmul(x, w, s, group_size=64)
    with pytest.raises(ValueError, match="weight_packed must be"):
        o.w4a16_matmul(x[:, :200], w, s)
    with pytest.raises(TypeError, match="weight_packed must be"):
        o.w4a16_matmul(x, w.long(), s)
    with pytest.raises(ValueError, match="weight_zero_point must be"):
        o.w4a16_matmul(x, w, s, z[:1])
    with pytest.raises(ValueError, match="no zero points"):
        o.w4a16_matmul(x, torch.zeros(16, 128, dtype=torch.uint8, device="cuda"),
                       torch.zeros(16, 8, dtype=torch.uint8, device="cuda"), z)
    with pytest.raises(ValueError, match="groups of 32"):
        o.w4a16_matmul(x[:, :40], torch.zeros(16, 20, dtype=torch.uint8, device="cuda"),
                       torch.zeros(16, 1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="gate and up"):
        o.w4a16_matmul(x, w[:15], s[:15], gated=True)
    with pytest.raises(ValueError, match="bias must be"):
        o.w4a16_matmul(x, w, s, bias=torch.zeros(15, device="cuda"))
    with pytest.raises(TypeError, match="out_dtype"):
        o.w4a16_matmul(x, w, s, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="GPU only"):
        o.w4a16_matmul(x, w.cpu(), s)
    with pytest.raises(TypeError, match="offsets must be"):
        o.w4a16_experts_matmul(x, None, torch.zeros(2, dtype=torch.int32, device="cuda"), w[None], s[None])
    with pytest.raises(TypeError, match="rows must be"):
        o.w4a16_experts_matmul(x, torch.zeros(4, dtype=torch.int64, device="cuda"),
                               torch.zeros(2, dtype=torch.int64, device="cuda"), w[None], s[None])
    ids = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    rows, slots, offsets = o.moe_plan(ids, 3)
    with pytest.raises(TypeError, match="int32 or int64"):
        o.moe_plan(ids.float(), 3)
    with pytest.raises(ValueError, match="positive"):
        o.moe_plan(ids, 0)
    with pytest.raises(RuntimeError, match="at most 2040"):
        o.moe_plan(ids, 2041)
    with pytest.raises(ValueError, match="rows"):
        o.moe_sort(x[:3], slots, offsets)
    with pytest.raises(ValueError, match="same shape"):
        o.moe_combine(torch.zeros(8, 4, device="cuda"), torch.ones(4, 1, device="cuda"), slots, offsets)
    with pytest.raises(ValueError, match="in its type"):
        o.moe_combine_backward(torch.zeros(4, 4, device="cuda"), torch.zeros(8, 4, device="cuda", dtype=BF16),
                               torch.ones(4, 2, device="cuda"), slots, offsets)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        o.moe_sort(torch.zeros(4, 4, dtype=torch.float64, device="cuda"), slots, offsets)


# ---------------------------------------------------------------- experts on sorted tokens, routing
@pytest.mark.parametrize("tokens,top", [(0, 2), (1, 2), (200, 3)])
def test_linear_experts_on_sorted_tokens(tokens, top):
    """Output and gradients against the loop over experts, both in fp32: each within the sums' roundings of the
    other (chains of up to 384 products twice and top terms: 2^-13 of the magnitudes is far above)."""
    torch.manual_seed(0)
    a = LinearExperts(5, 64, 96).cuda()
    b = LinearExperts(5, 64, 96, sorted_tokens=True).cuda()
    b.load_state_dict(a.state_dict())
    seen = {id(m): [] for m in (a, b)}
    for m in (a, b):
        for e in m:
            e.register_forward_pre_hook(lambda mod, args, m=m: seen[id(m)].append(args[0].detach()))
    x = torch.randn(tokens, 64, device="cuda")
    weights, ids = torch.softmax(torch.randn(tokens, 5, device="cuda"), 1).topk(top)
    d = torch.randn(tokens, 64, device="cuda")
    res = []
    for m in (a, b):
        xi, wi = x.clone().requires_grad_(), weights.clone().requires_grad_()
        y = m(xi, ids, wi)
        res.append([y, *torch.autograd.grad(y, [xi, wi, *m.parameters()], d, allow_unused=True)])
    for p, q in zip(*res):
        if p is None or q is None or p.numel() == 0:
            continue
        assert p.shape == q.shape and (p - q).detach().abs().max() <= 2.0 ** -13 * p.detach().abs().max()
    assert all(torch.equal(p, q) for p, q in zip(seen[id(a)], seen[id(b)]))     # the experts' inputs are the same
    with moe_calibration_context(), torch.no_grad():
        assert torch.equal(a(x, ids, weights), b(x, ids, weights))


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("tokens,top,experts", [(1, 1, 1), (300, 4, 16), (5000, 8, 128), (7, 2, 3000)])
def test_route_tokens_is_what_it_was(tokens, top, experts, dtype):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(0, experts, (tokens, top), generator=g).to(dtype)
    rows, offsets, pos = route_tokens(ids.cuda(), experts)
    want = route_tokens(ids, experts)
    assert rows.dtype == torch.int32 and pos.dtype == torch.int64
    assert torch.equal(rows.cpu(), want[0]) and offsets == want[1] and torch.equal(pos.cpu(), want[2])
    ids[0, 0] = experts + 2                                     # past the last expert: more offsets, as before
    rows, offsets, pos = route_tokens(ids.cuda(), experts)
    want = route_tokens(ids, experts)
    assert torch.equal(rows.cpu(), want[0]) and offsets == want[1] and torch.equal(pos.cpu(), want[2])


def test_example_serves_what_it_quantizes():
    path = Path(__file__).resolve().parents[1] / "examples" / "w4a16_experts.py"
    spec = importlib.util.spec_from_file_location("w4a16_experts", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    errors = mod.serve(experts=4, top=2, hidden=256, intermediate=128, tokens=512)
    assert len(errors) == 2 and all(e == e for e in errors)


def test_plan_types():
    plan = moe.plan_tokens(torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 4)
    assert isinstance(plan, moe.TokenPlan) and [t.dtype for t in plan] == [torch.int32, torch.int32, torch.int64]
