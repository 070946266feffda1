"""The operators of a 4-bit mixture of experts whose speed is measured.

A 4-bit weight here is what the package's checkpoints hold: int4 codes, eight
to an int32 (stored + 8), with a scale per row and group of columns and, where
asymmetric, zero points packed along the rows; or MXFP4, e2m1 codes two to a
byte with a power of two per row and 32 columns.  Kinds of cases:

* ``sort``     tokens into the order of the experts that they are routed to
* ``combine``  the experts' rows back to tokens, weighted and summed
* ``matmul``   Y = X W^T (+ bias), X of 16 bits, W of 4
* ``experts``  the same for rows grouped by expert, a weight per expert

``backward``: the gradients are part of the pass.  ``gated``: the weight holds
gate and up, one after the other, and the product is silu(gate) * up.  With
``own`` false ``run`` computes them with elementary torch operations in 32
bits, with ``own`` true through the package's entry points.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "llm-compressor_amd"))

own = False
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token on its way to its experts
        dict(name="sort_token", kind="sort", tokens=1, top=8, experts=128, cols=2048, dtype="bf16", dropped=0.0,
             backward=False),
        # a padded batch (ids of -1) through a few wide experts, in training
        dict(name="sort_padded", kind="sort", tokens=1333, top=2, experts=8, cols=4096, dtype="fp16", dropped=0.2,
             backward=True),
        # a training step's tokens
        dict(name="sort_step", kind="sort", tokens=8192, top=8, experts=128, cols=2048, dtype="bf16", dropped=0.0,
             backward=True),
        # one decoded token on its way back
        dict(name="combine_token", kind="combine", tokens=1, top=8, experts=128, cols=2048, dtype="bf16", dropped=0.0,
             backward=False),
        # rows of an odd width in fp32, in training
        dict(name="combine_odd", kind="combine", tokens=777, top=4, experts=60, cols=2001, dtype="fp32", dropped=0.1,
             backward=True),
        # a training step's tokens
        dict(name="combine_step", kind="combine", tokens=8192, top=8, experts=128, cols=2048, dtype="bf16",
             dropped=0.0, backward=True),
        # decoding one token through an up projection: the weight's bytes
        dict(name="matmul_token", kind="matmul", rows=1, out=14336, cols=4096, weight="int4", group=128, dtype="bf16",
             bias=False, gated=False),
        # a decoding batch through a down projection in MXFP4
        dict(name="matmul_batch", kind="matmul", rows=23, out=4096, cols=14336, weight="mxfp4", group=32,
             dtype="fp16", bias=True, gated=False),
        # a prompt through gate and up: the largest call
        dict(name="matmul_prompt", kind="matmul", rows=8192, out=28672, cols=4096, weight="int4", group=128,
             dtype="bf16", bias=False, gated=True),
        # one token through gate and up of its eight experts
        dict(name="experts_token", kind="experts", tokens=1, top=8, experts=128, out=1536, cols=2048, weight="int4",
             group=128, dtype="bf16", gated=True),
        # a decoding batch, asymmetric with small groups: nearly every expert is read for a few rows
        dict(name="experts_batch", kind="experts", tokens=61, top=8, experts=128, out=1536, cols=2048,
             weight="int4z", group=32, dtype="bf16", gated=True),
        # a prompt
        dict(name="experts_prompt", kind="experts", tokens=4096, top=8, experts=128, out=1536, cols=2048,
             weight="int4", group=128, dtype="bf16", gated=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly whole groups of 128, else whole groups of 32, now and then any number."""
    n, how = _log(rng, lo, hi), rng.random()
    if how < 0.6:
        return max(128, n // 128 * 128)
    return max(32, n // 32 * 32) if how < 0.85 else n


def draw(rng):
    kind = rng.choice(["sort", "combine", "matmul", "matmul", "experts", "experts"])
    if kind in ("sort", "combine"):
        experts = _log(rng, 2, 256)
        c = dict(kind=kind, experts=experts, top=rng.randint(1, min(8, experts)), cols=_width(rng, 64, 8192),
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), dropped=rng.choice([0.0, 0.0, 0.15]),
                 backward=rng.random() < 0.6)
        most = 8192 * 8 * 2048 * 2 // (c["top"] * c["cols"] * SIZES[c["dtype"]])
        return dict(c, tokens=_log(rng, 1, min(16384, most)))
    weight = rng.choice(["int4", "int4", "int4z", "mxfp4"])
    cols = _width(rng, 64, 14336)
    if weight == "mxfp4":
        cols = max(32, cols // 32 * 32)
    group = 32 if weight == "mxfp4" else rng.choice([128, 128, 64, 32, cols])
    c = dict(kind=kind, cols=cols, weight=weight, group=group, dtype=rng.choice(["bf16", "bf16", "fp16"]),
             gated=rng.random() < 0.4)
    if kind == "matmul":
        out = _width(rng, 64, 28672) * (2 if c["gated"] else 1)
        out = min(out, 28672)
        most = 8192 * 28672 * 4096 // (out * cols)
        return dict(c, out=out, rows=_log(rng, 1, min(8192, most)), bias=rng.random() < 0.3)
    c["cols"] = cols = min(cols, 4096)
    c["group"] = min(group, cols)
    experts = _log(rng, 2, 128)
    out = min(_width(rng, 64, 2048) * (2 if c["gated"] else 1), 128 * 1536 * 2048 // (experts * cols) // 2 * 2)
    top = rng.randint(1, min(8, experts))
    most = 4096 * 8 * 1536 * 2048 // (top * out * cols)
    return dict(c, experts=experts, out=out, top=top, tokens=_log(rng, 1, min(4096, most)))


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _activations(g, rows, cols, dtype):
    """Heavy-tailed activations: Student t with four degrees of freedom times a lognormal scale per channel."""
    chi = _randn(g, rows, cols).square_()
    for _ in range(3):
        chi += _randn(g, rows, cols).square_()
    x = _randn(g, rows, cols).div_(chi.mul_(0.25).sqrt_()).mul_(_randn(g, cols).exp_())
    return x.clamp_(-3e4, 3e4).to(dtype)


def _routing(g, tokens, top, experts, dropped):
    """A skewed router's choice: ids of the largest logits and their softmax; ids of padded tokens are -1."""
    logits = _randn(g, tokens, experts) + _randn(g, experts)
    best, ids = logits.topk(top, dim=1)
    if dropped:
        ids[torch.rand(tokens, generator=g, device=DEV) < dropped] = -1
    return ids, torch.softmax(best, 1)


def _int4(w, group, zeros):
    """w [n, cols] as int4: (packed words [n, ceil(cols / 8)], bf16 scales [n, groups], stored zero points [n, groups]
    or None), codes and zero points 0 .. 15."""
    n, cols = w.shape
    v = torch.nn.functional.pad(w, (0, -cols % group)).view(n, -1, group)
    if zeros:
        lo, hi = v.amin(2).clamp_max(0), v.amax(2).clamp_min(0)
        s = ((hi - lo) / 15).clamp_min(1e-6).bfloat16()
        z = torch.round(-lo / s.float()).clamp(0, 15)
    else:
        s = (v.abs().amax(2) / 7.5).clamp_min(1e-6).bfloat16()
        z = torch.full_like(s, 8, dtype=torch.float32)
    codes = (torch.round(v / s.float()[..., None]) + z[..., None]).clamp_(0, 15).int().view(n, -1)[:, :cols]
    codes = torch.nn.functional.pad(codes, (0, -cols % 8)).view(n, -1, 8)
    words = torch.zeros(codes.shape[:2], dtype=torch.int32, device=DEV)
    for i in range(8):
        words |= codes[..., i] << (4 * i)
    return words, s, z.int() if zeros else None


def _mxfp4(w):
    """w [n, cols] as MXFP4: (bytes [n, cols / 2], exponent bytes [n, cols / 32])."""
    n, cols = w.shape
    v = w.view(n, -1, 32)
    e = torch.floor(torch.log2(v.abs().amax(2).clamp_min(1e-30))) - 2
    a = (v.abs() / torch.exp2(e)[..., None]).view(n, cols)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    codes = torch.bucketize(a, edges).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _pack_rows(z):
    """Zero points [n, groups] eight rows to an int32: [ceil(n / 8), groups]."""
    z = torch.nn.functional.pad(z, (0, 0, 0, -z.shape[0] % 8)).view(-1, 8, z.shape[1])
    words = torch.zeros((z.shape[0], z.shape[2]), dtype=torch.int32, device=DEV)
    for i in range(8):
        words |= z[:, i] << (4 * i)
    return words


def _weight(g, c):
    """(packed, scales, packed zero points or None) of N(0, 0.02) with one entry in a thousand ten times larger."""
    def one():
        w = _randn(g, c["out"], c["cols"]).mul_(0.02)
        w[torch.rand(w.shape, generator=g, device=DEV) < 1e-3] *= 10
        if c["weight"] == "mxfp4":
            return (*_mxfp4(w), None)
        words, s, z = _int4(w, c["group"], c["weight"] == "int4z")
        return words, s, None if z is None else _pack_rows(z)

    if c["kind"] == "matmul":
        return one()
    parts = [one() for _ in range(c["experts"])]
    return tuple(None if p[0] is None else torch.stack(p) for p in zip(*parts))


def prepare(case, seed):
    g, c, kind = _gen(seed), case, case["kind"]
    dtype = DTYPES[c["dtype"]]
    if kind == "matmul":
        return dict(c, x=_activations(g, c["rows"], c["cols"], dtype), w=_weight(g, c),
                    b=_randn(g, c["out"]).to(dtype) if c["bias"] else None)
    ids, weights = _routing(g, c["tokens"], c["top"], c["experts"], c.get("dropped", 0.0))
    if kind == "experts":
        return dict(c, x=_activations(g, c["tokens"], c["cols"], dtype), w=_weight(g, c),
                    plan=_plain_plan(ids, c["experts"]))
    pairs = c["tokens"] * c["top"]
    if kind == "sort":
        return dict(c, x=_activations(g, c["tokens"], c["cols"], dtype), ids=ids,
                    d=_randn(g, pairs, c["cols"]).mul_(1e-3).to(dtype) if c["backward"] else None)
    return dict(c, x=_activations(g, pairs, c["cols"], dtype), weights=weights, plan=_plain_plan(ids, c["experts"]),
                d=_randn(g, c["tokens"], c["cols"]).mul_(1e-3).to(dtype) if c["backward"] else None)


# ---------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from llmcompressor_amd import moe, ops

    kind = s["kind"]
    if kind == "matmul":
        return ops.w4a16_matmul(s["x"], *s["w"], group_size=s["group"], bias=s["b"], gated=s["gated"])
    if kind == "experts":
        rows, _, offsets = s["plan"]
        return ops.w4a16_experts_matmul(s["x"], rows, offsets, *s["w"], group_size=s["group"], gated=s["gated"])
    x = s["x"].detach().requires_grad_(s["backward"])
    if kind == "sort":
        y, plan = moe.sort_tokens(x, s["ids"], s["experts"])
        return (y, *plan, *torch.autograd.grad(y, x, s["d"])) if s["backward"] else (y, *plan)
    weights = s["weights"].detach().requires_grad_(s["backward"])
    y = moe.combine_tokens(x, weights, moe.TokenPlan(*s["plan"]))
    return (y, *torch.autograd.grad(y, (x, weights), s["d"])) if s["backward"] else y


# ---------------------------------------------------------------- plain forms
def _plain_plan(ids, experts):
    """(rows, slots, offsets): pairs ordered by expert, then position, then token; ids of no expert come last."""
    tokens, top = ids.shape
    e = torch.where((ids >= 0) & (ids < experts), ids, experts).t().reshape(-1)
    order = torch.sort(e, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=DEV)
    counts = (e[:, None] == torch.arange(experts, device=DEV)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return (order % tokens).int(), slots.view(top, tokens).t().contiguous().int(), offsets


def _plain_values(c, w, scales, zeros):
    """The fp32 values of 4-bit weights [n, cols]."""
    cols = c["cols"]
    if c["weight"] == "mxfp4":
        codes = torch.stack([w & 15, w >> 4], -1).view(w.shape[0], -1).long()
        v = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=DEV)[codes]
        s = torch.exp2(scales.float() - 127)
    else:
        v = torch.stack([(w >> 4 * i) & 15 for i in range(8)], -1).view(w.shape[0], -1)[:, :cols]
        s = scales.float()
        z = 8
        if zeros is not None:
            z = torch.stack([(zeros >> 4 * i) & 15 for i in range(8)], 1).view(-1, zeros.shape[1])[:w.shape[0]]
            z = z.repeat_interleave(c["group"], 1)[:, :cols]
        v = (v - z).float()
    return v * s.repeat_interleave(c["group"], 1)[:, :cols]


def _plain_gate(y, gated):
    if not gated:
        return y
    gate, up = y[:, :y.shape[1] // 2], y[:, y.shape[1] // 2:]
    return gate / (1.0 + torch.exp(-gate)) * up


def _run_plain(s):
    kind, dtype = s["kind"], DTYPES[s["dtype"]]
    if kind == "matmul":
        y = s["x"].float() @ _plain_values(s, *s["w"]).t()
        return _plain_gate(y if s["b"] is None else y + s["b"].float(), s["gated"]).to(dtype)
    if kind == "experts":
        rows, _, offsets = s["plan"]
        ends = offsets.tolist()
        y = torch.zeros(rows.numel(), s["out"] // 2 if s["gated"] else s["out"], device=DEV)
        for e in range(s["experts"]):
            a, b = ends[e], ends[e + 1]
            if a < b:
                w = _plain_values(s, *(None if t is None else t[e] for t in s["w"]))
                y[a:b] = _plain_gate(s["x"][rows[a:b].long()].float() @ w.t(), s["gated"])
        return y.to(dtype)
    tokens, top = s["tokens"], s["top"]
    if kind == "sort":
        rows, slots, offsets = _plain_plan(s["ids"], s["experts"])
        kept = torch.arange(rows.numel(), device=DEV) < offsets[-1]
        y = torch.where(kept[:, None], s["x"][rows.long()], 0)
        if not s["backward"]:
            return y, rows, slots, offsets
        d = torch.where(kept[:, None], s["d"].float(), 0)[slots.long().view(-1)].view(tokens, top, -1)
        return y, rows, slots, offsets, d.sum(1).to(dtype)
    rows, slots, offsets = s["plan"]
    kept = slots < offsets[-1]
    x = s["x"].float()[slots.long().view(-1)].view(tokens, top, -1)
    x = torch.where(kept[..., None], x, 0)
    y = (s["weights"][..., None] * x).sum(1).to(dtype)
    if not s["backward"]:
        return y
    d = s["d"].float()
    dx = torch.zeros(rows.numel(), s["cols"], device=DEV)
    dx[slots.long().view(-1)] = torch.where(kept[..., None], s["weights"][..., None] * d[:, None], 0).view(
        rows.numel(), -1)
    return y, dx.to(dtype), (x * d[:, None]).sum(2)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, kind, size = case, case["kind"], SIZES[case["dtype"]]
    if kind in ("sort", "combine"):
        pairs = c["tokens"] * c["top"]
        one, all_ = c["tokens"] * c["cols"] * size, pairs * c["cols"] * size
        if kind == "sort":
            return dict(bytes=8 * pairs + (2 if c["backward"] else 1) * (one + all_) + 8 * pairs + 8 * c["experts"],
                        flops=pairs * c["cols"])
        # the backward pass reads d and the experts' rows and writes their gradient and the weights'
        both = 2 * (one + all_) + all_ + 8 * pairs if c["backward"] else one + all_
        return dict(bytes=both + 8 * pairs, flops=(6 if c["backward"] else 2) * pairs * c["cols"])
    groups = -(-c["cols"] // c["group"])
    weight = c["out"] * (-(-c["cols"] // 8) * 4 + groups * {"int4": 2, "int4z": 2.5, "mxfp4": 1}[c["weight"]])
    out = c["out"] // 2 if c["gated"] else c["out"]
    if kind == "matmul":
        return dict(bytes=weight + (c["rows"] * (c["cols"] + out) + c["out"] * c["bias"]) * size,
                    flops=2 * c["rows"] * c["out"] * c["cols"])
    pairs = c["tokens"] * c["top"]
    # every pair's expert is read once: in the mean over even routing, this many of them
    read = c["experts"] * (1 - (1 - c["top"] / c["experts"]) ** c["tokens"])
    return dict(bytes=weight * read + (c["tokens"] * c["cols"] + pairs * out) * size + 4 * pairs,
                flops=2 * pairs * c["out"] * c["cols"])


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_weight(c, w, scales, zeros):
    n, cols, group = w.shape[0], c["cols"], c["group"]
    k = torch.arange(cols, device=DEV)
    if c["weight"] == "mxfp4":
        codes = (w[:, k // 2] >> (4 * (k % 2)).to(torch.uint8)) & 15
        size = codes & 7                     # two bits of exponent, one of fraction
        e, f = (size >> 1).double(), (size & 1).double()
        v = torch.where(size < 2, f / 2, (1 + f / 2) * 2.0 ** (e - 1))
        return torch.where(codes > 7, -v, v) * 2.0 ** (scales[:, k // group].double() - 127)
    q = ((w[:, k // 8] >> (4 * (k % 8)).int()) & 15).double()
    z = 8.0
    if zeros is not None:
        r = torch.arange(n, device=DEV)
        z = ((zeros[r // 8][:, k // group] >> (4 * (r % 8)).int()[:, None]) & 15).double()
    return (q - z) * scales[:, k // group].double()


def _exact_product(c, x, w, b):
    y = torch.matmul(x.double(), _exact_weight(c, *w).T)
    y = y if b is None else y + b.double()
    if not c["gated"]:
        return y
    gate, up = y.chunk(2, 1)
    return gate * torch.sigmoid(gate) * up


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "matmul":
        return _exact_product(s, s["x"], s["w"], s["b"])
    if kind == "experts":
        rows, _, offsets = s["plan"]
        parts = []
        for e, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
            if a < b:
                parts.append(_exact_product(s, s["x"][rows[a:b].long()], [None if t is None else t[e] for t in s["w"]],
                                            None))
        return torch.cat(parts)
    tokens, top = s["tokens"], s["top"]
    if kind == "sort":
        # every expert's pairs in turn, position by position
        ids, order, offsets = s["ids"].t().contiguous(), [], [0]
        for e in range(s["experts"]):
            order.append((ids == e).reshape(-1).nonzero().view(-1))
            offsets.append(offsets[-1] + order[-1].numel())
        order.append(((ids < 0) | (ids >= s["experts"])).reshape(-1).nonzero().view(-1))
        order = torch.cat(order)
        n, token = offsets[-1], order % tokens
        slots = torch.zeros(tokens, top, dtype=torch.int64, device=DEV)
        slots[token, order // tokens] = torch.arange(order.numel(), device=DEV)
        y = s["x"].double()[token]
        y[n:] = 0
        plan = token, slots, torch.tensor(offsets, device=DEV)
        if not s["backward"]:
            return y, *plan
        dx = torch.zeros(tokens, s["cols"], dtype=torch.float64, device=DEV)
        return y, *plan, dx.index_add_(0, token[:n], s["d"][:n].double())
    rows, slots, offsets = s["plan"]
    n, x, token = int(offsets[-1]), s["x"].double(), rows.long()
    at = torch.zeros(rows.numel(), dtype=torch.float64, device=DEV)     # each row's weight
    at[slots.long().reshape(-1)] = s["weights"].double().reshape(-1)
    at[n:] = 0
    y = torch.zeros(tokens, s["cols"], dtype=torch.float64, device=DEV).index_add_(0, token[:n], at[:n, None] * x[:n])
    if not s["backward"]:
        return y
    d = s["d"].double()[token]
    dw = (d * x).sum(1)
    dw[n:] = 0
    return y, at[:, None] * d, dw[slots.long().reshape(-1)].view(tokens, top)
