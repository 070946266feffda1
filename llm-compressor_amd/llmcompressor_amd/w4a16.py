"""Linear layers and mixtures of experts on 4-bit weights, for serving what the
W4A16 and MXFP4 schemes compress without unpacking it.

A weight is what ``save.compress_module`` writes and a checkpoint holds:
``pack-quantized`` (int4, a scale per row and group of columns, zero points where
asymmetric) or ``mxfp4-pack-quantized``.  Activations stay bf16 or fp16.  MXFP4's
preset quantizes activations too; here they are not, so a layer differs from that
scheme by the rounding it leaves out.  The layers are for inference: inputs that
want gradients or carry tangents are refused.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import moe, ops, save
from .quant_args import QuantizationStrategy, resolve_args


def _no_derivatives(*tensors) -> None:
    for t in tensors:
        if (torch.is_grad_enabled() and t.requires_grad) or forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("4-bit layers have no derivatives: call them under torch.no_grad() or detach "
                                      "their inputs")


def _unpack(words: torch.Tensor, cols: int) -> torch.Tensor:
    """int32 words [rows, n] as nibbles [rows, cols], int8."""
    shift = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    return ((words.unsqueeze(-1) >> shift) & 15).flatten(-2)[..., :cols].to(torch.int8)


class _Weight(torch.nn.Module):
    """The tensors of one 4-bit weight [out, in], or of a stack [experts, out,
    in]; ``columns``: the order in which a row of x is multiplied with them
    (activation ordering's groups lie side by side then), or None."""

    def __init__(self, weight_packed, weight_scale, weight_zero_point, group_size, in_features, columns=None):
        super().__init__()
        self.in_features, self.group_size = in_features, group_size
        for name, t in (("weight_packed", weight_packed), ("weight_scale", weight_scale),
                        ("weight_zero_point", weight_zero_point), ("columns", columns)):
            self.register_buffer(name, None if t is None else t.detach())

    def _apply(self, fn, *args, **kwargs):
        # module.to(dtype) keeps the format's types and moves only between devices
        kept = dict(self._buffers)
        super()._apply(fn, *args, **kwargs)
        for name, t in kept.items():
            if t is not None and self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def parts(self):
        return self.weight_packed, self.weight_scale, self.weight_zero_point, self.group_size

    def rows(self, x: torch.Tensor) -> torch.Tensor:
        return x if self.columns is None else x.index_select(1, self.columns)


def _tensors(module: torch.nn.Module):
    """(packed, scales, zero points, group size, in features, g_idx) of a quantized module."""
    scheme = getattr(module, "quantization_scheme", None)
    if scheme is None or scheme.weights is None:
        raise ValueError(f"{type(module).__name__} has no quantized weight (quantization_scheme)")
    w, fmt = resolve_args(scheme.weights), save.infer_quantization_format(scheme)
    if fmt not in ("pack-quantized", "mxfp4-pack-quantized") or w.num_bits != 4:
        raise NotImplementedError(f"4-bit layers take int4 or MXFP4 weights, got {w.type.value}{w.num_bits} ({fmt})")
    if w.strategy not in (QuantizationStrategy.GROUP, QuantizationStrategy.CHANNEL) and fmt == "pack-quantized":
        raise NotImplementedError(f"4-bit layers take weights with group or channel scales, got {w.strategy.value}")
    t = save.compress_module(module, fmt)
    group = w.group_size if w.strategy == QuantizationStrategy.GROUP else None
    return (t["weight_packed"], t["weight_scale"], t.get("weight_zero_point"), group, module.weight.shape[1],
            t.get("weight_g_idx"))


def _by_group(packed, group, in_features, g_idx):
    """Codes with the columns of each group side by side, and that order of the
    columns; unchanged where they lie so."""
    if g_idx is None or group is None:
        return packed, None
    g_idx = g_idx.to(device=packed.device, dtype=torch.int64)
    order = torch.argsort(g_idx, stable=True)
    want = torch.arange(in_features, device=packed.device) // group
    if not torch.equal(g_idx[order], want):
        raise NotImplementedError("weight_g_idx must give every group group_size columns")
    if torch.equal(order, torch.arange(in_features, device=packed.device)):
        return packed, None
    codes = _unpack(packed, in_features)[:, order] - 8
    return ops.pack_int32(codes.contiguous(), 4), order


class W4A16Linear(torch.nn.Module):
    """``torch.nn.Linear`` on a 4-bit weight (``ops.w4a16_matmul``)."""

    def __init__(self, weight_packed: torch.Tensor, weight_scale: torch.Tensor,
                 weight_zero_point: torch.Tensor | None = None, group_size: int | None = 128,
                 bias: torch.Tensor | None = None, in_features: int | None = None,
                 weight_g_idx: torch.Tensor | None = None):
        """From a checkpoint's tensors (``weight_packed`` int32: int4, uint8:
        MXFP4); ``in_features`` where it is not a multiple of 8
        (``weight_shape[1]``)."""
        super().__init__()
        mx = weight_packed.dtype == torch.uint8
        cols = weight_packed.shape[1] * (2 if mx else 8)
        if in_features is not None and not (in_features == cols or not mx and cols - 8 < in_features < cols):
            raise ValueError(f"weight_packed {tuple(weight_packed.shape)} does not hold {in_features} columns")
        self.in_features, self.out_features = in_features or cols, weight_packed.shape[0]
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError(f"bias must be [{self.out_features}], got {tuple(bias.shape)}")
        packed, columns = _by_group(weight_packed, group_size, self.in_features, weight_g_idx)
        self.linear = _Weight(packed, weight_scale, weight_zero_point, 32 if mx else group_size, self.in_features,
                              columns)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_module(cls, module: torch.nn.Module) -> "W4A16Linear":
        """From a ``Linear`` that this package's modifiers quantized to int4
        (groups or channels, activation ordering included) or MXFP4."""
        packed, scale, zero, group, cols, g_idx = _tensors(module)
        return cls(packed, scale, zero, group, getattr(module, "bias", None), cols, g_idx)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise ValueError(f"input must be [..., {self.in_features}], got {tuple(x.shape)}")
        _no_derivatives(x)
        packed, scale, zero, group = self.linear.parts()
        y = ops.w4a16_matmul(self.linear.rows(x.reshape(-1, self.in_features)), packed, scale, zero, group, self.bias)
        return y.reshape(*x.shape[:-1], self.out_features)


class W4A16Experts(torch.nn.Module):
    """The experts of an MoE layer on stacked 4-bit weights: down(silu(gate x)
    * (up x)) of every token's experts, weighted and summed.  Three launches behind
    the plan's (one more before a product of many rows), whatever the number of
    experts, and none waits for the host."""

    def __init__(self, gate_up, down, num_experts: int, intermediate_size: int):
        """``gate_up`` [experts, 2 intermediate, hidden] (gate's rows first) and
        ``down`` [experts, hidden, intermediate], each (weight_packed,
        weight_scale, weight_zero_point or None, group_size)."""
        super().__init__()
        self.num_experts, self.intermediate_size = num_experts, intermediate_size
        if gate_up[0].dim() != 3 or tuple(gate_up[0].shape[:2]) != (num_experts, 2 * intermediate_size):
            raise ValueError(f"gate_up must be [{num_experts}, {2 * intermediate_size}, ...], got "
                             f"{tuple(gate_up[0].shape)}")
        if down[0].dim() != 3 or down[0].shape[0] != num_experts:
            raise ValueError(f"down must be [{num_experts}, hidden, ...], got {tuple(down[0].shape)}")
        self.hidden_size = down[0].shape[1]
        self.gate_up = _Weight(*gate_up, self.hidden_size)
        self.down = _Weight(*down, intermediate_size)

    @classmethod
    def from_experts(cls, experts: torch.nn.ModuleList) -> "W4A16Experts":
        """From a list of experts with ``gate_proj``, ``up_proj`` and
        ``down_proj`` (``moe.LinearExperts``) that this package's modifiers
        quantized, one scheme for all; SiLU, no biases, no activation ordering by
        groups."""
        parts = {}
        for expert in experts:
            act = getattr(expert, "act", getattr(expert, "act_fn", torch.nn.functional.silu))
            if act is not torch.nn.functional.silu and not isinstance(act, torch.nn.SiLU):
                raise NotImplementedError(f"the activation must be SiLU, got {act}")
            for name in ("gate_proj", "up_proj", "down_proj"):
                module = getattr(expert, name)
                if module.bias is not None:
                    raise NotImplementedError("experts with biases are not supported")
                *t, cols, g_idx = _tensors(module)
                if g_idx is not None and _by_group(t[0], t[3], cols, g_idx)[1] is not None:
                    raise NotImplementedError("experts with activation ordering by groups are not supported")
                parts.setdefault(name, []).append(t)
        inter = experts[0].gate_proj.weight.shape[0]
        if parts["gate_proj"][0][2] is not None and inter % 8:
            raise NotImplementedError("zero points of gate and up are packed eight rows to a word: the intermediate "
                                      "size must be a multiple of 8")

        def stacked(*names):
            kinds = {(t[0].dtype, t[1].dtype, t[2] is None, t[3]) for n in names for t in parts[n]}
            if len(kinds) != 1:
                raise ValueError(f"{' and '.join(names)} have several formats: {sorted(map(str, kinds))}")
            per = [[torch.cat([parts[n][e][i] for n in names]) if parts[names[0]][e][i] is not None else None
                    for e in range(len(experts))] for i in range(3)]
            return [None if p[0] is None else torch.stack(p) for p in per] + [parts[names[0]][0][3]]

        return cls(stacked("gate_proj", "up_proj"), stacked("down_proj"), len(experts), inter)

    def forward(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                top_k_weights: torch.Tensor) -> torch.Tensor:
        """hidden_states [tokens, hidden] (bf16 or fp16), top_k_index and
        top_k_weights [tokens, top]; ids outside [0, num_experts) take no
        part."""
        if hidden_states.dim() != 2 or top_k_index.dim() != 2 or top_k_index.shape[0] != hidden_states.shape[0]:
            raise ValueError(f"hidden_states [tokens, hidden] take ids of the same tokens, got "
                             f"{tuple(hidden_states.shape)} and {tuple(top_k_index.shape)}")
        _no_derivatives(hidden_states, top_k_weights)
        plan = moe.plan_tokens(top_k_index, self.num_experts)
        h = ops.w4a16_experts_matmul(hidden_states, plan.rows, plan.offsets, *self.gate_up.parts(), gated=True)
        out = ops.w4a16_experts_matmul(h, None, plan.offsets, *self.down.parts())
        return ops.moe_combine(out, top_k_weights, plan.slots, plan.offsets)
