"""Linear layers and gated MLPs in block-scaled fp8, for serving and for
training with 8-bit activation checkpoints.

A weight is e4m3 codes with one fp32 scale per 128 x 128 block, activations are
e4m3 codes with one scale per row and 128 columns: the FP8_BLOCK format
(compressed-tensors' preset of that name: float 8-bit weights of strategy
block [128, 128], dynamic group-128 activations).  Weights come from plain ones, which are quantized here
(``ops.fp8_quantize_blocks``), or from a checkpoint that another tool wrote: this package's
schemes, modifiers and save path do not write the format.

Without gradients a layer's input takes fp32 scales, as the scheme has them; the
gated MLP's inner activation has e8m0 scales in both cases.  With gradients all take
powers of two (e8m0), and the same codes that enter the product are all that is
kept of the activation for the backward pass: one byte per element and one per 128,
where the bf16 tensor takes two.  (A first pass without gradients that is run again
with them, as reentrant checkpointing does, therefore differs from the second by
the input's quantization.)

Backward formulas, for y = x W^T + b with X, W the values that the codes stand
for (quantization itself counts as the identity):

    dX = dY W,  dW = dY^T X,  db = sum of dY's rows

Gradients of activations are bf16 inside, whatever the layer's type: dY of another
type is rounded to it first, the input gradient (and in the MLP the gradients of the inner
activation and of gate and up) is a bf16 result, and dX is then converted to the input's type.
Each rounding is up to 2^-8 relative, beside 2^-4 of the codes it is multiplied
with.  Weight gradients are rounded once, to the master's type.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops

E8M0 = torch.float8_e8m0fnu
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _rows(x: torch.Tensor, width: int, what: str) -> torch.Tensor:
    """x [..., width] as a matrix."""
    if x.dtype not in _TYPES:
        raise TypeError(f"{what} must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] != width:
        raise ValueError(f"{what} must be [..., {width}], got {tuple(x.shape)}")
    return x.reshape(-1, width)


def _no_tangents(*tensors) -> None:
    """Refuses operands of forward-mode differentiation: the kernels would return their results without tangents."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("block-scaled fp8 layers have no forward-mode derivatives")


def _grad_rows(dy: torch.Tensor, width: int) -> torch.Tensor:
    return dy.reshape(-1, width).to(torch.bfloat16)


class _Linear(torch.autograd.Function):
    """x [rows, in] times the fp8 weight; ``weight`` is the tensor that takes
    the weight's gradient, or None.  Kept is what a gradient asked for reads."""

    @staticmethod
    def forward(ctx, x, weight, codes, scales, bias):
        xc, xs = ops.fp8_quantize_groups(x, E8M0)
        need = ctx.needs_input_grad
        ctx.save_for_backward(*((xc, xs) if need[1] else (None, None)), *((codes, scales) if need[0] else (None, None)))
        ctx.types = x.dtype, None if weight is None else weight.dtype, None if bias is None else bias.dtype
        return ops.fp8_block_matmul(xc, xs, codes, scales, bias, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xc, xs, codes, scales = ctx.saved_tensors
        need, (x_type, w_type, b_type) = ctx.needs_input_grad, ctx.types
        d = _grad_rows(dy, dy.shape[-1])
        dx = ops.fp8_block_grad_input(d, codes, scales).to(x_type) if need[0] else None
        dw = ops.fp8_block_grad_weight(d, xc, xs, w_type) if need[1] else None
        db = dy.sum(0, dtype=torch.float32).to(b_type) if need[4] else None
        return dx, dw, None, None, db


class _GatedMLP(torch.autograd.Function):
    """down(silu(gate x) * (up x)); keeps the codes of x, of gate and up's
    outputs and of their product, nothing wider, and of these what a gradient
    asked for reads."""

    @staticmethod
    def forward(ctx, x, gate_up_weight, down_weight, gu_codes, gu_scales, d_codes, d_scales):
        xc, xs = ops.fp8_quantize_groups(x, E8M0)
        gate_up = ops.fp8_block_matmul(xc, xs, gu_codes, gu_scales, None, x.dtype)
        need, none = ctx.needs_input_grad, (None, None)
        inner = need[0] or need[1]
        hc, hs, *kept = ops.fp8_silu_mul(gate_up, save=inner)
        ctx.save_for_backward(*((xc, xs) if need[1] else none), *((hc, hs) if need[2] else none), *(kept or none),
                              *((gu_codes, gu_scales) if need[0] else none),
                              *((d_codes, d_scales) if inner else none))
        ctx.types = x.dtype, *(None if w is None else w.dtype for w in (gate_up_weight, down_weight))
        return ops.fp8_block_matmul(hc, hs, d_codes, d_scales, None, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xc, xs, hc, hs, kept, ks, gu_codes, gu_scales, d_codes, d_scales = ctx.saved_tensors
        need, (x_type, gu_type, d_type) = ctx.needs_input_grad, ctx.types
        d = _grad_rows(dy, dy.shape[-1])
        d_down = ops.fp8_block_grad_weight(d, hc, hs, d_type) if need[2] else None
        dx = d_gate_up = None
        if need[0] or need[1]:
            dgu = ops.fp8_silu_mul_backward(ops.fp8_block_grad_input(d, d_codes, d_scales), kept, ks)
            if need[1]:
                d_gate_up = ops.fp8_block_grad_weight(dgu, xc, xs, gu_type)
            if need[0]:
                dx = ops.fp8_block_grad_input(dgu, gu_codes, gu_scales).to(x_type)
        return dx, d_gate_up, d_down, None, None, None, None


class _Weight(torch.nn.Module):
    """An fp8 weight: frozen codes and scales, or (``trainable``) a master
    parameter that is quantized again for every forward pass."""

    def __init__(self, weight: torch.Tensor, trainable: bool):
        super().__init__()
        if weight.dim() != 2 or weight.dtype not in _TYPES:
            raise ValueError(f"a weight must be a bf16, fp16 or fp32 matrix, got {tuple(weight.shape)} {weight.dtype}")
        self.shape = tuple(weight.shape)
        if trainable:
            self.master = torch.nn.Parameter(weight.detach().clone())
        else:
            self.register_parameter("master", None)
            codes, scales = ops.fp8_quantize_blocks(weight.detach())
            self.register_buffer("weight", codes)
            self.register_buffer("weight_scale", scales)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "_Weight":
        if codes.dim() != 2 or codes.dtype != torch.float8_e4m3fn:
            raise ValueError(f"codes must be a float8_e4m3fn matrix, got {tuple(codes.shape)} {codes.dtype}")
        want = tuple(-(-n // ops.FP8_GROUP) for n in codes.shape)
        if tuple(scales.shape) != want or scales.dtype not in _TYPES:
            raise ValueError(f"codes of {tuple(codes.shape)} take bf16, fp16 or fp32 scales of {want}, got "
                             f"{tuple(scales.shape)} {scales.dtype}")
        self = cls.__new__(cls)
        torch.nn.Module.__init__(self)
        self.shape = tuple(codes.shape)
        self.register_parameter("master", None)
        self.register_buffer("weight", codes.detach().clone(memory_format=torch.contiguous_format))
        self.register_buffer("weight_scale", scales.detach().to(torch.float32, copy=True))
        return self

    def _apply(self, fn, *args, **kwargs):
        # module.to(dtype) would turn codes into numbers of that type: the format
        # keeps its types and moves only between devices
        kept = dict(self._buffers)
        super()._apply(fn, *args, **kwargs)
        for name, t in kept.items():
            if self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def codes(self):
        if self.master is None:
            return self.weight, self.weight_scale
        return ops.fp8_quantize_blocks(self.master.detach())


class Fp8BlockLinear(torch.nn.Module):
    """``torch.nn.Linear`` with its weight in block-scaled fp8.

    ``trainable``: the weight stays as a master parameter (``linear.master``,
    in the type given) that receives gradients; otherwise only its codes and
    scales are kept (``linear.weight``, ``linear.weight_scale``: the tensors of an
    FP8_BLOCK checkpoint)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, trainable: bool = False):
        super().__init__()
        self._build(_Weight(weight, trainable), bias, trainable)

    def _build(self, linear: _Weight, bias: torch.Tensor | None, trainable: bool) -> None:
        self.linear = linear
        self.out_features, self.in_features = linear.shape
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError(f"bias must be [{self.out_features}], got {tuple(bias.shape)}")
        self.bias = None if bias is None else torch.nn.Parameter(bias.detach().clone(), requires_grad=trainable)

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, trainable: bool = False) -> "Fp8BlockLinear":
        return cls(linear.weight, linear.bias, trainable)

    @classmethod
    def from_compressed(cls, weight: torch.Tensor, weight_scale: torch.Tensor,
                        bias: torch.Tensor | None = None) -> "Fp8BlockLinear":
        """From a checkpoint's codes [out, in] and scales (one per 128 x 128
        block; bf16 and fp16 ones are widened, which is exact), frozen."""
        self = cls.__new__(cls)
        torch.nn.Module.__init__(self)
        self._build(_Weight.from_codes(weight, weight_scale), bias, False)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        rows = _rows(x, self.in_features, "input")
        master, bias = self.linear.master, self.bias
        _no_tangents(x, master, bias)
        codes, scales = self.linear.codes()
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, master, bias)):
            y = _Linear.apply(rows, master, codes, scales, bias)
        else:
            y = ops.fp8_block_matmul(*ops.fp8_quantize_groups(rows), codes, scales, bias, x.dtype)
        return y.reshape(*x.shape[:-1], self.out_features)


class Fp8GatedMLP(torch.nn.Module):
    """A gated MLP ``down(silu(gate x) * (up x))`` in block-scaled fp8, gate
    and up stacked into one weight [2 intermediate, hidden].

    The stacked weight is what is cut into 128 x 128 blocks.  Where the intermediate size is a
    multiple of 128 these are the blocks of gate and of up; elsewhere one row of blocks
    holds gate's last rows and up's first under shared scales and up's later blocks
    are shifted, so the codes are not those of the two projections quantized apart, and
    up to 127 rows of a projection much smaller than the other lose precision (two
    ``Fp8BlockLinear`` keep them apart).  There is no construction from a checkpoint's codes.

    The activation goes from the first product to the second in fp8 without a
    pass of its own; with gradients, 8-bit codes are what the backward pass gets
    (hidden + 3 intermediate bytes per token and their scales, where bf16
    tensors of the same would be twice that)."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, trainable: bool = False):
        super().__init__()
        if gate.shape != up.shape or tuple(down.shape) != (gate.shape[1], gate.shape[0]):
            raise ValueError(f"gate {tuple(gate.shape)}, up {tuple(up.shape)} and down {tuple(down.shape)} do not make "
                             "a gated MLP")
        self.intermediate_size, self.hidden_size = gate.shape
        self.gate_up = _Weight(torch.cat([gate.detach(), up.detach()]), trainable)
        self.down = _Weight(down, trainable)

    @classmethod
    def from_expert(cls, expert: torch.nn.Module, trainable: bool = False) -> "Fp8GatedMLP":
        """From a module with ``gate_proj``, ``up_proj`` and ``down_proj``
        linears without biases and SiLU between them (``moe.ExpertMLP``)."""
        projs = expert.gate_proj, expert.up_proj, expert.down_proj
        if any(p.bias is not None for p in projs):
            raise NotImplementedError("gated MLPs with biases are not supported")
        act = getattr(expert, "act", getattr(expert, "act_fn", torch.nn.functional.silu))
        if act is not torch.nn.functional.silu and not isinstance(act, torch.nn.SiLU):
            raise NotImplementedError(f"the activation must be SiLU, got {act}")
        return cls(*(p.weight for p in projs), trainable=trainable)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        rows = _rows(x, self.hidden_size, "input")
        masters = self.gate_up.master, self.down.master
        _no_tangents(x, *masters)
        gu, d = self.gate_up.codes(), self.down.codes()
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, *masters)):
            y = _GatedMLP.apply(rows, *masters, *gu, *d)
        else:
            h = ops.fp8_block_matmul(*ops.fp8_quantize_groups(rows), *gu, None, x.dtype)
            y = ops.fp8_block_matmul(*ops.fp8_silu_mul(h, save=False), *d, None, x.dtype)
        return y.reshape(x.shape)
