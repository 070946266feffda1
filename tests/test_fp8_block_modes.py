"""Block-scaled fp8 layers outside of reverse-mode gradients (CPU only: nothing is launched)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from llmcompressor_amd import Fp8BlockLinear, Fp8GatedMLP
from llmcompressor_amd.fp8_block import _Weight


def layers():
    codes, scales = torch.ones(128, 256).to(torch.float8_e4m3fn), torch.ones(1, 2)
    linear = Fp8BlockLinear.from_compressed(codes, scales, torch.zeros(128))
    mlp = Fp8GatedMLP.__new__(Fp8GatedMLP)      # the constructor quantizes, on a GPU
    torch.nn.Module.__init__(mlp)
    mlp.intermediate_size, mlp.hidden_size = 64, 256
    mlp.gate_up = _Weight.from_codes(codes, scales)
    mlp.down = _Weight.from_codes(codes[:64].reshape(256, 64), torch.ones(2, 1))
    return linear, mlp


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(which, grad):
    """An input with a tangent is refused whether or not it asks for a gradient too; the tangent is never dropped."""
    layer, x = layers()[which], torch.ones(3, 256, requires_grad=grad)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones(3, 256))
        for context in (torch.enable_grad(), torch.no_grad()):
            with context, pytest.raises(NotImplementedError, match="forward-mode"):
                layer(dual)
        with pytest.raises(RuntimeError, match="GPU only"):       # no tangent: as ever
            layer(x.detach())
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(layer, (x.detach(),), (torch.ones(3, 256),))


def test_forward_mode_derivatives_of_a_parameter_are_refused():
    linear, x = layers()[0], torch.ones(3, 256)
    with fwd.dual_level():
        dual = fwd.make_dual(linear.bias, torch.ones(128))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.functional_call(linear, {"bias": dual}, (x,))
