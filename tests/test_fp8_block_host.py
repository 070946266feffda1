"""Host-side checks of the block-scaled fp8 entry points (CPU only: no kernel
launches)."""
import ctypes as C

import pytest
import torch

from llmcompressor_amd import Fp8GatedMLP, _lib, ops
from llmcompressor_amd.fp8_block import _rows

P = C.c_void_p(256)


@pytest.mark.parametrize("call,needle", [
    (lambda l: l.mi355q_fp8_quantize_groups(P, 0, 4, 128, 64, P, 128, P, 0, 1, None), "bad shape"),
    (lambda l: l.mi355q_fp8_quantize_groups(P, 0, 4, 256, 256, P, 256, P, 0, 1, None), "bad shape"),
    (lambda l: l.mi355q_fp8_quantize_groups(None, 0, 4, 128, 128, P, 128, P, 0, 1, None), "null pointer"),
    (lambda l: l.mi355q_fp8_quantize_groups(P, 9, 4, 128, 128, P, 128, P, 0, 1, None), "dtype"),
    (lambda l: l.mi355q_fp8_quantize_groups(P, 0, 4, 128, 128, P, 128, P, 7, 1, None), "scale type"),
    (lambda l: l.mi355q_fp8_quantize_blocks(P, 0, 4, 0, 128, P, 128, P, 1, None), "bad shape"),
    (lambda l: l.mi355q_fp8_quantize_blocks(P, 0, 4, 128, 128, P, 128, None, 1, None), "null pointer"),
    (lambda l: l.mi355q_fp8_block_matmul(P, 128, P, 0, 1, P, 128, P, 1, None, 0, P, 0, 8, 4, 16, 128, None, 0, None),
     "bad shape"),
    (lambda l: l.mi355q_fp8_block_matmul(P, 128, P, 0, 1, P, 128, P, 1, None, 0, P, 5, 16, 4, 16, 128, None, 0, None),
     "output and bias"),
    (lambda l: l.mi355q_fp8_block_matmul(P, 128, P, 3, 1, P, 128, P, 1, None, 0, P, 0, 16, 4, 16, 128, None, 0, None),
     "scale type"),
    (lambda l: l.mi355q_fp8_block_grad_input(P, 16, P, 128, None, 1, P, 128, 4, 16, 128, None, 0, None), "null pointer"),
    (lambda l: l.mi355q_fp8_block_grad_input(P, 8, P, 128, P, 1, P, 128, 4, 16, 128, None, 0, None), "bad shape"),
    (lambda l: l.mi355q_fp8_block_grad_weight(P, 16, P, 128, P, 1, None, 0, 128, 4, 16, 128, None, 0, None),
     "null pointer"),
    (lambda l: l.mi355q_fp8_block_grad_weight(P, 16, P, 128, P, 1, P, 8, 128, 4, 16, 128, None, 0, None), "output is"),
    (lambda l: l.mi355q_fp8_silu_mul(P, 0, 4, 128, 255, P, 128, P, None, 256, None, None), "bad shape"),
    (lambda l: l.mi355q_fp8_silu_mul(P, 0, 4, 128, 256, P, 128, P, P, 256, None, None), "come together"),
    (lambda l: l.mi355q_fp8_silu_mul_backward(P, 0, 4, 128, 128, P, 255, P, 2, P, 256, None), "bad shape"),
])
def test_invalid_arguments_are_rejected_on_the_host(call, needle):
    lib = _lib.load_library()
    assert call(lib) == _lib.INVALID_ARGUMENT
    assert needle in lib.mi355q_last_error().decode()


def test_calls_without_rows_need_no_pointers():
    lib = _lib.load_library()
    assert lib.mi355q_fp8_quantize_groups(None, 0, 0, 128, 128, None, 128, None, 0, 1, None) == _lib.OK
    assert lib.mi355q_fp8_block_matmul(None, 128, None, 0, 1, None, 128, None, 1, None, 0, None, 0, 16, 0, 16, 128, None,
                                       0, None) == _lib.OK
    assert lib.mi355q_fp8_silu_mul(None, 0, 0, 128, 256, None, 128, None, None, 256, None, None) == _lib.OK


def test_workspaces():
    """Splits where tiles leave CUs idle, padded copies for odd widths, nothing else."""
    lib = _lib.load_library()
    assert lib.mi355q_fp8_block_matmul_workspace_size(1, 4096, 4096) == 0
    assert lib.mi355q_fp8_block_matmul_workspace_size(8192, 28672, 4096) == 0
    n = lib.mi355q_fp8_block_matmul_workspace_size(333, 4096, 14336)
    assert n > 0 and n % (333 // 64 * 64 * 4) == 0 or n % (128 * 128 * 4) == 0
    assert lib.mi355q_fp8_block_matmul_workspace_size(4096, 4096, 127) == (4096 + 4096) * 128
    assert lib.mi355q_fp8_block_grad_input_workspace_size(8192, 4096, 14336) == 0
    assert lib.mi355q_fp8_block_grad_weight_workspace_size(0, 16, 16) == 0
    assert lib.mi355q_fp8_block_grad_weight_workspace_size(32, 4096, 4096) == 0
    assert lib.mi355q_fp8_block_grad_weight_workspace_size(32, 4095, 4096) == 32 * 4096 * 2


def test_host_tensors_are_refused():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    c, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2)
    for call in (lambda: ops.fp8_quantize_groups(x), lambda: ops.fp8_quantize_blocks(x),
                 lambda: ops.fp8_block_matmul(c, s, c, s[:1]), lambda: ops.fp8_block_grad_input(x, c, s[:1]),
                 lambda: ops.fp8_silu_mul(x), lambda: ops.fp8_silu_mul_backward(x, c, s)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_module_shapes():
    w = torch.zeros(128, 256)
    with pytest.raises(ValueError, match="gated MLP"):
        Fp8GatedMLP(w, w, w)
    with pytest.raises(ValueError, match="256"):
        _rows(torch.zeros(3, 128), 256, "input")
    with pytest.raises(TypeError, match="bf16"):
        _rows(torch.zeros(3, 256, dtype=torch.int32), 256, "input")
    assert _rows(torch.zeros(2, 3, 256), 256, "input").shape == (6, 256)
