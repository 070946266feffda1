"""Argument checks of the 4-bit products and the token kernels that need no device."""
import ctypes as C

import pytest

from llmcompressor_amd import _lib

P = C.c_void_p(16)


def w4(lib, **k):
    a = dict(x=P, xt=_lib.BF16, n_x=4, ldx=256, rows_idx=None, offsets=None, experts=1, w=P, fmt=_lib.W4_INT4, ldw=128,
             sw=0, s=P, st=_lib.BF16, lds=2, ss=0, z=None, ldz=0, sz=0, group=128, bias=None, bt=0, gated=0, y=P,
             yt=_lib.BF16, ldy=16, rows=4, out=16, cols=256, ws=None, wsb=0)
    a.update(k)
    return lib.mi355q_w4a16_matmul(*a.values(), None)


@pytest.mark.parametrize("args,needle", [
    (dict(fmt=7), "format"), (dict(xt=_lib.F32), "bf16 or fp16"), (dict(yt=9), "dtype"), (dict(st=9), "dtype"),
    (dict(out=0), "sizes"), (dict(rows=-1), "sizes"), (dict(cols=7), "8 columns"), (dict(gated=1, out=15), "halves"),
    (dict(experts=2), "offsets"), (dict(n_x=3), "fewer rows"), (dict(group=48), "groups"), (dict(group=0), "groups"),
    (dict(fmt=_lib.W4_MXFP4, group=128), "MXFP4"), (dict(fmt=_lib.W4_MXFP4, group=32, z=P), "MXFP4"),
    (dict(fmt=_lib.W4_MXFP4, group=32, cols=264), "MXFP4"), (dict(x=None), "null"), (dict(w=None), "null"),
    (dict(ldw=64), "overlap"), (dict(ldw=130), "4-byte"), (dict(w=C.c_void_p(18)), "4-byte"), (dict(ldy=15), "overlap"),
    (dict(ldx=-256), "pitch"), (dict(group=2 ** 63 - 1, x=None), "null"),
    (dict(offsets=P, rows=2 ** 31, n_x=2 ** 31), "too many"),
])
def test_product_arguments(args, needle):
    lib = _lib.load_library()
    assert w4(lib, **args) == _lib.INVALID_ARGUMENT
    assert needle in lib.mi355q_last_error().decode()


def test_product_of_no_rows_needs_no_operands():
    assert w4(_lib.load_library(), rows=0, n_x=0, x=None, y=None) == _lib.OK


def test_workspaces():
    lib = _lib.load_library()
    f = lib.mi355q_w4a16_matmul_workspace_size
    assert f(1, 1, 1, 4096, 4096, _lib.W4_INT4, 128) == 0
    assert f(0, 0, 1, 4096, 4096, _lib.W4_INT4, 128) == 0
    assert f(-1, 4, 1, 16, 64, _lib.W4_INT4, 0) == 0
    assert f(256, 256, 1, 512, 1024, _lib.W4_INT4, 2 ** 63 - 1) == f(256, 256, 1, 512, 1024, _lib.W4_INT4, 1024)
    # many rows: sums of x and factors (three 16-bit pieces a group), scales in fp32, a copy of x
    assert f(256, 256, 1, 512, 1024, _lib.W4_INT4, 128) >= (256 + 512) * 3 * 16 * 2 + 512 * 16 * 4 + 256 * 1024 * 2
    g = lib.mi355q_moe_plan_workspace_size
    assert g(1, 8, 128) == 0 and g(256, 8, 128) == 0                  # one workgroup
    assert g(8192, 8, 128) == 32 * 129 * 4
    assert g(2 ** 31, 2, 4) == 0 and g(5, 1, 5000) == 0


@pytest.mark.parametrize("call,needle", [
    (lambda l: l.mi355q_moe_plan(P, 16, 4, 2, 2, 8, P, P, P, None, 0, None), "32 or 64"),
    (lambda l: l.mi355q_moe_plan(P, 64, 4, 0, 2, 8, P, P, P, None, 0, None), "top"),
    (lambda l: l.mi355q_moe_plan(P, 64, 2 ** 30, 4, 4, 8, P, P, P, None, 0, None), "2^31"),
    (lambda l: l.mi355q_moe_plan(P, 64, 4, 2, 2, 0, P, P, P, None, 0, None), "positive"),
    (lambda l: l.mi355q_moe_plan(None, 64, 4, 2, 2, 8, P, P, P, None, 0, None), "null"),
    (lambda l: l.mi355q_moe_plan(P, 64, 4, 2, 1, 8, P, P, P, None, 0, None), "overlap"),
    (lambda l: l.mi355q_moe_plan(P, 64, 8192, 8, 8, 128, P, P, P, P, 100, None), "workspace"),
    (lambda l: l.mi355q_moe_sort(P, 9, 4, 2, 8, 8, P, P, P, 8, None), "dtype"),
    (lambda l: l.mi355q_moe_sort(P, 0, 4, 2, 0, 8, P, P, P, 8, None), "cols"),
    (lambda l: l.mi355q_moe_sort(P, 0, 4, 2, 8, 8, None, P, P, 8, None), "slots"),
    (lambda l: l.mi355q_moe_sort(P, 0, 4, 2, 8, 8, P, P, P, 4, None), "overlap"),
    (lambda l: l.mi355q_moe_combine(P, 0, 4, 2, 8, 8, P, 9, P, P, P, 8, None), "weights"),
    (lambda l: l.mi355q_moe_combine(None, 0, 4, 2, 8, 8, P, 1, P, P, P, 8, None), "null"),
    (lambda l: l.mi355q_moe_combine_backward(P, 0, 4, 2, 8, 8, None, 8, P, 1, P, P, P, 8, P, None), "null"),
    (lambda l: l.mi355q_moe_combine_backward(P, 0, 4, 2, 8, 8, P, 8, P, 1, P, P, P, 4, P, None), "overlap"),
])
def test_token_arguments(call, needle):
    lib = _lib.load_library()
    assert call(lib) == _lib.INVALID_ARGUMENT
    assert needle in lib.mi355q_last_error().decode()


def test_too_many_experts_are_unsupported():
    lib = _lib.load_library()
    assert lib.mi355q_moe_plan(P, 64, 4, 2, 2, 2041, P, P, P, None, 0, None) == _lib.UNSUPPORTED


def test_host_tensors_are_refused():
    import torch

    from llmcompressor_amd import ops
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.moe_plan(torch.zeros(2, 2, dtype=torch.int64), 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.w4a16_matmul(torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.int32),
                         torch.zeros(4, 1, dtype=torch.bfloat16))


@pytest.mark.parametrize("cols,fmt,group", [(1024, _lib.W4_INT4, 128), (1032, _lib.W4_INT4, 32), (1024, _lib.W4_MXFP4, 32),
                                            (1023, _lib.W4_INT4, 128)])
def test_workspace_without_a_copy_of_x(cols, fmt, group):
    """Less by x with rows of whole steps of 128 columns; rows of an odd number of columns are copied all the same."""
    lib = _lib.load_library()
    for n_x, rows, experts in ((256, 256, 1), (1000, 4000, 4)):
        args = n_x, rows, experts, 512, cols, fmt, group
        copy = n_x * -(-cols // 128) * 128 * 2 if cols % 8 == 0 else 0
        assert lib.mi355q_w4a16_matmul_workspace_size(*args) - lib.mi355q_w4a16_matmul_workspace_size_in_place(*args) == copy
    assert lib.mi355q_w4a16_matmul_workspace_size_in_place(1, 1, 1, 4096, 4096, _lib.W4_INT4, 128) == 0
