"""Block-scaled fp8 at the ends of its ranges, against the 64-bit definitions of test_gpu_fp8_blocks."""
import math

import pytest
import torch

from test_gpu_fp8_blocks import E4M3, E8M0, G, check_codes, check_sum, gen, heavy, ops, values

pytestmark = pytest.mark.gpu


def smallest_steps(n):
    """Whole numbers as multiples of 2^-149, fp32's smallest step, exactly."""
    n = n.to(torch.int32)
    return torch.where(n < 0, n.abs() - 2 ** 31, n).to(torch.int32).view(torch.float32)


def ramps(tops, cols):
    """A row of ``cols`` numbers for each top: the top, and signed fractions of it."""
    part = torch.linspace(1, 0, cols, dtype=torch.float64) * (1 - 2 * (torch.arange(cols) % 2))
    return torch.round(tops.double()[:, None] * part)


@pytest.mark.parametrize("cols", [128, 131])
def test_groups_whose_scale_is_a_few_smallest_steps(dev, cols):
    """Largest magnitudes of n 2^-149: a / 448 is rounded to whole steps there, for n = 465 .. 671 to one step, and the
    quotients pass e4m3's largest value, by a half at the most.  They are clamped to it; finite groups hold no NaN."""
    x = smallest_steps(ramps(torch.arange(1, 7201), cols))
    codes, scales = ops().fp8_quantize_groups(x.to(dev))
    assert bool(torch.isfinite(codes.float()).all()) and bool(torch.isfinite(scales).all())
    check_codes(codes, scales, x, 1, torch.float32)
    codes, scales = ops().fp8_quantize_groups(x.to(dev), E8M0)
    check_codes(codes, scales, x, 1, E8M0)


@pytest.mark.parametrize("cols", [128, 200])
def test_blocks_whose_scale_is_a_few_smallest_steps(dev, cols):
    tops = torch.tensor([1, 224, 225, 464, 465, 500, 671, 672, 1100, 1119, 3000, 7000])
    x = smallest_steps(ramps(tops.repeat_interleave(G) - torch.arange(len(tops) * G) % G % tops.repeat_interleave(G), cols))
    codes, scales = ops().fp8_quantize_blocks(x.to(dev))
    assert bool(torch.isfinite(codes.float()).all()) and bool(torch.isfinite(scales).all())
    check_codes(codes, scales, x, G, torch.float32)
