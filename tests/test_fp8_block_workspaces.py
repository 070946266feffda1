"""Workspace sizes of the block-scaled fp8 products (CPU only: no kernel launches)."""
import pytest

from llmcompressor_amd import _lib

TILE = 64 * 128 * 4     # bytes of the smallest partial tile; the others are multiples of it


@pytest.mark.parametrize("query,rows,out,cols", [
    ("matmul", 333, 4096, 14336), ("matmul", 64, 512, 4096), ("matmul", 100, 4096, 4096),
    ("grad_input", 16, 4096, 4096), ("grad_input", 450, 12544, 7936),
    ("grad_weight", 8192, 1024, 4096), ("grad_weight", 8200, 136, 272),
])
def test_products_of_few_tiles_ask_for_split_sums(query, rows, out, cols):
    """Two parts or more of at least one tile, whole tiles only."""
    n = getattr(_lib.load_library(), f"mi355q_fp8_block_{query}_workspace_size")(rows, out, cols)
    assert n >= 2 * TILE and n % TILE == 0


@pytest.mark.parametrize("query,rows,out,cols,copies", [
    ("matmul", 100, 4096, 4095, (100 + 4096) * 4096),
    ("grad_input", 16, 4095, 4096, 16 * 4096 * 2),
    ("grad_input", 16, 4096, 4095, 4096 * 4096),
    ("grad_weight", 8192, 1023, 4096, 8192 * 1024 * 2),
    ("grad_weight", 8192, 1024, 4095, 8192 * 4096),
])
def test_odd_widths_add_their_padded_copies(query, rows, out, cols, copies):
    """To the same split sums as the next width of whole chunks has."""
    size = getattr(_lib.load_library(), f"mi355q_fp8_block_{query}_workspace_size")
    splits = size(rows, -(-out // 8) * 8, -(-cols // 16) * 16)
    assert splits > 0 and size(rows, out, cols) == splits + copies
