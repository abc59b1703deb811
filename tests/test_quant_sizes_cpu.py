"""Sizes at the end of 32 bits in the quantised operators' entry points, on a CPU-only machine: refused by name.

Each is refused before a pointer is touched or anything is launched, so no GPU and no memory of such a size is needed.
"""

from __future__ import annotations

import pytest
import torch

from vesper_b200 import _lib
from vesper_b200.contracts import ContractError
from vesper_b200.kernels.q8 import check_width

INT_MAX = 2**31 - 1


def _refused(name: str, *args: object, match: str) -> None:
    with pytest.raises(_lib.KernelError, match=match):
        _lib.call(name, *args)


@pytest.mark.parametrize(("m", "n"), [(INT_MAX, 16), (INT_MAX - 254, 16), (1, INT_MAX), (INT_MAX, INT_MAX)])
def test_products_whose_tiles_no_int_counts_are_refused(m: int, n: int) -> None:
    _refused("vb_linear_q8", None, 16, None, None, 16, None, None, m, n, 16, 0, None, None, match="of at most 2147483392")


def test_rows_whose_width_no_int_walks_are_refused() -> None:
    wide = 2**30 + 1
    _refused("vb_rms_norm_q8", None, None, None, None, None, wide, None, 1, wide, 1e-3, 1e-6, 0, 0, None, match="exceed 2\\^30")
    _refused("vb_quantize_rows_q8", None, INT_MAX, None, INT_MAX, None, 1, INT_MAX, 0, 0, None, match="exceed 2\\^30")
    _refused("vb_dequantize_rows_q8", None, wide, None, None, 1, wide, 0, None, match="exceed 2\\^30")


def test_chunks_whose_tokens_no_int_counts_are_refused() -> None:
    ring = [None] * 5
    _refused("vb_q4_write", *ring, None, 0, 0, None, 0, 0, None, 1, INT_MAX, 1, 64, 8, 64, 0, None, match="exceed the grid")
    _refused("vb_q4_read", *ring, None, None, None, None, 1, 2**30 + 1, 1, 64, 64, 64, 0, None, match="exceed the grid")


def test_the_python_entry_points_refuse_what_an_int_would_cut() -> None:
    """Views of one number stand for rows of 2^32 + 4 channels, of which an int holds 4."""
    wide = torch.zeros(1, device="meta").expand(1, 2**32 + 4)
    for call in (lambda: check_width("x", wide), lambda: check_width("q", wide.to(torch.int8))):
        with pytest.raises(ContractError, match="at most 1073741824 channels"):
            call()
