"""Sizes at the end of 32 bits in the quantised operators' entry points, on a CPU-only machine: refused by name.

Each is refused before a pointer is touched or anything is launched, so no GPU and no memory of such a size is needed.
"""

from __future__ import annotations

import pytest

from vesper_b200 import _lib

INT_MAX = 2**31 - 1


def _refused(name: str, *args: object, match: str) -> None:
    with pytest.raises(_lib.KernelError, match=match):
        _lib.call(name, *args)


@pytest.mark.parametrize(("m", "n"), [(INT_MAX, 16), (INT_MAX - 254, 16), (1, INT_MAX), (INT_MAX, INT_MAX)])
def test_products_whose_tiles_no_int_counts_are_refused(m: int, n: int) -> None:
    _refused("vb_linear_q8", None, 16, None, None, 16, None, None, m, n, 16, 0, None, None, match="of at most 2147483392")
