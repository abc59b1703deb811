"""The quantised operators' C entry points on a CPU-only machine: bad arguments are refused.

Each call returns an error status with the reason in its message before it touches a pointer or
launches anything, so no GPU is needed.
"""

from __future__ import annotations

import pytest

from vesper_b200 import _lib


def _refused(name: str, *args: object, match: str) -> None:
    with pytest.raises(_lib.KernelError, match=match):
        _lib.call(name, *args)


def test_the_8_bit_row_entry_points_refuse_bad_arguments_without_a_gpu() -> None:
    _refused("vb_rms_norm_q8", None, None, None, None, None, 8, None, 4, 16, 1e-3, 1e-6, 0, 0, None, match="row pitch=8")
    _refused("vb_rms_norm_q8", 16, 16, 16, None, 16, 16, 16, 4, 16, 1e-3, 1e-6, 0, 0, None, match="come together")
    _refused("vb_rms_norm_q8", 16, 16, 16, 16, 16, 16, 16, 4, 16, 1e-3, 1e-6, 1, 0, None, match="stream is float32")
    _refused("vb_rms_norm_q8", None, None, None, None, None, 16, None, 4, 16, 1e-3, 1e-6, 0, 0, None, match="null pointer")
    _refused("vb_quantize_rows_q8", None, 15, None, 16, None, 4, 16, 0, 0, None, match="row pitch 15")
    _refused("vb_quantize_rows_q8", None, 16, None, 16, None, 4, 16, 0, 7, None, match="dtype code 7")
    _refused("vb_dequantize_rows_q8", None, 16, None, None, 1 << 32, 16, 0, None, match="exceed 2")
    _refused("vb_linear_q8", None, 64, None, None, 64, None, None, 4, 0, 64, 0, None, None, match="bad shape")
    _refused("vb_linear_q8", None, 1 << 20, None, None, 1 << 20, None, None, 4, 4, 131072, 0, None, None, match="131056")
    _refused("vb_linear_q8", None, 64, None, None, 64, None, None, 4, 4, 64, 0, None, None, match="null pointer")


def test_the_4_bit_cache_entry_points_refuse_bad_arguments_without_a_gpu() -> None:
    ring = [None] * 5
    _refused("vb_q4_write", *ring, None, 0, 0, None, 0, 0, None, 1, 1, 1, 40, 8, 64, 0, None, match="multiple of 16")
    _refused("vb_q4_write", *ring, None, 0, 0, None, 0, 0, None, 1, 1, 1, 64, 65, 64, 0, None, match="holding the window 65")
    _refused("vb_q4_write", *ring, None, 0, 0, None, 0, 0, None, 1, 1, 1, 64, 64, 64, 0, None, match="null pointer")
    _refused("vb_q4_read", *ring, None, None, None, None, 1, 1, 1, 64, 64, 100, 0, None, match="multiple of 64")
    _refused("vb_q4_read", *ring, None, None, None, None, 1, 1, 1, 64, 64, 64, 9, None, match="dtype code 9")
    attend = [None, 0, None, 0, None, 0, None, *ring, None, None]
    _refused("vb_q4_attend", *attend, 1, 3, 2, 64, 64, 64, 0, None, match="not a multiple of 2 key heads")
    _refused("vb_q4_attend", *attend, 1, 2, 2, 64, 64, 64, 0, None, match="null pointer")
    assert _lib.query("vb_q4_attend_workspace", 64, 8, 2, 64, 512) == 0  # a CTA per row and key head
    assert _lib.query("vb_q4_attend_workspace", 1, 8, 2, 64, 4096) > 0
