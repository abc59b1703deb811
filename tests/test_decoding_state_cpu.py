"""A decoding state's windows on a CPU-only machine: 4 bits are held by rings only."""

from __future__ import annotations

import pytest
import torch

from vesper_b200.column import ColumnShape, init_column_state


def test_4_bit_windows_without_rings_are_refused() -> None:
    shape = ColumnShape(d=64, heads=4, kv_groups=2, head_dim=16, window=20, rotary_base=1e4, ffn_mult=2, block=16, key_conv=4)
    with pytest.raises(ValueError, match="needs ring=True"):
        init_column_state(shape, 1, 1, torch.bfloat16, torch.device("cpu"), q4=True)
