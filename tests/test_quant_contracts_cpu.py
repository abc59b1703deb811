"""The quantised operators' Python entry points on a CPU-only machine: what they refuse before any kernel runs."""

from __future__ import annotations

import pytest
import torch

from vesper_b200.column import ColumnShape, init_column_state, map_state, state_tensors
from vesper_b200.contracts import ContractError
from vesper_b200.kernels.q4_cache import Q4RingKVCache, group_size, q4_attend_, q4_read, q4_ring_empty, q4_write_
from vesper_b200.kernels.q8 import add_rms_norm_q8, dequantize_rows_q8, linear_q8, quantize_rows_q8, rms_norm_q8

CPU = torch.device("cpu")


def test_cpu_tensors_are_refused() -> None:
    x, w = torch.ones(2, 32), torch.ones(32)
    q, s = torch.ones(2, 32, dtype=torch.int8), torch.ones(2)
    with pytest.raises(ContractError, match="CUDA only"):
        rms_norm_q8(x, w, 1e-3, 1e-6)
    with pytest.raises(ContractError, match="CUDA only"):
        add_rms_norm_q8(x, x, w, 1e-3, 1e-6)
    with pytest.raises(ContractError, match="CUDA only"):
        quantize_rows_q8(x)
    with pytest.raises(ContractError, match="CUDA only"):
        dequantize_rows_q8(q, s)
    with pytest.raises(ContractError, match="CUDA only"):
        linear_q8(q, s, q, s)
    ring = q4_ring_empty(2, 1, 32, 10, CPU)
    k, pos = torch.zeros(2, 1, 1, 32), torch.zeros(2, 1, dtype=torch.long)
    for call in (lambda: q4_write_(ring, k, k, pos), lambda: q4_read(ring, pos), lambda: q4_attend_(k, k, k, pos, ring)):
        with pytest.raises(ContractError, match="CUDA only"):
            call()


@pytest.mark.parametrize(("dk", "groups"), [(16, 1), (32, 1), (48, 3), (64, 2), (80, 5), (96, 3), (112, 7), (128, 4)])
def test_an_empty_ring_has_the_layout_it_says(dk: int, groups: int) -> None:
    ring = q4_ring_empty(3, 2, dk, 65, CPU)
    assert ring.k_codes.shape == ring.v_codes.shape == (3, 2, 128, dk // 2) and ring.k_codes.dtype == torch.uint8
    assert ring.k_params.shape == ring.v_params.shape == (3, 2, 128, groups, 2) and ring.k_params.dtype == torch.bfloat16
    assert ring.pos.shape == (3, 128) and bool((ring.pos == -1).all()) and ring.window == 65
    assert ring.head_dim == dk and groups * group_size(dk) == dk


def test_bad_rings_are_refused() -> None:
    for dk in (0, 8, 24, 130, 144):
        with pytest.raises(ContractError, match="multiple of 16"):
            q4_ring_empty(1, 1, dk, 8, CPU)
    for window in (0, -1, 2**31):
        with pytest.raises(ValueError, match="window must be at least 1"):
            q4_ring_empty(1, 1, 64, window, CPU)


def test_a_decoding_state_can_carry_4_bit_rings() -> None:
    shape = ColumnShape(d=64, heads=4, kv_groups=2, head_dim=16, window=20, rotary_base=1e4, ffn_mult=2, block=16, key_conv=4)
    state = init_column_state(shape, 2, 3, torch.bfloat16, CPU, ring=True, q4=True)
    assert all(isinstance(c, Q4RingKVCache) for c in state.kv)
    assert len(state_tensors([state])) == 3 * (1 + 5 + 1)  # per pass a state, five ring tensors and a key history
    copy = map_state(state, torch.clone)
    assert copy.kv[0].window == 20 and torch.equal(copy.kv[2].pos, state.kv[2].pos)
    plain = init_column_state(shape, 2, 3, torch.bfloat16, CPU, ring=True)
    assert not any(isinstance(c, Q4RingKVCache) for c in plain.kv)
