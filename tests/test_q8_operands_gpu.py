"""The quantised operators' operands as callers have them (strided scales, positions), on a B200.

Tolerance: the int32 sum of the product is exact, its conversion and two products round three times, 3 * 2^-24 of each output.
"""

from __future__ import annotations

import pytest
import torch

from vesper_b200 import _lib
from vesper_b200.kernels.q4_cache import q4_read, q4_ring_empty, q4_write_
from vesper_b200.kernels.q8 import dequantize_rows_q8, linear_q8

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")


def _codes(n: int, k: int, seed: int) -> torch.Tensor:
    return torch.randint(-127, 128, (n, k), generator=torch.Generator().manual_seed(seed), dtype=torch.int8).to(CUDA)


def _scales(n: int, seed: int, strided: bool) -> torch.Tensor:
    t = (0.5 + torch.rand(n, 3, generator=torch.Generator().manual_seed(seed))).to(CUDA)
    return t[:, 1] if strided else t[:, 1].contiguous()


def _check(xq: torch.Tensor, xs: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor) -> None:
    y = linear_q8(xq, xs, wq, ws, torch.float32)
    want = (xq.cpu().double() @ wq.cpu().double().T) * xs.cpu().double()[:, None] * ws.cpu().double()
    assert bool(((y.cpu().double() - want).abs() <= 3 * 2.0**-24 * want.abs()).all())


@pytest.mark.parametrize(("m", "n"), [(64, 64), (1, 100), (128, 17), (300, 300), (700, 2000)])
@pytest.mark.parametrize(("x_strided", "w_strided"), [(True, True), (True, False), (False, True)])
def test_strided_scales_of_tokens_and_channels(m: int, n: int, x_strided: bool, w_strided: bool) -> None:
    """Each operand's scales keep their own copy, whichever of them are copied."""
    _check(_codes(m, 64, 1), _scales(m, 2, x_strided), _codes(n, 64, 3), _scales(n, 4, w_strided))


@pytest.mark.parametrize(("x_strided", "w_strided"), [(True, False), (False, True), (True, True)])
def test_strided_scales_in_a_process_s_first_product(monkeypatch: pytest.MonkeyPatch, x_strided: bool, w_strided: bool) -> None:
    """The device's status word is made on first use: it takes no operand's memory."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    xq, xs, wq, ws = _codes(5, 64, 5), _scales(5, 6, x_strided), _codes(7, 64, 7), _scales(7, 8, w_strided)
    monkeypatch.setattr(_lib, "_STATUS", {})
    _check(xq, xs, wq, ws)
    _lib.check_status(CUDA)


def test_strided_scales_and_positions_of_what_is_read_back() -> None:
    q, s = _codes(40, 96, 9), _scales(40, 10, True)
    assert torch.equal(dequantize_rows_q8(q, s), q.float() * s[:, None])
    ring = q4_ring_empty(2, 1, 32, 50, CUDA)
    k = torch.randn(2, 30, 1, 32, device=CUDA)
    at = torch.arange(30, device=CUDA).expand(2, 30)
    q4_write_(ring, k, k, at)
    got, want = q4_read(ring, at[:, ::3], torch.float32), q4_read(ring, at[:, ::3].contiguous(), torch.float32)
    assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True)) and bool(got[2].all())
