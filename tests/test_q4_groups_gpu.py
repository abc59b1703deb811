"""Groups at the end of float32's range in the 4-bit ring (``q4_write_``, ``q4_read``) on a B200: as long as a group's range is
finite it has the codes that its definition gives, bit for bit; one past it is NaN as a whole."""

from __future__ import annotations

import pytest
import torch

from test_q4_cache_gpu import _toward
from vesper_b200.kernels.q4_cache import group_size, q4_attend_, q4_read, q4_ring_empty, q4_write_

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
LARGEST = {torch.float32: torch.finfo(torch.float32).max, torch.bfloat16: torch.finfo(torch.bfloat16).max}


def _stored(x: torch.Tensor) -> torch.Tensor:
    """What a ring keeps of ``x [..., dk]``: codes by float32 steps, the value ``lo + code * step`` rounded once."""
    g = x.float().unflatten(-1, (-1, group_size(x.shape[-1])))
    lo = _toward(g.amin(-1, keepdim=True), False)
    span = g.amax(-1, keepdim=True) - lo
    step = _toward(span / 15, True)
    code = torch.round((g - lo) / step).clamp(max=15)
    value = (lo.double() + code.double() * step.double()).float()
    return torch.where(torch.isfinite(step) & torch.isfinite(lo), value, torch.nan).flatten(-2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk", [64, 48])
def test_ranges_up_to_the_largest_number(dk: int, dtype: torch.dtype) -> None:
    top = LARGEST[dtype]
    g = torch.Generator().manual_seed(61)
    x = torch.rand(1, 8, 1, dk, generator=g)
    lows = [0.0, -1.2e36, -1.3e36, 1e36, -0.5 * top, 0.9 * top, -top, -1.0]
    for i, low in enumerate(lows):
        high = top if i < 6 else 0.0 if i == 6 else 1.0
        x[0, i] = low + x[0, i] * (high * 0.5 - low * 0.5)
        x[0, i, 0, ::16] = low
        x[0, i, 0, 5::16] = high
    x = x.to(dtype)
    pos = torch.arange(8)[None].to(CUDA)
    for write in ("chunk", "tokens"):
        ring = q4_ring_empty(1, 1, dk, 8, CUDA)
        if write == "chunk":
            q4_write_(ring, x.to(CUDA), x.to(CUDA), pos)
        else:
            for i in range(8):
                t = x[:, i : i + 1].to(CUDA)
                q4_attend_(torch.zeros_like(t), t, t, pos[:, i : i + 1], ring)
        k, v, held = q4_read(ring, pos, torch.float32)
        want = _stored(x)
        assert bool(held.all())
        for got in (k.cpu(), v.cpu()):
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(got, 0.0, 7.0, -7.0), torch.nan_to_num(want, 0.0, 7.0, -7.0))
    # a range of 1.5 times the largest number; ranges of just the largest (float32) and just above 3.4e38 (bf16)
    assert bool(torch.isnan(want[0, 4]).all()) and not bool(torch.isnan(want[0, [0, 3, 5, 7]]).any())
    assert bool(torch.isnan(want[0, [1, 2]]).any()) == (dtype == torch.float32)
