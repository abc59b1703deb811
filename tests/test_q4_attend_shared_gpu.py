"""4-bit ring attention (``q4_attend_``) where its CTAs share rows' and heads' work, on a B200, against a masked softmax in
64 bits over what the ring holds.

Tolerances, derived before the first run: 1e-5 of a row's norm in float32 (a score is a sum of at most 128 products, off by
some 2^-22 of their magnitudes, which weights and output take over relatively), 5e-3 in 16 bits (the output's rounding, 2^-9).
"""

from __future__ import annotations

import pytest
import torch

from test_q4_attend_precision_gpu import _full, _rel, _step, _want
from vesper_b200.kernels.q4_cache import Q4RingKVCache, q4_attend_, q4_read, q4_write_

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
TOL = {torch.float32: 1e-5, torch.bfloat16: 5e-3, torch.float16: 5e-3}
NAMES = ("k_codes", "k_params", "v_codes", "v_params", "pos")


def _held(ring: Q4RingKVCache, lengths: list[int]) -> Q4RingKVCache:
    """``ring`` cut to the first ``lengths[i]`` positions of each row."""
    n = torch.tensor(lengths, device=CUDA)[:, None]
    ring.pos.masked_fill_(torch.arange(ring.pos.shape[1], device=CUDA) >= n, -1)
    return ring


def _check(ring: Q4RingKVCache, h: int, pos: list[int], seed: int, dtype: torch.dtype) -> None:
    b, hkv, dk = ring.k_codes.shape[0], ring.k_codes.shape[1], ring.head_dim
    q, k, v, at = _step(b, h, hkv, dk, pos, seed, dtype)
    other = Q4RingKVCache(*(getattr(ring, n).clone() for n in NAMES), ring.window)
    o = q4_attend_(q, k, v, at, ring)
    q4_write_(other, k, v, at)  # the token is in the ring as a chunk's write leaves it, and nothing else has changed
    for name in NAMES:
        assert torch.equal(getattr(ring, name), getattr(other, name)), name
    want = _want(ring, q, at)
    for i, p in enumerate(pos):
        if p < 0:
            assert not bool(o[i].any()), i
        else:
            assert _rel(o[i], want[i]) < TOL[dtype], (i, p)
    assert torch.equal(q4_attend_(q, k, v, at, ring), o)  # the same bits again


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("hkv", "h", "dk"), [(8, 32, 128), (8, 16, 64), (3, 24, 80)])
def test_rows_of_uneven_length_over_many_tiles(hkv: int, h: int, dk: int, dtype: torch.dtype) -> None:
    """Over 32 tiles a CTA, so that a unit's opening counts: shares begin and end in openings of rows of other lengths."""
    lengths = [40000, 100, 17, 31011, 0, 39999, 2048, 25601, 6000, 12345]
    ring = _held(_full(len(lengths), hkv, dk, 40000, 41, dtype), lengths)
    _check(ring, h, [-7 if i == 3 else x for i, x in enumerate(lengths)], 42, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(("hkv", "h"), [(1, 9), (1, 16), (2, 24), (1, 40), (2, 10)])
@pytest.mark.parametrize(("dk", "window"), [(64, 1500), (128, 9000)])
def test_more_than_eight_heads_to_a_key_head_share_long_windows(dk: int, window: int, hkv: int, h: int, dtype: torch.dtype) -> None:
    """Head tiles of their own spans and partials, the last of them not full; the first writes the token."""
    lengths = [window, 1, window // 3, window - 1]
    ring = _held(_full(len(lengths), hkv, dk, window, 43, dtype), lengths)
    _check(ring, h, lengths, 44, dtype)
