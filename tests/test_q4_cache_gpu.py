"""The 4-bit ring cache (``vesper_b200.kernels.q4_cache``) on a B200: written, read and attended.

Tolerances, derived before the first run:

- quantisation is float32 arithmetic without sums (extremes, directed roundings, a quotient), so what is read back equals
  the same steps written out in torch on the CPU, bit for bit, and lies within half a step of the input;
- attention over the values the ring holds, against a masked softmax in 64 bits: in float32 a score is a sum of at most
  128 products, off by some 2^-22 of the sum of their magnitudes (about 1e-6 for unit keys and queries), which a weight and
  then the output take over relatively: 1e-5 of the output's norm. In bf16 and f16 the weights are rounded to
  8 bits or more (2^-9 each, of both signs) and the output once (2^-9): 5e-3.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import rel
from vesper_b200.contracts import ContractError
from vesper_b200.kernels.q4_cache import Q4RingKVCache, group_size, q4_attend_, q4_read, q4_ring_empty, q4_write_

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
TOL = {torch.float32: 1e-5, torch.bfloat16: 5e-3, torch.float16: 5e-3}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _toward(x: torch.Tensor, up: bool) -> torch.Tensor:
    """Float32 to the nearest bf16 value not below (``up``) or not above ``x``."""
    near = x.to(torch.bfloat16)
    side = torch.full_like(near, math.inf if up else -math.inf)
    wrong = near.float() < x if up else near.float() > x
    return torch.where(wrong, torch.nextafter(near, side), near).float()


def _stored(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """What a ring keeps of ``x [..., dk]`` (float32 on the CPU), and its steps per channel."""
    size = group_size(x.shape[-1])
    g = x.float().cpu().unflatten(-1, (-1, size))
    lo = _toward(g.amin(-1, keepdim=True), False)
    span = g.amax(-1, keepdim=True) - lo
    step = torch.where(span < 2.0**-100, 0.0, _toward(span / 15, True))
    code = torch.where(step > 0, torch.round((g - lo) / step).clamp(max=15), 0.0)
    value = torch.where(torch.isfinite(step) & torch.isfinite(lo), lo + code * step, math.nan)
    return value.flatten(-2), step.expand_as(g).flatten(-2)


def _tokens(b: int, n: int, hkv: int, dk: int, seed: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    g = torch.Generator().manual_seed(seed)
    shift = 3 * torch.randn(hkv, dk, generator=g) * (torch.rand(hkv, dk, generator=g) < 0.2)
    k = (torch.randn(b, n, hkv, dk, generator=g) + shift).to(dtype)
    return k, torch.randn(b, n, hkv, dk, generator=g).to(dtype)


def _positions(first: list[int], n: int) -> torch.Tensor:
    return torch.tensor(first)[:, None] + torch.arange(n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk", [16, 32, 48, 64, 80, 96, 112, 128])
def test_what_is_read_back_is_the_nearest_code(dk: int, dtype: torch.dtype) -> None:
    b, n, hkv, window = 3, 21, 3, 40
    k, v = _tokens(b, n, hkv, dk, dk, dtype)
    pos = _positions([0, 35, 1000], n)
    ring = q4_write_(q4_ring_empty(b, hkv, dk, window, CUDA), k.to(CUDA), v.to(CUDA), pos.to(CUDA))
    k2, v2, held = q4_read(ring, pos.to(CUDA), torch.float32)
    assert bool(held.all())
    for got, x in ((k2, k), (v2, v)):
        want, step = _stored(x)
        assert torch.equal(got.cpu(), want)
        assert bool(((want - x.float()).abs() <= step / 2 * (1 + 2.0**-20)).all())
    k3, v3, _ = q4_read(ring, pos.to(CUDA), dtype)
    assert torch.equal(k3, k2.to(dtype)) and torch.equal(v3, v2.to(dtype))


def test_hard_groups() -> None:
    """Constant, zero, tiny, huge, far from zero, one outlier, not finite: each group on its own."""
    dk = 64
    k, v = _tokens(1, 16, 1, dk, 5, torch.float32)
    k[0, 0] = 0
    k[0, 1] = -3.3
    k[0, 2] *= 1e-33
    k[0, 3] *= 1e35
    k[0, 4] += 1e4
    k[0, 5, 0, 7] = 1e6
    k[0, 6, 0, 40] = math.nan
    k[0, 7, 0, 3] = math.inf
    k[0, 8, 0, 63] = -math.inf
    k[0, 9] *= 3e38 / k[0, 9].abs().max()
    k[0, 10, 0, :32] = 2.0**-60
    k[0, 11] = -0.0
    pos = _positions([0], 16).to(CUDA)
    ring = q4_write_(q4_ring_empty(1, 1, dk, 16, CUDA), k.to(CUDA), v.to(CUDA), pos)
    got, _, _ = q4_read(ring, pos, torch.float32)
    want, step = _stored(k)
    got = got.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert bool(torch.isnan(got[0, 6, 0, 32:]).all()) and not bool(torch.isnan(got[0, 6, 0, :32]).any())
    fine = ~torch.isnan(want)
    assert bool(((want - k).abs() <= step / 2 * (1 + 2.0**-20))[fine & (k.abs() > 2.0**-90)].all())


@pytest.mark.parametrize(("n", "window"), [(1, 1), (5, 1), (7, 3), (64, 64), (200, 64), (65, 100), (300, 129)])
def test_chunks_longer_than_the_window_keep_the_last(n: int, window: int) -> None:
    b, hkv, dk = 2, 2, 32
    k, v = _tokens(b, n, hkv, dk, n, torch.bfloat16)
    pos = _positions([3, 77], n)
    ring = q4_write_(q4_ring_empty(b, hkv, dk, window, CUDA), k.to(CUDA), v.to(CUDA), pos.to(CUDA))
    k2, v2, held = q4_read(ring, pos.to(CUDA), torch.float32)
    kept = min(n, window)
    assert not bool(held[:, : n - kept].any()) and bool(held[:, n - kept :].all())
    assert not bool(k2[:, : n - kept].any()) and not bool(v2[:, : n - kept].any())
    assert torch.equal(k2.cpu()[:, n - kept :], _stored(k)[0][:, n - kept :])
    assert torch.equal(v2.cpu()[:, n - kept :], _stored(v)[0][:, n - kept :])


def test_chunks_in_turn_equal_one_and_single_tokens() -> None:
    b, n, hkv, dk, window = 2, 150, 2, 64, 100
    k, v = (t.to(CUDA) for t in _tokens(b, n, hkv, dk, 8, torch.bfloat16))
    pos = _positions([11, 500], n).to(CUDA)
    whole = q4_write_(q4_ring_empty(b, hkv, dk, window, CUDA), k, v, pos)
    for cuts in ([0, 1, 40, 41, 150], list(range(151))):
        ring = q4_ring_empty(b, hkv, dk, window, CUDA)
        for i, j in zip(cuts[:-1], cuts[1:], strict=True):
            q4_write_(ring, k[:, i:j], v[:, i:j], pos[:, i:j])  # slices: other strides than dense
        for name in ("k_codes", "k_params", "v_codes", "v_params", "pos"):
            assert torch.equal(getattr(ring, name), getattr(whole, name)), name


def test_padding_is_not_written_and_other_strides_are_read() -> None:
    b, n, hkv, dk, window = 3, 20, 2, 64, 8
    k, v = (t.to(CUDA) for t in _tokens(b, n, hkv, dk, 9, torch.bfloat16))
    pos = torch.full((b, n), -1)
    pos[0, 15:] = torch.arange(5)  # padded in front
    pos[1, :12] = torch.arange(12)  # padded behind: a padding token takes no slot
    ring = q4_ring_empty(b, hkv, dk, window, CUDA)
    # heads and tokens swapped in memory, and both tensors slices of one projection
    both = torch.cat([k, v], 2).transpose(1, 2).contiguous().transpose(1, 2)
    q4_write_(ring, both[:, :, :hkv], both[:, :, hkv:], pos.to(CUDA))
    k2, v2, held = q4_read(ring, pos.to(CUDA), torch.float32)
    want_held = pos >= 0
    want_held[1, :4] = False
    assert torch.equal(held.cpu(), want_held)
    assert torch.equal(k2.cpu(), torch.where(want_held[..., None, None], _stored(k)[0], 0.0))
    assert torch.equal(v2.cpu(), torch.where(want_held[..., None, None], _stored(v)[0], 0.0))
    assert int((ring.pos >= 0).sum()) == 5 + 8


def _attend_want(ring: Q4RingKVCache, q: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """A masked softmax in 64 bits over what the ring holds after the token was written."""
    b, _, h, dk = q.shape
    hkv, w = ring.k_codes.shape[1], ring.window
    at = ring.pos[:, :w]
    k, v, held = q4_read(ring, at, torch.float32)
    out = torch.zeros(b, h, dk, dtype=torch.float64)
    for i in range(b):
        p = int(pos[i])
        if p < 0:
            continue
        seen = held[i] & (at[i] <= p) & (at[i] > p - w)
        ki, vi = k[i, seen].double().cpu(), v[i, seen].double().cpu()
        qi = q[i, 0].double().cpu().view(hkv, h // hkv, dk)
        wt = torch.softmax(torch.einsum("hgd,lhd->hgl", qi, ki) / math.sqrt(dk), -1)
        out[i] = torch.einsum("hgl,lhd->hgd", wt, vi).reshape(h, dk)
    return out[:, None]


def _filled(b: int, hkv: int, dk: int, window: int, held: list[int], seed: int, dtype: torch.dtype) -> Q4RingKVCache:
    """A ring whose row i holds positions 0 .. held[i] - 1 (the last ``window`` of them)."""
    ring = q4_ring_empty(b, hkv, dk, window, CUDA)
    n = max(held)
    if n:
        k, v = _tokens(b, n, hkv, dk, seed, dtype)
        pos = torch.arange(n).expand(b, n).clone()
        for i, x in enumerate(held):
            pos[i, x:] = -1
        q4_write_(ring, k.to(CUDA), v.to(CUDA), pos.to(CUDA))
    return ring


def _check_attend(ring: Q4RingKVCache, h: int, pos: list[int], seed: int, dtype: torch.dtype, scale: float = 1.0) -> None:
    b, hkv, dk = ring.k_codes.shape[0], ring.k_codes.shape[1], ring.head_dim
    g = torch.Generator().manual_seed(seed)
    q = (scale * torch.randn(b, 1, h, dk, generator=g)).to(dtype).to(CUDA)
    k, v = (t.to(CUDA) for t in _tokens(b, 1, hkv, dk, seed + 1, dtype))
    at = torch.tensor(pos, device=CUDA)[:, None]
    o = q4_attend_(q, k, v, at, ring)
    assert o.shape == q.shape and o.dtype == dtype
    k2, v2, held = q4_read(ring, at, torch.float32)
    assert torch.equal(held.cpu(), torch.tensor(pos)[:, None] >= 0)
    for i, p in enumerate(pos):
        if p >= 0:
            assert torch.equal(k2[i].cpu(), _stored(k[i])[0]) and torch.equal(v2[i].cpu(), _stored(v[i])[0])
    want = _attend_want(ring, q, at)
    for i in range(b):
        assert rel(o[i].double().cpu().numpy(), want[i].numpy()) < TOL[dtype], (i, pos[i])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk", [16, 32, 48, 64, 80, 96, 112, 128])
def test_attention_over_every_head_size(dk: int, dtype: torch.dtype) -> None:
    held = [0, 1, 63, 64, 65, 200, 333, 1000]
    ring = _filled(len(held), 2, dk, 200, held, dk, dtype)
    _check_attend(ring, 8, held, dk + 1, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("h", "hkv"), [(1, 1), (2, 1), (3, 3), (6, 2), (5, 1), (7, 1), (8, 1), (9, 1), (16, 1), (24, 2), (40, 8)])
def test_attention_over_every_head_layout(h: int, hkv: int, dtype: torch.dtype) -> None:
    held = [10, 500, 517]
    ring = _filled(3, hkv, 64, 512, held, h, dtype)
    _check_attend(ring, h, held, h + 1, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 127, 512, 1000, 4097, 20000])
def test_attention_over_short_and_long_windows(window: int, dtype: torch.dtype) -> None:
    held = [0, window // 2, window - 1, window, window + 1, 2 * window + window // 3, 7 * window]
    ring = _filled(len(held), 2, 64, window, held, window, dtype)
    _check_attend(ring, 4, held, window + 1, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_run_of_steps_wraps_the_ring(dtype: torch.dtype) -> None:
    ring = _filled(2, 1, 32, 70, [60, 3], 30, dtype)
    for i in range(150):
        _check_attend(ring, 4, [60 + i, 3 + i], 100 + 2 * i, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_only_positions_in_the_window_are_seen(dtype: torch.dtype) -> None:
    """Jumps leave old positions in the ring, and a token before others does not see them."""
    held = [300, 300, 300, 300, 300]
    ring = _filled(5, 2, 64, 256, held, 40, dtype)
    _check_attend(ring, 4, [300, 400, 555, 100000, 150], 41, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_a_masked_slot_holds_does_not_matter(dtype: torch.dtype) -> None:
    """NaN, infinities and garbage codes in slots outside the window or never written change nothing."""
    b, hkv, dk, window = 3, 2, 64, 200
    clean = _filled(b, hkv, dk, window, [50, 120, 200], 50, dtype)
    dirty = Q4RingKVCache(*(getattr(clean, n).clone() for n in ("k_codes", "k_params", "v_codes", "v_params", "pos")), window)
    unseen = clean.pos < 0
    for name in ("k_params", "v_params"):
        p = getattr(dirty, name)
        p.masked_fill_(unseen[:, None, :, None, None], math.nan)
        p[:, :, ::3].masked_fill_(unseen[:, None, ::3, None, None], -math.inf)
    for name in ("k_codes", "v_codes"):
        getattr(dirty, name).masked_fill_(unseen[:, None, :, None], 255)
    g = torch.Generator().manual_seed(51)
    q = torch.randn(b, 1, 8, dk, generator=g).to(dtype).to(CUDA)
    k, v = (t.to(CUDA) for t in _tokens(b, 1, hkv, dk, 52, dtype))
    pos = torch.tensor([[50], [120], [-5]], device=CUDA)
    o1, o2 = q4_attend_(q, k, v, pos, clean), q4_attend_(q, k, v, pos, dirty)
    assert torch.equal(o1, o2) and bool(torch.isfinite(o1).all())
    assert not bool(o1[2].any()) and torch.equal(dirty.pos, clean.pos)  # a negative position: zeros, nothing written


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_nan_that_is_seen_stays_in_its_head(dtype: torch.dtype) -> None:
    ring = _filled(2, 2, 64, 128, [100, 100], 60, dtype)
    k, v = (t.to(CUDA) for t in _tokens(2, 1, 2, 64, 61, dtype))
    q = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(62)).to(dtype).to(CUDA)
    pos = torch.tensor([[100], [100]], device=CUDA)
    v[0, 0, 1, 40] = math.nan
    k[1, 0, 0, 3] = math.inf
    o = q4_attend_(q, k, v, pos, ring)
    bad = torch.isnan(o[:, 0])
    assert bool(bad[0, 2:, 32:].all()) and not bool(bad[0, 2:, :32].any()) and not bool(bad[0, :2].any())
    assert bool(bad[1, :2].all()) and not bool(bad[1, 2:].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sharp_and_large_scores(dtype: torch.dtype) -> None:
    """Queries 30 times larger (one key takes almost all the weight), and values far apart in size."""
    ring = _filled(3, 2, 128, 300, [299, 600, 30], 70, dtype)
    _check_attend(ring, 8, [299, 600, 30], 71, dtype, scale=4.0)
    big = _filled(2, 1, 64, 100, [99, 99], 72, dtype)
    big.v_params[:, :, ::7] *= 512
    _check_attend(big, 4, [99, 99], 73, dtype)
    tiny = _filled(2, 1, 64, 100, [99, 99], 74, dtype)
    _check_attend(tiny, 4, [99, 99], 75, dtype, scale=1e-6)
    zero = _filled(2, 1, 64, 100, [99, 99], 76, dtype)
    _check_attend(zero, 4, [99, 99], 77, dtype, scale=0.0)


@pytest.mark.parametrize(("dk", "window"), [(64, 512), (128, 5000), (80, 3001)])
def test_an_f16_output_is_off_by_little_more_than_its_own_rounding(dk: int, window: int) -> None:
    """Rounding to f16 costs 2^-11 / sqrt(6) = 2.0e-4 of the norm (uniform errors, uniform mantissas); the float32 sums
    and products in 22 bits leave room for half as much again."""
    b, h, hkv = 3, 8, 2
    ring = _filled(b, hkv, dk, window, [window] * b, 65, torch.float16)
    q = torch.randn(b, 1, h, dk, generator=torch.Generator().manual_seed(66)).half().to(CUDA)
    k, v = (t.to(CUDA) for t in _tokens(b, 1, hkv, dk, 67, torch.float16))
    pos = torch.full((b, 1), window, device=CUDA)
    o = q4_attend_(q, k, v, pos, ring)
    assert rel(o.double().cpu().numpy(), _attend_want(ring, q, pos).numpy()) < 3e-4


@pytest.mark.parametrize("size", [2.0**-20, 1.0, 2.0**40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tiles_of_constant_values_among_large_ones(dtype: torch.dtype, size: float) -> None:
    """Whole tiles of zeros (no step at all) before, between and after others: they take their weight's part."""
    b, hkv, dk, window = 2, 1, 64, 1200
    k, v = _tokens(b, window, hkv, dk, 78, dtype)
    v = v * size
    v[:, :70] = 0
    v[:, 500:800] = 0
    v[:, 1100:] = 0
    pos = _positions([0, 0], window).to(CUDA)
    ring = q4_write_(q4_ring_empty(b, hkv, dk, window, CUDA), k.to(CUDA), v.to(CUDA), pos)
    _check_attend(ring, 4, [window - 1, window + 5], 79, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [2.0**12, 2.0**24, 2.0**60])
def test_large_values_of_no_weight_do_not_touch_the_others(dtype: torch.dtype, size: float) -> None:
    """Every 40th token has values ``size`` times larger and a key that no query attends (weights below e^-130)."""
    b, hkv, h, dk, window = 2, 1, 4, 64, 700
    g = torch.Generator().manual_seed(68)
    k, v = _tokens(b, window, hkv, dk, 69, dtype)
    u = torch.nn.functional.normalize(torch.randn(dk, generator=g), dim=0)
    v[:, 7::40] = v[:, 7::40] * size
    k[:, 7::40] = (-60 * u).to(dtype)
    ring = q4_write_(q4_ring_empty(b, hkv, dk, window, CUDA), k.to(CUDA), v.to(CUDA), _positions([0, 0], window).to(CUDA))
    q = (20 * u + torch.randn(b, 1, h, dk, generator=g)).to(dtype).to(CUDA)
    t, w = (x.to(CUDA) for x in _tokens(b, 1, hkv, dk, 70, dtype))
    pos = torch.full((b, 1), window, device=CUDA)
    o = q4_attend_(q, t, w, pos, ring)
    assert rel(o.double().cpu().numpy(), _attend_want(ring, q, pos).numpy()) < TOL[dtype]


def test_strided_tokens_and_streams() -> None:
    b, h, hkv, dk = 4, 8, 2, 64
    ring1, ring2 = (_filled(b, hkv, dk, 96, [95, 96, 97, 10], 80, torch.bfloat16) for _ in range(2))
    qkv = torch.randn(b, 1, (h + 2 * hkv) * dk, generator=torch.Generator().manual_seed(81)).bfloat16().to(CUDA)
    q, k, v = (t.unflatten(-1, (-1, dk)) for t in qkv.split([h * dk, hkv * dk, hkv * dk], -1))
    pos = torch.tensor([[95], [96], [97], [10]], device=CUDA)
    o1 = q4_attend_(q, k, v, pos, ring1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2 = q4_attend_(q.contiguous(), k.contiguous(), v.contiguous(), pos, ring2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o1, o2)
    for name in ("k_codes", "k_params", "v_codes", "v_params", "pos"):
        assert torch.equal(getattr(ring1, name), getattr(ring2, name))
    for _ in range(3):  # the same bits every time
        assert torch.equal(q4_attend_(q, k, v, pos, ring1), o1)


def test_steps_in_a_graph() -> None:
    b, h, hkv, dk, window = 2, 4, 2, 64, 100
    ring, eager = (_filled(b, hkv, dk, window, [90, 5], 90, torch.bfloat16) for _ in range(2))
    q, k, v = (torch.zeros(b, 1, x, dk, dtype=torch.bfloat16, device=CUDA) for x in (h, hkv, hkv))
    pos = torch.tensor([[90], [5]], device=CUDA)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = q4_attend_(q, k, v, pos, ring)
    for i in range(30):
        g = torch.Generator().manual_seed(i)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        assert torch.equal(out, q4_attend_(q, k, v, pos, eager))
        pos.add_(1)
    assert torch.equal(ring.pos, eager.pos)


def test_a_ring_without_key_heads_is_refused() -> None:
    ring = q4_ring_empty(2, 0, 64, 64, CUDA)
    q, kv = torch.zeros(2, 1, 4, 64, device=CUDA), torch.zeros(2, 1, 0, 64, device=CUDA)
    with pytest.raises(ContractError, match="key heads"):
        q4_attend_(q, kv, kv, torch.zeros(2, 1, dtype=torch.long, device=CUDA), ring)


def test_empty_batches_and_chunks() -> None:
    none = q4_ring_empty(0, 2, 64, 10, CUDA)
    e = torch.zeros(0, 1, 2, 64, device=CUDA)
    at = torch.zeros(0, 1, dtype=torch.long, device=CUDA)
    assert q4_attend_(e, e, e, at, none).shape == (0, 1, 2, 64)
    ring = q4_ring_empty(1, 2, 64, 10, CUDA)
    q4_write_(ring, torch.zeros(1, 0, 2, 64, device=CUDA), torch.zeros(1, 0, 2, 64, device=CUDA), torch.zeros(1, 0, dtype=torch.long, device=CUDA))
    assert not bool((ring.pos >= 0).any())
    k, v, held = q4_read(ring, torch.tensor([[0, -1, 5, 1 << 40]], device=CUDA), torch.float32)
    assert not bool(held.any()) and not bool(k.any()) and not bool(v.any())


def test_refusals() -> None:
    ring = q4_ring_empty(2, 2, 64, 10, CUDA)
    q, k = torch.zeros(2, 1, 4, 64, device=CUDA), torch.zeros(2, 1, 2, 64, device=CUDA)
    pos = torch.zeros(2, 1, dtype=torch.long, device=CUDA)
    with pytest.raises(ContractError, match="multiple of 16"):
        q4_ring_empty(2, 2, 40, 10, CUDA)
    with pytest.raises(ContractError, match="multiple of 16"):
        q4_ring_empty(2, 2, 144, 10, CUDA)
    with pytest.raises(ValueError, match="at least 1"):
        q4_ring_empty(2, 2, 64, 0, CUDA)
    with pytest.raises(ContractError, match="not a multiple of 2 key heads"):
        q4_attend_(q[:, :, :3], k, k, pos, ring)
    with pytest.raises(ContractError, match="one token per row"):
        q4_attend_(q, k.expand(2, 2, 2, 64).transpose(1, 2), k.expand(2, 2, 2, 64), pos.expand(2, 2), ring)
    with pytest.raises(ContractError, match="one dtype"):
        q4_attend_(q, k, k.bfloat16(), pos, ring)
    with pytest.raises(ContractError, match=r"\(q's\)"):
        q4_attend_(q.bfloat16(), k, k, pos, ring)
    with pytest.raises(ContractError, match="dtype must be torch.int64"):
        q4_write_(ring, k, k, pos.int())
    with pytest.raises(ContractError, match="axis"):
        q4_write_(ring, k[..., :32], k[..., :32], pos)
    with pytest.raises(ContractError, match="on cpu"):
        q4_write_(ring, k.cpu(), k, pos)
    with pytest.raises(ContractError, match="no gradient"):
        q4_write_(ring, k.clone().requires_grad_(), k, pos)
    bent = Q4RingKVCache(ring.k_codes.transpose(0, 1), ring.k_params, ring.v_codes, ring.v_params, ring.pos, 10)
    with pytest.raises(ContractError, match="contiguous"):
        q4_write_(bent, k, k, pos)
    small = Q4RingKVCache(ring.k_codes, ring.k_params, ring.v_codes, ring.v_params, ring.pos, 65)
    with pytest.raises(ContractError, match="holding the window"):
        q4_read(small, pos)
    with pytest.raises(ContractError, match="dtype: must be"):
        q4_read(ring, pos, torch.float64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_past_32_bits(dtype: torch.dtype) -> None:
    """A ring of 5 GB of key codes, its few tokens in the last head of the last row and across the ring's end."""
    b, hkv, dk, window = 2, 8, 128, 5_000_000
    ring = q4_ring_empty(b, hkv, dk, window, CUDA)
    assert ring.k_codes.numel() > 2**32
    n, last = 300, 2 * window + 100  # positions last - 299 .. last: slots window - 199 .. window - 1, 0 .. 100
    k, v = _tokens(b, n, hkv, dk, 95, dtype)
    pos = _positions([last - n + 1] * b, n)
    q4_write_(ring, k.to(CUDA), v.to(CUDA), pos.to(CUDA))
    k2, v2, held = q4_read(ring, pos.to(CUDA), torch.float32)
    assert bool(held.all()) and torch.equal(k2.cpu(), _stored(k)[0]) and torch.equal(v2.cpu(), _stored(v)[0])
    g = torch.Generator().manual_seed(96)
    q = torch.randn(b, 1, 16, dk, generator=g).to(dtype).to(CUDA)
    k1, v1 = (t.to(CUDA) for t in _tokens(b, 1, hkv, dk, 97, dtype))
    at = torch.full((b, 1), last + 1, device=CUDA)
    o = q4_attend_(q, k1, v1, at, ring)
    all_k = torch.cat([_stored(k)[0], _stored(k1)[0]], 1).double()
    all_v = torch.cat([_stored(v)[0], _stored(v1)[0]], 1).double()
    qs = q[:, 0].double().cpu().view(b, hkv, 2, dk)
    w = torch.softmax(torch.einsum("bhgd,blhd->bhgl", qs, all_k) / math.sqrt(dk), -1)
    want = torch.einsum("bhgl,blhd->bhgd", w, all_v).reshape(b, 1, 16, dk)
    for i in range(b):
        assert rel(o[i].double().cpu().numpy(), want[i].numpy()) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows_of_uneven_lengths_share_the_work(dtype: torch.dtype) -> None:
    """More rows than a warp has lanes, lengths from none to the window, and rows that attend nothing."""
    b, hkv, window = 75, 2, 3000
    held = [(i * 977) % 3100 for i in range(b)]
    ring = _filled(b, hkv, 64, window, held, 98, dtype)
    pos = [-1 if i % 11 == 5 else x for i, x in enumerate(held)]
    _check_attend(ring, 4, pos, 99, dtype)
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(b, 1, 4, 64, generator=g).to(dtype).to(CUDA), torch.randn(b, 1, hkv, 64, generator=g).to(dtype).to(CUDA)
    none = torch.full((b, 1), -1, device=CUDA)
    assert not bool(q4_attend_(q, k, k, none, ring).any())  # nothing to share at all
