"""What 4-bit ring attention (``q4_attend_``) keeps of 16-bit inputs, on a B200, against 64-bit arithmetic.

Tolerances, derived before the first run:

- rounding an output to f16 costs 2^-11 / sqrt(6) = 2.0e-4 of the norm (uniform errors, uniform mantissas); float32 sums, of
  however many positions, leave room for half as much again: 3e-4;
- a bf16 output is the float32 result rounded once. Float32 arithmetic leaves it within 1e-5 of the outputs' size (as for
  float32 inputs), which moves an output x across a rounding boundary, 2^-8 |x| or more apart, with a probability
  of at most 2 * 1e-5 * 2^8 / |x| (x in units of the outputs' size). Over normally distributed x that is 5e-3 E[min(1 / |x|,
  200)] = 5e-3 * sqrt(2 / pi) * (ln 200 + 0.06) = 2.1 %. So at least 97.5 % of the outputs equal the 64-bit result
  rounded to bf16.
"""

from __future__ import annotations

import pytest
import torch

from vesper_b200.kernels.q4_cache import Q4RingKVCache, q4_attend_, q4_read, q4_ring_empty, q4_write_

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")


def _want(ring: Q4RingKVCache, q: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """A masked softmax in 64 bits over what the ring holds, the token among it."""
    b, _, h, dk = q.shape
    hkv, w = ring.k_codes.shape[1], ring.window
    out = torch.zeros(b, 1, h, dk, dtype=torch.float64, device=CUDA)
    for i in range(b):
        p = int(pos[i])
        if p < 0:
            continue
        one = Q4RingKVCache(*(getattr(ring, n)[i : i + 1] for n in ("k_codes", "k_params", "v_codes", "v_params", "pos")), w)
        at = one.pos[:, :w]
        k, v, held = q4_read(one, at, torch.float32)
        seen = (held & (at <= p) & (at > p - w))[0]
        qi = q[i, 0].double().view(hkv, h // hkv, dk)
        wt = torch.softmax(torch.einsum("hgd,lhd->hgl", qi, k[0, seen].double()) / dk**0.5, -1)
        out[i, 0] = torch.einsum("hgl,lhd->hgd", wt, v[0, seen].double()).reshape(h, dk)
    return out


def _full(b: int, hkv: int, dk: int, window: int, seed: int, dtype: torch.dtype) -> Q4RingKVCache:
    """A ring that holds positions 0 .. window - 1 of normally distributed keys and values."""
    g = torch.Generator(device=CUDA).manual_seed(seed)
    ring = q4_ring_empty(b, hkv, dk, window, CUDA)
    k, v = (torch.randn(b, window, hkv, dk, generator=g, device=CUDA).to(dtype) for _ in range(2))
    return q4_write_(ring, k, v, torch.arange(window, device=CUDA).expand(b, window))


def _step(b: int, h: int, hkv: int, dk: int, pos: list[int], seed: int, dtype: torch.dtype) -> tuple[torch.Tensor, ...]:
    """A token's ``q``, ``k``, ``v`` and position."""
    g = torch.Generator(device=CUDA).manual_seed(seed)
    q, k, v = (torch.randn(b, 1, x, dk, generator=g, device=CUDA).to(dtype) for x in (h, hkv, hkv))
    return q, k, v, torch.tensor(pos, device=CUDA)[:, None]


def _rel(o: torch.Tensor, want: torch.Tensor) -> float:
    return float((o.double() - want).norm() / want.norm())


@pytest.mark.parametrize(("b", "h", "hkv", "dk", "window"), [(64, 2, 1, 16, 65536), (64, 4, 1, 64, 40000), (16, 7, 1, 128, 65536),
                                                           (48, 5, 1, 48, 30000)])  # fmt: skip
def test_long_sums_in_f16_are_float32_sums(b: int, h: int, hkv: int, dk: int, window: int) -> None:
    """Dozens of tiles a warp, every weight of the same order: the outputs are small against the values they average."""
    ring = _full(b, hkv, dk, window, 1, torch.float16)
    q, k, v, pos = _step(b, h, hkv, dk, [window] * b, 2, torch.float16)
    o = q4_attend_(q, k, v, pos, ring)
    assert _rel(o, _want(ring, q, pos)) < 3e-4


@pytest.mark.parametrize(("h", "hkv"), [(8, 2), (16, 2), (3, 1), (9, 1)])
@pytest.mark.parametrize(("dk", "window"), [(64, 512), (128, 5000), (80, 3001), (16, 100)])
def test_a_bf16_output_is_the_float32_result_rounded(dk: int, window: int, h: int, hkv: int) -> None:
    b = 8
    ring = _full(b, hkv, dk, window, 3, torch.bfloat16)
    q, k, v, pos = _step(b, h, hkv, dk, [window] * b, 4, torch.bfloat16)
    o = q4_attend_(q, k, v, pos, ring)
    equal = float((o == _want(ring, q, pos).to(torch.bfloat16)).double().mean())
    assert equal >= 0.975, equal


@pytest.mark.parametrize(("dk", "h"), [(64, 4), (128, 8)])
def test_offsets_of_groups_that_cancel(dk: int, h: int) -> None:
    """Keys whose groups stand far from zero, slot by slot, in amounts that the queries take from one another: parts of some
    2000 in the scores, of which float32 keeps 2^-22 at worst, 5e-4, and the output's rounding 2e-4."""
    b, hkv, window = 4, 1, 700
    g = torch.Generator(device=CUDA).manual_seed(5)
    ring = q4_ring_empty(b, hkv, dk, window, CUDA)
    k, v = (torch.randn(b, window, hkv, dk, generator=g, device=CUDA) for _ in range(2))
    far = 1000 * torch.randn(b, window, hkv, 1, generator=g, device=CUDA)
    k[..., :32] += far
    k[..., 32:64] -= far / 3
    q4_write_(ring, k.half(), v.half(), torch.arange(window, device=CUDA).expand(b, window))
    q, k, v, pos = _step(b, h, hkv, dk, [window] * b, 6, torch.float16)
    q[..., :32] = (0.5 + 0.3 * q[..., :32]).bfloat16()
    q[..., 32:64] = 3 * q[..., :32]
    o = q4_attend_(q, k, v, pos, ring)
    assert _rel(o, _want(ring, q, pos)) < 7e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("dk", "h"), [(64, 4), (128, 8), (16, 1)])
def test_scores_in_the_millions_and_far_beyond(dtype: torch.dtype, dk: int, h: int) -> None:
    """One key takes all the weight, and the output is its value: off by half a step of the output's type at most, 2^-9."""
    b, window = 3, 500
    ring = q4_ring_empty(b, 1, dk, window, CUDA)
    g = torch.Generator(device=CUDA).manual_seed(14)
    k, v = (torch.randn(b, window, 1, dk, generator=g, device=CUDA) for _ in range(2))
    q, k1, v1, pos = _step(b, h, 1, dk, [window] * b, 15, dtype)
    for size in (2.0**8, 2.0**11, 2.0**12) if dtype == torch.float16 else (2.0**10, 2.0**14, 2.0**25, 2.0**50):
        q4_write_(ring, (k * size).to(dtype), v.to(dtype), torch.arange(window, device=CUDA).expand(b, window))
        o = q4_attend_((q * size).to(dtype), (k1 * size).to(dtype), v1, pos, ring)
        assert _rel(o, _want(ring, (q * size).to(dtype), pos)) < 4e-3, size


@pytest.mark.parametrize("dk", [16, 64, 128])
@pytest.mark.parametrize("h", [3, 8])
def test_queries_at_the_upper_end_of_bf16(h: int, dk: int) -> None:
    """Scores that stay finite: tiny keys, or queries of different sizes in one unit. A bf16 output's rounding is 2^-9."""
    b, window = 2, 300
    ring = q4_ring_empty(b, 1, dk, window, CUDA)
    g = torch.Generator(device=CUDA).manual_seed(7)
    k, v = (torch.randn(b, window, 1, dk, generator=g, device=CUDA) for _ in range(2))
    q4_write_(ring, (k * 2.0**-95).bfloat16(), v.bfloat16(), torch.arange(window, device=CUDA).expand(b, window))
    q, k, v, pos = _step(b, h, 1, dk, [window] * b, 8, torch.bfloat16)
    sizes = [2.0**x for x in (95, 125, 103, 104, 105, 117, 118, 0)][:h]
    q = q / q.abs().amax(-1, keepdim=True) * torch.tensor(sizes, device=CUDA, dtype=torch.bfloat16)[:, None]
    k = k * 2.0**-95
    o = q4_attend_(q, k, v, pos, ring)
    assert bool(torch.isfinite(o).all())
    want = _want(ring, q, pos)
    for i in range(h):
        assert _rel(o[:, :, i], want[:, :, i]) < 5e-3, i


def _value_steps(kind: str, b: int, window: int, groups: int) -> torch.Tensor:
    """Powers of two ``[b, slots, groups]`` for the values of a ring's slots."""
    g = torch.Generator(device=CUDA).manual_seed(9)
    x = torch.zeros(b, window, groups, device=CUDA)
    if kind == "one group small":
        x[..., 1:] = -30
    elif kind == "one group large":
        x[..., 0] = 45
    elif kind == "small only later":
        x[:, window // 2 :, 1:] = -30
    elif kind == "small at first":
        x[:, : window // 2, 1:] = -30
    else:
        x = torch.randint(-40, 41, x.shape, generator=g, device=CUDA).float()
    return torch.exp2(x)


@pytest.mark.parametrize("kind", ["one group small", "one group large", "small only later", "small at first", "any sizes"])
@pytest.mark.parametrize(("dk", "h"), [(64, 4), (128, 8), (48, 3), (96, 6), (32, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_groups_of_very_different_size_keep_their_own_values(dtype: torch.dtype, dk: int, h: int, kind: str) -> None:
    """Each group of channels against its own norm, off by the output's rounding (2^-9 in bf16). f16 outputs hold no such
    sizes, so the ring's steps are made, and the outputs compared, where f16 can tell: groups of 2^-10 and less of another."""
    b, window, groups = 3, 1500, dk // (32 if dk % 32 == 0 else 16)
    ring = _full(b, 1, dk, window, 10, dtype)
    size = _value_steps(kind, b, window, groups)
    if dtype == torch.float16:
        size = torch.exp2(torch.log2(size) / 4)
    ring.v_params[:, 0, :window] = (ring.v_params[:, 0, :window].float() * size[..., None]).bfloat16()
    q, k, v, pos = _step(b, h, 1, dk, [window] * b, 11, dtype)
    o = q4_attend_(q, k, v, pos, ring)
    want = _want(ring, q, pos)
    for x, y in zip(o.chunk(groups, -1), want.chunk(groups, -1), strict=True):
        if dtype == torch.bfloat16 or float(y.abs().max()) > 2.0**-10:
            assert _rel(x, y) < 5e-3


def test_a_group_without_steps_before_one_of_small_steps() -> None:
    """Constant values (no step at all) in a group's first slots, small ones later, beside a group of ordinary values."""
    b, window, dk = 2, 1200, 64
    g = torch.Generator(device=CUDA).manual_seed(12)
    k, v = (torch.randn(b, window, 1, dk, generator=g, device=CUDA) for _ in range(2))
    v[..., 32:] *= 2.0**-30
    v[:, :700, :, 32:] = 0
    ring = q4_write_(q4_ring_empty(b, 1, dk, window, CUDA), k.bfloat16(), v.bfloat16(), torch.arange(window, device=CUDA).expand(b, window))
    q, k, v, pos = _step(b, 4, 1, dk, [window] * b, 13, torch.bfloat16)
    v[..., 32:] *= 2.0**-30
    o = q4_attend_(q, k, v, pos, ring)
    want = _want(ring, q, pos)
    for x, y in zip(o.chunk(2, -1), want.chunk(2, -1), strict=True):
        assert _rel(x, y) < 5e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize(("dk", "h"), [(64, 4), (128, 8), (48, 3)])
@pytest.mark.parametrize("kind", ["all large", "constant", "one group constant", "some tokens"])
def test_values_at_the_upper_end_of_float32(kind: str, dk: int, h: int, dtype: torch.dtype) -> None:
    """Outputs of up to 1e37, whole or beside small ones, constant (no step) or not: 1e-5 in float32, 2^-9 in bf16."""
    b, window, size = 2, 900, 16 if dk % 32 else 32
    g = torch.Generator(device=CUDA).manual_seed(16)
    k, v = (torch.randn(b, window, 1, dk, generator=g, device=CUDA) for _ in range(2))
    if kind == "all large":
        v *= 1e37
    elif kind == "constant":
        v = torch.full_like(v, 2.0**120)
    elif kind == "one group constant":
        v[..., :size] = 2.0**120
        v[..., size:] *= 1e-10
    else:
        v[:, 100:150] *= 1e36
        v[:, 400] = -(2.0**122)
    ring = q4_write_(q4_ring_empty(b, 1, dk, window, CUDA), k.to(dtype), v.to(dtype), torch.arange(window, device=CUDA).expand(b, window))
    q, k, v, pos = _step(b, h, 1, dk, [window] * b, 17, dtype)
    v *= 1e-10 if kind == "one group constant" else 1
    o = q4_attend_(q, k, v, pos, ring)
    want = _want(ring, q, pos)
    assert bool(torch.isfinite(o).all())
    for x, y in zip(o.split(size, -1), want.split(size, -1), strict=True):
        assert _rel(x, y) < (1e-5 if dtype == torch.float32 else 5e-3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk", [64, 48, 128])
def test_keys_at_the_upper_end_of_float32(dk: int, dtype: torch.dtype) -> None:
    """Keys of 1e36 and queries that bring them to ordinary scores, or to finite ones of which the largest takes all."""
    b, window = 2, 400
    g = torch.Generator(device=CUDA).manual_seed(18)
    k, v = (torch.randn(b, window, 1, dk, generator=g, device=CUDA) for _ in range(2))
    ring = q4_write_(q4_ring_empty(b, 1, dk, window, CUDA), (k * 2.0**119).to(dtype), v.to(dtype), torch.arange(window, device=CUDA).expand(b, window))
    q, k, v, pos = _step(b, 3, 1, dk, [window] * b, 19, dtype)
    q = q * torch.tensor([2.0**-119, 2.0**-100, 1.0], device=CUDA, dtype=dtype)[:, None]
    o = q4_attend_(q, (k.float() * 2.0**119).to(dtype), v, pos, ring)
    want = _want(ring, q, pos)
    assert bool(torch.isfinite(o).all())
    for i in range(3):
        assert _rel(o[:, :, i], want[:, :, i]) < (1e-5 if dtype == torch.float32 else 5e-3), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("order", ["ordinary first", "far below first", "in turn"])
@pytest.mark.parametrize(("dk", "h"), [(64, 4), (128, 7)])
def test_ordinary_scores_beside_scores_in_the_millions(dk: int, h: int, order: str, dtype: torch.dtype) -> None:
    """Tiles of ordinary keys and of keys 2^30 times as large: of those the one that scores most takes all, or, where they all
    score far below, the ordinary ones share it. Off by the output's rounding, 2^-9, in float32 by 1e-5."""
    b, window = 2, 1500
    g = torch.Generator(device=CUDA).manual_seed(71)
    k, v = (torch.randn(b, window, 1, dk, generator=g, device=CUDA) for _ in range(2))
    q, k1, v1, pos = _step(b, h, 1, dk, [window] * b, 72, dtype)
    if order == "ordinary first":
        k[:, window // 2 :] *= 2.0**30
    elif order == "far below first":
        k[:, : window // 2] = -(2.0**30) * q[:, :, :1].float().mean(2, keepdim=True)
        q = q[:, :, :1].expand(b, 1, h, dk).contiguous()
    else:
        k[:, ::3] *= 2.0**30
    ring = q4_write_(q4_ring_empty(b, 1, dk, window, CUDA), k.to(dtype), v.to(dtype), torch.arange(window, device=CUDA).expand(b, window))
    o = q4_attend_(q, k1, v1, pos, ring)
    assert _rel(o, _want(ring, q, pos)) < (1e-5 if dtype == torch.float32 else 4e-3)
