"""8-bit rows and the int8 product (``vesper_b200.kernels.q8``) on a B200 against 64-bit arithmetic.

Tolerances, derived before the first run:

- codes of plain and squared-ReLU rows are float32 arithmetic without sums (a maximum, one quotient, one
  product, a rounding), so they and the scales equal the same float32 steps on the CPU, bit for bit;
- a norm's scale carries a float32 sum of up to 20000 squares, spread over at least 32 partial sums: fewer
  than 700 additions in a row, each within 2^-24, errors of both signs: 4e-6 relative. A code is the nearest one of
  a quotient formed with a few roundings of 2^-24: |y - code * scale| <= scale * (1/2 + 127 * 8e-6);
- the product: the int32 sum is exact; its conversion and two products round three times, 3 * 2^-24,
  and the result once more to its type (unit roundoff 2^-8 for bf16, 2^-11 for f16).
"""

from __future__ import annotations

import math

import pytest
import torch

from vesper_b200 import _lib
from vesper_b200.contracts import ContractError
from vesper_b200.kernels.norm import add_rms_norm, fused_rms_norm
from vesper_b200.kernels.q8 import (
    add_rms_norm_q8,
    dequantize_rows_q8,
    linear_q8,
    quantize_rows_q8,
    rms_norm_q8,
)

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
FLOOR, EPS = 1e-3, 1e-6
ROUNDOFF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _rows(n: int, width: int, seed: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, width, generator=g) * torch.exp(0.7 * torch.randn(width, generator=g))).to(dtype)


def _want_rows(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of float32 rows on the CPU, in float32 steps."""
    amax = y.abs().amax(-1, keepdim=True)
    live = torch.isfinite(amax) & (amax >= 1e-35)
    most = torch.full_like(amax, 127.0)
    codes = torch.where(live, torch.round(y * (most / amax)), 0.0).to(torch.int8)
    scale = torch.where(live, amax / most, torch.where(torch.isfinite(amax), 0.0, math.nan))
    return codes, scale[..., 0]


def _norm64(s: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    s = s.double()
    return s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * w.double()


def _assert_codes(q: torch.Tensor, scale: torch.Tensor, y: torch.Tensor) -> None:
    want = y.abs().amax(-1) / 127
    got = scale.double().cpu()
    assert bool(((got - want).abs() <= 4e-6 * want).all()), float(((got - want).abs() / want).max())
    off = (q.cpu().double() * want[..., None] - y).abs()
    assert bool((off <= want[..., None] * (0.5 + 127 * 8e-6)).all()), float((off / want[..., None]).max())
    assert int(q.cpu().abs().amax()) == 127


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (64, 512), (7, 1000), (5, 1031), (130, 2048), (9, 5000), (3, 20000)])
def test_the_norm_in_8_bits(shape: tuple[int, int], dtype: torch.dtype) -> None:
    n, width = shape
    x = _rows(n, width, 1, dtype)
    w = 1 + 0.2 * _rows(1, width, 2)[0]
    q, scale = rms_norm_q8(x.to(CUDA), w.to(CUDA), FLOOR, EPS)
    assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == (n,)
    _assert_codes(q, scale, _norm64(x, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 4), (2, 3, 516), (64, 512), (33, 1003), (257, 1024), (6, 5000), (2, 9001), (2, 16400)])
def test_the_residual_add_and_the_norm_in_8_bits(shape: tuple[int, ...], dtype: torch.dtype) -> None:
    width = shape[-1]
    x = _rows(math.prod(shape[:-1]), width, 3).view(shape)
    r = _rows(math.prod(shape[:-1]), width, 4, dtype).view(shape)
    w = 1 + 0.2 * _rows(1, width, 5)[0]
    s, q, scale = add_rms_norm_q8(x.to(CUDA), r.to(CUDA), w.to(CUDA), FLOOR, EPS)
    total = x + r.float()
    assert torch.equal(s.cpu(), total)
    _assert_codes(q, scale, _norm64(total, w))


def test_the_norm_in_8_bits_is_the_framework_norm() -> None:
    """Against the float norm's own kernel on the same rows: half a step plus both norms' rounding."""
    x, r, w = _rows(100, 512, 6).to(CUDA), _rows(100, 512, 7, torch.bfloat16).to(CUDA), _rows(1, 512, 8)[0].to(CUDA)
    s, q, scale = add_rms_norm_q8(x, r, w, FLOOR, EPS)
    s2, y = add_rms_norm(x, r, w, FLOOR, EPS)
    assert torch.equal(s, s2)
    off = (dequantize_rows_q8(q, scale) - y).abs()
    assert bool((off <= scale[:, None] * (0.5 + 2e-3)).all())
    q1, s1 = rms_norm_q8(s, w, FLOOR, EPS)
    assert torch.equal(q1, q) and torch.equal(s1, scale)
    off = (dequantize_rows_q8(q1, s1) - fused_rms_norm(s, w, FLOOR, EPS)).abs()
    assert bool((off <= scale[:, None] * (0.5 + 2e-3)).all())


@pytest.mark.parametrize("width", [8, 512, 1003, 5000, 20000])
def test_rows_of_extreme_values(width: int) -> None:
    x = _rows(8, width, 9)
    x[1] = 0
    x[2] *= 1e30  # squares overflow float32: the norm is scale-safe
    x[3] *= 1e-30  # below the norm's floor: eps decides
    x[4, width // 2] = math.inf
    x[5, 1] = math.nan
    x[6] = 0
    x[6, width - 1] = -7.0
    w = 1 + 0.2 * _rows(1, width, 10)[0]
    q, scale = rms_norm_q8(x.to(CUDA), w.to(CUDA), FLOOR, EPS)
    assert bool(torch.isnan(scale[4:6]).all()) and not bool(q[4:6].any())
    assert bool(torch.isnan(dequantize_rows_q8(q, scale)[4:6]).all())
    assert float(scale[1]) == 0 and not bool(q[1].any())
    fine = [0, 2, 3, 6, 7]
    y = _norm64(x[fine], w)
    _assert_codes(q[fine], scale[fine], y)
    assert int(q[6, -1].abs()) == 127 and int(q[6].abs().sum()) == 127


@pytest.mark.parametrize("width", [96, 4096, 5001])
def test_norm_weights_at_the_ends_of_float32(width: int) -> None:
    """Rows of one spike, whose norm is sqrt(width) times the weight there: no infinite factor and no infinite scale."""
    x = torch.zeros(5, width)
    x[:, 3] = torch.tensor([2.0, -2.0, 5.0, 1.0, 3.0])
    for gain, zero, bad in ((1e-36, True, False), (1e-30, False, False), (2e38, False, True)):
        q, scale = rms_norm_q8(x.to(CUDA), torch.full((width,), gain, device=CUDA), FLOOR, EPS)
        if bad:  # the norm itself is infinite
            assert bool(torch.isnan(scale).all()) and not bool(q.any())
            continue
        spike = x[:, 3].double().abs()
        want = spike / torch.sqrt(spike.square() / width + EPS) * gain / 127
        assert torch.equal(q[:, 3].cpu(), torch.tensor([0, 0, 0, 0, 0] if zero else [127, -127, 127, 127, 127], dtype=torch.int8))
        assert bool((scale == 0).all() if zero else ((scale.cpu().double() - want).abs() <= 4e-6 * want).all())


@pytest.mark.parametrize("relu_square", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (64, 1536), (5, 17), (3, 4, 100), (40, 4097), (3, 20000)])
def test_plain_and_squared_relu_rows(shape: tuple[int, ...], dtype: torch.dtype, relu_square: bool) -> None:
    x = _rows(math.prod(shape[:-1]), shape[-1], 11, dtype).view(shape)
    q, scale = quantize_rows_q8(x.to(CUDA), relu_square=relu_square)
    y = torch.relu(x.float()).square() if relu_square else x.float()
    want, want_scale = _want_rows(y)
    assert torch.equal(q.cpu(), want) and torch.equal(scale.cpu(), want_scale)


def test_rows_that_are_zero_tiny_or_not_finite() -> None:
    x = _rows(8, 300, 12)
    x[0] = 0
    x[1] *= 1e-37 / x[1].abs().max()
    x[2, 7], x[3, 299], x[4, 0] = math.nan, -math.inf, math.inf
    x[5] = -x[5].abs()
    q, scale = quantize_rows_q8(x.to(CUDA))
    want, want_scale = _want_rows(x)
    assert torch.equal(q.cpu(), want)
    assert torch.equal(torch.isnan(scale.cpu()), torch.isnan(want_scale))
    assert torch.equal(scale.cpu().nan_to_num(), want_scale.nan_to_num()) and float(scale[1]) == 0
    q, scale = quantize_rows_q8(x.to(CUDA), relu_square=True)
    assert float(scale[5]) == 0 and not bool(q[5].any())  # nothing positive
    assert float(scale[3]) > 0  # relu drops -inf
    assert bool(torch.isnan(scale[[2, 4]]).all())


def test_slices_and_other_orders() -> None:
    x = _rows(40, 600, 13).to(CUDA)
    for part in (x[:, 100:356], x[::3, 1:90], x.t()[5:9], x[:, ::2], x[3], x[2:3, 7:99]):
        q, scale = quantize_rows_q8(part)
        want, want_scale = _want_rows(part.cpu())
        assert torch.equal(q.cpu(), want) and torch.equal(scale.cpu(), want_scale)
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            back = dequantize_rows_q8(q, scale, dtype)
            assert torch.equal(back.cpu(), (want.float() * want_scale[..., None]).to(dtype))
    back = dequantize_rows_q8(q.expand(5, *q.shape), scale.expand(5, *scale.shape))
    assert back.shape == (5, *q.shape)


def _operands(m: int, n: int, k: int, seed: int) -> tuple[torch.Tensor, ...]:
    g = torch.Generator().manual_seed(seed)
    xq = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    wq = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    return xq, torch.rand(m, generator=g) * 0.1 + 1e-3, wq, torch.rand(n, generator=g) * 0.1 + 1e-3


def _assert_product(y: torch.Tensor, xq, xs, wq, ws) -> None:
    want = (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()
    bound = want.abs() * (3 * 2.0**-24 + ROUNDOFF[y.dtype] * (y.dtype != torch.float32))
    if y.dtype == torch.float16:
        bound = bound + 2.0**-25  # subnormals
    off = (y.double().cpu() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize(
    ("m", "n", "k"),
    [(1, 1, 1), (1, 16, 32), (1, 1544, 512), (2, 8, 16), (7, 130, 48), (16, 128, 128), (17, 129, 144), (33, 300, 272),
     (64, 512, 1536), (64, 1544, 512), (65, 96, 4096), (100, 1000, 1000), (127, 255, 129), (128, 256, 256),
     (129, 257, 640), (200, 2001, 1040), (300, 64, 64), (257, 513, 8), (512, 512, 2048), (1000, 777, 130),
     (1300, 4100, 1040), (2200, 1290, 520), (700, 4160, 2304)],
)  # fmt: skip
def test_the_product(m: int, n: int, k: int, dtype: torch.dtype) -> None:
    xq, xs, wq, ws = _operands(m, n, k, 14)
    y = linear_q8(xq.to(CUDA), xs.to(CUDA), wq.to(CUDA), ws.to(CUDA), dtype)
    _lib.check_status(CUDA)
    assert y.shape == (m, n) and y.dtype == dtype
    _assert_product(y, xq, xs, wq, ws)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_sums_at_the_edge_of_int32(m: int) -> None:
    """Every product 127 * 127 or -128 * 127 with the longest inner dimension: sums of 2.1e9."""
    k = 131056
    for a, b in ((127, 127), (-128, 127), (-128, -128)):
        xq = torch.full((m, k), a, dtype=torch.int8, device=CUDA)
        wq = torch.full((130, k), b, dtype=torch.int8, device=CUDA)
        ones = torch.ones(130, device=CUDA)
        y = linear_q8(xq, torch.ones(m, device=CUDA), wq, ones, torch.float32)
        assert bool((y.double() == float(torch.tensor(float(a * b * k), dtype=torch.float32))).all())
    _lib.check_status(CUDA)


@pytest.mark.parametrize("m", [3, 70, 260])
def test_the_product_of_padded_sliced_and_unaligned_operands(m: int) -> None:
    xq, xs, wq, ws = _operands(m, 200, 256, 15)
    wide_x, wide_w = torch.zeros(m, 320, dtype=torch.int8), torch.zeros(200, 336, dtype=torch.int8)
    for at in (0, 16, 3):
        wide_x[:, at : at + 256], wide_w[:, at : at + 256] = xq, wq
        y = linear_q8(wide_x.to(CUDA)[:, at : at + 256], xs.to(CUDA), wide_w.to(CUDA)[:, at : at + 256], ws.to(CUDA), torch.float32)
        _assert_product(y, xq, xs, wq, ws)
    y = linear_q8(xq.t().contiguous().to(CUDA).t(), xs.to(CUDA), wq.to(CUDA), ws.to(CUDA), torch.float32)
    _assert_product(y, xq, xs, wq, ws)
    x3 = xq.to(CUDA).view(1, m, 256).expand(2, m, 256)
    y = linear_q8(x3, xs.to(CUDA).expand(2, m), wq.to(CUDA), ws.to(CUDA))
    assert y.shape == (2, m, 200) and torch.equal(y[0], y[1])
    _lib.check_status(CUDA)


def test_a_nan_scale_reaches_its_row_only() -> None:
    xq, xs, wq, ws = _operands(70, 130, 64, 16)
    xs[3], ws[5] = math.nan, math.inf
    y = linear_q8(xq.to(CUDA), xs.to(CUDA), wq.to(CUDA), ws.to(CUDA)).cpu()
    assert bool(torch.isnan(y[3]).all())
    assert not bool(torch.isfinite(y[:, 5]).any())
    rest = torch.isfinite(y)
    rest[3], rest[:, 5] = True, True
    assert bool(rest.all())


def test_the_chain_on_another_stream_and_in_a_graph() -> None:
    """Norm, product, squared ReLU and product as a captured step runs them, replayed on new inputs."""
    w1, s1 = quantize_rows_q8(_rows(1536, 512, 17).to(CUDA))
    w2, s2 = quantize_rows_q8(_rows(512, 1536, 18).to(CUDA))
    x, r = torch.empty(64, 512, device=CUDA), torch.empty(64, 512, device=CUDA, dtype=torch.bfloat16)
    gain = torch.ones(512, device=CUDA)

    def step() -> torch.Tensor:
        s, q, scale = add_rms_norm_q8(x, r, gain, FLOOR, EPS)
        h, hs = quantize_rows_q8(linear_q8(q, scale, w1, s1), relu_square=True)
        return s + linear_q8(h, hs, w2, s2)

    def load(seed: int) -> None:
        x.copy_(_rows(64, 512, seed))
        r.copy_(_rows(64, 512, seed + 1))

    load(19)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    assert torch.equal(out, first)
    load(21)
    graph.replay()
    assert torch.equal(out, step()) and not torch.equal(out, first)
    _lib.check_status(CUDA)


def test_empty_batches() -> None:
    none = torch.zeros(0, 64, device=CUDA)
    w = torch.ones(64, device=CUDA)
    q, scale = rms_norm_q8(none, w, FLOOR, EPS)
    assert q.shape == (0, 64) and scale.shape == (0,)
    s, q, scale = add_rms_norm_q8(none, none, w, FLOOR, EPS)
    assert s.shape == (0, 64)
    q, scale = quantize_rows_q8(none)
    wq, ws = quantize_rows_q8(torch.ones(8, 64, device=CUDA))
    assert linear_q8(q, scale, wq, ws).shape == (0, 8)
    assert dequantize_rows_q8(q, scale).shape == (0, 64)


def test_refusals() -> None:
    x, w = torch.ones(4, 64, device=CUDA), torch.ones(64, device=CUDA)
    q, scale = quantize_rows_q8(x)
    with pytest.raises(ContractError, match="expected shape"):
        rms_norm_q8(x, torch.ones(63, device=CUDA), FLOOR, EPS)
    with pytest.raises(ContractError, match="dtype must be"):
        rms_norm_q8(x.double(), w, FLOOR, EPS)
    with pytest.raises(ContractError, match="residual stream"):
        add_rms_norm_q8(x.bfloat16(), x, w, FLOOR, EPS)
    with pytest.raises(ContractError, match="expected shape"):
        add_rms_norm_q8(x, x[:2], w, FLOOR, EPS)
    with pytest.raises(ContractError, match="no gradient"):
        quantize_rows_q8(x.clone().requires_grad_())
    with pytest.raises(ContractError, match="at least one channel"):
        quantize_rows_q8(x[:, :0])
    with pytest.raises(ContractError, match="expected int8 rows"):
        linear_q8(q[:, :32], scale, q, scale)
    with pytest.raises(ContractError, match="one float32 scale per row"):
        linear_q8(q, scale[:2], q, scale)
    with pytest.raises(ContractError, match="out_dtype"):
        linear_q8(q, scale, q, scale, torch.float64)
    with pytest.raises(ContractError, match="131056"):
        big = torch.zeros(1, 131072, dtype=torch.int8, device=CUDA)
        linear_q8(big, scale[:1], big, scale[:1])
    with pytest.raises(ContractError, match="on cpu"):
        linear_q8(q, scale.cpu(), q, scale)
    with pytest.raises(ContractError, match="dtypes must be"):
        dequantize_rows_q8(q.float(), scale)
