"""Quantised decoding (``BatchedDecoder(quantized=True)``, ``vesper_b200.quant``) and ``extend`` on a B200.

Tolerances, derived before the first run:

- a quantised step against the same step with every product and the attention written out in float32 torch over the
  values that the codes stand for: the quantisers are the same kernels, so the two differ by float32 rounding of sums
  (1e-6) and, where that moves a value across the middle of a step, by one code: of the 64 to 128 values of a row, each a 127th
  of the largest, a few per thousand elements. 1e-2 of the output's norm covers all of them moving in some rows;
- quantised against float decoding: an 8-bit operand is off by about 0.6 % of a row's spread and a 4-bit key or value by
  8 % of a group's, on one of three sublayers of similar size; four column applications add up to some 10 % of
  the output. 25 % tells that apart from a wrong one, whose error is over 100 %;
- ``extend`` with float rings is the chunked forward cut at another place: 1e-4 in float32.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F  # noqa: N812

from conftest import rel
from vesper_b200 import _lib
from vesper_b200.attention import cache_from_ring, kv_ring_empty, q4_ring_from_cache, ring_from_cache
from vesper_b200.attention import KVCache
from vesper_b200.column import RMS_EPS, RMS_SCALE_FLOOR, ColumnShape, init_column_state, set_scan
from vesper_b200.contracts import ContractError
from vesper_b200.decode import BatchedDecoder
from vesper_b200.kernels.delta_scan import delta_scan_step_
from vesper_b200.kernels.q4_cache import q4_read, q4_write_
from vesper_b200.kernels.q8 import add_rms_norm_q8, dequantize_rows_q8, quantize_rows_q8, rms_norm_q8
from vesper_b200.kernels.rotary import rotary
from vesper_b200.model import Vesper
from vesper_b200.quant import QuantizedColumn, QuantizedVesper

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
SHAPE = ColumnShape(d=128, heads=4, kv_groups=2, head_dim=32, window=24, rotary_base=10000.0, ffn_mult=2, block=16, key_conv=4)
VOCAB, DEPTH = 96, 2


def _model(scan: str) -> Vesper:
    model = Vesper(SHAPE, VOCAB, 2, DEPTH, 0.01, torch.Generator().manual_seed(5)).to(CUDA)
    set_scan(model, scan)
    return model


def _tokens(b: int, n: int, seed: int) -> torch.Tensor:
    return torch.randint(0, VOCAB, (b, n), generator=torch.Generator().manual_seed(seed)).to(CUDA)


def _plain_step(column: QuantizedColumn, x, r, pos, state, t):
    """``QuantizedColumn.step_decode`` with its products and attention in float32 torch."""
    c, dk = column.column, column.column.rec.head_dim
    rec, attn, ring, history, h = c.rec, c.attn, state.kv[t], state.key_history[t], state.h[t]

    def linear(rows, weight):
        return F.linear(dequantize_rows_q8(*rows), dequantize_rows_q8(*weight))

    if r is None:
        rows = rms_norm_q8(x, c.norm_rec.weight, RMS_SCALE_FLOOR, RMS_EPS)
    else:
        x, *rows = add_rms_norm_q8(x, r, c.norm_rec.weight, RMS_SCALE_FLOOR, RMS_EPS)
    d = x.shape[-1]
    q, z, v, logits = linear(rows, column.rec_in).split([d, d, d, rec.heads], -1)
    k, new = rec.keys(z.contiguous(), history)
    history.copy_(new)
    q, v = (y.unflatten(-1, (rec.heads, dk)) for y in (q, v))
    o = delta_scan_step_(q, k, v, logits, h, from_logits=True)
    r = linear(quantize_rows_q8(o.flatten(2)), column.rec_out)
    x, *rows = add_rms_norm_q8(x, r, c.norm_attn.weight, RMS_SCALE_FLOOR, RMS_EPS)
    hd, kv = attn.heads * dk, attn.kv_heads * dk
    q, k, v = (y.unflatten(-1, (-1, dk)) for y in linear(rows, column.attn_in).split([hd, kv, kv], -1))
    q, k = rotary(q, pos, attn.rotary_base), rotary(k, pos, attn.rotary_base)
    q4_write_(ring, k, v, pos)
    at = ring.pos[:, : ring.window]
    kk, vv, held = q4_read(ring, at, torch.float32)
    seen = held & (at <= pos) & (at > pos - ring.window)
    rep = attn.heads // attn.kv_heads
    s = torch.einsum("bhd,blhd->bhl", q[:, 0], kk.repeat_interleave(rep, 2)) / math.sqrt(dk)
    w = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
    a = torch.einsum("bhl,blhd->bhd", w, vv.repeat_interleave(rep, 2))[:, None]
    r = linear(quantize_rows_q8(a.flatten(2)), column.attn_out)
    x, *rows = add_rms_norm_q8(x, r, c.norm_ffn.weight, RMS_SCALE_FLOOR, RMS_EPS)
    hidden = quantize_rows_q8(linear(rows, column.ffn_in), relu_square=True)
    return x, linear(hidden, column.ffn_out)


@torch.no_grad()
def test_a_quantised_column_step_is_its_formula() -> None:
    model = _model("fused-fp32")
    column = QuantizedColumn(model.loop.columns[0], torch.float32)
    b = 5
    ours, plain = (init_column_state(SHAPE, b, 1, torch.float32, CUDA, ring=True, q4=True) for _ in range(2))
    g = torch.Generator().manual_seed(6)
    for i in range(40):  # past the window
        x, r = (torch.randn(b, 1, SHAPE.d, generator=g).to(CUDA) for _ in range(2))
        pos = torch.full((b, 1), i, device=CUDA)
        got = column.step_decode(x, r if i % 3 else None, pos, ours, 0)
        want = _plain_step(column, x, r if i % 3 else None, pos, plain, 0)
        for y, z in zip(got, want, strict=True):
            assert rel(y.cpu().numpy(), z.cpu().numpy()) < 1e-2, i
        # what is carried on starts the next step equal, so that a code's difference does not add up over the steps
        for dst, src in zip((plain.h[0], plain.key_history[0]), (ours.h[0], ours.key_history[0]), strict=True):
            assert rel(dst.cpu().numpy(), src.cpu().numpy()) < 1e-2, i
            dst.copy_(src)
        for name in ("k_codes", "k_params", "v_codes", "v_params", "pos"):
            getattr(plain.kv[0], name).copy_(getattr(ours.kv[0], name))
    _lib.check_status(CUDA)


@pytest.mark.parametrize(("dtype", "scan"), [(torch.float32, "fused-fp32"), (torch.bfloat16, "fused")])
def test_quantised_decoding_follows_float_decoding(dtype: torch.dtype, scan: str) -> None:
    b, prompt, steps = 3, 37, 30
    model = _model(scan)
    tokens = _tokens(b, prompt + steps, 7)
    plain, quant = (BatchedDecoder(model, DEPTH, VOCAB, b, dtype, warm=2, quantized=x) for x in (False, True))
    first = plain.prefill(tokens[:, :prompt], chunk=16)
    assert torch.equal(first, quant.prefill(tokens[:, :prompt], chunk=16))  # prompts run in floats
    want, got = [], []
    for i in range(steps):
        want.append(plain.step(tokens[:, prompt + i : prompt + i + 1])[1].float().clone())
        ids, logits = quant.step(tokens[:, prompt + i : prompt + i + 1])
        assert logits.shape == (b, 1, VOCAB) and torch.equal(ids, logits.argmax(-1))
        got.append(logits.float().clone())
    a, w = torch.cat(got, 1).cpu().numpy(), torch.cat(want, 1).cpu().numpy()
    assert np.isfinite(a).all()
    assert rel(a, w) < 0.25, rel(a, w)
    _lib.check_status(CUDA)
    plain.release()
    quant.release()


def test_the_captured_quantised_step_is_the_eager_one() -> None:
    b, steps = 4, 40
    model = _model("fused")
    tokens = _tokens(b, steps, 8)
    eager, captured = (BatchedDecoder(model, DEPTH, VOCAB, b, torch.bfloat16, warm=w, quantized=True) for w in (steps, 1))
    for i in range(steps):
        _, want = eager.step(tokens[:, i : i + 1])
        _, got = captured.step(tokens[:, i : i + 1])
        assert torch.equal(got, want), i
    captured.release()


@pytest.mark.parametrize("quantized", [False, True])
def test_extend_goes_on_where_the_rings_are(quantized: bool) -> None:
    """Prefill, steps, extend and steps again, against the whole in one prefill (float rings: to float32 rounding)."""
    b = 2
    model = _model("fused-fp32")
    tokens = _tokens(b, 120, 9)
    dec = BatchedDecoder(model, DEPTH, VOCAB, b, torch.float32, warm=1, quantized=quantized)
    dec.prefill(tokens[:, :20], chunk=8)
    for i in range(20, 30):
        dec.step(tokens[:, i : i + 1])
    tail = dec.extend(tokens[:, 30:90], chunk=16, all_logits=True)
    for i in range(90, 95):
        _, logits = dec.step(tokens[:, i : i + 1])
    tail2 = dec.extend(tokens[:, 95:100])
    whole = BatchedDecoder(model, DEPTH, VOCAB, b, torch.float32).prefill(tokens[:, :100], chunk=32, all_logits=True)
    tol = 0.25 if quantized else 1e-4
    assert tail.shape == (b, 60, VOCAB) and tail2.shape == (b, 1, VOCAB)
    assert rel(tail.cpu().numpy(), whole[:, 30:90].cpu().numpy()) < tol
    assert rel(logits.cpu().numpy(), whole[:, 94:95].cpu().numpy()) < tol
    assert rel(tail2.cpu().numpy(), whole[:, 99:].cpu().numpy()) < tol
    assert int(dec.position[0, 0]) == 99 and dec.length == 100
    dec.release()


@pytest.mark.parametrize("m", [0, 1, 15, 24])
def test_rings_and_caches_turn_into_each_other(m: int) -> None:
    g = torch.Generator().manual_seed(10)
    k, v = (torch.randn(2, 24, 2, 32, generator=g).to(CUDA) for _ in range(2))
    pos = torch.arange(100, 124, device=CUDA).expand(2, 24).contiguous()
    cache = KVCache(k=k, v=v, pos=pos, window=24)
    last = pos[:, -1]
    back = cache_from_ring(ring_from_cache(cache), last, m, torch.float32)
    assert torch.equal(back.k, k[:, 24 - m :]) and torch.equal(back.v, v[:, 24 - m :]) and torch.equal(back.pos, pos[:, 24 - m :])
    ring = q4_ring_from_cache(cache)
    back = cache_from_ring(ring, last, m, torch.float32)
    want_k, want_v, _ = q4_read(ring, pos[:, 24 - m :], torch.float32)
    assert torch.equal(back.k, want_k) and torch.equal(back.v, want_v) and back.window == 24


def test_refusals() -> None:
    model = _model("fused")
    with pytest.raises(ContractError, match="carries a Q4RingKVCache"):
        state = init_column_state(SHAPE, 1, 1, torch.bfloat16, CUDA, ring=True)
        x, pos = torch.zeros(1, 1, SHAPE.d, device=CUDA), torch.zeros(1, 1, dtype=torch.long, device=CUDA)
        QuantizedColumn(model.loop.columns[0]).step_decode(x, None, pos, state, 0)
    with pytest.raises(ContractError, match="multiple of 16"):
        shape = ColumnShape(d=64, heads=8, kv_groups=2, head_dim=8, window=8, rotary_base=10000.0, ffn_mult=2, block=16, key_conv=4)
        QuantizedVesper(Vesper(shape, 16, 1, 1, 0.01).to(CUDA))
    with pytest.raises(ContractError, match="runs on CUDA"):
        QuantizedVesper(Vesper(SHAPE, 16, 1, 1, 0.01))
    with pytest.raises(ContractError, match="does not hold every position"):
        cache_from_ring(kv_ring_empty(1, 2, 32, 8, torch.float32, CUDA), torch.zeros(1, dtype=torch.long, device=CUDA), 1, torch.float32)
    with pytest.raises(ValueError, match="m must lie"):
        cache_from_ring(kv_ring_empty(1, 2, 32, 8, torch.float32, CUDA), torch.zeros(1, dtype=torch.long, device=CUDA), 9, torch.float32)
    dec = BatchedDecoder(model, DEPTH, VOCAB, 2, quantized=True)
    with pytest.raises(ContractError, match="prompt of 3 rows"):
        dec.extend(_tokens(3, 4, 11))
    dec.prefill(_tokens(2, 4, 11))
    with pytest.raises(ContractError, match="at least one token"):
        dec.extend(_tokens(2, 0, 11))
