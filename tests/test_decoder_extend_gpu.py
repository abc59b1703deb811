"""``BatchedDecoder`` at fewer passes than its model has, on a B200: ``extend`` carries on the passes that run.

Tolerances, derived before the first run: with float rings ``extend`` is the chunked forward cut at another place, 1e-4 in
float32; with 4-bit rings the windows' keys and values are off by 8 % of a group's spread, on one of three sublayers of
similar size: 25 % tells that apart from a wrong continuation, whose error is over 100 %.
"""

from __future__ import annotations

import pytest
import torch

from vesper_b200.column import ColumnShape, set_scan
from vesper_b200.contracts import ContractError
from vesper_b200.decode import BatchedDecoder
from vesper_b200.model import Vesper

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
SHAPE = ColumnShape(d=128, heads=4, kv_groups=2, head_dim=32, window=24, rotary_base=10000.0, ffn_mult=2, block=16, key_conv=4)
VOCAB, T_MAX = 96, 3


def _rel(a: torch.Tensor, b: torch.Tensor) -> float:
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("depth", [1, 2, 3])
def test_extend_at_any_depth(depth: int, quantized: bool) -> None:
    """Prefill, steps, extend, steps and extend again, against the whole in one prefill."""
    b = 2
    model = Vesper(SHAPE, VOCAB, 2, T_MAX, 0.01, torch.Generator().manual_seed(21)).to(CUDA)
    set_scan(model, "fused-fp32")
    tokens = torch.randint(0, VOCAB, (b, 100), generator=torch.Generator().manual_seed(22)).to(CUDA)
    dec = BatchedDecoder(model, depth, VOCAB, b, torch.float32, warm=1, quantized=quantized)
    dec.prefill(tokens[:, :20], chunk=8)
    for i in range(20, 30):
        dec.step(tokens[:, i : i + 1])
    tail = dec.extend(tokens[:, 30:90], chunk=16, all_logits=True)
    for i in range(90, 95):
        _, logits = dec.step(tokens[:, i : i + 1])
    last = dec.extend(tokens[:, 95:])
    whole = BatchedDecoder(model, depth, VOCAB, b, torch.float32).prefill(tokens, chunk=32, all_logits=True)
    tol = 0.25 if quantized else 1e-4
    assert _rel(tail, whole[:, 30:90]) < tol
    assert _rel(logits, whole[:, 94:95]) < tol
    assert _rel(last, whole[:, 99:]) < tol
    assert int(dec.position[0, 0]) == 99 and dec.length == 100
    for state in dec.states:  # the passes that do not run hold nothing
        for ring in state.kv[depth:]:
            assert not bool((ring.pos > 0).any())
    dec.release()


def test_extending_nothing_by_nothing_is_refused_by_name() -> None:
    model = Vesper(SHAPE, VOCAB, 1, T_MAX, 0.01, torch.Generator().manual_seed(23)).to(CUDA)
    dec = BatchedDecoder(model, 1, VOCAB, 1)
    with pytest.raises(ContractError, match="at least one token"):
        dec.extend(torch.zeros(1, 0, dtype=torch.long, device=CUDA))
