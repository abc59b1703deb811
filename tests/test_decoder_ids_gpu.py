"""Token ids outside the vocabulary in ``BatchedDecoder.step`` on a B200: an eager step refuses them, a captured one
records them in the status word; neither looks them up. What the word holds after a step is raised by the next call."""

from __future__ import annotations

import pytest
import torch

from vesper_b200 import _lib
from vesper_b200.column import ColumnShape, set_scan
from vesper_b200.contracts import ContractError
from vesper_b200.decode import BatchedDecoder
from vesper_b200.model import Vesper

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
SHAPE = ColumnShape(d=64, heads=2, kv_groups=1, head_dim=32, window=16, rotary_base=10000.0, ffn_mult=2, block=16, key_conv=4)
VOCAB = 50


def _decoder(quantized: bool, warm: int) -> BatchedDecoder:
    model = Vesper(SHAPE, VOCAB, 1, 2, 0.01, torch.Generator().manual_seed(31)).to(CUDA)
    set_scan(model, "fused")
    return BatchedDecoder(model, 2, VOCAB, 2, torch.bfloat16, warm=warm, quantized=quantized)


@pytest.mark.parametrize("bad", [VOCAB, -1, 1 << 40])
@pytest.mark.parametrize("quantized", [False, True])
def test_an_eager_step_refuses_an_id_outside_the_vocabulary(quantized: bool, bad: int) -> None:
    dec = _decoder(quantized, warm=3)
    with pytest.raises(ContractError, match="every id must lie in"):
        dec.step(torch.tensor([[1], [bad]], device=CUDA))


@pytest.mark.parametrize("bad", [VOCAB, -1, 1 << 40])
@pytest.mark.parametrize("quantized", [False, True])
def test_a_captured_step_records_an_id_outside_the_vocabulary(quantized: bool, bad: int) -> None:
    dec = _decoder(quantized, warm=1)
    good = torch.tensor([[1], [2]], device=CUDA)
    for _ in range(3):
        dec.step(good)
    _lib.check_status(CUDA)
    dec.step(torch.tensor([[1], [bad]], device=CUDA))
    with pytest.raises(_lib.KernelError, match="status 4"):
        _lib.check_status(CUDA)
    _, logits = dec.step(good)
    assert bool(torch.isfinite(logits).all())
    _lib.check_status(CUDA)
    dec.release()


@pytest.mark.parametrize("quantized", [False, True])
def test_a_refused_id_takes_no_position(quantized: bool) -> None:
    dec, other = (_decoder(quantized, warm=9) for _ in range(2))
    other.model.load_state_dict(dec.model.state_dict())
    tokens = torch.tensor([[3, 7, 11, 2], [4, 9, 1, 30]], device=CUDA)
    for x in (dec, other):
        x.prefill(tokens[:, :2])
    with pytest.raises(ContractError, match="every id must lie in"):
        dec.step(torch.tensor([[1], [VOCAB]], device=CUDA))
    torch.cuda.synchronize()
    assert torch.equal(dec.position, other.position) and dec.length == other.length
    for i in (2, 3):
        want, got = (x.step(tokens[:, i : i + 1])[1] for x in (other, dec))
        assert torch.equal(got, want)


@pytest.mark.parametrize("warm", [9, 1])
@pytest.mark.parametrize("quantized", [False, True])
def test_a_kernel_that_gave_up_is_raised_by_the_next_call(quantized: bool, warm: int) -> None:
    """The bit is set by hand, as a kernel whose wait ran out sets it."""
    dec = _decoder(quantized, warm)
    good = torch.tensor([[1], [2]], device=CUDA)
    calls = (lambda: dec.step(good), lambda: dec.extend(good), lambda: dec.prefill(good), dec.check)
    for call in calls:
        for _ in range(3):
            dec.step(good)
        _lib.status_word(CUDA).fill_(1)
        dec.step(good)
        torch.cuda.synchronize()
        with pytest.raises(_lib.KernelError, match="status 1"):
            call()
        dec.prefill(good)  # raised once
        dec.check()
    dec.release()


def test_a_bad_id_of_a_captured_step_is_raised_by_the_next_call() -> None:
    dec = _decoder(True, 1)
    good, bad = torch.tensor([[1], [2]], device=CUDA), torch.tensor([[1], [VOCAB]], device=CUDA)
    for _ in range(3):
        dec.step(good)
    dec.step(bad)
    torch.cuda.synchronize()
    with pytest.raises(_lib.KernelError, match="status 4"):
        dec.step(good)
    dec.release()
