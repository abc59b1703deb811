"""A whole quantised decoding step (``QuantizedVesper``) on a B200 against the same step with its products and attention in
float32 torch.

Tolerance, derived before the first run: a column's step is within 1e-2 of its formula (values that move across the middle of a
code's step, a few of a row's 64 to 128); the two passes of two columns and the head's own rows add up to 5e-2 at most.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F  # noqa: N812

from test_quantized_decode_gpu import DEPTH, SHAPE, VOCAB, _model, _plain_step, _tokens
from vesper_b200.column import RMS_EPS, RMS_SCALE_FLOOR, state_tensors
from vesper_b200.kernels.q8 import add_rms_norm_q8, dequantize_rows_q8
from vesper_b200.quant import QuantizedVesper

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")


def _rel(a: torch.Tensor, b: torch.Tensor) -> float:
    return float((a.double() - b.double()).norm() / b.double().norm())


@torch.no_grad()
def test_a_quantised_model_s_step_is_its_formula() -> None:
    b, steps = 4, 40
    model = _model("fused-fp32")
    quant = QuantizedVesper(model, torch.float32)
    ours, plain = (model.init_states(b, torch.float32, CUDA, ring=True, q4=True) for _ in range(2))
    tokens = _tokens(b, steps, 51)
    assert SHAPE.window < steps
    for i in range(steps):
        token, pos = tokens[:, i : i + 1], torch.full((b, 1), i, device=CUDA)
        x, r = quant.forward(token, pos, ours, DEPTH)
        logits = quant.logits(x, r)
        px, pr = model.embedding.embed(token).float(), None
        for t in range(DEPTH):
            px, pr = (px if pr is None else px + pr) + model.loop.u[t], None
            for c, column in enumerate(quant.columns):
                px, pr = _plain_step(column, px, pr, pos, plain[c], t)
        _, *rows = add_rms_norm_q8(px, pr, model.norm_out.weight, RMS_SCALE_FLOOR, RMS_EPS)
        want = F.linear(dequantize_rows_q8(*rows), dequantize_rows_q8(*quant.embedding))
        assert logits.shape == (b, 1, VOCAB)
        assert _rel(logits, want) < 5e-2, i
        # what is carried on starts the next step equal, so that a code's difference does not add up over the steps
        for dst, src in zip(state_tensors(plain), state_tensors(ours), strict=True):
            dst.copy_(src)
