"""Quantised one-token decoding of the looped model on a B200: int8 products over int8 weights, 4-bit rings.

``QuantizedVesper(model, dtype)`` quantises a ``Vesper``'s matrices once (8 bits, a float32 scale per output
channel, ``quantize_rows_q8``) and runs what ``vesper_b200.decode.decode_step`` runs (the contract of
``vesper/decode.py:29-46`` of mstampfli/vesper-preview) with them:

- every norm that feeds a product adds the sublayer's output to the float32 residual stream, normalises it and
  writes 8-bit rows, in one kernel (``add_rms_norm_q8``);
- the projections that share an input are one product (q, k, v and the write strengths; q, k, v of the attention),
  summed exactly in int32 (``linear_q8``); the scan's, the attention's and the feed-forward block's outputs are
  quantised by rows on their way to the next (``quantize_rows_q8``, with the squared ReLU in it for the last);
- the attention's window is a ``Q4RingKVCache``: its keys and values take 5 bits a channel, quantised as they
  are written, and the step attends them as they are held (``q4_attend_``);
- the recurrent state, the key filter and its history, the rotary turns and the residual stream stay as they are.

The float32 state update and everything the state feeds keep the precision of the float path; what the codes cost
is a relative error of about 0.6 % per 8-bit operand and 8 % of a spread per 4-bit key or value.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor

from vesper_b200.column import FUSED_INPUT_DTYPES, RMS_EPS, RMS_SCALE_FLOOR, Column, ColumnState
from vesper_b200.contracts import ContractError
from vesper_b200.kernels.act import residual_add
from vesper_b200.kernels.delta_scan import delta_scan_step_
from vesper_b200.kernels.q4_cache import Q4RingKVCache, q4_attend_
from vesper_b200.kernels.q8 import add_rms_norm_q8, linear_q8, quantize_rows_q8, rms_norm_q8
from vesper_b200.kernels.rotary import rotary
from vesper_b200.model import Vesper

Quantized = tuple[Tensor, Tensor]  # int8 rows and their float32 scales


@torch.no_grad()
def _quantize(*weights: Tensor) -> Quantized:
    """One matrix of the given ones' output channels, in 8 bits."""
    return quantize_rows_q8(torch.cat([w.detach().float() for w in weights]))


class QuantizedColumn:
    """A column's one-token step over 8-bit weights and 4-bit rings (``Column.step_decode``)."""

    def __init__(self, column: Column, dtype: torch.dtype = torch.bfloat16) -> None:
        self.column, self.dtype = column, dtype
        rec, attn, ffn = column.rec, column.attn, column.ffn
        self.rec_in = _quantize(rec.w_q, rec.w_k, rec.w_v, rec.w_beta)
        self.rec_out = _quantize(rec.w_o)
        self.attn_in = _quantize(attn.w_q, attn.w_k, attn.w_v)
        self.attn_out = _quantize(attn.w_o)
        self.ffn_in, self.ffn_out = _quantize(ffn.w1), _quantize(ffn.w2)

    def _linear(self, rows: Quantized, weight: Quantized) -> Tensor:
        return linear_q8(*rows, *weight, self.dtype)

    def step_decode(self, x: Tensor, r: Tensor | None, pos: Tensor, state: ColumnState, pass_index: int) -> tuple[Tensor, Tensor]:
        """One decoding token per row, ``state`` updated in place.

        ``x [b, 1, d]`` is the float32 residual stream and ``r`` the sublayer output still to be added to it (None
        where there is none); so are the stream and the output returned.
        """
        ring = state.kv[pass_index]
        if not isinstance(ring, Q4RingKVCache):
            msg = "a quantised step carries a Q4RingKVCache window (init_column_state(..., ring=True, q4=True))"
            raise ContractError(msg)
        column, dk = self.column, self.column.rec.head_dim
        rec, attn = column.rec, column.attn
        history, h = state.key_history[pass_index], state.h[pass_index]
        gain = column.norm_rec.weight
        if r is None:
            rows = rms_norm_q8(x, gain, RMS_SCALE_FLOOR, RMS_EPS)
        else:
            x, *rows = add_rms_norm_q8(x, r, gain, RMS_SCALE_FLOOR, RMS_EPS)
        d = x.shape[-1]
        q, z, v, logits = self._linear(rows, self.rec_in).split([d, d, d, rec.heads], dim=-1)
        z = z.contiguous()
        k, _ = rec.keys(z, history)
        if history.shape[1]:
            history.copy_(torch.cat([history[:, 1:], z.to(history.dtype)], dim=1))
        scan = FUSED_INPUT_DTYPES[rec.scan_impl]
        q, v = (t.unflatten(-1, (rec.heads, dk)).to(scan) for t in (q, v))
        o = delta_scan_step_(q, k.to(scan), v, logits.to(scan), h, from_logits=True)
        r = self._linear(quantize_rows_q8(o.flatten(2)), self.rec_out)

        x, *rows = add_rms_norm_q8(x, r, column.norm_attn.weight, RMS_SCALE_FLOOR, RMS_EPS)
        heads, kv = attn.heads * dk, attn.kv_heads * dk
        q, k, v = (t.unflatten(-1, (-1, dk)) for t in self._linear(rows, self.attn_in).split([heads, kv, kv], dim=-1))
        q, k = rotary(q, pos, attn.rotary_base), rotary(k, pos, attn.rotary_base)
        a = q4_attend_(q, k, v, pos, ring)
        r = self._linear(quantize_rows_q8(a.flatten(2)), self.attn_out)

        x, *rows = add_rms_norm_q8(x, r, column.norm_ffn.weight, RMS_SCALE_FLOOR, RMS_EPS)
        hidden = quantize_rows_q8(self._linear(rows, self.ffn_in), relu_square=True)
        return x, self._linear(hidden, self.ffn_out)


class QuantizedVesper:
    """A model's decoding step in 8-bit products and 4-bit rings; the model's own parameters are not touched.

    ``dtype`` (bf16 or float32) is what the products' outputs and the scan's inputs are rounded to. The model's scan
    (``set_scan``) must take it: ``"fused"`` for bf16, ``"fused-fp32"`` for float32.

    Raises:
        ContractError: if the model is not on CUDA or its head dimension is not one a 4-bit ring takes.
    """

    def __init__(self, model: Vesper, dtype: torch.dtype = torch.bfloat16) -> None:
        if next(model.parameters()).device.type != "cuda":
            msg = f"the quantised decoder runs on CUDA, the model is on {next(model.parameters()).device}"
            raise ContractError(msg)
        if model.shape.head_dim % 16 != 0 or model.shape.head_dim > 128:
            msg = f"head dimension {model.shape.head_dim} must be a multiple of 16 and not exceed 128"
            raise ContractError(msg)
        self.model, self.dtype = model, dtype
        self.columns = [QuantizedColumn(c, dtype) for c in model.loop.columns]
        self.embedding = _quantize(model.embedding.weight)

    @torch.no_grad()
    def forward(self, token: Tensor, position: Tensor, states: Sequence[ColumnState], depth: int) -> tuple[Tensor, Tensor]:
        """The stream and the last column's output ``[b, 1, d]`` after ``depth`` dense passes over one token per row
        (``vesper_b200.decode.decode_forward``), states advanced in place."""
        x, r = self.model.embedding.embed(token).float(), None
        for t in range(depth):
            if r is not None:
                x = residual_add(x, r)
            x, r = x + self.model.loop.u[t], None
            for c, column in enumerate(self.columns):
                x, r = column.step_decode(x, r, position, states[c], t)
        return x, r

    @torch.no_grad()
    def logits(self, x: Tensor, r: Tensor) -> Tensor:
        """The head ``[b, 1, V]``: the output norm of ``x + r``, then the tied embedding."""
        _, *rows = add_rms_norm_q8(x, r, self.model.norm_out.weight, RMS_SCALE_FLOOR, RMS_EPS)
        return linear_q8(*rows, *self.embedding, self.dtype)
