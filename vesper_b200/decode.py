"""Batched one-token decoding of the looped model on a B200, captured as one CUDA graph.

The contract of ``vesper/decode.py`` (``decode_step`` ``:29-46``, ``CapturedDecoder`` ``:49-97``)
of mstampfli/vesper-preview, batched: the reference decoder takes one row (its ring writes one
slot per row); here every row of a batch decodes its own stream in the same step. A step embeds
one token per row, runs the loop at a fixed depth with every token active in every pass (the
reference's ``DenseRule``: ``y`` is the last pass's output), applies the head to it and takes the
argmax over the first ``vocab`` ids. Every column keeps, per pass, its float32 recurrent state,
its key history and a ``RingKVCache``; the step updates all of them IN PLACE (``Column.step_decode``:
the one-token scan kernel, the batched ring-attention kernel), so their shapes and addresses never
change and one captured graph serves every step.

``prefill`` is the long-context half: the prompt runs through the ordinary chunked forward
(``Vesper.run`` with the dense rule, chronological ``KVCache`` windows, the chunked scan and
window-attention kernels), chunk by chunk with carried states, and its windows are then moved into
rings (``ring_from_cache``), so decoding continues exactly where the prompt ended. ``extend`` is the way
back: the rings' windows become chronological caches again (``cache_from_ring``), more prompt runs
through the chunked forward, and its tokens go into the rings.

``quantized=True`` decodes with int8 products and rings held in 4 bits (``vesper_b200.quant``).
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor

from vesper_b200 import _lib
from vesper_b200.attention import KVCache, RingKVCache, cache_from_ring, q4_ring_from_cache, ring_from_cache
from vesper_b200.column import ColumnState, state_tensors
from vesper_b200.contracts import ContractError
from vesper_b200.kernels.q4_cache import Q4RingKVCache, q4_write_
from vesper_b200.loop import DenseRule
from vesper_b200.model import Vesper
from vesper_b200.quant import QuantizedVesper


def decode_forward(model: Vesper, token: Tensor, position: Tensor, states: Sequence[ColumnState], depth: int) -> Tensor:
    """``y [b, 1, d]`` of one token per row at ``depth`` dense passes, states updated in place.

    The loop of ``vesper/loop.py:349-465`` under ``DenseRule`` (every token active in every pass;
    the output is the last pass's) for ``n = 1``.
    """
    x = model.embedding.embed(token)
    for t in range(depth):
        h = x + model.loop.u[t]
        for c, column in enumerate(model.loop.columns):
            h = column.step_decode(h, position, states[c], t)
        x = h
    return x


def decode_step(model: Vesper, depth: int, vocab: int, states: Sequence[ColumnState], token: Tensor,
                position: Tensor) -> tuple[Tensor, Tensor]:  # fmt: skip
    """``(ids [b, 1], logits [b, 1, vocab])`` of one token per row (``vesper/decode.py:29-46``),
    the states advanced in place."""
    y = decode_forward(model, token, position, states, depth)
    logits = model.head(y)[..., :vocab]
    return logits.argmax(-1), logits


class BatchedDecoder:
    """Greedy decoding of ``b`` rows at ``depth`` passes, the step captured after ``warm`` eager steps.

    ``prefill(tokens)`` runs a prompt ``[b, P]`` (positions ``0 .. P-1``) and returns the logits of
    every prompt position; ``step(token)`` advances every row by one token ``[b, 1]`` at the next
    position and returns ``(ids, logits)`` (the graph's buffers after a replay: read them before the
    next step). ``extend(tokens)`` runs more tokens of a prompt ``[b, P]`` at the positions that follow, after any
    number of steps. ``dtype``: the activation dtype (bfloat16 runs under autocast with the chunked and
    one-token bf16 kernels; float32 is the reference's precision). ``quantized``: the steps run int8
    products over weights quantised here, once, and attend rings held in 4 bits; prompts run in ``dtype``
    as ever, their windows quantised as they enter the rings.

    Raises:
        ContractError: if the model is not on CUDA or ``depth`` is outside ``1..t_max``, or ``quantized`` with a
            head dimension that is not a multiple of 16 up to 128.
    """

    def __init__(self, model: Vesper, depth: int, vocab: int, b: int, dtype: torch.dtype = torch.bfloat16,
                 warm: int = 2, *, quantized: bool = False) -> None:  # fmt: skip
        device = next(model.parameters()).device
        if device.type != "cuda":
            msg = f"the decoder runs on CUDA, the model is on {device}"
            raise ContractError(msg)
        if not 1 <= depth <= model.t_max:
            msg = f"depth {depth} is outside 1..{model.t_max}"
            raise ContractError(msg)
        self.model, self.depth, self.vocab, self.b, self.dtype, self.warm = model, depth, vocab, b, dtype, warm
        self.device = device
        self.quant = QuantizedVesper(model, dtype) if quantized else None
        self.states: list[ColumnState] = model.init_states(b, dtype, device, ring=True, q4=quantized)
        self.length, self.last = 0, 0  # tokens so far, and the last one's position, of every row
        self.token = torch.zeros(b, 1, dtype=torch.long, device=device)
        self.position = torch.zeros(b, 1, dtype=torch.long, device=device)
        self.graph: torch.cuda.CUDAGraph | None = None
        self.outputs: tuple[Tensor, Tensor] | None = None
        self.steps = 0
        # the device's status word as the last step left it, read by the next call without waiting
        _lib.status_word(device)
        self._status = torch.zeros(1, dtype=torch.int32, pin_memory=True)

    def check(self) -> None:
        """Wait for the steps so far and raise ``KernelError`` if a kernel gave up or an id was out of range in one."""
        try:
            _lib.check_status(self.device)
        finally:
            self._status.zero_()

    def _autocast(self):
        return torch.autocast("cuda", dtype=torch.bfloat16, enabled=self.dtype == torch.bfloat16)

    @torch.no_grad()
    def prefill(self, tokens: Tensor, chunk: int = 2048, *, all_logits: bool = False) -> Tensor:
        """Run the prompt ``[b, P]`` chunk by chunk; the rings then hold its last windows.

        Returns the logits of the last prompt position ``[b, 1, vocab]`` (of every position with
        ``all_logits``, ``[b, P, vocab]``: a long prompt's full logits are large)."""
        b, length = tokens.shape
        if b != self.b:
            msg = f"prompt of {b} rows for a decoder of {self.b}"
            raise ContractError(msg)
        if int(self._status):
            self.check()
        logits, states = self._chunks(tokens, self.model.init_states(b, self.dtype, self.device), 0, chunk, all_logits)
        to_ring = q4_ring_from_cache if self.quant else ring_from_cache
        rings = [ColumnState(h=s.h, kv=tuple(to_ring(c) for c in s.kv), key_history=s.key_history)
                 for s in states]  # fmt: skip
        # into the decoder's own (possibly captured) buffers
        for dst, src in zip(state_tensors(self.states), state_tensors(rings), strict=True):
            dst.copy_(src)
        self.position.fill_(length - 1)
        self.length, self.last = length, length - 1
        return logits

    def _chunks(self, tokens: Tensor, states: list[ColumnState], first: int, chunk: int,
                all_logits: bool) -> tuple[Tensor, list[ColumnState]]:  # fmt: skip
        """The chunked forward of ``tokens [b, P]`` from position ``first``: logits and new states."""
        b, length = tokens.shape
        outs = []
        for s in range(0, length, chunk):
            piece = tokens[:, s : s + chunk].to(self.device)
            pos = torch.arange(first + s, first + s + piece.shape[1], device=self.device).expand(b, -1).contiguous()
            with self._autocast():
                res = self.model.run(piece, pos, states, passes=self.depth, exit_rule=DenseRule())
                if all_logits or s + chunk >= length:
                    outs.append(self.model.head(res.y if all_logits else res.y[:, -1:])[..., : self.vocab])
            states = list(res.states)
        return torch.cat(outs, dim=1), states

    @torch.no_grad()
    def extend(self, tokens: Tensor, chunk: int = 2048, *, all_logits: bool = False) -> Tensor:
        """Run ``tokens [b, P]`` at the positions after every row's last one, as ``prefill`` runs a prompt.

        The windows are read out of the rings (4-bit ones as the values they stand for), the chunked forward carries
        them and the states on, and the new tokens are written into the rings; older entries of the rings stay as
        they are. Returns logits as ``prefill`` does."""
        b, length = tokens.shape
        if b != self.b:
            msg = f"prompt of {b} rows for a decoder of {self.b}"
            raise ContractError(msg)
        if length == 0:
            msg = "extend: at least one token is needed"
            raise ContractError(msg)
        if self.length == 0:
            return self.prefill(tokens, chunk, all_logits=all_logits)
        if int(self._status):
            self.check()
        last = self.position[:, 0]

        def cache(t: int, ring: RingKVCache | Q4RingKVCache) -> KVCache:  # a pass that is not run has nothing in its ring
            return cache_from_ring(ring, last, min(self.length, ring.window) if t < self.depth else 0, self.dtype)

        caches = [
            ColumnState(h=s.h, kv=tuple(cache(t, c) for t, c in enumerate(s.kv)), key_history=s.key_history)
            for s in self.states
        ]
        logits, states = self._chunks(tokens, caches, self.last + 1, chunk, all_logits)
        for old, new in zip(self.states, states, strict=True):
            for dst, src in zip((*old.h, *old.key_history), (*new.h, *new.key_history), strict=True):
                dst.copy_(src)
            for ring, window in zip(old.kv[: self.depth], new.kv[: self.depth], strict=True):
                self._into_ring(ring, window, min(length, window.window))
        self.position.add_(length)
        self.length, self.last = self.length + length, self.last + length
        return logits

    @staticmethod
    def _into_ring(ring: RingKVCache | Q4RingKVCache, cache: KVCache, n: int) -> None:
        """The newest ``n`` entries of ``cache`` into ``ring``, in place."""
        m = cache.k.shape[1]
        k, v, pos = cache.k[:, m - n :], cache.v[:, m - n :], cache.pos[:, m - n :]
        if isinstance(ring, Q4RingKVCache):
            q4_write_(ring, k, v, pos)
            return
        slot = pos % ring.window
        at = slot[:, :, None, None].expand_as(k)
        ring.k.scatter_(1, at, k.to(ring.k.dtype))
        ring.v.scatter_(1, at, v.to(ring.v.dtype))
        ring.pos.scatter_(1, slot, pos)
        ring.valid.scatter_(1, slot, torch.ones_like(slot, dtype=torch.bool))

    def _body(self) -> tuple[Tensor, Tensor]:
        self.position.add_(1)
        if self.quant is not None:
            x, r = self.quant.forward(self.token, self.position, self.states, self.depth)
            logits = self.quant.logits(x, r)[..., : self.vocab]
            out = logits.argmax(-1), logits
        else:
            with self._autocast():
                out = decode_step(self.model, self.depth, self.vocab, self.states, self.token, self.position)
        self._status.copy_(_lib.status_word(self.device), non_blocking=True)
        return out

    @torch.no_grad()
    def step(self, token: Tensor) -> tuple[Tensor, Tensor]:
        """One token per row ``[b, 1]`` at the next position: ``(ids [b, 1], logits [b, 1, vocab])``.

        A kernel of a step that gave up waiting, or an id outside the vocabulary in a captured one, makes that step's
        outputs and states wrong and raises ``KernelError`` from the first call after the step has ended (or from
        ``check()``, which waits for it): the decoder then starts again with ``prefill``."""
        if int(self._status):
            self.check()
        self.token.copy_(token)
        if self.steps < self.warm:  # eager, on a side stream joined to the current one
            side = torch.cuda.Stream(self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            try:
                with torch.cuda.stream(side):
                    out = self._body()
            except ContractError:  # a refused token takes no position
                torch.cuda.current_stream(self.device).wait_stream(side)
                self.position.sub_(1)
                raise
            torch.cuda.current_stream(self.device).wait_stream(side)
        else:
            if self.graph is None:
                # capturing records the step without running it: the live buffers are untouched
                torch.cuda.synchronize(self.device)
                self.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self.graph):
                    self.outputs = self._body()
            self.graph.replay()
            out = self.outputs
        self.steps += 1
        self.length, self.last = self.length + 1, self.last + 1
        return out

    def release(self) -> None:
        self.graph = None
        self.outputs = None

