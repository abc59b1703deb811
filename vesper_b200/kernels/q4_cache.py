"""A decoding ring cache held in 4 bits on a B200: written, read back and attended.

``Q4RingKVCache`` is a ``RingKVCache`` (``vesper/attention.py:63-139`` of mstampfli/vesper-preview)
whose keys and values take 4 bits a channel plus two bf16 numbers per group of channels (32 where
the head dimension is a multiple of 32, else 16): ``lo``, the group's minimum rounded down, and
``step``, ``(max - lo) / 15`` rounded up, with ``code = rint((x - lo) / step)`` and value ``lo + code *
step``. Every value is then at most half a step off, however large the group's common offset
is. A group of one value (a range below 2^-100) has step 0; one that holds an infinity or a NaN reads back as
NaN and is seen only by the tokens that attend its slot.

- ``q4_ring_empty(b, hkv, dk, window, device)``: an unwritten ring;
- ``q4_write_(ring, k, v, pos)``: tokens written in place, quantised as they go in (a prefill chunk,
  any length, or one token);
- ``q4_read(ring, pos, dtype) -> (k, v, held)``: the values at given positions;
- ``q4_attend_(q, k, v, pos, ring)``: a decode step's attention (``vesper/attention.py:298-338``): one
  token per row is written and attends the window, itself included, as the ring holds it.

Serving only: nothing here is differentiated. Everything runs on torch's current stream, allocates
only through torch and can be captured in a CUDA graph.
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch
from torch import Tensor

from vesper_b200 import _lib
from vesper_b200.contracts import ContractError, Dims, check_shape, require_cuda
from vesper_b200.kernels.q8 import serving_only

SUPPORTED = (torch.float32, torch.bfloat16, torch.float16)
MAX_HEAD_DIM = 128
SLOT_TILE = 64  # slots are allocated in whole tiles
MAX_SLOTS = 2**31 - SLOT_TILE
MAX_TOKENS = 2**30  # tokens of a row in one call


def group_size(dk: int) -> int:
    """Channels per group: 32 where ``dk`` is a multiple of 32, else 16."""
    return 32 if dk % 32 == 0 else 16


@dataclass(frozen=True, slots=True)
class Q4RingKVCache:
    """A ring of ``window`` positions in 4 bits. ``slots`` is the window rounded up to a multiple of
    64; a token at position ``p`` lives in slot ``p % window``. Codes ``[b, hkv, slots, dk / 2]`` uint8
    (two a byte, in the attention kernel's channel order), parameters ``[b, hkv, slots, groups, 2]``
    bf16 (step, lo), ``pos [b, slots]`` int64, -1 where nothing was written. Its shapes never change and it
    is updated in place, so a captured decode step carries it."""

    k_codes: Tensor
    k_params: Tensor
    v_codes: Tensor
    v_params: Tensor
    pos: Tensor
    window: int

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[-1]


def q4_ring_empty(b: int, hkv: int, dk: int, window: int, device: torch.device) -> Q4RingKVCache:
    """Every slot unwritten (position -1)."""
    if not 1 <= window <= MAX_SLOTS:
        msg = f"window must be at least 1 and at most {MAX_SLOTS}, got {window}"
        raise ValueError(msg)
    if dk % 16 != 0 or not 16 <= dk <= MAX_HEAD_DIM:
        msg = f"head dimension {dk} must be a multiple of 16 and not exceed {MAX_HEAD_DIM}"
        raise ContractError(msg)
    slots = -(-window // SLOT_TILE) * SLOT_TILE
    groups = dk // group_size(dk)

    def codes() -> Tensor:
        return torch.zeros(b, hkv, slots, dk // 2, dtype=torch.uint8, device=device)

    def params() -> Tensor:
        return torch.zeros(b, hkv, slots, groups, 2, dtype=torch.bfloat16, device=device)

    pos = torch.full((b, slots), -1, dtype=torch.long, device=device)
    return Q4RingKVCache(codes(), params(), codes(), params(), pos, window)


def _check_ring(ring: Q4RingKVCache, what: str) -> tuple[int, int, int, int]:
    """``(b, hkv, dk, slots)`` of a well-formed ring on CUDA: accepts in one expression what is
    well-formed, else finds out what is not."""
    kc, kp, vc, vp, pos = ring.k_codes, ring.k_params, ring.v_codes, ring.v_params, ring.pos
    if kc.dim() == 4:
        shape, device = kc.shape, kc.device
        b, hkv, slots, half = shape
        params = (b, hkv, slots, half // 16 if half % 16 == 0 else half // 8, 2)
        if (
            half % 8 == 0 and 8 <= half <= MAX_HEAD_DIM // 2 and slots % SLOT_TILE == 0 and MAX_SLOTS >= slots >= ring.window >= 1
            and vc.shape == shape and kp.shape == params and vp.shape == params and pos.shape == (b, slots)
            and kc.dtype == torch.uint8 == vc.dtype and kp.dtype == torch.bfloat16 == vp.dtype and pos.dtype == torch.int64
            and kc.is_cuda and kp.device == device and vc.device == device and vp.device == device and pos.device == device
            and kc.is_contiguous() and kp.is_contiguous() and vc.is_contiguous() and vp.is_contiguous()
            and pos.is_contiguous()
            and (kc.data_ptr() | kp.data_ptr() | vc.data_ptr() | vp.data_ptr() | pos.data_ptr()) % 16 == 0
        ):  # fmt: skip
            return b, hkv, 2 * half, slots
    return _explain_ring(ring, what)


def _explain_ring(ring: Q4RingKVCache, what: str) -> tuple[int, int, int, int]:
    dims: Dims = {}
    check_shape("ring.k_codes", ring.k_codes, ("b", "hkv", "slots", "half"), dims, torch.uint8)
    b, hkv, slots, dk = dims["b"], dims["hkv"], dims["slots"], 2 * dims["half"]
    if dk % 16 != 0 or not 16 <= dk <= MAX_HEAD_DIM:
        msg = f"head dimension {dk} must be a multiple of 16 and not exceed {MAX_HEAD_DIM}"
        raise ContractError(msg)
    if ring.window < 1 or slots % SLOT_TILE or slots < ring.window or slots > MAX_SLOTS:
        msg = f"ring: {slots} slots must be a multiple of {SLOT_TILE} up to {MAX_SLOTS} holding the window {ring.window}"
        raise ContractError(msg)
    params = ("b", "hkv", "slots", dk // group_size(dk), 2)
    check_shape("ring.k_params", ring.k_params, params, dims, torch.bfloat16)
    check_shape("ring.v_codes", ring.v_codes, ("b", "hkv", "slots", "half"), dims, torch.uint8)
    check_shape("ring.v_params", ring.v_params, params, dims, torch.bfloat16)
    check_shape("ring.pos", ring.pos, ("b", "slots"), dims, torch.long)
    require_cuda(what, ring.k_codes, k_params=ring.k_params, v_codes=ring.v_codes, v_params=ring.v_params, pos=ring.pos)
    for name in ("k_codes", "k_params", "v_codes", "v_params", "pos"):
        t = getattr(ring, name)
        if not t.is_contiguous() or t.data_ptr() % 16:
            msg = f"ring.{name}: must be contiguous from a 16-byte boundary (it is updated in place)"
            raise ContractError(msg)
    return b, hkv, dk, slots


def _tokens(t: Tensor) -> Tensor:
    """``t [b, n, heads, dk]`` with each token's heads and channels dense, copied if they are not."""
    if t.is_contiguous():
        return t
    _, _, heads, dk = t.shape
    _, _, head, channel = t.stride()
    dense = (channel == 1 or dk == 1) and (head == dk or heads == 1)
    return t if dense else t.contiguous()


def _ring_ptrs(ring: Q4RingKVCache) -> tuple[int, int, int, int, int]:
    return (ring.k_codes.data_ptr(), ring.k_params.data_ptr(), ring.v_codes.data_ptr(), ring.v_params.data_ptr(),
            ring.pos.data_ptr())  # fmt: skip


def _check_tokens(ring: Q4RingKVCache, k: Tensor, v: Tensor, pos: Tensor, what: str) -> tuple[int, int, int, int, int]:
    b, hkv, dk, slots = _check_ring(ring, what)
    device = ring.pos.device
    shape = k.shape
    if not (
        len(shape) == 4 and shape[0] == b and shape[1] <= MAX_TOKENS and shape[2] == hkv and shape[3] == dk and v.shape == shape
        and pos.shape == shape[:2] and pos.dtype == torch.int64 and k.dtype in SUPPORTED and v.dtype == k.dtype
        and k.device == device and v.device == device and pos.device == device
    ):  # fmt: skip
        dims: Dims = {"b": b, "hkv": hkv, "dk": dk}
        check_shape("k", k, ("b", "n", "hkv", "dk"), dims)
        check_shape("v", v, ("b", "n", "hkv", "dk"), dims)
        check_shape("pos", pos, ("b", "n"), dims, torch.long)
        if k.dtype not in SUPPORTED or v.dtype != k.dtype:
            msg = f"k, v: one dtype of {SUPPORTED}, got {k.dtype} and {v.dtype}"
            raise ContractError(msg)
        require_cuda(what, ring.pos, k=k, v=v, positions=pos)
        msg = f"k: at most {MAX_TOKENS} tokens a row, got shape {tuple(shape)}"
        raise ContractError(msg)
    serving_only(what, k, v)
    return b, shape[1], hkv, dk, slots


@lru_cache(maxsize=256)
def _attend_workspace(b: int, heads: int, hkv: int, dk: int, window: int) -> int:
    """The library's answer for these sizes (0: none needed)."""
    return _lib.query("vb_q4_attend_workspace", b, heads, hkv, dk, window)


def q4_write_(ring: Q4RingKVCache, k: Tensor, v: Tensor, pos: Tensor) -> Q4RingKVCache:
    """Write tokens ``k, v [b, n, hkv, dk]`` at positions ``pos [b, n]`` (int64) into ``ring``, in place.

    Positions are consecutive along a row, with negative ones (padding, at either end) not written.
    Of ``n > window`` tokens the last ``window`` are kept. Returns ``ring``.

    Raises:
        ContractError: on a shape, dtype or device mismatch, or a ring that is not dense.
    """
    b, n, hkv, dk, slots = _check_tokens(ring, k, v, pos, "4-bit cache")
    if b == 0 or n == 0:
        return ring
    k, v, pos = _tokens(k), _tokens(v), pos.contiguous()
    _lib.call(
        "vb_q4_write", *_ring_ptrs(ring), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
        v.stride(1), pos.data_ptr(), b, n, hkv, dk, ring.window, slots, _lib.DTYPE_CODE[k.dtype],
        _lib.stream(k.device),
    )  # fmt: skip
    return ring


def q4_read(ring: Q4RingKVCache, pos: Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor, Tensor]:
    """``(k, v [b, n, hkv, dk], held [b, n] bool)``: what ``ring`` holds at positions ``pos [b, n]``.

    The values are formed in float32 and rounded once to ``dtype``. Where the ring does not hold a
    position (never written, overwritten since, or negative) ``held`` is False and the values zero.

    Raises:
        ContractError: on a shape, dtype or device mismatch, or a ring that is not dense.
    """
    b, hkv, dk, slots = _check_ring(ring, "4-bit cache")
    device = ring.pos.device
    if not (
        pos.dim() == 2 and pos.shape[0] == b and pos.shape[1] <= MAX_TOKENS and pos.dtype == torch.int64
        and pos.device == device and dtype in SUPPORTED
    ):  # fmt: skip
        check_shape("pos", pos, ("b", "n"), {"b": b}, torch.long)
        require_cuda("4-bit cache", ring.pos, positions=pos)
        if pos.shape[1] > MAX_TOKENS:
            msg = f"pos: at most {MAX_TOKENS} positions a row, got shape {tuple(pos.shape)}"
            raise ContractError(msg)
        msg = f"dtype: must be one of {SUPPORTED}, got {dtype}"
        raise ContractError(msg)
    n, pos = pos.shape[1], pos.contiguous()
    k = torch.empty(b, n, hkv, dk, dtype=dtype, device=device)
    v = torch.empty_like(k)
    held = torch.empty_like(pos, dtype=torch.bool, memory_format=torch.contiguous_format)
    if b and n:
        _lib.call(
            "vb_q4_read", *_ring_ptrs(ring), pos.data_ptr(), k.data_ptr(), v.data_ptr(), held.data_ptr(),
            b, n, hkv, dk, ring.window, slots, _lib.DTYPE_CODE[dtype], _lib.stream(device),
        )  # fmt: skip
    return k, v, held


def q4_attend_(q: Tensor, k: Tensor, v: Tensor, pos: Tensor, ring: Q4RingKVCache) -> Tensor:
    """One decoding token per row: written into ``ring`` (in place), then attending it.

    ``q [b, 1, h, dk]``, ``k, v [b, 1, hkv, dk]`` of ``q``'s dtype, ``pos [b, 1]`` int64. The output
    ``[b, 1, h, dk]`` is ``softmax(q k^T / sqrt(dk)) v`` over the slots whose positions lie in
    ``(pos - window, pos]``, the token itself included, with the values the ring holds (head ``h``
    reads key head ``h // (h_q / hkv)``). A row with a negative position writes nothing and its output is zero.

    Raises:
        ContractError: on a shape, dtype or device mismatch, query heads that are not a multiple of
            the key heads, or a ring that is not dense.
    """
    b, n, hkv, dk, slots = _check_tokens(ring, k, v, pos, "4-bit ring attention")
    if not (q.dim() == 4 and q.shape[0] == b and q.shape[1] == 1 and q.shape[3] == dk):
        check_shape("q", q, ("b", "one", "h", "dk"), {"b": b, "one": 1, "dk": dk})
    if n != 1:
        msg = f"k: axis 1 must be 1, got {n} (one token per row)"
        raise ContractError(msg)
    heads = q.shape[2]
    if hkv < 1 or heads < 1 or heads % hkv != 0:
        msg = f"{heads} query heads are not a multiple of {hkv} key heads"
        raise ContractError(msg)
    if q.dtype != k.dtype:
        msg = f"k: dtype must be {q.dtype} (q's), got {k.dtype}"
        raise ContractError(msg)
    device = q.device
    if device != k.device:
        require_cuda("4-bit ring attention", ring.pos, q=q)
    serving_only("4-bit ring attention", q)
    o = torch.empty(b, 1, heads, dk, dtype=q.dtype, device=device)
    if b == 0:
        return o
    q, k, v, pos = _tokens(q), _tokens(k), _tokens(v), pos.contiguous()
    nbytes = _attend_workspace(b, heads, hkv, dk, ring.window)
    ws = _lib.workspace(nbytes, device) if nbytes else None
    _lib.call(
        "vb_q4_attend", q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
        pos.data_ptr(), *_ring_ptrs(ring), o.data_ptr(), _lib.ptr(ws), b, heads, hkv, dk, ring.window, slots,
        _lib.DTYPE_CODE[q.dtype], _lib.stream(device),
    )  # fmt: skip
    return o
