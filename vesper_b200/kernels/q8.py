"""Quantised linear layers on a B200: rows in 8 bits with a scale each, and the int8 product over them.

PRIMITIVES for serving (no gradients), what a decode step runs in place of a norm followed by a
bf16 ``F.linear`` (``vesper/column.py:159-188`` with ``:236-253``, ``vesper/ffn.py:44-56`` of
mstampfli/vesper-preview):

- ``rms_norm_q8(x, weight, floor, eps) -> (q, scale)``: the column's RMSNorm with its output in 8 bits;
- ``add_rms_norm_q8(x, r, weight, floor, eps) -> (s, q, scale)``: the same of ``s = x + r`` over a
  float32 residual stream, the sum stored too, one kernel;
- ``quantize_rows_q8(x, relu_square=False) -> (q, scale)``: any rows, or their squared ReLU;
- ``dequantize_rows_q8(q, scale, dtype)``: the values back;
- ``linear_q8(xq, xs, wq, ws, out_dtype)``: ``(xq @ wq.T) * xs[:, None] * ws``, summed exactly in int32.

A row ``y`` becomes codes ``rint(y * 127 / max|y|)`` in ``[-127, 127]`` and ``scale = max|y| / 127``
(float32). A row of magnitude below 1e-35 has scale 0; one that holds an infinity or a NaN has
codes 0 and a NaN scale, so whatever is made from it is NaN, as it would be without the codes.
A weight matrix is quantised once, by rows (output channels), with ``quantize_rows_q8``.

The code tensors are ``[..., W]`` with rows padded to a multiple of 16 bytes (the product's copies
start on 16-byte boundaries); ``linear_q8`` copies operands that are not laid out so.
"""

from __future__ import annotations

import torch
from torch import Tensor

from vesper_b200 import _lib
from vesper_b200.contracts import ContractError, Dims, check_shape, require_cuda

SUPPORTED = (torch.float32, torch.bfloat16, torch.float16)
MAX_K = 131056  # largest inner dimension whose int8 sums stay in int32
MAX_WIDTH = 2**30  # channels of a row
MAX_ROWS = 2**31 - 256  # rows of either operand: with a tile more still int32


def serving_only(what: str, *tensors: Tensor) -> None:
    """Refuse inputs that autograd is recording: these operators have no gradient."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                msg = f"the {what} has no gradient: call it under torch.no_grad()"
                raise ContractError(msg)


def check_width(name: str, x: Tensor) -> None:
    """Refuse rows whose width an entry point's int does not hold."""
    if x.shape[-1] > MAX_WIDTH:
        msg = f"{name}: rows of at most {MAX_WIDTH} channels, got shape {tuple(x.shape)}"
        raise ContractError(msg)


def _codes(x: Tensor) -> tuple[Tensor, Tensor, int]:
    """Empty codes and scales for ``x``'s rows, and the codes' row pitch."""
    *lead, width = x.shape
    device = x.device
    scale = torch.empty(*lead, dtype=torch.float32, device=device) if lead else torch.empty((), dtype=torch.float32, device=device)
    if width % 16 == 0:
        return torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format), scale, width
    pitch = -(-width // 16) * 16
    strides, step = [1], pitch
    for n in reversed(lead):
        strides.insert(0, step)
        step *= n
    return torch.empty_strided(x.shape, strides, dtype=torch.int8, device=device), scale, pitch


def _check_norm(x: Tensor, r: Tensor | None, weight: Tensor) -> None:
    """Accepts in one expression what is well-formed, else finds out what is not."""
    device = x.device
    if (
        x.is_cuda and x.dtype in SUPPORTED and x.dim() >= 1 and weight.dim() == 1 and MAX_WIDTH >= x.shape[-1] == weight.shape[0] >= 1
        and weight.device == device
        and (r is None or (x.dtype == torch.float32 and r.shape == x.shape and r.dtype in SUPPORTED and r.device == device))
    ):  # fmt: skip
        return
    require_cuda("8-bit RMSNorm", x, weight=weight, r=r)
    if x.dtype not in SUPPORTED:
        msg = f"x: dtype must be one of {SUPPORTED}, got {x.dtype}"
        raise ContractError(msg)
    if x.dim() < 1 or x.shape[-1] < 1:
        msg = f"x: expected rows of at least one channel, got shape {tuple(x.shape)}"
        raise ContractError(msg)
    check_width("x", x)
    if weight.shape != (x.shape[-1],):
        msg = f"weight: expected shape ({x.shape[-1]},), got {tuple(weight.shape)}"
        raise ContractError(msg)
    assert r is not None
    if x.dtype != torch.float32:
        msg = f"x: dtype must be {torch.float32} (the residual stream), got {x.dtype}"
        raise ContractError(msg)
    if r.shape != x.shape:
        msg = f"r: expected shape {tuple(x.shape)}, got {tuple(r.shape)}"
        raise ContractError(msg)
    msg = f"r: dtype must be one of {SUPPORTED}, got {r.dtype}"
    raise ContractError(msg)


def _norm(x: Tensor, r: Tensor | None, weight: Tensor, floor: float, eps: float):
    _check_norm(x, r, weight)
    width = weight.shape[0]
    x = x.contiguous()
    if weight.dtype != torch.float32 or not weight.is_contiguous():
        weight = weight.to(torch.float32).contiguous()
    q, scale, pitch = _codes(x)
    code = _lib.DTYPE_CODE
    if r is None:
        serving_only("8-bit RMSNorm", x, weight)
        total, total_ptr, r_ptr, r_code = None, None, None, 0
    else:
        serving_only("8-bit RMSNorm", x, r, weight)
        r = r.contiguous()
        total = torch.empty_like(x)
        total_ptr, r_ptr, r_code = total.data_ptr(), r.data_ptr(), code[r.dtype]
    _lib.call(
        "vb_rms_norm_q8", x.data_ptr(), r_ptr, weight.data_ptr(), total_ptr, q.data_ptr(), pitch, scale.data_ptr(),
        x.numel() // width, width, floor, eps, code[x.dtype], r_code, _lib.stream(x.device),
    )  # fmt: skip
    return total, q, scale


def rms_norm_q8(x: Tensor, weight: Tensor, floor: float, eps: float) -> tuple[Tensor, Tensor]:
    """``(q [..., W] int8, scale [...] float32)`` of ``fused_rms_norm(x, weight, floor, eps)``.

    The norm is computed and quantised in float32 whatever ``x``'s dtype (float32, bf16 or f16).

    Raises:
        ContractError: on a CPU tensor, an unsupported dtype or a weight of another width.
    """
    _, q, scale = _norm(x, None, weight, floor, eps)
    return q, scale


def add_rms_norm_q8(x: Tensor, r: Tensor, weight: Tensor, floor: float, eps: float) -> tuple[Tensor, Tensor, Tensor]:
    """``(s, q, scale)``: ``s = x + r`` (float32) and ``rms_norm_q8(s, weight, floor, eps)``, one kernel.

    ``x`` is the float32 residual stream, ``r`` a sublayer's output of the same shape (float32, bf16
    or f16); the sum is one IEEE float32 addition per channel, as torch's mixed-dtype add makes it.

    Raises:
        ContractError: as ``rms_norm_q8``, or where ``x`` is not float32 or ``r`` has another shape.
    """
    return _norm(x, r, weight, floor, eps)


def quantize_rows_q8(x: Tensor, *, relu_square: bool = False) -> tuple[Tensor, Tensor]:
    """``(q [..., W] int8, scale [...] float32)`` of ``x``'s rows, or of ``relu(x)^2`` (formed in float32).

    ``x`` may be a slice of wider rows (contiguous channels); anything else is copied first.

    Raises:
        ContractError: on a CPU tensor, an unsupported dtype or rows without channels.
    """
    require_cuda("8-bit rows", x)
    serving_only("8-bit quantisation", x)
    if x.dtype not in SUPPORTED:
        msg = f"x: dtype must be one of {SUPPORTED}, got {x.dtype}"
        raise ContractError(msg)
    if x.dim() < 1 or x.shape[-1] < 1:
        msg = f"x: expected rows of at least one channel, got shape {tuple(x.shape)}"
        raise ContractError(msg)
    check_width("x", x)
    width = x.shape[-1]
    if not (x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= width):
        x = x.contiguous()
    ldx = x.stride(0) if x.dim() == 2 and x.shape[0] > 1 else width
    q, scale, pitch = _codes(x)
    _lib.call(
        "vb_quantize_rows_q8", x.data_ptr(), ldx, q.data_ptr(), pitch, scale.data_ptr(), x.numel() // width, width,
        int(relu_square), _lib.DTYPE_CODE[x.dtype], _lib.stream(x.device),
    )  # fmt: skip
    return q, scale


def _pitched(t: Tensor) -> tuple[Tensor, int]:
    """``t [rows, K]`` int8 with rows a multiple of 16 bytes apart from a 16-byte boundary, and their
    pitch: ``t`` itself where it is laid out so (as this module's codes are), else a copy."""
    n, k = t.shape
    row, step = t.stride()
    if step == 1 or k == 1:
        pitch = row if n > 1 else -(-k // 16) * 16
        if pitch % 16 == 0 and pitch >= k and t.data_ptr() % 16 == 0:
            return t, pitch
    pitch = -(-k // 16) * 16
    copy = torch.zeros(n, pitch, dtype=torch.int8, device=t.device)
    copy[:, :k] = t
    return copy, pitch


def dequantize_rows_q8(q: Tensor, scale: Tensor, dtype: torch.dtype = torch.float32) -> Tensor:
    """The values ``q * scale`` of 8-bit rows ``[..., W]`` in ``dtype``, rounded once.

    Raises:
        ContractError: on a CPU tensor, codes that are not int8, scales that are not float32 of the
            rows' shape or an unsupported ``dtype``.
    """
    if not (
        q.is_cuda and scale.device == q.device and q.dtype == torch.int8 and scale.dtype == torch.float32 and q.dim() >= 1
        and MAX_WIDTH >= q.shape[-1] >= 1 and scale.shape == q.shape[:-1] and dtype in SUPPORTED
    ):  # fmt: skip
        require_cuda("8-bit rows", q, scale=scale)
        if q.dtype != torch.int8 or scale.dtype != torch.float32:
            msg = f"q, scale: dtypes must be {torch.int8} and {torch.float32}, got {q.dtype} and {scale.dtype}"
            raise ContractError(msg)
        if dtype not in SUPPORTED:
            msg = f"dtype: must be one of {SUPPORTED}, got {dtype}"
            raise ContractError(msg)
        if q.dim() >= 1:
            check_width("q", q)
        msg = f"scale: expected one per row of q {tuple(q.shape)}, got shape {tuple(scale.shape)}"
        raise ContractError(msg)
    width = q.shape[-1]
    rows = q.numel() // width
    if q.is_contiguous():
        flat, pitch = q, width
    else:
        flat = q if q.dim() == 2 else q.reshape(rows, width)  # a view of codes as this module lays them out
        if (width > 1 and flat.stride(1) != 1) or (rows > 1 and flat.stride(0) < width):
            flat = flat.contiguous()
        pitch = flat.stride(0) if rows > 1 else width
    scale = scale.contiguous()  # a copy is held until the launch: its memory is not to be had again before
    y = torch.empty(*q.shape, dtype=dtype, device=q.device)
    _lib.call(
        "vb_dequantize_rows_q8", flat.data_ptr(), pitch, scale.data_ptr(), y.data_ptr(), rows, width,
        _lib.DTYPE_CODE[dtype], _lib.stream(q.device),
    )  # fmt: skip
    return y


def _check_linear(xq: Tensor, xs: Tensor, wq: Tensor, ws: Tensor, out_dtype: torch.dtype) -> tuple[int, int]:
    """``(N, K)``: accepts in one expression what is well-formed, else finds out what is not."""
    if wq.dim() == 2 and xq.dim() >= 1:
        device, x_shape, (n, k) = xq.device, xq.shape, wq.shape
        if (
            wq.dtype == torch.int8 == xq.dtype and xs.dtype == torch.float32 == ws.dtype
            and 1 <= k <= MAX_K and 1 <= n <= MAX_ROWS and xs.numel() <= MAX_ROWS and x_shape[-1] == k
            and xs.shape == x_shape[:-1] and ws.shape == (n,) and out_dtype in SUPPORTED and xq.is_cuda
            and xs.device == device and wq.device == device and ws.device == device
        ):  # fmt: skip
            return n, k
    dims: Dims = {}
    check_shape("wq", wq, ("N", "K"), dims, torch.int8)
    check_shape("ws", ws, ("N",), dims, torch.float32)
    if xq.dim() < 1 or xq.dtype != torch.int8 or xq.shape[-1] != dims["K"]:
        msg = f"xq: expected int8 rows of {dims['K']} channels, got {xq.dtype} {tuple(xq.shape)}"
        raise ContractError(msg)
    if xs.shape != xq.shape[:-1] or xs.dtype != torch.float32:
        msg = f"xs: expected one float32 scale per row of xq {tuple(xq.shape)}, got {xs.dtype} {tuple(xs.shape)}"
        raise ContractError(msg)
    if out_dtype not in SUPPORTED:
        msg = f"out_dtype: must be one of {SUPPORTED}, got {out_dtype}"
        raise ContractError(msg)
    require_cuda("int8 product", xq, xs=xs, wq=wq, ws=ws)
    msg = (f"wq: expected 1 to {MAX_ROWS} rows of 1 to {MAX_K} channels for at most {MAX_ROWS} rows of xq, got shape "
           f"{tuple(wq.shape)} for {tuple(xq.shape)}")  # fmt: skip
    raise ContractError(msg)


def linear_q8(xq: Tensor, xs: Tensor, wq: Tensor, ws: Tensor, out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``y [..., N]``: the quantised linear layer, ``y[m, n] = (sum_k xq[m, k] wq[n, k]) * xs[m] * ws[n]``.

    Args:
        xq, xs: int8 rows ``[..., K]`` and their float32 scales ``[...]``.
        wq, ws: int8 weights ``[N, K]`` and their float32 scales ``[N]``.
        out_dtype: float32, bf16 or f16; the scaled float32 sum is rounded to it once.

    Raises:
        ContractError: on a shape or dtype mismatch, a CPU tensor or ``K`` above 131056 (where a sum
            of int8 products may leave int32).
    """
    n, k = _check_linear(xq, xs, wq, ws, out_dtype)
    device = xq.device
    flat = xq if xq.dim() == 2 else xq.reshape(-1, k)
    rows, ldx = _pitched(flat)
    weights, ldw = _pitched(wq)
    xs, ws = xs.contiguous(), ws.contiguous()  # copies are held until the launch: their memory is not to be had again before
    m = xs.numel()
    y = torch.empty(m, n, dtype=out_dtype, device=device)
    _lib.call(
        "vb_linear_q8", rows.data_ptr(), ldx, xs.data_ptr(), weights.data_ptr(), ldw, ws.data_ptr(), y.data_ptr(), m, n, k,
        _lib.DTYPE_CODE[out_dtype], _lib.status_word(device).data_ptr(), _lib.stream(device),
    )  # fmt: skip
    return y if flat is xq else y.view(*xq.shape[:-1], n)
