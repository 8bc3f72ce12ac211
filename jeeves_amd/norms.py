"""Norms around a block of a served model, on MI355X, fused with the block's
gate, its residual and the quantizer of the FP8 projection that follows (C ABI
``include/jeeves_norm.h``).

* ``add_norm``: a block's output, normed and gated where the model does that,
  onto the residual, and the norm of the sum for the next block;
* ``gated_norm``: per-head norm of a linear attention's output times its gate
  (without weight: the output gate of a softmax attention).

Both give the e4m3 codes of the projection that reads their output on request,
in the launch that works it out, for ``fp8_matmul_quantized`` or
``FP8Linear.forward_codes``. Tensors are bf16 or fp16. As in ``jeeves_amd.fp8``,
everything is enqueued on ``torch.cuda.current_stream()`` without host
synchronisation, outputs come from torch's caching allocator, and bad arguments
raise ``ValueError``. No gradients: the framework serves.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .attention import _FP16, _head_weight, _heads, _on, _refuse
from .fp8 import QUANT_MAX_PACKED_COLS, packed_codes_bytes
from .fp8_weights import FP8

ACTIVATIONS = {None: 0, "sigmoid": 1, "silu": 2}
QUANTIZE = (None, "rows", "packed")


class Normed(NamedTuple):
    """What ``add_norm`` gives; what was not asked for is None."""

    h: torch.Tensor
    y: torch.Tensor | None
    codes: torch.Tensor | None
    scales: torch.Tensor | None


def _operand(name: str, t: torch.Tensor, dtype: torch.dtype, index: int, shape: tuple) -> tuple:
    """``t`` [tokens, cols] with 16-byte aligned rows: (the tensor, its address and row stride)."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index:
        _refuse(name, t, f"{dtype} {list(shape)} on HIP device {index}")
    (ts, unit), ptr = t.stride(), t.data_ptr()
    if unit != 1 or ts & 7 or ptr & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        ts, ptr = t.stride(0), t.data_ptr()
    return t, ptr, ts


def _weight(name: str, w: torch.Tensor | None, channels: int, index: int) -> torch.Tensor | None:
    if w is None:
        return None
    w = _head_weight(name, w, channels, index)
    return w.clone() if w.data_ptr() & 15 else w


def _codes(quantize: str | None, tokens: int, cols: int, device: torch.device) -> tuple:
    """(codes, their row stride, scales) for a batch's rows."""
    if quantize is None:
        return None, 0, None
    packed = quantize == "packed"
    codes = torch.empty(packed_codes_bytes(tokens, cols) if packed else (tokens, cols), dtype=torch.uint8 if packed else FP8, device=device)
    return codes, 0 if packed else cols, torch.empty(tokens, dtype=torch.float32, device=device)


def _check(activation: str | None, quantize: str | None, cols: int) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if quantize not in QUANTIZE:
        raise ValueError(f"quantize must be one of {QUANTIZE}, got {quantize!r}")
    if cols % 8 or not 0 < cols <= QUANT_MAX_PACKED_COLS:
        raise ValueError(f"a row has a multiple of 8 channels up to {QUANT_MAX_PACKED_COLS}, got {cols}")
    return ACTIVATIONS[activation]


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def add_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, *, post_weight: torch.Tensor | None = None,
             gate: torch.Tensor | None = None, activation: str | None = "sigmoid", scale: float = 1.0, eps: float = 1e-6,
             quantize: str | None = None, keep_y: bool = True) -> Normed:
    """Between two blocks: a block's output ``x`` [tokens, hidden] onto the
    residual stream, and the next block's norm of it, in one pass:

        b = x, or its RMS norm times ``post_weight`` [hidden]
        b = b * act(``gate``)                (``gate`` [tokens, hidden]; None: no gate)
        h = ``residual`` + ``scale`` * b     (None: no residual)
        y = RMS norm of h times ``weight`` [hidden]

    ``activation``: ``"sigmoid"``, ``"silu"`` or None (the gate as it is).
    Norms are ``x * weight / sqrt(mean(x^2) + eps)`` (a model whose norms scale
    by 1 + w passes 1 + w). In 32 bits throughout, h and y rounded once, y from
    the h before its rounding. ``weight`` None: only h.

    ``quantize``: also the codes and scales of ``quantize_rows`` of the y before
    its rounding: ``"rows"`` (float8_e4m3fn [tokens, hidden]) or ``"packed"``
    (the GEMMs' fragment order, for ``packed_rows=tokens``; hidden a multiple
    of 128). ``keep_y`` False leaves y itself out where only its codes are read.
    """
    dtype, index, shape = x.dtype, x.get_device(), x.shape
    if len(shape) != 2 or dtype not in _FP16 or index < 0:
        _refuse("x", x, "bfloat16 or float16 [tokens, hidden] on a HIP device")
    tokens, cols = shape
    act = _check(activation, quantize, cols)
    x, x_ptr, x_ts = _operand("x", x, dtype, index, shape)
    r_ptr, r_ts, g_ptr, g_ts = None, 0, None, 0
    if residual is not None:
        residual, r_ptr, r_ts = _operand("residual", residual, dtype, index, shape)
    if gate is not None:
        gate, g_ptr, g_ts = _operand("gate", gate, dtype, index, shape)
    weight, post_weight = _weight("weight", weight, cols, index), _weight("post_weight", post_weight, cols, index)
    if weight is None and quantize is not None:
        raise ValueError("the codes are those of y, which needs its norm's weight")
    h = torch.empty(shape, dtype=dtype, device=x.device)
    y = torch.empty(shape, dtype=dtype, device=x.device) if weight is not None and (keep_y or quantize is None) else None
    codes, ldc, scales = _codes(quantize, tokens, cols, x.device)
    if tokens:
        with _on(index):
            _lib.check(_lib.lib().jv_block_norm(
                x_ptr, x_ts, 0, r_ptr, r_ts, g_ptr, g_ts, 0, act, _ptr(post_weight), scale, _ptr(weight), eps, h.data_ptr(), _ptr(y),
                _ptr(codes), ldc, _ptr(scales), tokens, 1, cols, _FP16[dtype], torch._C._cuda_getCurrentRawStream(index)))
    return Normed(h, y, codes, scales)


def gated_norm(x: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor | None, *, activation: str | None = "silu", eps: float = 1e-6,
               quantize: str | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``x`` [tokens, heads, dim] (dim 64, 128 or 256), each head's channels
    normed (``x * weight / sqrt(mean(x^2) + eps)``, ``weight`` [dim]; None: no
    norm), times act(``gate``), the gate of the same shape: what a linear
    attention's output goes through before the out projection (weight and
    ``"silu"``), and the output gate of an attention layer (no weight,
    ``"sigmoid"``). x and gate may be views of a merged projection's output.

    A new contiguous tensor of x's shape, or with ``quantize`` (``"rows"`` or
    ``"packed"``, as in ``add_norm``) the codes and scales of the tokens' rows
    of heads * dim channels, before any rounding. In 32 bits, rounded once.
    """
    dtype, index, shape = x.dtype, x.get_device(), x.shape
    if len(shape) != 3 or dtype not in _FP16 or index < 0 or shape[2] not in (64, 128, 256):
        _refuse("x", x, "bfloat16 or float16 [tokens, heads, 64, 128 or 256] on a HIP device")
    tokens, heads, dim = shape
    act = _check(activation, quantize, heads * dim)
    x, x_ptr, x_ts, x_hs, _ = _heads("x", x, dtype, index, tokens, dim)
    if gate.shape != shape:
        _refuse("gate", gate, f"{dtype} {list(shape)} on HIP device {index}")
    gate, g_ptr, g_ts, g_hs, _ = _heads("gate", gate, dtype, index, tokens, dim)
    weight = _weight("weight", weight, dim, index)
    y = torch.empty(shape, dtype=dtype, device=x.device) if quantize is None else None
    codes, ldc, scales = _codes(quantize, tokens, heads * dim, x.device)
    if tokens:
        with _on(index):
            _lib.check(_lib.lib().jv_block_norm(
                x_ptr, x_ts, x_hs, None, 0, g_ptr, g_ts, g_hs, act, _ptr(weight), 1.0, None, eps, _ptr(y), None, _ptr(codes), ldc,
                _ptr(scales), tokens, heads, dim, _FP16[dtype], torch._C._cuda_getCurrentRawStream(index)))
    return y if quantize is None else (codes, scales)
