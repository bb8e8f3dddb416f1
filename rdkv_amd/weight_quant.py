"""4-bit weights with group scales, and the products that read them.

The projections of a decode step read every weight once per token; as 4-bit codes with one scale
and zero point per group of 32, 64 or 128 columns they are a quarter of the bytes.  A matrix is
quantized (``quantize_weight``) or taken over from a checkpoint (``pack_weight``) once, into the
layout that the kernels stream, and used by ``linear`` (one activation row, a batch, a prompt
chunk), ``norm_linear`` and ``silu_linear`` (one row with the operation in front folded in, as the
decode loops use them).  ``fast_decode.quantize_weights`` does this for a whole model.

The reference has no quantized weights; the products stand where its loop calls ``F.linear``
(obkv_accel/fast_decode.py:1650-1656, 1786, 1797-1804, 1826).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib

GROUP_SIZES = (32, 64, 128)
_MAX_ROW_K = 32768          # what the one-row kernels hold of an activation row


@dataclass(frozen=True, eq=False)
class QuantizedWeight:
    """A matrix [N, K] as ``(q - zero) * scale`` with q and zero in 0 .. 15, in the kernels' layout
    (include/rdkv.h).  ``dtype``: the type of the activations it is multiplied with."""
    codes: torch.Tensor      # uint8, rdkv_w4_codes_bytes
    scales: torch.Tensor     # int32, rdkv_w4_scale_words
    N: int
    K: int
    group_size: int
    dtype: torch.dtype

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.N, self.K)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()


def _empty(N: int, K: int, group_size: int, dtype: torch.dtype, dev: torch.device) -> QuantizedWeight:
    assert group_size in GROUP_SIZES, f"group_size must be one of {GROUP_SIZES}, got {group_size}"
    assert dtype in (torch.float16, torch.bfloat16), f"fp16 or bf16, got {dtype}"
    assert N >= 0 and K >= 1, f"a matrix of {N} x {K}"
    lib = _lib.load()
    return QuantizedWeight(torch.empty(lib.rdkv_w4_codes_bytes(N, K), dtype=torch.uint8, device=dev),
                           torch.empty(lib.rdkv_w4_scale_words(N, K, group_size), dtype=torch.int32, device=dev),
                           N, K, group_size, dtype)


def quantize_weight(weight: torch.Tensor, group_size: int = 128) -> QuantizedWeight:
    """Round-to-nearest quantization of ``weight`` [N, K] (fp16 / bf16; rows of any stride) by groups
    of ``group_size`` columns, the last of a row may be short.  The range of a group takes in
    zero, so zeros stay zeros.  A group that holds a NaN or an infinity becomes NaN."""
    if weight.is_cuda:
        if _lib.native is None:
            _lib.load()
        pair = _lib.native.w4_quantize(weight, group_size, _lib.stream_of(weight.device))
        if pair is not None:
            return QuantizedWeight(*pair, *weight.shape, group_size, weight.dtype)
    dev = _lib.require_device(weight)
    assert weight.dim() == 2, f"a matrix, got {tuple(weight.shape)}"
    if weight.stride(1) != 1 or (weight.shape[0] > 1 and weight.stride(0) < weight.shape[1]):
        weight = weight.contiguous()
    q = _empty(weight.shape[0], weight.shape[1], group_size, weight.dtype, dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().rdkv_w4_quantize(weight.data_ptr(), weight.stride(0), q.N, q.K, group_size,
                                                _lib.DTYPE_CODE[q.dtype], _lib.ptr(q.codes), _lib.ptr(q.scales),
                                                _lib.stream_of(dev)))
    return q


def pack_weight(codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None, group_size: int = 128,
                dtype: Optional[torch.dtype] = None) -> QuantizedWeight:
    """A matrix quantized elsewhere: ``codes`` uint8 [N, K] with values 0 .. 15, ``scale`` [N, groups]
    (fp16, bf16, or fp32 rounded to 20 significant bits), ``zero`` integers 0 .. 15 of the same shape (None: 8).
    ``dtype``: of the activations (default: the scales', fp16 for fp32 scales)."""
    dev = _lib.require_device(codes, scale, zero)
    assert codes.dim() == 2 and codes.dtype == torch.uint8, "codes: a uint8 matrix"
    N, K = codes.shape
    if dtype is None:
        dtype = torch.float16 if scale.dtype == torch.float32 else scale.dtype
    q = _empty(N, K, group_size, dtype, dev)
    groups = -(-K // group_size)
    assert tuple(scale.shape) == (N, groups) and scale.dtype in _lib.DTYPE_CODE, \
        f"scale: {(N, groups)} floats, got {tuple(scale.shape)} {scale.dtype}"
    codes, scale = codes.contiguous(), scale.contiguous()
    if zero is not None:
        assert tuple(zero.shape) == (N, groups) and not zero.dtype.is_floating_point, \
            f"zero: {(N, groups)} integers, got {tuple(zero.shape)} {zero.dtype}"
        zero = zero.to(torch.uint8).contiguous()
    with torch.cuda.device(dev):
        _lib.check(_lib.load().rdkv_w4_pack(_lib.ptr(codes), K, _lib.ptr(scale), _lib.DTYPE_CODE[scale.dtype], groups,
                                            _lib.ptr(zero), groups, N, K, group_size, _lib.ptr(q.codes),
                                            _lib.ptr(q.scales), _lib.stream_of(dev)))
    return q


def dequantize_weight(q: QuantizedWeight, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The matrix [N, K] that the codes stand for, each value rounded to ``q.dtype``."""
    if out is None:
        w = _native("w4_dequantize", q, *_fields(q))
        if w is not None:
            return w
    dev = _lib.require_device(q.codes, q.scales, out)
    if out is None:
        out = torch.empty(q.N, q.K, dtype=q.dtype, device=dev)
    assert tuple(out.shape) == q.shape and out.dtype == q.dtype and out.stride(1) == 1, \
        f"out: {q.shape} {q.dtype} with unit column stride"
    with torch.cuda.device(dev):
        _lib.check(_lib.load().rdkv_w4_dequant(_lib.ptr(q.codes), _lib.ptr(q.scales), q.N, q.K, q.group_size,
                                               _lib.DTYPE_CODE[q.dtype], _lib.ptr(out), out.stride(0),
                                               _lib.stream_of(dev)))
    return out


def _fields(q: QuantizedWeight) -> tuple:
    return q.codes, q.scales, q.N, q.K, q.group_size, _lib.DTYPE_CODE[q.dtype]


def _native(name: str, q: QuantizedWeight, *args):
    """A call of csrc/native.cpp, which takes plain arguments (the checks, the result and the launch cost 9 us
    interpreted, next to 3.5 of a small product); None: the general path has to take it."""
    if not q.codes.is_cuda:
        return None
    if _lib.native is None:
        _lib.load()
    return getattr(_lib.native, name)(*args, _lib.stream_of(q.codes.device))


def _check_bias(q: QuantizedWeight, bias: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if bias is None:
        return None
    assert tuple(bias.shape) == (q.N,) and bias.dtype == q.dtype, f"bias: {q.N} values of {q.dtype}"
    return bias.contiguous()


def _overlap(out: torch.Tensor, t: Optional[torch.Tensor]) -> bool:
    if t is None or t.numel() == 0 or out.numel() == 0:
        return False
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
    return t.data_ptr() < out.data_ptr() + out.numel() * out.element_size() and out.data_ptr() < t.data_ptr() + last * t.element_size()


def linear(x: torch.Tensor, q: QuantizedWeight, bias: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``F.linear(x.to(q.dtype), W, bias)`` for ``x`` [..., K] of ``q.dtype`` or fp32 (rounded to it),
    any number of rows; the result has ``q.dtype``.  fp32 accumulation in an order that the shapes
    fix, so equal calls give equal bits."""
    if out is None:
        y = _native("w4_linear", q, x, *_fields(q), bias)
        if y is not None:
            return y
    dev = _lib.require_device(x, q.codes, bias, out)
    assert x.dim() >= 1 and x.shape[-1] == q.K, f"x: [..., {q.K}], got {tuple(x.shape)}"
    assert x.dtype in (q.dtype, torch.float32), f"x: {q.dtype} or fp32, got {x.dtype}"
    bias = _check_bias(q, bias)
    rows = x.reshape(-1, q.K)
    M = rows.shape[0]
    if rows.stride(1) != 1:
        rows = rows.contiguous()
    if out is None:
        out = torch.empty(x.shape[:-1] + (q.N,), dtype=q.dtype, device=dev)
    assert tuple(out.shape) == tuple(x.shape[:-1]) + (q.N,) and out.dtype == q.dtype and out.is_contiguous(), \
        "out: contiguous rows of the weights' type"
    assert not _overlap(out, rows) and not _overlap(out, bias), "out must not overlap the inputs (every workgroup reads them)"
    if M == 0 or q.N == 0:
        return out
    lib = _lib.load()
    with torch.cuda.device(dev):
        need = lib.rdkv_w4_linear_workspace_bytes(M, q.N, q.K)
        # (the call's own, so that graphs that hold such calls may replay side by side)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(lib.rdkv_w4_linear(q.codes.data_ptr(), q.scales.data_ptr(), rows.data_ptr(), _lib.DTYPE_CODE[x.dtype],
                                      rows.stride(0), _lib.ptr(bias), M, q.N, q.K, q.group_size, _lib.DTYPE_CODE[q.dtype],
                                      out.data_ptr(), q.N, _lib.ptr(ws), need, _lib.stream_of(dev)))
    return out


def _check_row(q: QuantizedWeight, name: str, t: torch.Tensor) -> None:
    assert t.numel() == q.K and t.dtype == q.dtype and t.stride(-1) == 1 and t.shape[-1] == q.K, \
        f"{name}: one row of {q.K} values of {q.dtype}"


def norm_linear(h: torch.Tensor, delta: Optional[torch.Tensor], norm_weight: torch.Tensor, eps: float,
                q: QuantizedWeight, bias: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Residual add, RMSNorm and product of one row: ``(linear(rms_norm(h + delta), q, bias), h + delta)``,
    one launch.  ``delta`` None: the row is ``h`` itself, which is handed back.  K at most 32768."""
    pair = _native("w4_norm_linear", q, h, delta, norm_weight, eps, *_fields(q), bias)
    if pair is not None:
        return pair
    dev = _lib.require_device(h, delta, norm_weight, q.codes, bias)
    _check_row(q, "h", h)
    if delta is not None:
        _check_row(q, "delta", delta)
    assert norm_weight.dtype == q.dtype and tuple(norm_weight.shape) == (q.K,) and norm_weight.is_contiguous()
    assert q.K <= _MAX_ROW_K, f"rows of {q.K} elements exceed {_MAX_ROW_K}"
    bias = _check_bias(q, bias)
    r = h if delta is None else torch.empty_like(h, memory_format=torch.contiguous_format)
    y = torch.empty(h.shape[:-1] + (q.N,), dtype=q.dtype, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().rdkv_w4_linear_norm(
            _lib.ptr(q.codes), _lib.ptr(q.scales), h.data_ptr(), _lib.ptr(delta), norm_weight.data_ptr(), float(eps),
            None if delta is None else r.data_ptr(), _lib.ptr(bias), q.N, q.K, q.group_size, _lib.DTYPE_CODE[q.dtype],
            _lib.ptr(y), _lib.stream_of(dev)))
    return y, r


def silu_linear(gate: torch.Tensor, up: torch.Tensor, q: QuantizedWeight,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``linear(silu(gate) * up, q, bias)`` of one row, the activation rounded to the type before the product
    with ``up``, one launch.  K at most 32768."""
    y = _native("w4_silu_linear", q, gate, up, *_fields(q), bias)
    if y is not None:
        return y
    dev = _lib.require_device(gate, up, q.codes, bias)
    _check_row(q, "gate", gate)
    _check_row(q, "up", up)
    assert q.K <= _MAX_ROW_K, f"rows of {q.K} elements exceed {_MAX_ROW_K}"
    bias = _check_bias(q, bias)
    y = torch.empty(gate.shape[:-1] + (q.N,), dtype=q.dtype, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().rdkv_w4_linear_silu(_lib.ptr(q.codes), _lib.ptr(q.scales), gate.data_ptr(), up.data_ptr(),
                                                   _lib.ptr(bias), q.N, q.K, q.group_size, _lib.DTYPE_CODE[q.dtype],
                                                   _lib.ptr(y), _lib.stream_of(dev)))
    return y
