"""Sampling of the next token: temperature, top-k, top-p and min-p over rows of logits, from given
uniform random numbers.

The reference decodes greedily (obkv_accel/fast_decode.py:1827); ``sample_tokens`` stands beside that
choice for programs that sample, and ``fast_decode.greedy_decode_fast(..., sampling=...)`` takes
its tokens this way, inside the captured step too.  Random numbers are an argument: the same
numbers give the same tokens, whatever the batch and the launch.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib

Setting = Union[float, int, torch.Tensor]


@dataclass(frozen=True)
class Sampling:
    """Settings of one decode loop.  ``temperature`` not above 0: the largest logit; ``top_k`` 0, ``top_p`` 1 and
    ``min_p`` 0 are off."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


def _check_value(name: str, v: Setting) -> None:
    assert not math.isnan(v), f"{name} is NaN"
    if name == "top_k":
        assert v == int(v) and v < 1 << 31, f"top_k: a whole number below 2^31, got {v}"
    elif name in ("top_p", "min_p"):
        assert 0.0 <= v <= 1.0, f"{name}: between 0 and 1, got {v}"


def _settings(dev: torch.device, rows: int, temperature: Setting, top_k: Setting, top_p: Setting, min_p: Setting):
    """The library's settings, and the tensors that they point to."""
    s, held = _lib.RdkvSampling(), []
    for name, v in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        if torch.is_tensor(v):
            assert v.device == dev, f"{name}: on {v.device}, the logits on {dev}"
            assert tuple(v.shape) == (rows,), f"{name}: one value per row ({rows}), got {tuple(v.shape)}"
            if name == "top_k":
                assert not v.dtype.is_floating_point and v.dtype != torch.bool, f"top_k: integers, got {v.dtype}"
                v = v if v.dtype == torch.int32 else v.clamp(0, (1 << 31) - 1).to(torch.int32)
            else:
                v = v.to(torch.float32)
            v = v.contiguous()
            held.append(v)
            setattr(s, name, _lib.ptr(v))
        else:
            _check_value(name, v)
            setattr(s, name + "_value", max(int(v), 0) if name == "top_k" else float(v))
    return s, held


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens (int64) and their log probabilities (fp32) for ``logits`` [..., vocab] (fp16 / bf16 / fp32) and
    ``uniform`` [...] (fp32 in [0, 1)), one number per row.

    Per row, with ``w = exp((logit - max) / temperature)`` and the tokens in descending order (equal logits by
    index): ``top_k`` > 0 keeps the first so many; ``top_p`` < 1 keeps, of those, the shortest run from the front
    whose sum reaches ``top_p`` of theirs; ``min_p`` > 0 keeps the tokens with ``w >= min_p``; the first token always
    stays.  The token is the first one whose running sum exceeds ``uniform`` times the sum of what stays, the log
    probability its share of that sum.  A ``temperature`` that is not above 0 takes the largest logit (log probability
    0).  Each setting is a number or a tensor with one value per row, on the logits' device (and not looked
    at by the host: values out of range act as the nearest one in range, NaN as off).  NaN and -inf logits are masked, +inf
    counts as the largest number of fp32; a row with nothing left has token -1 and log probability -inf."""
    if logits.is_cuda:              # plain arguments: csrc/native.cpp (the checks and the launch cost 27 us interpreted)
        if _lib.native is None:
            _lib.load()
        pair = _lib.native.sample_rows(logits, uniform, temperature, top_k, top_p, min_p, _lib.stream_of(logits.device))
        if pair is not None:
            return pair
    dev = _lib.require_device(logits, uniform)
    assert logits.dim() >= 1 and logits.dtype in _lib.DTYPE_CODE, f"logits: fp32, fp16 or bf16, got {logits.dtype}"
    shape, vocab = logits.shape[:-1], logits.shape[-1]
    assert 1 <= vocab <= 1 << 24, f"a vocabulary of {vocab}"
    assert uniform.dtype == torch.float32 and uniform.shape == shape, \
        f"uniform: fp32 {tuple(shape)}, got {uniform.dtype} {tuple(uniform.shape)}"
    rows = logits.reshape(-1, vocab)
    if rows.stride(1) != 1 or rows.stride(0) < 0:
        rows = rows.contiguous()
    B = rows.shape[0]
    token = torch.empty(shape, dtype=torch.int64, device=dev)
    logprob = torch.empty(shape, dtype=torch.float32, device=dev)
    flat = lambda v: v.reshape(-1) if torch.is_tensor(v) and v.shape == shape else v  # noqa: E731
    with torch.cuda.device(dev):
        s, held = _settings(dev, B, flat(temperature), flat(top_k), flat(top_p), flat(min_p))
        if B == 0:
            return token, logprob
        uniform = uniform.contiguous()
        lib = _lib.load()
        need = lib.rdkv_sample_workspace_bytes(B, vocab, _lib.DTYPE_CODE[rows.dtype])
        # (the call's own, so that graphs that hold such calls may replay side by side)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(lib.rdkv_sample_rows(rows.data_ptr(), rows.stride(0), B, vocab, _lib.DTYPE_CODE[rows.dtype],
                                        uniform.data_ptr(), ctypes.addressof(s), token.data_ptr(), logprob.data_ptr(),
                                        _lib.ptr(ws), need, _lib.stream_of(dev)))
    return token, logprob


def _sample_advance(logits: torch.Tensor, token: torch.Tensor, sampling: Sampling, uniforms: torch.Tensor,
                    position: torch.Tensor, write_row: torch.Tensor, n_new: Optional[torch.Tensor] = None,
                    word: Optional[_lib.StepWord] = None) -> None:
    """``fast_decode._argmax_advance`` with a sampled token: ``token <- `` the choice for the one row of
    ``logits`` with ``uniforms[write_row]``, then the counters advanced by one."""
    dev = _lib.require_device(logits, token, uniforms, position, write_row, n_new)
    row = logits.reshape(-1)
    assert row.is_contiguous() and row.dtype in _lib.DTYPE_CODE
    for t in (token, position, write_row):
        assert t.dtype == torch.int64 and t.numel() == 1
    assert uniforms.dtype == torch.float32 and uniforms.is_contiguous() and uniforms.numel() >= 1
    assert n_new is None or (n_new.dtype == torch.int32 and n_new.is_contiguous() and n_new.numel() <= 1024)
    lib = _lib.load()
    with torch.cuda.device(dev):
        s, _ = _settings(dev, 1, sampling.temperature, sampling.top_k, sampling.top_p, sampling.min_p)
        need = lib.rdkv_sample_workspace_bytes(1, row.numel(), _lib.DTYPE_CODE[row.dtype])
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(lib.rdkv_sample_advance(
            row.data_ptr(), row.numel(), _lib.DTYPE_CODE[row.dtype], uniforms.data_ptr(), uniforms.numel(),
            write_row.data_ptr(), ctypes.addressof(s), token.data_ptr(), position.data_ptr(), write_row.data_ptr(),
            _lib.ptr(n_new), 0 if n_new is None else n_new.numel(), word.ptr if word is not None else None,
            word.tag_base if word is not None else 0, _lib.ptr(ws), need, _lib.stream_of(dev)))
