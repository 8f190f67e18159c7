"""Drafted tokens checked against the target's probabilities.

A server that drafts tokens attends to a tree of them in one call (`paged_attention` with `parents`), has the target's probabilities behind each of its rows
from that, and keeps a branch of it such that the tokens are distributed as the target's own.  No counterpart in the reference, which
samples nothing.  include/moba_b200.h has the rules in full.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .paged import _check_parents, _i32_rows, _run_on

__all__ = ["verify_drafts"]

_DTYPES = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_TOKEN_BITS = {torch.int32: 32, torch.int64: 64}
#: struct moba_drafts, field by field
_CALL = struct.Struct("@2q4i3q")
assert _CALL.size == C.sizeof(_lib.Drafts)


def _check_drafts(target, draft, tokens, cu_seqlens, accept, sample, max_new) -> None:
    if target.ndim != 2 or target.shape[1] == 0:
        raise ValueError(f"target must have shape [tokens, vocabulary], got {tuple(target.shape)}")
    if target.dtype not in _DTYPES:
        raise TypeError(f"probabilities are float32, bfloat16 or float16, got {target.dtype}")
    index = target.get_device()
    if index < 0:
        raise ValueError("target must be an accelerator tensor")
    rows = target.shape[0]
    for name, x in (("target", target), ("draft", draft)):
        if x is None:
            continue
        if x.shape != target.shape:
            raise ValueError(f"draft must have the shape of target, {tuple(target.shape)}, got {tuple(x.shape)}")
        if x.dtype != target.dtype or x.get_device() != index:
            raise TypeError("draft must have target's dtype and device")
        if x.stride(1) != 1 and x.shape[1] > 1:
            raise NotImplementedError(f"{name} must be contiguous in its last dimension")
    if tokens.shape != (rows,):
        raise ValueError(f"tokens must have shape [{rows}], got {tuple(tokens.shape)}")
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.get_device() != index:
        raise TypeError("tokens must be an int32 or int64 tensor on target's device")
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be a one-dimensional tensor of length >= 2")
    _i32_rows("cu_seqlens", cu_seqlens, cu_seqlens.shape, index)
    for name, x, shape in (("accept", accept, (rows,)), ("sample", sample, (cu_seqlens.numel() - 1,))):
        if x.shape != shape:
            raise ValueError(f"{name} must have shape {list(shape)}, got {list(x.shape)}")
        if x.dtype != torch.float32 or x.get_device() != index:
            raise TypeError(f"{name} must be a float32 tensor on target's device")
    for name, x in (("tokens", tokens), ("accept", accept), ("sample", sample)):
        if x.shape[0] > 1 and x.stride(0) != 1:
            raise NotImplementedError(f"{name} must be contiguous")
    if not isinstance(max_new, int) or max_new <= 0:
        raise ValueError(f"max_new must be a positive int, got {max_new}")
    if max_new > 1024:
        raise NotImplementedError(f"at most 1024 packed tokens of a sequence, got max_new = {max_new}")
    if target.shape[1] > 2 ** 22:
        raise NotImplementedError(f"vocabularies of at most 2**22 tokens, got {target.shape[1]}")


def verify_drafts(target: torch.Tensor, draft: Optional[torch.Tensor], tokens: torch.Tensor, cu_seqlens: torch.Tensor,
                  accept: torch.Tensor, sample: torch.Tensor, max_new: int, *,
                  parents: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens stand, and the token behind them.  The packed rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 are a tree (`parents` as
    in `paged_attention`; without it each row follows the one before): row 0 is the last accepted token, the others are drafted ones.

    `target`, `draft` [T, V] (float32, bfloat16 or float16): the target's and the draft's probabilities of the token behind each row; a row's children
    were drawn from its `draft` one by one.  draft = None: children are given tokens, such as the draft's likeliest.  `tokens` [T] int32 or int64,
    `accept` [T] and `sample` [batch] float32: random numbers from [0, 1), for each drafted row and each sequence.  `max_new`: the most rows of a
    sequence, at most 1024; rows beyond are not looked at.

    A child with token x of row r is accepted where accept * draft[r, x] < target[r, x]; after one that is not, its siblings are tried against what is
    left, max(target[r] - draft[r], 0) over its sum (draft = None: target[r] without x over 1 - target[r, x]: its rows are taken to add up to 1), and so on;
    the walk goes on from an accepted one.
    The next token is drawn from what is left of the last row's target by `sample`.

    Returns (path, count, next): path int32 [batch, max_new], the accepted rows counted from the sequence's first (row 0 among them), -1 behind
    them; count int32 [batch]; next [batch] of tokens' dtype.  A sequence without rows has 0 and -1; a next token of -1 else means that the row's
    probabilities are all zeros.  Computed in 64 bits; values that are not above 0 and finite count as 0."""
    # each attribute is read once: this runs in every step of a server
    shape, dtype, index, token = target.shape, target.dtype, target.get_device(), tokens.dtype
    good = len(shape) == 2 and index >= 0 and dtype in _DTYPES and token in _TOKEN_BITS and isinstance(max_new, int) and 0 < max_new <= 1024
    if good:
        (rows, vocabulary), (ts, t1), i32, f32, ds = shape, target.stride(), torch.int32, torch.float32, 0
        batch = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else 0
        good = (0 < vocabulary <= 2 ** 22 and (t1 == 1 or vocabulary == 1) and batch > 0 and cu_seqlens.dtype == i32 and cu_seqlens.get_device() == index
                and cu_seqlens.stride(0) == 1 and tokens.shape == (rows,) and tokens.get_device() == index and tokens.is_contiguous()
                and accept.shape == (rows,) and accept.dtype == f32 and accept.get_device() == index and accept.is_contiguous()
                and sample.shape == (batch,) and sample.dtype == f32 and sample.get_device() == index and sample.is_contiguous())
        if good and draft is not None:
            ds, d1 = draft.stride() if draft.dim() == 2 else (0, 0)
            good = draft.shape == shape and draft.dtype == dtype and draft.get_device() == index and (d1 == 1 or vocabulary == 1)
    if not good:
        _check_drafts(target, draft, tokens, cu_seqlens, accept, sample, max_new)
        raise ValueError("target, draft, tokens, cu_seqlens, accept and sample do not describe a call")
    if parents is not None:
        _check_parents(parents, rows, index)
    for x in (target, draft, accept, sample):
        if x is not None and ((x.requires_grad and torch.is_grad_enabled())
                              or (getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(x).tangent is not None)):
            raise NotImplementedError("whole numbers have no derivatives: verify_drafts takes no tensors that autograd follows")
    path = torch.empty((batch, max_new), dtype=i32, device=target.device)
    count, following = torch.empty(batch, dtype=i32, device=target.device), torch.empty(batch, dtype=token, device=target.device)
    if rows == 0:
        return path.fill_(-1), count.zero_(), following.fill_(-1)
    call = _CALL.pack(rows, vocabulary, batch, max_new, _DTYPES[dtype], _TOKEN_BITS[token], ts if rows > 1 else 0, ds if rows > 1 else 0, 0)
    _run_on(index, _lib.lib().moba_verify_drafts, call, target.data_ptr(), None if draft is None else draft.data_ptr(), tokens.data_ptr(),
            cu_seqlens.data_ptr(), None if parents is None else parents.data_ptr(), accept.data_ptr(), sample.data_ptr(), path.data_ptr(),
            count.data_ptr(), following.data_ptr())
    return path, count, following
