"""Rotary positions of queries and keys, in front of the attention over packed rows (`parallel_moba`) and over pages (`paged_append`).

The reference's operator takes queries and keys that are turned already (benchmarks/moba_compare.py draws them at random).  A table
holds, for each pair of dims, the part of a whole turn that one position makes, in 64 bits of fixed point: angles of far positions lose
nothing.  include/moba_b200.h has the rules in full.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from fractions import Fraction
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .paged import _check_written, _run_on, _written
from .parallel import HEAD_DIMS

__all__ = ["RotaryTable", "rotary", "rotary_frequencies"]

#: 2 ** 160 units of a turn in a radian
_PER_RADIAN = round(2 ** 160 / (2 * Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)))
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
#: struct moba_rotary, field by field (filling a ctypes structure by name takes ten times as long)
_CALL = struct.Struct("@q8ifi8q")
assert _CALL.size == C.sizeof(_lib.Rotary)


def _turns(x: float) -> int:
    """x radians as a part of a turn in units of 2 ** -64, whole turns dropped, as a signed 64-bit number."""
    m, e = math.frexp(x)
    n, shift = int(m * 2 ** 53) * _PER_RADIAN, 149 - e       # x = m * 2 ** 53 * 2 ** (e - 53)
    n = ((n + (1 << (shift - 1))) >> shift if shift > 0 else n << -shift) % 2 ** 64
    return n - 2 ** 64 if n >= 2 ** 63 else n


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                       original: Optional[int] = None, fast: float = 32.0, slow: float = 1.0) -> torch.Tensor:
    """Radians that a position turns each of rotary_dim / 2 pairs by: base ** (-2 j / rotary_dim), float64 on the CPU.  `scaling` for contexts
    `factor` times as long as those the model was trained on:

        "linear"  every frequency divided by the factor
        "base"    the base times factor ** (rotary_dim / (rotary_dim - 2)): the slowest pair is divided by the factor, the fastest stays
        "parts"   pairs that turn `fast` times or more within the `original` context stay, those that turn `slow` times or less are divided by the
                  factor; of those between a part stays that is linear in their turns, (original f / (2 pi) - slow) / (fast - slow): f times
                  the part, and f / factor times the rest.  (Another rule in use is linear in the pair's index: its frequencies go to
                  `RotaryTable` as they are.)"""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even int, got {rotary_dim}")
    if scaling not in ("none", "linear", "base", "parts"):
        raise ValueError(f"scaling must be none, linear, base or parts, got {scaling}")
    if not (base > 0 and factor > 0):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling by the base needs two pairs")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = torch.tensor([base ** (-j / rotary_dim) for j in range(0, rotary_dim, 2)], dtype=torch.float64)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        if original is None or original <= 0 or not fast > slow:
            raise ValueError(f"scaling by parts needs the original context and fast > slow, got {original}, {fast} and {slow}")
        stay = ((original * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * stay + f / factor * (1 - stay)
    return f


class RotaryTable:
    """What `rotary` turns by, kept for all layers and calls: `frequencies`, radians a position for each pair (rotary_dim / 2 of them: see
    `rotary_frequencies`); `interleaved`: pairs are dims 2 j and 2 j + 1, else j and j + rotary_dim / 2; `magnitude`: factor of the turned dims."""

    def __init__(self, frequencies: torch.Tensor, *, interleaved: bool = False, magnitude: float = 1.0, device: Optional[torch.device] = None):
        f = torch.as_tensor(frequencies, dtype=torch.float64).detach().cpu()
        if f.ndim != 1 or f.numel() == 0:
            raise ValueError(f"frequencies must have shape [rotary_dim / 2], got {tuple(f.shape)}")
        radians = f.tolist()
        if not all(map(math.isfinite, radians)):
            raise ValueError("frequencies must be finite")
        if not 0.0 < C.c_float(float(magnitude)).value <= 3.0e38:
            raise ValueError(f"magnitude must be a positive number of 32 bits, got {magnitude}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.rotary_dim, self.interleaved, self.magnitude = 2 * f.numel(), bool(interleaved), float(magnitude)
        self.turns = torch.tensor([_turns(x) for x in radians], dtype=torch.int64).to(device)
        self.index = self.turns.get_device()


def _check_rotary(q, k, positions, table) -> None:
    for name, x in (("q", q), ("k", k)):
        if x is None:
            continue
        if x.ndim != 3:
            raise ValueError(f"{name} must have shape [tokens, heads, head_dim], got {tuple(x.shape)}")
        if x.shape[0] != q.shape[0] or x.shape[2] != q.shape[2] or x.shape[1] == 0:
            raise ValueError(f"q and k must have the same token count and head dimension, and heads, got {tuple(q.shape)} and {tuple(x.shape)}")
        if x.dtype not in _DTYPES:
            raise TypeError(f"only float16 and bfloat16 are supported, got {x.dtype}")
        if x.dtype != q.dtype:
            raise TypeError("q and k must have the same dtype")
        if x.get_device() < 0 or x.get_device() != q.get_device():
            raise ValueError("q and k must be accelerator tensors on the same device")
        if x.stride(2) != 1:
            raise NotImplementedError(f"{name} must be contiguous in its last dimension")
    if q.shape[2] not in HEAD_DIMS:
        raise NotImplementedError(f"this build supports head_dim {HEAD_DIMS} only")
    if table.rotary_dim > q.shape[2]:
        raise ValueError(f"the table turns {table.rotary_dim} dims, head_dim is {q.shape[2]}")
    if positions.shape != (q.shape[0],):
        raise ValueError(f"positions must have shape [{q.shape[0]}], got {tuple(positions.shape)}")
    if positions.dtype != torch.int32 or positions.get_device() != q.get_device() or table.index != q.get_device():
        raise TypeError("positions must be an int32 tensor, and the table, on the device of q")
    if q.shape[0] > 1 and positions.stride(0) != 1:
        raise NotImplementedError("positions must be contiguous")


def _strides(x) -> Tuple[int, int]:
    """Of tokens and heads (one token or head may have any: it is never stepped over)."""
    (tokens, heads, _), (t, h, _) = x.shape, x.stride()
    return t if tokens > 1 else 0, h if heads > 1 else 0


def _turn(q, k, positions, table, inverse, out=None):
    """(q, k) turned, in `out` or in new tensors; looks at q, k, positions and the table first, each attribute once."""
    shape, index, dtype = q.shape, q.get_device(), q.dtype
    good = len(shape) == 3 and index >= 0 and dtype in _DTYPES
    if good:
        tokens, heads, dim = shape
        qt, qh, qd = q.stride()
        good = (qd == 1 and heads > 0 and dim in HEAD_DIMS and table.rotary_dim <= dim and positions.shape == (tokens,)
                and positions.dtype == torch.int32 and positions.get_device() == index and table.index == index
                and (tokens < 2 or positions.stride(0) == 1))
        ks, heads_k = (0, 0), 0
        if good and k is not None:
            other = k.shape
            good = len(other) == 3 and other[0] == tokens and other[2] == dim and other[1] > 0 and k.dtype == dtype and k.get_device() == index
            if good:
                heads_k, (kt, kh, kd) = other[1], k.stride()
                good, ks = kd == 1, (kt if tokens > 1 else 0, kh if heads_k > 1 else 0)
    if not good:
        _check_rotary(q, k, positions, table)
        raise ValueError("q, k, positions and the table do not describe a call")
    if out is None:
        device = q.device
        out = (torch.empty(shape, dtype=dtype, device=device), None if k is None else torch.empty(other, dtype=dtype, device=device))
        strides = (heads * dim, dim, heads_k * dim, dim)
    else:
        _check_out(q, k, out)
        strides = (*_strides(out[0]), *((0, 0) if k is None else _strides(out[1])))
    if tokens > 0:
        call = _CALL.pack(tokens, heads, heads_k, dim, table.rotary_dim, table.interleaved, inverse, _DTYPES[dtype], 0, table.magnitude, 0,
                          qt if tokens > 1 else 0, qh if heads > 1 else 0, *ks, *strides)
        qo, ko = out
        _run_on(index, _lib.lib().moba_rotary, call, q.data_ptr(), None if k is None else k.data_ptr(), positions.data_ptr(), table.turns.data_ptr(),
                qo.data_ptr(), None if k is None else ko.data_ptr())
    return out


def _check_out(q, k, out) -> None:
    qo, ko = out
    if (k is None) != (ko is None):
        raise ValueError("out must have a tensor for each of q and k")
    for name, x, y in (("out[0]", q, qo), ("out[1]", k, ko)):
        if x is None or x is y:
            continue
        if y.shape != x.shape or y.dtype != x.dtype or y.get_device() != x.get_device():
            raise ValueError(f"{name} must have the shape, dtype and device of what is turned")
        if y.stride(2) != 1:
            raise NotImplementedError(f"{name} must be contiguous in its last dimension")
    _check_written(qo, ko)


def _kernel_rows(x):
    """A gradient or tangent as the kernel takes it: whatever autograd makes of it is not the caller's to lay out."""
    t, h, d = x.stride()
    return x if d == 1 and not (t | h) & 7 and not x.data_ptr() & 15 else x.clone(memory_format=torch.contiguous_format)


class _Rotary(torch.autograd.Function):
    """The operator is linear: its gradient is the turn back, its tangent the turn itself, and both may be differentiated again."""

    @staticmethod
    def forward(ctx, q, k, positions, table, inverse):
        qo, ko = _turn(q, k, positions, table, inverse)
        ctx.save_for_backward(positions)
        ctx.table, ctx.inverse, ctx.alone = table, inverse, k is None
        ctx.set_materialize_grads(False)
        if getattr(forward_ad, "_current_level", 0) >= 0:
            ctx.save_for_forward(positions)
            ctx.like = tuple((x.shape, x.dtype, x.device) for x in (q, k) if x is not None)
        return qo if k is None else (qo, ko)

    @staticmethod
    def _each(ctx, tensors, inverse):
        """Each of (dq, dk) turned; what is None stays None."""
        positions, = ctx.saved_tensors
        given = [None if x is None else _kernel_rows(x) for x in tensors]
        if all(x is None for x in given):
            return given
        if not torch.is_grad_enabled() and getattr(forward_ad, "_current_level", 0) < 0:
            if len(given) == 2 and given[0] is not None and given[1] is not None:
                return list(_turn(*given, positions, ctx.table, inverse))
            return [None if x is None else _turn(x, None, positions, ctx.table, inverse)[0] for x in given]
        if len(given) == 2 and given[0] is not None and given[1] is not None:
            return list(_Rotary.apply(given[0], given[1], positions, ctx.table, inverse))
        return [None if x is None else _Rotary.apply(x, None, positions, ctx.table, inverse) for x in given]

    @staticmethod
    def backward(ctx, *grads):
        wanted = [g if need else None for g, need in zip(grads, ctx.needs_input_grad)]
        dq, *dk = _Rotary._each(ctx, wanted, not ctx.inverse)
        return dq, dk[0] if dk else None, None, None, None

    @staticmethod
    def jvp(ctx, dq, dk, *_):
        tangents = [dq] if ctx.alone else [dq, dk]
        tangents = [torch.zeros(s, dtype=t, device=d) if x is None else x for x, (s, t, d) in zip(tangents, ctx.like)]
        got = _Rotary._each(ctx, tangents, ctx.inverse)
        return got[0] if ctx.alone else tuple(got)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, table: RotaryTable, *,
           out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None):
    """Queries q [T, Hq, D] and keys k [T, Hkv, D] turned to positions [T] (int32; `paged_reserve` gives them): the first table.rotary_dim dims of
    each head, rounded once; the others, and rows with a position below 0, are copied.  k may be None.

    Returns (q, k) turned, as new tensors, or written to `out`, which may be (q, k) themselves; tensors that lie on them otherwise are not
    allowed.  Gradients of both orders, and forward derivatives, are followed (not with `out`)."""
    followed = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
    if not followed and getattr(forward_ad, "_current_level", 0) >= 0:
        followed = any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in (q, k))
    if out is None:
        if not followed:
            return _turn(q, k, positions, table, False)
        got = _Rotary.apply(q, k, positions, table, False)
        return (got, None) if k is None else got
    if followed:
        raise NotImplementedError("out is for rows that autograd does not follow")
    _turn(q, k, positions, table, False, out)
    _written(*out)
    return out
