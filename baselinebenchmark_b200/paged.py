"""Keys and values of many sequences in pages: written, read back and attended to.

The reference's operator takes whole packed sequences and keeps nothing between calls (backends/_mthreads/ops/moba/parallel.py:253-374);
`IncrementalMoba` keeps one sequence in a cache of its own.  A server has many, of any length: their rows live in one pool of pages,
in 16 bits or quantised to 8, and a call concerns a packed batch of new tokens.

    k_pages, v_pages   [pages, page_size, Hkv, D]: bfloat16, float16, float8_e4m3fn or int8, any strides with a contiguous last
                       dimension (head-major pages read fastest: see `PagedKV`); page_size a power of two, at least 16
    k_scales, v_scales [pages, Hkv, page_size] uint8, for 8-bit pages: a code c with byte s stands for c * 2**(s - 127)
    page_table         int32 [batch, pages of a sequence]: position x is slot x % page_size of page page_table[b, x // page_size];
                       an entry that is no page's number is a page that is not there
    cu_seqlens         int32 [batch + 1]: sequence b has the packed rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, its last tokens
    seq_lens           int32 [batch]: its tokens, the packed ones included

All of them stay on the device; nothing is read back to the host, so that calls may be captured in a CUDA graph and replayed
with other numbers in the same tensors.  include/moba_b200.h has the rules in full.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .parallel import HEAD_DIMS, _workspace

__all__ = ["PagedKV", "PagePool", "paged_store", "paged_load", "paged_attention", "paged_append", "paged_keep", "paged_reserve", "paged_release"]

_STORES = {torch.float8_e4m3fn: _lib.STORE_E4M3, torch.int8: _lib.STORE_INT8}
_ROWS = (torch.float16, torch.bfloat16)


def _check_pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales) -> None:
    shape, dtype, dev = k_pages.shape, k_pages.dtype, k_pages.device
    if len(shape) != 4:
        raise ValueError("k_pages and v_pages must have shape [pages, page_size, heads, head_dim]")
    if shape != v_pages.shape:
        raise ValueError(f"k_pages and v_pages must have identical shapes, got {shape} and {v_pages.shape}")
    if dtype != v_pages.dtype:
        raise TypeError("k_pages and v_pages must have the same dtype")
    if dtype not in _STORES and dtype not in _ROWS:
        raise TypeError(f"pages hold float16, bfloat16, float8_e4m3fn or int8, got {dtype}")
    if 0 in shape:
        raise ValueError("k_pages and v_pages dimensions must be non-zero")
    if dev.type != "cuda" or v_pages.device != dev:
        raise ValueError("k_pages and v_pages must be accelerator tensors on the same device")
    if shape[1] < 16 or shape[1] & (shape[1] - 1):
        raise NotImplementedError(f"page_size must be a power of two and at least 16, got {shape[1]}")
    if shape[3] not in HEAD_DIMS:
        raise NotImplementedError(f"this build supports head_dim {HEAD_DIMS} only")
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        if x.stride(3) != 1:
            raise NotImplementedError(f"{name} must be contiguous in its last dimension")
    if dtype in _STORES:
        want = (shape[0], shape[2], shape[1])
        for name, x in (("k_scales", k_scales), ("v_scales", v_scales)):
            if x is None or x.shape != want or x.dtype != torch.uint8 or x.device != dev or not x.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 tensor of shape {want} on the pages' device")
    elif k_scales is not None or v_scales is not None:
        raise ValueError("pages of 16-bit rows have no scales")
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be a one-dimensional tensor of length >= 2")
    batch = cu_seqlens.numel() - 1
    if page_table.ndim != 2 or page_table.shape[0] != batch or page_table.shape[1] == 0:
        raise ValueError(f"page_table must have shape [{batch}, pages of a sequence], got {tuple(page_table.shape)}")
    if seq_lens.shape != (batch,):
        raise ValueError(f"seq_lens must have shape [{batch}], got {tuple(seq_lens.shape)}")
    for name, x in (("cu_seqlens", cu_seqlens), ("seq_lens", seq_lens), ("page_table", page_table)):
        if x.device != dev or x.dtype != torch.int32:
            raise TypeError(f"{name} must be an int32 tensor on the pages' device")
        if x.stride(-1) != 1 and x.shape[-1] > 1:
            raise NotImplementedError(f"{name} must be contiguous in its last dimension")


def _check_rows(name, x, k_pages, heads: Optional[int], tokens: Optional[int]) -> None:
    if x.ndim != 3 or x.shape[2] != k_pages.shape[3] or (heads is not None and x.shape[1] != heads) \
            or (tokens is not None and x.shape[0] != tokens):
        raise ValueError(f"{name} must have shape [tokens, heads, head_dim] in line with the pages {tuple(k_pages.shape)}, "
                         f"got {tuple(x.shape)}")
    if x.dtype not in _ROWS:
        raise TypeError(f"only float16 and bfloat16 are supported, got {x.dtype}")
    if k_pages.dtype in _ROWS and x.dtype != k_pages.dtype:
        raise TypeError(f"{name} must have the dtype of the pages, {k_pages.dtype}, got {x.dtype}")
    if x.device != k_pages.device:
        raise ValueError(f"{name} must be on the pages' device")
    if x.shape[1] == 0:
        raise ValueError(f"{name} must have heads")
    if x.stride(2) != 1:
        raise NotImplementedError(f"{name} must be contiguous in its last dimension")
    if x.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} requires grad: a paged cache is state of a server, its operators have no backward")


#: struct moba_paged, field by field (filling a ctypes structure by name takes ten times as long)
_PAGED = struct.Struct("@q10ifi15q")
assert _PAGED.size == C.sizeof(_lib.Paged)
_STORE_OF = {torch.bfloat16: _lib.STORE_SAME, torch.float16: _lib.STORE_SAME, **_STORES}
_DTYPE_OF = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}


class _Pages:
    """The tensors that describe a call, checked, with what the C structure needs of them; each attribute is read once, because this
    runs on every call of a decode step."""
    __slots__ = ("index", "shape", "dtype", "store", "batch", "per_seq", "strides", "where")

    def __init__(self, k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales):
        shape, dtype, index = k_pages.shape, k_pages.dtype, k_pages.get_device()
        store, table, cu, i32 = _STORE_OF.get(dtype), page_table.shape, cu_seqlens.shape, torch.int32
        good = (index >= 0 and store is not None and len(shape) == 4 == len(v_pages.shape) and len(table) == 2 and len(cu) == 1)
        if good:
            (pages, size, heads, dim), batch = shape, cu[0] - 1
            (kp, kt, kh, kd), (vp, vt, vh, vd), (ts, td) = k_pages.stride(), v_pages.stride(), page_table.stride()
            per_seq = table[1]
            good = (kd == 1 == vd and v_pages.shape == shape and v_pages.dtype == dtype and v_pages.get_device() == index
                    and dim in HEAD_DIMS and size >= 16 and not size & (size - 1) and pages > 0 and heads > 0 and batch > 0
                    and table[0] == batch and per_seq > 0 and (td == 1 or per_seq == 1) and seq_lens.shape == (batch,)
                    and page_table.dtype == i32 and cu_seqlens.dtype == i32 and seq_lens.dtype == i32
                    and page_table.get_device() == index and cu_seqlens.get_device() == index and seq_lens.get_device() == index
                    and cu_seqlens.stride(0) == 1 and (batch == 1 or seq_lens.stride(0) == 1))
            if store == _lib.STORE_SAME:
                good = good and k_scales is None and v_scales is None
            elif good:
                want = (pages, heads, size)
                good = (k_scales is not None and v_scales is not None and k_scales.shape == want and v_scales.shape == want
                        and k_scales.dtype == torch.uint8 == v_scales.dtype and k_scales.get_device() == index
                        and v_scales.get_device() == index and k_scales.is_contiguous() and v_scales.is_contiguous())
        if not good:
            _check_pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
            raise ValueError("k_pages, v_pages, page_table, cu_seqlens and seq_lens do not describe a paged cache")
        # a dimension of one page or head may have any stride: it is never stepped over
        if pages == 1:
            kp = vp = heads * size * dim
        if heads == 1:
            kh = vh = size * dim
        self.index, self.shape, self.dtype, self.store, self.batch, self.per_seq = index, shape, dtype, store, batch, per_seq
        self.strides = (kp, kt, kh, vp, vt, vh, ts if batch > 1 else per_seq)
        # as the C calls take them
        self.where = (cu_seqlens.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                      None if k_scales is None else k_scales.data_ptr(), None if v_scales is None else v_scales.data_ptr())

    def pack(self, tokens, q_heads, max_new, dtype, scale, q=(0, 0), o=(0, 0), k=(0, 0), v=(0, 0)) -> bytes:
        pages, size, heads, dim = self.shape
        try:
            return _PAGED.pack(tokens, self.batch, q_heads, heads, dim, pages, size, self.per_seq, min(max_new, 0x7fffffff), _DTYPE_OF[dtype],
                               self.store, scale, 0, *q, *o, *k, *v, *self.strides)
        except struct.error as e:
            raise NotImplementedError("pages, columns of the table and sequences are counted in 32 bits") from e

    def run(self, call, *args) -> None:
        """`call(*args, stream)` with the pages' device current."""
        index = self.index
        if index != torch.cuda.current_device():
            with torch.cuda.device(index):
                _lib.check(call(*args, torch._C._cuda_getCurrentRawStream(index)))
        else:
            _lib.check(call(*args, torch._C._cuda_getCurrentRawStream(index)))


def _rows(name, x, g: _Pages, heads: Optional[int], tokens: Optional[int], k_pages) -> Tuple[int, int]:
    """A packed tensor, checked; its strides of tokens and heads (one token or head may have any, it is never stepped over)."""
    shape, dtype, (t, h, d) = x.shape, x.dtype, x.stride() if x.dim() == 3 else (0, 0, 0)
    if not (d == 1 and shape[2] == g.shape[3] and shape[1] > 0 and (heads is None or shape[1] == heads) and (tokens is None or shape[0] == tokens)
            and dtype in _DTYPE_OF and (g.store != _lib.STORE_SAME or dtype == g.dtype) and x.get_device() == g.index
            and not (x.requires_grad and torch.is_grad_enabled())):
        _check_rows(name, x, k_pages, heads, tokens)
    return t if shape[0] > 1 else 0, h if shape[1] > 1 else 0


def _check_not_followed(**tensors) -> None:
    """Nothing here has a backward or a forward derivative: what autograd follows is refused, not dropped."""
    if torch.is_grad_enabled():
        for name, x in tensors.items():
            if x is not None and x.requires_grad:
                raise NotImplementedError(f"{name} requires grad: a paged cache is state of a server, its operators have no backward")
    if getattr(forward_ad, "_current_level", 0) >= 0:        # (-1: outside of forward mode, where a look at each tensor is saved)
        for name, x in tensors.items():
            if x is not None and forward_ad.unpack_dual(x).tangent is not None:
                raise NotImplementedError(f"{name} has a tangent: the operators of a paged cache have no derivatives")


def _check_written(*tensors) -> None:
    inference = torch.is_inference_mode_enabled()
    for x in tensors:
        if x is not None:
            if not inference and x.is_inference():
                raise RuntimeError("tensors made in inference mode can only be written in inference mode")
            if x.requires_grad:
                raise NotImplementedError("tensors that require grad cannot be written")


def _written(*tensors) -> None:
    """As after an in-place torch operation: what autograd saved of them is stale."""
    torch.autograd.graph.increment_version([x for x in tensors if x is not None and not x.is_inference()])


def paged_store(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, *, k_scales: Optional[torch.Tensor] = None,
                v_scales: Optional[torch.Tensor] = None) -> None:
    """Writes the packed rows k, v [T, Hkv, D] into the pages of their sequences; 8-bit pages are quantised to, each row
    and head with a power of two of its own.  Rows behind the last sequence, and rows whose page is not there, are not written.
    A slot that two rows of a call are for (a page in two sequences' tables) is undefined."""
    g = _Pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    heads, tokens = g.shape[2], k.shape[0] if k.dim() else None
    ks = _rows("k", k, g, heads, None, k_pages)
    vs = _rows("v", v, g, heads, tokens, k_pages)
    if k.dtype != v.dtype:
        raise TypeError("k and v must have the same dtype")
    _check_written(k_pages, v_pages, k_scales, v_scales)
    _check_not_followed(k=k, v=v, k_pages=k_pages, v_pages=v_pages)
    if tokens == 0:
        return
    prob = g.pack(tokens, heads, 1, k.dtype, 0.0, k=ks, v=vs)
    g.run(_lib.lib().moba_paged_store, prob, k.data_ptr(), v.data_ptr(), *g.where)
    _written(k_pages, v_pages, k_scales, v_scales)


def paged_load(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
               seq_lens: torch.Tensor, total_tokens: int, *, dtype: Optional[torch.dtype] = None,
               k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Reads rows back: (k, v), each [total_tokens, Hkv, D] packed as cu_seqlens says, of `dtype` (8-bit pages: bfloat16 unless
    given).  With seq_lens the lengths of whole sequences this is the packed batch that `parallel_moba` takes.  Rows whose page is not
    there are zeros; rows behind the last sequence are left as they were (undefined without `out`)."""
    g = _Pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    if not isinstance(total_tokens, int) or total_tokens < 0:
        raise ValueError(f"total_tokens must be an int that is not negative, got {total_tokens}")
    same = g.store == _lib.STORE_SAME
    if dtype is None:
        dtype = g.dtype if same else out[0].dtype if out is not None else torch.bfloat16
    _, _, heads, dim = g.shape
    if out is None:
        if dtype not in _DTYPE_OF:
            raise TypeError(f"only float16 and bfloat16 are supported, got {dtype}")
        if same and dtype != g.dtype:
            raise TypeError(f"rows of {g.dtype} pages are {g.dtype}, got {dtype}")
        k = k_pages.new_empty((total_tokens, heads, dim), dtype=dtype)
        v = torch.empty_like(k)
        ks = vs = (heads * dim, dim)
    else:
        k, v = out
        ks = _rows("out[0]", k, g, heads, total_tokens, k_pages)
        vs = _rows("out[1]", v, g, heads, total_tokens, k_pages)
        if k.dtype != dtype or v.dtype != dtype:
            raise TypeError(f"out must be of {dtype}, got {k.dtype} and {v.dtype}")
        _check_written(k, v)
    _check_not_followed(k_pages=k_pages, v_pages=v_pages, **{"out[0]": k, "out[1]": v})
    if total_tokens == 0:
        return k, v
    prob = g.pack(total_tokens, heads, 1, dtype, 0.0, k=ks, v=vs)
    g.run(_lib.lib().moba_paged_load, prob, *g.where, k.data_ptr(), v.data_ptr())
    if out is not None:
        _written(*out)
    return k, v


def _check_attention(q, k_pages, max_new, scale, out) -> None:
    if q.shape[1] % k_pages.shape[2] != 0:
        raise ValueError(f"q heads ({q.shape[1]}) must be divisible by kv heads ({k_pages.shape[2]})")
    if not isinstance(max_new, int) or max_new <= 0:
        raise ValueError(f"max_new must be a positive int, got {max_new}")
    # (in the structure 0 stands for none given; times log2(e) it has to be finite)
    if scale is not None and not (0.0 < C.c_float(float(scale)).value and float(scale) <= 2.3e38):
        raise ValueError(f"scale must be a positive number of 32 bits, at most 2.3e38, got {scale}")
    if out is not None and out.dtype != q.dtype:
        raise TypeError(f"out must be of {q.dtype}, got {out.dtype}")


def _check_parents(parents, tokens: int, index: int) -> None:
    """`parents` of the packed rows, on device number `index`."""
    if parents.ndim != 1 or parents.shape[0] != tokens:
        raise ValueError(f"parents must have shape [{tokens}], got {tuple(parents.shape)}")
    if parents.dtype != torch.int32 or parents.get_device() != index:
        raise TypeError("parents must be an int32 tensor on the device of the call's other tensors")
    if tokens > 1 and parents.stride(0) != 1:
        raise NotImplementedError("parents must be contiguous")


def _attention(g: _Pages, q, kv, k_pages, v_pages, max_new, scale, return_lse, out, parents, written=()):
    """Attention of q; with `kv` the rows of k and v are stored first, in the tensors of `written`."""
    _check_not_followed(q=q, k=kv and kv[0], v=kv and kv[1], k_pages=k_pages, v_pages=v_pages, out=out)
    qs = _rows("q", q, g, None, None, k_pages)
    tokens, heads, _ = q.shape
    _check_attention(q, k_pages, max_new, scale, out)
    if parents is not None:
        _check_parents(parents, tokens, g.index)
    dtype, given, ks, vs = q.dtype, out is not None, (0, 0), (0, 0)
    if given:
        os = _rows("out", out, g, heads, tokens, k_pages)
        _check_written(out)
    else:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os = (heads * g.shape[3], g.shape[3])
    if kv is not None:
        k, v = kv
        ks = _rows("k", k, g, g.shape[2], tokens, k_pages)
        vs = _rows("v", v, g, g.shape[2], tokens, k_pages)
        if k.dtype != dtype or v.dtype != dtype:
            raise TypeError("q, k, and v must have the same dtype")
    lse = q.new_empty((heads, tokens), dtype=torch.float32) if return_lse else None
    if tokens > 0:
        lib, need = _lib.lib(), C.c_size_t(0)
        prob = g.pack(tokens, heads, max_new, dtype, 0.0 if scale is None else float(scale), qs, os, ks, vs)
        _lib.check((lib.moba_paged_workspace_size if parents is None else lib.moba_paged_tree_workspace_size)(prob, C.byref(need)))
        ws = _workspace(q.device, need.value)                # (the caching allocator goes by the current stream of the device given)
        if kv is not None:
            # what only the attention would refuse comes before anything is written
            if (q.data_ptr() | out.data_ptr()) & 15:
                _lib.check(_lib.E_ALIGN)
            if (os[0] == 0 and tokens > 1) or (os[1] == 0 and heads > 1):
                _lib.check(_lib.E_SHAPE)
            g.run(lib.moba_paged_store, prob, k.data_ptr(), v.data_ptr(), *g.where)
            _written(*written)
        g.run(lib.moba_paged_tree_attention, prob, q.data_ptr(), None if parents is None else parents.data_ptr(), *g.where, out.data_ptr(), None if lse is None else lse.data_ptr(),
              ws.data_ptr(), need.value)
        if given:
            _written(out)
    return (out, lse) if return_lse else out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, max_new: int, *, scale: Optional[float] = None,
                    k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
                    return_lse: bool = False, out: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None):
    """Causal softmax attention of the packed new tokens q [T, Hq, D] over the pages of their sequences: every token sees the
    positions of its sequence up to its own, which the pages hold already (`paged_append` writes them first).  One token a sequence
    is a decode step, a few are drafted tokens, many a block of a prompt; a batch may mix them.

    `max_new`: the most new tokens that a sequence has (the kernel is chosen by it; another number costs time only).  `scale`:
    factor of the scores, head_dim ** -0.5 unless given.  Returns out [T, Hq, D], with `return_lse` (out, lse [Hq, T] fp32, natural
    log).  A token that sees nothing is zeros and -inf.  `out`: a tensor to write to; rows behind the last sequence are left as
    they were (undefined without it).  8-bit pages are attended to as the rows that `paged_load` gives in the queries' dtype,
    whichever they were written from: a value beyond float16 is an infinity to float16 queries.

    `parents` [T] int32: the packed tokens are trees of drafted ones.  parents[row] is the row of the same sequence, counted from its
    first packed one, that the token follows; what is not an earlier row (-1) is none.  A token then sees the tokens in front of
    the packed ones, its ancestors and itself.  Rows keep their places in the pages, whatever branch they are of.  Small trees are fastest with
    no more columns of the table than the longest sequence needs (a view, page_table[:, :n], will do): which kernel takes them goes by its room."""
    g = _Pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    return _attention(g, q, None, k_pages, v_pages, max_new, scale, return_lse, out, parents)


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, max_new: int, *,
                 scale: Optional[float] = None, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None,
                 parents: Optional[torch.Tensor] = None):
    """`paged_store` of the new tokens' k and v, then `paged_attention` of their q: a layer's step of a server."""
    g = _Pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    _check_written(k_pages, v_pages, k_scales, v_scales)
    return _attention(g, q, (k, v), k_pages, v_pages, max_new, scale, return_lse, out, parents, (k_pages, v_pages, k_scales, v_scales))


def _i32_rows(name, x, shape, index) -> None:
    """An int32 tensor of this shape, contiguous in its last dimension, on device number `index`."""
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(x.shape)}")
    if x.dtype != torch.int32 or x.get_device() != index:
        raise TypeError(f"{name} must be an int32 tensor on the device of the call's other tensors")
    if x.stride(-1) != 1 and shape[-1] > 1:
        raise NotImplementedError(f"{name} must be contiguous in its last dimension")


def paged_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor,
               path: torch.Tensor, count: torch.Tensor, *, k_scales: Optional[torch.Tensor] = None,
               v_scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Moves the rows of an accepted branch together: of the packed tokens of sequence b, which the pages hold, rows path[b, 0] < path[b, 1]
    < .. (count[b] of them; `verify_drafts` gives both) go to the places of rows 0, 1, ..  Returns the sequences' lengths then, int32 [batch]: the tokens in
    front of the packed ones and the kept ones; what is behind them is no longer the sequence's.  8-bit rows are moved as they are, with
    their powers of two; a slot that two sequences' tables have is undefined.  A path ends in front of an entry that is no later row of the sequence than the one before it.  Each layer's pages are
    moved with the same seq_lens, those with the drafted tokens."""
    g = _Pages(k_pages, v_pages, page_table, cu_seqlens, seq_lens, k_scales, v_scales)
    if path.ndim != 2 or path.shape[1] == 0:
        raise ValueError(f"path must have shape [{g.batch}, rows], got {tuple(path.shape)}")
    _i32_rows("path", path, (g.batch, path.shape[1]), g.index)
    _i32_rows("count", count, (g.batch,), g.index)
    _check_written(k_pages, v_pages, k_scales, v_scales)
    _check_not_followed(k_pages=k_pages, v_pages=v_pages)
    lens = torch.empty(g.batch, dtype=torch.int32, device=k_pages.device)
    dtype = g.dtype if g.store == _lib.STORE_SAME else torch.bfloat16
    cu, old, table, k, v, ks, vs = g.where
    columns = path.shape[1]
    g.run(_lib.lib().moba_paged_keep, g.pack(1, g.shape[2], 1, dtype, 0.0), cu, old, table, path.data_ptr(),
          path.stride(0) if g.batch > 1 else columns, columns, count.data_ptr(), k, v, ks, vs, lens.data_ptr())
    _written(k_pages, v_pages, k_scales, v_scales)
    return lens


#: struct moba_page_pool, field by field
_POOL = struct.Struct("@q4i2q")
assert _POOL.size == C.sizeof(_lib.PagePool)


def _check_pool(page_table, free_pages, free_count, page_size, total_tokens, lens_name, lens) -> None:
    index = page_table.get_device()
    if index < 0:
        raise ValueError("page_table must be an accelerator tensor")
    if page_table.ndim != 2 or 0 in page_table.shape:
        raise ValueError(f"page_table must have shape [batch, pages of a sequence], got {tuple(page_table.shape)}")
    if free_pages.ndim != 1 or free_pages.shape[0] == 0:
        raise ValueError(f"free_pages must have shape [pages], got {tuple(free_pages.shape)}")
    if not isinstance(page_size, int) or page_size <= 0:
        raise ValueError(f"page_size must be a positive int, got {page_size}")
    if page_size < 16 or page_size & (page_size - 1):
        raise NotImplementedError(f"page_size must be a power of two and at least 16, got {page_size}")
    batch, per_seq = page_table.shape
    _i32_rows("page_table", page_table, page_table.shape, index)
    _i32_rows("free_pages", free_pages, free_pages.shape, index)
    _i32_rows("free_count", free_count, (1,), index)
    _i32_rows(lens_name, lens, (batch,), index)
    if batch > 1 and page_table.stride(0) < per_seq:
        raise ValueError("rows of page_table must not lie on one another")
    if not isinstance(total_tokens, int) or total_tokens < 0:
        raise ValueError(f"total_tokens must be an int that is not negative, got {total_tokens}")


def _pool_call(page_table, free_pages, free_count, page_size, total_tokens, lens_name, lens) -> Tuple[bytes, int, int]:
    """The structure of a call on a pool, with its tensors checked, their device's number and the sequences."""
    table, pages, index, i32 = page_table.shape, free_pages.shape, page_table.get_device(), torch.int32
    good = len(table) == 2 and index >= 0 and len(pages) == 1 and isinstance(page_size, int) and isinstance(total_tokens, int)
    if good:
        (batch, per_seq), (ts, td) = table, page_table.stride()
        good = (batch > 0 and per_seq > 0 and pages[0] > 0 and page_size >= 16 and not page_size & (page_size - 1) and total_tokens >= 0
                and (td == 1 or per_seq == 1) and (batch == 1 or ts >= per_seq) and page_table.dtype == i32
                and free_pages.dtype == i32 and free_pages.get_device() == index and (pages[0] == 1 or free_pages.stride(0) == 1)
                and free_count.shape == (1,) and free_count.dtype == i32 and free_count.get_device() == index
                and lens.shape == (batch,) and lens.dtype == i32 and lens.get_device() == index and (batch == 1 or lens.stride(0) == 1))
    if not good:
        _check_pool(page_table, free_pages, free_count, page_size, total_tokens, lens_name, lens)
        raise ValueError("page_table, free_pages, free_count and the lengths do not describe a call")
    _check_written(page_table, free_pages, free_count)
    try:
        return _POOL.pack(total_tokens, batch, per_seq, pages[0], page_size, ts if batch > 1 else per_seq, 0), index, batch
    except struct.error as e:
        raise NotImplementedError("pages, columns of the table, tokens and sequences are counted in 32 bits") from e


def _run_on(index: int, call, *args) -> None:
    """`call(*args, stream)` with device number `index` current."""
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            _lib.check(call(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        _lib.check(call(*args, torch._C._cuda_getCurrentRawStream(index)))


def paged_reserve(page_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int, total_tokens: int, *,
                  parents: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Pages for the packed tokens of a call, and where they lie.  Every entry of the tables that a packed token's position is in and that is no
    page's number gets one from the stack of free pages (free_pages int32 [pages], of which the first free_count, int32 [1], are free ones; the last
    is taken first), in the order of the sequences and entries.  The table, the stack and its count are written.

    Returns (slots, positions, missing): slots int64 [total_tokens], page * page_size + place of each packed row, -1 where it has no page;
    positions int32 [total_tokens], as `rotary` takes them, with `parents` (see `paged_attention`) those of a row's depth in its tree; missing int32
    [1], the entries for which no page was left.  Rows of no sequence have -1 in both.  Calls on one pool are ordered by the caller's
    streams.  At most 16384 sequences."""
    call, index, batch = _pool_call(page_table, free_pages, free_count, page_size, total_tokens, "seq_lens", seq_lens)
    _i32_rows("cu_seqlens", cu_seqlens, (batch + 1,), index)
    if parents is not None:
        _check_parents(parents, total_tokens, index)
    device, i32 = page_table.device, torch.int32
    slots = torch.empty(total_tokens, dtype=torch.int64, device=device)
    positions, missing = torch.empty(total_tokens, dtype=i32, device=device), torch.empty(1, dtype=i32, device=device)
    _run_on(index, _lib.lib().moba_paged_reserve, call, cu_seqlens.data_ptr(), seq_lens.data_ptr(),
            parents.data_ptr() if parents is not None else None, page_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
            slots.data_ptr(), positions.data_ptr(), missing.data_ptr())
    _written(page_table, free_pages, free_count)
    return slots, positions, missing


def paged_release(page_table: torch.Tensor, keep_lens: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  page_size: int) -> None:
    """Gives pages back: those behind the first keep_lens[b] (int32) tokens of sequence b, all of them for 0, go to the stack of free pages and
    their entries become -1.  The other way round of `paged_reserve`: what one call took, a release leaves as it was.  Pages that other
    sequences share must not be given back."""
    call, index, _ = _pool_call(page_table, free_pages, free_count, page_size, 0, "keep_lens", keep_lens)
    _run_on(index, _lib.lib().moba_paged_release, call, keep_lens.data_ptr(), page_table.data_ptr(), free_pages.data_ptr(),
            free_count.data_ptr())
    _written(page_table, free_pages, free_count)


class PagePool:
    """The free pages of a `PagedKV` (of all layers' caches, which share one page table): `free_pages` int32 [num_pages], the stack of their
    numbers, and `free_count` int32 [1].  All are free at first."""

    def __init__(self, num_pages: int, page_size: int, device: Optional[torch.device] = None):
        if num_pages <= 0:
            raise ValueError(f"num_pages must be positive, got {num_pages}")
        if page_size < 16 or page_size & (page_size - 1):
            raise NotImplementedError(f"page_size must be a power of two and at least 16, got {page_size}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page_size = page_size
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)

    def reserve(self, page_table, cu_seqlens, seq_lens, total_tokens: int, parents=None):
        return paged_reserve(page_table, cu_seqlens, seq_lens, self.free_pages, self.free_count, self.page_size, total_tokens, parents=parents)

    def release(self, page_table, keep_lens) -> None:
        paged_release(page_table, keep_lens, self.free_pages, self.free_count, self.page_size)


class PagedKV:
    """A layer's pool of pages.  `k`, `v`: [pages, page_size, Hkv, D], in memory head by head within a page, so that the rows of
    one head that attention reads together lie together; `k_scales`, `v_scales` for 8-bit pages, else None.  `dtype` is that of the
    rows written and read, `store` that of the pages: the same, torch.float8_e4m3fn or torch.int8."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 store: Optional[torch.dtype] = None, device: Optional[torch.device] = None):
        store = dtype if store is None else store
        if dtype not in _ROWS:
            raise TypeError(f"only float16 and bfloat16 are supported, got {dtype}")
        if store != dtype and store not in _STORES:
            raise TypeError(f"pages hold the rows' own dtype, float8_e4m3fn or int8, got {store}")
        if num_pages <= 0 or num_kv_heads <= 0:
            raise ValueError(f"num_pages and num_kv_heads must be positive, got {num_pages} and {num_kv_heads}")
        if page_size < 16 or page_size & (page_size - 1):
            raise NotImplementedError(f"page_size must be a power of two and at least 16, got {page_size}")
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"this build supports head_dim {HEAD_DIMS} only")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.dtype = dtype
        self.k, self.v = (torch.zeros(num_pages, num_kv_heads, page_size, head_dim, device=device, dtype=torch.int8 if store in _STORES else store)
                          .view(store).transpose(1, 2) for _ in range(2))
        self.k_scales = self.v_scales = None
        if store in _STORES:
            self.k_scales, self.v_scales = (torch.full((num_pages, num_kv_heads, page_size), 127, device=device, dtype=torch.uint8)
                                            for _ in range(2))

    def _scales(self):
        return {"k_scales": self.k_scales, "v_scales": self.v_scales}

    def store(self, k, v, page_table, cu_seqlens, seq_lens) -> None:
        paged_store(k, v, self.k, self.v, page_table, cu_seqlens, seq_lens, **self._scales())

    def load(self, page_table, cu_seqlens, seq_lens, total_tokens: int, out=None):
        return paged_load(self.k, self.v, page_table, cu_seqlens, seq_lens, total_tokens, dtype=self.dtype, out=out, **self._scales())

    def attend(self, q, page_table, cu_seqlens, seq_lens, max_new: int, **options):
        return paged_attention(q, self.k, self.v, page_table, cu_seqlens, seq_lens, max_new, **self._scales(), **options)

    def append(self, q, k, v, page_table, cu_seqlens, seq_lens, max_new: int, **options):
        return paged_append(q, k, v, self.k, self.v, page_table, cu_seqlens, seq_lens, max_new, **self._scales(), **options)

    def keep(self, page_table, cu_seqlens, seq_lens, path, count):
        return paged_keep(self.k, self.v, page_table, cu_seqlens, seq_lens, path, count, **self._scales())
