"""A cache of keys and values in pages, with attention on it: the serving side of :mod:`semicat_amd.packed`.  No counterpart in
olsdavis/semicat, which generates whole sequences.

* :class:`PagedCache` holds the pages, as numbers of 16 bits or, quantised as they are written, of 8.
* :func:`paged_write` puts new tokens' keys and values to their places, :func:`paged_attention` attends from the new tokens to all that
  the cache holds of their sequences, :func:`paged_read` hands back what it holds.

All of them take the same description of the sequences: ``tables`` (int32 ``[B,P]``, position ``x`` of sequence ``b`` stands in row
``x % page_size`` of page ``tables[b, x // page_size]``), ``lengths`` (int32 ``[B]``, the tokens of each sequence with those of the call) and
``offsets`` (int32 ``[B+1]``, where the call's new tokens of each sequence stand in its ``[T,...]`` tensors, as in
:func:`semicat_amd.packed_attention`; None: one token of each sequence).  A page number that the cache has not reads as zeros and takes no writes;
positions behind the end of a table (a length of more than ``P * page_size``) take no writes and hold no keys.  The host looks at none of them.  None of the ops has a gradient: with an input, or a tensor of the
cache, that requires one they raise, as they do with forward-mode tangents.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as fwAD
from torch import Tensor

from . import _lib
from .kernels import _host_result, _on_gpu, _scale_arg
from .packed import _DTYPES, _check_indices, _check_offsets, _check_query, _check_rows

GROUP = 32  # columns of a row that share a scale
_SCALES = (torch.float8_e8m0fnu, torch.uint8)


class PagedCache:
    """``pages`` pages of ``page_size`` tokens for ``heads`` key heads: ``k`` and ``v`` ``[pages,heads,page_size,head_dim]``, so that what a head holds
    of a page is one piece of memory.

    ``quantized``: 8-bit numbers (``torch.float8_e4m3fn``) and, in ``k_scales`` and ``v_scales`` ``[pages,heads,page_size,ceil(head_dim/32)]``
    (``torch.float8_e8m0fnu``), a power of two for each 32 columns of a row: the least one by which none of their numbers goes
    beyond 448, the largest that the 8 bits have, within the range in which every 8-bit number stands for one of ``dtype``.  Numbers
    are rounded to nearest even, at most 2^-4 of themselves (or 2^-10 of the scale) off; what is not finite becomes NaN.  Reading rounds nothing.

    ``head_dim`` is a multiple of 8 (16 if quantised) within 16 and 128."""

    __slots__ = ("k", "v", "k_scales", "v_scales", "dtype", "_strides")

    def __init__(self, pages: int, page_size: int, heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 quantized: bool = False, device: Union[str, torch.device] = "cuda"):
        shape = (pages, heads, page_size, head_dim)
        new = lambda s, t: torch.zeros(s, dtype=torch.uint8, device=device).view(t) if t.itemsize == 1 else torch.zeros(s, dtype=t, device=device)
        store = torch.float8_e4m3fn if quantized else dtype
        scales = [new((*shape[:3], -(-head_dim // GROUP)), torch.float8_e8m0fnu) for _ in range(2)] if quantized else (None, None)
        self._take(new(shape, store), new(shape, store), *scales, dtype)

    @classmethod
    def of(cls, k: Tensor, v: Tensor, k_scales: Optional[Tensor] = None, v_scales: Optional[Tensor] = None,
           dtype: Optional[torch.dtype] = None) -> "PagedCache":
        """A cache in tensors that the caller has, of any strides whose pages, heads and rows are multiples of 16 bytes apart, pages
        and rows less than 4 GiB, the same of k and v.  ``dtype``: the 16-bit type that quantised numbers stand for (bfloat16 if not said)."""
        cache = cls.__new__(cls)
        cache._take(k, v, k_scales, v_scales, dtype)
        return cache

    def _take(self, k, v, k_scales, v_scales, dtype) -> None:
        quantized = k_scales is not None or v_scales is not None
        if k.ndim != 4:
            raise AssertionError(f"pages must be [pages, heads, page_size, head_dim], got {tuple(k.shape)}")
        if quantized and (k_scales is None or v_scales is None):
            raise AssertionError("k and v must both have scales, or neither")
        dtype = dtype or (torch.bfloat16 if quantized else k.dtype)
        if dtype not in _DTYPES or k.dtype != (torch.float8_e4m3fn if quantized else dtype):
            raise TypeError(f"pages hold bfloat16 or float16 numbers, or float8_e4m3fn ones with scales; got {k.dtype} for {dtype}")
        _check_rows("v", v, k.shape, k)
        _check_rows("k", k, k.shape, k)
        D, item = k.shape[3], k.dtype.itemsize
        if not 16 <= D <= 128 or D % (16 // item):
            raise ValueError(f"the head dimension must lie within 16 and 128 and be a multiple of {16 // item}, got {D}")
        if min(k.shape) < 1 or max(k.shape) > 1 << 29:
            raise ValueError(f"a cache has at least one page, head and row, got {tuple(k.shape)}")
        places = lambda t: tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))  # (of one page, head or row: no stride)
        strides = tuple(s * item for s in places(k))
        if places(v) != places(k) or any(s % 16 for s in strides) or (k.data_ptr() | v.data_ptr()) % 16:
            raise AssertionError("pages, heads and rows of k and v must stand at the same multiples of 16 bytes")
        if quantized:
            shape = (*k.shape[:3], -(-D // GROUP))
            if k_scales.dtype not in _SCALES:
                raise TypeError(f"scales must be float8_e8m0fnu or uint8, got {k_scales.dtype}")
            _check_rows("v_scales", v_scales, shape, k_scales)
            _check_rows("k_scales", k_scales, shape, k_scales)
            if k_scales.device != k.device or places(k_scales) != places(v_scales):
                raise AssertionError("scales of k and v must have the same strides, on the pages' device")
            strides += places(k_scales)
        if any(not 0 <= s < 1 << 32 for i, s in enumerate(strides) if i % 3 != 1):
            raise AssertionError("pages, and the rows of a page, must be less than 4 GiB apart")
        self.k, self.v, self.k_scales, self.v_scales, self.dtype = k, v, k_scales, v_scales, dtype
        self._strides = strides + (0,) * (6 - len(strides))

    def _storage(self):
        return self.k, self.v, self.k_scales, self.v_scales, self.dtype

    pages = property(lambda self: self.k.shape[0])
    heads = property(lambda self: self.k.shape[1])
    page_size = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])
    quantized = property(lambda self: self.k_scales is not None)


def _describe(cache: PagedCache, tables: Tensor, lengths: Tensor, offsets: Optional[Tensor], T: int) -> _lib.Paged:
    """The sequences' side of a call, checked."""
    if not cache.k.is_cuda:
        raise RuntimeError(f"semicat_amd kernels run on an AMD GPU only; got a cache on {cache.k.device} (there is no CPU fallback)")
    if tables.ndim != 2 or tables.shape[0] < 1 or tables.shape[1] < 1:
        raise AssertionError(f"tables must be [sequences, pages], got {tuple(tables.shape)}")
    if tables.dtype != torch.int32:
        raise TypeError(f"tables must be int32, got {tables.dtype}")
    if tables.device != cache.k.device:
        raise ValueError(f"tables is on {tables.device}, expected {cache.k.device}")
    if tables.stride(1) != 1 and tables.shape[1] > 1:
        raise AssertionError("tables: the last dimension must have unit stride")
    B = tables.shape[0]
    _check_indices("lengths", lengths, (B,), cache.k)
    if offsets is not None:
        _check_offsets(offsets, cache.k)
        if offsets.shape[0] != B + 1:
            raise AssertionError(f"offsets of {B} sequences are {B + 1}, got {offsets.shape[0]}")
    elif T >= 0 and T != B:
        raise AssertionError(f"without offsets there is one token of each of the {B} sequences, got {T}")
    t = _lib.Paged()
    t.k_pages, t.v_pages = cache.k.data_ptr(), cache.v.data_ptr()
    if cache.quantized:
        t.k_scales, t.v_scales = cache.k_scales.data_ptr(), cache.v_scales.data_ptr()
    t.page_strides[:] = cache._strides
    t.tables, t.table_stride, t.table_pages = tables.data_ptr(), tables.stride(0), tables.shape[1]
    t.lengths, t.offsets = lengths.data_ptr(), None if offsets is None else offsets.data_ptr()
    t.pages, t.Hkv, t.page_size, t.D = cache.k.shape
    t.B, t.T, t.Hq = B, max(T, 0), t.Hkv
    return t


def _put(t: _lib.Paged, i: int, x: Tensor, row: int = 0, head: int = 1) -> None:
    setattr(t, _lib.P_TENSORS[i], x.data_ptr())
    t.strides[3 * i:3 * i + 3] = x.stride(head), x.stride(row), x.stride(0) if head == 2 else 0


def _launch(fn: str, t: _lib.Paged, cache: PagedCache) -> None:
    lib = _lib.load()
    with torch.cuda.device(cache.k.device):
        workspace = None
        if fn == "sjvp_paged_attention":
            t.workspace_bytes = lib.sjvp_paged_workspace_bytes(ctypes.byref(t))
            if t.workspace_bytes:
                workspace = torch.empty((t.workspace_bytes,), device=cache.k.device, dtype=torch.uint8)
                t.workspace = workspace.data_ptr()
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        _lib.check(getattr(lib, fn)(ctypes.byref(t), _DTYPES[cache.dtype], stream))


def _no_gradient(what: str, cache: PagedCache, *tensors: Tensor) -> None:
    for t in (*tensors, *(x for x in cache._storage()[:4] if x is not None)):
        if fwAD.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"forward mode of {what} is not implemented")
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad() or with detached tensors")


@torch._dynamo.disable
def paged_write(cache: PagedCache, k: Tensor, v: Tensor, tables: Tensor, lengths: Tensor, offsets: Optional[Tensor] = None) -> None:
    """Writes the new tokens' ``k`` and ``v`` ``[T,Hkv,D]`` to the last positions of their sequences: token ``i`` of ``n`` new ones of a
    sequence has the position ``length - n + i``.  A page that is written to must belong to one sequence.  Tensors of another type than the cache's are
    rounded to it first.  The cache's tensors count as changed in place."""
    if _on_gpu(k):
        status = _lib.host().paged_write(k, v, *cache._storage(), tables, lengths, offsets)
        if status is not None:
            return _lib.check(status)
    _no_gradient("paged_write", cache, k, v)
    if k.ndim != 3:
        raise AssertionError(f"k must have three dimensions, got {tuple(k.shape)}")
    t = _describe(cache, tables, lengths, offsets, k.shape[0])
    k, v = (x if x.dtype == cache.dtype else x.to(cache.dtype) for x in (k, v))
    if k.shape[0] > 1 << 29:
        raise ValueError(f"at most 2^29 rows, got {tuple(k.shape)}")
    for name, x in (("k", k), ("v", v)):
        if x.device != cache.k.device:
            raise ValueError(f"{name} is on {x.device}, expected {cache.k.device}")
        _check_rows(name, x, (k.shape[0], cache.heads, cache.head_dim), k)
    if k.shape[0] == 0:
        return
    _put(t, 2, k), _put(t, 3, v)
    _launch("sjvp_paged_write", t, cache)
    # (a change in place, for what autograd has saved of these tensors)
    torch.autograd.graph.increment_version([x for x in cache._storage()[:4] if x is not None])


@torch._dynamo.disable
def paged_read(cache: PagedCache, tables: Tensor, lengths: Tensor, size: int) -> Tuple[Tensor, Tensor]:
    """What the cache holds of each sequence's first ``size`` positions: ``(k, v)`` ``[B,size,Hkv,D]``, zeros behind a sequence, as
    :func:`semicat_amd.cross_attention` takes them with ``key_lengths``."""
    if _on_gpu(cache.k):
        both = _lib.host().paged_read(*cache._storage(), tables, lengths, None, size)
        if both is not None:
            return _host_result(both)
    _no_gradient("paged_read", cache)
    t = _describe(cache, tables, lengths, None, -1)
    t.size = size
    k, v = (torch.empty((tables.shape[0], size, cache.heads, cache.head_dim), device=cache.k.device, dtype=cache.dtype) for _ in range(2))
    if size:
        _put(t, 2, k, 1, 2), _put(t, 3, v, 1, 2)
        _launch("sjvp_paged_read", t, cache)
    return k, v


@torch._dynamo.disable
def paged_attention(q: Tensor, cache: PagedCache, tables: Tensor, lengths: Tensor, offsets: Optional[Tensor] = None,
                    scale: Optional[float] = None) -> Tensor:
    """Attention of the new tokens ``q`` ``[T,Hq,D]`` on all tokens that the cache holds of their sequences, causal: token ``i`` of ``n`` new ones
    has the position ``length - n + i`` and sees the positions up to its own, which :func:`paged_write` has filled before.  Returns
    ``[T,Hq,D]``; rows that see nothing, and rows outside the sequences, are zeros.  ``Hq`` is a multiple of the cache's heads, ``scale``
    defaults to ``1/sqrt(D)``.  Sequences with one new token and with whole chunks of a prompt may stand in one call.  What the
    pages hold behind a token's position, NaN included, does not reach its result.  ``q`` of
    another type than the cache's is computed in the cache's and handed back as it came."""
    if _on_gpu(q):
        o = _lib.host().paged_attention(q, *cache._storage(), tables, lengths, offsets, scale)
        if o is not None:
            return _host_result(o)
    _no_gradient("paged_attention", cache, q)
    dtype = q.dtype
    q = q if dtype == cache.dtype else q.to(cache.dtype)
    _check_query(q)
    t = _describe(cache, tables, lengths, offsets, q.shape[0])
    if q.device != cache.k.device:
        raise ValueError(f"q is on {q.device}, expected {cache.k.device}")
    if q.shape[1] < 1 or q.shape[1] % cache.heads or q.shape[2] != cache.head_dim:
        raise AssertionError(f"queries {tuple(q.shape)} do not fit a cache of {cache.heads} heads of {cache.head_dim}")
    _check_rows("q", q, q.shape, q)
    o = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if q.shape[0]:
        t.Hq, t.scale = q.shape[1], _scale_arg(scale)
        _put(t, 0, q), _put(t, 1, o)
        _launch("sjvp_paged_attention", t, cache)
    return o if dtype == o.dtype else o.to(dtype)
