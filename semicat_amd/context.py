"""Attention of queries on keys of another length, beside the attention-JVP op: cross attention to an encoder's states and
attention with a learned relative position bias, with reverse mode, on ``[B,S,H,D]`` tensors as :func:`semicat_amd.safe_sdpa_jvp`
takes them.  No counterpart in olsdavis/semicat, whose attention has one length, no mask and no bias.

* :func:`cross_attention` and :func:`relative_attention` are the ops, for training, for a forward without gradients and for the
  few query rows of a generation step (the kernels split the key axis by themselves where the rows are few).
* :func:`context_forward` and :func:`context_backward` are their launches on ``[B,H,L,D]`` views, for callers with autograd glue of
  their own.

Forward mode (``torch.func.jvp``) and double backward are not implemented and raise.
"""
from __future__ import annotations

import ctypes
import functools
import operator
from typing import Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as fwAD
from torch import Tensor

from . import _lib
from .kernels import _host_result, _on_gpu, _scale_arg

_DTYPES = {torch.bfloat16: _lib.SJVP_BF16, torch.float16: _lib.SJVP_FP16}
_TABLE_DTYPES = {torch.bfloat16: _lib.SJVP_BF16, torch.float16: _lib.SJVP_FP16, torch.float32: _lib.SJVP_FP32}


@functools.lru_cache(maxsize=64, typed=True)
def relative_bucket_starts(buckets: int, max_distance: int = 128) -> Tuple[int, ...]:
    """The first distance of each bucket of one direction.  The lower half of the ``n`` buckets are single distances; bucket
    ``single + k`` begins at the least ``d`` with ``(d / single) ** (n - single) >= (max_distance / single) ** k``, so that the
    upper ones grow evenly in the logarithm and the last one has no end.  In whole numbers: no rounding at a border."""
    buckets, max_distance = operator.index(buckets), operator.index(max_distance)
    single = buckets // 2
    if buckets < 2 or buckets > _lib.SJVP_CTX_MAX_BUCKETS:
        raise ValueError(f"a direction has 2 to {_lib.SJVP_CTX_MAX_BUCKETS} buckets, got {buckets}")
    if max_distance <= single or max_distance > _lib.SJVP_CTX_MAX_DISTANCE:
        raise ValueError(f"max_distance must lie above the {single} single distances and within "
                         f"{_lib.SJVP_CTX_MAX_DISTANCE}, got {max_distance}")
    above, starts = buckets - single, list(range(single + 1))
    for k in range(1, above):
        d = starts[-1]
        while d ** above * single ** k < max_distance ** k * single ** above:
            d += 1
        starts.append(d)
    return tuple(starts)


@functools.lru_cache(maxsize=64, typed=True)
def _packed_starts(rows: int, max_distance: int, bidirectional: bool) -> bytes:
    """The first distances as the host extension takes them, for a table of that many rows."""
    if bidirectional and rows % 2:
        raise ValueError(f"two directions share an even number of buckets, got {rows}")
    starts = relative_bucket_starts(rows // 2 if bidirectional else rows, max_distance)
    return bytes((ctypes.c_int32 * len(starts))(*starts))


class RelativeBias:
    """A bias table of a call with the map of its buckets, checked: ``table`` is ``[num_buckets, Hq]``."""

    __slots__ = ("table", "starts", "bidirectional", "causal")

    def __init__(self, table: Tensor, max_distance: int = 128, bidirectional: bool = True, causal: bool = False):
        if table.ndim != 2:
            raise AssertionError(f"the table must be [num_buckets, heads], got {tuple(table.shape)}")
        if table.dtype not in _TABLE_DTYPES:
            raise TypeError(f"the table must be bfloat16, float16 or float32, got {table.dtype}")
        n = table.shape[0]
        if bidirectional and n % 2:
            raise ValueError(f"two directions share an even number of buckets, got {n}")
        self.table, self.bidirectional, self.causal = table, bool(bidirectional), bool(causal)
        self.starts = relative_bucket_starts(n // 2 if bidirectional else n, max_distance)


def _check(name: str, t: Tensor, shape, q: Tensor) -> None:
    if tuple(t.shape) != tuple(shape):
        raise AssertionError(f"{name} shape mismatch: {tuple(t.shape)} != {tuple(shape)}")
    if t.dtype != q.dtype:
        raise TypeError(f"{name} dtype {t.dtype} != {q.dtype}")
    if t.device != q.device:
        raise ValueError(f"{name} is on {t.device}, expected {q.device}")
    if t.stride(-1) != 1 and t.numel():
        raise AssertionError(f"{name}: the last dimension must have unit stride")


def _check_indices(name: str, t: Optional[Tensor], q: Tensor) -> None:
    if t is None:
        return
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if tuple(t.shape) != (q.shape[0],) or not t.is_contiguous():
        raise AssertionError(f"{name} must be a contiguous tensor of shape {(q.shape[0],)}, got {tuple(t.shape)}")
    if t.device != q.device:
        raise ValueError(f"{name} is on {t.device}, expected {q.device}")


def _check_inputs(q, k, v, bias, key_lengths, query_lengths, query_start) -> None:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.ndim != 4:
            raise AssertionError(f"{name} must have four dimensions, got {tuple(t.shape)}")
    if not q.is_cuda:
        raise RuntimeError(f"semicat_amd kernels run on an AMD GPU only; got a tensor on {q.device} (there is no CPU fallback)")
    if q.dtype not in _DTYPES:
        raise TypeError(f"context attention kernels support bfloat16 and float16, got {q.dtype}")
    B, H, Lq, D = q.shape
    if D < 16 or D > 128:
        raise ValueError(f"the head dimension must lie within 16 and 128, got {D}")
    if max(*q.shape, *k.shape) > _lib.SJVP_CTX_MAX_POSITION:
        raise ValueError(f"sizes must not exceed {_lib.SJVP_CTX_MAX_POSITION}, got {tuple(q.shape)} and {tuple(k.shape)}")
    if k.shape[1] < 1 or H % max(k.shape[1], 1):
        raise AssertionError(f"{H} query heads cannot share {k.shape[1]} key heads")
    _check("q", q, q.shape, q)
    _check("k", k, (B, k.shape[1], k.shape[2], D), q)
    _check("v", v, k.shape, q)
    _check_indices("key_lengths", key_lengths, q)
    _check_indices("query_lengths", query_lengths, q)
    if isinstance(query_start, Tensor):
        _check_indices("query_start", query_start, q)
    elif not -_lib.SJVP_CTX_MAX_POSITION <= operator.index(query_start) <= _lib.SJVP_CTX_MAX_POSITION:
        raise ValueError(f"query_start must lie within +-{_lib.SJVP_CTX_MAX_POSITION}, got {query_start}")
    if bias is not None:
        if bias.table.shape[1] != H:
            raise AssertionError(f"the table has {bias.table.shape[1]} heads, the queries {H}")
        if bias.table.device != q.device:
            raise ValueError(f"the table is on {bias.table.device}, expected {q.device}")


def _call(backward: bool, tensors, lse, bias, key_lengths, query_lengths, query_start, scale, dtable=None) -> None:
    """``tensors``: q, k, v, o, o_rest, dO, dq, dk, dv, as the C ABI orders them."""
    q, k = tensors[0], tensors[1]
    ptr = lambda t: None if t is None else t.data_ptr()
    t = _lib.Ctx()
    for i, (name, x) in enumerate(zip(_lib.C_TENSORS, tensors)):
        setattr(t, name, ptr(x))
        if x is not None:
            t.strides[3 * i:3 * i + 3] = x.stride()[:3]
    t.lse, t.key_lengths, t.query_lengths = ptr(lse), ptr(key_lengths), ptr(query_lengths)
    if isinstance(query_start, Tensor):
        t.query_start = ptr(query_start)
    else:
        t.query_start0 = operator.index(query_start)
    if bias is not None:
        t.table, t.table_dtype = ptr(bias.table), _TABLE_DTYPES[bias.table.dtype]
        t.table_stride[:] = bias.table.stride()
        t.buckets, t.bidirectional, t.causal = len(bias.starts), bias.bidirectional, bias.causal
        starts = (ctypes.c_int32 * len(bias.starts))(*bias.starts)
        t.bucket_first = ctypes.cast(starts, ctypes.c_void_p)
        if dtable is not None:
            t.dtable = ptr(dtable)
            t.dtable_stride[:] = dtable.stride()
    t.B, t.Hq, t.Lq, t.D = q.shape
    t.Hkv, t.Lk = k.shape[1:3]
    t.scale = _scale_arg(scale)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        t.workspace_bytes = lib.sjvp_ctx_workspace_bytes(ctypes.byref(t), int(backward))
        workspace = torch.empty((t.workspace_bytes,), device=q.device, dtype=torch.uint8) if t.workspace_bytes else None
        t.workspace = ptr(workspace)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        _lib.check((lib.sjvp_ctx_bwd if backward else lib.sjvp_ctx_fwd)(ctypes.byref(t), _DTYPES[q.dtype], stream))


def context_forward(q: Tensor, k: Tensor, v: Tensor, bias: Optional[RelativeBias] = None, key_lengths: Optional[Tensor] = None,
                    query_lengths: Optional[Tensor] = None, query_start: Union[int, Tensor] = 0, scale: Optional[float] = None,
                    o: Optional[Tensor] = None, o_rest: Optional[Tensor] = None, with_lse: bool = True
                    ) -> Tuple[Tensor, Optional[Tensor]]:
    """Forward on ``[B,H,L,D]`` views: ``(o, lse)``, with ``lse`` fp32 ``[B,Hq,Lq,2]``, or None without ``with_lse``: two numbers ``m``,
    ``l`` to a row, of which the logarithm of the sum of its scores' exponentials is ``m ln 2 + ln l`` (in one number, ``l`` would be lost
    beside large scores or biases), ``(0, 0)`` for a row that sees no key.  ``o`` may be passed in to be filled, and ``o_rest``, a tensor like it, to receive what the rounding of ``o`` leaves (16 bits
    in a form of their own), for :func:`context_backward`."""
    _check_inputs(q, k, v, bias, key_lengths, query_lengths, query_start)
    B, H, Lq, D = q.shape
    if o is None:
        o = torch.empty((B, Lq, H, D), device=q.device, dtype=q.dtype).transpose(1, 2)
    _check("o", o, q.shape, q)
    if o_rest is not None:
        _check("o_rest", o_rest, q.shape, q)
    lse = torch.empty((B, H, Lq, 2), device=q.device, dtype=torch.float32) if with_lse else None
    if q.numel() == 0 or k.numel() == 0:  # no row, or no key for any row
        if o_rest is not None:
            o_rest.zero_()
        return o.zero_(), None if lse is None else lse.zero_()
    _call(False, (q, k, v, o, o_rest, None, None, None, None), lse, bias, key_lengths, query_lengths, query_start, scale)
    return o, lse


def context_backward(q: Tensor, k: Tensor, v: Tensor, o: Tensor, lse: Tensor, dO: Tensor, bias: Optional[RelativeBias] = None,
                     key_lengths: Optional[Tensor] = None, query_lengths: Optional[Tensor] = None,
                     query_start: Union[int, Tensor] = 0, scale: Optional[float] = None, o_rest: Optional[Tensor] = None,
                     with_keys: bool = True, with_table: bool = True
                     ) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """Backward on ``[B,H,L,D]`` views for the cotangent ``dO``, with the forward's arguments and results:
    ``(dq, dk, dv, dtable)``.  Without ``o_rest`` the row sums of ``dO * o`` carry the rounding of ``o``, which the gradients of
    sharp rows and of a float32 table show.  ``with_keys=False`` leaves out dk and dv (frozen states), ``with_table=False`` the table's."""
    _check_inputs(q, k, v, bias, key_lengths, query_lengths, query_start)
    B, H, Lq, D = q.shape
    if dO.stride(-1) != 1 or dO.stride(2) >= 1 << 24:
        dO = dO.contiguous()
    for name, t in (("o", o), ("dO", dO)) + ((("o_rest", o_rest),) if o_rest is not None else ()):
        _check(name, t, q.shape, q)
    if tuple(lse.shape) != (B, H, Lq, 2) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != q.device:
        raise AssertionError(f"lse must be a contiguous float32 tensor of shape {(B, H, Lq, 2)}, got {tuple(lse.shape)} {lse.dtype}")
    like = lambda t: torch.empty((t.shape[0], t.shape[2], t.shape[1], D), device=t.device, dtype=t.dtype).transpose(1, 2)
    dq, dk, dv = like(q), *((like(k), like(v)) if with_keys else (None, None))
    dtable = torch.empty(bias.table.shape, device=q.device, dtype=bias.table.dtype) if bias is not None and with_table else None
    if q.numel() == 0 or k.numel() == 0:
        return tuple(None if t is None else t.zero_() for t in (dq, dk, dv, dtable))
    _call(True, (q, k, v, o, o_rest, dO, dq, dk, dv), lse, bias, key_lengths, query_lengths, query_start, scale, dtable)
    return dq, dk, dv, dtable


class ContextAttentionFunction(torch.autograd.Function):
    """The op on ``[B,S,H,D]`` tensors as one autograd node; ``table`` is None for plain cross attention."""

    @staticmethod
    def forward(q, k, v, table, key_lengths, query_lengths, query_start, scale, max_distance, bidirectional, causal):
        bias = None if table is None else RelativeBias(table, max_distance, bidirectional, causal)
        rest = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        o, lse = context_forward(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), bias, key_lengths, query_lengths,
                                 query_start, scale, o_rest=rest.transpose(1, 2))
        return o.transpose(1, 2), lse, rest

    @staticmethod
    def setup_context(ctx, inputs, output) -> None:
        q, k, v, table, key_lengths, query_lengths, query_start, *ctx.options = inputs
        o, lse, rest = output
        ctx.start = None if isinstance(query_start, Tensor) else query_start
        ctx.save_for_backward(q, k, v, table, key_lengths, query_lengths, None if ctx.start is not None else query_start, o, lse, rest)
        ctx.mark_non_differentiable(lse, rest)
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, d_o, *_):
        if d_o is None:
            return (None,) * 11
        q, k, v, table, key_lengths, query_lengths, query_start, o, lse, rest = ctx.saved_tensors
        needs = ctx.needs_input_grad
        grads = ContextAttentionBackwardFunction.apply(
            q, k, v, table, o, lse, rest, d_o, key_lengths, query_lengths, query_start if ctx.start is None else ctx.start,
            *ctx.options, needs[1] or needs[2], needs[3])
        return *(g if need else None for g, need in zip(grads, needs)), *(None,) * 7


class ContextAttentionBackwardFunction(torch.autograd.Function):
    """Gradients of q, k, v and the table for the cotangent of the output."""

    @staticmethod
    def forward(q, k, v, table, o, lse, rest, d_o, key_lengths, query_lengths, query_start, scale, max_distance,
                bidirectional, causal, with_keys, with_table):
        bias = None if table is None else RelativeBias(table, max_distance, bidirectional, causal)
        heads = [None if t is None else t.transpose(1, 2) for t in (q, k, v, o, d_o, rest)]
        dq, dk, dv, dtable = context_backward(*heads[:4], lse, heads[4], bias, key_lengths, query_lengths, query_start, scale,
                                              o_rest=heads[5], with_keys=with_keys, with_table=with_table)
        return *(None if t is None else t.transpose(1, 2) for t in (dq, dk, dv)), dtable

    @staticmethod
    def setup_context(ctx, inputs, output) -> None:
        pass

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("double backward of the context attention ops is not implemented")


def _attend(q, k, v, table, key_lengths, query_lengths, query_start, scale, max_distance=128, bidirectional=True,
            causal=False) -> Tensor:
    if _on_gpu(q):
        first = None if table is None or table.ndim != 2 else _packed_starts(table.shape[0], max_distance, bool(bidirectional))
        o = _lib.host().context(q, k, v, table, key_lengths, query_lengths, query_start, scale, first, bool(bidirectional), bool(causal))
        if o is not None:
            return _host_result(o)
    for t in (q, k, v, table):
        if t is not None and fwAD.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward mode of the context attention ops is not implemented")
    dtype = q.dtype
    if dtype not in _DTYPES:
        # the dtype policy of safe_sdpa_jvp: computed in bfloat16, handed back in the caller's type
        q, k, v = (t.to(torch.bfloat16) for t in (q, k, v))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, table)):
        o, _, _ = ContextAttentionFunction.apply(q, k, v, table, key_lengths, query_lengths, query_start, scale, max_distance,
                                              bidirectional, causal)
    else:
        bias = None if table is None else RelativeBias(table, max_distance, bidirectional, causal)
        o, _ = context_forward(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), bias, key_lengths, query_lengths,
                               query_start, scale, with_lse=False)
        o = o.transpose(1, 2)
    return o if o.dtype == dtype else o.to(dtype)


@torch._dynamo.disable
def cross_attention(q: Tensor, k: Tensor, v: Tensor, key_lengths: Optional[Tensor] = None,
                    query_lengths: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
    """Attention of ``q`` ``[B,Sq,Hq,D]`` on the states ``k``, ``v`` ``[B,Sk,Hkv,D]`` of another length: ``[B,Sq,Hq,D]``.

    ``Hq`` is a multiple of ``Hkv``; query head ``h`` reads key head ``h // (Hq // Hkv)``.  ``key_lengths`` / ``query_lengths``
    (int32 ``[B]``) are the lengths of the sequences of a padded batch: what lies behind them is not used, results and gradients
    there are zeros, and a sequence without keys gives zeros.  ``scale`` defaults to ``1/sqrt(D)``.  bfloat16 and float16,
    16 <= D <= 128; other types are computed in bfloat16 and handed back as they came."""
    return _attend(q, k, v, None, key_lengths, query_lengths, 0, scale)


@torch._dynamo.disable
def relative_attention(q: Tensor, k: Tensor, v: Tensor, table: Tensor, max_distance: int = 128, bidirectional: bool = True,
                       causal: bool = False, key_lengths: Optional[Tensor] = None, query_lengths: Optional[Tensor] = None,
                       query_start: Union[int, Tensor] = 0, scale: Optional[float] = None) -> Tensor:
    """:func:`cross_attention` with ``table[bucket(j - (query_start + i)), h]`` added to the score of query ``i`` and key ``j``, in float32
    (keys that all have the lowest number weigh alike, ``-inf`` leaves its keys out).

    ``table`` is ``[num_buckets, Hq]`` (float32, bfloat16 or float16; its gradient is summed in float32, and formed to some
    1e-6 for a float32 table).  Buckets go by distance (:func:`relative_bucket_starts`): with ``bidirectional`` the second half of
    them belongs to keys behind the query, without it these count as distance 0.  ``causal`` hides the keys behind a query.
    ``query_start`` (an int, or int32 ``[B]``) is the position of the first query among the keys: a generation step passes
    the tokens that the cache held before it, and ``key_lengths`` the tokens that it holds with the step's own."""
    return _attend(q, k, v, table, key_lengths, query_lengths, query_start, scale, max_distance, bidirectional, causal)
