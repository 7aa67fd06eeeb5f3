"""Attention over packed sequences: whole sequences of different lengths one behind the other in ``[T,H,D]`` tensors, with reverse mode.
No counterpart in olsdavis/semicat, whose sequences all have one length.

* :func:`packed_attention` is the op, for training and for a forward without gradients (a prompt's first pass, causal).
* :func:`packed_forward` and :func:`packed_backward` are its launches, for callers with autograd glue of their own.

Forward mode (``torch.func.jvp``) and double backward are not implemented and raise.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as fwAD
from torch import Tensor

from . import _lib
from .kernels import _host_result, _on_gpu, _scale_arg

_DTYPES = {torch.bfloat16: _lib.SJVP_BF16, torch.float16: _lib.SJVP_FP16}


def _check_rows(name: str, t: Tensor, shape, like: Tensor) -> None:
    if tuple(t.shape) != tuple(shape):
        raise AssertionError(f"{name} shape mismatch: {tuple(t.shape)} != {tuple(shape)}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} dtype {t.dtype} != {like.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if t.stride(-1) != 1 and t.numel():
        raise AssertionError(f"{name}: the last dimension must have unit stride")


def _check_indices(name: str, t: Tensor, shape, like: Tensor) -> None:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise AssertionError(f"{name} must be a contiguous tensor of shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")


def _check_query(q: Tensor) -> None:
    if q.ndim != 3:
        raise AssertionError(f"q must have three dimensions, got {tuple(q.shape)}")
    if not q.is_cuda:
        raise RuntimeError(f"semicat_amd kernels run on an AMD GPU only; got a tensor on {q.device} (there is no CPU fallback)")
    if q.dtype not in _DTYPES:
        raise TypeError(f"packed and paged attention kernels support bfloat16 and float16, got {q.dtype}")
    if not 16 <= q.shape[2] <= 128:
        raise ValueError(f"the head dimension must lie within 16 and 128, got {q.shape[2]}")
    if q.shape[0] * q.shape[1] >= 1 << 31 or q.shape[0] > 1 << 29:
        raise ValueError(f"at most 2^29 rows and 2^31 - 1 of all heads, got {tuple(q.shape)}")


def _check_offsets(offsets: Tensor, like: Tensor) -> None:
    if offsets.ndim != 1 or offsets.shape[0] < 2:
        raise AssertionError(f"offsets must be [sequences + 1], got {tuple(offsets.shape)}")
    _check_indices("offsets", offsets, offsets.shape, like)


def _check_packed(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor) -> None:
    _check_query(q)
    T, H, D = q.shape
    if k.ndim != 3 or k.shape[1] < 1 or H % max(k.shape[1], 1):
        raise AssertionError(f"{H} query heads cannot share the key heads of {tuple(k.shape)}")
    _check_rows("q", q, q.shape, q)
    _check_rows("k", k, (T, k.shape[1], D), q)
    _check_rows("v", v, k.shape, q)
    _check_offsets(offsets, q)


def _call(backward: bool, tensors, lse, offsets: Tensor, causal: bool, scale) -> None:
    """``tensors``: q, k, v, o, dO, dq, dk, dv, as the C ABI orders them."""
    q, k = tensors[:2]
    ptr = lambda t: None if t is None else t.data_ptr()
    t = _lib.Packed()
    for i, (name, x) in enumerate(zip(_lib.S_TENSORS, tensors)):
        setattr(t, name, ptr(x))
        if x is not None:
            t.strides[2 * i:2 * i + 2] = x.stride(1), x.stride(0)
    t.lse, t.offsets, t.B, t.causal = ptr(lse), ptr(offsets), offsets.shape[0] - 1, causal
    t.T, t.Hq, t.D = q.shape
    t.Hkv = k.shape[1]
    t.scale = _scale_arg(scale)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        t.workspace_bytes = lib.sjvp_packed_workspace_bytes(ctypes.byref(t), int(backward))
        workspace = torch.empty((t.workspace_bytes,), device=q.device, dtype=torch.uint8) if t.workspace_bytes else None
        t.workspace = ptr(workspace)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        _lib.check((lib.sjvp_packed_bwd if backward else lib.sjvp_packed_fwd)(ctypes.byref(t), _DTYPES[q.dtype], stream))


def _like(t: Tensor) -> Tensor:
    return torch.empty(t.shape, device=t.device, dtype=t.dtype)


def packed_forward(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, causal: bool = True, scale: Optional[float] = None,
                   with_lse: bool = True) -> Tuple[Tensor, Optional[Tensor]]:
    """Forward: ``(o, lse)``, with ``lse`` fp32 ``[Hq,T,2]``, or None without ``with_lse``: two numbers ``m``, ``l`` to a row, of which the
    logarithm of the sum of its scores' exponentials is ``m ln 2 + ln l``."""
    _check_packed(q, k, v, offsets)
    o = _like(q)
    lse = torch.zeros((q.shape[1], q.shape[0], 2), device=q.device, dtype=torch.float32) if with_lse and not q.numel() else \
        torch.empty((q.shape[1], q.shape[0], 2), device=q.device, dtype=torch.float32) if with_lse else None
    if q.numel():
        _call(False, (q, k, v, o, None, None, None, None), lse, offsets, causal, scale)
    return o, lse


def packed_backward(q: Tensor, k: Tensor, v: Tensor, o: Tensor, lse: Tensor, dO: Tensor, offsets: Tensor, causal: bool = True,
                    scale: Optional[float] = None, with_keys: bool = True) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """Backward for the cotangent ``dO``, with the forward's arguments and results: ``(dq, dk, dv)``.  ``with_keys=False`` leaves
    out dk and dv."""
    _check_packed(q, k, v, offsets)
    if dO.stride(-1) != 1 or dO.stride(0) >= 1 << 24:
        dO = dO.contiguous()
    _check_rows("o", o, q.shape, q)
    _check_rows("dO", dO, q.shape, q)
    shape = (q.shape[1], q.shape[0], 2)
    if tuple(lse.shape) != shape or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != q.device:
        raise AssertionError(f"lse must be a contiguous float32 tensor of shape {shape}, got {tuple(lse.shape)} {lse.dtype}")
    dq, dk, dv = _like(q), *((_like(k), _like(v)) if with_keys else (None, None))
    if q.numel():
        _call(True, (q, k, v, o, dO, dq, dk, dv), lse, offsets, causal, scale)
    elif with_keys:
        dk.zero_(), dv.zero_()  # (keys that no query reads)
    return dq, dk, dv


class PackedAttentionFunction(torch.autograd.Function):
    """The op as one autograd node."""

    @staticmethod
    def forward(q, k, v, offsets, causal, scale):
        return packed_forward(q, k, v, offsets, causal, scale)

    @staticmethod
    def setup_context(ctx, inputs, output) -> None:
        q, k, v, offsets, *ctx.options = inputs
        ctx.save_for_backward(q, k, v, offsets, *output)
        ctx.mark_non_differentiable(output[1])
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, d_o, *_):
        if d_o is None:
            return (None,) * 6
        q, k, v, offsets, o, lse = ctx.saved_tensors
        needs = ctx.needs_input_grad
        grads = PackedAttentionBackwardFunction.apply(q, k, v, o, lse, d_o, offsets, *ctx.options, needs[1] or needs[2])
        return *(g if need else None for g, need in zip(grads, needs)), None, None, None


class PackedAttentionBackwardFunction(torch.autograd.Function):
    """Gradients of q, k and v for the cotangent of the output."""

    @staticmethod
    def forward(q, k, v, o, lse, d_o, offsets, causal, scale, with_keys):
        return packed_backward(q, k, v, o, lse, d_o, offsets, causal, scale, with_keys)

    @staticmethod
    def setup_context(ctx, inputs, output) -> None:
        pass

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("double backward of packed attention is not implemented")


@torch._dynamo.disable
def packed_attention(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, causal: bool = True, scale: Optional[float] = None) -> Tensor:
    """Attention within each of several sequences that stand one behind the other: ``q`` ``[T,Hq,D]``, ``k`` and ``v`` ``[T,Hkv,D]``;
    returns ``[T,Hq,D]``.

    ``offsets`` (int32 ``[sequences + 1]``, ascending, on the GPU) says where: sequence ``b`` has the rows ``offsets[b]`` up to
    ``offsets[b + 1]``; sequences may be empty.  Rows in front of the first sequence and behind the last one are not used, results and
    gradients there are zeros.  The lengths are not looked at by the host.  ``causal`` hides the tokens behind a query: infinities and
    NaN among them reach neither its result nor its gradient.  ``Hq`` is a
    multiple of ``Hkv``; query head ``h`` reads key head ``h // (Hq // Hkv)``.  ``scale`` defaults to ``1/sqrt(D)``.  bfloat16 and float16,
    16 <= D <= 128; other types are computed in bfloat16 and handed back as they came."""
    if _on_gpu(q):
        o = _lib.host().packed(q, k, v, offsets, bool(causal), scale)
        if o is not None:
            return _host_result(o)
    for t in (q, k, v):
        if fwAD.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward mode of packed attention is not implemented")
    dtype = q.dtype
    if dtype not in _DTYPES:
        # the dtype policy of safe_sdpa_jvp: computed in bfloat16, handed back in the caller's type
        q, k, v = (t.to(torch.bfloat16) for t in (q, k, v))
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        o, _ = PackedAttentionFunction.apply(q, k, v, offsets, bool(causal), scale)
    else:
        o, _ = packed_forward(q, k, v, offsets, bool(causal), scale, with_lse=False)
    return o if o.dtype == dtype else o.to(dtype)
