"""CPU tests of the context attention ops: the oracle, the map of the buckets, refusals."""
import ctypes

import pytest
import torch

from oracle import context_oracle as orc
from semicat_amd import RelativeBias, _lib, context_forward, cross_attention, relative_attention, relative_bucket_starts


@pytest.mark.parametrize("n,distance", [(2, 2), (3, 2), (5, 9), (16, 128), (32, 128), (7, 1024), (32, 17), (256, 1024), (10, 1000)])
def test_bucket_starts(n, distance):
    starts = relative_bucket_starts(n, distance)
    assert len(starts) == n and starts[0] == 0 and list(starts) == sorted(starts) and starts[-1] <= distance
    for d in range(0, distance + 1, 1 if n < 64 else 37):
        assert orc.bucket_of(d, n, distance) == max(b for b in range(n) if starts[b] <= d), d


def test_bucket_starts_of_the_usual_table():
    assert relative_bucket_starts(16, 128) == (0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91)


@pytest.mark.parametrize("n,distance", [(1, 8), (257, 512), (8, 4), (8, 1025)])
def test_bucket_starts_refused(n, distance):
    with pytest.raises(ValueError):
        relative_bucket_starts(n, distance)


def test_oracle_gradients_are_those_of_differences():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    x = {"q": r(2, 5, 4, 16), "k": r(2, 7, 2, 16), "v": r(2, 7, 2, 16), "table": r(6, 4)}
    options = dict(max_distance=5, bidirectional=True, key_lengths=torch.tensor([7, 3]), query_lengths=torch.tensor([4, 5]), start=1)
    dO = r(2, 5, 4, 16)
    values, sizes = orc.attention(**x, dO=dO, **options)
    f = lambda **y: (orc.attention(**{**x, **y}, **options)[0]["o"] * dO).sum()
    for n in x:
        step = r(*x[n].shape)
        slope = (f(**{n: x[n] + 1e-5 * step}) - f(**{n: x[n] - 1e-5 * step})) / 2e-5
        assert abs(float((values["d" + n] * step).sum() - slope)) < 1e-7
        assert bool((values["d" + n].abs() <= sizes["d" + n][0] * (1 + 1e-12)).all())


def test_oracle_is_torch_attention_where_nothing_is_hidden():
    q, k = torch.randn(2, 6, 3, 32, dtype=torch.float64), torch.randn(2, 9, 3, 32, dtype=torch.float64)
    want = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, k))).transpose(1, 2)
    assert torch.allclose(orc.attention(q, k, k)[0]["o"], want, atol=1e-12)


class _Gpu(torch.Tensor):
    """A host tensor that says it is on the GPU, for checks that come before any launch."""
    is_cuda = True


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Gpu)


@pytest.mark.parametrize("error,call", [
    (RuntimeError, lambda: cross_attention(torch.zeros(1, 2, 2, 32, dtype=torch.bfloat16), *[torch.zeros(1, 2, 2, 32, dtype=torch.bfloat16)] * 2)),
    (AssertionError, lambda: context_forward(_t(1, 2, 32), _t(1, 2, 32), _t(1, 2, 32))),
    (TypeError, lambda: context_forward(*[_t(1, 2, 3, 32, dtype=torch.float32)] * 3)),
    (ValueError, lambda: context_forward(*[_t(1, 2, 3, 8)] * 3)),
    (ValueError, lambda: context_forward(*[_t(1, 2, 3, 136)] * 3)),
    (AssertionError, lambda: context_forward(_t(1, 3, 3, 32), _t(1, 2, 3, 32), _t(1, 2, 3, 32))),
    (AssertionError, lambda: context_forward(_t(1, 2, 3, 32), _t(1, 2, 3, 32), _t(1, 2, 4, 32))),
    (AssertionError, lambda: context_forward(_t(1, 2, 3, 32), _t(2, 2, 3, 32), _t(2, 2, 3, 32))),
    (TypeError, lambda: context_forward(_t(1, 2, 3, 32), *[_t(1, 2, 3, 32, dtype=torch.float16)] * 2)),
    (AssertionError, lambda: context_forward(_t(1, 2, 32, 3).transpose(2, 3), *[_t(1, 2, 3, 32)] * 2)),
    (TypeError, lambda: context_forward(*[_t(1, 2, 3, 32)] * 3, key_lengths=_t(1, dtype=torch.int64))),
    (AssertionError, lambda: context_forward(*[_t(1, 2, 3, 32)] * 3, key_lengths=_t(2, dtype=torch.int32))),
    (TypeError, lambda: context_forward(*[_t(1, 2, 3, 32)] * 3, query_lengths=_t(1, dtype=torch.float32))),
    (AssertionError, lambda: context_forward(*[_t(1, 2, 3, 32)] * 3, query_start=_t(1, 1, dtype=torch.int32))),
    (ValueError, lambda: context_forward(*[_t(1, 2, 3, 32)] * 3, query_start=1 << 30)),
    (ValueError, lambda: context_forward(_t(1, 2, 3, 32), *[_t(1, 2, 1, 32).expand(1, 2, (1 << 32) + 3, 32)] * 2)),
    (ValueError, lambda: context_forward(*[_t(1, 2, 3, 32)] * 3, scale=-1.0)),
    (AssertionError, lambda: context_forward(*[_t(1, 2, 3, 32)] * 3, bias=RelativeBias(_t(8, 3)))),
    (ValueError, lambda: RelativeBias(_t(7, 2))),
    (TypeError, lambda: RelativeBias(_t(8, 2, dtype=torch.int32))),
    (AssertionError, lambda: RelativeBias(_t(8))),
    (ValueError, lambda: RelativeBias(_t(8, 2), max_distance=1)),
])
def test_refusals(error, call):
    with pytest.raises(error):
        call()


def _ctx(**fields):
    t = _lib.Ctx()
    t.B, t.Hq, t.Hkv, t.Lq, t.Lk, t.D = 2, 4, 2, 8, 8, 64
    for n in _lib.C_TENSORS:
        setattr(t, n, 64)  # never read: every call below is refused before a launch
    t.lse = 64
    for n, value in fields.items():
        setattr(t, n, value)
    return t


@pytest.mark.parametrize("status,fields", [
    (_lib.SJVP_ERR_SHAPE, dict(B=0)), (_lib.SJVP_ERR_SHAPE, dict(Lk=0)), (_lib.SJVP_ERR_SHAPE, dict(Hkv=3)),
    (_lib.SJVP_ERR_SHAPE, dict(Lq=(1 << 29) + 1)), (_lib.SJVP_ERR_SHAPE, dict(query_start0=-(1 << 30))),
    (_lib.SJVP_ERR_HEAD_DIM, dict(D=15)), (_lib.SJVP_ERR_HEAD_DIM, dict(D=129)),
    (_lib.SJVP_ERR_SCALE, dict(scale=-1.0)), (_lib.SJVP_ERR_SCALE, dict(scale=float("inf"))),
    (_lib.SJVP_ERR_SCALE, dict(scale=float("nan"))), (_lib.SJVP_ERR_NULL, dict(q=None)), (_lib.SJVP_ERR_NULL, dict(o=None)),
    (_lib.SJVP_ERR_BUCKETS, dict(causal=1)), (_lib.SJVP_ERR_BUCKETS, dict(dtable=64)),
    (_lib.SJVP_ERR_NULL, dict(table=64, table_dtype=2)), (_lib.SJVP_ERR_DTYPE, dict(table=64, table_dtype=3)),
])
def test_status_of_the_c_abi(status, fields):
    lib = _lib.load()
    assert lib.sjvp_ctx_fwd(ctypes.byref(_ctx(**fields)), 0, None) == status
    assert lib.sjvp_ctx_bwd(ctypes.byref(_ctx(**fields)), 0, None) == status


def test_status_of_the_c_abi_beyond_the_fields():
    lib = _lib.load()
    assert lib.sjvp_ctx_fwd(None, 0, None) == _lib.SJVP_ERR_NULL
    assert lib.sjvp_ctx_fwd(ctypes.byref(_ctx()), 2, None) == _lib.SJVP_ERR_DTYPE
    assert lib.sjvp_ctx_bwd(ctypes.byref(_ctx(dk=None)), 0, None) == _lib.SJVP_ERR_NULL
    assert lib.sjvp_ctx_bwd(ctypes.byref(_ctx(Lk=300)), 0, None) == _lib.SJVP_ERR_WORKSPACE
    assert lib.sjvp_ctx_bwd(ctypes.byref(_ctx(Lk=300, workspace=64, workspace_bytes=4)), 0, None) == _lib.SJVP_ERR_WORKSPACE
    t = _ctx()
    t.strides[2] = 1 << 24
    assert lib.sjvp_ctx_fwd(ctypes.byref(t), 0, None) == _lib.SJVP_ERR_SHAPE
    for starts in ([1], [0, 5, 4], [0, 1025], list(range(257))):
        first = (ctypes.c_int32 * len(starts))(*starts)
        t = _ctx(table=64, table_dtype=2, buckets=len(starts), bucket_first=ctypes.cast(first, ctypes.c_void_p))
        assert lib.sjvp_ctx_fwd(ctypes.byref(t), 0, None) == _lib.SJVP_ERR_BUCKETS
    # launches of too many workgroups: no work is done, and nothing wraps round
    for sizes in (dict(B=1 << 24), dict(B=1 << 30), dict(B=(1 << 31) - 1, Lq=1), dict(B=1 << 28, Hq=16, Hkv=16), dict(Lq=1 << 29, B=64, D=96)):
        assert lib.sjvp_ctx_fwd(ctypes.byref(_ctx(**sizes)), 0, None) == _lib.SJVP_ERR_SHAPE, sizes
        assert lib.sjvp_ctx_bwd(ctypes.byref(_ctx(**sizes)), 0, None) == _lib.SJVP_ERR_SHAPE, sizes
    assert b"bias" in lib.sjvp_strerror(_lib.SJVP_ERR_BUCKETS)
