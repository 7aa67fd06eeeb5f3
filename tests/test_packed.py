"""CPU tests of the attention over packed sequences and of the paged cache: the oracle, refusals, the C ABI's checks."""
import ctypes
import math

import pytest
import torch

import semicat_amd
from oracle import packed_oracle as orc
from semicat_amd import PagedCache, _lib, packed, paged, packed_attention, packed_backward, packed_forward, paged_attention, paged_read, paged_write

BF16, FP16, FP8, E8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def test_entry_points_are_public():
    for name in ("packed_attention", "packed_forward", "packed_backward", "PagedCache", "paged_write", "paged_read", "paged_attention"):
        assert name in semicat_amd.__all__ and getattr(semicat_amd, name).__doc__, name


def test_oracle_gradients_are_those_of_differences():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    x, dO, offsets = {"q": r(11, 4, 16), "k": r(11, 2, 16), "v": r(11, 2, 16)}, r(11, 4, 16), [1, 6, 6, 10]
    for causal in (True, False):
        values, sizes = orc.packed(**x, offsets=offsets, causal=causal, dO=dO)
        f = lambda **y: (orc.packed(**{**x, **y}, offsets=offsets, causal=causal)[0]["o"] * dO).sum()
        for n in x:
            step = r(*x[n].shape)
            slope = (f(**{n: x[n] + 1e-5 * step}) - f(**{n: x[n] - 1e-5 * step})) / 2e-5
            assert abs(float((values["d" + n] * step).sum() - slope)) < 1e-7
            assert bool((values["d" + n].abs() <= sizes["d" + n][0] * (1 + 1e-12)).all())


def test_oracle_is_torch_attention():
    q, k, v = (torch.randn(9, h, 32, dtype=torch.float64) for h in (4, 2, 2))
    for causal in (True, False):
        got = orc.packed(q, k, v, [0, 4, 9], causal)[0]["o"]
        for s, e in ((0, 4), (4, 9)):
            want = torch.nn.functional.scaled_dot_product_attention(q[s:e].transpose(0, 1), *(t[s:e].repeat_interleave(2, 1).transpose(0, 1) for t in (k, v)),
                                                                    is_causal=causal).transpose(0, 1)
            assert torch.allclose(got[s:e], want, atol=1e-12)
    # one new token on a cache is the last row of a causal pass
    last = orc.paged(q[8:], [k], [v], [9], [0, 1])[0]
    assert torch.allclose(last[0], orc.packed(q, k, v, [0, 9], True)[0]["o"][8], atol=1e-12)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_oracle_numbers_of_eight_bits(dtype):
    values = orc.e4m3_values()
    torch_values = torch.arange(256).to(torch.uint8).view(FP8).double()
    assert torch.equal(values.nan_to_num(nan=1e9), torch_values.nan_to_num(nan=1e9))
    rows = (torch.randn(40, 3, 2, 80, generator=torch.Generator().manual_seed(1)) * torch.logspace(-6, 4, 40)[:, None, None, None]).to(dtype)
    codes, powers = orc.quantise(rows)
    assert codes.shape == rows.shape and powers.shape == (40, 3, 2, 3)
    scale = torch.exp2(powers.double() - 127).repeat_interleave(32, -1)[..., :80]
    back = torch_values[codes.long()] * scale
    assert bool((back.to(dtype).double() == back).all())  # exactly numbers of the type
    off = (back - rows.double()).abs()
    clipped = rows.double().abs() > 240 * scale if dtype == FP16 else torch.zeros_like(off, dtype=torch.bool)
    assert bool(((off <= torch.maximum(rows.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)) | clipped).all())


class _Gpu(torch.Tensor):
    """A host tensor that says it is on the GPU, for checks that come before any launch."""
    is_cuda = True


def _t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Gpu)


def _i(*shape, dtype=torch.int32):
    return _t(*shape, dtype=dtype)


def _q(T=6, H=2, D=32, dtype=BF16):
    return _t(T, H, D, dtype=dtype)


@pytest.fixture(autouse=True)
def _general_form(monkeypatch):
    for module in (packed, paged):
        monkeypatch.setattr(module, "_on_gpu", lambda q: False)


@pytest.mark.parametrize("error,call", [
    (RuntimeError, lambda: packed_attention(*[torch.zeros(6, 2, 32, dtype=BF16)] * 3, torch.zeros(2, dtype=torch.int32))),
    (AssertionError, lambda: packed_forward(_t(6, 32), _t(6, 32), _t(6, 32), _i(2))),
    (AssertionError, lambda: packed_forward(_t(1, 6, 2, 32), *[_q()] * 2, _i(2))),
    (TypeError, lambda: packed_forward(*[_q(dtype=torch.float32)] * 3, _i(2))),
    (ValueError, lambda: packed_forward(*[_q(D=8)] * 3, _i(2))),
    (ValueError, lambda: packed_forward(*[_q(D=136)] * 3, _i(2))),
    (AssertionError, lambda: packed_forward(_q(H=3), *[_q()] * 2, _i(2))),
    (AssertionError, lambda: packed_forward(_q(), *[_q(H=0)] * 2, _i(2))),
    (AssertionError, lambda: packed_forward(_q(), *[_q(T=7)] * 2, _i(2))),
    (AssertionError, lambda: packed_forward(_q(), _q(), _q(H=1), _i(2))),
    (AssertionError, lambda: packed_forward(_q(), _q(D=16), _q(D=16), _i(2))),
    (TypeError, lambda: packed_forward(_q(), *[_q(dtype=FP16)] * 2, _i(2))),
    (AssertionError, lambda: packed_forward(_t(6, 32, 2).transpose(1, 2), *[_q()] * 2, _i(2))),
    (ValueError, lambda: packed_forward(_t(1, 1, 32).expand((1 << 29) + 1, 1, 32), *[_t(1, 1, 32).expand((1 << 29) + 1, 1, 32)] * 2, _i(2))),
    (TypeError, lambda: packed_forward(*[_q()] * 3, _i(2, dtype=torch.int64))),
    (AssertionError, lambda: packed_forward(*[_q()] * 3, _i(1))),
    (AssertionError, lambda: packed_forward(*[_q()] * 3, _i(1, 2))),
    (AssertionError, lambda: packed_forward(*[_q()] * 3, _i(4)[::2])),
    (ValueError, lambda: packed_forward(*[_q()] * 3, _i(2), scale=0.0)),
    (ValueError, lambda: packed_forward(*[_q()] * 3, _i(2), scale=math.inf)),
    (ValueError, lambda: packed_forward(*[_q()] * 3, _i(2), scale=math.nan)),
    (AssertionError, lambda: packed_backward(*[_q()] * 4, _t(2, 6, 1, dtype=torch.float32), _q(), _i(2))),
    (AssertionError, lambda: packed_backward(*[_q()] * 4, _t(2, 6, 2), _q(), _i(2))),
    (AssertionError, lambda: packed_backward(*[_q()] * 3, _q(T=5), _t(2, 6, 2, dtype=torch.float32), _q(), _i(2))),
    (TypeError, lambda: packed_backward(*[_q()] * 4, _t(2, 6, 2, dtype=torch.float32), _q(dtype=FP16), _i(2))),
])
def test_refusals_of_packed_sequences(error, call):
    with pytest.raises(error):
        call()


def test_no_higher_derivatives_of_packed_sequences():
    import torch.autograd.forward_ad as fwAD
    q = torch.zeros(6, 2, 32, dtype=BF16)
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        packed_attention(fwAD.make_dual(q, q), q, q, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(NotImplementedError):
        packed.PackedAttentionBackwardFunction.backward(None)


def _cache(pages=4, size=8, heads=2, D=32, dtype=BF16, scales=False):
    if not scales:
        return PagedCache.of(_t(pages, heads, size, D, dtype=dtype), _t(pages, heads, size, D, dtype=dtype))
    new = lambda d, t: torch.zeros(pages, heads, size, d, dtype=torch.uint8).view(t).as_subclass(_Gpu)
    return PagedCache.of(new(D, FP8), new(D, FP8), new(-(-D // 32), E8), new(-(-D // 32), E8), dtype)


def test_cache_of_the_caller_s_tensors():
    cache = _cache(scales=True, D=80, dtype=FP16)
    assert (cache.pages, cache.heads, cache.page_size, cache.head_dim, cache.quantized, cache.dtype) == (4, 2, 8, 80, True, FP16)
    assert cache._strides == (2 * 8 * 80, 8 * 80, 80, 2 * 8 * 3, 8 * 3, 3)
    assert not _cache().quantized and _cache(dtype=FP16).dtype == FP16
    # [pages, size, heads, D] in memory, one page alone, and the scales as plain bytes
    wide = torch.zeros(4, 8, 2, 32, dtype=BF16).transpose(1, 2)
    assert PagedCache.of(wide, wide)._strides[:3] == (2 * 8 * 2 * 32, 64, 128)
    assert PagedCache.of(wide[:1], wide[1:2])._strides[0] == 0
    bytes_ = torch.zeros(4, 2, 8, 1, dtype=torch.uint8)
    assert PagedCache.of(*[torch.zeros(4, 2, 8, 32, dtype=torch.uint8).view(FP8)] * 2, bytes_, bytes_).dtype == BF16
    new = PagedCache(3, 5, 2, 48, quantized=True, device="cpu")
    assert new.k.shape == (3, 2, 5, 48) and new.k.dtype == FP8 and new.v_scales.shape == (3, 2, 5, 2) and not new.k.view(torch.uint8).any()


@pytest.mark.parametrize("error,call", [
    (AssertionError, lambda: PagedCache.of(_t(2, 8, 32), _t(2, 8, 32))),
    (AssertionError, lambda: PagedCache.of(_t(4, 2, 8, 32), _t(4, 2, 9, 32))),
    (TypeError, lambda: PagedCache.of(_t(4, 2, 8, 32), _t(4, 2, 8, 32, dtype=FP16))),
    (TypeError, lambda: PagedCache.of(*[_t(4, 2, 8, 32, dtype=torch.float32)] * 2)),
    (TypeError, lambda: PagedCache.of(*[_t(4, 2, 8, 32)] * 2, dtype=FP16)),
    (TypeError, lambda: PagedCache.of(*[torch.zeros(4, 2, 8, 32, dtype=torch.uint8).view(FP8)] * 2)),
    (AssertionError, lambda: PagedCache.of(*[torch.zeros(4, 2, 8, 32, dtype=torch.uint8).view(FP8)] * 2, _i(4, 2, 8, 1, dtype=torch.uint8))),
    (TypeError, lambda: PagedCache.of(*[_t(4, 2, 8, 32)] * 2, *[_i(4, 2, 8, 1, dtype=torch.uint8)] * 2)),
    (TypeError, lambda: PagedCache.of(*[torch.zeros(4, 2, 8, 32, dtype=torch.uint8).view(FP8)] * 2, *[torch.zeros(4, 2, 8, 1)] * 2)),
    (AssertionError, lambda: PagedCache.of(*[torch.zeros(4, 2, 8, 48, dtype=torch.uint8).view(FP8)] * 2, *[torch.zeros(4, 2, 8, 1, dtype=torch.uint8)] * 2)),
    (ValueError, lambda: _cache(D=8)), (ValueError, lambda: _cache(D=136)), (ValueError, lambda: _cache(D=20)),
    (ValueError, lambda: _cache(D=24, scales=True)), (ValueError, lambda: _cache(pages=0)), (ValueError, lambda: _cache(size=0)),
    (AssertionError, lambda: PagedCache.of(*[_t(4, 2, 8, 36)[..., :32]] * 2)),           # rows 72 bytes apart
    (AssertionError, lambda: PagedCache.of(*[_t(4, 2, 8, 40)[..., 4:36]] * 2)),          # 8 bytes off
    (AssertionError, lambda: PagedCache.of(_t(4, 2, 8, 32), _t(4, 8, 2, 32).transpose(1, 2))),
    (AssertionError, lambda: PagedCache.of(*[_t(4, 2, 32, 8).transpose(2, 3)] * 2)),
    (AssertionError, lambda: PagedCache.of(*[torch.empty_strided((2, 2, 8, 32), (1 << 31, 256, 32, 1), dtype=BF16, device="meta")] * 2)),
    (AssertionError, lambda: PagedCache.of(*[torch.empty_strided((2, 2, 8, 32), (256, 512, 1 << 31, 1), dtype=BF16, device="meta")] * 2)),
    (RuntimeError, lambda: paged_read(PagedCache(4, 8, 2, 32, device="cpu"), _i(3, 2), _i(3), 4)),
    (AssertionError, lambda: paged_read(_cache(), _i(3), _i(3), 4)),
    (TypeError, lambda: paged_read(_cache(), _i(3, 2, dtype=torch.int64), _i(3), 4)),
    (AssertionError, lambda: paged_read(_cache(), _i(3, 4)[:, ::2], _i(3), 4)),
    (AssertionError, lambda: paged_read(_cache(), _i(3, 0), _i(3), 4)),
    (AssertionError, lambda: paged_read(_cache(), _i(3, 2), _i(2), 4)),
    (TypeError, lambda: paged_read(_cache(), _i(3, 2), _i(3, dtype=torch.int64), 4)),
    (AssertionError, lambda: paged_attention(_q(T=4), _cache(), _i(3, 2), _i(3))),
    (AssertionError, lambda: paged_attention(_q(), _cache(), _i(3, 2), _i(3), _i(3))),
    (TypeError, lambda: paged_attention(_q(), _cache(), _i(3, 2), _i(3), _i(4, dtype=torch.int64))),
    (AssertionError, lambda: paged_attention(_q(H=3), _cache(), _i(3, 2), _i(3), _i(4))),
    (AssertionError, lambda: paged_attention(_q(D=64), _cache(), _i(3, 2), _i(3), _i(4))),
    (AssertionError, lambda: paged_attention(_t(6, 64), _cache(), _i(3, 2), _i(3), _i(4))),
    (ValueError, lambda: paged_attention(_q(), _cache(), _i(3, 2), _i(3), _i(4), scale=-1.0)),
    (NotImplementedError, lambda: paged_attention(_q().requires_grad_(), _cache(), _i(3, 2), _i(3), _i(4))),
    (NotImplementedError, lambda: paged_write(_cache(), _q(), _q().requires_grad_(), _i(3, 2), _i(3), _i(4))),
    (AssertionError, lambda: paged_write(_cache(), _t(6, 64), _q(), _i(3, 2), _i(3), _i(4))),
    (AssertionError, lambda: paged_write(_cache(), _q(), _q(T=5), _i(3, 2), _i(3), _i(4))),
    (AssertionError, lambda: paged_write(_cache(), _q(H=4), _q(H=4), _i(3, 2), _i(3), _i(4))),
    (AssertionError, lambda: paged_write(_cache(), _q(T=4), _q(T=4), _i(3, 2), _i(3))),
])
def test_refusals_of_the_paged_cache(error, call):
    with pytest.raises(error):
        call()


def _packed(**fields):
    t = _lib.Packed()
    t.B, t.T, t.Hq, t.Hkv, t.D = 3, 40, 4, 2, 64
    for n in _lib.S_TENSORS:
        setattr(t, n, 64)  # never read: every call below is refused before a launch
    t.lse = t.offsets = 64
    for n, value in fields.items():
        setattr(t, n, value)
    return t


@pytest.mark.parametrize("status,fields", [
    (_lib.SJVP_ERR_SHAPE, dict(B=0)), (_lib.SJVP_ERR_SHAPE, dict(T=0)), (_lib.SJVP_ERR_SHAPE, dict(Hkv=0)), (_lib.SJVP_ERR_SHAPE, dict(Hkv=3)),
    (_lib.SJVP_ERR_SHAPE, dict(B=(1 << 29) + 1)), (_lib.SJVP_ERR_SHAPE, dict(T=(1 << 29) + 1)), (_lib.SJVP_ERR_SHAPE, dict(T=1 << 29)),
    (_lib.SJVP_ERR_SHAPE, dict(B=1 << 24)),                                     # launches of too many workgroups
    (_lib.SJVP_ERR_HEAD_DIM, dict(D=15)), (_lib.SJVP_ERR_HEAD_DIM, dict(D=129)),
    (_lib.SJVP_ERR_SCALE, dict(scale=-1.0)), (_lib.SJVP_ERR_SCALE, dict(scale=math.inf)), (_lib.SJVP_ERR_SCALE, dict(scale=math.nan)),
    (_lib.SJVP_ERR_NULL, dict(q=None)), (_lib.SJVP_ERR_NULL, dict(v=None)), (_lib.SJVP_ERR_NULL, dict(o=None)), (_lib.SJVP_ERR_NULL, dict(offsets=None)),
])
def test_status_of_packed_sequences(status, fields):
    lib = _lib.load()
    assert lib.sjvp_packed_fwd(ctypes.byref(_packed(**fields)), 0, None) == status
    assert lib.sjvp_packed_bwd(ctypes.byref(_packed(**fields)), 0, None) == status


def test_status_of_packed_sequences_beyond_the_fields():
    lib = _lib.load()
    assert lib.sjvp_packed_fwd(None, 0, None) == lib.sjvp_packed_bwd(None, 0, None) == _lib.SJVP_ERR_NULL
    assert lib.sjvp_packed_fwd(ctypes.byref(_packed()), 2, None) == lib.sjvp_packed_bwd(ctypes.byref(_packed()), 2, None) == _lib.SJVP_ERR_DTYPE
    for fields in (dict(dO=None), dict(dq=None), dict(lse=None), dict(dk=None), dict(dv=None)):
        assert lib.sjvp_packed_bwd(ctypes.byref(_packed(**fields)), 0, None) == _lib.SJVP_ERR_NULL, fields
    need = lib.sjvp_packed_workspace_bytes(ctypes.byref(_packed()), 1)
    assert need >= 3 * 4 * 40 * 4 and lib.sjvp_packed_workspace_bytes(ctypes.byref(_packed()), 0) == 0
    assert lib.sjvp_packed_workspace_bytes(ctypes.byref(_packed(D=200)), 1) == 0 and lib.sjvp_packed_workspace_bytes(None, 1) == 0
    for fields in (dict(), dict(workspace=64, workspace_bytes=need - 1), dict(workspace=72, workspace_bytes=need)):
        assert lib.sjvp_packed_bwd(ctypes.byref(_packed(**fields)), 0, None) == _lib.SJVP_ERR_WORKSPACE, fields
    for i in (0, 1, 2):
        t = _packed()
        t.strides[2 * i + 1] = 1 << 24
        assert lib.sjvp_packed_fwd(ctypes.byref(t), 0, None) == _lib.SJVP_ERR_SHAPE
        t.strides[2 * i + 1] = -64
        assert lib.sjvp_packed_fwd(ctypes.byref(t), 0, None) == _lib.SJVP_ERR_SHAPE
    # the sums of the column-owned launch are split where there are few blocks of keys, and over heads alone
    size = lambda **f: lib.sjvp_packed_workspace_bytes(ctypes.byref(_packed(**f)), 1)
    assert size(Hkv=4) == 4 * 3 * 4 * 40 < size()


def _pages(**fields):
    t = _lib.Paged()
    t.B, t.T, t.Hq, t.Hkv, t.D, t.size = 3, 3, 4, 2, 64, 8
    t.pages, t.page_size, t.table_pages, t.table_stride = 9, 16, 4, 4
    for n in (*_lib.P_TENSORS, "k_pages", "v_pages", "tables", "lengths"):
        setattr(t, n, 64)
    for n, value in fields.items():
        setattr(t, n, value)
    return t


CALLS = ("sjvp_paged_write", "sjvp_paged_read", "sjvp_paged_attention")


@pytest.mark.parametrize("status,fields", [
    (_lib.SJVP_ERR_SHAPE, dict(B=0)), (_lib.SJVP_ERR_SHAPE, dict(Hkv=0)), (_lib.SJVP_ERR_SHAPE, dict(Hkv=3)), (_lib.SJVP_ERR_SHAPE, dict(B=(1 << 29) + 1)),
    (_lib.SJVP_ERR_HEAD_DIM, dict(D=8)), (_lib.SJVP_ERR_HEAD_DIM, dict(D=136)), (_lib.SJVP_ERR_SCALE, dict(scale=math.nan)),
    (_lib.SJVP_ERR_PAGES, dict(pages=0)), (_lib.SJVP_ERR_PAGES, dict(page_size=0)), (_lib.SJVP_ERR_PAGES, dict(table_pages=0)),
    (_lib.SJVP_ERR_PAGES, dict(page_size=(1 << 29) + 1)), (_lib.SJVP_ERR_PAGES, dict(D=36)), (_lib.SJVP_ERR_PAGES, dict(D=40, k_scales=64, v_scales=64)),
    (_lib.SJVP_ERR_PAGES, dict(k_pages=72)), (_lib.SJVP_ERR_PAGES, dict(v_pages=68)),
    (_lib.SJVP_ERR_NULL, dict(k_pages=None)), (_lib.SJVP_ERR_NULL, dict(tables=None)), (_lib.SJVP_ERR_NULL, dict(lengths=None)),
    (_lib.SJVP_ERR_NULL, dict(k_scales=64)), (_lib.SJVP_ERR_NULL, dict(v_scales=64)),
])
def test_status_of_the_paged_cache(status, fields):
    lib = _lib.load()
    for fn in CALLS:
        assert getattr(lib, fn)(ctypes.byref(_pages(**fields)), 0, None) == status, fn


def test_status_of_the_paged_cache_beyond_the_fields():
    lib = _lib.load()
    call = lambda fn, dtype=0, **f: getattr(lib, "sjvp_paged_" + fn)(ctypes.byref(_pages(**f)), dtype, None)
    for fn in CALLS:
        assert getattr(lib, fn)(None, 0, None) == _lib.SJVP_ERR_NULL
    for fn in ("write", "read", "attention"):
        assert call(fn, 2) == _lib.SJVP_ERR_DTYPE
    for i in (0, 2, 3, 5):
        for stride in (1 << 32, -16):
            t = _pages(k_scales=64, v_scales=64)
            t.page_strides[i] = stride
            assert lib.sjvp_paged_read(ctypes.byref(t), 0, None) == _lib.SJVP_ERR_PAGES
    for stride, status in ((8, _lib.SJVP_ERR_PAGES), (-16, _lib.SJVP_ERR_PAGES)):
        for i in range(3):
            t = _pages()
            t.page_strides[i] = stride
            assert lib.sjvp_paged_read(ctypes.byref(t), 0, None) == status
    assert call("write", k=None) == call("read", v=None) == call("attention", q=None) == call("attention", o=None) == _lib.SJVP_ERR_NULL
    assert call("write", T=4) == call("attention", T=4) == _lib.SJVP_ERR_NULL           # without offsets: one token each
    assert call("write", T=0) == call("attention", T=0) == _lib.SJVP_ERR_SHAPE
    assert call("read", size=0) == call("read", size=1 << 30) == call("read", B=1 << 20, size=1 << 20) == _lib.SJVP_ERR_SHAPE
    # launches of too many threads
    assert call("write", T=1 << 26, offsets=64) == call("read", B=1 << 13, size=1 << 13) == _lib.SJVP_ERR_SHAPE
    assert call("attention", T=1 << 28, Hq=4, Hkv=4, offsets=64) == _lib.SJVP_ERR_SHAPE
    assert b"page" in lib.sjvp_strerror(_lib.SJVP_ERR_PAGES)
    # few rows on long sequences are split over the keys
    size = lambda **f: lib.sjvp_paged_workspace_bytes(ctypes.byref(_pages(**f)))
    assert size() == 0 and size(pages=0) == 0 and lib.sjvp_paged_workspace_bytes(None) == 0
    need = size(table_pages=4096)
    assert need > 0
    for f in (dict(), dict(workspace=64, workspace_bytes=need - 1), dict(workspace=72, workspace_bytes=need)):
        assert call("attention", table_pages=4096, **f) == _lib.SJVP_ERR_WORKSPACE, f
