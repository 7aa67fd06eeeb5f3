"""The host extension serves packed sequences and the paged cache exactly as the general form of the entry points does, and leaves what it does
not serve to the general form's errors."""
import pytest
import torch

from semicat_amd import PagedCache, packed, packed_attention, paged, paged_attention, paged_read, paged_write

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture
def general(monkeypatch):
    def switch():
        for module in (packed, paged):
            monkeypatch.setattr(module, "_on_gpu", lambda q: False)
    return switch


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def normal(*shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.stride() == y.stride() and torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("H,G,D,dtype,causal,scale", [(4, 2, 64, BF16, True, None), (2, 1, 33, FP16, False, 0.3), (8, 8, 128, BF16, True, None),
                                                       (2, 1, 64, torch.float32, True, None), (3, 3, 48, torch.float64, False, None)])
def test_packed_attention(general, H, G, D, dtype, causal, scale):
    offsets = ints(3, 50, 50, 181)
    q, k, v, dO = (normal(190, h, D, dtype=dtype, seed=i) for i, h in enumerate((H, H // G, H // G, H)))

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = packed_attention(*leaves, offsets, causal, scale)
        with torch.no_grad():
            plain = packed_attention(*leaves, offsets, causal=causal, scale=scale)
        return [o.detach(), plain, *torch.autograd.grad(o, leaves, dO)]

    first = run()
    general()
    same(first, run())


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("dtype,given", [(BF16, BF16), (FP16, FP16), (BF16, torch.float32)])
def test_paged_cache(general, dtype, given, quantized):
    tables, lengths, offsets = ints([4, 2, -1], [0, 5, 1], [3, -1, -1]), ints(20, 33, 7), ints(1, 6, 39, 40)
    new, q = [normal(41, 2, 64, dtype=given, seed=i) for i in (1, 2)], normal(41, 6, 64, dtype=given, seed=3)

    def run():
        cache = PagedCache(6, 16, 2, 64, dtype, quantized)
        paged_write(cache, *new, tables, lengths, offsets)
        paged_write(cache, new[0][:3], new[1][:3], tables, lengths)
        out = [cache.k, cache.v, *paged_read(cache, tables, lengths, 40), paged_attention(q, cache, tables, lengths, offsets),
               paged_attention(q[:3], cache, tables, lengths, scale=0.2)]
        return out + ([cache.k_scales, cache.v_scales] if quantized else [])

    first = run()
    general()
    same(first, run())


def both_ways(general, error, call):
    with pytest.raises(error):
        call()
    general()
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("error,spoil", [
    (TypeError, lambda a: a.__setitem__("offsets", a["offsets"].long())), (ValueError, lambda a: a.__setitem__("offsets", a["offsets"].cpu())),
    (ValueError, lambda a: a.__setitem__("k", a["k"].cpu())), (TypeError, lambda a: a.__setitem__("v", a["v"].half())),
    (AssertionError, lambda a: a.__setitem__("k", a["k"][:, :1])), (AssertionError, lambda a: a.__setitem__("q", a["q"][:9])),
    (AssertionError, lambda a: a.__setitem__("q", a["q"].transpose(1, 2).contiguous().transpose(1, 2))),
    (ValueError, lambda a: a.__setitem__("scale", -1.0)), (ValueError, lambda a: [a.__setitem__(n, a[n][..., :8]) for n in "qkv"]),
])
def test_refusals_of_packed_attention(general, error, spoil):
    a = {n: normal(20, 2, 32, dtype=BF16) for n in "qkv"} | {"offsets": ints(0, 20)}
    spoil(a)
    both_ways(general, error, lambda: packed_attention(**a))


@pytest.mark.parametrize("error,spoil", [
    (TypeError, lambda a: a.__setitem__("tables", a["tables"].long())), (ValueError, lambda a: a.__setitem__("tables", a["tables"].cpu())),
    (TypeError, lambda a: a.__setitem__("lengths", a["lengths"].long())), (AssertionError, lambda a: a.__setitem__("lengths", a["lengths"][:1])),
    (AssertionError, lambda a: a.__setitem__("offsets", None)), (AssertionError, lambda a: a.__setitem__("offsets", a["offsets"][:2])),
    (AssertionError, lambda a: a.__setitem__("x", a["x"][:, :1])), (AssertionError, lambda a: a.__setitem__("x", a["x"][..., :16])),
    (RuntimeError, lambda a: a.__setitem__("x", a["x"].cpu())), (NotImplementedError, lambda a: a["x"].requires_grad_()),
])
def test_refusals_of_the_paged_cache(general, error, spoil):
    cache = PagedCache(4, 8, 2, 32)
    a = {"tables": ints([0, 1], [2, 3]), "lengths": ints(9, 7), "offsets": ints(0, 5, 8), "x": normal(8, 2, 32, dtype=BF16)}
    spoil(a)
    rest = (a["tables"], a["lengths"], a["offsets"])
    if error is RuntimeError:  # (q is looked at first, k behind the cache)
        with pytest.raises(ValueError):
            paged_write(cache, a["x"], a["x"], *rest)
    else:
        both_ways(general, error, lambda: paged_write(cache, a["x"], a["x"], *rest))
    both_ways(general, error, lambda: paged_attention(a["x"], cache, *rest))


def test_no_double_backward(general):
    for _ in range(2):
        q = normal(20, 2, 32, dtype=BF16).requires_grad_()
        d, = torch.autograd.grad(packed_attention(q, q, q, ints(0, 20)).float().sum(), [q], create_graph=True)
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.autograd.grad(d.float().sum(), [q])
        general()


def test_no_forward_mode(general):
    import torch.autograd.forward_ad as fwAD
    q, cache = normal(2, 2, 32, dtype=BF16), PagedCache(4, 8, 2, 32)
    for _ in range(2):
        with fwAD.dual_level():
            dual = fwAD.make_dual(q, q)
            for call in (lambda: packed_attention(dual, q, q, ints(0, 2)), lambda: paged_attention(dual, cache, ints([0], [1]), ints(1, 1)),
                         lambda: paged_write(cache, q, dual, ints([0], [1]), ints(1, 1))):
                with pytest.raises(NotImplementedError):
                    call()
        general()


def test_calls_without_rows():
    q = torch.empty(0, 2, 32, dtype=BF16, device="cuda").requires_grad_()
    o = packed_attention(q, q, q, ints(0, 0))
    assert o.shape == q.shape and torch.autograd.grad(o.sum(), [q])[0].shape == q.shape
    cache = PagedCache(4, 8, 2, 32)
    assert paged_attention(q.detach(), cache, ints([0], [1]), ints(1, 1), ints(0, 0, 0)).shape == q.shape
    paged_write(cache, q.detach(), q.detach(), ints([0], [1]), ints(1, 1), ints(0, 0, 0))
    assert paged_read(cache, ints([0]), ints(3), 0)[0].shape == (1, 0, 2, 32)
    assert not cache.k.any()
