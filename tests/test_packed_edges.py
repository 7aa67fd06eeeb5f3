"""CPU tests of the packed sequences and the paged cache: gradients that are not there raise, a write is a change in place, calls without query rows."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from semicat_amd import PagedCache, packed, packed_attention, packed_backward, packed_forward, paged, paged_attention, paged_read, paged_write
from tests.test_packed import BF16, E8, FP8, _Gpu, _i, _q, _t


@pytest.fixture(autouse=True)
def _general_form(monkeypatch):
    monkeypatch.setattr(paged, "_on_gpu", lambda q: False)


def _storage(scales):
    if not scales:
        return [_t(4, 2, 8, 32), _t(4, 2, 8, 32)]
    return [torch.zeros(4, 2, 8, d, dtype=torch.uint8).view(t).as_subclass(_Gpu) for d, t in ((32, FP8), (32, FP8), (1, E8), (1, E8))]


CALLS = {"attention": lambda cache: paged_attention(_q(), cache, _i(3, 2), _i(3), _i(4)), "read": lambda cache: paged_read(cache, _i(3, 2), _i(3), 4),
         "write": lambda cache: paged_write(cache, _q(), _q(), _i(3, 2), _i(3), _i(4))}


@pytest.mark.parametrize("which", range(2))
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("scales", [False, True])
def test_no_gradient_through_the_cache(monkeypatch, call, scales, which):
    launched = []
    monkeypatch.setattr(paged, "_launch", lambda *a: launched.append(a))
    tensors = _storage(scales)
    tensors[which].requires_grad_()
    cache = PagedCache.of(*tensors)
    with pytest.raises(NotImplementedError):
        CALLS[call](cache)
    assert not launched
    with torch.no_grad():
        CALLS[call](cache)
    assert len(launched) == 1


@pytest.mark.parametrize("which", range(2))
@pytest.mark.parametrize("call", CALLS)
def test_no_forward_mode_through_the_cache(monkeypatch, call, which):
    monkeypatch.setattr(paged, "_launch", lambda *a: pytest.fail("launched"))
    tensors = [torch.zeros(4, 2, 8, 32, dtype=BF16) for _ in range(2)]
    with fwAD.dual_level():
        tensors[which] = fwAD.make_dual(tensors[which], torch.ones_like(tensors[which]))
        cache = PagedCache.of(*tensors)
        with pytest.raises(NotImplementedError):
            CALLS[call](cache)


def test_dual_levels_without_tangents(monkeypatch):
    """Tensors of 8 bits have none, and are looked at all the same."""
    launched = []
    monkeypatch.setattr(paged, "_launch", lambda *a: launched.append(a))
    with fwAD.dual_level():
        for call in CALLS.values():
            for scales in (False, True):
                call(PagedCache.of(*_storage(scales)))
    assert len(launched) == 6


@pytest.mark.parametrize("scales", [False, True])
def test_a_write_counts_as_a_change_in_place(monkeypatch, scales):
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    tensors = _storage(scales)
    cache = PagedCache.of(*tensors)
    versions = lambda: [t._version for t in tensors]
    before = versions()
    paged_attention(_q(), cache, _i(3, 2), _i(3), _i(4)), paged_read(cache, _i(3, 2), _i(3), 4)
    paged_write(cache, _q(T=0), _q(T=0), _i(3, 2), _i(3), _i(4))
    assert versions() == before
    paged_write(cache, _q(), _q(), _i(3, 2), _i(3), _i(4))
    assert all(now > was for now, was in zip(versions(), before))
    with torch.inference_mode():
        kept = PagedCache.of(*_storage(scales))  # (such tensors have no count)
        paged_write(kept, _q(), _q(), _i(3, 2), _i(3), _i(4))


@pytest.fixture
def filled_memory():
    """New tensors hold NaN until they are written."""
    torch.use_deterministic_algorithms(True)
    yield
    torch.use_deterministic_algorithms(False)


@pytest.mark.parametrize("H,T", [(0, 6), (0, 0), (2, 0)])
def test_calls_without_query_rows(filled_memory, H, T):
    """Keys that no query reads have gradients of zero."""
    q, k = _q(T=T, H=H), _q(T=T)
    o, lse = packed_forward(q, k, k, _i(2))
    assert o.shape == (T, H, 32) and lse.shape == (H, T, 2)
    dq, dk, dv = packed_backward(q, k, k, o, lse.as_subclass(_Gpu), _q(T=T, H=H), _i(2))
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
    assert not dk.any() and not dv.any()
    assert packed_backward(q, k, k, o, lse.as_subclass(_Gpu), _q(T=T, H=H), _i(2), with_keys=False)[1:] == (None, None)


def test_training_without_query_heads(filled_memory, monkeypatch):
    monkeypatch.setattr(packed, "_on_gpu", lambda q: False)
    q, k, v = (_q(T=6, H=h).requires_grad_() for h in (0, 2, 2))
    grads = torch.autograd.grad(packed_attention(q, k, v, _i(2)).float().sum(), [q, k, v])
    assert [g.shape for g in grads] == [t.shape for t in (q, k, v)] and not any(g.any() for g in grads)
