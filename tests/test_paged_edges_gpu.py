"""The paged cache at its edges: offsets that descend, lengths beyond the table, NaN among what a row sees, gradients that are not there, the count of
changes in place."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from oracle import packed_oracle as orc
from semicat_amd import PagedCache, paged, paged_attention, paged_read, paged_write
from tests.test_paged_gpu import BF16, attend, cache_of, held_rows, ints, normal, offsets_of, tables_of

pytestmark = pytest.mark.gpu


def bits(cache):
    return [t.view(torch.uint8).cpu().clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("offsets", [[9, 2, 3], [12, 0, 5], [7, 3, -4], [40, 3, 1 << 30], [5, 9, 2]])
def test_offsets_that_descend_reach_no_other_pages(offsets, quantized):
    """Rows of no use, but nothing beside the sequences' own table rows is read and no position behind their lengths is written: the table stands
    between numbers of pages that exist, the pages between others, and both sequences are as long as their table is."""
    size, H, T = 8, 2, 12
    pages = cache_of(20, size, H, 64, BF16, quantized)
    wide = torch.tensor([[10, 11, 1, 2, 12, 13], [14, 15, 3, 4, 16, 17]], dtype=torch.int32).cuda()
    tables = wide[:, 2:4]
    for held in ([2 * size] * 2, [2 * size, 11]):
        before = bits(pages)
        paged_write(pages, normal(T, H, 64, dtype=BF16).cuda(), normal(T, H, 64, dtype=BF16, seed=2).cuda(), tables, ints(held), ints(offsets))
        for was, now in zip(before, bits(pages)):
            changed = (was != now).flatten(3).any(3).any(1)  # [pages, rows]
            for b, n in enumerate(held):
                for x in range(n):
                    changed[tables[b, x // size].item(), x % size] = False
            assert not changed.any()
        o = paged_attention(normal(T, 4, 64, dtype=BF16, seed=3).cuda(), pages, tables, ints(held), ints(offsets))
        torch.cuda.synchronize()
        assert o.shape == (T, 4, 64)


NAN_CASES = [  # held, new, heads, group, head dimension
    ([1, 7, 33, 0, 64, 257], None, 4, 2, 64),                                # seq_few, whole
    ([1, 40, 17], [1, 6, 5], 4, 4, 128),
    ([5000, 1, 3000, 700], None, 8, 4, 128),                                 # split
    ([4000, 6, 900], [4, 9, 2], 8, 2, 64),                                   # (more new tokens than are held)
    ([30] * 40, [20] * 40, 4, 1, 48),                                        # workgroups of one wave
    ([900, 17, 1400], [300, 17, 200], 8, 2, 64),                             # blocks of 128 rows
    ([8000, 5000], [700, 500], 32, 4, 128),                                  # split
    ([5000, 1, 3333, 900, 2048, 2], [1000, 1, 900, 700, 17, 2], 16, 4, 64),  # both launches
]


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("held,new,H,G,D", NAN_CASES)
def test_nan_queries_have_nan_results(held, new, H, G, D, quantized):
    """A NaN in a query makes all of its scores NaN: its result is NaN, in whichever launch and split, and zero only where it sees nothing."""
    pages = sum(-(-n // 16) for n in held) + 3
    cache = cache_of(pages, 16, H // G, D, BF16, quantized)
    tables = tables_of(held, 16, pages)
    offsets = offsets_of(new or [1] * len(held))
    q = normal(offsets[-1], H, D, dtype=BF16)
    want = attend(cache, q, tables, held, new and offsets)
    seen, spoilt = torch.zeros(q.shape[:2], dtype=torch.bool), torch.zeros(q.shape[:2], dtype=torch.bool)
    for b, n in enumerate(held):
        count = offsets[b + 1] - offsets[b]
        for i in range(count):
            seen[offsets[b] + i] = n - count + i >= 0
        for i in {0, count // 2, count - 1}:
            spoilt[offsets[b] + i, (b + i) % H] = True
    q[spoilt, D // 2] = float("nan")
    got = attend(cache, q, tables, held, new and offsets)
    assert got[spoilt & seen].isnan().all() and not got[~seen].any()
    assert torch.equal(got[~spoilt], want[~spoilt])


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("held,new,H,G,D", NAN_CASES)
def test_rows_whose_keys_are_all_nan(held, new, H, G, D, quantized):
    """A sequence with NaN in all its keys, one of one key among them, has NaN results; the others keep theirs."""
    pages = sum(-(-n // 16) for n in held) + 3
    cache = cache_of(pages, 16, H // G, D, BF16, quantized)
    tables = tables_of(held, 16, pages)
    offsets = offsets_of(new or [1] * len(held))
    q = normal(offsets[-1], H, D, dtype=BF16)
    want = attend(cache, q, tables, held, new and offsets)
    bad = torch.tensor([0x7f], dtype=torch.uint8) if quantized else torch.tensor([float("nan")], dtype=BF16)
    nan = torch.zeros(offsets[-1], dtype=torch.bool)
    for b, n in enumerate(held):
        if b % 2 == 0:
            mine = tables[b, :-(-n // 16)].long().cuda()
            (cache.k.view(torch.uint8) if quantized else cache.k)[mine, :, :, 3] = bad.cuda()
            count = offsets[b + 1] - offsets[b]
            for i in range(count):
                nan[offsets[b] + i] = n - count + i >= 0
    got = attend(cache, q, tables, held, new and offsets)
    assert got[nan].isnan().all() and torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("more,new", [((1, 0, 3), (1, 1, 1)), ((5, 2, 0), (4, 9, 30)), ((100, 1, 1 << 30), (100, 40, 60)), ((0, 60, 0), (0, 64, 1))])
def test_tokens_behind_their_table(more, new, quantized):
    """A token has the position length - n + i, also where the length goes beyond the table: behind its end it is not written, and what stands in the
    table stays; its query sees all of the table, one within it the positions up to its own."""
    size, H, D, room = 8, 2, 64, 64
    cache = cache_of(26, size, H, D, BF16, quantized)
    tables = torch.randperm(26, generator=torch.Generator().manual_seed(5))[:24].view(3, 8).int()
    held, offsets = [room + m for m in more], offsets_of(new)
    k, v = normal(sum(new), H, D, dtype=BF16), normal(sum(new), H, D, dtype=BF16, seed=2)
    want = bits(cache)
    paged_write(cache, k.cuda(), v.cuda(), tables.cuda(), ints(held), ints(offsets))
    for b, n in enumerate(new):
        for i in range(n):
            x = held[b] - n + i
            if x < room:
                page, row = int(tables[b, x // size]), x % size
                for j, numbers in enumerate((k[offsets[b] + i], v[offsets[b] + i])):
                    if quantized:
                        want[j][page, :, row], want[2 + j][page, :, row] = orc.quantise(numbers)
                    else:
                        want[j][page, :, row] = numbers.contiguous().view(torch.uint8)
    assert all(torch.equal(a, b) for a, b in zip(bits(cache), want))
    rows = {which: held_rows(cache, tables, [room] * 3, which) for which in "kv"}
    for got, which in zip(paged_read(cache, tables.cuda(), ints(held), room + 2), "kv"):
        assert not got[:, room:].any()
        assert all(torch.equal(got[b, :room].cpu().double(), rows[which][b]) for b in range(3))
    for H in (4, 16):
        q = normal(sum(new), H, D, dtype=BF16, seed=7)
        got = attend(cache, q, tables, held, offsets)
        value, sizes = orc.paged(q, rows["k"], rows["v"], held, offsets)
        assert bool(((got.double() - value).abs() <= orc.limit(value, sizes, BF16)).all())


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("name", ["k", "v"])
def test_no_gradient_through_the_cache(monkeypatch, name, quantized):
    """A cache whose tensors require gradients, or have tangents, is refused, by the host extension as by the general form; without recording it serves."""
    cache = cache_of(3, 16, 2, 64, BF16, quantized)
    tables, lengths, q, k = ints([[0, 1, 2]]), ints([40]), normal(1, 4, 64, dtype=BF16).cuda(), normal(1, 2, 64, dtype=BF16).cuda()
    calls = (lambda: paged_write(cache, k, k, tables, lengths), lambda: paged_attention(q, cache, tables, lengths),
             lambda: paged_read(cache, tables, lengths, 40)[0])
    want = [call() for call in calls]
    pages = getattr(cache, name)
    for general in (False, True):
        if general:
            monkeypatch.setattr(paged, "_on_gpu", lambda q: False)
        pages.requires_grad_()
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
        with torch.no_grad():
            got = [call() for call in calls]
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        pages.requires_grad_(False)
        if not quantized:
            with fwAD.dual_level():
                setattr(cache, name, fwAD.make_dual(pages, torch.ones_like(pages)))
                for call in calls:
                    with pytest.raises(NotImplementedError):
                        call()
                setattr(cache, name, pages)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("general", [False, True])
def test_a_write_counts_as_a_change_in_place(monkeypatch, general, quantized):
    """What autograd has saved of a cache's tensors, or of what they are views of, is not used after a write has changed it."""
    if general:
        monkeypatch.setattr(paged, "_on_gpu", lambda q: False)
    cache = cache_of(3, 16, 2, 64, BF16, quantized)
    tables, lengths, k = ints([[0, 1, 2]]), ints([40]), normal(1, 2, 64, dtype=BF16).cuda()
    tensors = [t for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]
    before = [t._version for t in tensors]
    paged_read(cache, tables, lengths, 40), paged_attention(normal(1, 4, 64, dtype=BF16).cuda(), cache, tables, lengths)
    assert [t._version for t in tensors] == before
    paged_write(cache, k, k, tables, lengths)
    assert all(t._version > n for t, n in zip(tensors, before))
    if not quantized:
        room = torch.zeros(2, 3, 2, 16, 64, dtype=BF16, device="cuda")
        views = PagedCache.of(room[0], room[1])
        weight = torch.ones((), dtype=BF16, device="cuda", requires_grad=True)
        y = (room * weight).float().sum()
        paged_write(views, k, k, tables, lengths)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        kept = PagedCache(3, 16, 2, 64, BF16, quantized)
    paged_write(kept, k, k, tables, lengths)  # (its tensors have no count)
    assert paged_read(kept, tables, lengths, 40)[0][0, 39].any()
