"""The paged cache (csrc/sjvp_paged.hip, sjvp_seq*): written and read numbers bit by bit against the format's definition, attention against
the definition in float64 with the tolerances at packed_oracle.limit."""
import math

import pytest
import torch

from oracle import packed_oracle as orc

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def cache_of(pages, size, heads, D, dtype, quantized, seed=0, spread=1.0):
    """A cache full of numbers, pages of nobody included."""
    from semicat_amd import PagedCache
    g = torch.Generator().manual_seed(seed)
    cache = PagedCache(pages, size, heads, D, dtype, quantized)
    for x, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        numbers = (torch.randn(pages, heads, size, D, generator=g) * spread).to(dtype)
        if quantized:
            codes, powers = orc.quantise(numbers)
            x.view(torch.uint8).copy_(codes), scales.view(torch.uint8).copy_(powers)
        else:
            x.copy_(numbers)
    return cache


def tables_of(held, size, pages, extra=1, seed=0):
    """Pages of the sequences in a mixed order; -1 behind them."""
    g = torch.Generator().manual_seed(seed)
    free = torch.randperm(pages, generator=g).tolist()
    out = torch.full((len(held), max(1, max(-(-n // size) for n in held)) + extra), -1, dtype=torch.int32)
    for b, n in enumerate(held):
        for i in range(-(-n // size)):
            out[b, i] = free.pop()
    return out


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def held_rows(cache, tables, held, which):
    pages, scales = (cache.k, cache.k_scales) if which == "k" else (cache.v, cache.v_scales)
    bits = lambda t: None if t is None else t.view(torch.uint8).cpu()
    numbers = pages.cpu() if scales is None else bits(pages)
    return [orc.rows(numbers, bits(scales), tables[b], n, cache.page_size) for b, n in enumerate(held)]


def offsets_of(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def attend(cache, q, tables, held, offsets, scale=None):
    from semicat_amd import paged_attention
    o = paged_attention(q.cuda(), cache, tables.cuda(), ints(held), None if offsets is None else ints(offsets), scale)
    torch.cuda.synchronize()
    return o.cpu()


def check_attention(cache, q, tables, held, offsets, scale=None, got=None):
    got = attend(cache, q, tables, held, offsets, scale) if got is None else got
    offsets = list(range(len(held) + 1)) if offsets is None else offsets
    want, size = orc.paged(q, held_rows(cache, tables, held, "k"), held_rows(cache, tables, held, "v"), held, offsets, scale)
    off, limit = (got.double() - want).abs(), orc.limit(want, size, q.dtype)
    assert bool((off <= limit).all()), (float((off / limit).max()), int((off > limit).sum()))


def normal(*shape, dtype, seed=1):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 48), (FP16, 128), (FP16, 16), (BF16, 112)])
def test_written_numbers_are_the_format_s(dtype, D):
    """Every scale that a type has, numbers at and next to the borders between two 8-bit numbers and between two scales, zeros, infinities and NaN."""
    from semicat_amd import PagedCache, paged_read, paged_write
    g = torch.Generator().manual_seed(D)
    T, H = 300, 3
    info = torch.finfo(dtype)
    powers = torch.linspace(math.log2(info.smallest_normal) - 2, math.log2(info.max), T)[:, None, None]
    x = torch.randn(T, H, D, generator=g, dtype=torch.float64) * torch.pow(2.0, powers.double())
    y = orc.e4m3_values()[torch.randint(0, 127, (T, H, D), generator=g)] * torch.pow(2.0, torch.randint(-12, 5, (T, H, 1), generator=g).double())
    y *= 1 + torch.randint(-2, 3, y.shape, generator=g) / 16  # (numbers of the format, and in the middle between two)
    k, v = x.to(dtype), y.to(dtype)
    k[0], v[1] = 0.0, -0.0
    k[2, 0, 3], k[2, 1, 5], k[2, 2, 7] = math.inf, -math.inf, math.nan
    v[3] = info.max
    v[4, :, 0] = info.max
    v[5] = math.nan
    k[6], k[6, :, -1] = info.tiny / 4, 1.0
    k[7] = 448.0
    k[8], k[9] = 450.0, 1.75 * info.tiny
    cache = PagedCache(40, 8, H, D, dtype, quantized=True)
    tables = tables_of([T], 8, 40)
    paged_write(cache, k.cuda(), v.cuda(), tables.cuda(), ints([T]), ints([0, T]))
    order = tables[0, torch.arange(T) // 8].long(), torch.arange(T) % 8
    for numbers, pages, scales in ((k, cache.k, cache.k_scales), (v, cache.v, cache.v_scales)):
        codes, powers = orc.quantise(numbers)
        got = pages.view(torch.uint8).cpu()[order[0], :, order[1]]
        same = (got == codes) | ((got & 127 == 127) & (codes & 127 == 127))
        assert bool(same.all()), (got[~same][:8], codes[~same][:8], numbers[~same][:8])
        assert torch.equal(scales.view(torch.uint8).cpu()[order[0], :, order[1]], powers)
    # reading rounds nothing: what the 8 bits stand for is one of the type's numbers
    for got, pages, scales in zip(paged_read(cache, tables.cuda(), ints([T]), T), (cache.k, cache.v), (cache.k_scales, cache.v_scales)):
        want = orc.dequantise(pages.view(torch.uint8).cpu()[order[0], :, order[1]], scales.view(torch.uint8).cpu()[order[0], :, order[1]])
        assert torch.equal(got[0].cpu().double().nan_to_num(-1.0), want.nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_every_code_and_scale_reads_back(dtype):
    from semicat_amd import PagedCache, paged_read
    low, high = orc.LOWEST[dtype], orc.HIGHEST[dtype]
    n = high - low + 1
    cache = PagedCache(n, 8, 1, 32, dtype, quantized=True)
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 8, 32).expand(n, 1, 8, 32).clone()
    codes[-1][(codes[-1] & 127) > 0x77] = 0x77  # (240 is the last number at the largest scale)
    scales = (torch.arange(low, high + 1) + 127).to(torch.uint8).view(n, 1, 1, 1).expand(n, 1, 8, 1).contiguous()
    for pages, powers in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        pages.view(torch.uint8).copy_(codes), powers.view(torch.uint8).copy_(scales)
    tables = torch.arange(n, dtype=torch.int32)[None]
    want = orc.dequantise(codes, scales).reshape(1, n * 8, 1, 32)
    assert torch.equal(want.to(dtype).double().nan_to_num(-1.0), want.nan_to_num(-1.0))
    for got in paged_read(cache, tables.cuda(), ints([n * 8]), n * 8):
        assert torch.equal(got.cpu().double().nan_to_num(-1.0), want.nan_to_num(-1.0))


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("size,H,D,dtype", [(16, 2, 64, BF16), (7, 3, 48, FP16), (1, 1, 16, BF16), (64, 5, 128, BF16), (100, 1, 80, FP16)])
def test_write_and_read(size, H, D, dtype, quantized):
    """Ragged writes at the ends of their sequences; rows and pages of others stay as they were."""
    from semicat_amd import paged_read, paged_write
    held, new = [0, 33, 1, 129, 64, 20, 2], [0, 33, 1, 5, 1, 0, 2]
    T = sum(new) + 3
    pages = sum(-(-n // size) for n in held) + 4
    cache = cache_of(pages, size, H, D, dtype, quantized)
    tables = tables_of(held, size, pages)
    before = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]
    k, v = normal(T, H, D, dtype=dtype), normal(T, H, D, dtype=dtype, seed=2)
    offsets = [n + 2 for n in offsets_of(new)]  # (two tokens of nobody in front, one behind)
    paged_write(cache, k.cuda(), v.cuda(), tables.cuda(), ints(held), ints(offsets))
    want = [t.cpu().clone() for t in before]
    for b, n in enumerate(new):
        for i in range(n):
            x = held[b] - n + i
            page, row = int(tables[b, x // size]), x % size
            for j, numbers in enumerate((k[offsets[b] + i], v[offsets[b] + i])):
                if quantized:
                    want[j][page, :, row], want[2 + j][page, :, row] = orc.quantise(numbers)
                else:
                    want[j][page, :, row] = numbers.contiguous().view(torch.uint8)
    for t, w in zip((cache.k, cache.v, cache.k_scales, cache.v_scales), want):
        assert torch.equal(t.view(torch.uint8).cpu(), w)
    for most in (1, 64, 140):
        for which, got in zip("kv", paged_read(cache, tables.cuda(), ints(held), most)):
            rows = held_rows(cache, tables, held, which)
            assert got.shape == (len(held), most, H, D) and got.dtype == dtype
            for b, n in enumerate(held):
                m = min(n, most)
                assert torch.equal(got[b, :m].cpu().double(), rows[b][:m]) and not got[b, m:].any()


CASES = [  # heads, group, head dimension, page size, type
    (2, 1, 64, 16, BF16), (4, 4, 128, 32, BF16), (6, 3, 48, 7, FP16), (8, 8, 128, 64, FP16), (3, 1, 16, 1, BF16), (5, 5, 80, 48, BF16), (12, 2, 96, 16, FP16),
    (32, 32, 64, 128, BF16), (40, 40, 32, 16, BF16), (2, 2, 112, 300, BF16)]


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("H,G,D,size,dtype", CASES)
def test_one_token_each(H, G, D, size, dtype, quantized):
    held = [1, 2, 31, 32, 33, 0, 64, 100, 257]
    pages = sum(-(-n // size) for n in held) + 3
    cache = cache_of(pages, size, H // G, D, dtype, quantized)
    tables = tables_of(held, size, pages)
    check_attention(cache, normal(len(held), H, D, dtype=dtype), tables, held, None)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("H,G,D,size,dtype", CASES)
def test_chunks(H, G, D, size, dtype, quantized):
    """New tokens from none to more than the cache holds (those in front of position 0 see nothing), rows of nobody in front and behind."""
    held, new = [40, 70, 5, 0, 300, 129, 3], [1, 70, 0, 2, 33, 2, 5]
    pages = sum(-(-n // size) for n in held) + 3
    cache = cache_of(pages, size, H // G, D, dtype, quantized)
    tables = tables_of(held, size, pages)
    offsets = [n + 1 for n in offsets_of(new)]
    q = normal(offsets[-1] + 2, H, D, dtype=dtype)
    q[0], q[-2:] = float("nan"), float("inf")
    got = attend(cache, q, tables, held, offsets)
    q[0], q[-2:] = 0.0, 0.0
    check_attention(cache, q, tables, held, offsets, got=got)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("H,G,D,dtype", [(16, 4, 128, BF16), (8, 1, 64, FP16), (6, 6, 48, BF16)])
def test_long_caches_and_mixed_batches(H, G, D, dtype, quantized):
    """Long sequences are split over workgroups; with enough rows single tokens and whole chunks go through launches of their own."""
    held = [5000, 1, 3333, 900, 513, 0, 2048]
    pages = sum(-(-n // 32) for n in held) + 3
    cache = cache_of(pages, 32, H // G, D, dtype, quantized)
    tables = tables_of(held, 32, pages, extra=9)
    check_attention(cache, normal(len(held), H, D, dtype=dtype), tables, held, None)
    new = [3, 1, 700, 64, 513, 0, 17]
    check_attention(cache, normal(sum(new), H, D, dtype=dtype), tables, held, offsets_of(new))


def test_many_rows_of_many_sequences():
    """Enough rows for the launch of 128-row blocks beside the one of few rows, at both sides of the border between them."""
    g = torch.Generator().manual_seed(3)
    held, new = [], []
    for n in (15, 16, 17, 1, 200, 33, 0, 64, 400, 129, 31, 32, 500, 480, 300, 256):
        new.append(n)
        held.append(n + int(torch.randint(0, 700, (1,), generator=g)))
    pages = sum(-(-n // 16) for n in held) + 3
    for quantized in (True, False):
        cache = cache_of(pages, 16, 8, 64, BF16, quantized)
        tables = tables_of(held, 16, pages)
        check_attention(cache, normal(sum(new), 32, 64, dtype=BF16), tables, held, offsets_of(new))


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("most,B,H,G,D,dtype", [(40, 50, 4, 1, 64, BF16), (64, 9, 4, 2, 128, FP16), (1, 70, 3, 3, 16, BF16), (200, 150, 32, 1, 48, BF16),
                                                 (120, 64, 40, 2, 96, FP16), (130, 40, 40, 1, 112, BF16)])
def test_short_caches(most, B, H, G, D, dtype, quantized):
    """Caches that a wave reads by itself, and their neighbours."""
    g = torch.Generator().manual_seed(most)
    held = torch.randint(0, most + 1, (B,), generator=g).tolist()
    held[0], held[-1] = most, 0
    new = [min(n, int(torch.randint(0, 1 + min(most, 12), (1,), generator=g))) for n in held]
    pages = sum(-(-n // 8) for n in held) + 3
    cache = cache_of(pages, 8, H // G, D, dtype, quantized)
    tables = tables_of(held, 8, pages, extra=0)
    check_attention(cache, normal(sum(new), H, D, dtype=dtype), tables, held, offsets_of(new))
    check_attention(cache, normal(B, H, D, dtype=dtype), tables, held, None)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("B,G,D,dtype", [(7, 4, 128, BF16), (62, 2, 64, FP16), (63, 2, 96, BF16), (1, 8, 80, BF16)])
def test_chunks_on_caches_of_all_lengths(B, G, D, dtype, quantized):
    """Blocks of 128 rows in the order of their sequences' lengths, up to 62 sequences, and in the plain order with more."""
    g = torch.Generator().manual_seed(B)
    new = [int(n) for n in torch.randint(128 // G, 512 // G, (B,), generator=g)]
    held = [n + int(m) for n, m in zip(new, torch.randint(0, 3000 if B < 10 else 200, (B,), generator=g))]
    new[B // 2] = 0
    if B > 2:
        held[1], held[2] = held[0], 0
        new[2] = 3  # (more new tokens than the cache has)
    H = 12 * G if B < 10 else 2 * G
    pages = sum(-(-n // 64) for n in held) + 3
    cache = cache_of(pages, 64, H // G, D, dtype, quantized)
    tables = tables_of(held, 64, pages)
    new[1 % B] = min(new[1 % B], held[1 % B])
    check_attention(cache, normal(max(1, sum(new)), H, D, dtype=dtype)[:sum(new)], tables, held, offsets_of(new))


@pytest.mark.parametrize("D,dtype", [(128, BF16), (48, FP16)])
@pytest.mark.parametrize("G,few", [(4, (7, 8, 9)), (1, (31, 32, 33)), (8, (3, 4, 5))])
def test_the_border_of_few_rows(G, few, D, dtype):
    """Sequences of 32 rows and their neighbours in number beside long ones, split over the keys or not."""
    new = [*few, 1, 0, 700 // G, *few, 2100 // G]
    for more in (0, 2500):
        held = [n + more * (i % 2) for i, n in enumerate(new)]
        pages = sum(-(-n // 16) for n in held) + 3
        cache = cache_of(pages, 16, 8, D, dtype, True)
        check_attention(cache, normal(sum(new), 8 * G, D, dtype=dtype), tables_of(held, 16, pages), held, offsets_of(new))


@pytest.mark.parametrize("quantized", [True, False])
def test_pages_that_the_cache_has_not(quantized):
    """They read as zeros and take no writes; lengths beyond the table end there."""
    from semicat_amd import paged_read, paged_write
    cache = cache_of(9, 16, 2, 64, BF16, quantized)
    tables = torch.tensor([[3, -1, 5, 1 << 30], [9, 0, -(1 << 31), 7]], dtype=torch.int32)
    held = [64, 50]
    q = normal(2, 4, 64, dtype=BF16)
    check_attention(cache, q, tables, held, None)
    assert torch.equal(attend(cache, q, tables, [1 << 30, 50], None), attend(cache, q, tables, [64, 50], None))
    assert not attend(cache, q, tables, [-5, 0], None).any()
    chunk = normal(90, 4, 64, dtype=BF16, seed=4)
    check_attention(cache, chunk, tables, held, [0, 60, 90])
    for got, which in zip(paged_read(cache, tables.cuda(), ints(held), 70), "kv"):
        for b, rows in enumerate(held_rows(cache, tables, held, which)):
            assert torch.equal(got[b, :held[b]].cpu().double(), rows)
    before = [t.view(torch.uint8).clone() for t in (cache.k, cache.v)]
    k = normal(4, 2, 64, dtype=BF16)
    paged_write(cache, k.cuda(), k.cuda(), torch.tensor([[-1, 9], [1 << 30, -7]], dtype=torch.int32).cuda(), ints([17, 2]), ints([0, 2, 4]))
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip((cache.k, cache.v), before))


@pytest.mark.parametrize("quantized", [True, False])
def test_numbers_of_nobody_are_not_used(quantized):
    """NaN in pages of others, behind a sequence within its last page, and in what a row ends before."""
    held, size = [21, 40], 16
    cache = cache_of(8, size, 2, 64, BF16, quantized)
    tables = tables_of(held, size, 8)
    q = normal(2, 4, 64, dtype=BF16)
    want = attend(cache, q, tables, held, None)
    mine = torch.zeros(8, size, dtype=torch.bool)
    for b, n in enumerate(held):
        for x in range(n):
            mine[tables[b, x // size].long(), x % size] = True
    for pages in (cache.k, cache.v):
        t = pages.view(torch.uint8)
        t.copy_(torch.where(mine[:, None, :, None].cuda(), t, 255))  # (NaN in both forms)
    assert torch.equal(attend(cache, q, tables, held, None), want)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("new,held", [([5, 1, 3], [40, 33, 70]), ([300, 17, 200], [900, 17, 1400]), ([90] * 30, [100 + 20 * i for i in range(30)])])
def test_numbers_that_a_token_does_not_see(new, held, quantized):
    """The last token's keys and values are not finite: only its own output is not."""
    size, H, D = 16, 8, 64
    pages = sum(-(-n // size) for n in held) + 1
    cache = cache_of(pages, size, 4, D, BF16, quantized)
    tables = tables_of(held, size, pages)
    offsets = offsets_of(new)
    q = normal(sum(new), H, D, dtype=BF16)
    want, sizes = orc.paged(q, held_rows(cache, tables, held, "k"), held_rows(cache, tables, held, "v"), held, offsets)
    bad = torch.tensor([float("nan")], dtype=BF16).view(torch.uint8) if not quantized else torch.tensor([127], dtype=torch.uint8)
    for b, n in enumerate(held):
        page, row = int(tables[b, (n - 1) // size]), (n - 1) % size
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[page, :, row] = bad.repeat(D).cuda()
    got = attend(cache, q, tables, held, offsets)
    last = torch.zeros(sum(new), dtype=torch.bool)
    last[torch.tensor(offsets[1:]) - 1] = True
    off = (got.double() - want).abs()
    assert bool((off <= orc.limit(want, sizes, BF16))[~last].all()) and got[last].isnan().all()


def test_rows_of_nobody_beside_many():
    """Rows outside the sequences are zeros whichever launch they fall to."""
    new, held = [300] * 12 + [3], [400] * 13
    cache = cache_of(13 * 25 + 1, 16, 4, 64, BF16, True)
    tables = tables_of(held, 16, 13 * 25 + 1)
    for front, behind in ((1, 2), (200, 300)):
        offsets = [n + front for n in offsets_of(new)]
        q = normal(offsets[-1] + behind, 16, 64, dtype=BF16)
        got = attend(cache, q, tables, held, offsets)
        assert not got[:front].any() and not got[-behind:].any()
        inner = attend(cache, q[front:-behind], tables, held, offsets_of(new))
        assert torch.equal(got[front:-behind], inner)


def test_places_in_memory():
    """A cache in slices of a caller's tensors, tensors of any stride, a table that is a slice of a larger one."""
    from semicat_amd import PagedCache, paged_attention, paged_write
    held, size, H, D = [35, 20], 16, 2, 64
    tables = tables_of(held, size, 6)
    room = torch.zeros(6, 2, size, H, D, dtype=BF16, device="cuda")  # K and V of a page side by side, tokens before heads
    cache = PagedCache.of(room[:, 0].transpose(1, 2), room[:, 1].transpose(1, 2))
    plain = PagedCache(6, size, H, D)
    wide = torch.zeros(2, 99, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + tables.shape[1]] = tables.cuda()
    sliced = wide[:, 5:5 + tables.shape[1]]
    kv = normal(55, 2, H, D, dtype=BF16).cuda()  # [T,2,H,D]
    offsets = ints([0, 35, 55])
    paged_write(cache, kv[:, 0], kv[:, 1], sliced, ints(held), offsets)
    paged_write(plain, kv[:, 0].contiguous(), kv[:, 1].contiguous(), tables.cuda(), ints(held), offsets)
    assert torch.equal(cache.k, plain.k) and torch.equal(cache.v, plain.v)
    q = torch.zeros(2, 4, D + 3, dtype=BF16, device="cuda")[:, :, 1:1 + D]
    q.copy_(normal(2, 4, D, dtype=BF16))
    got = paged_attention(q, cache, sliced, ints(held))
    assert torch.equal(got, paged_attention(q.contiguous(), plain, tables.cuda(), ints(held)))
    check_attention(plain, q.cpu().contiguous(), tables, held, None, got=got.cpu())


def test_large_caches():
    """Pages beyond 4 GiB from the first one."""
    from semicat_amd import PagedCache, paged_read, paged_write
    size, H, D = 256, 8, 128
    pages = (5 << 30) // (size * H * D * 2)
    cache = PagedCache(pages, size, H, D)
    tables = torch.tensor([[pages - 1, 0, pages - 2], [pages // 2, 1, 2]], dtype=torch.int32)
    held = [600, 300]
    k, v = normal(900, H, D, dtype=BF16), normal(900, H, D, dtype=BF16, seed=2)
    paged_write(cache, k.cuda(), v.cuda(), tables.cuda(), ints(held), ints([0, 600, 900]))
    got = paged_read(cache, tables.cuda(), ints(held), 600)
    assert torch.equal(got[0][0].cpu(), k[:600]) and torch.equal(got[1][1, :300].cpu(), v[600:])
    q = normal(40, 16, D, dtype=BF16)
    want, sizes = orc.paged(q, [k[:600], k[600:]], [v[:600], v[600:]], held, [0, 38, 40])
    off = (attend(cache, q, tables, held, [0, 38, 40]).double() - want).abs()
    assert bool((off <= orc.limit(want, sizes, BF16)).all())


def test_a_run_of_generation():
    """Prompts in one packed tensor, their keys and values written, then steps of one token and a chunk: every token's output is the one that attention
    over the whole sequence gives it."""
    from semicat_amd import PagedCache, packed_attention, paged_attention, paged_read, paged_write
    H, Hkv, D, size = 8, 2, 64, 16
    final, prompts = [70, 41, 100], [50, 41, 77]
    whole = {n: [normal(m, h, D, dtype=BF16, seed=10 * i + j) for i, m in enumerate(final)] for j, (n, h) in enumerate((("q", H), ("k", Hkv), ("v", Hkv)))}
    want = [orc.packed(*(whole[n][i] for n in "qkv"), [0, m], True) for i, m in enumerate(final)]
    cache = PagedCache(20, size, Hkv, D)
    tables = tables_of(final, size, 20).cuda()

    def rows(name, spans):
        return torch.cat([whole[name][i][a:b] for i, (a, b) in enumerate(spans)]).cuda()

    def check(o, spans):
        at = 0
        for i, (a, b) in enumerate(spans):
            off = (o[at:at + b - a].cpu().double() - want[i][0]["o"][a:b]).abs()
            assert bool((off <= orc.limit(want[i][0]["o"], want[i][1]["o"], BF16)[a:b]).all())
            at += b - a

    spans = [(0, n) for n in prompts]
    offsets = ints(offsets_of(prompts))
    check(packed_attention(rows("q", spans), rows("k", spans), rows("v", spans), offsets), spans)
    paged_write(cache, rows("k", spans), rows("v", spans), tables, ints(prompts), offsets)
    held = list(prompts)
    while held != final:
        new = [min(1 if i == 0 else 9, m - n) for i, (m, n) in enumerate(zip(final, held))]
        spans = [(n, n + x) for n, x in zip(held, new)]
        held = [b for _, b in spans]
        paged_write(cache, rows("k", spans), rows("v", spans), tables, ints(held), ints(offsets_of(new)))
        check(paged_attention(rows("q", spans), cache, tables, ints(held), ints(offsets_of(new))), spans)
    k, v = paged_read(cache, tables, ints(final), max(final))
    for i, n in enumerate(final):
        assert torch.equal(k[i, :n].cpu(), whole["k"][i]) and torch.equal(v[i, :n].cpu(), whole["v"][i])


def test_read_pages_fit_the_attention_on_states():
    """What is read back is what cross_attention takes."""
    from semicat_amd import cross_attention, paged_attention, paged_read
    held, size = [45, 130, 7], 16
    cache = cache_of(14, size, 2, 64, BF16, True)
    tables = tables_of(held, size, 14)
    q = normal(3, 4, 64, dtype=BF16).cuda()
    k, v = paged_read(cache, tables.cuda(), ints(held), 130)
    dense = cross_attention(q[:, None], k, v, key_lengths=ints(held))[:, 0]
    check_attention(cache, q.cpu(), tables, held, None, got=dense.cpu())
    check_attention(cache, q.cpu(), tables, held, None, got=paged_attention(q, cache, tables.cuda(), ints(held)).cpu())


def test_steps_in_graphs():
    """Two captured steps with different lengths, replayed in turn with eager calls between them."""
    from semicat_amd import paged_attention, paged_write
    held, size = [900, 1700], 32
    caches = [cache_of(120, size, 2, 64, BF16, q) for q in (True, False)]
    tables = tables_of([1800, 1800], size, 120)
    tables, lengths = tables.cuda(), ints(held)
    q, k, v = normal(2, 8, 64, dtype=BF16).cuda(), normal(2, 2, 64, dtype=BF16, seed=3).cuda(), normal(2, 2, 64, dtype=BF16, seed=4).cuda()
    graphs, outs = [], []
    for cache in caches:
        paged_attention(q, cache, tables, lengths)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_write(cache, k, v, tables, lengths)
            outs.append(paged_attention(q, cache, tables, lengths))
        graphs.append(graph)
    for step in range(4):
        lengths.copy_(torch.tensor([900 + 200 * step, 1700 - 500 * step], dtype=torch.int32))
        q.copy_(normal(2, 8, 64, dtype=BF16, seed=20 + step))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for cache, out in zip(caches, outs):
            assert torch.equal(out, paged_attention(q, cache, tables, lengths))


def test_other_streams_and_repeats():
    from semicat_amd import paged_attention
    held = [3000, 40, 777]
    cache = cache_of(130, 32, 4, 128, BF16, True)
    tables, lengths, q = tables_of(held, 32, 130).cuda(), ints(held), normal(3, 16, 128, dtype=BF16).cuda()
    first = paged_attention(q, cache, tables, lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(paged_attention(q, cache, tables, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_other_types():
    from semicat_amd import PagedCache, paged_attention, paged_write
    cache = PagedCache(4, 16, 2, 64, quantized=True)
    tables, lengths = torch.tensor([[2, 1]], dtype=torch.int32).cuda(), ints([20])
    k = normal(20, 2, 64, dtype=torch.float32).cuda()
    paged_write(cache, k, k, tables, lengths, ints([0, 20]))
    other = PagedCache(4, 16, 2, 64, quantized=True)
    paged_write(other, k.bfloat16(), k.bfloat16(), tables, lengths, ints([0, 20]))
    assert torch.equal(cache.k.view(torch.uint8), other.k.view(torch.uint8))
    q = normal(1, 4, 64, dtype=torch.float32).cuda()
    o = paged_attention(q, cache, tables, lengths)
    assert o.dtype == torch.float32 and torch.equal(o, paged_attention(q.bfloat16(), cache, tables, lengths).float())
