"""The paged cache where a call's description of its sequences ends: offsets that descend."""
import pytest
import torch

from semicat_amd import paged_attention, paged_write
from tests.test_paged_gpu import BF16, cache_of, ints, normal

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
