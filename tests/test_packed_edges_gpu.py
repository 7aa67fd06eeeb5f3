"""Packed sequences of one or two tiles of keys, which the row-owned backward holds at once."""
import pytest
import torch

from semicat_amd import packed_attention
from tests.test_packed_gpu import BF16, FP16, check, make, offsets_of, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,G,D,dtype", [(2, 1, 32, BF16), (4, 2, 64, FP16), (3, 1, 50, BF16), (2, 2, 96, BF16), (4, 4, 128, BF16), (2, 1, 100, FP16)])
def test_two_tiles_of_keys(H, G, D, dtype, causal):
    lengths = [128, 65, 96, 127, 64, 97, 66, 128]
    offsets = offsets_of(lengths)
    x = make(offsets[-1], H, G, D, dtype, seed=D)
    check(run(x, offsets, causal), x, offsets, causal)


@pytest.mark.parametrize("H,G,D,dtype", [(12, 1, 64, BF16), (8, 4, 128, BF16), (6, 3, 36, FP16)])
def test_two_tiles_of_keys_have_the_same_bits_every_time(H, G, D, dtype):
    """More workgroups than run at once, with waves that see different numbers of keys."""
    g = torch.Generator().manual_seed(D)
    offsets = offsets_of(torch.randint(65, 129, (200,), generator=g).tolist())
    x = {n: t.cuda() for n, t in make(offsets[-1], H, G, D, dtype).items()}
    leaves, at = [x[n].requires_grad_() for n in "qkv"], torch.tensor(offsets, dtype=torch.int32, device="cuda")
    grads = [torch.autograd.grad(packed_attention(*leaves, at), leaves, x["dO"]) for _ in range(5)]
    assert all(torch.equal(a, b) for other in grads[1:] for a, b in zip(grads[0], other))
