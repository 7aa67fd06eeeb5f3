"""Cross attention and attention with a relative position bias at the ends of their range: tables that hide every key of a row alike,
few-bit tensors of small numbers, bucket lists of their own, how near the gradient of a float32 table comes.  Limits of single elements as in
test_context_gpu.py."""
import pytest
import torch

from oracle import context_oracle as orc
from tests.test_context_gpu import BF16, FP16, make, run

pytestmark = pytest.mark.gpu
LOW = torch.finfo(torch.float32).min

# the single backward launch by four waves and by eight, the pair, the pair with split axes, few rows in splits, rows of odd length
FORMS = [(2, 4, 2, 50, 90, 64), (2, 9, 3, 60, 250, 40), (3, 2, 1, 140, 300, 32), (1, 2, 2, 130, 1500, 96), (2, 4, 4, 3, 3000, 128),
         (20, 8, 1, 150, 290, 48)]


def near(got, want, sizes, x, names=None):
    for name in names or got:
        t = got[name]
        key = "o" if name == "plain" else name
        u = torch.finfo(t.dtype).eps / 2
        a, b, c = sizes[key]
        limit = 2.0 ** -15 * a if name == "dtable" else u * a + (u * u + 2.0 ** -14) * (a + b)
        limit = limit + u * want[key].abs() + (2.0 ** -25 * (1.0 + c) if x["q"].dtype == FP16 else 0.0) + 1e-30
        off = (t.cpu().double() - want[key]).abs()
        assert bool((off <= limit).all()), f"{name}: {float((off / limit).max()):.3g} times the limit"


@pytest.mark.parametrize("value", [-1e9, LOW])
@pytest.mark.parametrize("shape", FORMS + [(6, 8, 1, 700, 900, 64), (9, 8, 2, 500, 600, 128)])
def test_a_bias_that_leaves_nothing_of_the_scores_does_so_at_every_distance(shape, value):
    """The output of rows whose keys all have it: near the diagonal and far from it they have the same weight, as scores and bias added in
    float32 have."""
    x = make(*shape, BF16, seed=4, table=(32, torch.float32))
    x["table"][:] = value
    x.pop("dO")
    want, sizes = orc.attention(**x, max_distance=60, scores_in=torch.float32)
    x["dO"] = torch.zeros_like(x["q"])
    near(run(x, max_distance=60), want, sizes, x, ("o", "plain"))
