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


@pytest.mark.parametrize("both,causal", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("shape", FORMS[:3])
def test_bucket_lists_with_buckets_that_no_distance_has(shape, both, causal):
    """Equal first distances: all but the last bucket of them are empty.  Results are those of the list without the empty ones, whose
    entries have no gradient."""
    from semicat_amd import RelativeBias, context_backward, context_forward
    firsts, used = (0, 0, 0, 2, 7, 7, 40), [2, 3, 5, 6]
    x = make(*shape, BF16, seed=5, table=(14 if both else 7, torch.float32))
    d = {n: t.cuda() if n == "table" else t.cuda().transpose(1, 2) for n, t in x.items()}
    rows = used + [7 + i for i in used] if both else used

    def passes(table, starts):
        bias = RelativeBias(table, 40, both, causal)
        bias.starts = starts
        rest = torch.empty_like(d["q"])
        o, lse = context_forward(d["q"], d["k"], d["v"], bias, o_rest=rest)
        return o, *context_backward(d["q"], d["k"], d["v"], o, lse, d["dO"], bias, o_rest=rest)

    got = passes(d["table"], firsts)
    want = passes(d["table"][rows].contiguous(), tuple(firsts[i] for i in used))
    for a, b in zip(got[:-1], want[:-1]):
        assert torch.equal(a, b)
    full = torch.zeros_like(got[-1])
    full[rows] = want[-1]
    assert torch.equal(got[-1], full)


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


@pytest.mark.parametrize("value", [-1e9, LOW])
@pytest.mark.parametrize("dtype,shape", [(BF16, s) for s in FORMS] + [(FP16, FORMS[0]), (FP16, FORMS[3])])
def test_rows_whose_keys_all_have_one_large_bias(shape, dtype, value):
    """Beside a bias of 1e9 nothing of the scores is left in float32: all keys of the row have the same weight, in the output
    and in every gradient."""
    x = make(*shape, dtype, seed=1, table=(32, torch.float32))
    x["table"][:] = value
    want, sizes = orc.attention(**x, max_distance=60, scores_in=torch.float32)
    near(run(x, max_distance=60), want, sizes, x)


@pytest.mark.parametrize("value", [-1e9, LOW])
@pytest.mark.parametrize("shape", FORMS[:4])
def test_rows_that_see_hidden_keys_alone_beside_others(shape, value):
    """Causal rows near the first key see nothing but the distances that the table hides; the others see keys that it does not."""
    x = make(*shape, BF16, seed=2, table=(24, torch.float32))
    x["table"][:5] = value
    options = dict(max_distance=60, bidirectional=False, causal=True, key_lengths=torch.tensor([shape[4] - 7] * shape[0], dtype=torch.int32))
    want, sizes = orc.attention(**x, scores_in=torch.float32, **options)
    near(run(x, **options), want, sizes, x)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", FORMS)
def test_weights_of_large_scores_sum_to_one(shape, dtype):
    """Keys in groups of three alike, with scores of some millions: a row's weights are thirds.  With a cotangent of ones each row hands
    a weight of one on to dv, whose sum over the keys is the number of rows: P is rounded once and so is dv, by u each, and fp16
    numbers below 2^-14 by 2^-25."""
    B, H, G, Lq, Lk, _ = shape
    x = make(*shape, dtype, seed=3)
    x["q"], x["k"] = x["q"] * 2048, x["k"][:, torch.arange(Lk) // 3] * 2048
    x["dO"] = torch.ones_like(x["dO"])
    got = run(x)
    assert all(t.isfinite().all() for t in got.values())
    total, rows = got["dv"].cpu().double().sum(1), G * Lq
    limit = (2 * torch.finfo(dtype).eps / 2 + 2.0 ** -14) * rows + (2.0 ** -25 * Lk * (1 + rows) if dtype == FP16 else 0.0)
    assert bool(((total - rows).abs() <= limit).all()), float((total - rows).abs().max() / limit)


@pytest.mark.parametrize("value", [-1e4, -1e5, -1e6, 1e6])
@pytest.mark.parametrize("shape", FORMS)
def test_weights_beside_a_large_bias_sum_to_one(shape, value):
    """As above, with a bias that leaves some of the scores: forward and backward round score plus bias alike."""
    B, H, G, Lq, Lk, _ = shape
    x = make(*shape, FP16, seed=6, table=(32, torch.float32))
    x["table"][:] = value
    x["dO"] = torch.ones_like(x["dO"])
    total, rows = run(x, max_distance=60)["dv"].cpu().double().sum(1), G * Lq
    limit = (2 * torch.finfo(FP16).eps / 2 + 2.0 ** -14) * rows + 2.0 ** -25 * Lk * (1 + rows)
    assert bool(((total - rows).abs() <= limit).all()), float((total - rows).abs().max() / limit)


def off_in_norm(x, **options):
    """How far the table's gradient is off, relative to its norm."""
    want = orc.attention(**x, **options)[0]["dtable"]
    return float((run(x, **options)["dtable"].cpu().double() - want).norm() / want.norm())


# the single backward launch by four waves and by eight, the pair, split axes, a long causal sequence
EXACT = [((2, 4, 2, 128, 128, 64), {}), ((3, 2, 2, 200, 250, 64), {}), ((4, 2, 1, 100, 90, 32), {}), ((1, 1, 1, 300, 300, 128), {}),
         ((1, 2, 1, 1500, 1500, 64), dict(bidirectional=False, causal=True))]


@pytest.mark.parametrize("small", [0.01, 0.002])
@pytest.mark.parametrize("shape,options", EXACT)
def test_table_gradient_of_small_values_in_fp16(shape, options, small):
    """Outputs of 1e-4: delta = dO.o is formed from o to 2^-22 of it or 2^-36, 1.5e-7 of such an output.  With what float32 adds (see
    the next test) 3e-6 of the norm."""
    x = make(*shape, FP16, seed=7, table=(32, torch.float32))
    x["v"] = (x["v"].float() * small).to(FP16)
    assert off_in_norm(x, **options) <= 3e-6


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape,options", EXACT + [((1, 2, 1, 512, 512, 64), {}), ((2, 4, 4, 7, 2500, 128), {})])
@pytest.mark.parametrize("spread,added", [(1.0, 0.0), (2.0, 0.0), (1.0, 30.0)])
def test_table_gradient_is_off_by_some_1e_6(shape, options, dtype, spread, added):
    """Limits in the norm, which the terms of dS all but cancel in as they do in a sum of random signs, so that relative errors of single
    terms come through as they are.  P = 2^x is off by half a step of x, i.e. by 2^-24 X ln 2 for |x| up to X, and is formed twice, for o and for dS.
    Scores have a deviation of 1.44 spread^2 in units of log2 and the bias one of 1.44, largest among 1e5 pairs 5 of them: X is 16 for the
    first, 32 with a spread of 2 (5 x 5.9) and 64 with 30 / ln 2 in every entry: 1.3e-6, 2.6e-6, 5.3e-6.  Contractions of 128 products and
    delta add 2^-22 = 2.4e-7 each: 7e-7 with both.
    P in one rounding (2^-9 of it in bf16), delta of a rounded o (2^-9, 2^-12) or, with bf16, P in two roundings (2^-18 of it at worst,
    4e-6) do not stay below 2e-6."""
    x = make(*shape, dtype, seed=7, table=(32, torch.float32), spread=spread)
    x["table"] += added
    assert off_in_norm(x, **options) <= 7e-7 + 2 * 2.0 ** -24 * 0.6932 * (64 if added else 32 if spread > 1.0 else 16)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", FORMS)
def test_backward_without_what_the_rounding_of_o_left(shape, dtype):
    """delta is off by u |dO||o| then: u (a + b) more than the limits of single elements, for the table u a."""
    from semicat_amd import RelativeBias, context_backward, context_forward
    x = make(*shape, dtype, seed=8, table=(32, torch.float32))
    d = {n: t.cuda() if n == "table" else t.cuda().transpose(1, 2) for n, t in x.items()}
    bias = RelativeBias(d["table"], 60)
    o, lse = context_forward(d["q"], d["k"], d["v"], bias)
    dq, dk, dv, dtable = context_backward(d["q"], d["k"], d["v"], o, lse, d["dO"], bias)
    got = {"o": o.transpose(1, 2), "dq": dq.transpose(1, 2), "dk": dk.transpose(1, 2), "dv": dv.transpose(1, 2), "dtable": dtable}
    want, sizes = orc.attention(**x, max_distance=60)
    u = torch.finfo(dtype).eps / 2
    for name, t in got.items():
        a, b, c = sizes[name]
        own = torch.finfo(t.dtype).eps / 2 * want[name].abs()
        limit = (2.0 ** -15 + u) * a + own if name == "dtable" else u * a + (u + 2.0 ** -14) * (a + b) + own
        limit = limit + (2.0 ** -25 * (1.0 + c) if dtype == FP16 else 0.0) + 1e-30
        off = (t.cpu().double() - want[name]).abs()
        assert bool((off <= limit).all()), f"{name}: {float((off / limit).max()):.3g} times the limit"


def test_strides_of_axes_of_one_row():
    """A sequence axis of size one has no stride that anything depends on."""
    from semicat_amd import cross_attention
    x = make(2, 4, 2, 1, 1, 64, BF16, seed=9)
    y = make(2, 4, 2, 5, 7, 64, BF16, seed=9)

    def far(t):
        return t.as_strided(t.shape, (t.stride(0), (1 << 24) + 4, t.stride(2), 1))

    def passes(q, k, v, dO):
        leaves = [t.requires_grad_() for t in (q, k, v)]
        o = cross_attention(*leaves)
        with torch.no_grad():
            plain = cross_attention(*leaves)
        return (o.detach(), plain, *torch.autograd.grad(o, leaves, dO))

    for a, b in ((x, x), (x, y), (y, x)):  # one row on both sides, one query, one key
        d = [t.cuda() for t in (a["q"], b["k"], b["v"], a["dO"])]
        want = passes(*(t.clone() for t in d))
        got = passes(*(far(t.clone()) if t.shape[1] == 1 else t.clone() for t in d))
        assert all(torch.equal(s, t) for s, t in zip(got, want))


@pytest.mark.parametrize("training", [False, True])
def test_sizes_beyond_the_range_raise_what_the_checks_raise(training):
    """Expanded tensors of one row; nothing is launched.  More sequences than a launch has workgroups for: the library's own error."""
    from semicat_amd import _lib, cross_attention
    q, k = (torch.zeros(1, 1, 1, 16, device="cuda", dtype=BF16, requires_grad=training) for _ in range(2))
    with pytest.raises(ValueError):
        cross_attention(q, k.expand(1, (1 << 29) + 1, 1, 16), k.expand(1, (1 << 29) + 1, 1, 16))
    many = (1 << 24) + 8
    with pytest.raises(_lib.SjvpError) as info:
        cross_attention(q.expand(many, 1, 1, 16), k.expand(many, 1, 1, 16), k.expand(many, 1, 1, 16))
    assert info.value.status == _lib.SJVP_ERR_SHAPE
