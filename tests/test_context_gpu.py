"""Cross attention and attention with a relative position bias (csrc/sjvp_ctx*.hip) against the definition in float64.

Tolerances, element by element.  Each contraction rounds one of its operands (P or dS) to 16 bits and its result once more, by at
most half a step each, u = eps/2 of the type relative to the value.  With a = sum |p||v| (and the like for the gradients) that is
u a + u |result|.  What float32 contractions of up to 128 products, the exponentials and the reduction over the keys add
is bounded by 2^-14 (a + b), b = |sum p k| sum |dO||o| scale and the like: what a relative error of delta = dO.o does, for which P
and o are held to two roundings, u^2 b.  fp16 numbers below 2^-14 are rounded in steps of 2^-24: 2^-25 c + 2^-25, c = sum |v| and the like.
The float32 table's gradient rounds nothing to 16 bits either: 2^-15 a."""
import ctypes

import pytest
import torch

from oracle import context_oracle as orc

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def make(B, H, G, Lq, Lk, D, dtype, seed=0, table=None, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    x = {"q": r(B, Lq, H, D) * spread, "k": r(B, Lk, H // G, D) * spread, "v": r(B, Lk, H // G, D), "dO": r(B, Lq, H, D)}
    x = {n: t.to(dtype) for n, t in x.items()}
    if table is not None:
        x["table"] = r(table[0], H).to(table[1])
    return x


def run(x, **options):
    """Output and gradients through the autograd surface, on the GPU."""
    from semicat_amd import cross_attention, relative_attention
    d = {n: t.cuda() for n, t in x.items()}
    leaves = {n: d[n].requires_grad_() for n in ("q", "k", "v", "table") if n in d}
    options = {n: t.cuda() if torch.is_tensor(t) else t for n, t in options.items()}
    op = relative_attention if "table" in d else cross_attention
    o = op(**leaves, **options)
    grads = torch.autograd.grad(o, list(leaves.values()), d["dO"])
    with torch.no_grad():
        plain = op(**leaves, **options)  # (rounds P, which the forward of a training pass does not)
    torch.cuda.synchronize()
    return {"o": o.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}, "plain": plain}


def check(got, x, **options):
    if "query_start" in options:
        options["start"] = options.pop("query_start")
    want, sizes = orc.attention(**{n: x[n] for n in ("q", "k", "v", "dO")}, table=x.get("table"), **options)
    for name, t in got.items():
        name = "o" if name == "plain" else name
        assert t.dtype == (x["table"].dtype if name == "dtable" else x["q"].dtype) and t.shape == want[name].shape, name
        u = torch.finfo(t.dtype).eps / 2
        a, b, c = sizes[name]
        if name == "dtable":
            limit = 2.0 ** -15 * a + u * want[name].abs()
        else:
            limit = u * a + (u * u + 2.0 ** -14) * (a + b) + u * want[name].abs()
        if x["q"].dtype == FP16:
            limit += 2.0 ** -25 * (1.0 + c)
        off = (t.cpu().double() - want[name]).abs()
        assert bool((off <= limit + 1e-30).all()), f"{name}: {float((off / (limit + 1e-30)).max()):.3g} times the limit"
    return want


SHAPES = [  # B, H, G, Lq, Lk, D
    (1, 1, 1, 1, 1, 16), (2, 4, 2, 1, 7, 64), (1, 2, 1, 33, 64, 32), (2, 2, 1, 128, 128, 64), (1, 3, 3, 130, 65, 128),
    (3, 4, 4, 17, 200, 36), (1, 2, 1, 257, 300, 20), (2, 6, 2, 64, 129, 80), (1, 8, 8, 5, 513, 96), (1, 2, 2, 300, 31, 18),
    (1, 1, 1, 65, 1, 127), (2, 4, 2, 140, 270, 40), (1, 3, 3, 330, 257, 64), (20, 8, 1, 150, 90, 48), (30, 10, 2, 129, 63, 33),
    (16, 8, 1, 100, 256, 64), (9, 30, 2, 66, 250, 57),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES)
def test_cross(shape, dtype):
    x = make(*shape, dtype, seed=shape[3])
    check(run(x), x)


@pytest.mark.parametrize("shape", SHAPES[:13])
@pytest.mark.parametrize("buckets,distance,both,causal,dtype,table", [
    (32, 128, True, False, BF16, torch.float32), (32, 128, False, True, FP16, torch.float32), (5, 9, False, False, BF16, BF16),
    (8, 1024, True, True, BF16, torch.float32), (64, 90, False, True, FP16, FP16)])
def test_relative(shape, buckets, distance, both, causal, dtype, table):
    x = make(*shape, dtype, seed=shape[3], table=(buckets, table))
    options = dict(max_distance=distance, bidirectional=both, causal=causal)
    check(run(x, **options), x, **options)


@pytest.mark.parametrize("relative", [False, True])
@pytest.mark.parametrize("shape", [(5, 4, 2, 70, 150, 64), (6, 4, 2, 65, 100, 64), (5, 2, 1, 200, 300, 64), (5, 2, 1, 3, 400, 40), (5, 4, 4, 140, 140, 128), (6, 2, 1, 1, 2, 32),
                                   (5, 2, 1, 190, 150, 64), (6, 2, 1, 130, 100, 64), (5, 3, 3, 60, 250, 52), (6, 2, 2, 40, 128, 33)])
def test_lengths_hide_what_lies_behind_them(shape, relative):
    """Lengths of zero, one and all; NaN and infinities behind them; results there are zeros."""
    B, _, _, Lq, Lk, _ = shape
    x = make(*shape, BF16, table=(16, torch.float32) if relative else None)
    klen = torch.tensor([0, 1, Lk, Lk // 2, Lk + 5, -3][:B], dtype=torch.int32)
    qlen = torch.tensor([Lq, Lq, 1, 0, Lq // 2 + 1, Lq][:B], dtype=torch.int32)
    options = dict(key_lengths=klen, query_lengths=qlen)
    if relative:
        options.update(max_distance=40, bidirectional=False, causal=True,
                       query_start=torch.tensor([0, 0, Lk - Lq, 3, -2, 1][:B], dtype=torch.int32))
    clean = run(x, **options)
    check(clean, x, **options)
    dirty = {n: t.clone() for n, t in x.items()}
    for b in range(B):
        for n, t in dirty.items():
            if n != "table":
                t[b, max(int((klen if n in "kv" else qlen)[b]), 0):] = float("nan") if b % 2 else float("inf")
    for n, t in run(dirty, **options).items():
        assert torch.equal(t, clean[n]), n
    for b in range(B):
        assert clean["o"][b, int(qlen[b]):].eq(0).all() and clean["dq"][b, int(qlen[b]):].eq(0).all()
        for n in ("dk", "dv"):
            assert clean[n][b, max(int(klen[b]), 0):].eq(0).all()


@pytest.mark.parametrize("start,Lq,Lk", [(0, 100, 100), (50, 20, 80), (-30, 64, 40), (700, 3, 703), (5, 200, 7), (-400, 90, 90)])
@pytest.mark.parametrize("both,causal", [(True, False), (False, True)])
def test_positions(start, Lq, Lk, both, causal):
    """Differences far on either side, rows before the first key (which see none where causal)."""
    x = make(2, 2, 1, Lq, Lk, 32, BF16, table=(12, torch.float32))
    options = dict(max_distance=50, bidirectional=both, causal=causal, query_start=start)
    check(run(x, **options), x, **options)


def in_one_launch(B, H, G, Lq, Lk, D):
    """Whether the backward of such a call is a single launch, which alone needs no workspace (without a table)."""
    from semicat_amd import _lib
    t = _lib.Ctx()
    t.B, t.Hq, t.Hkv, t.Lq, t.Lk, t.D, t.dk = B, H, H // G, Lq, Lk, D, 64  # (no pointer is read)
    return _lib.load().sjvp_ctx_workspace_bytes(ctypes.byref(t), 1) == 0


# the single backward launch over several tiles and heads, by eight waves and by four; the pair
@pytest.mark.parametrize("shape,one", [((40, 8, 2, 150, 220, 64), True), ((65, 4, 2, 150, 100, 64), True), ((33, 8, 2, 150, 220, 64), False),
                                       ((2, 9, 3, 60, 256, 40), True), ((3, 2, 2, 33, 128, 50), True), ((80, 2, 1, 200, 140, 36), True)])
def test_many_units_with_a_bias(shape, one):
    x = make(*shape, BF16, table=(32, torch.float32))
    B, Lk = shape[0], shape[4]
    options = dict(max_distance=60, key_lengths=torch.randint(0, Lk + 1, (B,), generator=torch.Generator().manual_seed(0)).int())
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:  # (the rule asks for their number)
        assert in_one_launch(*shape) == one
    check(run(x, **options), x, **options)


@pytest.mark.parametrize("relative", [False, True])
def test_rows_that_see_one_key_have_no_score_gradient(relative):
    """Exactly none: whoever divides by the gradient's norm sees it.  The value's gradient is the cotangent."""
    x = make(2, 4, 2, 5, 1, 64, BF16, table=(8, torch.float32) if relative else None)
    got = run(x)
    assert all(got[n].eq(0).all() for n in ("dq", "dk") + ("dtable",) * relative)
    check({n: got[n] for n in ("o", "dv")}, x)
    if relative:  # the first row of a causal sequence
        x = make(2, 4, 2, 1, 7, 64, BF16, table=(8, torch.float32))
        got = run(x, max_distance=5, bidirectional=False, causal=True)
        assert all(got[n].eq(0).all() for n in ("dq", "dk", "dtable"))
        check(got, x, max_distance=5, bidirectional=False, causal=True)


def test_masking_entries_of_the_table():
    """The lowest float32 as a bias leaves the other keys their weight, and a row with nothing else its even one; -inf excludes."""
    low = torch.finfo(torch.float32).min
    for value in (low, -float("inf")):
        x = make(1, 2, 1, 40, 40, 32, BF16, table=(8, torch.float32))
        x["table"][3:, 0] = value   # head 0: keys three or more behind
        x["table"][:, 1] = value    # head 1: every key
        options = dict(max_distance=20, bidirectional=False, causal=True)
        got = run(x, **options)
        assert all(t.isfinite().all() for t in got.values())
        if value == low:  # even weights over the keys that the row sees
            v = x["v"][0, :, 1].double()
            even = v.cumsum(0) / torch.arange(1, 41)[:, None]
            a = v.abs().cumsum(0) / torch.arange(1, 41)[:, None]
            off = (got["o"][0, :, 1].cpu().double() - even).abs()
            assert bool((off <= 2.0 ** -8 * (a + even.abs()) + 2.0 ** -14 * a).all())
        else:
            assert got["o"][0, :, 1].eq(0).all() and got["dq"][0, :, 1].eq(0).all() and got["dtable"][:, 1].eq(0).all()
            check(got, x, **options)


def test_sharp_rows():
    """Scores of some hundreds: rows with one key."""
    x = make(2, 2, 1, 150, 150, 64, BF16, spread=6.0, table=(32, torch.float32))
    check(run(x), x)


@pytest.mark.parametrize("dtype,D,gap,offset", [(BF16, 64, 1, 1), (FP16, 48, 3, 5), (BF16, 127, 0, 0), (BF16, 128, 8, 8), (FP16, 17, 0, 1)])
def test_views_of_any_alignment(dtype, D, gap, offset):
    """Rows with gaps of NaN between them at odd addresses, and the heads in front of the sequence: the same bits as dense tensors."""
    x = make(2, 4, 2, 70, 90, D, dtype, table=(16, torch.float32))

    def spread(t, heads_first):
        t = t.transpose(1, 2) if heads_first else t
        buf = torch.full((t.numel() // D * (D + gap) + offset + 8,), float("nan"), dtype=dtype)
        view = buf[offset:offset + t.numel() // D * (D + gap)].view(*t.shape[:3], D + gap)[..., :D]
        view.copy_(t)
        view = buf.cuda()[offset:offset + t.numel() // D * (D + gap)].view(*t.shape[:3], D + gap)[..., :D]
        return view.transpose(1, 2) if heads_first else view

    from semicat_amd import relative_attention
    outs = []
    for place in (lambda t, i: t.cuda(), lambda t, i: spread(t, i % 2 == 1)):
        d = [place(x[n], i) for i, n in enumerate(("q", "k", "v", "dO"))]
        table = x["table"].cuda().requires_grad_()
        leaves = [t.requires_grad_() for t in d[:3]]
        o = relative_attention(*leaves, table)
        outs.append((o, *torch.autograd.grad(o, (*leaves, table), d[3])))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_broadcast_inputs():
    """States shared by the batch, a cotangent of one number, a table read through strides."""
    x = make(3, 4, 2, 40, 70, 64, BF16, table=(16, torch.float32))
    from semicat_amd import relative_attention
    k, v = (x[n][:1].cuda().requires_grad_() for n in "kv")
    q = x["q"].cuda().requires_grad_()
    table = x["table"].t().contiguous().cuda().requires_grad_()
    o = relative_attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), table.t())
    o.sum().backward()
    full = dict(x, dO=torch.ones_like(x["dO"]), k=x["k"][:1].expand(3, -1, -1, -1), v=x["v"][:1].expand(3, -1, -1, -1))
    check({"o": o.detach(), "dq": q.grad, "dtable": table.grad.t()}, full)
    each = run({n: t.contiguous() for n, t in full.items()})
    for g, n in ((k.grad, "dk"), (v.grad, "dv")):
        assert torch.equal(g, each[n].sum(0, keepdim=True)), n


def test_gradients_against_differences():
    """Of a smooth function of the output, in the direction of each input (float32 callers: computed in bfloat16)."""
    from semicat_amd import relative_attention
    x = make(1, 2, 1, 50, 60, 64, BF16, table=(16, torch.float32))
    d = {n: t.cuda() for n, t in x.items()}
    table = d["table"].requires_grad_()
    o = relative_attention(d["q"], d["k"], d["v"], table, max_distance=30)
    (g,) = torch.autograd.grad(o, table, d["dO"])
    step = torch.randn(table.shape, generator=torch.Generator().manual_seed(1)).cuda()
    value = lambda t: (orc.attention(x["q"], x["k"], x["v"], table=t, max_distance=30)[0]["o"] * x["dO"].double()).sum()
    h = 1e-4
    slope = (value(x["table"].double() + h * step.cpu()) - value(x["table"].double() - h * step.cpu())) / (2 * h)
    assert abs(float((g.double().cpu() * step.cpu()).sum() - slope)) <= 1e-4 * float((g.abs() * step.abs()).sum())


def test_same_bits_every_time():
    for shape in ((2, 4, 2, 200, 333, 64), (1, 8, 4, 2, 3000, 128), (1, 2, 1, 40, 2000, 32)):
        x = make(*shape, BF16, table=(32, torch.float32))
        first = run(x)
        for _ in range(3):
            for n, t in run(x).items():
                assert torch.equal(t, first[n]), n


def test_frozen_states_and_table():
    x = make(2, 4, 2, 100, 130, 64, BF16, table=(32, torch.float32))
    from semicat_amd import relative_attention
    d = {n: t.cuda() for n, t in x.items()}
    q = d["q"].requires_grad_()
    relative_attention(q, d["k"], d["v"], d["table"]).backward(d["dO"])
    table = d["table"].requires_grad_()
    relative_attention(d["q"].detach(), d["k"], d["v"], table).backward(d["dO"])
    check({"dq": q.grad, "dtable": table.grad}, x)
    assert d["k"].grad is None and d["v"].grad is None


def test_a_decoder_layer_by_tokens_gives_its_training_pass():
    """Self attention with the bias over a growing cache, then cross attention to ragged states, token by token (and three at a
    time), against the same layer over the whole sequence at once."""
    from semicat_amd import cross_attention, relative_attention
    B, S, H, G, D, Lk = 3, 37, 6, 2, 64, 90
    x = make(B, H, G, S, S, D, BF16, table=(16, torch.float32))
    enc = make(B, H, G, S, Lk, D, BF16, seed=5)
    d, e = ({n: t.cuda() for n, t in z.items()} for z in (x, enc))
    klen = torch.tensor([90, 1, 41], dtype=torch.int32, device="cuda")
    bias = dict(table=d["table"], max_distance=20, bidirectional=False, causal=True)
    a = relative_attention(d["q"], d["k"], d["v"], **bias)
    whole = cross_attention(a, e["k"], e["v"], key_lengths=klen)
    cache_k, cache_v = (torch.full((B, 64, H // G, D), float("nan"), device="cuda", dtype=BF16) for _ in range(2))
    i = 0
    while i < S:
        n = min(3 if i % 2 else 1, S - i)
        cache_k[:, i:i + n], cache_v[:, i:i + n] = d["k"][:, i:i + n], d["v"][:, i:i + n]
        held = torch.full((B,), i + n, device="cuda", dtype=torch.int32)
        step = relative_attention(d["q"][:, i:i + n], cache_k, cache_v, key_lengths=held, query_start=i, **bias)
        # both round P and o: they differ by at most two roundings of each
        limit = 4 * 2.0 ** -8 * (a[:, i:i + n].abs().float() + 2.0)
        assert bool(((step.float() - a[:, i:i + n].float()).abs() <= limit).all())
        out = cross_attention(a[:, i:i + n], e["k"], e["v"], key_lengths=klen)
        assert bool(((out.float() - whole[:, i:i + n].float()).abs() <= 4 * 2.0 ** -8 * (whole[:, i:i + n].abs().float() + 2.0)).all())
        i += n


def test_streams_and_graphs():
    """On a stream of its own, and captured: forward and backward launches replayed among eager work on other inputs."""
    from semicat_amd import RelativeBias, context_backward, context_forward
    xs = [make(2, 4, 2, 5, 1500, 64, BF16, seed=s, table=(16, torch.float32)) for s in range(3)]
    ds = [{n: t.cuda().transpose(1, 2) if n != "table" else t.cuda() for n, t in x.items()} for x in xs]

    def both(d):
        bias = RelativeBias(d["table"], 64)
        rest = torch.empty_like(d["q"])
        o, lse = context_forward(d["q"], d["k"], d["v"], bias, o_rest=rest)
        return o, *context_backward(d["q"], d["k"], d["v"], o, lse, d["dO"], bias, o_rest=rest)

    want = [both(d) for d in ds]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = both(ds[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(aside, want[1]))
    held = {n: t.clone(memory_format=torch.preserve_format) for n, t in ds[0].items()}
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both(held))
        graphs.append(graph)
    for i in (0, 1, 2, 0, 1):
        for n, t in held.items():
            t.copy_(ds[i][n])
        for graph, out in zip(graphs, outs):
            for t in out:
                t.zero_()
            graph.replay()
            eager = both(ds[(i + 1) % 3])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
            assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3]))
        both(held)


# one launch, a pair of launches, a pair with split axes; few rows in splits
@pytest.mark.parametrize("B,H,G,Lq,Lk,D,table", [(2, 4, 1, 70, 90, 64, None), (3, 4, 2, 70, 300, 32, (16, torch.float32)),
                                                 (1, 2, 2, 130, 1500, 96, (8, BF16)), (2, 4, 4, 3, 3000, 128, None)])
def test_training_passes_in_a_graph(B, H, G, Lq, Lk, D, table):
    """Forward and backward through the autograd surface, captured and replayed on other inputs among eager passes."""
    from semicat_amd import cross_attention, relative_attention
    xs = [{n: t.cuda() for n, t in make(B, H, G, Lq, Lk, D, BF16, seed=s, table=table).items()} for s in range(3)]
    lengths = [torch.tensor([Lk - s] + [Lk // (2 + s)] * (B - 1), dtype=torch.int32, device="cuda") for s in range(3)]

    def step(x, n):
        leaves = [x[m].detach().requires_grad_() for m in ("q", "k", "v", "table") if m in x]
        o = cross_attention(*leaves, key_lengths=n) if table is None else relative_attention(*leaves, 64, key_lengths=n)
        return o.detach(), *torch.autograd.grad(o, leaves, x["dO"])

    want = [step(x, n) for x, n in zip(xs, lengths)]
    held, n = {m: t.clone() for m, t in xs[0].items()}, lengths[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held, n)
    for i in (0, 1, 2, 1):
        for m, t in held.items():
            t.copy_(xs[i][m])
        n.copy_(lengths[i])
        for t in out:
            t.zero_()
        graph.replay()
        eager = step(xs[(i + 1) % 3], lengths[(i + 1) % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3]))


@pytest.mark.parametrize("D,Lk", [(64, 100), (32, 300)])
def test_table_entries_beyond_the_range(D, Lk):
    """NaN in the table is not hidden where a key has it; -inf and the lowest float32 hide their keys."""
    x = make(1, 2, 1, 40, Lk, D, BF16, table=(8, torch.float32))
    x["table"][2, 0] = float("nan")
    got = run(x, max_distance=16)
    assert bool(got["o"][:, 2:, 0].isnan().all()) and bool(got["plain"][:, 2:, 0].isnan().all()) and bool(got["dtable"][2, 0].isnan())
    assert not any(bool(got[n][:, :, 1].isnan().any()) for n in ("o", "plain", "dq", "dk", "dv")) and not bool(got["dtable"][:, 1].isnan().any())
    for low in (float("-inf"), torch.finfo(torch.float32).min):
        x["table"][2, 0] = low
        check(run(x, max_distance=16), x, max_distance=16)


def test_rows_without_work():
    """No batch entry, no query, no key."""
    from semicat_amd import cross_attention
    for B, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        q = torch.randn(B, Lq, 2, 32, device="cuda", dtype=BF16, requires_grad=True)
        k = torch.randn(B, Lk, 2, 32, device="cuda", dtype=BF16, requires_grad=True)
        o = cross_attention(q, k, k)
        assert o.shape == q.shape and o.eq(0).all()
        grads = torch.autograd.grad(o.sum(), (q, k))
        assert all(g.shape == t.shape and g.eq(0).all() for g, t in zip(grads, (q, k)))


def test_long_cache_beyond_32_bits():
    """Rows whose offsets in elements pass 2^31."""
    from semicat_amd import cross_attention
    B, S, H, D = 3, 70000, 96, 128  # 2.6e9 elements
    big = torch.zeros(B, S, H, D, device="cuda", dtype=BF16)
    k, v = (torch.randn(2, 300, H, D, device="cuda", dtype=BF16) for _ in range(2))
    q = torch.randn(2, 2, H, D, device="cuda", dtype=BF16)
    want = cross_attention(q, k, v)
    big[1:, S - 300:], spare = k, torch.zeros_like(big)
    spare[1:, S - 300:] = v
    got = cross_attention(q, big[1:, S - 300:], spare[1:, S - 300:])
    assert torch.equal(got, want)


def test_double_backward_and_forward_mode_are_refused():
    from semicat_amd import cross_attention
    q = torch.randn(1, 8, 2, 32, device="cuda", dtype=BF16, requires_grad=True)
    (g,) = torch.autograd.grad(cross_attention(q, q, q).sum(), q, create_graph=True)
    with pytest.raises(NotImplementedError):
        g.sum().backward()
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: cross_attention(t, t, t), (q.detach(),), (q.detach(),))


def test_ctypes_path_gives_the_same_bits(monkeypatch):
    from semicat_amd import _lib
    x = make(2, 4, 2, 50, 90, 64, BF16, table=(16, torch.float32))
    options = dict(key_lengths=torch.tensor([70, 90], dtype=torch.int32), query_start=torch.tensor([3, -4], dtype=torch.int32), scale=0.3)
    first = run(x, **options)
    plain = run({n: t for n, t in x.items() if n != "table"})
    monkeypatch.setattr(_lib, "_host", False)
    for a, b in ((first, run(x, **options)), (plain, run({n: t for n, t in x.items() if n != "table"}))):
        assert all(torch.equal(a[n], b[n]) for n in a)
    q = torch.randn(1, 8, 2, 32, device="cuda", dtype=BF16, requires_grad=True)
    test_double_backward_and_forward_mode_are_refused()
    g = torch.func.grad(lambda t: run_sum(t))(q.detach())  # (functorch's wrappers take this path always)
    monkeypatch.undo()
    assert torch.equal(g, torch.func.grad(lambda t: run_sum(t))(q.detach()))
    assert torch.equal(g, torch.autograd.grad(run_sum(q), q)[0])


def run_sum(t):
    from semicat_amd import cross_attention
    return cross_attention(t, t, t).float().sum()


def test_other_types_are_computed_in_bfloat16():
    from semicat_amd import cross_attention
    x = make(1, 2, 1, 20, 30, 64, BF16)
    q, k, v = (x[n].float().cuda().requires_grad_() for n in "qkv")
    o = cross_attention(q, k, v)
    g = torch.autograd.grad(o, (q, k, v), x["dO"].float().cuda())
    want = run(x)
    assert o.dtype == torch.float32 and torch.equal(o, want["o"].float())
    assert all(a.dtype == torch.float32 and torch.equal(a, want[n].float()) for a, n in zip(g, ("dq", "dk", "dv")))


def test_strides_that_are_not_served():
    from semicat_amd import _lib, cross_attention
    buf = torch.zeros((1 << 24) + 64, device="cuda", dtype=BF16)
    far = buf.as_strided((1, 2, 1, 32), (1 << 25, 1 << 24, 32, 1))
    with pytest.raises(_lib.SjvpError):
        cross_attention(far, far, far)
    q = torch.randn(1, 2, 1, 32, device="cuda", dtype=BF16, requires_grad=True)
    (got,) = torch.autograd.grad(cross_attention(q, q, q), q, far + 1)
    g = far.copy_(torch.randn(1, 2, 1, 32, device="cuda"))
    assert torch.equal(torch.autograd.grad(cross_attention(q, q, q), q, g)[0], torch.autograd.grad(cross_attention(q, q, q), q, g.contiguous())[0])
