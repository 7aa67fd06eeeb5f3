"""Attention over packed sequences (csrc/sjvp_seq*) against the definition in float64; the tolerances stand at packed_oracle.limit."""
import pytest
import torch

from oracle import packed_oracle as orc

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def make(T, H, G, D, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda h, s=1.0: (torch.randn(T, h, D, generator=g) * s).to(dtype)
    return {"q": r(H, spread), "k": r(H // G, spread), "v": r(H // G), "dO": r(H)}


def offsets_of(lengths, front=0):
    out = [front]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def run(x, offsets, causal, scale=None):
    from semicat_amd import packed_attention
    d = {n: t.cuda() for n, t in x.items()}
    leaves = [d[n].requires_grad_() for n in "qkv"]
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    o = packed_attention(*leaves, at, causal=causal, scale=scale)
    grads = torch.autograd.grad(o, leaves, d["dO"])
    with torch.no_grad():
        plain = packed_attention(*leaves, at, causal=causal, scale=scale)
    torch.cuda.synchronize()
    assert torch.equal(plain, o)
    return {"o": o.detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def check(got, x, offsets, causal, scale=None):
    want, sizes = orc.packed(x["q"], x["k"], x["v"], offsets, causal, x["dO"], scale)
    for name, t in got.items():
        assert t.dtype == x["q"].dtype and t.shape == want[name].shape, name
        off = (t.cpu().double() - want[name]).abs()
        limit = orc.limit(want[name], sizes[name], t.dtype)
        assert bool((off <= limit).all()), (name, float((off / limit).max()), int((off > limit).sum()))
        empty = torch.ones(t.shape[0], dtype=torch.bool)
        empty[offsets[0]:offsets[-1]] = False
        assert not t.cpu()[empty].any(), name


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,G,D,dtype", [(2, 1, 64, BF16), (4, 2, 128, BF16), (6, 3, 36, FP16), (3, 1, 16, BF16), (5, 5, 20, BF16),
                                         (2, 2, 80, FP16), (2, 1, 96, BF16), (8, 8, 128, FP16), (1, 1, 33, BF16), (4, 1, 127, FP16)])
def test_lengths_heads_and_types(H, G, D, dtype, causal):
    lengths = [1, 0, 37, 128, 2, 129, 0, 0, 63, 64, 65, 200]
    offsets = offsets_of(lengths)
    x = make(offsets[-1], H, G, D, dtype, seed=D + causal)
    check(run(x, offsets, causal), x, offsets, causal)


@pytest.mark.parametrize("lengths,front,behind", [([1], 0, 0), ([0], 0, 3), ([0, 0], 0, 140), ([1, 1, 1], 0, 0), ([5], 7, 0), ([130, 3], 129, 261),
                                                  ([700], 0, 1), ([33] * 70, 1, 2), ([0] * 80 + [9] + [0] * 80, 0, 0), ([127, 1, 129], 0, 0)])
@pytest.mark.parametrize("causal", [True, False])
def test_places_of_the_sequences(lengths, front, behind, causal):
    offsets = offsets_of(lengths, front)
    x = make(offsets[-1] + behind, 2, 2, 64, BF16, seed=len(lengths))
    check(run(x, offsets, causal), x, offsets, causal)


@pytest.mark.parametrize("D,dtype,G", [(64, BF16, 1), (128, BF16, 4), (48, FP16, 2)])
def test_long_sequences(D, dtype, G):
    offsets = offsets_of([1500, 77, 1025])
    x = make(offsets[-1], 4, G, D, dtype)
    for causal in (True, False):
        check(run(x, offsets, causal), x, offsets, causal)


@pytest.mark.parametrize("spread,scale", [(6.0, None), (30.0, None), (1.0, 3.0), (0.0, None)])
def test_sharp_rows_and_scales(spread, scale):
    """Scores of some hundreds to some thousands: the statistics are two numbers, so that the backward's P does not lose its sum beside them."""
    offsets = offsets_of([90, 1, 140])
    x = make(offsets[-1], 4, 2, 64, BF16, spread=spread)
    check(run(x, offsets, True, scale), x, offsets, True, scale)


def test_equal_large_scores():
    """Keys that are all alike beside scores of 1e6 share the weight, in the gradients too."""
    offsets = [0, 100]
    x = make(100, 2, 1, 64, BF16)
    x["q"][:], x["k"][:] = 320.0, 400.0  # (scale 1/8: 1.024e6)
    got = run(x, offsets, True)
    want, _ = orc.packed(x["q"], x["k"], x["v"], offsets, True, x["dO"])
    for name in ("o", "dv"):
        assert float((got[name].cpu().double() - want[name]).abs().max()) <= 2.0 ** -6 * float(want[name].abs().max()), name


def test_one_key_has_no_gradient_of_its_score():
    offsets = offsets_of([1, 1, 1, 1])
    x = make(4, 4, 2, 64, BF16)
    for causal in (True, False):
        got = run(x, offsets, causal)
        assert not got["dq"].any() and not got["dk"].any()
        assert torch.equal(got["o"].cpu(), x["v"].repeat_interleave(2, 1))
    x = make(5, 2, 1, 64, BF16)
    got = run(x, [0, 3, 5], True)
    assert not got["dq"].cpu()[[0, 3]].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_nobody_are_not_used(bad):
    offsets = offsets_of([70, 0, 61], 9)
    x = make(offsets[-1] + 40, 4, 2, 64, BF16)
    for t in x.values():
        t[:9], t[offsets[-1]:] = bad, bad
    clean = {n: t.clone() for n, t in x.items()}
    for t in clean.values():
        t[:9], t[offsets[-1]:] = 0.0, 0.0
    check(run(x, offsets, True), clean, offsets, True)


@pytest.mark.parametrize("D,G", [(64, 1), (128, 2), (48, 4), (96, 1), (20, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_numbers_that_a_row_does_not_see(D, G, bad):
    """Tokens with infinities or NaN among their numbers do not reach the tokens in front of them (but for the last bits: rows of a wave raise
    their maxima together)."""
    from semicat_amd import packed_attention
    offsets, hurt = offsets_of([70, 1, 300, 129]), {0: 33, 2: 130, 3: 128}  # (sequence: its first such token)
    x = make(offsets[-1], 4, G, D, BF16)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    want, sizes = orc.packed(x["q"], x["k"], x["v"], offsets, True)
    limit = orc.limit(want["o"], sizes["o"], BF16)
    for b, i in hurt.items():
        x["v"][offsets[b] + i, :, 3], x["v"][offsets[b + 1] - 1] = bad, bad
        x["k"][offsets[b] + i, :, 1] = bad
        x["q"][offsets[b] + i, 0] = bad
    got = packed_attention(*(x[n].cuda() for n in "qkv"), at).cpu()
    off = (got.double() - want["o"]).abs()
    for b, (s, e) in enumerate(zip(offsets, offsets[1:])):
        i = s + hurt.get(b, e - s)
        assert bool((off[s:i] <= limit[s:i]).all()), b
        assert not got[i:e].isfinite().all(-1).any(), b


@pytest.mark.parametrize("D,G", [(64, 1), (128, 2), (48, 4), (96, 1), (20, 2), (128, 8)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_gradients_of_numbers_that_a_row_does_not_see(D, G, bad):
    """Infinities and NaN of a key or value do not reach the gradients of queries in front of it, those of a query or of its
    result's gradient not the keys behind it."""
    from semicat_amd import packed_attention
    offsets = offsets_of([70, 200, 300, 129, 260])
    hurt_keys, hurt_rows = {0: 33, 2: 130, 3: 128}, {1: 70, 4: 128}  # (sequence: the token)
    x = make(offsets[-1], 8, G, D, BF16)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    want, sizes = orc.packed(x["q"], x["k"], x["v"], offsets, True, x["dO"])
    for b, i in hurt_keys.items():
        x["k"][offsets[b] + i, :, 5] = bad
        x["v"][offsets[b] + i, :, 3], x["v"][offsets[b + 1] - 1] = bad, bad
    for b, i in hurt_rows.items():
        x["q"][offsets[b] + i, :, 7], x["dO"][offsets[b] + i, :, 9] = bad, bad
    leaves = [x[n].cuda().requires_grad_() for n in "qkv"]
    grads = torch.autograd.grad(packed_attention(*leaves, at), leaves, x["dO"].cuda())
    for name, t in zip(("dq", "dk", "dv"), grads):
        off, limit = (t.cpu().double() - want[name]).abs(), orc.limit(want[name], sizes[name], BF16)
        for b, (s, e) in enumerate(zip(offsets, offsets[1:])):
            clean = torch.arange(s, e)
            if b in hurt_keys:
                i = s + hurt_keys[b]
                clean, rest = clean[:i - s if name == "dq" else 0], torch.arange(i, e) if name == "dq" else clean
            else:
                i = s + hurt_rows[b]
                clean, rest = (clean[clean != i], torch.tensor([i])) if name == "dq" else (clean[i - s + 1:], torch.arange(s, i + 1))
            assert bool((off[clean] <= limit[clean]).all()), (name, b)
            if name == "dv" and b in hurt_keys and bad == bad:
                continue  # (a score of -inf is a probability of zero)
            assert not t.cpu()[rest].isfinite().all(-1).any(), (name, b)


def test_neighbours_do_not_mix():
    """NaN in one sequence stays there."""
    offsets = offsets_of([40, 50, 60])
    x = make(150, 2, 1, 64, BF16)
    clean = run(x, offsets, True)
    for t in x.values():
        t[40:90] = float("nan")
    from semicat_amd import packed_attention
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    leaves = [x[n].cuda().requires_grad_() for n in "qkv"]
    o = packed_attention(*leaves, at)
    grads = torch.autograd.grad(o, leaves, x["dO"].cuda())
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        assert torch.equal(t[:40], clean[name][:40]) and torch.equal(t[90:], clean[name][90:]), name
        # (the first token sees one key: no gradient of its score, whatever the numbers)
        assert t[41:90].isnan().all() and (name == "dq" or t[40].isnan().all()), name


@pytest.mark.parametrize("D", [64, 36, 128])
def test_strides_and_alignment(D):
    """q, k and v as slices of one projection, and at odd places."""
    from semicat_amd import packed_attention
    offsets = offsets_of([100, 30])
    x = make(130, 2, 1, D, BF16)
    want = run(x, offsets, True)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    fused = torch.stack([x[n] for n in "qkv"], 1).cuda().requires_grad_()  # [T,3,H,D]
    o = packed_attention(fused[:, 0], fused[:, 1], fused[:, 2], at)
    d, = torch.autograd.grad(o, [fused], x["dO"].cuda())
    for i, n in enumerate(("dq", "dk", "dv")):
        assert torch.equal(d[:, i], want[n]), n
    assert torch.equal(o, want["o"])
    odd = []
    for n in "qkv":
        room = torch.zeros(130, 3, D + 5, dtype=BF16, device="cuda")
        room[:, 1:, 3:3 + D] = x[n].cuda()
        odd.append(room[:, 1:, 3:3 + D].requires_grad_())
    wide = torch.zeros(2, 130, D, dtype=BF16, device="cuda").transpose(0, 1)
    wide.copy_(x["dO"])
    o = packed_attention(*odd, at)
    grads = torch.autograd.grad(o, odd, wide)
    tight = {n: t for n, t in zip(("o", "dq", "dk", "dv"), (o, *grads))}
    check({n: t.detach() for n, t in tight.items()}, x, offsets, True)


def test_other_types_and_partial_gradients():
    from semicat_amd import packed_attention
    offsets = offsets_of([33, 20])
    x = make(53, 2, 1, 64, BF16)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    want = run(x, offsets, True)
    q, k, v = (x[n].float().cuda() for n in "qkv")
    q.requires_grad_()
    o = packed_attention(q, k, v, at)
    assert o.dtype == torch.float32 and torch.equal(o, want["o"].float())
    dq, = torch.autograd.grad(o, [q], x["dO"].float().cuda())
    assert dq.dtype == torch.float32 and torch.equal(dq, want["dq"].float())
    q, k, v = (x[n].cuda() for n in "qkv")
    v.requires_grad_()
    dv, = torch.autograd.grad(packed_attention(q, k, v, at), [v], x["dO"].cuda())
    assert torch.equal(dv, want["dv"])


def test_gradients_against_differences():
    """The three gradients along a direction against central differences of the float64 definition."""
    offsets, causal = offsets_of([24, 9]), True
    x = make(33, 2, 2, 32, FP16)
    got = run(x, offsets, causal)
    g = torch.Generator().manual_seed(5)
    for name in "qkv":
        way = torch.randn(x[name].shape, generator=g).double()
        value = lambda s: float((orc.packed(*((x[n].double() + s * way if n == name else x[n].double()) for n in "qkv"), offsets, causal)[0]["o"]
                                 * x["dO"].double()).sum())
        slope = (value(1e-4) - value(-1e-4)) / 2e-4
        got_slope = float((got["d" + name].cpu().double() * way).sum())
        # each of the gradient's numbers is off by its limit at most, and the differences by their third order
        _, sizes = orc.packed(x["q"], x["k"], x["v"], offsets, causal, x["dO"])
        want = orc.packed(x["q"], x["k"], x["v"], offsets, causal, x["dO"])[0]["d" + name]
        most = float((orc.limit(want, sizes["d" + name], FP16) * way.abs()).sum()) + 1e-5 * abs(slope) + 1e-5
        assert abs(slope - got_slope) <= most, name


def test_the_same_bits_every_time():
    offsets = offsets_of([300, 17, 256])
    x = make(573, 4, 2, 64, BF16)
    first = run(x, offsets, True)
    for _ in range(3):
        again = run(x, offsets, True)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_descending_offsets_stay_in_bounds():
    """Offsets that make no sense give rows of no use; what lies around the tensors is not touched."""
    from semicat_amd import packed_attention
    T = 200
    room = torch.full((3, 3 * T, 2, 64), 7.0, dtype=BF16, device="cuda")
    q, k, v = (room[i, T:2 * T] for i in range(3))
    for bad in ([50, 20, 180], [0, 500, 100], [-5, 90, 1 << 30], [300, 300, -1]):
        at = torch.tensor(bad, dtype=torch.int32, device="cuda")
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = packed_attention(*leaves, at)
        torch.autograd.grad(o, leaves, torch.ones_like(o))
    torch.cuda.synchronize()
    assert bool((room == 7.0).all())


def test_streams_and_graph_replays():
    from semicat_amd import packed_attention
    offsets = offsets_of([100, 150])
    x = make(250, 4, 2, 64, BF16)
    want = run(x, offsets, True)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    q, k, v = (x[n].cuda() for n in "qkv")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = packed_attention(q, k, v, at)
    side.synchronize()
    assert torch.equal(got, want["o"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = packed_attention(q, k, v, at)
    other = offsets_of([30, 0])
    y = make(250, 4, 2, 64, BF16, seed=9)
    for offs, z in ((offsets, x), (other, y), (offsets, x)):
        for t, n in zip((q, k, v), "qkv"):
            t.copy_(z[n])
        at.copy_(torch.tensor(offs, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, run(z, offs, True)["o"])


def test_a_captured_backward_replays():
    from semicat_amd import packed_backward, packed_forward
    offsets = offsets_of([100, 150])
    x = make(250, 4, 2, 64, BF16)
    want = run(x, offsets, True)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    q, k, v, g = (x[n].cuda() for n in ("q", "k", "v", "dO"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = packed_forward(q, k, v, at)
        grads = packed_backward(q, k, v, o, lse, g, at)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for t, n in zip((o, *grads), ("o", "dq", "dk", "dv")):
            assert torch.equal(t, want[n]), n
        run(x, offsets, False)


@pytest.mark.parametrize("causal", [True, False])
def test_thousands_of_sequences(causal):
    g = torch.Generator().manual_seed(0)
    offsets = offsets_of(torch.randint(0, 3, (4200,), generator=g).tolist(), 3)  # (a search in three steps)
    x = make(offsets[-1] + 2, 1, 1, 16, BF16)
    check(run(x, offsets, causal), x, offsets, causal)


@pytest.mark.parametrize("D,G", [(64, 2), (128, 1), (36, 2)])
def test_broadcast_inputs(D, G):
    """Keys, values and cotangents that are one row seen many times: the same numbers as their copies, gradients summed over the broadcast."""
    from semicat_amd import packed_attention
    T, offsets = 200, offsets_of([150, 50])
    x = make(T, 4, G, D, BF16)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    q = x["q"].cuda()
    for shape in ((1, 1, D), (T, 1, D), (1, 4 // G, D)):
        k, v = (x[n][:shape[0], :shape[1]].cuda() for n in "kv")
        cot = x["dO"][:shape[0], :1].cuda().expand(T, 4, D)
        wide = [t.expand(T, 4 // G, D) for t in (k, v)]
        leaves = [q.clone().requires_grad_(), *(t.clone().requires_grad_() for t in wide)]
        want = torch.autograd.grad(packed_attention(*leaves, at), leaves, cot.contiguous())
        leaves = [q.clone().requires_grad_(), *(t.clone().requires_grad_() for t in (k, v))]
        got = torch.autograd.grad(packed_attention(leaves[0], *(t.expand(T, 4 // G, D) for t in leaves[1:]), at), leaves, cot)
        assert torch.equal(got[0], want[0])
        for a, b, t in zip(got[1:], want[1:], (k, v)):
            assert torch.equal(a, b.sum_to_size(t.shape))


def test_function_transforms():
    from semicat_amd import packed_attention
    offsets = offsets_of([40, 33])
    x = make(73, 2, 1, 64, BF16)
    want = run(x, offsets, True)
    at = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    q, k, v, dO = (x[n].cuda() for n in ("q", "k", "v", "dO"))
    o, pull = torch.func.vjp(lambda *t: packed_attention(*t, at), q, k, v)
    assert torch.equal(o, want["o"])
    for a, n in zip(pull(dO), ("dq", "dk", "dv")):
        assert torch.equal(a, want[n])
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: packed_attention(t, k, v, at), (q,), (q,))
    with pytest.raises(Exception):
        torch.func.vmap(lambda t: packed_attention(t, k, v, at))(q[None])
    torch.cuda.synchronize()


def test_places_beyond_32_bits():
    """The last rows of tensors of more than 4 GiB."""
    from semicat_amd import packed_attention
    T, H, D, tail = 2_200_000, 8, 128, 330
    x = make(tail, H, 1, D, BF16)
    big = {n: torch.zeros(T, H, D, dtype=BF16, device="cuda") for n in x}
    for n, t in x.items():
        big[n][T - tail:] = t.cuda()
    results = []
    for tensors, first in (({n: t.cuda() for n, t in x.items()}, 0), (big, T - tail)):
        at = torch.tensor([first, first + 200, first + tail], dtype=torch.int32, device="cuda")
        leaves = [tensors[n].requires_grad_() for n in "qkv"]
        o = packed_attention(*leaves, at)
        results.append([o.detach(), *torch.autograd.grad(o, leaves, tensors["dO"])])
    for small, large in zip(*results):
        assert torch.equal(small, large[T - tail:]) and not large[:T - tail].any()
