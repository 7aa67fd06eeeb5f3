"""Attention over packed sequences and over a paged cache, as it is timed: whole sequences of different lengths one behind the
other in one tensor (training, and the forward of long prompts), the writing of new keys and values into pages with their
quantisation, the reading back of pages, and the attention of new tokens on what the pages hold.

A case is a plain dict.  ``kind`` says which call it is:

* ``packed_train`` / ``packed_forward``: ``packed_attention(q, k, v, offsets, causal=...)`` on ``[T,H,D]`` tensors that hold ``B``
  sequences of up to ``L`` tokens and ``pad`` rows behind the last one; keys have ``G`` times fewer heads.
* ``paged_write``: ``paged_write(cache, k, v, tables, lengths, offsets)``, the step's up to ``L`` new tokens of each sequence into the pages
  of a cache whose sequences are up to ``K`` tokens long then.
* ``paged_read``: ``paged_read(cache, tables, lengths, K)``, what the cache holds as ``[B,K,H/G,D]`` tensors.
* ``paged_attention``: ``paged_attention(q, cache, tables, lengths, offsets)``, the up to ``L`` newest tokens of each sequence on all tokens
  that the cache holds of it, causal.

The sequences' lengths are spread evenly between ``fill`` times the longest and the longest, in an order of the seed's own.  ``stored`` is
the form of the cache's numbers: ``"same"`` (the type of the tensors) or ``"e4m3"`` (8 bits, and for each 32 columns of a row an 8-bit exponent).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# exponents that a scale may have, by type: within these every number that the 8 bits stand for is one of the type's own
EXPONENTS = {torch.bfloat16: (-117, 120), torch.float16: (-15, 8)}
DEVICE = "cuda"
GROUP = 32


def _packed(name, kind, B, L, fill, pad, H, G, D, dtype, causal):
    c = {"kind": kind, "B": B, "L": L, "fill": fill, "pad": pad, "H": H, "G": G, "D": D, "dtype": dtype, "causal": causal}
    return {"name": name, **c} if name else c


def _paged(name, kind, B, L, K, fill, H, G, D, dtype, page, stored):
    c = {"kind": kind, "B": B, "L": L, "K": K, "fill": fill, "H": H, "G": G, "D": D, "dtype": dtype, "page": page, "stored": stored}
    return {"name": name, **c} if name else c


def listed():
    return [
        # A few short sequences of any length, one of them empty, rows without 16-byte alignment: what a call costs.
        _packed("packed_train_odd", "packed_train", 7, 301, 0.0, 5, 6, 3, 36, "fp16", True),
        # The LM1B network's batch with its sentences packed in place of padded.
        _packed("packed_train_lm1b", "packed_train", 64, 128, 0.125, 0, 12, 1, 64, "bf16", False),
        # Training on long documents with shared key heads.
        _packed("packed_train_long", "packed_train", 4, 6000, 0.25, 0, 16, 4, 128, "bf16", True),
        # Two long prompts before their first token is drawn.
        _packed("packed_prompt_long", "packed_forward", 2, 8192, 0.6, 0, 16, 8, 128, "bf16", True),
        # A generation step writes one token of each sequence.
        _paged("paged_write_step", "paged_write", 64, 1, 4096, 0.3, 16, 4, 128, "bf16", 16, "e4m3"),
        # Whole prompts are written.
        _paged("paged_write_prompt", "paged_write", 8, 4096, 4096, 0.5, 32, 4, 128, "bf16", 64, "e4m3"),
        # A few short sequences are read back, pages of a size that is no power of two.
        _paged("paged_read_odd", "paged_read", 3, 0, 333, 0.1, 6, 3, 80, "fp16", 24, "e4m3"),
        # A serving batch is read back.
        _paged("paged_read_batch", "paged_read", 32, 0, 4096, 0.5, 16, 4, 128, "bf16", 16, "e4m3"),
        # One token of one sequence: latency.
        _paged("paged_step_one", "paged_attention", 1, 1, 128, 1.0, 12, 1, 64, "bf16", 16, "same"),
        # A full serving batch, one token each: reading the quantised cache.
        _paged("paged_step_batch", "paged_attention", 64, 1, 8192, 0.25, 16, 4, 128, "bf16", 16, "e4m3"),
        # Two very long sequences with four draft tokens each: few rows, the cache has to be split.
        _paged("paged_step_long", "paged_attention", 2, 4, 32769, 0.9, 16, 8, 128, "bf16", 64, "same"),
        # Prompts are taken in by chunks, on what is there of them.
        _paged("paged_chunk", "paged_attention", 8, 512, 8192, 0.25, 16, 4, 128, "bf16", 32, "e4m3"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    kind = rng.choice(("packed_train", "packed_train", "packed_forward", "paged_write", "paged_read", "paged_attention", "paged_attention",
                       "paged_attention"))
    while True:
        G = rng.choice((1, 1, 2, 4, 8))
        H = G * rng.randint(1, max(1, 32 // G))
        B, dtype, fill = _log_int(rng, 1, 128), rng.choice(("bf16", "bf16", "fp16")), rng.choice((1.0, 0.5, 0.25, 0.0))
        if kind.startswith("packed"):
            D = rng.choice((16, 20, 32, 36, 48, 64, 64, 64, 80, 96, 128, 128))
            c = _packed(None, kind, B, _log_int(rng, 1, 8192), fill, rng.choice((0, 0, 1, 37)), H, G, D, dtype, rng.random() < 0.8)
            if B * H * c["L"] ** 2 > 5 << 29 or B * c["L"] * H * D > 1 << 27:
                continue
        else:
            D, stored = rng.choice((16, 32, 48, 64, 64, 80, 96, 112, 128, 128)), rng.choice(("same", "e4m3", "e4m3"))
            K = _log_int(rng, 1, 32768 if kind == "paged_attention" else 8192)
            L = 0 if kind == "paged_read" else K if kind == "paged_write" and rng.random() < 0.5 else min(K, _log_int(rng, 1, 1024))
            L = rng.randint(1, 8) if kind == "paged_attention" and rng.random() < 0.5 else L
            c = _paged(None, kind, B, min(L, K), K, fill, H, G, D, dtype, rng.choice((7, 16, 16, 32, 48, 64, 128, 256)), stored)
            if B * K * H // G * D > 1 << 28 or B * H * c["L"] * K > 1 << 31 or B * c["L"] * H * D > 1 << 27:
                continue
        w = work(c)
        if w["flops"] <= most and w["bytes"] <= 2e9:
            return c


def _spread(longest, fill, B):
    """B lengths, evenly from ``fill * longest`` to ``longest``; a batch of one has the longest."""
    least = int(fill * longest)
    return [longest - (longest - least) * i // max(1, B - 1) for i in range(B)]


def _lengths(case):
    """(new, held): the tokens of each sequence that the call brings, and that the cache holds with them."""
    new = _spread(case["L"], case["fill"], case["B"])
    if "K" not in case:
        return new, new
    return new, [max(n, m) for n, m in zip(new, _spread(case["K"], case["fill"], case["B"]))]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    B, H, G, D, dt = case["B"], case["H"], case["G"], case["D"], DTYPES[case["dtype"]]
    ints = {"dtype": torch.int32, "device": DEVICE}

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE).to(dt)

    new, held = (torch.tensor(x, **ints) for x in _lengths(case))
    order = torch.randperm(B, generator=g, device=DEVICE)
    new, held = new[order], held[order]
    offsets = torch.nn.functional.pad(new.cumsum(0), (1, 0)).int()
    T = sum(_lengths(case)[0]) + case.get("pad", 0)
    s = {"case": case, "offsets": offsets}
    if "K" not in case:
        s |= {"q": normal(T, H, D), "k": normal(T, H // G, D), "v": normal(T, H // G, D), "dout": None}
        if case["kind"] == "packed_train":
            s["dout"] = normal(T, H, D)
            for name in "qkv":
                s[name].requires_grad_()
        return s
    # Pages in the order that they came free in, some of them of nobody; what stands in a table behind a sequence's pages is no page.
    size, most = case["page"], -(-max(_lengths(case)[1]) // case["page"])
    count = (held + size - 1) // size
    needed = sum(-(-n // size) for n in _lengths(case)[1])
    pages = needed + needed // 8 + 1
    used = torch.arange(most, device=DEVICE) < count[:, None]
    tables = torch.full((B, most), -1, **ints)
    tables[used] = torch.randperm(pages, generator=g, device=DEVICE)[:needed].int()
    s |= {"tables": tables, "lengths": held, "size": size}
    # Keys have columns that are larger than others; what was written earlier is of that kind.
    column = torch.exp(torch.randn(D, generator=g, device=DEVICE))
    column /= column.square().mean().sqrt()
    shape = (pages, H // G, size, D)
    s["pages"] = [(torch.randn(shape, generator=g, device=DEVICE) * column).to(dt), normal(*shape)]
    if case["stored"] == "e4m3":
        s["pages"] = [y for x in s["pages"] for y in _quantised(x)]
    if case["kind"] == "paged_write":
        s["k"] = (torch.randn((T, H // G, D), generator=g, device=DEVICE) * column).to(dt)
        s["v"] = normal(T, H // G, D)
    elif case["kind"] == "paged_attention":
        s["q"] = normal(T, H, D)
    return s


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    import semicat_amd as sa
    case = state["case"]
    if "K" not in case:
        inputs = [state["q"], state["k"], state["v"]]
        out = sa.packed_attention(*inputs, state["offsets"], causal=case["causal"])
        return out if state["dout"] is None else (out, *torch.autograd.grad(out, inputs, state["dout"]))
    if "cache" not in state:  # the handle that a program makes once
        k, v, *scales = state["pages"] if case["stored"] == "same" else state["pages"][::2] + state["pages"][1::2]
        state["cache"] = sa.PagedCache.of(k, v, *scales, dtype=DTYPES[case["dtype"]])
    cache, tables, lengths = state["cache"], state["tables"], state["lengths"]
    if case["kind"] == "paged_write":
        sa.paged_write(cache, state["k"], state["v"], tables, lengths, state["offsets"])
        return state["pages"]
    if case["kind"] == "paged_read":
        return sa.paged_read(cache, tables, lengths, case["K"])
    return sa.paged_attention(state["q"], cache, tables, lengths, state["offsets"])


def _power(e):
    """2^e for whole numbers e, exactly, as float32 (pow, and ldexp with it, may be off by a rounding)."""
    return ((e + 127).int() << 23).view(torch.float32)


def _quantised(x):
    """``[...,D]`` numbers as 8-bit ones and, for each 32 columns, the exponent of the least power of two by which none of them goes
    beyond 448, the largest 8-bit number.  (With the largest exponent of all, 8-bit numbers end at 240: 256 would be none of the type's.)"""
    lowest, highest = EXPONENTS[x.dtype]
    groups = -(-x.shape[-1] // GROUP)
    y = torch.nn.functional.pad(x.float(), (0, groups * GROUP - x.shape[-1])).unflatten(-1, (groups, GROUP))
    most, power = torch.frexp(torch.where(y.isfinite(), y.abs(), 0.0).amax(-1))
    power = torch.where(most > 0, power - torch.where(most <= 0.875, 9, 8), lowest).clamp(min=lowest)
    y = y * _power(-power[..., None])
    top = torch.where(power == highest, 240.0, 448.0)[..., None]
    y = torch.where(y.isfinite(), torch.minimum(torch.maximum(y, -top), top), math.nan)
    codes = y.flatten(-2)[..., :x.shape[-1]].to(torch.float8_e4m3fn).contiguous()
    return codes, (power + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(pages, k_or_v):
    """The numbers that pages of the cache stand for, in float32."""
    if len(pages) == 2:
        return pages[k_or_v].float()
    codes, scales = pages[2 * k_or_v], pages[2 * k_or_v + 1]
    return codes.float() * scales.float().repeat_interleave(GROUP, -1)[..., :codes.shape[-1]]


def _rows_of(state, positions, seen):
    """The page and the row in it of positions [B,N]; page 0 for those that are not seen."""
    page = state["tables"].gather(1, (positions // state["size"]).clamp(max=state["tables"].shape[1] - 1).long())
    return torch.where(seen, page, 0).long(), torch.where(seen, positions % state["size"], 0).long()


def _held(state, seen):
    """Keys and values of all positions, float32 [B,H,K,D], zeros where a sequence has none."""
    page, row = _rows_of(state, torch.arange(seen.shape[1], device=seen.device).expand_as(seen), seen)
    out = []
    for i in (0, 1):
        pages = [p.view(torch.uint8) if p.dtype.itemsize == 1 else p for p in state["pages"]]
        picked = [p[page, :, row] for p in pages]
        picked = [p.view(q.dtype) for p, q in zip(picked, state["pages"])]
        out.append((_values(picked, i) * seen[:, :, None, None]).transpose(1, 2))
    return out


def _padded(state, x, most):
    """Rows of packed sequences as [B, most, ...], zeros behind each, and which of them there are."""
    start, end = state["offsets"][:-1, None].long(), state["offsets"][1:, None].long()
    at = start + torch.arange(most, device=x.device)
    there = at < end
    return torch.where(there.view(*there.shape, *[1] * (x.ndim - 1)), x[torch.where(there, at, 0)], 0), there


def _unpadded(state, x, there, rows):
    """[B, most, ...] back to packed rows, zeros behind the last sequence."""
    out = torch.zeros(rows, *x.shape[2:], dtype=x.dtype, device=x.device)
    out[:int(there.sum())] = x[there]
    return out


@torch.no_grad()
def _plain(state):
    case = state["case"]
    B, H, G, D = (case[n] for n in "BHGD")
    dt = DTYPES[case["dtype"]]
    device = state["offsets"].device
    if case["kind"] == "paged_write":
        new = state["offsets"].diff()[:, None]
        i = torch.arange(case["L"], device=device)
        page, row = _rows_of(state, (state["lengths"][:, None] - new + i).clamp(min=0), i < new)
        page, row = page[i < new], row[i < new]
        for j, name in enumerate("kv"):
            rows = [state[name]] if case["stored"] == "same" else _quantised(state[name])
            for k, x in enumerate(rows):
                x, to = (t.view(torch.uint8) if t.dtype.itemsize == 1 else t for t in (x, state["pages"][len(rows) * j + k]))
                to[page, :, row] = x
        return state["pages"]
    if case["kind"] == "paged_read":
        seen = torch.arange(case["K"], device=device) < state["lengths"][:, None]
        return tuple(x.transpose(1, 2).to(dt).contiguous() for x in _held(state, seen))
    most = case["L"]
    q, there = _padded(state, state["q"].float(), most)
    q = q.transpose(1, 2)  # [B,H,L,D]
    if "K" in case:
        seen = (torch.arange(case["K"], device=device) < state["lengths"][:, None])
        k, v = _held(state, seen)
        start = (state["lengths"] - state["offsets"].diff())[:, None, None]
    else:
        k, v = (_padded(state, state[n].float(), most)[0].transpose(1, 2) for n in "kv")
        seen, start = there, 0
    keys = k.shape[2]
    grouped = lambda x: x.reshape(B, H // G, G * most, D)  # noqa: E731  (the heads that share a key head, one behind the other)
    scores = (grouped(q) @ k.transpose(-1, -2).contiguous() / math.sqrt(D)).view(B, H // G, G, most, keys)
    mask = seen[:, None, :].expand(B, most, keys)
    if case.get("causal", True):
        mask = mask & (torch.arange(keys, device=device) <= start + torch.arange(most, device=device)[:, None])
    scores.masked_fill_(~mask[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, 1.0)).view(B, H // G, G * most, keys)
    rows = state["q"].shape[0]
    back = lambda x: _unpadded(state, x.reshape(B, -1, most, D).transpose(1, 2), there, rows).to(dt)  # noqa: E731
    out = back(p @ v)
    if state.get("dout") is None:
        return out
    dout = grouped(_padded(state, state["dout"].float(), most)[0].transpose(1, 2))
    dp = dout @ v.transpose(-1, -2).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = ds @ k / math.sqrt(D)
    dk = ds.transpose(-1, -2).contiguous() @ grouped(q) / math.sqrt(D)
    dv = p.transpose(-1, -2).contiguous() @ dout
    return out, back(dq), back(dk), back(dv)


def work(case):
    B, H, G, D = (case[n] for n in "BHGD")
    new, held = _lengths(case)
    if "K" not in case:
        pairs = H * sum(n * (n + 1) / 2 if case["causal"] else n * n for n in new)
        rows, cols = (sum(new) + case["pad"]) * H * D * 2, (sum(new) + case["pad"]) * H // G * D * 2
        if case["kind"] == "packed_train":  # q, o, dO and dq; k, v, dk and dv; seven contractions, each input of both passes once
            return {"bytes": 4 * rows + 4 * cols, "flops": 14 * pairs * D}
        return {"bytes": 2 * rows + 2 * cols, "flops": 4 * pairs * D}
    # a row of a page: K and V of all heads
    stored = 2 * H // G * (2 * D if case["stored"] == "same" else D + -(-D // GROUP))
    dense = 2 * H // G * 2 * D
    if case["kind"] == "paged_write":
        return {"bytes": sum(new) * (dense + stored), "flops": 0}
    if case["kind"] == "paged_read":  # what lies behind a length is written as zeros
        return {"bytes": sum(held) * stored + B * case["K"] * dense, "flops": 0}
    pairs = H * sum(n * (m - n) + n * (n + 1) / 2 for n, m in zip(new, held))
    return {"bytes": sum(held) * stored + 2 * sum(new) * H * D * 2, "flops": 4 * pairs * D}


def _eight_bits(x, dtype):
    """What 8-bit numbers and their exponents hold of ``[...,D]``, by the definition: the format's numbers are multiples of
    2^(max(e, -6) - 3) for a number in [2^e, 2^(e+1)), the nearest one counts and of two the even multiple."""
    lowest, highest = EXPONENTS[dtype]
    D = x.shape[-1]
    codes, scales = torch.empty_like(x), torch.empty(*x.shape[:-1], -(-D // GROUP), dtype=x.dtype, device=x.device)
    powers = torch.tensor([2.0 ** e for e in range(lowest, highest + 1)], dtype=x.dtype, device=x.device)
    for g in range(scales.shape[-1]):
        part = x[..., g * GROUP:(g + 1) * GROUP]
        biggest = part.abs().amax(-1, keepdim=True)
        scale = powers[(biggest > 448 * powers).sum(-1, keepdim=True).clamp(max=len(powers) - 1)]
        y = part / scale
        e = sum((y.abs() >= 2.0 ** k).to(x.dtype) for k in range(-5, 9)) - 6
        unit = torch.tensor([2.0 ** k for k in range(-9, 6)], dtype=x.dtype, device=x.device)[(e + 6).long()]
        limit = torch.where(scale == powers[-1], 240.0, 448.0)
        codes[..., g * GROUP:(g + 1) * GROUP] = (torch.round(y / unit) * unit).clamp(-limit, limit)
        scales[..., g:g + 1] = scale
    return codes, scales


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    B, H, G, D = (case[n] for n in "BHGD")
    f64 = torch.float64
    offsets = state["offsets"].tolist()
    paged = "K" in case
    if paged:
        # the row of the flattened pages that each sequence's positions have
        lengths, size = state["lengths"].tolist(), state["size"]
        at = [(state["tables"][b, torch.arange(lengths[b], device=DEVICE) // size].long(), torch.arange(lengths[b], device=DEVICE) % size)
              for b in range(B)]

        def stored(x, b, h):
            """K (x = 0) or V of a sequence's head in the cache."""
            if case["stored"] == "same":
                return state["pages"][x][at[b][0], h, at[b][1]].to(f64)
            codes = state["pages"][2 * x].view(torch.uint8)[at[b][0], h, at[b][1]].view(torch.float8_e4m3fn).float().to(f64)
            scale = state["pages"][2 * x + 1].view(torch.uint8)[at[b][0], h, at[b][1]].long()
            scale = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=f64, device=DEVICE)[scale]
            return codes * scale[:, torch.arange(D, device=DEVICE) // GROUP]

    if case["kind"] == "paged_read":
        out = [torch.zeros(B, case["K"], H // G, D, dtype=f64, device=DEVICE) for _ in range(2)]
        for b in range(B):
            for h in range(H // G):
                for x in (0, 1):
                    out[x][b, :lengths[b], h] = stored(x, b, h)
        return tuple(out)
    if case["kind"] == "paged_write":
        out = [p.float().to(f64) for p in state["pages"]]
        for b in range(B):
            n = offsets[b + 1] - offsets[b]
            page, row = (t[lengths[b] - n:] for t in at[b])
            for x, name in enumerate("kv"):
                rows = state[name][offsets[b]:offsets[b + 1]].to(f64)
                parts = [rows] if case["stored"] == "same" else _eight_bits(rows, state[name].dtype)
                for y, part in enumerate(parts):
                    out[len(parts) * x + y][page, :, row] = part
        return out
    out = torch.zeros(state["q"].shape, dtype=f64, device=DEVICE)
    train = state.get("dout") is not None
    dq = torch.zeros_like(out)
    dk, dv = (torch.zeros(state["q"].shape[0], H // G, D, dtype=f64, device=DEVICE) for _ in range(2))
    for b in range(B):
        rows = slice(offsets[b], offsets[b + 1])
        n = offsets[b + 1] - offsets[b]
        if n == 0:
            continue
        held = lengths[b] if paged else n
        hidden = torch.arange(held, device=DEVICE) > held - n + torch.arange(n, device=DEVICE)[:, None]
        for h in range(H):
            q = state["q"][rows, h].to(f64)
            k, v = (stored(x, b, h // G) if paged else state["kv"[x]][rows, h // G].to(f64) for x in (0, 1))
            s = q @ k.t() / D ** 0.5
            if case.get("causal", True):
                s[hidden] = -math.inf
            p = torch.softmax(s, dim=-1)
            out[rows, h] = p @ v
            if train:
                do = state["dout"][rows, h].to(f64)
                ds = p * (do @ v.t() - (do * out[rows, h]).sum(-1, keepdim=True))
                dq[rows, h] = ds @ k / D ** 0.5
                dk[rows, h // G] += ds.t() @ q / D ** 0.5
                dv[rows, h // G] += p.t() @ do
    return (out, dq, dk, dv) if train else out
