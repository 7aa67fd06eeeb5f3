"""The attention operators beside the attention-JVP op, as they are timed: cross attention to an encoder's states and
attention with a learned relative position bias, each in training (forward and every gradient), in a forward without
gradients and for the few query rows of a generation step.

A case is a plain dict.  ``kind`` says which call it is:

* ``cross_train`` / ``cross_forward`` / ``cross_step``: ``cross_attention(q, k, v, key_lengths=...)`` on ``[B,S,H,D]`` tensors,
  keys of another length and, with ``G`` > 1, of ``G`` times fewer heads than the queries.
* ``relative_train`` / ``relative_forward`` / ``relative_step``: ``relative_attention(q, k, v, table, ...)``, scores with
  ``table[bucket(key position - query position), head]`` added; in a step the keys are a cache whose rows lie ahead of the queries.

``fill`` is the least share of ``Lk`` that a sequence of the batch has (1.0: no lengths are handed over).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


def _cross(name, kind, B, H, G, Lq, Lk, D, dtype, fill):
    c = {"kind": kind, "B": B, "H": H, "G": G, "Lq": Lq, "Lk": Lk, "D": D, "dtype": dtype, "fill": fill}
    return {"name": name, **c} if name else c


def _relative(name, kind, B, H, G, Lq, Lk, D, dtype, fill, buckets, distance, both, causal, table):
    return {**_cross(name, kind, B, H, G, Lq, Lk, D, dtype, fill), "buckets": buckets, "distance": distance, "both": both,
            "causal": causal, "table": table}


def listed():
    return [
        # One token of one sequence that looks at 128 states: what a call costs when there is next to nothing to do.
        _cross("cross_step_one", "cross_step", 1, 12, 1, 1, 128, 64, "bf16", 1.0),
        # A full serving batch, one token each, on the states of long inputs with shared key heads: reading the states.
        _cross("cross_step_batch", "cross_step", 64, 16, 4, 1, 2048, 128, "bf16", 0.5),
        # Two sequences with a very long input, four draft tokens each: few rows, the key axis has to be split.
        _cross("cross_step_long", "cross_step", 2, 16, 8, 4, 16385, 128, "bf16", 0.9),
        # The LM1B network's batch conditioned on 256 encoder states of ragged lengths.
        _cross("cross_train_lm1b", "cross_train", 64, 12, 1, 128, 256, 64, "bf16", 0.25),
        # Ragged lengths on both sides, shared heads, a head dimension between the usual ones.
        _cross("cross_train_ragged", "cross_train", 4, 6, 3, 333, 205, 48, "fp16", 0.0),
        # Long documents at the widest head with shared key heads.
        _cross("cross_train_long", "cross_train", 8, 16, 4, 2048, 1024, 128, "bf16", 0.5),
        # Sampling: a forward of long sequences on a long condition.
        _cross("cross_forward_long", "cross_forward", 8, 16, 1, 4096, 1024, 64, "bf16", 0.5),
        # A decoder's step on its cache, 32 sequences.
        _relative("relative_step_batch", "relative_step", 32, 12, 1, 1, 1024, 64, "bf16", 0.25, 32, 128, False, True, "bf16"),
        # The LM1B network with buckets in place of its rotary embedding; the table is a float32 parameter.
        _relative("relative_train_lm1b", "relative_train", 64, 12, 1, 128, 128, 64, "bf16", 1.0, 32, 128, True, False, "fp32"),
        # The character-level network, twice the batch and the sequence.
        _relative("relative_train_text8", "relative_train", 128, 12, 1, 256, 256, 64, "bf16", 1.0, 32, 128, True, False, "fp32"),
        # Rows without 16-byte alignment, causal, padded batch.
        _relative("relative_train_odd", "relative_train", 8, 8, 2, 300, 300, 36, "fp16", 0.3, 24, 77, False, True, "fp16"),
        # The longest sequences of the sweep, causal.
        _relative("relative_train_long", "relative_train", 8, 16, 1, 4096, 4096, 64, "bf16", 1.0, 32, 128, False, True, "fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = work(listed()[-1])["flops"] / 2
    kind = rng.choice(("cross_train", "cross_train", "cross_forward", "cross_step", "relative_train", "relative_train",
                       "relative_forward", "relative_step"))
    while True:
        step, relative = kind.endswith("step"), kind.startswith("relative")
        G = rng.choice((1, 1, 2, 4, 8))
        H = G * rng.randint(1, max(1, 16 // G))
        D = rng.choice((16, 20, 32, 36, 48, 64, 64, 64, 80, 96, 128, 128))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        Lk = _log_int(rng, 1, 32768 if step else 4096)
        Lq = rng.randint(1, min(8, Lk)) if step else Lk if relative and rng.random() < 0.8 else _log_int(rng, 1, 4096)
        args = (None, kind, _log_int(rng, 1, 128), H, G, Lq, Lk, D, dtype, rng.choice((1.0, 0.5, 0.25, 0.0)))
        if relative:
            both = not step and rng.random() < 0.5
            buckets = rng.choice((8, 16, 32, 32, 64))
            c = _relative(*args, buckets, rng.randint(buckets, 512), both, step or (not both and rng.random() < 0.8),
                          rng.choice((dtype, "fp32")))
        else:
            c = _cross(*args)
        w = work(c)
        if w["flops"] <= most and w["bytes"] <= 2e9 and c["B"] * H * Lq * Lk <= 1 << 31 and max(Lq, Lk) * c["B"] * H * D <= 1 << 26:
            return c


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    B, H, Lq, Lk, D, dt = case["B"], case["H"], case["Lq"], case["Lk"], case["D"], DTYPES[case["dtype"]]
    train, relative, step = case["kind"].endswith("train"), case["kind"].startswith("relative"), case["kind"].endswith("step")

    def normal(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=DEVICE).to(dtype)

    s = {"case": case, "q": normal(B, Lq, H, D), "k": normal(B, Lk, H // case["G"], D), "v": normal(B, Lk, H // case["G"], D),
         "lengths": None, "start": 0, "table": None, "dout": normal(B, Lq, H, D) if train else None}
    if case["fill"] < 1.0:
        # the longest sequence fills the batch's tensor; a step's cache holds at least the step's own rows
        least = max(int(case["fill"] * Lk), Lq if step and relative else 0)
        share = torch.rand(B, generator=g, device=DEVICE)
        share[0] = 1.0
        s["lengths"] = (least + (share * (Lk + 1 - least)).int()).clamp(max=Lk).int()
    if relative:
        s["table"] = normal(case["buckets"], H, dtype=DTYPES[case["table"]])
        if step:
            s["start"] = Lk - Lq if s["lengths"] is None else s["lengths"] - Lq
    for name in ("q", "k", "v", "table"):
        if train and s[name] is not None:
            s[name].requires_grad_()
    return s


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from semicat_amd import cross_attention, relative_attention
    case, inputs = state["case"], [state["q"], state["k"], state["v"]]
    if state["table"] is None:
        out = cross_attention(*inputs, key_lengths=state["lengths"])
    else:
        inputs.append(state["table"])
        out = relative_attention(*inputs, max_distance=case["distance"], bidirectional=case["both"], causal=case["causal"],
                                 key_lengths=state["lengths"], query_start=state["start"])
    if state["dout"] is None:
        return out
    return (out, *torch.autograd.grad(out, inputs, state["dout"]))


def _buckets(relative, case):
    """The bucket of every position difference (key minus query): half of the buckets of a direction are single distances, the
    others grow with the distance's logarithm up to ``distance``.  The logarithms are taken in 64 bits and lifted by more
    than their rounding and less than the least gap of a distance below a border."""
    n = case["buckets"] // 2 if case["both"] else case["buckets"]
    single = n // 2
    d = relative.abs() if case["both"] else (-relative).clamp(min=0)
    far = torch.log(d.clamp(min=1).double() / single) / math.log(case["distance"] / single) * (n - single)
    bucket = torch.where(d < single, d, (single + torch.floor(far + 1e-9).long()).clamp(max=n - 1))
    return bucket + (relative > 0).long() * n if case["both"] else bucket


@torch.no_grad()
def _plain(state):
    case, dt = state["case"], state["q"].dtype
    B, H, G, Lq, Lk, D = (case[n] for n in ("B", "H", "G", "Lq", "Lk", "D"))
    q, k, v = (state[n].float().transpose(1, 2) for n in "qkv")
    k, v = (t.repeat_interleave(G, dim=1) for t in (k, v))
    scores = q @ k.transpose(-1, -2).contiguous() / math.sqrt(D)
    keys = torch.arange(Lk, device=q.device)
    seen = torch.ones(1, 1, 1, Lk, dtype=torch.bool, device=q.device)
    if state["lengths"] is not None:
        seen = (keys < state["lengths"][:, None])[:, None, None]
    if state["table"] is not None:
        start = torch.as_tensor(state["start"], device=q.device).reshape(-1, 1, 1)
        relative = keys - (start + torch.arange(Lq, device=q.device)[:, None])  # [B or 1, Lq, Lk]
        scores += state["table"].float()[_buckets(relative, case)].permute(0, 3, 1, 2)
        if case["causal"]:
            seen = seen & (relative <= 0)[:, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    out = (p @ v).transpose(1, 2).to(dt)
    if state["dout"] is None:
        return out
    dout = state["dout"].float().transpose(1, 2)
    dp = dout @ v.transpose(-1, -2).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = (ds @ k).transpose(1, 2) / math.sqrt(D)
    dk = (ds.transpose(-1, -2).contiguous() @ q).view(B, H // G, G, Lk, D).sum(2).transpose(1, 2) / math.sqrt(D)
    dv = (p.transpose(-1, -2).contiguous() @ dout).view(B, H // G, G, Lk, D).sum(2).transpose(1, 2)
    grads = [out, dq.to(dt), dk.to(dt), dv.to(dt)]
    if state["table"] is not None:
        # Sums along the diagonals: rows in reverse order, padded to Lk + Lq columns, read again as rows of one column less,
        # stand one column further right from each row to the next.  They are long, so in 64 bits.
        rows = torch.nn.functional.pad(ds.sum(0, dtype=torch.float64).flip(1), (0, Lq)).flatten(1)
        diagonals = rows[:, :Lq * (Lq + Lk - 1)].view(H, Lq, Lq + Lk - 1).sum(1)
        bucket = _buckets(torch.arange(1 - Lq, Lk, device=q.device), case)
        hot = (bucket[:, None] == torch.arange(case["buckets"], device=q.device)).double()
        grads.append((diagonals @ hot).t().to(state["table"].dtype))
    return tuple(grads)


def work(case):
    """Sequences of a ragged batch have lengths between ``fill`` and all of ``Lk``; causal rows see the keys up to their own."""
    B, H, G, Lq, Lk, D = (case[n] for n in ("B", "H", "G", "Lq", "Lk", "D"))
    keys = Lk * (1.0 + case["fill"]) / 2
    pairs = B * H * Lq * keys
    if case.get("causal") and not case["kind"].endswith("step"):
        pairs = B * H * (min(Lq, keys) * (min(Lq, keys) + 1) / 2 + max(0.0, Lq - keys) * keys)
    rows, cols = B * Lq * H * D * 2, B * keys * (H // G) * D * 2
    if case["kind"].endswith("train"):  # q, o, dO and dq; k, v, dk and dv; seven contractions, each input of both passes once
        return {"bytes": 4 * rows + 4 * cols, "flops": 14 * pairs * D}
    return {"bytes": 2 * rows + 2 * cols, "flops": 4 * pairs * D}


def _bucket_of(d, n, distance):
    """The bucket of a distance in whole numbers: bucket single + k begins at the least d with
    (d / single) ** (n - single) >= (distance / single) ** k."""
    single = n // 2
    if d < single:
        return d
    above = n - single
    return max(single + k for k in range(above) if d ** above * single ** k >= distance ** k * single ** above)


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    B, H, G, Lq, Lk, D = (case[n] for n in ("B", "H", "G", "Lq", "Lk", "D"))
    if B * H * Lq * Lk > 1 << 32:
        return None
    f64, train = torch.float64, state["dout"] is not None
    out = torch.zeros(B, Lq, H, D, dtype=f64, device=DEVICE)
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(B, Lk, H // G, D, dtype=f64, device=DEVICE) for _ in range(2))
    lengths = [Lk] * B if state["lengths"] is None else state["lengths"].tolist()
    starts = state["start"].tolist() if torch.is_tensor(state["start"]) else [state["start"]] * B
    table = dtable = None
    if state["table"] is not None:
        table, dtable = state["table"].to(f64), torch.zeros(case["buckets"], H, dtype=f64, device=DEVICE)
        n = case["buckets"] // 2 if case["both"] else case["buckets"]
        side = [_bucket_of(d, n, case["distance"]) for d in range(case["distance"] + 1)]
        side = torch.tensor(side, device=DEVICE)
    for b in range(B):
        L = lengths[b]
        if L == 0:
            continue
        if table is not None:
            away = torch.arange(L, device=DEVICE) - starts[b] - torch.arange(Lq, device=DEVICE)[:, None]
            at = side[(away.abs() if case["both"] else -away).clamp(0, case["distance"])]
            at = at + n * (away > 0) if case["both"] else at
            order = at.flatten().sort(stable=True) if train else None
        for h in range(H):
            q, k, v = state["q"][b, :, h].to(f64), state["k"][b, :L, h // G].to(f64), state["v"][b, :L, h // G].to(f64)
            s = q @ k.t() / D ** 0.5
            if table is not None:
                s += table[:, h][at]
                if case["causal"]:
                    s[away > 0] = -math.inf
            p = torch.softmax(s, dim=-1).nan_to_num(0.0)
            out[b, :, h] = p @ v
            if train:
                do = state["dout"][b, :, h].to(f64)
                dp = do @ v.t()
                ds = p * (dp - (do * out[b, :, h]).sum(-1, keepdim=True))
                dq[b, :, h] = ds @ k / D ** 0.5
                dk[b, :L, h // G] += ds.t() @ q / D ** 0.5
                dv[b, :L, h // G] += p.t() @ do
                if table is not None:
                    ends = torch.searchsorted(order.values, torch.arange(case["buckets"] + 1, device=DEVICE))
                    sums = torch.nn.functional.pad(ds.flatten()[order.indices].cumsum(0), (1, 0))[ends]
                    dtable[:, h] += sums[1:] - sums[:-1]
    if not train:
        return out
    return (out, dq, dk, dv) if table is None else (out, dq, dk, dv, dtable)
