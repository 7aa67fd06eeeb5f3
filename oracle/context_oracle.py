"""Cross attention and attention with a relative position bias in float64 (torch on the CPU), for the tests: the definition, its
gradients by autograd, and for each result the magnitudes that rounding errors are bounded by."""
from __future__ import annotations

import math

import torch


def bucket_of(distance: int, buckets: int, max_distance: int) -> int:
    """The bucket of a distance in one direction, by its definition in whole numbers: single distances below buckets // 2, then the
    last k with (distance / single) ** (buckets - single) >= (max_distance / single) ** k."""
    single = buckets // 2
    if distance < single:
        return distance
    n = buckets - single
    return max(single + k for k in range(n) if distance ** n * single ** k >= max_distance ** k * single ** n)


def bucket_map(Lq, Lk, start, buckets, max_distance, bidirectional):
    """[Lq, Lk] bucket of each pair for one sequence."""
    n = buckets // 2 if bidirectional else buckets
    far = [bucket_of(d, n, max_distance) for d in range(max_distance + 1)]
    out = torch.empty(Lq, Lk, dtype=torch.long)
    for i in range(Lq):
        for j in range(Lk):
            rel = j - (start + i)
            d = abs(rel) if bidirectional else max(-rel, 0)
            out[i, j] = far[min(d, max_distance)] + (n if bidirectional and rel > 0 else 0)
    return out


def attention(q, k, v, dO=None, table=None, max_distance=128, bidirectional=True, causal=False, key_lengths=None,
              query_lengths=None, start=0, scale=None, scores_in=None):
    """``[B,S,H,D]`` tensors.  ``scores_in``: a type that the scores with their bias are rounded to (their gradient passes as it is), which
    a bias of 1e8 or more hides the scores in.  Returns ``(values, sizes)``, dicts of o, lse and, with dO, dq, dk, dv, dtable.  ``sizes[name]`` holds
    (a, b, c): a is the magnitude that a relative rounding of the 16-bit operands of the last contraction meets (sum of
    |p||v| and the like), b what a relative error of delta = dO.o meets, c what an absolute error of those operands meets."""
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1:3]
    G = H // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    tab = None if table is None else table.detach().double().requires_grad_()
    z = lambda *s: torch.zeros(s, dtype=torch.float64)
    o, lse = z(B, Lq, H, D), torch.full((B, H, Lq), -math.inf, dtype=torch.float64)
    size = {n: [z(*s) for _ in range(3)] for n, s in (("o", o.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    if tab is not None:
        size["dtable"] = [z(*tab.shape) for _ in range(3)]
    for b in range(B):
        nq = Lq if query_lengths is None else min(max(int(query_lengths[b]), 0), Lq)
        nk = Lk if key_lengths is None else min(max(int(key_lengths[b]), 0), Lk)
        if nq == 0 or nk == 0:
            continue
        s0 = int(start[b]) if torch.is_tensor(start) else start
        rel = torch.arange(nk) - s0 - torch.arange(nq)[:, None]
        seen = rel <= 0 if causal else torch.ones(nq, nk, dtype=torch.bool)
        at = None if tab is None else bucket_map(nq, nk, s0, table.shape[0], max_distance, bidirectional)
        for h in range(H):
            Q, K, V = leaves[0][b, :nq, h], leaves[1][b, :nk, h // G], leaves[2][b, :nk, h // G]
            s = Q @ K.T * scale
            if tab is not None:
                s = s + tab[:, h][at]
            if scores_in is not None:
                s = s + (s.detach().to(scores_in).double() - s.detach()).nan_to_num(0.0)  # (-inf stays)
            hidden = ~seen | (s == -math.inf)
            some = (~hidden).any(1)
            s = s.masked_fill(hidden, -math.inf)[some]
            p = torch.softmax(s, -1)
            rows = torch.arange(nq)[some]
            out = p @ V
            o = o.index_put((torch.tensor(b), rows, torch.tensor(h)), out)
            lse[b, h, rows] = torch.logsumexp(s.detach(), -1)
            with torch.no_grad():
                size["o"][0][b, rows, h] = p @ V.abs()
                size["o"][2][b, rows, h] = V.abs().sum(0).expand(len(rows), D)
                if dO is None:
                    continue
                g = dO[b, rows, h].double()
                dp, delta = g @ V.T, (g * out).sum(-1, keepdim=True)
                ds, dd = p * (dp - delta), p * (g.abs() * out.abs()).sum(-1, keepdim=True)
                size["dq"][0][b, rows, h] = ds.abs() @ K.abs() * scale
                size["dq"][1][b, rows, h] = (dd @ K).abs() * scale + (p * (g.abs() @ V.abs().T)) @ K.abs() * scale * 2.0 ** -6
                size["dq"][2][b, rows, h] = K.abs().sum(0).expand(len(rows), D) * scale
                size["dk"][0][b, :nk, h // G] += ds.abs().T @ Q[rows].abs() * scale
                size["dk"][1][b, :nk, h // G] += dd.T @ Q[rows].abs() * scale + (p * (g.abs() @ V.abs().T)).T @ Q[rows].abs() * scale * 2.0 ** -6
                size["dk"][2][b, :nk, h // G] += Q[rows].abs().sum(0) * scale
                size["dv"][0][b, :nk, h // G] += p.T @ g.abs()
                size["dv"][2][b, :nk, h // G] += g.abs().sum(0)
                if tab is not None:
                    size["dtable"][0][:, h].index_add_(0, at[rows].flatten(), (p * (g.abs() @ V.abs().T) + dd).flatten())
    values = {"o": o.detach(), "lse": lse}
    if dO is not None:
        ins = leaves + ([] if tab is None else [tab])
        grads = torch.autograd.grad(o, ins, dO.double(), allow_unused=True) if o.requires_grad else [None] * len(ins)
        for name, t, g in zip(("dq", "dk", "dv", "dtable"), ins, grads):
            values[name] = torch.zeros_like(t) if g is None else g
    return values, size
