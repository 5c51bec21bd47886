"""The operators' formulas in float64 on the CPU, one document at a time, with bounds on what a
computation in a narrower type may be off by.

A bound is worked out element by element from the same intermediate values: `u` is the unit
roundoff of the inputs' type (each rounding of P, dS, o and a result to it is off by at most u times
the value), and `eta` bounds the relative error of P in float32: a score is a sum of dim products and
a few terms, each rounded (2^-24 of the sum of their absolute values each), the exponential and
tanh functions are good to a few units in the last place, and a softmax over n keys adds n roundings.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32 = 2.0 ** -24
# Below this a value of the type has fewer bits (float16's subnormals; the others' are out of reach).
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}


def documents(mask_kind, q_lens, k_lens, prefix=None):
    """[(position of the first query, lq, lk, keys a query may see as a bool matrix)]."""
    out = []
    for w, (a, b) in enumerate(zip(q_lens, k_lens)):
        pos = torch.arange(a)[:, None] + (b - a)
        key = torch.arange(b)[None]
        seen = torch.ones(a, b, dtype=torch.bool)
        if mask_kind != "full":
            seen = key <= pos
            if mask_kind == "prefix":
                seen = seen | (key < prefix[w]).expand(a, b)
        out.append((b - a, a, b, seen))
    return out


def score_terms(x, dim, scale, softcap, table, buckets, slopes, hop, gap):
    """(scores, d score / d x, sum of absolute terms) of scaled products x [h, a, b]."""
    s, slope, size = x, torch.ones_like(x), x.abs()
    if softcap:
        t = torch.tanh(x / softcap)
        s, slope = softcap * t, 1 - t * t
        size = size + softcap
    if table is not None:
        reach = buckets.shape[0] // 2
        bias = table[:, buckets.long()[hop.clamp(-reach, reach) + reach]]
        s = s + bias
        size = size + bias.clamp_min(-1e4).abs()
    if slopes is not None:
        s = s - slopes[:, None, None] * gap.abs()
        size = size + (slopes[:, None, None] * gap).abs()
    return s, slope, size


def attention(q, k, v, docs, *, scale=None, softcap=0.0, table=None, buckets=None, slopes=None,
              q_times=None, k_times=None, d_out=None, dtype=torch.float32, starts=None):
    """q [rows, heads, dim], k, v [rows, kv_heads, dim] in float64 (already rounded to `dtype`);
    `starts`: first query and key row of each document (packed one after another by default).
    Returns {name: (value, bound)}."""
    rows, heads, dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    u, tiny = U[dtype], TINY[dtype]
    z = lambda x: torch.zeros(x.shape, dtype=torch.float64)  # noqa: E731
    out, out_b = z(q), z(q)
    grads = {n: (z(x), z(x)) for n, x in (("d_q", q), ("d_k", k), ("d_v", v))}
    d_table = None if table is None else (z(table), z(table))
    if starts is None:
        starts, a0, b0 = [], 0, 0
        for _, a, b, _ in docs:
            starts.append((a0, b0))
            a0, b0 = a0 + a, b0 + b
    of = torch.arange(heads) // group
    for (first, a, b, seen), (a0, b0) in zip(docs, starts):
        if a == 0:
            continue
        qs = q[a0:a0 + a].transpose(0, 1)
        ks = k[b0:b0 + b].transpose(0, 1)[of]
        vs = v[b0:b0 + b].transpose(0, 1)[of]
        hop = first + torch.arange(a)[:, None] - torch.arange(b)[None]
        gap = hop.double()
        if q_times is not None:
            gap = q_times[a0:a0 + a, None] - k_times[None, b0:b0 + b]
        x = qs @ ks.mT * scale
        s, slope, size = score_terms(x, dim, scale, softcap, table, buckets, slopes, hop, gap)
        size = size + (qs.abs() @ ks.abs().mT) * abs(scale)
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True).clamp_min(-1e300) if b else s.new_zeros(heads, a, 1)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        p = e / total.clamp_min(1e-300) if b else e
        o = p @ vs
        worst = (size.masked_fill(~seen, 0).amax(-1, keepdim=True) if b
                 else s.new_zeros(heads, a, 1))
        eta = F32 * ((dim + 24) * (1 + worst) * 2 + b)
        weight = p @ vs.abs()
        o_b = u * o.abs() + (u + eta) * weight * 1.01 + tiny * (1 + (seen[None] * vs.abs().amax(-1)[:, None]).sum(-1, keepdim=True))
        out[a0:a0 + a] = o.transpose(0, 1)
        out_b[a0:a0 + a] = o_b.transpose(0, 1)
        if d_out is None:
            continue
        do = d_out[a0:a0 + a].transpose(0, 1)
        dp = do @ vs.mT
        delta = (do * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        dx = ds * slope * scale
        # dS: P's relative error, dP's and D's own
        dp_b = F32 * dim * (do.abs() @ vs.abs().mT)
        delta_b = (do.abs() * o_b).sum(-1, keepdim=True) + F32 * dim * (do.abs() * o.abs()).sum(-1, keepdim=True)
        ds_b = eta * ds.abs() + p * (dp_b + delta_b) * 1.01
        slope_b = 0.0 if not softcap else 8 * F32
        dx_b = ((ds_b * slope + ds.abs() * slope_b) + u * (ds * slope).abs() + tiny) * abs(scale)
        dx_b = dx_b.masked_fill(~seen, 0)
        n_f32 = F32 * 2  # of the sums, times their length
        dq = dx @ ks
        dq_b = (dx_b + n_f32 * b * dx.abs()) @ ks.abs() + u * dq.abs() + tiny
        dk = (dx.mT @ qs).unflatten(0, (kv_heads, group)).sum(1)
        dk_b = ((dx_b + n_f32 * a * group * dx.abs()).mT @ qs.abs()).unflatten(0, (kv_heads, group)).sum(1)
        dv = (p.mT @ do).unflatten(0, (kv_heads, group)).sum(1)
        dv_b = (((u + eta + n_f32 * a * group) * p + tiny * seen).mT @ do.abs()).unflatten(
            0, (kv_heads, group)).sum(1)
        for n, val, bound, at, m in (("d_q", dq, dq_b, a0, a), ("d_k", dk, dk_b + u * dk.abs() + tiny, b0, b),
                                     ("d_v", dv, dv_b + u * dv.abs() + tiny, b0, b)):
            grads[n][0][at:at + m] = val.transpose(0, 1)
            grads[n][1][at:at + m] = bound.transpose(0, 1)
        if table is not None:
            reach = buckets.shape[0] // 2
            bucket = buckets.long()[hop.clamp(-reach, reach) + reach]
            for t in range(table.shape[1]):
                at = (bucket == t) & seen
                d_table[0][:, t] += (ds * at).sum((1, 2))
                d_table[1][:, t] += ((ds_b + F32 * 64 * ds.abs()) * at).sum((1, 2))
    res = {"out": (out, out_b)}
    if d_out is not None:
        res.update(grads)
        if table is not None:
            res["d_table"] = (d_table[0], d_table[1] + F32 * d_table[0].abs())
    return res


def check(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), f"{name}: not finite"
    off = (got - want).abs() - bound
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, (f"{name}: off by {(got - want).abs().flatten()[off.argmax()].item():.3g}, "
                        f"bound {bound.flatten()[off.argmax()].item():.3g}")
