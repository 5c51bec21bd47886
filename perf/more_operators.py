"""Performance cases of the operators that serve a model over walks from paged caches: keys and values
written to pages (8 bits with a scale for each row, or as they are) and read back, the attention of one
new event over them, and beam search over a walk's next nodes.

``kind`` of a case:

``step``    `paged_attention_step`: one new event of each walk, appended to its pages;
``write``   `paged_write`: the rows of prompts (walks, histories) go to their pages;
``read``    `paged_read`: pages back to rows, as `walk_attention` takes them;
``select``  `beam_select`: the best continuations of each group's beams;
``reorder`` `beam_reorder`: the beams' pages follow that choice, in every layer.

Where `own` is false `run` computes the formulas with elementary torch operations; where it is true it
calls the framework.  `exact` works them out once more in float64, walk by walk.
"""
import math
import os
import sys

import torch

own = False

DEFAULTS = {
    "kind": "step",
    "dtype": "bf16",      # of the rows (kind select: of the logits)
    "eight": False,       # pages hold e4m3 and a scale for each row and head
    "page": 16,           # rows of a page
    "walks": 1,
    "min_len": 1,         # cached events of a walk; kinds write, read: rows of a walk
    "max_len": 20,
    "skew": 1.0,          # lengths min + (max - min) u^skew, u even in (0, 1)
    "heads": 8,
    "kv_heads": 8,
    "dim": 64,
    "window": 0,          # kind step: a walk sees no more than so many events back (0: all)
    "padded": False,      # kinds write, read: [walks, max_len, ...] and lengths, else rows and offsets
    "held": 0,            # kind write: up to so many rows are in the pages before
    "softcap": 0.0,
    "buckets": 0,         # of the learned bias (0: none)
    "reach": 0,
    "slopes": False,      # bias -slope |t_i - t_j|
    "times": False,       # t: event times (else positions)
    "beams": 4,           # kinds select, reorder: walks are groups of so many beams
    "nodes": 1000,        # kind select: the logits' length
    "ended": 0.0,         # kind select: share of beams that have ended
    "barred": 0.0,        # kind select: share of nodes that cannot come next (logit -inf)
    "layers": 1,          # kind reorder: caches that share one table
}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _full(case):
    c = dict(DEFAULTS)
    c.update(case)
    return c


def listed():
    return [
        # The smallest request: one event of a few short walks, in pages of the type that came in.
        {"name": "step few walks", "walks": 4, "min_len": 0, "max_len": 79, "buckets": 32,
         "reach": 32},
        # A served batch of histories of up to 4095 events, in 8 bits.
        {"name": "step batch in 8 bits", "eight": True, "page": 64, "walks": 64, "min_len": 100,
         "max_len": 4095, "heads": 32, "kv_heads": 8, "dim": 128, "softcap": 50.0},
        # A stream with a window: each walk's older events have left it; an odd head size, 16 bits.
        {"name": "step in a window", "dtype": "fp16", "page": 32, "walks": 101, "min_len": 0,
         "max_len": 2999, "heads": 12, "kv_heads": 4, "dim": 96, "window": 2048, "slopes": True,
         "times": True},
        # Few very long histories in 8 bits: the work of one walk over many compute units.
        {"name": "step long histories", "dtype": "fp16", "eight": True, "page": 256, "walks": 3,
         "min_len": 60001, "max_len": 100000, "heads": 16, "kv_heads": 2, "dim": 128,
         "slopes": True, "times": True},
        # The first events of a few walks as the sampler pads them, float32 to 8 bits.
        {"name": "write few walks", "kind": "write", "dtype": "fp32", "eight": True, "walks": 64,
         "max_len": 20, "kv_heads": 4, "dim": 32, "padded": True, "times": True},
        # Prompts of very different lengths, some over pages that hold events already.
        {"name": "write prompts", "kind": "write", "eight": True, "page": 64, "walks": 201,
         "min_len": 0, "max_len": 1999, "kv_heads": 8, "dim": 128, "held": 555},
        # A few histories for the prompts of their next events.
        {"name": "read few histories", "kind": "read", "page": 32, "walks": 13, "min_len": 0,
         "max_len": 301, "kv_heads": 4, "dim": 96},
        # Long histories from 8 bits, for a pass over all of them.
        {"name": "read long histories", "kind": "read", "eight": True, "page": 128, "walks": 23,
         "min_len": 7, "max_len": 9999, "kv_heads": 8, "dim": 128},
        # The smallest choice: four forecasts over a small graph's nodes.
        {"name": "select few beams", "kind": "select", "dtype": "fp32", "walks": 4, "beams": 4,
         "nodes": 4000},
        # A served batch of forecasts over the nodes of a larger graph, most of which no edge leads
        # to, some of them at their end.
        {"name": "select batch", "kind": "select", "walks": 64, "beams": 8, "nodes": 50021,
         "ended": 0.1, "barred": 0.5},
        # The same groups' pages: only the last page of a beam that was chosen twice moves.
        {"name": "reorder few beams", "kind": "reorder", "page": 16, "walks": 4, "beams": 4,
         "min_len": 20, "max_len": 79, "kv_heads": 2, "layers": 2},
        # A served batch, several layers in 8 bits.
        {"name": "reorder batch", "kind": "reorder", "eight": True, "page": 64, "walks": 32,
         "beams": 8, "min_len": 100, "max_len": 1023, "kv_heads": 8, "dim": 128, "layers": 4,
         "times": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "write", "read", "select", "select", "reorder"])
    c = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "select":
        c["walks"] = _log_int(rng, 1, 128)
        c["beams"] = rng.choice([1, 2, 3, 4, 5, 8, 8, 10, 16, 32])
        most = 64 * 8 * 50021 // (c["walks"] * c["beams"])
        c["nodes"] = _log_int(rng, 33, min(1000003, most))
        c["ended"] = rng.choice([0.0, rng.uniform(0.05, 0.4)])
        c["barred"] = rng.choice([0.0, rng.uniform(0.1, 0.9)])
        return c
    c["page"] = rng.choice([16, 16, 32, 64, 128, 256])
    c["kv_heads"] = rng.choice([1, 2, 3, 4, 8])
    c["eight"] = rng.random() < 0.6
    c["dim"] = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128] if c["eight"]
                          else [8, 24, 32, 40, 64, 64, 96, 104, 128])
    c["skew"] = rng.choice([0.5, 1.0, 2.0])
    row = c["kv_heads"] * c["dim"]
    if kind == "reorder":
        c["layers"] = rng.randint(1, 4)
        c["beams"] = rng.choice([2, 3, 4, 5, 8, 16, 32])
        c["times"] = rng.random() < 0.5
        c["max_len"] = _log_int(rng, 8, 1023)
        room = 32 * 8 * 1023 * 8 * 128 // (c["max_len"] * row * c["beams"])
        c["walks"] = _log_int(rng, 1, max(1, min(256, room)))
        c["min_len"] = rng.randint(1, c["max_len"])
        return c
    if kind in ("write", "read"):
        c["padded"] = rng.random() < 0.5
        c["times"] = rng.random() < 0.3
        c["max_len"] = _log_int(rng, 1, 4096)
        c["held"] = rng.choice([0, rng.randint(0, 2000)]) if kind == "write" else 0
        room = 201 * 1000 * 8 * 128 // ((c["max_len"] + c["held"]) * row)
        c["walks"] = _log_int(rng, 1, max(1, min(20000, room)))
        c["min_len"] = rng.randint(0, c["max_len"])
        return c
    c["heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 4, 6])
    c["softcap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    if rng.random() < 0.5:
        c.update(buckets=rng.randint(2, 48), reach=_log_int(rng, 4, 256))
    if rng.random() < 0.4:
        c.update(slopes=True, times=rng.random() < 0.5)
    c["max_len"] = _log_int(rng, 15, 99999)
    c["min_len"] = rng.randint(0, c["max_len"])
    c["window"] = rng.choice([0, 0, _log_int(rng, 10, 5000)])
    room = 64 * 4096 * 8 * 128 // ((c["max_len"] + 1) * row)
    c["walks"] = _log_int(rng, 1, max(1, min(512, room)))
    return c


# ---- inputs -------------------------------------------------------------------------------------
def _lengths(n, lo, hi, skew):
    """n lengths of lo..hi: the same ones for every seed (which only orders them)."""
    return [lo + int((hi - lo) * ((i + 1) / n) ** skew + 0.5) for i in range(n)]


def _held(c):
    """Rows in the pages before, by walk: 0 where there are none."""
    return _lengths(c["walks"], 0, c["held"], 1.0)[::-1]


class _State:
    pass


def _bucket_ids(buckets, reach):
    """Bucket of every distance -reach..reach: one hop each, then buckets that widen by a constant
    factor; keys after the query (a step has none) share the first."""
    exact = max(1, buckets // 2)

    def of(n):
        if n < exact:
            return min(n, buckets - 1)
        wide = math.log(max(2.0, (reach + 1) / exact))
        return min(buckets - 1, exact + int(math.log(n / exact) / wide * (buckets - exact)))

    return torch.tensor([of(max(d, 0)) for d in range(-reach, reach + 1)], dtype=torch.int32,
                        device="cuda")


def _eight_bits(x):
    """e4m3 of rows [..., dim] and the scales' exponents (biased, as bytes): the smallest power of two
    that brings a row's largest value to 448 or less.  Dividing by it is exact in float32."""
    x = x.float()
    top, e = torch.frexp(x.abs().amax(-1))  # top in [1/2, 1): 448 is 7/8 of 2^9
    e = (e - 9 + (top > 0.875)).masked_fill(top == 0, -117).clamp(-117, 120)
    codes = (x * _power(127 - e)[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _power(biased):
    """2^(biased - 127), exactly."""
    return (biased.int() << 23).view(torch.float32)


def _wide(codes, scale):
    return codes.float() * _power(scale)[..., None]


def _table(c, pages_of, gen):
    """The walks' pages in a pool, in no order: ids [walks, most], -1 where a walk has none, and the
    pool's size."""
    most, total = max(pages_of), sum(pages_of)
    n = torch.tensor(pages_of, device="cuda")
    order = torch.randperm(c["walks"], generator=gen, device="cuda")
    n = n[order]
    ids = torch.randperm(total + 3, generator=gen, device="cuda").int()
    p = torch.arange(most, device="cuda")
    at = (n.cumsum(0) - n)[:, None] + p
    return order, torch.where(p < n[:, None], ids[at.clamp(max=total + 2)], -1), total + 3


def prepare(case, seed):
    c = _full(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    s = _State()
    s.case = c

    def normal(*shape, std=1.0, of=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(of)

    n, h, hk, dim, page = c["walks"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    if c["kind"] == "select":
        # a trained model's logits: most nodes far below a few
        s.logits = normal(n, c["beams"], c["nodes"], std=3.0)
        if c["barred"]:
            bar = torch.rand(n, 1, c["nodes"], generator=gen, device="cuda") < c["barred"]
            s.logits.masked_fill_(bar, -math.inf)
        s.scores = -10.0 * torch.rand(n, c["beams"], generator=gen, device="cuda")
        s.ended = torch.rand(n, c["beams"], generator=gen, device="cuda") < c["ended"]
        torch.cuda.synchronize()
        return s

    def pool(count):
        """Keys (values) [pages, kv_heads, rows, dim], and scales; heads differ in size."""
        size = torch.exp2(torch.randint(-3, 3, (hk, 1, 1), generator=gen, device="cuda").float())
        x = torch.randn(count, hk, page, dim, generator=gen, device="cuda") * size
        return _eight_bits(x) if c["eight"] else (x.to(dtype), None)

    lens = _lengths(n, c["min_len"], c["max_len"], c["skew"])
    if c["kind"] == "reorder":
        beams = c["beams"]
        own_pages = -(-(c["max_len"] + 1) // page)
        s.table = torch.randperm(n * beams * own_pages, generator=gen, device="cuda").int()
        s.table = s.table.view(n * beams, own_pages)
        order = torch.randperm(n, generator=gen, device="cuda")
        s.lens = torch.tensor(lens, device="cuda")[order].repeat_interleave(beams)
        s.parents = torch.randint(beams, (n, beams), generator=gen, device="cuda")
        s.layers = [pool(s.table.numel()) + pool(s.table.numel()) for _ in range(c["layers"])]
        s.k_times = torch.rand(s.table.numel(), page, generator=gen, device="cuda")
        torch.cuda.synchronize()
        return s
    held = _held(c)
    room = 1 if c["kind"] == "step" else 0  # the new event
    order, s.table, pages = _table(
        c, [-(-max(1, a + b + room) // page) for a, b in zip(lens, held)], gen)
    s.lens = torch.tensor(lens, device="cuda")[order]
    s.starts = torch.tensor(held, device="cuda")[order]
    s.rows = sum(lens)
    s.offsets = torch.nn.functional.pad(torch.cumsum(s.lens, 0), (1, 0))
    s.k_times = s.times = None
    if c["times"]:
        s.k_times = 100.0 * torch.rand(pages, page, generator=gen, device="cuda")
    if c["kind"] == "write":
        rows = (n, c["max_len"]) if c["padded"] else (s.rows,)
        s.k, s.v = normal(*rows, hk, dim), normal(*rows, hk, dim)
        if c["times"]:
            s.times = torch.rand(*rows, generator=gen, device="cuda")
        kind = torch.float8_e4m3fn if c["eight"] else dtype
        empty = torch.zeros(pages, hk, page, dim, device="cuda").to(kind)
        scale = torch.zeros(pages, hk, page, dtype=torch.uint8, device="cuda")
        s.pages = [empty, scale if c["eight"] else None, empty.clone(),
                   scale.clone() if c["eight"] else None]
        torch.cuda.synchronize()
        return s
    s.pages = pool(pages) + pool(pages)
    if c["kind"] == "step":
        s.q, s.k, s.v = normal(n, h, dim), normal(n, hk, dim), normal(n, hk, dim)
        s.first = (s.lens - c["window"] + 1).clamp(min=0) if c["window"] else None
        s.bias = s.buckets = s.slopes = None
        if c["buckets"]:
            s.bias = normal(h, c["buckets"], std=0.5)
            s.buckets = _bucket_ids(c["buckets"], c["reach"])
        if c["slopes"]:
            s.slopes = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h)
        if c["times"]:
            s.times = 100.0 + torch.rand(n, generator=gen, device="cuda")
    torch.cuda.synchronize()
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _slots(s, walk, position):
    """Page and row in it of walks' positions."""
    page = s.case["page"]
    return s.table[walk, position // page].long(), position % page


def _store(s, at, k, v, times):
    """Rows [n, kv_heads, dim] to the pages at `at`."""
    for x, (codes, scale) in ((k, s.pages[:2]), (v, s.pages[2:])):
        if scale is None:
            codes[at[0], :, at[1]] = x
        else:
            x, e = _eight_bits(x)
            codes.view(torch.uint8)[at[0], :, at[1]] = x.view(torch.uint8)
            scale[at[0], :, at[1]] = e
    if s.k_times is not None:
        s.k_times[at] = times


def _load(s, at):
    """Keys and values at `at`, float32 [..., kv_heads, dim]."""
    got = []
    for codes, scale in (s.pages[:2], s.pages[2:]):
        if scale is None:
            got.append(codes[at[0], :, at[1]].float())
        else:
            x = codes.view(torch.uint8)[at[0], :, at[1]].view(torch.float8_e4m3fn)
            got.append(_wide(x, scale[at[0], :, at[1]]))
    return got


def _of_rows(s):
    """Walk and number in it of every row: of the packed rows, or of the padded ones that count."""
    c = s.case
    if c["padded"]:
        return torch.nonzero(torch.arange(c["max_len"], device="cuda") < s.lens[:, None],
                             as_tuple=True)
    walk = torch.repeat_interleave(torch.arange(c["walks"], device="cuda"), s.lens,
                                   output_size=s.rows)
    return walk, torch.arange(s.rows, device="cuda") - s.offsets[walk]


def _plain_write(s):
    walk, i = _of_rows(s)
    k, v, times = s.k, s.v, s.times
    if s.case["padded"]:
        k, v = k[walk, i], v[walk, i]
        times = None if times is None else times[walk, i]
    _store(s, _slots(s, walk, s.starts[walk] + i), k, v, times)


def _plain_read(s):
    c = s.case
    walk, i = _of_rows(s)
    at = _slots(s, walk, i)
    got = _load(s, at) + ([] if s.k_times is None else [s.k_times[at]])
    if c["padded"]:
        rows = [x.new_zeros(c["walks"], c["max_len"], *x.shape[1:]) for x in got]
        for r, x in zip(rows, got):
            r[walk, i] = x
        got = rows
    return [x.to(TYPES[c["dtype"]]) for x in got[:2]] + got[2:]


def _plain_step(s):
    c = s.case
    n, h, hk = c["walks"], c["heads"], c["kv_heads"]
    walk = torch.arange(n, device="cuda")
    _store(s, _slots(s, walk, s.lens), s.k, s.v, s.times)
    j = torch.arange(s.table.shape[1] * c["page"], device="cuda")
    back = s.lens[:, None] - j
    seen = back >= 0
    if s.first is not None:
        seen = seen & (j >= s.first[:, None])
    at = _slots(s, walk[:, None], j.expand(n, -1))
    at = at[0].clamp(min=0), at[1]
    k, v = (x.masked_fill(~seen[..., None, None], 0).transpose(1, 2) for x in _load(s, at))
    q = s.q.float().view(n, hk, h // hk, -1)
    x = (q @ k.transpose(-1, -2).contiguous() * c["dim"] ** -0.5).view(n, h, -1)
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    if s.bias is not None:
        by_distance = s.bias.float()[:, s.buckets.long()]
        x = x + by_distance[:, back.clamp(-c["reach"], c["reach"]) + c["reach"]].transpose(0, 1)
    if s.slopes is not None:
        gap = s.times[:, None] - s.k_times[at] if c["times"] else back.float()
        x = x - s.slopes[:, None] * gap.abs()[:, None]
    x = x.masked_fill(~seen[:, None], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = (e.view(n, hk, h // hk, -1) @ v.contiguous()).view(n, h, -1)
    return (o / e.sum(-1, keepdim=True)).to(s.q.dtype)


def _plain_select(s):
    """In float64: candidates of different beams may be near to each other."""
    n, beams, nodes = s.logits.shape
    x = s.logits.double()
    top = x.amax(-1, keepdim=True)
    total = torch.log(torch.exp(x - top.clamp(min=-1e300)).sum(-1, keepdim=True)) + top
    at = s.scores.double()[..., None] + (x - total)
    at = at.masked_fill(~torch.isfinite(total) | ~torch.isfinite(s.scores)[..., None], -math.inf)
    first = torch.arange(nodes, device="cuda") == 0  # node 0 ends a walk
    kept = torch.where(first, s.scores.double()[..., None], -math.inf)
    at = torch.where(s.ended[..., None], kept, at).flatten(1)
    best, which = torch.sort(at, dim=-1, descending=True, stable=True)
    best, which = best[:, :beams], which[:, :beams]
    none = best == -math.inf
    parents = (which // nodes).masked_fill(none, 0)
    tokens = (which % nodes).masked_fill(none, 0)
    ended = s.ended.gather(1, parents) | (tokens == 0) | none
    return {"scores": best.float(), "tokens": tokens, "parents": parents, "ended": ended}


def _plain_reorder(s):
    """A beam's first child takes over its last page, every further one that of a beam without
    children, with a copy of its rows."""
    c = s.case
    n, beams, page = c["walks"], c["beams"], c["page"]
    b = torch.arange(beams, device="cuda")
    same = s.parents[:, :, None] == s.parents[:, None, :]
    further = (same & (b < b[:, None])).any(-1)
    childless = ~(s.parents[:, :, None] == b).any(1)
    spare = torch.sort(~childless, dim=-1, stable=True)[1]
    place = (further.long().cumsum(-1) - 1).clamp(min=0)
    taken = torch.where(further, spare.gather(1, place), s.parents)
    base = torch.arange(n, device="cuda")[:, None] * beams
    parent, taken = (s.parents + base).flatten(), (taken + base).flatten()
    lens = s.lens[parent]
    full = (lens // page)[:, None]
    p = torch.arange(s.table.shape[1], device="cuda")
    table = torch.where(p < full, s.table[parent], s.table[taken])
    moved = torch.nonzero(further.flatten() & (lens % page > 0))[:, 0]
    source = s.table[parent[moved], full[moved, 0]].long()
    target = s.table[taken[moved], full[moved, 0]].long()
    mine = torch.arange(page, device="cuda") < (lens[moved] % page)[:, None]
    for layer in s.layers:
        for x in layer:
            if x is not None:
                x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
                which = mine[:, None, :, None] if x.dim() == 4 else mine[:, None]
                x[target] = torch.where(which, x[source], x[target])
    if c["times"]:
        s.k_times[target] = torch.where(mine, s.k_times[source], s.k_times[target])
    return {"table": table, "lens": lens}


# ---- the framework's calls ----------------------------------------------------------------------
def _operators():
    package = os.path.join(os.getcwd(), "temporal-random-walk_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from temporal_random_walk import operators
    return operators


def _pages(ops, x):
    k, k_scale, v, v_scale = x
    return ops.Pages(k, v, k_scale, v_scale)


def _own_write(s):
    ops = _operators()
    more = {"counts": s.lens} if s.case["padded"] else {"offsets": s.offsets}
    ops.paged_write(_pages(ops, s.pages), s.table, s.starts, s.k, s.v, times=s.times,
                    k_times=s.k_times, **more)


def _own_read(s):
    ops, c = _operators(), s.case
    if c["padded"]:
        more = {"lens": s.lens, "length": c["max_len"]}
    else:
        more = {"offsets": s.offsets, "rows": s.rows}
    return ops.paged_read(_pages(ops, s.pages), s.table, dtype=TYPES[c["dtype"]],
                          k_times=s.k_times, **more)


def _own_step(s):
    ops = _operators()
    return ops.paged_attention_step(
        s.q, s.k, s.v, _pages(ops, s.pages), s.table, s.lens, first=s.first,
        softcap=s.case["softcap"], bias_table=s.bias, buckets=s.buckets, slopes=s.slopes,
        times=s.times, k_times=s.k_times)


def _own_select(s):
    got = _operators().beam_select(s.logits, s.scores, s.case["beams"], ended=s.ended, end_token=0)
    return {"scores": got.scores, "tokens": got.tokens, "parents": got.parents,
            "ended": got.ended}


def _own_reorder(s):
    ops = _operators()
    table, lens = ops.beam_reorder(s.table, s.lens, s.parents, [_pages(ops, x) for x in s.layers],
                                   k_times=s.k_times if s.case["times"] else None)
    return {"table": table, "lens": lens}


def _held_in_pages(s):
    names = ("k", "k_scale", "v", "v_scale")
    got = {name: x for name, x in zip(names, s.pages) if x is not None}
    if s.k_times is not None:
        got["k_times"] = s.k_times
    return got


def run(state):
    s = state
    kind = s.case["kind"]
    if kind == "select":
        return _own_select(s) if own else _plain_select(s)
    if kind == "reorder":
        got = _own_reorder(s) if own else _plain_reorder(s)
        return {**got, "layers": s.layers, "k_times": s.k_times}
    if kind == "read":
        return list(_own_read(s) if own else _plain_read(s))
    if kind == "write":
        if own:
            _own_write(s)
        else:
            _plain_write(s)
        return _held_in_pages(s)
    out = _own_step(s) if own else _plain_step(s)
    return {"out": out, **_held_in_pages(s)}


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    c = _full(case)
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "select":
        n = c["walks"] * c["beams"] * c["nodes"]
        return {"bytes": n * size, "flops": 4 * n}  # subtract, exp, add, compare
    lens = _lengths(c["walks"], c["min_len"], c["max_len"], c["skew"])
    row = c["kv_heads"] * c["dim"]
    in_page = row + c["kv_heads"] if c["eight"] else row * size  # of a key row or a value row
    if c["kind"] == "reorder":
        # of b beams that choose among themselves, (1 - 1/b)^b of them have no child
        b = c["beams"]
        rows = sum(n % c["page"] for n in lens) * b * (1 - 1 / b) ** b
        table = c["walks"] * b * -(-(c["max_len"] + 1) // c["page"]) * 8
        return {"bytes": 2 * rows * (2 * in_page * c["layers"] + 4 * c["times"]) + table,
                "flops": 0}
    if c["kind"] in ("write", "read"):
        rows = sum(lens)
        return {"bytes": rows * (2 * (row * size + in_page) + 8 * c["times"]),
                "flops": rows * row * 4 * c["eight"]}
    n = c["walks"]
    events = sum(min(x, c["window"] - 1) if c["window"] else x for x in lens)
    nbytes = events * (2 * in_page + 4 * c["times"]) + n * 2 * in_page
    nbytes += n * size * (2 * c["heads"] * c["dim"] + 2 * row)
    return {"bytes": nbytes, "flops": 4 * c["dim"] * c["heads"] * (events + n)}


# ---- the same in 64 bits ------------------------------------------------------------------------
def _exact_codes(x):
    """The nearest e4m3 values of float64 rows over their scales, ties to even, and the scales."""
    top = x.abs().amax(-1)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -109) / 448)).clamp(-117, 120)
    scale = torch.exp2(e)[..., None]
    y = x / scale
    place = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / place) * place, scale


def _exact_cells(s, w, count, start=0):
    """Pages and rows of a walk's positions start .. start + count - 1."""
    page = s.case["page"]
    at = [start + i for i in range(count)]
    ids = s.table[w].tolist()
    return (torch.tensor([ids[p // page] for p in at], dtype=torch.long, device="cuda"),
            torch.tensor([p % page for p in at], dtype=torch.long, device="cuda"))


def _exact_values(codes, scale, cells):
    x = codes.double()[cells[0], :, cells[1]]
    if scale is not None:
        x = x * torch.exp2(scale[cells[0], :, cells[1]].double() - 127)[..., None]
    return x


def _exact_pages(s, cells, k, v, times):
    """The pages' contents as float64 after rows of theirs are written."""
    res = {}
    for name, x, codes, scale in (("k", k, *s.pages[:2]), ("v", v, *s.pages[2:])):
        held = codes.double()
        if scale is None:
            held[cells[0], :, cells[1]] = x.double()
        else:
            values, factor = _exact_codes(x.double())
            held[cells[0], :, cells[1]] = values
            scale[cells[0], :, cells[1]] = (torch.log2(factor[..., 0]) + 127).to(torch.uint8)
            res[name + "_scale"] = scale
        res[name] = held
    if s.k_times is not None:
        s.k_times[cells] = times
        res["k_times"] = s.k_times
    return res


def _exact_write(s):
    c = s.case
    cells, picked = [], []
    for w, (n, start) in enumerate(zip(s.lens.tolist(), s.starts.tolist())):
        cells.append(_exact_cells(s, w, n, start))
        first = w * c["max_len"] if c["padded"] else int(s.offsets[w])
        picked.append(torch.arange(first, first + n, device="cuda"))
    cells, picked = tuple(torch.cat(x) for x in zip(*cells)), torch.cat(picked)
    flat = [x.flatten(0, 1) if c["padded"] else x for x in (s.k, s.v)]
    times = None if s.times is None else s.times.flatten()[picked]
    return _exact_pages(s, cells, flat[0][picked], flat[1][picked], times)


def _exact_read(s):
    c = s.case
    shape = (c["walks"], c["max_len"]) if c["padded"] else (s.rows,)
    tail = (c["kv_heads"], c["dim"])
    res = [torch.zeros(math.prod(shape), *t, dtype=torch.float64, device="cuda")
           for t in (tail, tail, ())]
    for w, n in enumerate(s.lens.tolist()):
        cells = _exact_cells(s, w, n)
        first = w * c["max_len"] if c["padded"] else int(s.offsets[w])
        res[0][first:first + n] = _exact_values(*s.pages[:2], cells)
        res[1][first:first + n] = _exact_values(*s.pages[2:], cells)
        if c["times"]:
            res[2][first:first + n] = s.k_times[cells].double()
    return [x.view(*shape, *x.shape[1:]) for x in res[:2 + c["times"]]]


def _exact_step(s):
    c = s.case
    group = c["heads"] // c["kv_heads"]
    lens = s.lens.tolist()
    new = [_exact_cells(s, w, 1, n) for w, n in enumerate(lens)]
    res = _exact_pages(s, tuple(torch.cat(x) for x in zip(*new)), s.k, s.v, s.times)
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    for w, n in enumerate(lens):
        first = max(0, n - c["window"] + 1) if c["window"] else 0
        cells = _exact_cells(s, w, n + 1 - first, first)
        k, v = (res[x][cells[0], :, cells[1]] for x in "kv")
        if c["eight"]:
            k, v = (y * torch.exp2(res[x][cells[0], :, cells[1]].double() - 127)[..., None]
                    for x, y in (("k_scale", k), ("v_scale", v)))
        k, v = (x.repeat_interleave(group, 1) for x in (k, v))
        x = (k * s.q[w].double()).sum(-1) / math.sqrt(c["dim"])  # [events, heads]
        if c["softcap"]:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        back = torch.arange(n - first, -1, -1, device="cuda")
        if s.bias is not None:
            x = x + s.bias.double()[:, s.buckets.long()[c["reach"] + back.clamp(max=c["reach"])]].T
        if s.slopes is not None:
            gap = s.times[w].double() - s.k_times[cells].double() if c["times"] else back.double()
            x = x - s.slopes.double() * gap.abs()[:, None]
        out[w] = (torch.softmax(x, 0)[..., None] * v).sum(0)
    return {"out": out, **res}


def _exact_select(s):
    c = s.case
    beams, nodes = c["beams"], c["nodes"]
    res = {"scores": torch.full((c["walks"], beams), -math.inf, dtype=torch.float64, device="cuda"),
           "tokens": torch.zeros(c["walks"], beams, dtype=torch.long, device="cuda"),
           "parents": torch.zeros(c["walks"], beams, dtype=torch.long, device="cuda"),
           "ended": torch.ones(c["walks"], beams, dtype=torch.bool, device="cuda")}
    for g in range(c["walks"]):
        share = torch.log_softmax(s.logits[g].double(), -1).nan_to_num(nan=-math.inf, neginf=-math.inf)
        gone = s.ended[g]
        share[gone] = -math.inf
        share[gone, 0] = 0.0
        at = (share + s.scores[g].double()[:, None]).flatten()
        for place in range(beams):
            best = at.max()
            if best == -math.inf:
                break
            which = int(torch.nonzero(at == best)[0])
            at[which] = -math.inf
            parent, token = divmod(which, nodes)
            res["scores"][g, place], res["tokens"][g, place] = best, token
            res["parents"][g, place] = parent
            res["ended"][g, place] = bool(gone[parent]) or token == 0
    return res


def _exact_reorder(s):
    c = s.case
    beams, page = c["beams"], c["page"]
    table, lens, parents = s.table.tolist(), s.lens.tolist(), s.parents.tolist()
    new, new_lens, moves = [], [], []
    for g in range(c["walks"]):
        spare = [b for b in range(beams) if b not in parents[g]]
        seen = set()
        for p in parents[g]:
            row, n = table[g * beams + p], lens[g * beams + p]
            last = row
            if p in seen:
                last = table[g * beams + spare.pop(0)]
                if n % page:
                    moves.append((row[n // page], last[n // page], n % page))
            seen.add(p)
            new.append(row[:n // page] + last[n // page:])
            new_lens.append(n)
    # no page is both read and written: the order of the moves does not matter
    source, target, count = (torch.tensor(x, dtype=torch.long, device="cuda").view(-1)
                             for x in (zip(*moves) if moves else ((), (), ())))
    move, row = torch.nonzero(torch.arange(page, device="cuda") < count[:, None], as_tuple=True)
    layers = []
    for layer in s.layers:
        layers.append([])
        for x in layer:
            if x is not None:
                whole = x.dtype == torch.uint8
                x = x.long() if whole else x.double()
                x[target[move], :, row] = x[source[move], :, row]
            layers[-1].append(x)
    if c["times"]:
        s.k_times[target[move], row] = s.k_times[source[move], row]
    return {"table": torch.tensor(new, device="cuda").int(),
            "lens": torch.tensor(new_lens, device="cuda"), "layers": layers, "k_times": s.k_times}


def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_step, "write": _exact_write, "read": _exact_read,
            "select": _exact_select, "reorder": _exact_reorder}[s.case["kind"]](s)
