"""Performance cases of the operators that consume walks: attention inside each walk (training and
prompts), its single-event form over a cache, and the learned bias by distance buckets.

``kind`` of a case:

``train``   `walk_attention` forward and backward: the output, the gradients of q, k, v and, with
            buckets, of the bias table;
``prompt``  `walk_attention` forward: each document's queries are its last rows, over keys that
            hold ``cached`` rows more;
``step``    `walk_attention_step`: one new event of each walk, appended to its cache;
``bias``    `relative_bias` and its gradient.

Where `own` is false `run` computes the formulas with elementary torch operations in float32;
where it is true it calls the framework.  `exact` works them out once more in float64, documents
of equal length at a time, with the gradients written out.
"""
import math
import os
import sys

import torch

own = False

DEFAULTS = {
    "kind": "train",
    "dtype": "bf16",
    "layout": "padded",   # padded: [docs, max_len, ...] and lens; packed: rows and offsets
    "docs": 1,            # walks (documents); kind step: walks in the batch
    "min_len": 1,         # query rows of a document; kind step: cached events of a walk
    "max_len": 20,
    "skew": 1.0,          # lengths min + (max - min) u^skew, u even in (0, 1)
    "cached": 0,          # kind prompt: up to so many key rows before a document's queries
    "capacity": 0,        # kind step: slots of a cache
    "heads": 8,
    "kv_heads": 8,
    "dim": 64,
    "fused": False,       # q, k and v are slices of one projection's output
    "mask": "causal",     # causal, full, prefix
    "softcap": 0.0,
    "buckets": 0,         # of the learned bias (0: none)
    "reach": 0,           # distances past it share the outermost buckets
    "slopes": False,      # bias -slope |t_i - t_j|
    "times": False,       # t: event times (else positions)
    "q_len": 0,           # kind bias
    "k_len": 0,
    "q_offset": 0,
}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _full(case):
    c = dict(DEFAULTS)
    c.update(case)
    return c


def listed():
    return [
        # The smallest training step of the tests' size: a few walks of a small graph, where the
        # launches are the time.
        {"name": "train few walks", "dtype": "fp32", "docs": 64, "max_len": 20, "heads": 4,
         "kv_heads": 4, "dim": 32, "buckets": 16, "reach": 16},
        # A training batch of walks of 80 as the sampler leaves them (padded, many ending early),
        # older events fading with the time that has passed.
        {"name": "train walks of 80", "docs": 20000, "max_len": 80, "skew": 0.6, "slopes": True,
         "times": True},
        # Walks of 40 packed without padding, q, k and v from one projection, shared key heads,
        # a learned bias by hops.
        {"name": "train packed walks", "layout": "packed", "docs": 8001, "max_len": 40,
         "kv_heads": 2, "fused": True, "buckets": 32, "reach": 32},
        # Histories of very different lengths in one packed batch, each with a prefix that sees
        # itself whole; capped scores, an odd head size.
        {"name": "train ragged prefix", "dtype": "fp16", "layout": "packed", "docs": 23,
         "max_len": 1999, "skew": 1.5, "dim": 80, "mask": "prefix", "softcap": 30.0,
         "buckets": 32, "reach": 128},
        # One long event stream, forward and backward: the largest training case.
        {"name": "train one long stream", "layout": "packed", "min_len": 8192, "max_len": 8192,
         "heads": 16, "kv_heads": 4, "dim": 128, "fused": True, "softcap": 50.0},
        # The longest prompt, a bias that falls with distance: the largest case.
        {"name": "prompt one long stream", "kind": "prompt", "layout": "packed",
         "min_len": 16384, "max_len": 16384, "heads": 16, "kv_heads": 4, "dim": 128,
         "slopes": True},
        # New events of several histories at once, each over what its cache already holds.
        {"name": "prompt over caches", "kind": "prompt", "layout": "packed", "docs": 13,
         "max_len": 301, "cached": 3001, "heads": 12, "kv_heads": 4, "dim": 96, "buckets": 32,
         "reach": 128},
        # The smallest request: one event of a few short walks.
        {"name": "step few walks", "kind": "step", "docs": 4, "min_len": 0, "max_len": 79,
         "capacity": 80, "buckets": 32, "reach": 32},
        # A served batch of histories of up to 4095 events.
        {"name": "step batch", "kind": "step", "docs": 64, "min_len": 100, "max_len": 4095,
         "capacity": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "softcap": 50.0},
        # Few very long histories: the work of one walk over many compute units.
        {"name": "step long histories", "kind": "step", "dtype": "fp16", "docs": 3,
         "min_len": 60001, "max_len": 100000, "capacity": 100001, "heads": 16, "kv_heads": 2,
         "dim": 128, "slopes": True, "times": True},
        # The bias of walks of 80, as a model with an attention of its own adds it.
        {"name": "bias walks of 80", "kind": "bias", "dtype": "fp32", "buckets": 32, "reach": 79,
         "q_len": 80, "k_len": 80},
        # The bias of long rows against a longer cache: all bandwidth.
        {"name": "bias long rows", "kind": "bias", "heads": 16, "buckets": 64, "reach": 512,
         "q_len": 4096, "k_len": 4199, "q_offset": 103},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


# Scores of the padded batch (what a plain form holds) that a drawn case may have, by kind: not
# more than the largest listed case of the kind.
MOST_SCORES = {"train": 16 * 8192 * 8192, "prompt": 16 * 16384 * 16384}


def draw(rng):
    kind = rng.choice(["train", "train", "train", "prompt", "step", "step", "bias"])
    c = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "bias":
        c.update(heads=rng.randint(1, 16), q_len=_log_int(rng, 1, 4096),
                 k_len=_log_int(rng, 8, 4199), buckets=rng.randint(2, 64),
                 reach=_log_int(rng, 1, 512))
        c["q_offset"] = rng.choice([0, rng.randint(0, c["k_len"]), rng.randint(0, 100)])
        return c
    c["kv_heads"] = rng.choice([1, 2, 3, 4, 8])
    c["heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 4])
    c["dim"] = rng.choice([16, 24, 32, 40, 64, 64, 64, 80, 96, 128, 128])
    c["softcap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    if rng.random() < 0.5:
        c.update(buckets=rng.randint(2, 48), reach=_log_int(rng, 4, 256))
    if rng.random() < 0.4:
        c.update(slopes=True, times=rng.random() < 0.5)
    if kind == "step":
        c["capacity"] = _log_int(rng, 16, 100000)
        c["max_len"] = c["capacity"] - 1
        c["min_len"] = rng.randint(0, c["max_len"])
        room = 64 * 4096 * 8 * 128 // (c["capacity"] * c["kv_heads"] * c["dim"])
        c["docs"] = _log_int(rng, 1, max(1, min(512, room)))
        return c
    c["mask"] = rng.choice(["causal", "causal", "full", "prefix"])
    c["layout"] = rng.choice(["padded", "packed"])
    c["skew"] = rng.choice([0.5, 1.0, 2.0])
    if kind == "prompt":
        c["layout"] = "packed"
        c["max_len"] = _log_int(rng, 1, 4096)
        c["cached"] = rng.choice([0, _log_int(rng, 1, 8192)])
    else:
        c["max_len"] = rng.choice([20, 40, 80, _log_int(rng, 2, 4096)])
        c["fused"] = rng.random() < 0.5
    c["min_len"] = rng.randint(0 if kind == "train" else 1, c["max_len"])
    pairs = c["heads"] * c["max_len"] * (c["max_len"] + c["cached"] if "cached" in c
                                         else c["max_len"])
    rows = max(1, 20000 * 80 * 8 * 64 // (c["max_len"] * c["heads"] * c["dim"]))
    c["docs"] = _log_int(rng, 1, max(1, min(20000, rows, MOST_SCORES[kind] // (4 * pairs))))
    return c


# ---- inputs -------------------------------------------------------------------------------------
def _lengths(n, lo, hi, skew):
    """n lengths of lo..hi: the same ones for every seed (which only orders them)."""
    return [lo + int((hi - lo) * ((i + 1) / n) ** skew + 0.5) for i in range(n)]


def _doc_lengths(c):
    q = _lengths(c["docs"], c["min_len"], c["max_len"], c["skew"])
    return q, [a + b for a, b in zip(q, _lengths(c["docs"], 0, c["cached"], 1.0)[::-1])]


class _State:
    pass


def _offsets(lens):
    return torch.nn.functional.pad(torch.cumsum(lens, 0), (1, 0))


def _bucket_ids(buckets, reach):
    """Bucket of every distance -reach..reach: keys after the query by halves, then buckets of one
    hop each, then buckets that widen by a constant factor."""
    after, before = buckets // 4, buckets - buckets // 4

    def of(n, count):
        exact = max(1, count // 2)
        if n < exact or count == exact:
            return min(n, count - 1)
        return min(count - 1, exact + int(math.log(n / exact) / math.log(max(2.0, (reach + 1) / exact))
                                          * (count - exact)))

    ids = [before + of(-d - 1, after) if d < 0 and after else of(max(d, 0), before)
           for d in range(-reach, reach + 1)]
    return torch.tensor(ids, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = _full(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    s = _State()
    s.case = c

    def normal(*shape, std=1.0, of=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(of)

    h, hk, dim = c["heads"], c["kv_heads"], c["dim"]
    s.table = s.buckets = s.slopes = s.times = s.k_times = s.prefix = None
    if c["buckets"]:
        s.table = normal(h, c["buckets"], std=0.5)
        s.buckets = _bucket_ids(c["buckets"], c["reach"])
    if c["kind"] == "bias":
        s.grad = normal(h, c["q_len"], c["k_len"])
        s.table.requires_grad_()
        torch.cuda.synchronize()
        return s
    if c["slopes"]:
        s.slopes = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h)
    q_lens, k_lens = _doc_lengths(c)
    order = torch.randperm(c["docs"], generator=gen, device="cuda")
    s.lens = torch.tensor(q_lens, device="cuda")[order]
    s.k_lens = torch.tensor(k_lens, device="cuda")[order]

    def clock(*shape):
        """Event times: exponential gaps of mean one."""
        return torch.cumsum(torch.empty(*shape, device="cuda").exponential_(generator=gen), -1)

    if c["kind"] == "step":
        n, room = c["docs"], c["capacity"]
        s.q, s.k, s.v = normal(n, h, dim), normal(n, hk, dim), normal(n, hk, dim)
        s.k_cache, s.v_cache = normal(n, room, hk, dim), normal(n, room, hk, dim)
        if c["times"]:
            s.k_times = clock(n, room)
            s.times = s.k_times.gather(1, s.lens[:, None])[:, 0].contiguous()
        torch.cuda.synchronize()
        return s
    if c["layout"] == "padded":
        rows = k_rows = (c["docs"], c["max_len"])
    else:
        s.offsets, s.k_offsets = _offsets(s.lens), _offsets(s.k_lens)
        rows, k_rows = (sum(q_lens),), (sum(k_lens),)
    if c["fused"]:
        qkv = normal(*rows, (h + 2 * hk) * dim).unflatten(-1, (h + 2 * hk, dim))
        s.q, s.k, s.v = qkv.split([h, hk, hk], -2)
    else:
        s.q, s.k, s.v = normal(*rows, h, dim), normal(*k_rows, hk, dim), normal(*k_rows, hk, dim)
    if c["times"]:
        s.k_times = clock(*k_rows)
        s.times = s.k_times
        if c["cached"]:
            first = torch.repeat_interleave(s.k_offsets[1:] - s.offsets[1:], s.lens)
            s.times = s.k_times[torch.arange(rows[0], device="cuda") + first].contiguous()
    if c["mask"] == "prefix":
        s.prefix = (torch.rand(c["docs"], generator=gen, device="cuda") * (s.k_lens + 1)).long()
    if c["kind"] == "train":
        s.grad = normal(*rows, h, dim)
        s.inputs = [x.detach().requires_grad_() for x in (s.q, s.k, s.v)]
        s.q, s.k, s.v = s.inputs
        if s.table is not None:
            s.inputs.append(s.table.requires_grad_())
    torch.cuda.synchronize()
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _masked_attention(q, k, v, seen, bias, slopes, gap, softcap):
    """q [n, heads, lq, dim], k and v [n, kv_heads, lk, dim], all float32; `seen` [n, 1, lq, lk];
    `gap` the times between, broadcast over the scores."""
    n, h, lq, dim = q.shape
    hk, lk = k.shape[1], k.shape[2]
    q = q.unflatten(1, (hk, h // hk)).flatten(2, 3)  # the heads that share keys are more rows
    x = (q @ k.transpose(-1, -2) * dim ** -0.5).view(n, h, lq, lk)
    if softcap:
        x = torch.tanh(x / softcap) * softcap
    if bias is not None:
        x = x + bias
    if slopes is not None:
        x = x - slopes[:, None, None] * gap.abs()
    x = x.masked_fill(~seen, -math.inf)
    top = x.detach().amax(-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    o = (e.view(n, hk, h // hk * lq, lk) @ v).view(n, h, lq, dim)
    return o / total.clamp_min(1e-30)


def _by_distance(s):
    """The bias of every distance -reach..reach: table columns picked by a product, so that its
    gradient is one too."""
    one_hot = s.buckets[:, None] == torch.arange(s.table.shape[1], device="cuda")
    return s.table.float() @ one_hot.float().T


def _toeplitz(by_distance, q_len, k_len, offset):
    """[heads, q_len, k_len] of i + offset - j."""
    reach = by_distance.shape[1] // 2
    d = torch.arange(offset + q_len - 1, offset - k_len, -1, device="cuda").clamp(-reach, reach)
    at = (d + reach)[:, None] == torch.arange(2 * reach + 1, device="cuda")
    line = by_distance @ at.float().T  # distances falling from the last row's first column
    return line.unfold(1, k_len, 1).flip(1)


def _padded(x, slot, docs, length):
    if slot is None:
        return x.transpose(1, 2).float()
    rows = x.new_zeros(docs * length, *x.shape[1:], dtype=torch.float32)
    return rows.index_copy(0, slot, x.float()).unflatten(0, (docs, length)).transpose(1, 2)


def _slots(offsets, rows, length):
    at = torch.arange(rows, device="cuda")
    doc = torch.searchsorted(offsets, at, right=True) - 1
    return doc * length + at - offsets[doc]


def _plain_attention(s):
    c = s.case
    docs, lq = c["docs"], c["max_len"]
    packed = c["layout"] == "packed"
    lk = max(_doc_lengths(c)[1]) if packed else lq
    slot = k_slot = None
    if packed:
        slot = _slots(s.offsets, s.q.shape[0], lq)
        k_slot = _slots(s.k_offsets, s.k.shape[0], lk)
    q = _padded(s.q, slot, docs, lq)
    k, v = _padded(s.k, k_slot, docs, lk), _padded(s.v, k_slot, docs, lk)
    i = torch.arange(lq, device="cuda")[:, None]
    j = torch.arange(lk, device="cuda")
    ahead = (s.k_lens - s.lens)[:, None, None]  # keys before a document's first query
    seen = (i < s.lens[:, None, None]) & (j < s.k_lens[:, None, None])
    if c["mask"] != "full":
        past = j <= i + ahead
        if c["mask"] == "prefix":
            past = past | (j < s.prefix[:, None, None])
        seen = seen & past
    bias = gap = None
    if c["buckets"]:
        if c["cached"]:
            reach = c["reach"]
            d = (i + ahead - j).clamp(-reach, reach) + reach
            bias = _by_distance(s)[:, d].transpose(0, 1)
        else:
            bias = _toeplitz(_by_distance(s), lq, lk, 0)
    if c["slopes"]:
        gap = (i + ahead - j).float()[:, None]
        if c["times"]:
            tq, tk = s.times[..., None], s.k_times[..., None]
            if packed:
                tq = _padded(tq[..., None], slot, docs, lq)[:, 0]
                tk = _padded(tk[..., None], k_slot, docs, lk)[:, 0]
            gap = (tq - tk.transpose(1, 2))[:, None]
    o = _masked_attention(q, k, v, seen[:, None], bias, s.slopes, gap, c["softcap"])
    o = o.transpose(1, 2)
    if packed:
        o = o.flatten(0, 1).index_select(0, slot)
    return o.to(s.q.dtype)


def _plain_step(s):
    c = s.case
    at = torch.arange(c["docs"], device="cuda")
    s.k_cache[at, s.lens] = s.k
    s.v_cache[at, s.lens] = s.v
    if c["times"]:
        s.k_times[at, s.lens] = s.times
    j = torch.arange(c["capacity"], device="cuda")
    d = s.lens[:, None] - j
    bias = gap = None
    if c["buckets"]:
        bias = _by_distance(s)[:, d.clamp(-c["reach"], c["reach"]) + c["reach"]]
        bias = bias.transpose(0, 1)[:, :, None]
    if c["slopes"]:
        gap = (s.times[:, None] - s.k_times if c["times"] else d.float())[:, None, None]
    o = _masked_attention(s.q.float()[:, :, None], s.k_cache.transpose(1, 2).float(),
                          s.v_cache.transpose(1, 2).float(), (d >= 0)[:, None, None], bias,
                          s.slopes, gap, c["softcap"])
    return o[:, :, 0].to(s.q.dtype)


def _plain_bias(s):
    c = s.case
    return _toeplitz(_by_distance(s), c["q_len"], c["k_len"], c["q_offset"]).to(s.table.dtype)


# ---- the framework's calls ----------------------------------------------------------------------
def _operators():
    package = os.path.join(os.getcwd(), "temporal-random-walk_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from temporal_random_walk import operators
    return operators


def _own_attention(s):
    c, ops = s.case, _operators()
    if c["layout"] == "padded":
        mask = ops.WalkMask.padded(s.lens, c["max_len"], kind=c["mask"], prefix=s.prefix)
    else:
        mask = ops.WalkMask.packed(s.offsets, s.q.shape[0], k_offsets=s.k_offsets,
                                   k_rows=s.k.shape[0], kind=c["mask"], prefix=s.prefix)
    return ops.walk_attention(s.q, s.k, s.v, mask, softcap=c["softcap"], bias_table=s.table,
                              buckets=s.buckets, slopes=s.slopes, times=s.times,
                              k_times=s.k_times)


def _own_step(s):
    return _operators().walk_attention_step(
        s.q, s.k, s.v, s.k_cache, s.v_cache, s.lens, softcap=s.case["softcap"],
        bias_table=s.table, buckets=s.buckets, slopes=s.slopes, times=s.times, k_times=s.k_times)


def _own_bias(s):
    c = s.case
    return _operators().relative_bias(s.table, s.buckets, c["q_len"], c["k_len"],
                                      q_offset=c["q_offset"])


def run(state):
    s = state
    kind = s.case["kind"]
    if kind == "step":
        out = {"out": _own_step(s) if own else _plain_step(s), "k_cache": s.k_cache,
               "v_cache": s.v_cache}
        if s.k_times is not None:
            out["k_times"] = s.k_times
        return out
    if kind == "prompt":
        with torch.no_grad():
            return {"out": _own_attention(s) if own else _plain_attention(s)}
    if kind == "bias":
        out = _own_bias(s) if own else _plain_bias(s)
        return {"out": out.detach(), "d_table": torch.autograd.grad(out, s.table, s.grad)[0]}
    out = _own_attention(s) if own else _plain_attention(s)
    grads = torch.autograd.grad(out, s.inputs, s.grad)
    return {"out": out.detach(), **dict(zip(("d_q", "d_k", "d_v", "d_table"), grads))}


# ---- what a pass cannot do without --------------------------------------------------------------
def _pairs(c):
    """Query and key pairs that the mask leaves (prefixes, which the seed makes, are half a document
    at the mean)."""
    total = 0
    for a, b in zip(*_doc_lengths(c)):
        causal = a * (b - a) + a * (a + 1) // 2
        total += {"causal": causal, "full": a * b, "prefix": causal + a * b // 8}[c["mask"]]
    return total


def work(case):
    c = _full(case)
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "bias":
        n = c["heads"] * c["q_len"] * c["k_len"]
        return {"bytes": 2 * n * size, "flops": n}
    q_lens, k_lens = _doc_lengths(c)
    wide = c["dim"] * size
    if c["kind"] == "step":
        events, n = sum(q_lens), c["docs"]
        nbytes = 2 * events * c["kv_heads"] * wide + (2 * c["heads"] + 4 * c["kv_heads"]) * n * wide
        return {"bytes": nbytes + 4 * events * c["times"],
                "flops": 4 * c["dim"] * c["heads"] * (events + n)}
    nq, nk, pairs = sum(q_lens), sum(k_lens), _pairs(c)
    nbytes = (2 * nq * c["heads"] + 2 * nk * c["kv_heads"]) * wide
    flops = 4 * c["dim"] * c["heads"] * pairs
    if c["kind"] == "train":  # q k v o and o's gradient read again, three gradients written
        return {"bytes": nbytes + (4 * nq * c["heads"] + 4 * nk * c["kv_heads"]) * wide,
                "flops": 3 * flops}
    return {"bytes": nbytes, "flops": flops}


# ---- the same in 64 bits ------------------------------------------------------------------------
def _exact_scores(c, q, k, first, slopes, table, ids, tq, tk, prefix):
    """Scores before the softmax and what the cap left of their slope.  q [n, h, a, dim],
    k [n, h, b, dim]; the queries' positions are first.., the keys' 0.."""
    x = torch.matmul(q, k.mT) / math.sqrt(c["dim"])
    slope = torch.ones((), dtype=torch.float64, device="cuda")
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
        slope = 1 - (x / c["softcap"]) ** 2
    a, b = q.shape[2], k.shape[2]
    hop = first + torch.arange(a, device="cuda")[:, None] - torch.arange(b, device="cuda")[None]
    bucket = None
    if table is not None:
        bucket = ids.long()[torch.clamp(hop, -c["reach"], c["reach"]) + c["reach"]]
        x = x + table[:, bucket]
    if slopes is not None:
        apart = hop.double() if tq is None else tq[:, None, :, None] - tk[:, None, None, :]
        x = x - slopes[:, None, None] * torch.abs(apart)
    if c["mask"] == "causal":
        x = torch.where(hop < 0, -math.inf, x)
    elif c["mask"] == "prefix":
        inside = torch.arange(b, device="cuda") < prefix[:, None]
        x = torch.where((hop < 0) & ~inside[:, None, None], -math.inf, x)
    return x, slope, bucket


def _exact_attention(s):
    c = s.case
    h, hk = c["heads"], c["kv_heads"]
    group = h // hk
    packed = c["layout"] == "packed"
    train = c["kind"] == "train"
    q, k, v = (x.detach().flatten(0, -3) for x in (s.q, s.k, s.v))
    do = s.grad.flatten(0, -3) if train else None
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = ([torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k, v)]
                  if train else (None, None, None))
    table = None if s.table is None else s.table.detach().double()
    d_table = None if table is None else torch.zeros_like(table)
    slopes = None if s.slopes is None else s.slopes.double()
    groups = {}
    for w, (a, b) in enumerate(zip(s.lens.tolist(), s.k_lens.tolist())):
        if a and b:
            groups.setdefault((a, b), []).append(w)
    starts = (s.offsets[:-1] if packed else
              torch.arange(c["docs"], device="cuda") * c["max_len"])
    k_starts = s.k_offsets[:-1] if packed else starts
    tq, tk = (None if t is None else t.double().flatten() for t in (s.times, s.k_times))
    for (a, b), members in groups.items():
        many = max(1, (1 << 27) // (a * b))  # documents and heads at a time
        for w0 in range(0, len(members), many):
            w = torch.tensor(members[w0:w0 + many], device="cuda")
            rows = starts[w][:, None] + torch.arange(a, device="cuda")
            k_rows = k_starts[w][:, None] + torch.arange(b, device="cuda")
            heads = max(1, many // len(w) // group)
            for g0 in range(0, hk, heads):
                gs = torch.arange(g0, min(hk, g0 + heads), device="cuda")
                hs = (gs[:, None] * group + torch.arange(group, device="cuda")).flatten()
                of = torch.arange(len(gs), device="cuda").repeat_interleave(group)
                qs = q[rows][:, :, hs].transpose(1, 2).double()
                ks = k[k_rows][:, :, gs].transpose(1, 2).double()[:, of]
                vs = v[k_rows][:, :, gs].transpose(1, 2).double()[:, of]
                x, slope, bucket = _exact_scores(
                    c, qs, ks, b - a, None if slopes is None else slopes[hs],
                    None if table is None else table[hs], s.buckets,
                    None if tq is None else tq[rows], None if tk is None else tk[k_rows],
                    None if s.prefix is None else s.prefix[w])
                p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)  # a row without keys
                o = torch.matmul(p, vs)
                at = (rows[:, None, :], hs[None, :, None])
                out[at] = o
                if not train:
                    continue
                dos = do[rows][:, :, hs].transpose(1, 2).double()
                ds = p * (torch.matmul(dos, vs.mT) - (dos * o).sum(-1, keepdim=True))
                if table is not None:
                    for t in range(table.shape[1]):
                        d_table[hs, t] += (ds * (bucket == t)).sum((0, 2, 3))
                dx = ds * slope / math.sqrt(c["dim"])
                dq[at] = torch.matmul(dx, ks)
                k_at = (k_rows[:, None, :], gs[None, :, None])
                dk[k_at] = torch.matmul(dx.mT, qs).unflatten(1, (len(gs), group)).sum(2)
                dv[k_at] = torch.matmul(p.mT, dos).unflatten(1, (len(gs), group)).sum(2)
    res = {"out": out.view(s.q.shape)}
    if train:
        res.update(d_q=dq.view(s.q.shape), d_k=dk.view(s.k.shape), d_v=dv.view(s.v.shape))
        if table is not None:
            res["d_table"] = d_table
    return res


def _exact_step(s):
    c = s.case
    group = c["heads"] // c["kv_heads"]
    table = None if s.table is None else s.table.double()
    slopes = None if s.slopes is None else s.slopes.double()
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    for w, n in enumerate(s.lens.tolist()):
        for x, new in ((s.k_cache, s.k), (s.v_cache, s.v), (s.k_times, s.times)):
            if x is not None:
                x[w, n] = new[w]
        for g in range(c["kv_heads"]):
            hs = slice(g * group, (g + 1) * group)
            times = [None if t is None else t.double() for t in (s.times, s.k_times)]
            x, _, _ = _exact_scores(
                dict(c, mask="full"), s.q[w, hs].double()[None, :, None],
                s.k_cache[w, :n + 1, g].double()[None, None], n,
                None if slopes is None else slopes[hs], None if table is None else table[hs],
                s.buckets, None if times[0] is None else times[0][w].view(1, 1),
                None if times[1] is None else times[1][w, :n + 1][None], None)
            p = torch.softmax(x[0, :, 0], -1)
            out[w, hs] = p @ s.v_cache[w, :n + 1, g].double()
    res = {"out": out, "k_cache": s.k_cache, "v_cache": s.v_cache}
    if s.k_times is not None:
        res["k_times"] = s.k_times
    return res


def _exact_bias(s):
    c = s.case
    hop = (c["q_offset"] + torch.arange(c["q_len"], device="cuda")[:, None]
           - torch.arange(c["k_len"], device="cuda"))
    bucket = s.buckets.long()[hop.clamp(-c["reach"], c["reach"]) + c["reach"]]
    d_table = torch.empty(s.table.shape, dtype=torch.float64, device="cuda")
    for h in range(c["heads"]):
        d_table[h] = torch.bincount(bucket.flatten(), s.grad[h].double().flatten(),
                                    minlength=c["buckets"])
    return {"out": s.table.detach().double()[:, bucket], "d_table": d_table}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"step": _exact_step, "bias": _exact_bias}.get(s.case["kind"], _exact_attention)(s)
