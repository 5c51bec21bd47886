"""Pages and beam search against their formulas in float64 (tests/serving_formulas.py,
tests/walk_formulas.py)."""
import math

import pytest
import torch

from tests import serving_formulas as sf
from tests import walk_formulas as wf

pytestmark = pytest.mark.gpu

BF, HF, SF, E8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
DTYPES = [BF, HF, SF]


@pytest.fixture(scope="module")
def ops():
    from temporal_random_walk import operators
    return operators


def _normal(gen, *shape, dtype=SF, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def _raw(x):
    """Comparable bits: codes as bytes, other types with one NaN."""
    x = x.cpu()
    return x.view(torch.uint8) if x.dtype == E8 else torch.nan_to_num(x.float(), nan=77.0)


class Pool:
    """A pool on the device and its rows on the CPU: [walks, capacity, kv_heads, dim] in float64, as
    the pages hold them (NaN where nothing has been written)."""

    def __init__(self, ops, walks, capacity, kv_heads, dim, *, rows=16, dtype=BF, eight=False,
                 seed=0, times=False):
        gen = torch.Generator().manual_seed(seed + 99)
        self.rows, self.eight, self.dtype = rows, eight, dtype
        each = -(-capacity // rows)
        total = walks * each + 3
        ids = torch.randperm(total, generator=gen)[:walks * each].int().view(walks, each)
        self.table = ids.cuda()
        self.pages = ops.Pages.empty(total, rows, kv_heads, dim, dtype=E8 if eight else dtype)
        for x in self.pages:  # what no walk has written is nobody's business
            if x is not None:
                x.view(torch.uint8).fill_(0xff)
        self.k = torch.full((walks, each * rows, kv_heads, dim), math.nan, dtype=torch.float64)
        self.v = self.k.clone()
        self.k_times = torch.full((total, rows), math.nan, device="cuda") if times else None

    def held(self, x):
        """Rows as the pages hold them."""
        if not self.eight:
            return x.to(self.dtype).double()
        codes, e = sf.eight_bits(x.double())
        return codes * torch.exp2(e)[..., None]

    def note(self, w, start, k, v):
        n = k.shape[0]
        self.k[w, start:start + n], self.v[w, start:start + n] = self.held(k), self.held(v)

    def values(self):
        """What the device's pages hold, in walks' order."""
        got = []
        for x, s in ((self.pages.k, self.pages.k_scale), (self.pages.v, self.pages.v_scale)):
            x = sf.CODES[x.cpu().view(torch.uint8).long()] if self.eight else x.cpu().double()
            if self.eight:
                x = x * torch.exp2(s.cpu().double() - 127)[..., None]
            got.append(x[self.table.cpu().long()].transpose(2, 3).flatten(1, 2))
        return got

    def check(self):
        for name, got, want in zip("kv", self.values(), (self.k, self.v)):
            same = (got == want) | (got.isnan() & want.isnan())
            written = ~want.isnan().all(-1)  # (bytes 0xff are NaN, and as scales not a row's)
            assert same[written].all(), name
            assert got[~written].isnan().all(), name


# ---- rows to pages and back ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight,dim,rows", [(False, 8, 16), (False, 40, 32), (False, 128, 16),
                                            (True, 16, 16), (True, 48, 64), (True, 128, 128)])
@pytest.mark.parametrize("padded", [False, True])
def test_write_and_read(ops, dtype, eight, dim, rows, padded):
    lens, starts = [5, 0, 1, 37, 16, 33, 9, 4], [0, 3, 15, 20, 16, 0, -1, 70]
    gen = torch.Generator().manual_seed(dim)
    pool = Pool(ops, len(lens), 72, 3, dim, rows=rows, dtype=dtype, eight=eight, times=True)
    pool.table[7, 64 // rows:] = -1  # positions from 64 on have no page
    room = [pool.k.shape[1]] * 7 + [64 // rows * rows]
    length = 37
    k, v = (_normal(gen, len(lens), length, 3, dim, dtype=dtype, std=3.0) for _ in range(2))
    t = torch.rand(len(lens), length, generator=gen)
    seen = torch.arange(length) < torch.tensor(lens)[:, None]
    if padded:
        ops.paged_write(pool.pages, pool.table, torch.tensor(starts).cuda(), k.cuda(), v.cuda(),
                        counts=torch.tensor(lens).cuda(), times=t.cuda(), k_times=pool.k_times)
    else:
        offsets = torch.tensor([0] + lens).cumsum(0) + 2  # rows before and behind are no walk's
        wide = lambda x: torch.cat([x[:1, :2].flatten(0, 1), x[seen], x[0, :3]]).cuda()  # noqa: E731
        ops.paged_write(pool.pages, pool.table, torch.tensor(starts).cuda(), wide(k), wide(v),
                        offsets=offsets.cuda(), times=wide(t[..., None])[:, 0].contiguous(),
                        k_times=pool.k_times)
    want_t = torch.full(pool.k.shape[:2], math.nan)
    for w, (n, s) in enumerate(zip(lens, starts)):
        n = min(n, room[w] - s) if s >= 0 else 0
        if n > 0:
            pool.note(w, s, k[w, :n], v[w, :n])
            want_t[w, s:s + n] = t[w, :n]
    # the last walk's rows have no page: its table names none that could be looked at
    pool.k, pool.v, pool.table = pool.k[:7], pool.v[:7], pool.table[:7]
    pool.check()
    got = ops.paged_read(pool.pages, pool.table, lens=torch.tensor([72] * 7).cuda(), length=72,
                         dtype=SF if eight else None, k_times=pool.k_times)
    for x, y in zip(got, (pool.k, pool.v, want_t[:7])):
        assert torch.equal(_raw(x), _raw(y[:, :72].float()))


def test_read_leaves_nothing(ops):
    """Rows of no walk, of no position and of no page are 0, whatever the pages hold."""
    pool = Pool(ops, 3, 48, 2, 64, rows=16, eight=True)
    pool.table[1, 1] = -1
    pool.table[2, 0] = pool.pages.k.shape[0]
    gen = torch.Generator().manual_seed(0)
    k, v = (_normal(gen, 3, 48, 2, 64, dtype=BF) for _ in range(2))
    ops.paged_write(pool.pages, pool.table, None, k.cuda(), v.cuda())
    want = [pool.held(x) for x in (k, v)]
    for x in want:
        x[1, 16:32], x[2, :16] = 0, 0
    lens = [48, 40, 20]
    got = ops.paged_read(pool.pages, pool.table, lens=torch.tensor(lens).cuda(), length=50)
    for x, y in zip(got, want):
        for w, n in enumerate(lens):
            assert torch.equal(x[w, :n].cpu().double(), y[w, :n]) and (x[w, n:] == 0).all()
    offsets = torch.tensor([1, 49, 49, 69])
    got = ops.paged_read(pool.pages, pool.table, offsets=offsets.cuda(), rows=75)
    for x, y in zip(got, want):
        x = x.cpu().double()
        assert torch.equal(x[1:49], y[0]) and torch.equal(x[49:69], y[2, :20])
        assert (x[:1] == 0).all() and (x[69:] == 0).all()
    far = ops.paged_read(pool.pages, pool.table[:1], lens=torch.tensor([90]).cuda(), length=90)
    assert (far[0][0, 48:] == 0).all()
    none = ops.paged_read(pool.pages, pool.table[:0], offsets=torch.tensor([0]).cuda(), rows=7)
    assert none[0].shape == (7, 2, 64) and (none[0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_eight_bits_of_any_rows(ops, dtype):
    """Zeros, borders between exponents, ties, the smallest and largest values, values that are not
    finite."""
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    rows = torch.zeros(12, 1, 16, dtype=torch.float64)
    rows[1, 0, 3] = 448.0
    rows[2, 0, :2] = torch.tensor([449.0 if dtype == SF else 450.0, -1.0])
    rows[3, 0] = torch.arange(16) * 28 + 14.0  # halves between codes
    rows[4, 0] = torch.linspace(-top, top, 16, dtype=torch.float64)
    rows[5, 0, 5] = tiny
    rows[6, 0] = torch.exp2(-torch.arange(16).double())
    rows[7, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 5.0])
    rows[8, 0, :3] = torch.tensor([1.75, 1.76, -1.0])
    rows[9, 0] = math.inf
    rows[10, 0] = torch.arange(16) * tiny
    rows[11, 0] = torch.randn(16, generator=torch.Generator().manual_seed(4)) * 1e-3
    rows = rows.to(dtype)
    pages = ops.Pages.empty(1, 16, 1, 16, dtype=E8)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    ops.paged_write(pages, table, None, rows[None].cuda(), -rows[None].cuda())
    codes, e = sf.eight_bits(rows.double())
    for x, s, sign in ((pages.k, pages.k_scale, 1), (pages.v, pages.v_scale, -1)):
        got = sf.CODES[x[0, 0, :12].cpu().view(torch.uint8).long()] * sign
        assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(codes[:, 0], nan=1e9))
        assert torch.equal(s[0, 0, :12].cpu().double() - 127, e[:, 0])
    back = ops.paged_read(pages, table, lens=torch.tensor([12]).cuda(), length=12, dtype=SF)[0]
    assert torch.equal(_raw(back[0]), _raw((codes * torch.exp2(e)[..., None]).float()))


def test_offsets_past_32_bits(ops):
    """Pools of more than 2^32 bytes and elements, and pages that lie past both."""
    count, rows, heads, dim = (1 << 18) + 5, 64, 2, 128
    assert count * rows * heads * dim > 1 << 32
    k = torch.empty(count, heads, rows, dim, dtype=E8, device="cuda")
    scale = torch.empty(count, heads, rows, dtype=torch.uint8, device="cuda")
    pages = ops.Pages(k, k.clone(), scale, scale.clone())
    table = torch.tensor([[count - 1, 3, count - 2]], dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(3)
    rows_k, rows_v = (_normal(gen, 1, 150, heads, dim, dtype=BF) for _ in range(2))
    ops.paged_write(pages, table, None, rows_k.cuda(), rows_v.cuda())
    got = ops.paged_read(pages, table, lens=torch.tensor([150]).cuda(), length=150)
    held = [(lambda c, e: c * torch.exp2(e)[..., None])(*sf.eight_bits(x.double()))
            for x in (rows_k, rows_v)]
    for x, y in zip(got, held):
        assert torch.equal(x.cpu().double(), y)
    q, new = _normal(gen, 1, 4, dim, dtype=BF), _normal(gen, 1, heads, dim, dtype=BF)
    out = ops.paged_attention_step(q.cuda(), new.cuda(), new.cuda(), pages, table,
                                   torch.tensor([150]).cuda())
    c, e = sf.eight_bits(new.double())
    last = c * torch.exp2(e)[..., None]
    want = wf.attention(q.double(), torch.cat([held[0][0], last]), torch.cat([held[1][0], last]),
                        wf.documents("causal", [1], [151]), dtype=BF)["out"]
    wf.check("out", out, *want)


# ---- one event over pages -------------------------------------------------------------------------
def _step(ops, dtype, lens, capacity, heads, kv_heads, dim, *, eight=False, rows=16, first=None,
          holes=(), softcap=0.0, num=0, reach=0, slopes=False, times=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = len(lens)
    pool = Pool(ops, n, capacity, kv_heads, dim, rows=rows, dtype=dtype, eight=eight, seed=seed,
                times=times)
    capacity = pool.k.shape[1]
    q = _normal(gen, n, heads, dim, dtype=dtype)
    k, v = (_normal(gen, n, kv_heads, dim, dtype=dtype) for _ in range(2))
    kc, vc = (_normal(gen, n, capacity, kv_heads, dim, dtype=dtype) for _ in range(2))
    kt = torch.rand(n, capacity, generator=gen).cumsum(1)
    tq = torch.tensor([float(kt[b, max(0, min(m, capacity) - 1)]) + 0.5 for b, m in enumerate(lens)])
    counts = torch.tensor([max(0, min(m, capacity)) for m in lens])
    ops.paged_write(pool.pages, pool.table, None, kc.cuda(), vc.cuda(), counts=counts.cuda(),
                    times=kt.cuda() if times else None, k_times=pool.k_times)
    for b in range(n):
        pool.note(b, 0, kc[b, :counts[b]], vc[b, :counts[b]])
    gone = torch.zeros(n, capacity, dtype=torch.bool)
    table = pool.table.clone()
    for b, page in holes:
        table[b, page] = -1 if page % 2 else pool.pages.k.shape[0] + 5
        gone[b, page * rows:(page + 1) * rows] = True
    bias = _normal(gen, heads, num) if num else None
    ids = ops.distance_buckets(num, reach, device="cpu") if num else None
    slope = torch.rand(heads, generator=gen) * 0.1 if slopes else None
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    out = ops.paged_attention_step(
        q.cuda(), k.cuda(), v.cuda(), pool.pages, table, torch.tensor(lens).cuda(),
        first=None if first is None else torch.tensor(first).cuda(), softcap=softcap,
        bias_table=dev(bias), buckets=dev(ids), slopes=dev(slope), times=dev(tq) if times else None,
        k_times=pool.k_times)
    d = lambda x: None if x is None else x.double()  # noqa: E731
    for b, m in enumerate(lens):
        if m < 0:
            assert (out[b] == 0).all(), b
            continue
        if m >= capacity or gone[b, m]:
            assert torch.isnan(out[b]).all(), b
            continue
        pool.note(b, m, k[b:b + 1], v[b:b + 1])
        kt[b, m] = tq[b]
        begin = 0 if first is None else min(max(first[b], 0), m)
        seen = (torch.arange(m + 1) >= begin) & ~gone[b, :m + 1]
        held = [x[b, :m + 1].nan_to_num(0.0) for x in (pool.k, pool.v)]
        want = wf.attention(
            q[b:b + 1].double(), *held, [(m, 1, m + 1, seen[None])], softcap=softcap, table=d(bias),
            buckets=ids, slopes=d(slope), q_times=tq[b:b + 1].double() if times else None,
            k_times=kt[b, :m + 1].double() if times else None, dtype=dtype)["out"]
        wf.check(f"out[{b}] of {m}", out[b:b + 1], *want)
    pool.check()
    if times:
        got = pool.k_times.cpu()[pool.table.cpu().long()].flatten(1)
        for b, m in enumerate(lens):
            if 0 <= m < capacity and not gone[b, m]:
                assert torch.equal(got[b, :m + 1], kt[b, :m + 1])


LENS = [0, 1, 15, 16, 17, 31, 32, 47, 63, 64, 127, 128, 199, -1, 208, 7]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight,dim", [(False, 8), (False, 40), (False, 64), (False, 96), (False, 128),
                                       (True, 16), (True, 48), (True, 64), (True, 80), (True, 128)])
def test_step_lengths(ops, dtype, eight, dim):
    _step(ops, dtype, LENS, 200, 4, 2, dim, eight=eight, seed=dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("rows", [16, 32, 128, 1024])
def test_step_pages(ops, dtype, eight, rows):
    """Pages of every kind, of walks that are cut among workgroups."""
    _step(ops, dtype, [0, 700, 1023, 1024, 100, 33, -5, 2000], 2048, 6, 2, 64, eight=eight, rows=rows,
          slopes=True, seed=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("terms", [
    dict(softcap=4.0), dict(softcap=3000.0), dict(slopes=True), dict(slopes=True, times=True),
    dict(num=16, reach=20), dict(num=32, reach=1024, softcap=9.0, slopes=True, times=True),
    dict(num=1, reach=0)])
@pytest.mark.parametrize("eight", [False, True])
def test_step_terms(ops, dtype, terms, eight):
    _step(ops, dtype, [0, 5, 90, 300, -7, 415], 416, 6, 2, 64, eight=eight, **terms)
    _step(ops, dtype, [0, 5, 690, 300, -7, 1415], 1456, 6, 2, 64, eight=eight, **terms)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (16, 1), (17, 1), (33, 1), (70, 2), (5, 5)])
def test_step_shared_heads(ops, heads, kv_heads, eight):
    _step(ops, BF, [100, 0, 64], 128, heads, kv_heads, 64, eight=eight)
    _step(ops, BF, [900, 0, 64], 1000, heads, kv_heads, 64, eight=eight)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("capacity", [208, 1040])
def test_step_windows_and_holes(ops, dtype, eight, capacity):
    """Firsts inside pages, at borders, past the end and below 0; pages that a table does not name."""
    lens = [200, 150, 100, 64, 63, 31, 5, 207, 190, 120]
    first = [0, 149, 101, 33, 32, 16, -3, 100, 176, 1 << 40]
    _step(ops, dtype, lens, capacity, 4, 2, 64, eight=eight, first=first, seed=capacity)
    holes = [(0, 0), (0, 3), (1, 9), (2, 6), (3, 1), (3, 2), (7, 5), (7, 6), (8, 11), (4, 0), (4, 1)]
    _step(ops, dtype, lens, capacity, 4, 2, 64, eight=eight, holes=holes, slopes=True)
    _step(ops, dtype, lens, capacity, 4, 2, 64, eight=eight, first=first, holes=holes, times=True,
          slopes=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight", [False, True])
def test_step_many_walks(ops, dtype, eight):
    """More walks than a wave has lanes, and more than a workgroup has threads; walks of very
    different lengths, of which the tables leave room for long ones."""
    _step(ops, dtype, [(37 * i) % 97 - 2 for i in range(130)] + [800], 816, 2, 1, 32, eight=eight)
    _step(ops, dtype, [(7 * i) % 20 - 1 for i in range(300)], 520, 1, 1, 32, eight=eight)


@pytest.mark.parametrize("dtype,eight", [(BF, True), (HF, True), (SF, True), (BF, False)])
def test_step_long_histories(ops, dtype, eight):
    _step(ops, dtype, [9000, 3, 20001], 20016, 4, 1, 64, eight=eight, rows=64, slopes=True, times=True)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_stays_in_its_walk(ops, eight, bad):
    gen = torch.Generator().manual_seed(0)
    pool = Pool(ops, 3, 640, 1, 64, eight=eight)
    lens = torch.tensor([620, 100, 33])
    kc, vc = (_normal(gen, 3, 640, 1, 64, dtype=BF) for _ in range(2))
    q, k, v = (_normal(gen, 3, 1, 64, dtype=BF) for _ in range(3))

    def run():
        ops.paged_write(pool.pages, pool.table, None, kc.cuda(), vc.cuda(), counts=lens.cuda())
        return ops.paged_attention_step(q.cuda(), k.cuda(), v.cuda(), pool.pages, pool.table,
                                        lens.cuda(), first=torch.tensor([0, 50, 0]).cuda())

    fine = run()
    kc[1, 20, 0, 3], vc[1, 49] = bad, bad  # before the window
    assert torch.equal(run(), fine)
    vc[1, 60, 0, 5] = bad
    got = run()
    assert torch.equal(got[[0, 2]], fine[[0, 2]]) and not torch.isfinite(got[1, 0, 5])


# ---- choice among beams -----------------------------------------------------------------------------
def _choose(ops, logits, scores, width, ended=None, end=None):
    got = ops.beam_select(logits.cuda(), scores.cuda(), width,
                          ended=None if ended is None else ended.cuda(), end_token=end)
    x = logits.double()
    for g in range(x.shape[0]):
        s, t, p, e = sf.choice(x[g], scores[g], width, None if ended is None else ended[g], end)
        assert got.tokens[g].tolist() == t and got.parents[g].tolist() == p, g
        assert got.ended[g].tolist() == e, g
        want = torch.tensor(s, dtype=torch.float64)
        # a sum of exponentials: 64 terms a lane, 6 joins of lanes, and of chunks, each rounded;
        # exponentials are good to 2 units; scores are rounded once
        bound = 90 * 2.0 ** -24 + want.abs().nan_to_num(posinf=0.0) * 2.0 ** -24
        off = (got.scores[g].cpu().double() - want).nan_to_num(0.0).abs()
        assert (torch.isinf(got.scores[g].cpu()) == torch.isinf(want)).all()
        assert (off <= bound).all(), (off - bound).max()


SIZES = [(2, 3, 100, 5), (3, 4, 9000, 8), (1, 8, 50021, 8), (1, 32, 20000, 32), (2, 1, 70001, 32),
         (1, 5, 4097, 1), (2, 2, 5, 32), (1, 1, 1, 3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,beams,nodes,width", SIZES)
def test_choice(ops, dtype, groups, beams, nodes, width):
    gen = torch.Generator().manual_seed(nodes)
    logits = _normal(gen, groups, beams, nodes, dtype=dtype, std=3.0)
    scores = -5 * torch.rand(groups, beams, generator=gen)
    _choose(ops, logits, scores, width)
    ended = torch.rand(groups, beams, generator=gen) < 0.3
    _choose(ops, logits, scores, width, ended, nodes // 2)
    _choose(ops, logits, scores, width, torch.ones_like(ended), 0)
    # rows of any alignment
    wide = _normal(gen, groups, beams + 1, nodes + 3, dtype=dtype, std=3.0)
    _choose(ops, wide[:, 1:, 1:nodes + 1], scores, width)
    _choose(ops, wide.transpose(1, 2).contiguous().transpose(1, 2)[:, :beams, :nodes], scores, width)
    _choose(ops, wide[:, :1, :nodes].expand(groups, beams, nodes), scores[:, :1].expand(-1, beams),
            width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,beams,nodes,width", SIZES)
def test_choice_among_equals(ops, dtype, groups, beams, nodes, width):
    """Constant rows, rows of few values, rising and falling ones, full lanes of large ones."""
    gen = torch.Generator().manual_seed(nodes + 1)
    x = _normal(gen, groups, beams, nodes)
    zero = torch.zeros(groups, beams)
    for logits in (torch.full_like(x, -1.5), (2 * x).round(), torch.where(x > 0, 0.0, -0.0),
                   torch.arange(nodes).float().expand_as(x), -torch.arange(nodes).float().expand_as(x),
                   torch.where((torch.arange(nodes) // 8) % 64 < width + 3, x.abs() + 5, x)):
        logits = logits.to(dtype).contiguous()
        _choose(ops, logits, zero, width)
        _choose(ops, logits, -torch.rand(groups, beams, generator=gen), width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,beams,nodes,width", SIZES)
def test_choice_of_masked_nodes(ops, dtype, groups, beams, nodes, width):
    gen = torch.Generator().manual_seed(nodes + 2)
    x = _normal(gen, groups, beams, nodes, dtype=dtype)
    scores = -torch.rand(groups, beams, generator=gen)
    for low in (torch.finfo(dtype).min, -math.inf):
        y = torch.full_like(x, low)
        y[..., 3::1999] = x[..., 3::1999]
        _choose(ops, y, scores, width)
        _choose(ops, torch.full_like(x, low), scores, width, None, nodes - 1)
    y = x.clone()
    y[0, 0, nodes // 2] = math.nan
    y[-1, -1, 0] = math.inf
    _choose(ops, y, scores, width)
    scores[0, 0], scores[-1, -1] = -math.inf, math.nan
    _choose(ops, x, scores, width)
    _choose(ops, x, torch.full_like(scores, -math.inf), width, None, 0)


def test_choice_over_a_large_graph(ops):
    """More chunks than are ranked at once, also where all are equal."""
    gen = torch.Generator().manual_seed(8)
    x = _normal(gen, 1, 16, 1000003, dtype=HF)
    scores = -torch.rand(1, 16, generator=gen)
    _choose(ops, x, scores, 16)
    _choose(ops, torch.ones_like(x), scores, 32)
    _choose(ops, torch.ones_like(x), torch.zeros(1, 16), 32)


# ---- reordering ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("groups,beams,rows,layers", [(1, 1, 16, 1), (3, 2, 16, 2), (5, 4, 32, 3),
                                                      (2, 32, 64, 1), (1, 8, 1024, 9)])
def test_reorder(ops, eight, groups, beams, rows, layers):
    gen = torch.Generator().manual_seed(rows + beams)
    each, kv_heads = 4, [1 + n % 3 for n in range(layers)]
    count = groups * beams * each
    table = torch.randperm(count, generator=gen).int().view(-1, each)
    caches = []
    for h in kv_heads:
        dim = 16 * h
        bits = lambda *s: torch.randint(0, 127, (count, h, rows, *s), dtype=torch.uint8,  # noqa: E731
                                        generator=gen).cuda()
        if eight:
            caches.append(ops.Pages(bits(dim).view(E8), bits(dim).view(E8), bits(), bits()))
        else:
            caches.append(ops.Pages(bits(2 * dim).view(HF), bits(2 * dim).view(HF)))
    times = torch.rand(count, rows, generator=gen).cuda()
    for turn in range(4):
        length = [0, rows, rows + 5, 4 * rows][turn]
        lens = torch.full((groups * beams,), length)
        lens[::3] = min(length, 7)  # beams that have ended are shorter
        parents = torch.randint(beams, (groups, beams), generator=gen)
        if turn == 3:
            parents[:] = 0
        want = [[None if x is None else x.clone() for x in c] for c in caches]
        want_times = times.clone()
        rows_of, lens_of = [], []
        for g in range(groups):
            a = g * beams
            # only beams that still grow have several children
            here = parents[g].tolist()
            grow = [b for b in range(beams) if lens[a + b] == length]
            taken = set()
            for i, p in enumerate(here):
                if lens[a + p] < length and p in taken:
                    here[i] = grow[i % len(grow)] if grow else p
                taken.add(here[i])
            parents[g] = torch.tensor(here)
            r, n, copies = sf.reorder(table[a:a + beams].tolist(), lens[a:a + beams].tolist(), here,
                                      rows)
            rows_of += r
            lens_of += n
            for source, target, left in copies:
                for c in want:
                    for x in c:
                        if x is not None:
                            x.view(torch.uint8)[target, :, :left] = x.view(torch.uint8)[source, :, :left]
                want_times[target, :left] = want_times[source, :left]
        before = table.clone()
        got, got_lens = ops.beam_reorder(table.cuda(), lens.cuda(), parents.cuda(), caches,
                                         k_times=times)
        assert got.tolist() == rows_of and got_lens.tolist() == lens_of
        assert torch.equal(table, before)
        for c, d in zip(caches, want):
            for x, y in zip(c, d):
                if x is not None:
                    assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        assert torch.equal(times, want_times)
        table = got.cpu()


def test_reorder_out_of_range(ops):
    """Parents outside the group count as its first or last beam; pages outside the pool stay out."""
    pages = ops.Pages.empty(4, 16, 1, 8)
    for x in pages[:2]:
        x.fill_(1.0)
    table = torch.tensor([[0, -1], [1 << 30, 2]], dtype=torch.int32).cuda()
    got, lens = ops.beam_reorder(table, torch.tensor([3, 3]).cuda(), torch.tensor([[-5, 0]]).cuda(),
                                 [pages])
    assert got.tolist() == [[0, -1], [1 << 30, 2]] and lens.tolist() == [3, 3]
    got, _ = ops.beam_reorder(table, torch.tensor([3, 1 << 50]).cuda(), torch.tensor([[7, 9]]).cuda(),
                              [pages])
    assert got.tolist() == [[1 << 30, 2], [1 << 30, 2]]
    empty = torch.tensor([[0, 1], [2, -1], [3, -1]], dtype=torch.int32).cuda()
    got, _ = ops.beam_reorder(empty, torch.full((3,), 20).cuda(), torch.tensor([[0, 0, 1]]).cuda(),
                              [pages])
    assert got.tolist() == [[0, 1], [0, -1], [2, -1]]
    assert (pages.k == 1).all() and (pages.v == 1).all()


@pytest.mark.parametrize("lens,table", [
    # Beam 0 has ended early; beams 1 to 3 went on together, from page 1 on.
    ([10, 40, 40, 40], [[0, 4, 5], [1, 6, 7], [1, 6, 8], [1, 9, 10]]),
    # Beam 2 holds what ended beam 1 does, and beam 3, the longest, is dropped.
    ([25, 20, 20, 50], [[0, 4, 5, 11], [1, 6, 7, 12], [1, 6, 8, 13], [2, 9, 10, 14]]),
    # Nothing is shared: a short beam's rows are copied.
    ([10, 40, 40, 40], [[0, 4, 5], [1, 6, 7], [2, 9, 8], [3, 11, 10]])])
def test_more_children_of_a_short_beam(ops, lens, table):
    """A choice of fewer than its width names beam 0 as the rest's parent, which may have ended
    before the others: its children take no page that another child's history lies in."""
    gen = torch.Generator().manual_seed(3)
    pages = ops.Pages(*(_normal(gen, 15, 2, 16, 64, dtype=BF).cuda() for _ in "kv"))
    times = torch.rand(15, 16, generator=gen).cuda()
    table = torch.tensor(table, dtype=torch.int32).cuda()
    lens = torch.tensor(lens).cuda()
    read = lambda t, n: ops.paged_read(pages, t, lens=n, length=64, k_times=times)  # noqa: E731
    before = read(table, lens)
    for parents in ([0, 1, 0, 0], [1, 0, 0, 0]):
        chosen = torch.tensor(parents).cuda()
        new, new_lens = ops.beam_reorder(table, lens, chosen[None], [pages], k_times=times)
        after = read(new, new_lens)
        for x, y in zip(before, after):
            assert torch.equal(y, x[chosen])
        assert new_lens.tolist() == lens[chosen].tolist()
        table, lens, before = new, new_lens, after


def test_offsets_of_no_walk(ops):
    """Offsets that are not walks' write nothing, and what is read for their rows is 0."""
    pages = ops.Pages.empty(4, 16, 1, 8)
    for x in pages[:2]:
        x.fill_(1.0)
    table = torch.arange(4, dtype=torch.int32).cuda().view(2, 2)
    rows = torch.full((6, 1, 8), 2.0, dtype=BF, device="cuda")
    far = (1 << 63) - 1
    for offsets in ([-far, -far, -far], [-far, 0, 0], [far, far, far], [-far, -far, 6], [5, -9, far]):
        offsets = torch.tensor(offsets).cuda()
        k, v = ops.paged_read(pages, table, offsets=offsets, rows=6)
        assert ((k == 0) | (k == 1)).all() and torch.equal(k, v)
        if offsets[1] != -9:
            ops.paged_write(pages, table, torch.tensor([7, 8]).cuda(), rows, rows, offsets=offsets)
            assert (k == 0).all() and (pages.k == 1).all() and (pages.v == 1).all()


# ---- together ---------------------------------------------------------------------------------------
def _model(gen, nodes, heads, kv_heads, dim):
    """A layer of its own for a walk's last node: rows of q, k, v, and logits of an output."""
    return {n: _normal(gen, nodes, h, dim, dtype=BF) for n, h in
            (("q", heads), ("k", kv_heads), ("v", kv_heads))} | {
                "head": _normal(gen, heads * dim, nodes, std=0.3)}


@pytest.mark.parametrize("eight", [False, True])
def test_a_forecast(ops, eight):
    """Prompts into pages, then steps, choices and reorderings: every beam's history and scores are
    those of a model that recomputes each from its own events."""
    gen = torch.Generator().manual_seed(21)
    nodes, heads, kv_heads, dim, beams, steps, rows = 50, 4, 2, 32, 4, 22, 16
    prompts = [13, 16, 1]
    groups, total = len(prompts), len(prompts) * beams
    m = _model(gen, nodes, heads, kv_heads, dim)
    dev = {n: x.cuda() for n, x in m.items()}
    pool = Pool(ops, total, 64, kv_heads, dim, rows=rows, eight=eight)
    walks = [torch.randint(1, nodes, (n,), generator=gen).tolist() for n in prompts]
    held = [torch.tensor(w[:-1], dtype=torch.int64) for w in walks]  # the last is the first step's
    starts = torch.full((total,), -1)
    starts[::beams] = 0
    length = max(prompts)
    padded = torch.zeros(total, length, dtype=torch.int64)
    counts = torch.zeros(total, dtype=torch.int64)
    for g, h in enumerate(held):
        padded[g * beams, :len(h)] = h
        counts[g * beams] = len(h)
    at = padded.cuda()
    ops.paged_write(pool.pages, pool.table, starts.cuda(), dev["k"][at], dev["v"][at],
                    counts=counts.cuda())
    lens = torch.tensor([len(h) for h in held]).repeat_interleave(beams)
    spread = torch.zeros(groups, beams, dtype=torch.int64).cuda()
    table, lens = ops.beam_reorder(pool.table, lens.cuda(), spread, [pool.pages])
    last = torch.tensor([w[-1] for w in walks]).repeat_interleave(beams).cuda()
    scores = torch.full((groups, beams), -math.inf, device="cuda")
    scores[:, 0] = 0
    ended = torch.zeros(groups, beams, dtype=torch.bool, device="cuda")
    histories = [[list(w) for _ in range(beams)] for w in walks]
    kept = {n: pool.held(m[n]) for n in "kv"}

    def plain(history):
        """Logits after a history, in float64, with the output rounded as the step's is."""
        i = torch.tensor(history)
        o = wf.attention(m["q"][i[-1:]].double(), kept["k"][i], kept["v"][i],
                         wf.documents("causal", [1], [len(i)]), dtype=BF)["out"]
        return o

    for _ in range(steps):
        live = torch.where(ended.flatten(), -1, lens)
        out = ops.paged_attention_step(dev["q"][last], dev["k"][last], dev["v"][last], pool.pages,
                                       table, live)
        for g in range(groups):
            for b in range(beams):
                if not ended[g, b] and torch.isfinite(scores[g, b]):
                    wf.check(f"out[{g}, {b}]", out[g * beams + b][None], *plain(histories[g][b]))
        lens = lens + (live >= 0)
        logits = (out.flatten(1).float() @ dev["head"]).view(groups, beams, nodes)
        choice = ops.beam_select(logits, scores, beams, ended=ended, end_token=0)
        for g in range(groups):
            s, t, p, e = sf.choice(logits[g].cpu().double(), scores[g].cpu(), beams, ended[g].cpu(), 0)
            assert choice.tokens[g].tolist() == t and choice.parents[g].tolist() == p
            histories[g] = [histories[g][a] + ([] if ended[g, a] else [x]) for a, x in zip(p, t)]
        table, lens = ops.beam_reorder(table, lens, choice.parents, [pool.pages])
        scores, ended, last = choice.scores, choice.ended, choice.tokens.flatten()
    assert any(len(h) > 16 for g in histories for h in g)


def test_prompts_over_pages(ops):
    """Pages read back are keys of a pass over new events, as walk_attention takes them."""
    gen = torch.Generator().manual_seed(31)
    held, new, heads, kv_heads, dim = [20, 0, 70], [5, 9, 33], 4, 2, 64
    pool = Pool(ops, 3, 128, kv_heads, dim, rows=32, eight=True)
    k, v = (_normal(gen, 3, 70, kv_heads, dim, dtype=BF) for _ in range(2))
    ops.paged_write(pool.pages, pool.table, None, k.cuda(), v.cuda(), counts=torch.tensor(held).cuda())
    q, nk, nv = (_normal(gen, sum(new), h, dim, dtype=BF) for h in (heads, kv_heads, kv_heads))
    offsets = torch.tensor([0] + new).cumsum(0)
    ops.paged_write(pool.pages, pool.table, torch.tensor(held).cuda(), nk.cuda(), nv.cuda(),
                    offsets=offsets.cuda())
    whole = [a + b for a, b in zip(held, new)]
    k_offsets = torch.tensor([0] + whole).cumsum(0)
    keys, values = ops.paged_read(pool.pages, pool.table, offsets=k_offsets.cuda(), rows=sum(whole))
    mask = ops.WalkMask.packed(offsets.cuda(), sum(new), k_offsets=k_offsets.cuda(), k_rows=sum(whole))
    out = ops.walk_attention(q.cuda(), keys, values, mask)
    rows = []
    for w in range(3):
        part = slice(int(offsets[w]), int(offsets[w + 1]))
        rows.append([pool.held(torch.cat([x[w, :held[w]], y[part]])) for x, y in ((k, nk), (v, nv))])
    want = wf.attention(q.double(), torch.cat([r[0] for r in rows]), torch.cat([r[1] for r in rows]),
                        wf.documents("causal", new, whole), dtype=BF)["out"]
    wf.check("out", out, *want)


# ---- how they are called ------------------------------------------------------------------------------
def _served(ops, seed, eight=True):
    gen = torch.Generator().manual_seed(seed)
    pool = Pool(ops, 8, 640, 2, 64, rows=16, eight=eight, seed=seed, times=True)
    lens = torch.tensor([600, 3, 40, 17, 0, 630, 99, 16]).cuda()
    kc, vc = (_normal(gen, 8, 640, 2, 64, dtype=BF).cuda() for _ in range(2))
    t = torch.rand(8, 640, generator=gen).cuda()
    ops.paged_write(pool.pages, pool.table, None, kc, vc, counts=lens, times=t, k_times=pool.k_times)
    x = {n: _normal(gen, 8, h, 64, dtype=BF).cuda() for n, h in (("q", 4), ("k", 2), ("v", 2))}
    slopes, now = torch.rand(4, generator=gen).cuda(), torch.rand(8, generator=gen).cuda() + 2
    head = _normal(gen, 256, 5000).cuda()
    scores = -torch.rand(2, 4, generator=gen).cuda()
    held = [(y, y.clone()) for y in (*pool.pages, pool.k_times) if y is not None]

    def run():
        for y, was in held:  # a run writes rows and moves some: equal inputs are equal pages as well
            y.view(torch.uint8).copy_(was.view(torch.uint8))
        out = ops.paged_attention_step(x["q"], x["k"], x["v"], pool.pages, pool.table, lens,
                                       slopes=slopes, times=now, k_times=pool.k_times)
        choice = ops.beam_select((out.flatten(1).float() @ head).view(2, 4, -1), scores, 4)
        table, new = ops.beam_reorder(pool.table, lens, choice.parents, [pool.pages],
                                      k_times=pool.k_times)
        read = ops.paged_read(pool.pages, table, lens=new, length=64, k_times=pool.k_times)
        return [out, *choice, table, new, *read]

    return x, pool, run


def _same(a, b):
    return all(torch.equal(_raw(x) if x.is_floating_point() else x,
                           _raw(y) if y.is_floating_point() else y) for x, y in zip(a, b))


@pytest.mark.parametrize("eight", [False, True])
def test_equal_inputs_give_equal_bits(ops, eight):
    _, _, run = _served(ops, 5, eight)
    first = run()
    for _ in range(3):
        assert _same(run(), first)


def test_in_a_graph(ops):
    x, pool, run = _served(ops, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    gen = torch.Generator().manual_seed(7)
    for _ in range(4):
        for name, y in x.items():
            y.copy_(_normal(gen, *y.shape, dtype=BF))
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in held]
        assert _same(run(), got)


def test_on_another_stream(ops):
    _, _, run = _served(ops, 8)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert _same(got, want)


def test_layouts(ops):
    """Keys and values of one pool, slices of one projection, tables and lengths of other layouts."""
    gen = torch.Generator().manual_seed(9)
    both = torch.zeros(40, 2, 2, 16, 64, dtype=BF, device="cuda")
    pages = ops.Pages(both[:, 0], both[:, 1])
    ids = torch.randperm(40, generator=gen).int().view(4, 10).cuda()
    qkv = _normal(gen, 4, 12, 64, dtype=BF).cuda()
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    lens = torch.tensor([33, 5, 159, -1])
    rows = _normal(gen, 4, 159, 4, 64, dtype=BF).cuda()
    for table in (ids, ids.t().contiguous().t(), torch.cat([ids, ids], 1)[:, :10]):
        ops.paged_write(pages, table, None, rows[:, :, :2], rows[:, :, 2:])
        for n in (lens.cuda(), lens.int().cuda(), torch.stack([lens, lens], 1).cuda()[:, 0]):
            out = ops.paged_attention_step(q, k, v, pages, table, n)
            for b, m in enumerate(lens.tolist()):
                if m < 0:
                    assert (out[b] == 0).all()
                    continue
                ks, vs = (torch.cat([r[b, :m], x[b:b + 1]]).cpu().double()
                          for r, x in ((rows[:, :, :2], k), (rows[:, :, 2:], v)))
                want = wf.attention(q[b:b + 1].cpu().double(), ks, vs,
                                    wf.documents("causal", [1], [m + 1]), dtype=BF)["out"]
                wf.check("out", out[b:b + 1], *want)
    odd = torch.zeros(4, 2, 65, dtype=BF, device="cuda")[:, :, 1:]  # rows that are not 16-byte pieces
    odd.copy_(k)
    assert torch.equal(ops.paged_attention_step(q, odd, v, pages, ids, lens.cuda()),
                       ops.paged_attention_step(q, k, v, pages, ids, lens.cuda()))


def test_nothing_at_all(ops):
    pages = ops.Pages.empty(0, 16, 2, 64, dtype=E8)
    rows = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    table = torch.zeros(0, 0, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    ops.paged_write(pages, table, none, rows, rows, offsets=torch.zeros(1, dtype=torch.int64).cuda())
    out = ops.paged_attention_step(rows, rows, rows, pages, table, none)
    assert out.shape == (0, 2, 64)
    new = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    out = ops.paged_attention_step(new, new, new, pages, table.new_zeros(3, 4),
                                   torch.tensor([-1, 0, 5]).cuda())
    assert (out[0] == 0).all() and torch.isnan(out[1:]).all()
    got = ops.beam_select(torch.zeros(0, 2, 9, device="cuda"), torch.zeros(0, 2, device="cuda"), 3)
    assert got.scores.shape == (0, 3)
    got = ops.paged_read(pages, table.new_zeros(2, 3), lens=torch.tensor([2, 5]).cuda(), length=4,
                         k_times=torch.zeros(0, 16, device="cuda"))
    assert all((x == 0).all() for x in got) and got[2].shape == (2, 4)
    a, b = ops.beam_reorder(table, none, torch.zeros(0, 2, dtype=torch.int64).cuda(), [pages])
    assert a.shape == (0, 0) and b.shape == (0,)


def test_gradients_are_refused(ops):
    gen = torch.Generator().manual_seed(1)
    pool = Pool(ops, 2, 32, 2, 64)
    x = _normal(gen, 2, 2, 64, dtype=BF).cuda().requires_grad_()
    lens = torch.zeros(2, dtype=torch.int64).cuda()
    out = ops.paged_attention_step(x, x, x, pool.pages, pool.table, lens)
    with pytest.raises(RuntimeError, match="has no gradient"):
        out.sum().backward()
    with pytest.raises(ValueError, match="has no gradient"):
        ops.paged_write(pool.pages, pool.table, None, x[:, None], x[:, None])
    with torch.no_grad():
        ops.paged_write(pool.pages, pool.table, None, x[:, None], x[:, None])
    logits = torch.zeros(1, 2, 9, device="cuda", requires_grad=True)
    got = ops.beam_select(logits, torch.zeros(1, 2, device="cuda"), 2)
    with pytest.raises(RuntimeError, match="has no gradient"):
        got.scores.sum().backward()
    before = pool.pages.k._version
    ops.paged_attention_step(x.detach(), x.detach(), x.detach(), pool.pages, pool.table, lens)
    assert pool.pages.k._version > before


def test_refusals(ops):
    pool = Pool(ops, 2, 32, 2, 64)
    p, table = pool.pages, pool.table
    new = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
    lens = torch.zeros(2, dtype=torch.int64, device="cuda")
    step = lambda *a, **k: ops.paged_attention_step(*a, **k)  # noqa: E731
    for call, message in (
            (lambda: step(new, new, new, p, table.long(), lens), "int32"),
            (lambda: step(new, new, new, p, table[:1], lens), "row for each"),
            (lambda: step(new.half(), new.half(), new.half(), p, table, lens), "pages' type"),
            (lambda: step(new, new, new, p, table.cpu(), lens), "on the GPU"),
            (lambda: step(new, new, new, ops.Pages(p.k, p.v, lens, lens), table, lens), "have scales"),
            (lambda: step(new, new, new, ops.Pages(p.k.transpose(1, 2), p.v.transpose(1, 2)), table,
                          lens), "contiguous|heads"),
            (lambda: step(new, new, new, ops.Pages(p.k[:1].expand_as(p.v), p.v), table, lens),
             "share memory"),
            (lambda: step(new, new, new, ops.Pages(p.k, p.k), table, lens), "share memory"),
            (lambda: step(new, new, new, ops.Pages.empty(4, 24, 2, 64), table, lens), "power of two"),
            (lambda: step(new[..., :24].contiguous(), new[..., :24].contiguous(),
                          new[..., :24].contiguous(), ops.Pages.empty(4, 16, 2, 24, dtype=E8), table,
                          lens), "multiple of 16"),
            (lambda: step(new, new, new, p, table, lens, times=torch.zeros(2).cuda()), "go together"),
            (lambda: ops.paged_write(p, table, None, new, new), "walks, length"),
            (lambda: ops.paged_write(p, table, None, new[None], new[None]), "walks, length"),
            (lambda: ops.paged_write(p, table, None, new[:, None], new[:, None], times=lens.float()),
             "go together"),
            (lambda: ops.paged_read(p, table), "either"),
            (lambda: ops.paged_read(p, table, lens=lens, length=3, offsets=lens, rows=1), "either"),
            (lambda: ops.paged_read(p, table, lens=lens, length=3, dtype=SF), "pages' type"),
            (lambda: ops.paged_read(p, table, lens=lens, length=-1), "rows"),
            (lambda: ops.beam_select(new, torch.zeros(2, 2).cuda(), 33), "1 to 32"),
            (lambda: ops.beam_select(new, torch.zeros(2, 3).cuda(), 2), "shape"),
            (lambda: ops.beam_select(new, torch.zeros(2, 2).cuda(), 2, end_token=64), "a node"),
            (lambda: ops.beam_select(new, torch.zeros(2, 2).cuda(), 2,
                                     ended=torch.zeros(2, 2, dtype=torch.bool).cuda()), "end_token"),
            (lambda: ops.beam_reorder(table, lens, lens[None], []), "at least one"),
            (lambda: ops.beam_reorder(table, lens, lens, [p]), "groups, beams"),
            (lambda: ops.beam_reorder(table, lens[:1], lens[None], [p]), "shape"),
            (lambda: ops.beam_reorder(table, lens, lens[None], [p, ops.Pages.empty(4, 16, 2, 64)]),
             "pages alike")):
        with pytest.raises(ValueError, match=message):
            call()


def test_example():
    """The forecast of examples/walk_model.py runs: paths of nodes, distinct, best first."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "walk_model.py")
    spec = importlib.util.spec_from_file_location("walk_model", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    at, times, lens = example.sample_walks(100, 20, 24, 20, seed=1)
    model = example.WalkModel(100).cuda()
    nodes, scores = example.forecast(model, at, times, lens, 5, beams=3)
    assert nodes.shape == (at.shape[0], 3, 5) and ((nodes >= 0) & (nodes < 100)).all()
    assert torch.isfinite(scores).all() and (scores[:, :-1] >= scores[:, 1:]).all()
    assert all(len(set(map(tuple, x))) == 3 for x in nodes.tolist())
