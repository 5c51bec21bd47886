"""Pages and beam search where rounding, masks and lengths are extreme, against their formulas in
float64 (tests/serving_formulas.py, tests/walk_formulas.py, tests/beam_orders.py)."""
import math
import random

import pytest
import torch

from tests import beam_orders as bo
from tests import walk_formulas as wf
from tests.test_cpu_beam_orders import TWO_SHORT
from tests.test_gpu_serving import (BF, DTYPES, E8, HF, SF, SIZES, Pool, _choose,  # noqa: F401
                                    _normal, _step, ops)

pytestmark = pytest.mark.gpu


# ---- one event over pages -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("cached,capacity", [(100, 128), (700, 768)])
def test_step_of_small_weights(ops, dtype, eight, cached, capacity):  # noqa: F811
    """A key that takes nearly all of the weight and has no values, and many of weights that are
    subnormal numbers of float16 relative to it: the output is theirs, as near as a computation in
    float32 rounded once has it."""
    dim = 64
    pool = Pool(ops, 1, capacity, 1, dim, dtype=dtype, eight=eight)
    # scores are k[..., 0]: q is 8 there and the scale 1 / 8
    k = torch.zeros(1, cached + 1, 1, dim)
    k[0, 1:, 0, 0] = -15.5  # 3.11 times float16's smallest number
    v = torch.full((1, cached + 1, 1, dim), 100.0)
    v[0, 0] = 0.0
    q = torch.zeros(1, 2, dim)
    q[..., 0] = 8.0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    ops.paged_write(pool.pages, pool.table, None, k[:, :-1].cuda(), v[:, :-1].cuda())
    out = ops.paged_attention_step(q.cuda(), k[:, -1].cuda(), v[:, -1].cuda(), pool.pages, pool.table,
                                   torch.tensor([cached]).cuda())
    held = [pool.held(x[0]) for x in (k, v)]
    o, bound = wf.attention(q.double(), *held, wf.documents("causal", [1], [cached + 1]))["out"]
    # besides float32's: the output's rounding; weights in two parts, of 8 bits each at least, or of
    # 2^-39 of the largest weight where the type has no smaller numbers
    bound = bound + (wf.U[dtype] + 2.0 ** -16) * o.abs() + cached * 2.0 ** -39 * 100.0
    wf.check("out", out, o, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 24, 40, 72, 104, 128])
def test_step_over_infinite_keys(ops, dtype, dim):  # noqa: F811
    """A key with an infinity against a query of the other sign has weight 0, at every head size."""
    gen = torch.Generator().manual_seed(dim)
    pool = Pool(ops, 1, 64, 1, dim, dtype=dtype)
    q, k, v = (_normal(gen, 1, n, 1, dim, dtype=dtype) for n in (1, 41, 41))
    q[..., 0] = 0.5 + q[..., 0].abs()
    k[0, 7, 0, 0] = -torch.inf
    ops.paged_write(pool.pages, pool.table, None, k[:, :-1].cuda(), v[:, :-1].cuda())
    out = ops.paged_attention_step(q[0].cuda(), k[:, -1].cuda(), v[:, -1].cuda(), pool.pages,
                                   pool.table, torch.tensor([40]).cuda())
    seen = torch.arange(41) != 7
    k[0, 7] = 0  # not seen: the formula's -inf
    want = wf.attention(q[0].double(), k[0].double(), v[0].double(), [(40, 1, 41, seen[None])],
                        dtype=dtype)["out"]
    wf.check("out", out, *want)


@pytest.mark.parametrize("dtype,eight", [(BF, False), (HF, True), (SF, False)])
def test_step_of_a_long_walk_in_a_large_batch(ops, dtype, eight):  # noqa: F811
    """Enough walks and heads for every place that a device has, several times, and one walk that is
    longer than they are."""
    _step(ops, dtype, [(7 * i) % 20 - 1 for i in range(520)] + [550], 560, 8, 8, 16, eight=eight)
    _step(ops, dtype, [(7 * i) % 20 - 1 for i in range(520)], 520, 8, 8, 16, eight=eight)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("cached,capacity", [(100, 128), (700, 768)])
@pytest.mark.parametrize("low", ["-inf", "lowest"])
def test_step_of_masked_distances(ops, dtype, eight, cached, capacity, low):  # noqa: F811
    """A bias that masks some distances, those of the nearest events, and all of them: -inf leaves
    nothing and the output is 0, the lowest finite value leaves equal weights."""
    low = -math.inf if low == "-inf" else torch.finfo(SF).min
    gen = torch.Generator().manual_seed(cached)
    pool = Pool(ops, 1, capacity, 2, 64, dtype=dtype, eight=eight)
    q, k, v = (_normal(gen, 1, m, n, 64, dtype=dtype) for m, n in
               ((1, 4), (cached + 1, 2), (cached + 1, 2)))
    ops.paged_write(pool.pages, pool.table, None, k[:, :-1].cuda(), v[:, :-1].cuda())
    held = [pool.held(x[0]) for x in (k, v)]
    ids = ops.distance_buckets(8, 64, device="cpu")
    for masked in ([0], [0, 1, 2, 3, 4], [7], [2, 6], range(8)):
        table = _normal(gen, 4, 8)
        table[:, list(masked)] = low
        table[0] = 1.0  # a head that sees everything
        out = ops.paged_attention_step(q[0].cuda(), k[:, -1].cuda(), v[:, -1].cuda(), pool.pages,
                                       pool.table, torch.tensor([cached]).cuda(),
                                       bias_table=table.cuda(), buckets=ids.cuda())
        want = wf.attention(q[0].double(), *held, wf.documents("causal", [1], [cached + 1]),
                            table=table.double(), buckets=ids, dtype=dtype)["out"]
        wf.check("out", out, *want)
        if low == -math.inf and len(masked) == 8:
            assert (out[:, 1:] == 0).all()


def test_pages_as_records(ops):  # noqa: F811
    """Keys, values and scales of a page in one record hold what they do in memory of their own;
    scales of one memory are refused."""
    gen = torch.Generator().manual_seed(5)
    heads, rows, dim, count = 2, 32, 64, 9
    sizes = [heads * rows * dim] * 2 + [heads * rows] * 2
    pool = torch.zeros(count, sum(sizes), dtype=torch.uint8, device="cuda")
    k, v, ks, vs = pool.split(sizes, 1)
    shape = (heads, rows)
    record = ops.Pages(*(x.view(E8).unflatten(1, (*shape, dim)) for x in (k, v)),
                       *(x.unflatten(1, shape) for x in (ks, vs)))
    whole = ops.Pages(*(None if x is None else x.contiguous() for x in record))
    table = torch.randperm(count, generator=gen).int().view(3, 3).cuda()
    lens = torch.tensor([90, 33, 64]).cuda()
    kc, vc = (_normal(gen, 3, 90, heads, dim, dtype=BF).cuda() for _ in "kv")
    q, new_k, new_v = (_normal(gen, 3, n, dim, dtype=BF).cuda() for n in (4, heads, heads))
    got = []
    for pages in (record, whole):
        ops.paged_write(pages, table, None, kc, vc, counts=lens)
        out = ops.paged_attention_step(q, new_k, new_v, pages, table, lens)
        new, n = ops.beam_reorder(table, lens, torch.tensor([[1, 1, 0]]).cuda(), [pages])
        got.append((out, *ops.paged_read(pages, new, lens=n, length=90)))
    for x, y in zip(*got):
        assert torch.equal(x, y)
    for x, y in zip(record, whole):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    one = whole._replace(v_scale=whole.k_scale)
    for call in (lambda: ops.paged_write(one, table, None, kc, vc),
                 lambda: ops.paged_read(one, table, lens=lens, length=4),
                 lambda: ops.paged_attention_step(q, new_k, new_v, one, table, lens),
                 lambda: ops.beam_reorder(table, lens, torch.tensor([[1, 1, 0]]).cuda(), [one])):
        with pytest.raises(ValueError, match="share memory"):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("capacity", [128, 768])
def test_step_over_infinite_values(ops, dtype, dim, capacity):  # noqa: F811
    """An infinity among the values that are seen makes its column that infinity, whatever its weight is
    and wherever it lies, beside rows that are not seen too; other columns are as without it."""
    gen = torch.Generator().manual_seed(dim)
    lens, first = [100, 17, 64, 0, 40, 95], [0, 5, 33, 0, 40, 50]
    walks = len(lens)
    pool = Pool(ops, walks, capacity, 1, dim, dtype=dtype)
    q, k, v = (_normal(gen, walks, m, 1, dim, dtype=dtype) for m in (1, 101, 101))
    # the new event, the first and the last one that are cached; -26 and -40 are weights of 2^-38 and 2^-58
    spots = [(w, j, c) for w in range(walks) for c, j in enumerate((lens[w], first[w], lens[w] - 1))
             if j >= first[w]] + [(0, 50, 3), (0, 51, 4)]
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[0, 50, 0, 0], k[0, 51, 0, 0] = -26.0 * dim ** 0.5, -40.0 * dim ** 0.5

    def run(x):
        ops.paged_write(pool.pages, pool.table, None, k.cuda(), x.cuda(),
                        counts=torch.tensor(lens).cuda())
        new_k, new_v = (torch.stack([y[w, n] for w, n in enumerate(lens)]).cuda() for y in (k, x))
        return ops.paged_attention_step(q[:, 0].cuda(), new_k, new_v, pool.pages, pool.table,
                                        torch.tensor(lens).cuda(), first=torch.tensor(first).cuda())

    fine = run(v)
    assert torch.isfinite(fine).all()
    for sign in (1, -1):
        x, want = v.clone(), fine.clone()
        for w, j, c in spots:
            x[w, j, 0, c] = want[w, 0, c] = sign * math.inf
        assert torch.equal(run(x), want)


# ---- choice among beams -----------------------------------------------------------------------------
LOWS = [-(10.0 ** n) for n in range(3, 38)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,beams,nodes,width", [(2, 3, 9000, 8), (1, 2, 70001, 5)])
def test_choice_of_finitely_masked_nodes(ops, dtype, groups, beams, nodes, width):  # noqa: F811
    """Masks of any size over whole chunks beside ordinary ones, and over whole rows."""
    gen = torch.Generator().manual_seed(nodes)
    x = _normal(gen, groups, beams, nodes, dtype=dtype, std=3.0)
    scores = -torch.rand(groups, beams, generator=gen)
    for low in LOWS:
        if low < torch.finfo(dtype).min:
            break
        y = x.clone()
        y[..., 4096:] = low
        _choose(ops, y, scores, width)
        y = torch.full_like(x, low)
        y[..., 8200:8300] = x[..., 8200:8300]
        _choose(ops, y, scores, width)
        _choose(ops, torch.full_like(x, low), scores, width)
        _choose(ops, torch.full_like(x, -low), scores, width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,beams,nodes,width", SIZES)
@pytest.mark.parametrize("far", [100.0, 1e3, 3e3, 1e4, -1e4, 6e4, 1e6, -1e6, 1e8, -1e8])
def test_choice_far_from_zero(ops, dtype, groups, beams, nodes, width, far):  # noqa: F811
    """Rows shifted by a constant choose as they do around zero."""
    if abs(far) > torch.finfo(dtype).max:
        return
    gen = torch.Generator().manual_seed(nodes)
    x = (_normal(gen, groups, beams, nodes, std=3.0) + far).to(dtype)
    _choose(ops, x, -torch.rand(groups, beams, generator=gen), width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nodes,width", [(100, 8), (9000, 5), (50021, 32)])
@pytest.mark.parametrize("score", [-1e20, -1e30, -3e38])
def test_choice_among_sums_that_round_to_one(ops, dtype, nodes, width, score):  # noqa: F811
    """Scores, or a row's maximum, next to which the other logits are lost: equal sums come by their
    beam, then by their node, whatever their logits are."""
    gen = torch.Generator().manual_seed(nodes)
    x = _normal(gen, 2, 3, nodes, dtype=dtype, std=3.0)
    x[0, 0, 2:] = -math.inf  # the beam that counts has two ways on
    scores = torch.tensor([[-0.5, score, score], [score, score, score]])
    got = ops.beam_select(x.cuda(), scores.cuda(), width)
    rest = list(range(width))
    best = [0, 1] if x[0, 0, 0] >= x[0, 0, 1] else [1, 0]
    assert got.tokens.tolist() == [best + rest[:-2], rest]
    assert got.parents.tolist() == [[0, 0] + [1] * (width - 2), [0] * width]
    assert (got.scores[:, 2:].cpu() == torch.tensor(score)).all()
    if abs(score) <= torch.finfo(dtype).max:
        x[..., nodes - 3] = -score  # of float32 and bfloat16: the rest is 1e20 and more below
        got = ops.beam_select(x.cuda(), torch.zeros(2, 3).cuda(), width)
        assert got.tokens.tolist() == [[nodes - 3] * 3 + rest[:2] + rest[:width - 5]] + [
            [nodes - 3] * 3 + rest[:width - 3]]
        assert got.parents.tolist() == [[0, 1, 2, 0, 0] + [1] * (width - 5),
                                        [0, 1, 2] + [0] * (width - 3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nodes", [3, 10, 100, 777, 4097, 50021, 70001])
def test_scores_are_rounded_once(ops, dtype, nodes):  # noqa: F811
    """Rows of zeros have sums that float32 holds exactly: what is left is the result's rounding."""
    scores = -20 * torch.rand(3, 4, generator=torch.Generator().manual_seed(nodes))
    got = ops.beam_select(torch.zeros(3, 4, nodes, dtype=dtype).cuda(), scores.cuda(), 1)
    want = scores.double().amax(1) - math.log(nodes)
    assert ((got.scores[:, 0].cpu().double() - want).abs() <= want.abs() * (2.0 ** -24 + 1e-12)).all()


# ---- reordering ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("table,lens,parents,page_rows", [
    TWO_SHORT,
    ([[0, 4, 5], [1, 6, 7], [2, 8, 9], [2, 8, 10]], [10, 12, 40, 40], [0, 0, 1, 1], 16),
    # three short parents, and dropped beams of one past and of another
    ([[0, 1], [2, 3], [4, 5], [6, 7], [6, 8], [9, 10]], [10, 12, 14, 20, 20, 30], [2, 1, 0, 0, 1, 2],
     16)])
def test_children_of_several_short_beams(ops, table, lens, parents, page_rows):  # noqa: F811
    """Rows of different parents never go to one page."""
    gen = torch.Generator().manual_seed(3)
    pages = ops.Pages(*(_normal(gen, 16, 2, page_rows, 64).cuda() for _ in "kv"))
    times = torch.rand(16, page_rows, generator=gen).cuda()
    length = len(table[0]) * page_rows
    read = lambda t, n: ops.paged_read(pages, t, lens=n, length=length, k_times=times)  # noqa: E731
    rows, _, _ = bo.order(table, lens, parents, page_rows)
    table, lens, chosen = torch.tensor(table).int().cuda(), torch.tensor(lens).cuda(), parents
    before = read(table, lens)
    new, new_lens = ops.beam_reorder(table, lens, torch.tensor([parents]).cuda(), [pages],
                                     k_times=times)
    assert new.tolist() == rows and new_lens.tolist() == lens[chosen].tolist()
    for x, y in zip(before, read(new, new_lens)):
        assert torch.equal(y, x[chosen])


def test_any_parents(ops):  # noqa: F811
    """Searches whose parents are any beams, those that ended early among them: tables are the
    formula's, and every beam keeps its history."""
    pages = ops.Pages.empty(64, 16, 1, 8, dtype=SF)
    for seed in range(12):
        gen = torch.Generator().manual_seed(seed)

        def orders(table, lens, parents, page_rows):
            want, want_lens, _ = bo.order(table, lens, parents, page_rows)
            t, n = torch.tensor(table).int().cuda(), torch.tensor(lens).cuda()
            for x in pages[:2]:
                x.copy_(torch.randn(x.shape, generator=gen))
            before = ops.paged_read(pages, t, lens=n, length=128)
            new, new_lens = ops.beam_reorder(t, n, torch.tensor([parents]).cuda(), [pages])
            assert new.tolist() == want and new_lens.tolist() == want_lens
            for x, y in zip(before, ops.paged_read(pages, new, lens=new_lens, length=128)):
                assert torch.equal(y, x[parents])
            return want, want_lens, None

        for _ in bo.search(random.Random(seed), orders, 16):
            pass
