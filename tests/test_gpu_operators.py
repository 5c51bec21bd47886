"""Operators on walks against their formulas in float64 (tests/walk_formulas.py)."""
import math

import pytest
import torch

from tests import walk_formulas as wf

pytestmark = pytest.mark.gpu

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
DTYPES = [BF, HF, SF]


@pytest.fixture(scope="module")
def ops():
    from temporal_random_walk import operators
    return operators


def _normal(gen, *shape, dtype=SF, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def _offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0)


class Batch:
    """A packed batch on the CPU with all terms of a score, and its device copies."""

    def __init__(self, q_lens, k_lens=None, *, heads=2, kv_heads=2, dim=64, dtype=BF, kind="causal",
                 prefix=None, softcap=0.0, buckets=None, num_buckets=0, slopes=False, times=False,
                 scale=None, seed=0):
        gen = torch.Generator().manual_seed(seed)
        k_lens = q_lens if k_lens is None else k_lens
        self.q_lens, self.k_lens, self.kind, self.prefix = q_lens, k_lens, kind, prefix
        self.dtype, self.scale, self.softcap = dtype, scale, softcap
        nq, nk = sum(q_lens), sum(k_lens)
        self.q = _normal(gen, nq, heads, dim, dtype=dtype)
        self.k = _normal(gen, nk, kv_heads, dim, dtype=dtype)
        self.v = _normal(gen, nk, kv_heads, dim, dtype=dtype)
        self.d_out = _normal(gen, nq, heads, dim, dtype=dtype)
        self.buckets = buckets
        self.table = _normal(gen, heads, num_buckets) if num_buckets else None
        self.slopes = torch.rand(heads, generator=gen) * 0.2 if slopes else None
        self.q_times = self.k_times = None
        if times:
            self.k_times = torch.rand(nk, generator=gen).cumsum(0)
            self.q_times = (self.k_times.clone() if k_lens == q_lens
                            else torch.rand(nq, generator=gen).cumsum(0))

    def reference(self, backward=True):
        d = lambda x: None if x is None else x.double()  # noqa: E731
        return wf.attention(
            d(self.q), d(self.k), d(self.v),
            wf.documents(self.kind, self.q_lens, self.k_lens, self.prefix), scale=self.scale,
            softcap=self.softcap, table=d(self.table), buckets=self.buckets,
            slopes=d(self.slopes), q_times=d(self.q_times), k_times=d(self.k_times),
            d_out=d(self.d_out) if backward else None, dtype=self.dtype)

    def mask(self, ops):
        own = self.k_lens == self.q_lens
        return ops.WalkMask.packed(
            _offsets(self.q_lens).cuda(), sum(self.q_lens),
            k_offsets=None if own else _offsets(self.k_lens).cuda(),
            k_rows=None if own else sum(self.k_lens), kind=self.kind,
            prefix=None if self.prefix is None else torch.tensor(self.prefix).cuda())

    def terms(self, table=None):
        c = lambda x: None if x is None else x.cuda()  # noqa: E731
        return dict(scale=self.scale, softcap=self.softcap,
                    bias_table=c(self.table) if table is None else table, buckets=c(self.buckets),
                    slopes=c(self.slopes), times=c(self.q_times),
                    k_times=None if self.q_times is None else c(self.k_times))

    def run(self, ops, backward=True):
        q, k, v = (x.cuda().requires_grad_(backward) for x in (self.q, self.k, self.v))
        table = None if self.table is None else self.table.cuda().requires_grad_(backward)
        out = ops.walk_attention(q, k, v, self.mask(ops), **self.terms(table))
        res = {"out": out}
        if backward:
            out.backward(self.d_out.cuda())
            res.update(d_q=q.grad, d_k=k.grad, d_v=v.grad)
            if table is not None:
                res["d_table"] = table.grad
        return res


def _check(ops, batch, backward=True):
    got, want = batch.run(ops, backward), batch.reference(backward)
    assert got.keys() == want.keys()
    for name, (value, bound) in want.items():
        wf.check(name, got[name], value, bound)


LENS = [1, 0, 2, 31, 32, 33, 5, 64, 65, 1, 1, 127, 0, 128, 129, 20, 200]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["causal", "full", "prefix"])
def test_documents_of_many_lengths(ops, dtype, kind):
    prefix = [(7 * w) % (n + 3) for w, n in enumerate(LENS)] if kind == "prefix" else None
    _check(ops, Batch(LENS, heads=3, kv_heads=1, dtype=dtype, kind=kind, prefix=prefix))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 72, 80, 96, 104, 128])
def test_head_sizes(ops, dtype, dim):
    _check(ops, Batch([70, 3, 150], dim=dim, dtype=dtype, seed=dim))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["causal", "full", "prefix"])
def test_queries_over_other_keys(ops, dtype, kind):
    """Prompts over caches, more queries than keys (the first see nothing), documents without keys
    or without queries."""
    q_lens, k_lens = [5, 1, 40, 33, 3, 0, 130, 64], [5, 300, 7, 97, 0, 50, 131, 4]
    prefix = [2, 10, 0, 97, 0, 9, 64, 4] if kind == "prefix" else None
    _check(ops, Batch(q_lens, k_lens, heads=4, kv_heads=2, dtype=dtype, kind=kind, prefix=prefix))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("terms", [
    dict(softcap=5.0), dict(slopes=True), dict(slopes=True, times=True), dict(table=(8, 5)),
    dict(table=(32, 128)), dict(softcap=20.0, slopes=True, times=True, table=(16, 40)),
    dict(scale=-0.3), dict(scale=0.0, table=(4, 3))])
@pytest.mark.parametrize("kind", ["causal", "full"])
def test_terms_of_the_score(ops, dtype, terms, kind):
    terms = dict(terms)
    n, reach = terms.pop("table", (0, 0))
    buckets = ops.distance_buckets(n, reach, kind == "full", "cpu") if n else None
    _check(ops, Batch([90, 1, 37, 260], heads=4, kv_heads=2, dtype=dtype, kind=kind,
                      buckets=buckets, num_buckets=n, seed=n, **terms))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,group,most,kind", [(64, 2, 36, "causal"), (32, 1, 68, "prefix"),
                                                 (96, 2, 66, "causal")])
def test_many_walks_of_many_lengths(ops, dtype, dim, group, most, kind):
    """So many packed walks that those of each number of 32 rows have a launch of their own in the
    backward pass, and some that none of those takes."""
    gen = torch.Generator().manual_seed(dim)
    lens = torch.randint(0, most, (130,), generator=gen).tolist()
    lens[40:52] = [0, 1, 31, 32, 33, 64, 65, 96, 97, 130, 200, 2]
    prefix = [(5 * w) % (n + 2) for w, n in enumerate(lens)] if kind == "prefix" else None
    _check(ops, Batch(lens, heads=16 * group, kv_heads=16, dim=dim, dtype=dtype, kind=kind,
                      prefix=prefix, buckets=ops.distance_buckets(4, 50, device="cpu"),
                      num_buckets=4, softcap=30.0))


def _padded(x, lens, length):
    rows = x.new_full((len(lens), length) + x.shape[1:], math.nan)
    for w, part in enumerate(x.split(lens)):
        rows[w, :lens[w]] = part
    return rows


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["causal", "full"])
@pytest.mark.parametrize("padded", [False, True])
def test_many_tiny_walks(ops, dtype, kind, padded):
    """Walks of a few rows share tiles; padding holds NaN."""
    gen = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 9, (130,), generator=gen).tolist()
    if not padded:
        lens[100:104] = [40, 97, 0, 260]
    b = Batch(lens, heads=32, kv_heads=16, dim=64, dtype=dtype, kind=kind, slopes=True,
              buckets=ops.distance_buckets(4, 5, kind == "full", "cpu"), num_buckets=4)
    if not padded:
        return _check(ops, b)
    q, k, v = (_padded(x, lens, 8).cuda().requires_grad_() for x in (b.q, b.k, b.v))
    table = b.table.cuda().requires_grad_()
    mask = ops.WalkMask.padded(torch.tensor(lens).cuda(), 8, kind=kind)
    out = ops.walk_attention(q, k, v, mask, **b.terms(table))
    out.backward(_padded(b.d_out, lens, 8).cuda())
    seen = torch.arange(8) < torch.tensor(lens)[:, None]
    got = {"out": out, "d_q": q.grad, "d_k": k.grad, "d_v": v.grad}
    for name, (value, bound) in b.reference().items():
        if name == "d_table":
            wf.check(name, table.grad, value, bound)
            continue
        rows = got[name].detach().cpu()
        assert not rows[~seen].any()
        wf.check(name, rows[seen], value, bound)


def test_many_padded_walks(ops):
    """A batch with launches by length against the same walks in smaller batches without: one
    float32 rounding of each of at most 80 terms either way, of values of the order of one."""
    gen = torch.Generator().manual_seed(4)
    n, length, heads = 8200, 40, 8
    lens = torch.randint(0, length + 1, (n,), generator=gen).cuda()
    x = torch.randn(4, n, length, heads, 8, generator=gen).cuda()
    table = torch.randn(heads, 6, generator=gen).cuda()
    buckets = ops.distance_buckets(6, 36)

    def run(part):
        q, k, v = (y[part].clone().requires_grad_() for y in x[:3])
        t = table.clone().requires_grad_()
        out = ops.walk_attention(q, k, v, ops.WalkMask.padded(lens[part], length), bias_table=t,
                                 buckets=buckets)
        out.backward(x[3][part])
        return [out.detach(), q.grad, k.grad, v.grad], t.grad.double()

    got, got_table = run(slice(0, n))
    want_table = torch.zeros_like(got_table)
    scale = torch.zeros_like(got_table)
    for w in range(0, n, 2050):
        part = slice(w, w + 2050)
        want, t = run(part)
        want_table += t
        scale += t.abs()
        for a, b in zip(got, want):
            torch.testing.assert_close(a[part], b, rtol=1e-4, atol=2e-4)
    # sums of a few million products, of which the float32 ones hold a few thousand each
    assert ((got_table - want_table).abs() <= 1e-3 * (scale + 1.0)).all()


@pytest.mark.parametrize("k_lens", [None, [50, 1, 400]])
@pytest.mark.parametrize("reach,num", [(0, 1), (0, 3), (1, 3), (31, 7), (300, 256), (1024, 64)])
def test_bias_reaches(ops, reach, num, k_lens):
    """Bucket ids in any order, some without a distance, one distance or all of them."""
    gen = torch.Generator().manual_seed(reach)
    ids = torch.randint(0, num, (2 * reach + 1,), generator=gen, dtype=torch.int32)
    _check(ops, Batch([50, 1, 170], k_lens, kind="full", buckets=ids, num_buckets=num))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (6, 3), (40, 2)])
def test_shared_heads(ops, dtype, heads, kv_heads):
    _check(ops, Batch([33, 100], heads=heads, kv_heads=kv_heads, dim=32, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF, SF])
def test_a_long_document(ops, dtype):
    """Enough keys for many tiles, and key heads whose query heads are split over workgroups."""
    _check(ops, Batch([1500], heads=2, kv_heads=1, dim=64, dtype=dtype,
                      buckets=ops.distance_buckets(32, 128, device="cpu"), num_buckets=32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_keys_of_few_queries(ops, dtype):
    _check(ops, Batch([1, 3, 17], [3001, 700, 2000], heads=4, kv_heads=2, dtype=dtype,
                      slopes=True), backward=dtype == SF)


def test_nothing_at_all(ops):
    for lens in ([], [0], [0, 0, 0]):
        got = Batch(lens).run(ops)
        assert all(x.numel() == 0 for x in got.values())
    b = Batch([0, 0], [3, 4], buckets=ops.distance_buckets(4, 2, device="cpu"), num_buckets=4)
    got = b.run(ops)
    assert got["d_k"].abs().sum() == 0 and got["d_v"].abs().sum() == 0
    assert got["d_table"].abs().sum() == 0
    b = Batch([3, 4], [0, 0])
    got = b.run(ops)
    assert got["out"].abs().sum() == 0 and got["d_q"].abs().sum() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_walks(ops, dtype):
    """Padded rows, whatever they hold, leave zeros and reach nothing."""
    lens, length = [0, 1, 80, 33, 64, 7, 100, 80], 80  # a length past the row is the row's
    gen = torch.Generator().manual_seed(3)
    shape = (len(lens), length, 2, 64)
    q, k, v, d_out = (_normal(gen, *shape, dtype=dtype) for _ in range(4))
    real = [min(n, length) for n in lens]
    pad = torch.arange(length)[None] >= torch.tensor(real)[:, None]
    for fill in (0.0, math.nan, math.inf):
        dev = []
        for x in (q, k, v, d_out):
            x = x.clone()
            x[pad] = fill
            dev.append(x.cuda())
        qkv = [x.requires_grad_() for x in dev[:3]]
        mask = ops.WalkMask.padded(torch.tensor(lens).cuda(), length)
        out = ops.walk_attention(*qkv, mask)
        out.backward(dev[3])
        flat = lambda x: x.double().flatten(0, 1)  # noqa: E731
        want = wf.attention(flat(q), flat(k), flat(v), wf.documents("causal", real, real),
                            d_out=flat(d_out), dtype=dtype,
                            starts=[(w * length, w * length) for w in range(len(lens))])
        for name, x in zip(("out", "d_q", "d_k", "d_v"), [out] + [x.grad for x in qkv]):
            wf.check(name, x.flatten(0, 1), *want[name])
            assert (x.cpu()[pad] == 0).all(), name


def test_lens_of_other_integer_types(ops):
    q = torch.randn(3, 10, 1, 32, device="cuda")
    a = ops.walk_attention(q, q, q, ops.WalkMask.padded(torch.tensor([10, 2, 5]).cuda(), 10))
    b = ops.walk_attention(q, q, q, ops.WalkMask.padded(
        torch.tensor([10, 2, 5], dtype=torch.int32).cuda(), 10))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_stays_in_its_walk(ops, dtype, bad):
    lens = [9, 30, 4, 70, 12]
    clean = Batch(lens, dtype=dtype, kind="full", buckets=ops.distance_buckets(8, 9, device="cpu"),
                  num_buckets=8)
    want = clean.run(ops)
    for name in ("q", "k", "v", "d_out"):
        b = Batch(lens, dtype=dtype, kind="full", buckets=clean.buckets, num_buckets=8)
        getattr(b, name)[9 + 7, 1, 5] = bad  # a row of the second walk
        got = b.run(ops)
        other = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
        other[9:39] = False
        for x in ("out", "d_q", "d_k", "d_v"):
            assert torch.equal(got[x][other], want[x][other]), (name, x)
            assert torch.equal(got[x][:, 0], want[x][:, 0]), (name, x)  # nor in another head
        reached = {"d_out": ("d_q", "d_k", "d_v")}.get(name, ("out", "d_q", "d_k", "d_v"))
        assert any(not torch.isfinite(got[x][9:39, 1]).all() for x in reached), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_tables_that_mask(ops, dtype):
    """-inf masks; the type's lowest value too, and a row of nothing else is a uniform row."""
    ids = torch.tensor([0, 1, 2, 2, 3], dtype=torch.int32)  # distances -2..2
    for low in (-math.inf, torch.finfo(torch.float32).min):
        b = Batch([6, 40], dtype=dtype, kind="full", buckets=ids, num_buckets=4)
        b.table[0] = torch.tensor([low, low, 0.5, low])  # hops 0 and 1 back alone
        b.table[1] = low
        got = b.run(ops)
        ref = Batch([6, 40], dtype=dtype, kind="full", buckets=ids, num_buckets=4)
        ref.table[0] = torch.tensor([-1e9, -1e9, 0.5, -1e9])
        want = ref.reference()
        wf.check("out", got["out"][:, 0], *(x[:, 0] for x in want["out"]))
        wf.check("d_q", got["d_q"][:, 0], *(x[:, 0] for x in want["d_q"]))
        if low == -math.inf:
            assert got["out"][:, 1].abs().sum() == 0
            assert got["d_v"][:, 1].abs().sum() == 0 and got["d_q"][:, 1].abs().sum() == 0
        else:  # a uniform row: the mean of v, and its gradient
            u = wf.U[dtype]
            for a, n in ((0, 6), (6, 40)):
                v, do = b.v[a:a + n, 1].double(), b.d_out[a:a + n, 1].double()
                bound = 2.1 * (u + n * wf.F32) * (v.abs().mean(0) + 1e-6)
                wf.check("out", got["out"][a:a + n, 1], v.mean(0).expand(n, -1),
                         bound.expand(n, -1))
                bound = 2.1 * (u + n * wf.F32) * (do.abs().mean(0) + 1e-6)
                wf.check("d_v", got["d_v"][a:a + n, 1], do.mean(0).expand(n, -1),
                         bound.expand(n, -1))


@pytest.mark.parametrize("dtype", [BF, SF])
def test_layouts(ops, dtype):
    """Slices of one projection, heads first, one key row for all, rows that are not 16-byte pieces:
    the same values give the same results, bit for bit."""
    b = Batch([40, 100, 3], heads=4, kv_heads=2, dtype=dtype)
    want = b.run(ops)
    n = sum(b.q_lens)

    def again(q, k, v, d_out):
        inputs = [x.detach().requires_grad_() for x in (q, k, v)]
        out = ops.walk_attention(*inputs, b.mask(ops))
        return dict(zip(("out", "d_q", "d_k", "d_v"),
                        (out, *torch.autograd.grad(out, inputs, d_out))))

    q, k, v, d_out = (x.cuda() for x in (b.q, b.k, b.v, b.d_out))
    fused = torch.cat([q, k, v], 1)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, d_out)]
    odd = []
    for x in (q, k, v, d_out):
        y = torch.empty(n, x.shape[1], 67, dtype=dtype, device="cuda")[:, :, 3:]
        y.copy_(x)
        odd.append(y)
    columns = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, d_out)]
    for layout in (list(fused.split([4, 2, 2], 1)) + [d_out], heads_first, odd, columns):
        got = again(*layout)
        for name in want:
            assert torch.equal(got[name], want[name]), name

    one = k[:1].expand(n, -1, -1)
    got, same = again(q, one, one, d_out), again(q, one.contiguous(), one.contiguous(), d_out)
    for name in want:
        assert torch.equal(got[name], same[name]), name
    leaf = k[:1].clone().requires_grad_()
    out = ops.walk_attention(q, leaf.expand(n, -1, -1), v, b.mask(ops))
    (grad,) = torch.autograd.grad(out, leaf, d_out)
    full = leaf.detach().expand(n, -1, -1).contiguous().requires_grad_()
    out = ops.walk_attention(q, full, v, b.mask(ops))
    (rows,) = torch.autograd.grad(out, full, d_out)
    assert torch.allclose(grad.float(), rows.float().sum(0, keepdim=True), rtol=2 * wf.U[dtype],
                          atol=n * wf.U[dtype] * rows.abs().max().item())


@pytest.mark.parametrize("dtype", [BF, SF])
def test_equal_inputs_give_equal_bits(ops, dtype):
    b = Batch([300, 5, 80, 500], heads=8, kv_heads=2, dtype=dtype, softcap=10.0,
              buckets=ops.distance_buckets(16, 30, device="cpu"), num_buckets=16)
    first = b.run(ops)
    for _ in range(3):
        again = b.run(ops)
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_another_stream(ops):
    b = Batch([100, 60], heads=2, dtype=BF)
    want = b.run(ops)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = b.run(ops)
    side.synchronize()
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_in_a_graph(ops):
    """Forward, backward and a step captured once and replayed on changed inputs."""
    b = Batch([50, 70], heads=4, kv_heads=2, dtype=BF,
              buckets=ops.distance_buckets(8, 20, device="cpu"), num_buckets=8)
    q, k, v = (x.cuda().requires_grad_() for x in (b.q, b.k, b.v))
    table, d_out = b.table.cuda().requires_grad_(), b.d_out.cuda()
    mask, terms = b.mask(ops), b.terms()
    terms["bias_table"] = table

    def both():
        out = ops.walk_attention(q, k, v, mask, **terms)
        return (out, *torch.autograd.grad(out, (q, k, v, table), d_out))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for step in range(4):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            table.copy_(torch.randn_like(table))
        want = [x.clone() for x in both()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x, y), step


def test_gradients_against_differences(ops):
    """Central differences of a scalar along random directions.  In float32 a loss of size S is
    rounded by about S 2^-24 sqrt(terms); with the step h the quotient is off by that over h, and
    by the third derivative times h^2 / 6."""
    b = Batch([30, 9, 50], heads=4, kv_heads=2, dim=32, dtype=SF, softcap=3.0, slopes=True,
              buckets=ops.distance_buckets(6, 8, device="cpu"), num_buckets=6)
    mask = b.mask(ops)
    weight = b.d_out.cuda().double()
    inputs = [x.cuda() for x in (b.q, b.k, b.v, b.table)]

    def loss(xs):
        terms = b.terms(xs[3])
        return (ops.walk_attention(*xs[:3], mask, **terms).double() * weight).sum().item()

    leaves = [x.clone().requires_grad_() for x in inputs]
    out = ops.walk_attention(*leaves[:3], mask, **b.terms(leaves[3]))
    grads = torch.autograd.grad(out, leaves, b.d_out.cuda())
    gen = torch.Generator().manual_seed(5)
    h = 1e-2
    for n, (x, g) in enumerate(zip(inputs, grads)):
        d = torch.randn(x.shape, generator=gen).cuda()
        d /= d.norm()
        moved = lambda t: [y + t * d if m == n else y for m, y in enumerate(inputs)]  # noqa: E731,B023
        # fourth order: (8 (f(h) - f(-h)) - (f(2h) - f(-2h))) / 12h
        slope = (8 * (loss(moved(h)) - loss(moved(-h)))
                 - (loss(moved(2 * h)) - loss(moved(-2 * h)))) / (12 * h)
        want = (g.double() * d.double()).sum().item()
        # 11392 outputs of size about 1 off by about 1e-6 each at random: 1e-4 in all, over h;
        # the fifth derivative's share is below 1e-3 |slope| for steps of norm 1e-2
        assert abs(slope - want) <= 1.5e-2 + 1e-3 * abs(want), (n, slope, want)


# ---- one event over a cache ------------------------------------------------------------------
def _step(ops, dtype, lens, capacity, heads, kv_heads, dim, *, softcap=0.0, num=0, reach=0,
          slopes=False, times=False, order="bshd", seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = len(lens)
    q = _normal(gen, n, heads, dim, dtype=dtype)
    k, v = (_normal(gen, n, kv_heads, dim, dtype=dtype) for _ in range(2))
    kc, vc = (_normal(gen, n, capacity, kv_heads, dim, dtype=dtype) for _ in range(2))
    used = torch.arange(capacity)[None] < torch.tensor(lens)[:, None]
    kc[~used], vc[~used] = math.nan, math.nan  # what the cache's end holds is nobody's business
    table = _normal(gen, heads, num) if num else None
    ids = ops.distance_buckets(num, reach, device="cpu") if num else None
    slope = torch.rand(heads, generator=gen) * 0.1 if slopes else None
    kt = torch.rand(n, capacity, generator=gen).cumsum(1) if times else None
    tq = None
    if times:
        tq = torch.tensor([kt[b, max(0, min(m, capacity) - 1)] + 0.5 for b, m in enumerate(lens)])
        kt[~used] = math.nan
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    if order == "bhsd":
        kcd, vcd = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (kc, vc))
    else:
        kcd, vcd = kc.cuda(), vc.cuda()
    ktd = dev(kt)
    out = ops.walk_attention_step(dev(q), dev(k), dev(v), kcd, vcd, torch.tensor(lens).cuda(),
                                  softcap=softcap, bias_table=dev(table), buckets=dev(ids),
                                  slopes=dev(slope), times=dev(tq), k_times=ktd)
    for b, m in enumerate(lens):
        if m < 0 or m >= capacity:
            if m < 0:
                assert (out[b] == 0).all()
            else:
                assert torch.isnan(out[b]).all()
            continue
        kc[b, m], vc[b, m] = k[b], v[b]
        if times:
            kt[b, m] = tq[b]
        d = lambda x: None if x is None else x.double()  # noqa: E731
        want = wf.attention(
            q[b:b + 1].double(), kc[b, :m + 1].double(), vc[b, :m + 1].double(),
            wf.documents("causal", [1], [m + 1]), softcap=softcap, table=d(table), buckets=ids,
            slopes=d(slope), q_times=None if tq is None else tq[b:b + 1].double(),
            k_times=None if kt is None else kt[b, :m + 1].double(), dtype=dtype)["out"]
        wf.check(f"out[{b}] of {m}", out[b:b + 1], *want)
    for x, y in ((kcd, kc), (vcd, vc)) + (((ktd, kt),) if times else ()):
        assert torch.equal(torch.nan_to_num(x.cpu().float(), nan=77.0),
                           torch.nan_to_num(y.float(), nan=77.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 32, 64, 80, 128])
def test_step_lengths(ops, dtype, dim):
    _step(ops, dtype, [0, 1, 30, 31, 32, 63, 127, 128, 199, -1, 200, 7], 200, 4, 2, dim, seed=dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("terms", [
    dict(softcap=4.0), dict(slopes=True), dict(slopes=True, times=True), dict(num=16, reach=20),
    dict(num=32, reach=1024, softcap=9.0, slopes=True, times=True), dict(num=1, reach=0)])
def test_step_terms(ops, dtype, terms):
    _step(ops, dtype, [0, 5, 90, 300, -7, 411], 412, 6, 2, 64, **terms)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 1), (33, 1), (70, 2)])
def test_step_shared_heads(ops, heads, kv_heads):
    _step(ops, BF, [100, 0, 64], 128, heads, kv_heads, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_long_histories(ops, dtype):
    _step(ops, dtype, [9000, 3, 4097], 9001, 4, 1, 64, slopes=True, times=True, order="bhsd")


def test_steps_follow_a_prompt(ops):
    """A walk taken event by event gives what one causal pass gives."""
    gen = torch.Generator().manual_seed(1)
    n, heads, dim = 40, 4, 64
    q, k, v = (_normal(gen, n, h, dim, dtype=BF) for h in (heads, 2, 2))
    table, ids = _normal(gen, heads, 8).cuda(), ops.distance_buckets(8, 12)
    mask = ops.WalkMask.packed(torch.tensor([0, n]).cuda(), n)
    whole = ops.walk_attention(q.cuda(), k.cuda(), v.cuda(), mask, bias_table=table, buckets=ids)
    kc, vc = (torch.full((1, 64, 2, dim), math.nan, dtype=BF, device="cuda") for _ in range(2))
    lens = torch.zeros(1, dtype=torch.int64, device="cuda")
    for i in range(n):
        out = ops.walk_attention_step(q[i:i + 1].cuda(), k[i:i + 1].cuda(), v[i:i + 1].cuda(), kc,
                                      vc, lens, bias_table=table, buckets=ids)
        lens += 1
        # each is within u (|o| + sum P |v|) of the formula
        bound = 2.2 * wf.U[BF] * (whole[i].abs().float().cpu() + v[:i + 1].abs().float().amax())
        assert ((out[0].float() - whole[i].float()).abs().cpu() <= bound).all(), i


def test_step_offsets_past_32_bits(ops):
    """A cache of more than 2^32 bytes and elements: the last walk's rows lie past both."""
    capacity, heads, dim = 1 << 18, 2, 128
    n = 65  # 65 * 2^18 * 2 * 128 elements > 2^32
    kc = torch.zeros(n, capacity, heads, dim, dtype=BF, device="cuda")
    vc = torch.zeros(n, capacity, heads, dim, dtype=BF, device="cuda")
    gen = torch.Generator().manual_seed(2)
    k, v, q = (_normal(gen, n, heads, dim, dtype=BF) for _ in range(3))
    lens = torch.full((n,), -1)
    lens[-1] = 1000
    rows_k, rows_v = (_normal(gen, 1000, heads, dim, dtype=BF) for _ in range(2))
    kc[-1, :1000], vc[-1, :1000] = rows_k.cuda(), rows_v.cuda()
    out = ops.walk_attention_step(q.cuda(), k.cuda(), v.cuda(), kc, vc, lens.cuda())
    want = wf.attention(q[-1:].double(), torch.cat([rows_k, k[-1:]]).double(),
                        torch.cat([rows_v, v[-1:]]).double(), wf.documents("causal", [1], [1001]),
                        dtype=BF)["out"]
    wf.check("out", out[-1:], *want)
    assert torch.equal(kc[-1, 1000].cpu(), k[-1]) and torch.equal(vc[-1, 1000].cpu(), v[-1])
    assert out[:-1].abs().sum() == 0


# ---- the dense bias -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len,offset", [
    (1, 1, 0), (1, 300, 299), (300, 1, 0), (80, 80, 0), (33, 65, 32), (7, 1031, -5),
    (130, 577, 447), (64, 64, 1000), (64, 64, -1000), (5, 8, 3), (600, 130, 0)])
def test_relative_bias(ops, dtype, q_len, k_len, offset):
    heads, num, reach = 3, 17, 40
    gen = torch.Generator().manual_seed(q_len + k_len)
    table = _normal(gen, heads, num, dtype=dtype)
    ids = torch.randint(0, num, (2 * reach + 1,), generator=gen, dtype=torch.int32)
    d_out = _normal(gen, heads, q_len, k_len, dtype=dtype)
    leaf = table.cuda().requires_grad_()
    out = ops.relative_bias(leaf, ids.cuda(), q_len, k_len, offset)
    hop = torch.arange(q_len)[:, None] + offset - torch.arange(k_len)
    bucket = ids.long()[hop.clamp(-reach, reach) + reach]
    assert torch.equal(out.detach().cpu(), table[:, bucket])
    (grad,) = torch.autograd.grad(out, leaf, d_out.cuda())
    want = torch.zeros(heads, num, dtype=torch.float64)
    size = torch.zeros(heads, num, dtype=torch.float64)
    for b in range(num):
        want[:, b] = (d_out.double() * (bucket == b)).sum((1, 2))
        size[:, b] = (d_out.double().abs() * (bucket == b)).sum((1, 2))
    # a lane adds up to 64 rows, then up to 64 distances and 3 waves, in float32
    wf.check("d_table", grad, want, wf.U[dtype] * want.abs() + 160 * wf.F32 * size + 1e-30)


@pytest.mark.parametrize("reach", [0, 1, 2, 7, 8, 1024])
@pytest.mark.parametrize("dtype", [BF, SF])
def test_relative_bias_reaches(ops, dtype, reach):
    num = min(256, 2 * reach + 1)
    table = torch.randn(2, num).to(dtype)
    ids = (torch.arange(2 * reach + 1) * 7 % num).int()
    hop = torch.arange(90)[:, None] - torch.arange(2500) + 1200
    for q_len, k_len in ((90, 2500), (90, 83)):
        out = ops.relative_bias(table.cuda(), ids.cuda(), q_len, k_len, 1200)
        bucket = ids.long()[hop[:q_len, :k_len].clamp(-reach, reach) + reach]
        assert torch.equal(out.cpu(), table[:, bucket])


def test_relative_bias_gradient_layouts(ops):
    table = torch.randn(2, 5, device="cuda", requires_grad=True)
    ids = ops.distance_buckets(5, 9)
    out = ops.relative_bias(table, ids, 50, 70, 20)
    d = torch.randn(2, 50, 70, device="cuda")
    (want,) = torch.autograd.grad(out, table, d, retain_graph=True)
    wide = torch.zeros(2, 50, 99, device="cuda")
    wide[:, :, 17:87] = d
    for layout in (wide[:, :, 17:87], d.transpose(1, 2).contiguous().transpose(1, 2),
                   d.transpose(0, 1).contiguous().transpose(0, 1)):
        (got,) = torch.autograd.grad(out, table, layout, retain_graph=True)
        assert torch.equal(got, want)
    (got,) = torch.autograd.grad(out, table, torch.ones(1, 1, 1, device="cuda").expand(2, 50, 70))
    counts = torch.bincount(ids.cpu().long()[(torch.arange(50)[:, None] + 20 - torch.arange(70)).clamp(-9, 9) + 9].flatten(), minlength=5)
    assert torch.equal(got.cpu(), counts.float().expand(2, 5))


def test_dense_and_fused_bias_agree(ops):
    """The table's gradient through the dense bias and an attention of torch's own operations, and
    inside walk_attention."""
    n, heads, dim = 60, 2, 32
    gen = torch.Generator().manual_seed(9)
    q, k, v, d_out = (_normal(gen, n, heads, dim).cuda() for _ in range(4))
    ids = ops.distance_buckets(8, 16, bidirectional=True)
    table = _normal(gen, heads, 8).cuda().requires_grad_()
    s = (q.transpose(0, 1) @ k.permute(1, 2, 0)) * dim ** -0.5 + ops.relative_bias(table, ids, n, n)
    a = (torch.softmax(s, -1) @ v.transpose(0, 1)).transpose(0, 1)
    (ga,) = torch.autograd.grad(a, table, d_out)
    mask = ops.WalkMask.packed(torch.tensor([0, n]).cuda(), n, kind="full")
    b = ops.walk_attention(q, k, v, mask, bias_table=table, buckets=ids)
    (gb,) = torch.autograd.grad(b, table, d_out)
    # both are float32: sums of 60 by 60 terms of size about 0.1
    assert torch.allclose(a, b, rtol=0, atol=2e-5) and torch.allclose(ga, gb, rtol=0, atol=1e-4)


# ---- refusals -----------------------------------------------------------------------------------
def test_refusals(ops):
    q = torch.randn(10, 4, 64, device="cuda", dtype=BF)
    kv = torch.randn(10, 2, 64, device="cuda", dtype=BF)
    off = torch.tensor([0, 4, 10]).cuda()
    mask = ops.WalkMask.packed(off, 10)
    ids = ops.distance_buckets(4, 8)
    table = torch.randn(4, 4, device="cuda")
    att = lambda *a, **kw: ops.walk_attention(*a, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="on the GPU"):
        att(q.cpu(), kv, kv, mask)
    with pytest.raises(ValueError, match="same type"):
        att(q, kv.float(), kv, mask)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        att(q.double(), kv.double(), kv.double(), mask)
    with pytest.raises(ValueError, match="multiple of the key heads"):
        att(q[:, :3], kv, kv, mask)
    with pytest.raises(ValueError, match="head size"):
        att(q[..., :60], kv[..., :60], kv[..., :60], mask)
    with pytest.raises(ValueError, match="head size"):
        x = torch.randn(10, 1, 136, device="cuda")
        att(x, x, x, mask)
    with pytest.raises(ValueError, match="rows of heads"):
        att(q[:9], kv, kv, mask)
    with pytest.raises(ValueError, match="rows of heads"):
        att(q, kv[:9], kv[:9], mask)
    with pytest.raises(ValueError, match="same shape"):
        att(q, kv, kv[:, :1], mask)
    with pytest.raises(ValueError, match="go together"):
        att(q, kv, kv, mask, bias_table=table)
    with pytest.raises(ValueError, match="num_buckets"):
        att(q, kv, kv, mask, bias_table=table[:3], buckets=ids)
    with pytest.raises(ValueError, match="2 reach"):
        att(q, kv, kv, mask, bias_table=table, buckets=ids[:-1])
    with pytest.raises(ValueError, match="2 reach"):
        att(q, kv, kv, mask, bias_table=table, buckets=ids.long())
    with pytest.raises(ValueError, match="softcap"):
        att(q, kv, kv, mask, softcap=-1.0)
    with pytest.raises(ValueError, match="finite"):
        att(q, kv, kv, mask, scale=math.inf)
    with pytest.raises(ValueError, match="slopes"):
        att(q, kv, kv, mask, times=torch.zeros(10, device="cuda"))
    with pytest.raises(ValueError, match="no gradient"):
        att(q, kv, kv, mask, slopes=torch.ones(4, device="cuda", requires_grad=True))
    with pytest.raises(ValueError, match="WalkMask"):
        att(q, kv, kv, None)
    with pytest.raises(ValueError, match="kind"):
        ops.WalkMask.packed(off, 10, kind="local")
    with pytest.raises(ValueError, match="prefix"):
        ops.WalkMask.packed(off, 10, kind="prefix")
    with pytest.raises(ValueError, match="whole numbers"):
        ops.WalkMask.padded(torch.ones(3, device="cuda"), 5)
    with pytest.raises(ValueError, match="reach"):
        ops.distance_buckets(4, 1025)
    with pytest.raises(ValueError, match="buckets"):
        ops.distance_buckets(257, 5)
    x = q.clone().requires_grad_()
    (g,) = torch.autograd.grad(att(x, kv, kv, mask).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    cache = torch.randn(10, 16, 2, 64, device="cuda", dtype=BF)
    lens = torch.zeros(10, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="capacity"):
        ops.walk_attention_step(q, kv, kv, cache[:9], cache[:9], lens)
    with pytest.raises(ValueError, match="16-byte"):
        ops.walk_attention_step(q, kv, kv, cache.transpose(1, 3).contiguous().transpose(1, 3),
                                cache, lens)
    with pytest.raises(ValueError, match="lens"):
        ops.walk_attention_step(q, kv, kv, cache, cache, lens[:9])
    with pytest.raises(ValueError, match="go together"):
        ops.walk_attention_step(q, kv, kv, cache, cache, lens,
                                slopes=torch.ones(4, device="cuda"),
                                times=torch.zeros(10, device="cuda"))
    with pytest.raises(ValueError, match="negative"):
        ops.relative_bias(table, ids, -1, 4)
    with pytest.raises(ValueError, match="table"):
        ops.relative_bias(table[0], ids, 4, 4)


def test_a_dropped_result_frees_its_memory(ops):
    """The output's history holds nothing that holds the output."""
    q, k, v = (torch.randn(2000, 4, 64, device="cuda", dtype=BF, requires_grad=True)
               for _ in range(3))
    table = torch.randn(4, 8, device="cuda", requires_grad=True)
    ids = ops.distance_buckets(8, 16)
    mask = ops.WalkMask.packed(torch.tensor([0, 700, 2000]).cuda(), 2000)

    def both():
        ops.walk_attention(q, k, v, mask, bias_table=table, buckets=ids)
        ops.relative_bias(table, ids, 100, 100)

    both()
    held = torch.cuda.memory_allocated()
    for _ in range(5):
        both()
    assert torch.cuda.memory_allocated() == held


def test_gradients_are_differentiable_once(ops):
    b = Batch([20, 5], dtype=SF)
    q, k, v = (x.cuda().requires_grad_() for x in (b.q, b.k, b.v))
    out = ops.walk_attention(q, k, v, b.mask(ops))
    (d_q,) = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        d_q.sum().backward()
    table = torch.randn(2, 4, device="cuda", requires_grad=True)
    bias = ops.relative_bias(table, ops.distance_buckets(4, 3), 6, 6)
    (d_table,) = torch.autograd.grad(bias.square().sum(), table, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        d_table.sum().backward()


def test_outputs_changed_in_place(ops):
    """What the backward pass reads again must be as it was; the rest is the caller's."""
    b = Batch([20, 5], dtype=SF)
    want = b.run(ops)
    q, k, v = (x.cuda().requires_grad_() for x in (b.q, b.k, b.v))
    out = ops.walk_attention(q, k, v, b.mask(ops))
    with torch.no_grad():
        q.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(b.d_out.cuda())
    with torch.no_grad():
        q.copy_(b.q)
    out = ops.walk_attention(q, k, v, b.mask(ops))
    out.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(b.d_out.cuda())
    out = ops.walk_attention(q, k, v, b.mask(ops)) * 1
    out.mul_(1)
    out.backward(b.d_out.cuda())
    assert torch.equal(q.grad, want["d_q"])


def test_no_memory(ops):
    with pytest.raises(torch.OutOfMemoryError):
        ops.relative_bias(torch.zeros(1, 4, device="cuda"), ops.distance_buckets(4, 3),
                          1 << 20, 1 << 20)


def test_a_mask_on_another_stream(ops):
    """A mask made on one stream, used on another and dropped at once."""
    b = Batch([300, 60], heads=2, dtype=BF)
    want = b.run(ops)["out"]
    q, k, v = (x.cuda() for x in (b.q, b.k, b.v))
    mask = b.mask(ops)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = ops.walk_attention(q, k, v, mask)
    mask.record_stream(side)
    del mask
    for _ in range(8):  # would take the mask's place
        b.mask(ops)._mask.info.zero_()
    side.synchronize()
    assert torch.equal(got, want)


def test_example():
    """examples/walk_model.py at a small size: it learns, and its steps agree with one pass.  Both
    paths round to bfloat16 six times a layer and twelve in all, each by at most 2^-8 of a value."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "walk_model.py")
    spec = importlib.util.spec_from_file_location("walk_model", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, served, off, far = example.main(["--nodes", "200", "--walks", "400", "--length", "24",
                                             "--batch", "200", "--steps", "30"])
    assert losses[-1] < losses[0] - 1
    assert served > 1000 and off < 12 * 2 ** -8
    assert ((far >= 0) & (far < 24)).all()
