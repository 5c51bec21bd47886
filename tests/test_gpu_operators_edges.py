"""The operators at the ends of their ranges, against their formulas in float64."""
import math

import pytest
import torch

from tests import walk_formulas as wf
from tests.test_gpu_operators import BF, DTYPES, HF, SF, Batch, _check, _normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from temporal_random_walk import operators
    return operators


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reach", [0, 1, 2, 7, 8, 1024])
@pytest.mark.parametrize("q_len,k_len,offset", [(10, 10, 0), (80, 80, 0), (90, 2500, 1200),
                                                (90, 83, 1200), (130, 600, 0), (70, 65, -30)])
def test_bias_gradient_of_every_reach(ops, dtype, reach, q_len, k_len, offset):
    """Each pair counts once, keys after the query too where all distances share one bucket."""
    gen = torch.Generator().manual_seed(reach + q_len)
    num = min(256, 2 * reach + 2)
    ids = (torch.arange(2 * reach + 1) * 7 % num).int()
    leaf = _normal(gen, 2, num, dtype=dtype).cuda().requires_grad_()
    # nothing cancels, and no sum leaves float16
    d_out = ((torch.rand(2, q_len, k_len, generator=gen) + 0.5) / 16).to(dtype)
    out = ops.relative_bias(leaf, ids.cuda(), q_len, k_len, offset)
    (grad,) = torch.autograd.grad(out, leaf, d_out.cuda())
    hop = torch.arange(q_len)[:, None] + offset - torch.arange(k_len)
    bucket = ids.long()[hop.clamp(-reach, reach) + reach].flatten()
    want = torch.stack([torch.bincount(bucket, d.flatten().double(), minlength=num) for d in d_out])
    # A lane adds up to 64 rows of at most ten pieces of eight values in float32, then come its
    # wave's and the workgroups' sums; all terms have one sign.
    wf.check("d_table", grad, want, (wf.U[dtype] + 900 * wf.F32) * want.abs() + 1e-30)


ONE_DISTANCE = [(0, 1), (0, 3), (1, 3)]


@pytest.mark.parametrize("kind", ["full", "prefix", "causal"])
@pytest.mark.parametrize("reach,num", ONE_DISTANCE)
@pytest.mark.parametrize("lens", [[20, 1, 33, 40], [50, 1, 170], [260]])
def test_table_gradient_of_one_distance(ops, kind, reach, num, lens):
    """Where all distances share a bucket its gradient is a sum that cancels, so a pair that is
    lost or counted twice shows.  float32: the bound is far below one pair's share."""
    ids = torch.arange(2 * reach + 1).int() % num
    prefix = [n // 2 for n in lens] if kind == "prefix" else None
    _check(ops, Batch(lens, dtype=SF, kind=kind, prefix=prefix, buckets=ids, num_buckets=num))


@pytest.mark.parametrize("kind", ["full", "prefix", "causal"])
@pytest.mark.parametrize("reach,num", ONE_DISTANCE)
@pytest.mark.parametrize("q_lens,k_lens", [([5, 9, 4], [50, 20, 300]), ([100, 31, 2], [160, 31, 9])])
def test_table_gradient_of_one_distance_over_caches(ops, kind, reach, num, q_lens, k_lens):
    """Prompts of several walks in one wave, whose rows have no diagonal in common."""
    ids = torch.arange(2 * reach + 1).int() % num
    prefix = [n // 2 for n in k_lens] if kind == "prefix" else None
    _check(ops, Batch(q_lens, k_lens, dtype=SF, kind=kind, prefix=prefix, buckets=ids,
                      num_buckets=num))


def _masked_steps(ops, dtype, lens, capacity, table, ids, heads=4, kv_heads=2, dim=64):
    """A step under a table that masks: against the formula, zeros where nothing is left."""
    gen = torch.Generator().manual_seed(capacity)
    n = len(lens)
    q = _normal(gen, n, heads, dim, dtype=dtype)
    k, v = (_normal(gen, n, kv_heads, dim, dtype=dtype) for _ in range(2))
    kc, vc = (_normal(gen, n, capacity, kv_heads, dim, dtype=dtype) for _ in range(2))
    out = ops.walk_attention_step(q.cuda(), k.cuda(), v.cuda(), kc.cuda(), vc.cuda(),
                                  torch.tensor(lens).cuda(), bias_table=table.cuda(),
                                  buckets=ids.cuda()).cpu()
    reach = ids.shape[0] // 2
    for b, m in enumerate(lens):
        kc[b, m], vc[b, m] = k[b], v[b]
        hop = (m - torch.arange(m + 1)).clamp(max=reach) + reach
        left = torch.isfinite(table[:, ids.long()[hop]]).any(-1)
        assert not out[b][~left].any()  # and no NaN
        low = table.double().clamp_min(-1e9)
        want = wf.attention(q[b:b + 1].double(), kc[b, :m + 1].double(), vc[b, :m + 1].double(),
                            wf.documents("causal", [1], [m + 1]), table=low, buckets=ids,
                            dtype=dtype)["out"]
        wf.check(f"out[{b}] of {m}", out[b:b + 1, left], *(x[:, left] for x in want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("capacity", [100, 9000])  # one workgroup a walk, and several
def test_steps_that_a_table_masks(ops, dtype, capacity):
    """Head 0 does not see the own event, head 1 nothing, head 2 the own event alone, head 3 all but
    what is far: an empty cache, every position masked, a whole workgroup's share masked."""
    ids = torch.arange(9, dtype=torch.int32)  # reach 4: distances -4..4, 0 is id 4
    inf = -math.inf
    table = torch.zeros(4, 9)
    table[0, 4] = inf
    table[1] = inf
    table[2, 5:] = inf
    table[3, 8] = inf
    lens = [n for n in (0, 1, 3, 31, 64, 99, 4000, 8999) if n < capacity]
    _masked_steps(ops, dtype, lens, capacity, table, ids)


def test_steps_agree_with_a_pass_where_a_table_masks(ops):
    n, heads, dim = 12, 2, 32
    gen = torch.Generator().manual_seed(7)
    q, k, v = (_normal(gen, n, heads, dim).cuda() for _ in range(3))
    table = torch.tensor([[-math.inf, 0.3], [-math.inf, -math.inf]]).cuda()
    ids = torch.tensor([0, 0, 0, 0, 1], dtype=torch.int32).cuda()  # two events back or more
    whole = ops.walk_attention(q, k, v, ops.WalkMask.packed(torch.tensor([0, n]).cuda(), n),
                               bias_table=table, buckets=ids)
    assert not whole[:2].any() and not whole[:, 1].any() and whole[2:, 0].any()
    kc, vc = (torch.zeros(1, n, heads, dim, device="cuda") for _ in range(2))
    for i in range(n):
        out = ops.walk_attention_step(q[i:i + 1], k[i:i + 1], v[i:i + 1], kc, vc,
                                      torch.tensor([i]).cuda(), bias_table=table, buckets=ids)
        # float32, at most 12 keys: a few units in the last place of sums of terms up to 4
        assert torch.allclose(out[0], whole[i], rtol=0, atol=1e-5), i


@pytest.mark.parametrize("dtype,gap", [(BF, 1 << 22), (SF, 1 << 21)])
def test_not_finite_beside_a_walk_of_far_rows(ops, dtype, gap):
    """Rows 8 MB apart, the furthest that are read in place: a walk of 300 rows is longer than 2^31
    bytes.  Walks share tiles, and those of the second are taken alone where the first is not
    finite: the second's results do not change."""
    lens, dim = [40, 300], 8
    n = sum(lens)
    gen = torch.Generator().manual_seed(11)
    values = _normal(gen, 4, n, 1, dim, dtype=dtype)
    far = torch.empty(n, gap, dtype=dtype, device="cuda")  # 2.9 GB

    def run(bad):
        rows = [far[:, m * dim:(m + 1) * dim].unflatten(1, (1, dim)) for m in range(4)]
        for x, y in zip(rows, values):
            x.copy_(y)
        if bad is not None:
            rows[bad][7, 0, 3] = math.nan
        leaves = [x.detach().requires_grad_() for x in rows[:3]]
        mask = ops.WalkMask.packed(torch.tensor([0, 40, n]).cuda(), n, kind="full")
        out = ops.walk_attention(*leaves, mask)
        return [out.detach(), *torch.autograd.grad(out, leaves, rows[3])]

    want = run(None)
    for bad in range(4):
        got = run(bad)
        for x, y in zip(got, want):
            assert torch.equal(x[40:], y[40:])
        assert any(torch.isnan(x[:40]).any() for x in got)


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("longest", [0, 5])
def test_rows_of_no_document(ops, dtype, longest):
    """The C ABI with packed offsets and the longest document stated: rows before the first one and
    after the last are zero, in every output."""
    import ctypes

    from temporal_random_walk import operators_capi as abi
    lib, rows, heads, kv_heads, dim = abi.lib(), 20, 4, 2, 64
    offsets = torch.tensor([2, 7, 8, 12]).cuda()
    gen = torch.Generator().manual_seed(longest)
    q, d_out = (_normal(gen, rows, heads, dim, dtype=dtype).cuda() for _ in range(2))
    k, v = (_normal(gen, rows, kv_heads, dim, dtype=dtype).cuda() for _ in range(2))
    out, d_q, low = (torch.full_like(q, math.nan) for _ in range(3))
    d_k, d_v = (torch.full_like(k, math.nan) for _ in range(2))
    info = torch.zeros(2, rows, 4, dtype=torch.int32, device="cuda")
    docs = torch.zeros(3, 8, dtype=torch.int32, device="cuda")
    stats = torch.zeros(2, heads, rows, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    mask = abi.MaskParams(docs=3, q_rows=rows, k_rows=rows, q_offsets=offsets.data_ptr(), kind=1,
                          q_rows_info=info[0].data_ptr(), k_rows_info=info[1].data_ptr(),
                          docs_info=docs.data_ptr())
    abi.call(lib.trw_ops_walk_mask, ctypes.byref(mask), stream)
    at = lambda x: abi.Rows(x.data_ptr(), x.stride(0), x.stride(1))  # noqa: E731
    p = abi.AttentionParams(
        dtype={SF: 0, BF: 2}[dtype], heads=heads, kv_heads=kv_heads, dim=dim, q_rows=rows,
        k_rows=rows, q_rows_info=info[0].data_ptr(), k_rows_info=info[1].data_ptr(),
        docs_info=docs.data_ptr(), docs=3, longest=longest, own_causal=1,
        score=abi.Score(dim ** -0.5, 0.0), q=at(q), k=at(k), v=at(v), out=at(out),
        out_low=at(low), stats=stats.data_ptr(), d_out=at(d_out), d_q=at(d_q), d_k=at(d_k),
        d_v=at(d_v))
    for backward, run in ((0, lib.trw_ops_attention_forward), (1, lib.trw_ops_attention_backward)):
        size = ctypes.c_uint64()
        abi.call(lib.trw_ops_attention_workspace, ctypes.byref(p), backward, ctypes.byref(size))
        space = torch.empty(size.value + 16, dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_bytes = space.data_ptr(), size.value
        abi.call(run, ctypes.byref(p), stream)
        torch.cuda.synchronize()
    d = lambda x: x[2:12].double().cpu()  # noqa: E731
    want = wf.attention(d(q), d(k), d(v), wf.documents("causal", [5, 1, 4], [5, 1, 4]),
                        d_out=d(d_out), dtype=dtype)
    for name, x in (("out", out), ("d_q", d_q), ("d_k", d_k), ("d_v", d_v)):
        assert not x[:2].any() and not x[12:].any(), name
        wf.check(name, x[2:12], *want[name])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [3000.0, 1e6, 1e30])
@pytest.mark.parametrize("lens", [[20, 1, 33, 40], [130, 260]])
def test_caps_far_above_the_scores(ops, dtype, softcap, lens):
    """cap(x) is then x but for its cube over 3 softcap^2, and as exact as x: within the bounds of the
    formula without a cap."""
    b = Batch(lens, dtype=dtype, softcap=softcap, scale=0.5)
    got, want = b.run(ops), b.reference()
    b.softcap = 0.0
    for name, (_, bound) in b.reference().items():
        wf.check(name, got[name], want[name][0], bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [3000.0, 1e6, 1e30])
def test_step_caps_far_above_the_scores(ops, dtype, softcap):
    gen = torch.Generator().manual_seed(5)
    n, dim, lens = 3, 64, [0, 40, 299]
    q, k, v = (_normal(gen, n, 2, dim, dtype=dtype) for _ in range(3))
    kc, vc = (_normal(gen, n, 300, 2, dim, dtype=dtype) for _ in range(2))
    out = ops.walk_attention_step(q.cuda(), k.cuda(), v.cuda(), kc.cuda(), vc.cuda(),
                                  torch.tensor(lens).cuda(), softcap=softcap, scale=0.5).cpu()
    for b, m in enumerate(lens):
        kc[b, m], vc[b, m] = k[b], v[b]
        args = (q[b:b + 1].double(), kc[b, :m + 1].double(), vc[b, :m + 1].double(),
                wf.documents("causal", [1], [m + 1]))
        want = wf.attention(*args, softcap=softcap, scale=0.5, dtype=dtype)["out"][0]
        bound = wf.attention(*args, scale=0.5, dtype=dtype)["out"][1]
        wf.check(f"out[{b}]", out[b:b + 1], want, bound)


def test_steps_over_one_shared_row(ops):
    """Caches that walks share are refused; one walk's has any stride there."""
    q, kv = torch.randn(3, 2, 64, device="cuda"), torch.randn(3, 2, 64, device="cuda")
    cache, lens = torch.randn(1, 8, 2, 64, device="cuda"), torch.tensor([1, 2, 3]).cuda()
    own = cache.repeat(3, 1, 1, 1)
    for caches in ((cache.expand(3, -1, -1, -1), own), (own, own[:, :, :1].expand(-1, -1, 2, -1))):
        with pytest.raises(ValueError, match="share memory"):
            ops.walk_attention_step(q, kv, kv, *caches, lens)
    want = ops.walk_attention_step(q, kv, kv, own.clone(), own.clone(), lens)
    one = ops.walk_attention_step(q[:1], kv[:1], kv[:1], cache.as_strided(cache.shape, (0, 128, 64, 1)),
                                  own[:1].clone(), lens[:1])
    assert torch.equal(one, want[:1])


@pytest.mark.parametrize("q_lens,k_lens", [([3, 0], [0, 0]), ([0, 0], [5, 2]), ([0], [0])])
def test_times_of_no_rows(ops, q_lens, k_lens):
    """Queries without keys, keys without queries: an empty tensor of times is one."""
    got = Batch(q_lens, k_lens, slopes=True, times=True, kind="full").run(ops)
    assert got["out"].shape[0] == sum(q_lens) and got["d_k"].shape[0] == sum(k_lens)
    assert not any(x.any() for x in got.values())


def test_step_over_a_cache_of_no_slots(ops):
    q, kv = torch.randn(2, 2, 64, device="cuda"), torch.randn(2, 2, 64, device="cuda")
    caches = [torch.empty(2, 0, 2, 64, device="cuda") for _ in range(2)]
    out = ops.walk_attention_step(q, kv, kv, *caches, torch.tensor([0, -1]).cuda(),
                                  slopes=torch.ones(2, device="cuda"),
                                  times=torch.ones(2, device="cuda"),
                                  k_times=torch.empty(2, 0, device="cuda"))
    assert torch.isnan(out[0]).all() and not out[1].any()
