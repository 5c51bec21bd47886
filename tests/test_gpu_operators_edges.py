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
