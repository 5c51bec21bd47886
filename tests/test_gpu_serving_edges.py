"""Pages and beam search where rounding, masks and lengths are extreme, against their formulas in
float64 (tests/serving_formulas.py, tests/walk_formulas.py)."""
import pytest
import torch

from tests import walk_formulas as wf
from tests.test_gpu_serving import DTYPES, Pool, ops  # noqa: F401

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
