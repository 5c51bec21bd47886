"""Pages and beam search where rounding, masks and lengths are extreme, against their formulas in
float64 (tests/serving_formulas.py, tests/walk_formulas.py)."""
import pytest
import torch

from tests import walk_formulas as wf
from tests.test_gpu_serving import DTYPES, SIZES, Pool, _choose, _normal, ops  # noqa: F401

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
