"""CPU checks of the operators' boundary: the library exports what its header declares, refuses what
it cannot run before it touches a GPU, and the formulas that the GPU tests use hold."""
import ctypes
import math
import os
import re

import pytest
import torch

from tests import walk_formulas as wf

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "trw_operators.h")


def _ops():
    from temporal_random_walk import operators
    return operators


def _abi():
    from temporal_random_walk import operators_capi
    return operators_capi


def test_library_exports_every_declared_symbol():
    ops, abi = _ops(), _abi()
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(trw_ops_[a-z_]+)\s*\(", text)))
    assert declared == sorted(abi.EXPORTS)
    lib = abi.lib()
    assert not [n for n in declared if not hasattr(lib, n)]
    version = int(re.search(r"#define TRW_OPS_ABI_VERSION (\d+)", open(HEADER).read()).group(1))
    assert lib.trw_ops_abi_version() == abi.ABI_VERSION == version
    assert b"gfx950" in open(abi.LIB_PATH, "rb").read()
    limits = dict(re.findall(r"#define TRW_OPS_(MAX_\w+) (\d+)", open(HEADER).read()))
    assert {k: int(v) for k, v in limits.items()} == {"MAX_REACH": ops.MAX_REACH,
                                                      "MAX_BUCKETS": ops.MAX_BUCKETS}


def _attention(abi, **changes):
    """Arguments that pass every check (their addresses are never followed: each test breaks one
    of them, or asks for a size only)."""
    rows = lambda h: abi.Rows(4096, h * 64, 64)  # noqa: E731
    p = abi.AttentionParams(dtype=2, heads=4, kv_heads=2, dim=64, q_rows=100, k_rows=100,
                             q_rows_info=4096, k_rows_info=4096,
                             score=abi.Score(0.125, 0.0), q=rows(4), k=rows(2), v=rows(2),
                             out=rows(4), stats=4096, d_out=rows(4), d_q=rows(4), d_k=rows(2),
                             d_v=rows(2))
    for name, value in changes.items():
        at, *path = name.split("__")
        target = p
        while path:
            target, at = getattr(target, at), path.pop(0)
        setattr(target, at, value)
    return p


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=3), "dtype"), (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "heads"),
    (dict(dim=60), "head size"), (dict(dim=136), "head size"), (dict(q_rows=-1), "rows"),
    (dict(q_rows=1 << 30), "rows"), (dict(k_rows=1 << 31), "rows"),
    (dict(q__data=None), "q is null"), (dict(k__data=4104), "16-byte aligned"),
    (dict(v__row_stride=129), "strides"), (dict(out__head_stride=4), "strides"),
    (dict(q_rows_info=None), "q_rows_info"), (dict(score__scale=math.nan), "scale"),
    (dict(score__softcap=-1.0), "softcap"), (dict(score__table=4096), "bucket"),
    (dict(score__table=4096, score__buckets=4096), "256 buckets"),
    (dict(score__table=4096, score__buckets=4096, score__num_buckets=257), "256 buckets"),
    (dict(score__table=4096, score__buckets=4096, score__num_buckets=4, score__reach=1025), "reach"),
    (dict(score__q_times=4096), "times"),
    (dict(score__q_times=4096, score__k_times=4096), "slopes"),
])
def test_attention_refusals(changes, message):
    abi = _abi()
    for function in (abi.lib().trw_ops_attention_forward, abi.lib().trw_ops_attention_backward):
        with pytest.raises(ValueError, match=message):
            abi.call(function, ctypes.byref(_attention(abi, **changes)), None)


@pytest.mark.parametrize("changes,message", [
    (dict(stats=None), "stats"), (dict(k_rows_info=None), "k_rows_info"),
    (dict(d_out__data=None), "d_out"), (dict(d_k__data=4100), "aligned"), ({}, "workspace"),
    (dict(score__table=4096, score__buckets=4096, score__num_buckets=4), "d_table"),
])
def test_backward_refusals(changes, message):
    abi = _abi()
    with pytest.raises(ValueError, match=message):
        abi.call(abi.lib().trw_ops_attention_backward, ctypes.byref(_attention(abi, **changes)),
                  None)


def test_null_arguments():
    abi = _abi()
    lib = abi.lib()
    for function in (lib.trw_ops_walk_mask, lib.trw_ops_attention_forward,
                     lib.trw_ops_attention_backward, lib.trw_ops_attention_step,
                     lib.trw_ops_relative_bias, lib.trw_ops_relative_bias_backward):
        with pytest.raises(ValueError, match="null"):
            abi.call(function, None, None)
    with pytest.raises(ValueError, match="null"):
        abi.call(lib.trw_ops_attention_workspace, ctypes.byref(_attention(abi)), 1, None)


@pytest.mark.parametrize("changes,message", [
    (dict(docs=-1), "docs"), (dict(kind=3), "kind"), (dict(q_rows=31), "docs"),
    (dict(k_rows=29), "docs"), (dict(q_rows_info=None), "info"), (dict(kind=2), "prefix"),
    (dict(q_offsets=4096), "lens"), (dict(k_offsets=4096), "q_offsets"),
    (dict(q_rows_info=4104), "aligned"),
])
def test_mask_refusals(changes, message):
    abi = _abi()
    p = abi.MaskParams(docs=3, q_rows=30, k_rows=30, q_length=10, k_length=10, q_lens=4096,
                        kind=1, q_rows_info=4096, k_rows_info=4096)
    for name, value in changes.items():
        setattr(p, name, value)
    with pytest.raises(ValueError, match=message):
        abi.call(abi.lib().trw_ops_walk_mask, ctypes.byref(p), None)


@pytest.mark.parametrize("changes,message", [
    (dict(batch=-1), "batch"), (dict(capacity=-1), "capacity"), (dict(lens=None), "lens"),
    (dict(k_cache=None), "k_cache"), (dict(v_cache=4104), "aligned"),
    (dict(k_batch_stride=1001), "batch strides"), (dict(v_pos_stride=129), "strides"),
    (dict(batch=1 << 20), "too many"),
])
def test_step_refusals(changes, message):
    abi = _abi()
    rows = lambda h: abi.Rows(4096, h * 64, 64)  # noqa: E731
    p = abi.StepParams(dtype=2, heads=4, kv_heads=2, dim=64, batch=3, capacity=50, lens=4096,
                        score=abi.Score(0.125, 0.0), q=rows(4), k=rows(2), v=rows(2), out=rows(4),
                        k_cache=4096, v_cache=4096, k_batch_stride=6400, k_pos_stride=128,
                        k_head_stride=64, v_batch_stride=6400, v_pos_stride=128, v_head_stride=64)
    for name, value in changes.items():
        setattr(p, name, value)
    with pytest.raises(ValueError, match=message):
        abi.call(abi.lib().trw_ops_attention_step, ctypes.byref(p), None)


@pytest.mark.parametrize("changes,message", [
    (dict(heads=0), "heads"), (dict(q_len=-1), "lengths"), (dict(reach=-1), "reach"),
    (dict(num_buckets=0), "buckets"), (dict(out=4100), "aligned"), (dict(out=None), "out is null"),
    (dict(q_offset=1 << 40), "q_offset"), (dict(dtype=-1), "dtype"),
])
def test_bias_refusals(changes, message):
    abi = _abi()
    p = abi.BiasParams(dtype=0, heads=2, num_buckets=4, reach=8, q_len=5, k_len=6, table=4096,
                        buckets=4096, out=4096)
    for name, value in changes.items():
        setattr(p, name, value)
    with pytest.raises(ValueError, match=message):
        abi.call(abi.lib().trw_ops_relative_bias, ctypes.byref(p), None)


def test_tensors_on_the_cpu_are_refused():
    ops = _ops()
    x = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.WalkMask.padded(torch.tensor([1, 2]), 4)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.relative_bias(torch.zeros(2, 4), ops.distance_buckets(4, 3, device="cpu"), 4, 4)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.walk_attention_step(x, x, x, x[None], x[None], torch.zeros(4))
    with pytest.raises(TypeError):
        ops.WalkMask.padded([1, 2], 4)


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("num,reach", [(1, 0), (2, 1), (8, 5), (32, 128), (256, 1024), (16, 3)])
def test_distance_buckets(num, reach, both):
    ids = _ops().distance_buckets(num, reach, both, device="cpu").tolist()
    assert len(ids) == 2 * reach + 1 and min(ids) >= 0 and max(ids) < num
    back = ids[reach:]
    assert back == sorted(back) and back[0] == 0
    count = num - (num // 2 if both else 0)
    exact = max(1, count // 2)
    assert back[:exact] == list(range(min(exact, reach + 1)))
    ahead = ids[:reach][::-1]
    if both and num > 1:
        assert ahead == sorted(ahead) and all(b >= count for b in ahead)
    else:
        assert all(b == 0 for b in ahead)


def test_formulas_against_autograd():
    """The gradients written out in walk_formulas are those of its own forward formula."""
    gen = torch.Generator().manual_seed(0)
    lens, heads, dim, cap = [5, 0, 9], 4, 8, 2.0
    q, do = (torch.randn(14, heads, dim, generator=gen, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(14, 2, dim, generator=gen, dtype=torch.float64) for _ in range(2))
    table = torch.randn(heads, 3, generator=gen, dtype=torch.float64)
    ids = torch.tensor([0, 0, 1, 2, 1], dtype=torch.int32)
    slopes = torch.rand(heads, generator=gen, dtype=torch.float64)
    docs = wf.documents("prefix", lens, lens, [2, 0, 20])
    got = wf.attention(q, k, v, docs, softcap=cap, table=table, buckets=ids, slopes=slopes, d_out=do)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, table)]
    outs = []
    a = 0
    for first, n, _, seen in docs:
        qs, ks, vs = (x[a:a + n].transpose(0, 1) for x in leaves[:3])
        ks, vs = ks.repeat_interleave(2, 0), vs.repeat_interleave(2, 0)
        hop = torch.arange(n)[:, None] - torch.arange(n)
        s = cap * torch.tanh(qs @ ks.mT / math.sqrt(dim) / cap)
        s = s + leaves[3][:, ids.long()[hop.clamp(-2, 2) + 2]]
        s = s - slopes[:, None, None] * hop.abs()
        outs.append((torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ vs).transpose(0, 1))
        a += n
    out = torch.cat(outs)
    assert torch.allclose(out, got["out"][0], atol=1e-12)
    for name, g in zip(("d_q", "d_k", "d_v", "d_table"), torch.autograd.grad(out, leaves, do)):
        assert torch.allclose(g, got[name][0], atol=1e-11), name
