"""CPU checks of pages and beam search: what they cannot run is refused before a GPU is touched, and
the formulas that the GPU tests use hold."""
import ctypes
import math

import pytest
import torch

from tests import serving_formulas as sf


def _abi():
    from temporal_random_walk import operators_capi
    return operators_capi


def _ops():
    from temporal_random_walk import operators
    return operators


def _changed(p, changes):
    for name, value in changes.items():
        at, *path = name.split("__")
        target = p
        while path:
            target, at = getattr(target, at), path.pop(0)
        setattr(target, at, value)
    return p


def _pages(abi, **changes):
    """Pages that pass every check (their addresses are never followed)."""
    return _changed(abi.Pages(dtype=3, kv_heads=2, dim=64, page_rows=16, pages=9, k=4096, v=4096,
                              k_scale=4096, v_scale=4096, k_stride=2048, v_stride=2048,
                              k_scale_stride=32, v_scale_stride=32, table=4096, table_stride=4,
                              table_pages=4, walks=3), changes)


PAGES = [
    (dict(dtype=4), "dtype"), (dict(dim=24), "multiple of 16"), (dict(dtype=2, dim=12), "head size"),
    (dict(dim=144), "head size"), (dict(kv_heads=0), "heads"), (dict(page_rows=8), "page_rows"),
    (dict(page_rows=48), "page_rows"), (dict(page_rows=2048), "page_rows"), (dict(pages=-1), "pages"),
    (dict(pages=1 << 31), "pages"), (dict(k=None), "null"), (dict(v=4100), "aligned"),
    (dict(k_stride=2032), "share memory"), (dict(v_stride=2056), "16 bytes"),
    (dict(k_stride=1 << 41), "2.40"), (dict(k_scale=None), "scales are null"),
    (dict(v_scale=4104), "scales must be"), (dict(k_scale_stride=16), "share memory"),
    (dict(v_scale_stride=40), "16 bytes"), (dict(walks=-1), "walks"), (dict(walks=1 << 30), "walks"),
    (dict(table=None), "table is null"), (dict(table_stride=-4), "table_stride"),
    (dict(table_pages=1 << 26), "rows"), (dict(table_pages=-1), "rows"),
]


def _copy(abi, **changes):
    p = abi.PagedCopyParams(pages=_pages(abi), dtype=2, rows=30, length=10, k=abi.Rows(4096, 128, 64),
                            v=abi.Rows(4096, 128, 64))
    return _changed(p, changes)


def _step(abi, **changes):
    p = abi.PagedStepParams(pages=_pages(abi), dtype=2, heads=4, lens=4096, score=abi.Score(0.125, 0.0),
                            q=abi.Rows(4096, 256, 64), k=abi.Rows(4096, 128, 64),
                            v=abi.Rows(4096, 128, 64), out=abi.Rows(4096, 256, 64))
    return _changed(p, changes)


@pytest.mark.parametrize("changes,message", PAGES)
def test_pages_refusals(changes, message):
    abi = _abi()
    lib = abi.lib()
    inside = {"pages__" + n: x for n, x in changes.items()}
    size = ctypes.c_uint64()
    for call in (lambda: abi.call(lib.trw_ops_paged_write, ctypes.byref(_copy(abi, **inside)), None),
                 lambda: abi.call(lib.trw_ops_paged_read, ctypes.byref(_copy(abi, **inside)), None),
                 lambda: abi.call(lib.trw_ops_paged_step, ctypes.byref(_step(abi, **inside)), None),
                 lambda: abi.call(lib.trw_ops_paged_step_workspace, ctypes.byref(_step(abi, **inside)),
                                  ctypes.byref(size))):
        with pytest.raises(ValueError, match=message):
            call()


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=3), "dtype"), (dict(pages__dtype=1), "pages' type"), (dict(rows=31), "walks"),
    (dict(rows=-1), "rows"), (dict(rows=1 << 30), "rows"), (dict(offsets=4096, counts=4096), "counts"),
    (dict(k__data=None), "k is null"), (dict(v__row_stride=130), "strides"),
    (dict(k__row_stride=1 << 23), "strides"), (dict(times=4096), "go together"),
    (dict(k_times=4096), "go together"),
])
def test_copy_refusals(changes, message):
    abi = _abi()
    for function in (abi.lib().trw_ops_paged_write, abi.lib().trw_ops_paged_read):
        with pytest.raises(ValueError, match=message):
            abi.call(function, ctypes.byref(_copy(abi, **changes)), None)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=3), "dtype"), (dict(pages__dtype=0), "pages' type"), (dict(heads=3), "heads"),
    (dict(lens=None), "lens"), (dict(q__data=4104), "aligned"), (dict(out__head_stride=4), "strides"),
    (dict(score__scale=math.inf), "scale"), (dict(score__softcap=-1.0), "softcap"),
    (dict(score__table=4096), "bucket"), (dict(score__q_times=4096), "times"),
    (dict(score__q_times=4096, score__k_times=4096), "slopes"),
    (dict(pages__walks=1 << 20), "too many"), (dict(workspace=4104), "workspace"),
    (dict(pages__table_pages=64), "workspace is too small"),
])
def test_step_refusals(changes, message):
    abi = _abi()
    with pytest.raises(ValueError, match=message):
        abi.call(abi.lib().trw_ops_paged_step, ctypes.byref(_step(abi, **changes)), None)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=3), "dtype"), (dict(beams=0), "1 to 32"), (dict(beams=33), "1 to 32"),
    (dict(width=0), "1 to 32"), (dict(width=33), "1 to 32"), (dict(groups=-1), "groups"),
    (dict(nodes=0), "nodes"), (dict(nodes=1 << 30), "nodes"), (dict(end_token=9000), "end_token"),
    (dict(end_token=-2), "end_token"), (dict(ended=4096, end_token=-1), "end_token"),
    (dict(logits=None), "logits"), (dict(logits=4097), "misaligned"), (dict(out_tokens=None), "outputs"),
    (dict(workspace=4104), "workspace"), (dict(workspace_bytes=8), "too small"),
    (dict(groups=1 << 24, workspace_bytes=1 << 62), "too many"),
])
def test_select_refusals(changes, message):
    abi = _abi()
    p = abi.BeamSelectParams(dtype=2, beams=8, width=8, groups=3, nodes=9000, logits=4096,
                             group_stride=72000, beam_stride=9000, scores=4096, end_token=-1,
                             out_scores=4096, out_tokens=4096, out_parents=4096, out_ended=4096,
                             workspace=4096, workspace_bytes=1 << 20)
    with pytest.raises(ValueError, match=message):
        abi.call(abi.lib().trw_ops_beam_select, ctypes.byref(_changed(p, changes)), None)


@pytest.mark.parametrize("changes,message", [
    (dict(beams=0), "beams"), (dict(beams=33), "beams"), (dict(groups=-1), "groups"),
    (dict(count=0), "at least one"), (dict(caches=None), "at least one"),
    (dict(page_rows=24), "page_rows"), (dict(pages=-1), "pages"), (dict(pages=8), "alike"),
    (dict(page_rows=32), "alike"), (dict(lens=None), "lens"), (dict(out_lens=8192), "lens"),
    (dict(table=None), "table is null"), (dict(out_table=None), "out_table"),
    (dict(out_table=4096), "out_table"), (dict(table_stride=-1), "table_stride"),
])
def test_reorder_refusals(changes, message):
    abi = _abi()
    caches = (abi.Pages * 1)(_pages(abi))
    p = abi.BeamReorderParams(beams=4, page_rows=16, count=1, groups=3, pages=9, table_pages=4,
                              table_stride=4, table=4096, out_table=1 << 20, lens=8192,
                              out_lens=1 << 21, parents=4096, caches=caches)
    with pytest.raises(ValueError, match=message):
        abi.call(abi.lib().trw_ops_beam_reorder, ctypes.byref(_changed(p, changes)), None)


def test_null_arguments():
    abi = _abi()
    lib = abi.lib()
    for function in (lib.trw_ops_paged_write, lib.trw_ops_paged_read, lib.trw_ops_paged_step,
                     lib.trw_ops_beam_select, lib.trw_ops_beam_reorder):
        with pytest.raises(ValueError, match="null"):
            abi.call(function, None, None)
    with pytest.raises(ValueError, match="null"):
        abi.call(lib.trw_ops_paged_step_workspace, ctypes.byref(_step(abi)), None)


def test_tensors_on_the_cpu_are_refused():
    ops = _ops()
    pages = ops.Pages.empty(3, 16, 2, 64, dtype=torch.float8_e4m3fn, device="cpu")
    assert pages.k.shape == pages.v.shape == (3, 2, 16, 64) and pages.k_scale.dtype == torch.uint8
    x, n = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int64)
    table = torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: ops.paged_write(pages, table, None, x[None], x[None]),
                 lambda: ops.paged_read(pages, table, lens=n, length=4),
                 lambda: ops.paged_attention_step(x, x, x, pages, table, n),
                 lambda: ops.beam_select(x, n.float(), 2),
                 lambda: ops.beam_reorder(table, n, n[None], [pages])):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


def test_the_limits_of_the_header():
    import os
    import re

    from tests.test_cpu_operators import HEADER
    assert os.path.exists(HEADER)
    assert int(re.search(r"#define TRW_OPS_BEAMS (\d+)", open(HEADER).read()).group(1)) == \
        _ops().MAX_BEAMS


def test_codes_are_the_nearest_ones():
    """The formula's rounding is PyTorch's, and no value is further off than the documentation says."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(200, 16, generator=gen, dtype=torch.float32) * torch.exp2(
        torch.randint(-60, 60, (200, 1), generator=gen).float())
    codes, e = sf.eight_bits(x.double())
    scaled = x.double() / torch.exp2(e)[:, None]
    assert torch.equal(codes, scaled.float().to(torch.float8_e4m3fn).double())
    top = scaled.abs().amax(-1)
    assert (top <= 448).all() and (top > 224).all()
    assert ((codes - scaled).abs() <= (scaled.abs() / 16).clamp(min=2.0 ** -10)).all()


def test_a_choice_against_all_sums():
    gen = torch.Generator().manual_seed(1)
    logits = torch.randn(3, 40, generator=gen, dtype=torch.float64)
    scores = torch.tensor([-1.0, -0.5, -3.0])
    s, t, p, e = sf.choice(logits, scores, 6)
    all_of = (scores.double()[:, None] + torch.log_softmax(logits, -1)).flatten()
    best, at = all_of.sort(descending=True, stable=True)
    assert [a * 40 + b for a, b in zip(p, t)] == at[:6].tolist() and not any(e)
    assert torch.allclose(torch.tensor(s, dtype=torch.float64), best[:6], atol=1e-12)
    s, t, p, e = sf.choice(logits, torch.tensor([-1.0, -math.inf, 0.0]), 2,
                           [False, False, True], 7)
    assert (s[0], t[0], p[0], e[0]) == (0.0, 7, 2, True)


def test_a_reordering_moves_only_what_it_must():
    table = [[0, 1], [2, 3], [4, 5]]
    rows, lens, copies = sf.reorder(table, [20, 20, 20], [1, 1, 0], 16)
    assert rows == [[2, 3], [2, 5], [0, 1]] and lens == [20, 20, 20] and copies == [(3, 5, 4)]
    assert sf.reorder(table, [16, 16, 16], [2, 2, 2], 16)[2] == []
