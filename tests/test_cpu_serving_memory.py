"""CPU checks of where pages lie: keys, values and their scales that share memory are refused before a
GPU is touched."""
import ctypes

import pytest

from temporal_random_walk import operators_capi as abi

HEADS, DIM, ROWS, COUNT = 2, 64, 16, 5
LINES = HEADS * ROWS


def _write(dtype, k, v, k_scale=None, v_scale=None, strides=None, pages=COUNT, rows=0):
    """Addresses, and strides in bytes; of no rows unless given, so that nothing is launched."""
    size = 1 if dtype == 3 else 2
    strides = strides or [LINES * DIM * size] * 2 + [LINES] * 2
    p = abi.PagedCopyParams(
        pages=abi.Pages(dtype=dtype, kv_heads=HEADS, dim=DIM, page_rows=ROWS, pages=pages, k=k, v=v,
                        k_scale=k_scale, v_scale=v_scale, k_stride=strides[0] // size,
                        v_stride=strides[1] // size, k_scale_stride=strides[2],
                        v_scale_stride=strides[3], table=4096, table_stride=4, table_pages=4, walks=3),
        dtype=2, rows=3 * rows, length=rows, k=abi.Rows(4096, HEADS * DIM, DIM),
        v=abi.Rows(4096, HEADS * DIM, DIM))
    abi.call(abi.lib().trw_ops_paged_write, ctypes.byref(p), None)


PAGE8 = LINES * DIM
FAR = 1 << 30


@pytest.mark.parametrize("dtype", [2, 3])
def test_pools_that_share_memory(dtype):
    page = LINES * DIM * (1 if dtype == 3 else 2)
    scales = (3 * FAR, 4 * FAR) if dtype == 3 else ()
    _write(dtype, FAR, FAR + COUNT * page, *scales)
    _write(dtype, FAR + COUNT * page, FAR, *scales)
    for off in (0, 16, page, COUNT * page - 16):
        for a, b in ((FAR, FAR + off), (FAR + off, FAR)):
            for rows in (0, 10):
                with pytest.raises(ValueError, match="share memory"):
                    _write(dtype, a, b, *scales, rows=rows)
    _write(dtype, FAR, FAR + page, *scales, pages=1)
    with pytest.raises(ValueError, match="share memory"):
        _write(dtype, FAR, FAR + page - 16, *scales, pages=1)
    with pytest.raises(ValueError, match="share memory"):
        _write(dtype, FAR, FAR + page, *scales, strides=[2 * page, 3 * page, LINES, LINES])
    _write(dtype, FAR, FAR, *scales, pages=0)


def test_scales_that_share_memory():
    own = dict(k=FAR, v=2 * FAR, k_scale=3 * FAR, v_scale=4 * FAR)
    _write(3, **own)
    for name, other in (("k_scale", "v_scale"), ("v_scale", "k_scale"), ("k_scale", "k"),
                        ("v_scale", "k"), ("k_scale", "v"), ("v_scale", "v")):
        with pytest.raises(ValueError, match="share memory"):
            _write(3, **{**own, name: own[other]})
        size = LINES if "scale" in other else PAGE8
        with pytest.raises(ValueError, match="share memory"):
            _write(3, **{**own, name: own[other] + COUNT * size - 16})
        _write(3, **{**own, name: own[other] + COUNT * size})


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (3, 2, 1, 0), (2, 0, 3, 1)])
def test_records(order):
    """Keys, values and scales of a page in one record."""
    sizes = [PAGE8, PAGE8, LINES, LINES]
    at, place = FAR, [0] * 4
    for i in order:
        place[i], at = at, at + sizes[i]
    record = at - FAR
    _write(3, *place, strides=[record] * 4)
    for i in range(4):
        for by in (-16, 16, 5 * record + 16, -record - 16):
            moved = list(place)
            moved[i] += by
            if abs(by) < 4 * record:
                with pytest.raises(ValueError, match="share memory"):
                    _write(3, *moved, strides=[record] * 4)
    # other pages of the same pool
    apart = [place[0], place[1] + record, place[2] - record, place[3] + 2 * record]
    _write(3, *apart, strides=[record] * 4)


def test_every_call_refuses_them():
    p = abi.Pages(dtype=2, kv_heads=HEADS, dim=DIM, page_rows=ROWS, pages=COUNT, k=FAR, v=FAR + 16,
                  k_stride=PAGE8, v_stride=PAGE8, table=4096, table_stride=4, table_pages=4, walks=3)
    lib = abi.lib()
    rows = abi.Rows(4096, HEADS * DIM, DIM)
    copy = abi.PagedCopyParams(pages=p, dtype=2, rows=3, length=1, k=rows, v=rows)
    step = abi.PagedStepParams(pages=p, dtype=2, heads=HEADS, lens=4096, score=abi.Score(0.125, 0.0),
                               q=rows, k=rows, v=rows, out=rows)
    caches = (abi.Pages * 1)(p)
    reorder = abi.BeamReorderParams(beams=1, page_rows=ROWS, count=1, groups=3, pages=COUNT,
                                    table_pages=4, table_stride=4, table=4096, out_table=1 << 20,
                                    lens=8192, out_lens=1 << 21, parents=4096, caches=caches)
    for call, x in ((lib.trw_ops_paged_write, copy), (lib.trw_ops_paged_read, copy),
                    (lib.trw_ops_paged_step, step), (lib.trw_ops_beam_reorder, reorder)):
        with pytest.raises(ValueError, match="share memory"):
            abi.call(call, ctypes.byref(x), None)
