"""What a launch or a cache cannot take is refused as an argument, before anything is queued (no GPU
needed: the addresses are never followed)."""
import ctypes

import pytest

from tests.test_cpu_operators import _abi, _attention


def _sized(abi, backward, **changes):
    """The pass itself and its workspace's size refuse alike."""
    lib = abi.lib()
    p = _attention(abi, docs_info=4096, d_table=4096, workspace=4096, workspace_bytes=1 << 62,
                   **changes)
    size = ctypes.c_uint64()
    run = lib.trw_ops_attention_backward if backward else lib.trw_ops_attention_forward
    for call in (lambda: abi.call(run, ctypes.byref(p), None),
                 lambda: abi.call(lib.trw_ops_attention_workspace, ctypes.byref(p), backward,
                                  ctypes.byref(size))):
        with pytest.raises(ValueError, match="too many rows, documents or heads"):
            call()


WALKS = dict(longest=80, covered=1, q_rows=(1 << 29) - 64, k_rows=(1 << 29) - 64)


@pytest.mark.parametrize("backward,changes", [
    # 64 threads for a walk and key head (forward): 2^26 of them are too many
    (0, dict(WALKS, docs=(1 << 24), heads=4, kv_heads=4)),
    # 192 where walks have up to 96 rows (backward)
    (1, dict(WALKS, docs=(1 << 24), heads=2, kv_heads=2)),
    # 256 for a tile of 128 rows and a head
    (0, dict(docs=1, q_rows=(1 << 30) - 1, heads=4, kv_heads=2, k_rows=100)),
    (1, dict(docs=1, q_rows=(1 << 30) - 1, heads=4, kv_heads=2, k_rows=100)),
    (1, dict(docs=1, q_rows=100, k_rows=(1 << 30) - 1, heads=8, kv_heads=4)),
])
def test_launches_of_too_many_threads(backward, changes):
    _sized(_abi(), backward, **changes)


def test_bias_of_too_many_rows():
    abi = _abi()
    p = abi.BiasParams(dtype=0, heads=2, num_buckets=4, reach=8, q_len=1 << 27, k_len=1 << 20,
                       table=4096, buckets=4096, out=4096)
    with pytest.raises(ValueError, match="too many rows, documents or heads"):
        abi.call(abi.lib().trw_ops_relative_bias, ctypes.byref(p), None)


@pytest.mark.parametrize("stride", ["k_batch_stride", "v_batch_stride", "k_pos_stride",
                                    "v_pos_stride", "k_head_stride", "v_head_stride"])
def test_caches_whose_rows_share_memory(stride):
    """An expanded view: two walks would write to one row."""
    abi = _abi()
    rows = lambda h: abi.Rows(4096, h * 64, 64)  # noqa: E731
    p = abi.StepParams(dtype=2, heads=4, kv_heads=2, dim=64, batch=3, capacity=50, lens=4096,
                       score=abi.Score(0.125, 0.0), q=rows(4), k=rows(2), v=rows(2), out=rows(4),
                       k_cache=4096, v_cache=4096, k_batch_stride=6400, k_pos_stride=128,
                       k_head_stride=64, v_batch_stride=6400, v_pos_stride=128, v_head_stride=64,
                       workspace=4096, workspace_bytes=1 << 40)
    setattr(p, stride, 0)
    with pytest.raises(ValueError, match="share memory"):
        abi.call(abi.lib().trw_ops_attention_step, ctypes.byref(p), None)


def test_sizes_below_the_limits():
    """A size's call goes through, so that the refusals are the limits' own."""
    abi = _abi()
    size = ctypes.c_uint64()
    for backward, changes in ((0, dict(WALKS, docs=(1 << 24) - 16, heads=3, kv_heads=3)),
                              (1, dict(WALKS, docs=(1 << 23), heads=2, kv_heads=2)),
                              (0, dict(docs=1, q_rows=(1 << 30) - 2048, heads=1, kv_heads=1))):
        p = _attention(abi, docs_info=4096, **changes)
        abi.call(abi.lib().trw_ops_attention_workspace, ctypes.byref(p), backward,
                 ctypes.byref(size))
