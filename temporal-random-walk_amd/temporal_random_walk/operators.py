"""Operators of a sequence model over walks, on PyTorch tensors.

The sampler leaves walks in device memory as padded rows with lengths; these
are the operators that a model trained on them, and asked one event at a time,
spends its time in:

* :func:`walk_attention` -- attention inside each walk, forward and backward;
* :func:`walk_attention_step` -- one new event of each walk over its cache;
* :func:`relative_bias` -- a learned bias by buckets of distance as a dense
  array, for models with an attention of their own (the other two take the
  table itself).

They run hand-written gfx950 kernels (``libtrw_operators.so``, whose C ABI is
``include/trw_operators.h``; ``operators_capi`` has it by ctypes) on the current
stream of the tensors' device, wait for nothing, and follow PyTorch's rules for
tensors used on several streams.  There is no CPU path.  Import ``torch`` before the engine in one process:
PyTorch brings a HIP runtime of its own, which has to come up first.

Scores, softmax, sums and gradients are float32 whatever the inputs' type.  The
softmax's weights and their gradients are rounded to float16 or bfloat16 where
those are the inputs' type, as operands of the matrix instructions, so results
are up to 1.5 times as far from exact ones as if they had been rounded once, at
the end.
"""
from __future__ import annotations

import math
import os

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
if not os.path.exists(os.path.join(HERE, "libtrw_operators.so")):
    raise ImportError("libtrw_operators.so is missing: build it first "
                      "(python temporal-random-walk_amd/build.py)")

from . import _operators  # noqa: E402

MAX_REACH = 1024
MAX_BUCKETS = 256


def _require(ok, message):
    if not ok:
        raise ValueError(message)


def distance_buckets(num_buckets, reach, bidirectional=False, device="cuda"):
    """Bucket ids of the distances -reach..reach (query position minus key
    position), as the operators take them: an int32 tensor of 2 reach + 1.

    Distances 0, 1, ... back in time have a bucket each up to half of the
    buckets, then buckets that widen by a constant factor up to ``reach``.
    ``bidirectional``: the upper half of the buckets serves keys after the
    query alike; else those share bucket 0 (a causal mask sees none).  Any
    other tensor of 2 reach + 1 ids will do as well."""
    num_buckets, reach = int(num_buckets), int(reach)
    _require(1 <= num_buckets <= MAX_BUCKETS, f"1 to {MAX_BUCKETS} buckets")
    _require(0 <= reach <= MAX_REACH, f"reach must be 0 to {MAX_REACH}")
    after = num_buckets // 2 if bidirectional else 0
    before = num_buckets - after

    def of(n, count):
        exact = max(1, count // 2)
        if n < exact:
            return n
        wide = math.log(max(2.0, (reach + 1) / exact))
        return min(count - 1, exact + int(math.log(n / exact) / wide * (count - exact)))

    ids = []
    for d in range(-reach, reach + 1):
        if d >= 0:
            ids.append(of(d, before))
        else:
            ids.append(before + of(-d - 1, after) if after else 0)
    return torch.tensor(ids, dtype=torch.int32, device=device)


class WalkMask:
    """Which keys each query of a batch of walks sees; built on the device once
    per batch and used by every layer, forward and backward.

    A document (walk, history) of ``a`` queries over ``b`` keys has its queries
    at the last ``a`` of the keys' positions.  ``kind``: ``"full"`` (all keys of
    the document), ``"causal"`` (up to the query's own position) or
    ``"prefix"`` (causal, and the document's first ``prefix`` keys).  Rows of
    padding, rows of no document and queries that come before every key see
    nothing: their output and gradients are zero.

    Lengths and offsets stay on the device and are not read back; values out of
    range are clamped.

    :meth:`record_stream` is for a mask that is used on another stream than the
    one that was current when it was made, as a tensor's is."""

    def __init__(self, mask, kind):
        self._mask = mask
        self.kind = kind
        self.q_rows, self.k_rows = mask.q_rows, mask.k_rows
        # leading dimensions of q; of k and v
        self.q_shape, self.k_shape = tuple(mask.q_shape), tuple(mask.k_shape)
        self.device = mask.info.device

    def record_stream(self, stream):
        self._mask.info.record_stream(stream)

    @classmethod
    def padded(cls, lens, length, *, k_lens=None, k_length=None, kind="causal", prefix=None):
        """Walks as the sampler leaves them: ``[walks, length]`` rows, of which
        the first ``lens[w]`` are walk w's.  ``k_lens``/``k_length``: keys that
        are not the queries' own rows."""
        return cls(_operators.padded_mask(lens, length, k_lens, k_length, kind, prefix), kind)

    @classmethod
    def packed(cls, offsets, rows, *, k_offsets=None, k_rows=None, kind="causal", prefix=None):
        """Documents one after another: document w has the rows
        ``offsets[w]`` up to ``offsets[w + 1]`` of ``rows``."""
        return cls(_operators.packed_mask(offsets, rows, k_offsets, k_rows, kind, prefix), kind)


def walk_attention(q, k, v, mask, *, scale=None, softcap=0.0, bias_table=None, buckets=None,
                   slopes=None, times=None, k_times=None):
    """Attention inside each walk (document) of a batch.

    ``q``: ``[walks, length, heads, dim]`` for a padded mask, ``[rows, heads,
    dim]`` for a packed one; ``k`` and ``v`` alike with ``kv_heads``, which the
    query heads share in order (head h reads key head h // (heads // kv_heads)).
    float32, float16 or bfloat16; ``dim`` a multiple of 8 up to 128.  Strides
    are free where rows are 16-byte pieces (slices of one projection are);
    others are copied.

    score(i, j) = cap(scale q_i . k_j) + bias_table[h, buckets[reach + d]]
    - slopes[h] |t_i - t_j|, where cap(x) = softcap tanh(x / softcap)
    (``softcap`` 0: none), d is the distance in positions clamped to
    [-reach, reach] (``buckets``: int32 ids of 2 reach + 1 distances,
    :func:`distance_buckets`) and t are ``times`` and ``k_times`` (float32, of
    the rows' shape; without them, positions; subtract an origin from integer
    timestamps first, of which float32 holds 24 bits).  ``scale``: 1 / sqrt(dim)
    unless given.  -inf in the table masks.

    Returns the output in q's shape; differentiable by q, k, v and bias_table
    (once), also under checkpointing.  Arguments that change between the passes
    are an error, as PyTorch's own.  Equal inputs give equal results, bit for bit.  A row that sees no
    key is zero.  Values that are not finite stay within their own walk."""
    _require(isinstance(mask, WalkMask), "mask must be a WalkMask")
    return _operators.walk_attention(q, k, v, mask._mask, scale, softcap, bias_table, buckets,
                                     slopes, times, k_times)


def walk_attention_step(q, k, v, k_cache, v_cache, lens, *, scale=None, softcap=0.0,
                        bias_table=None, buckets=None, slopes=None, times=None, k_times=None):
    """One new event of each of a batch of walks: appends ``k`` and ``v``
    (``[batch, kv_heads, dim]``) to the caches at position ``lens[b]`` and
    returns the attention of ``q`` (``[batch, heads, dim]``) over positions 0
    to ``lens[b]``.  The caller counts ``lens`` up.

    ``k_cache``, ``v_cache``: ``[batch, capacity, kv_heads, dim]`` (a transposed
    view of another order will do; dim contiguous, rows 16-byte pieces, none of
    them shared: no expanded view).  With
    ``times`` (``[batch]``), ``k_times`` (``[batch, capacity]``, contiguous) is
    a cache as well and is written at ``lens[b]``.  The other arguments are
    :func:`walk_attention`'s; there is no gradient, and a result that is
    differentiated says so.

    A negative length is an idle row: output 0, caches untouched.  Where the
    table masks every position the output is 0 too.  A full cache
    (``lens[b] >= capacity``) gives NaN and leaves the caches untouched."""
    return _operators.walk_attention_step(q, k, v, k_cache, v_cache, lens, scale, softcap,
                                          bias_table, buckets, slopes, times, k_times)


def relative_bias(table, buckets, q_len, k_len, q_offset=0):
    """``out[h, i, j] = table[h, buckets[reach + clamp(i + q_offset - j, -reach,
    reach)]]``: the dense ``[heads, q_len, k_len]`` bias of a learned table
    ``[heads, num_buckets]``, in the table's type; differentiable by the table
    (once).  ``buckets``: as for :func:`walk_attention`."""
    return _operators.relative_bias(table, buckets, q_len, k_len, q_offset)
