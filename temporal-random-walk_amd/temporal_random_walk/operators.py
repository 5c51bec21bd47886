"""Operators of a sequence model over walks, on PyTorch tensors.

The sampler leaves walks in device memory as padded rows with lengths; these
are the operators that a model trained on them, and asked one event at a time,
spends its time in:

* :func:`walk_attention` -- attention inside each walk, forward and backward;
* :func:`walk_attention_step` -- one new event of each walk over its cache;
* :func:`relative_bias` -- a learned bias by buckets of distance as a dense
  array, for models with an attention of their own (the other two take the
  table itself);
* :class:`Pages`, :func:`paged_write`, :func:`paged_read`,
  :func:`paged_attention_step` -- caches in pages of a common pool, in 8 bits or
  as they are, for walks of very different and growing lengths;
* :func:`beam_select`, :func:`beam_reorder` -- forecasts of several events by
  beam search, over such caches.

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
from typing import NamedTuple, Optional

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
if not os.path.exists(os.path.join(HERE, "libtrw_operators.so")):
    raise ImportError("libtrw_operators.so is missing: build it first "
                      "(python temporal-random-walk_amd/build.py)")

from . import _operators  # noqa: E402

MAX_REACH = 1024
MAX_BUCKETS = 256
MAX_BEAMS = 32


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


class Pages(NamedTuple):
    """Keys and values of many walks in pages of one pool.

    ``k``, ``v``: ``[pages, kv_heads, page_rows, dim]``, each page contiguous
    (``page_rows``: a power of two, 16 to 1024), of memory of their own or parts of
    one record for each page.  Which pages are a walk's says a
    table, int32 ``[walks, pages of a walk]``, that all layers share: position p
    of walk w is row p % page_rows of page ``table[w, p // page_rows]``.  Entries
    outside the pool (-1, say) are no pages: nothing is written there, 0 is read,
    and steps do not see their positions.

    Rows are kept as they are (float32, float16, bfloat16), or in 8 bits: ``k``
    and ``v`` of ``torch.float8_e4m3fn``, and for each row and head a byte b of
    ``k_scale`` or ``v_scale`` (uint8 ``[pages, kv_heads, page_rows]``); a value
    is its code times 2^(b - 127), off by at most 1/16 of it or 2^-10 of that
    power (for rows whose largest value is below 2^-109, of 2^-117).  What is not
    finite becomes NaN.  ``dim`` is a multiple of 8 up to 128, of 16 in 8 bits."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages, page_rows, kv_heads, dim, *, dtype=torch.bfloat16, device="cuda"):
        """A pool whose rows are still to be written; ``dtype``
        ``torch.float8_e4m3fn`` for 8 bits."""
        def one(*shape, of=dtype):
            return torch.empty(pages, kv_heads, page_rows, *shape, dtype=of, device=device)

        k, v = one(dim), one(dim)
        if dtype != torch.float8_e4m3fn:
            return cls(k, v)
        return cls(k, v, one(of=torch.uint8), one(of=torch.uint8))

    def record_stream(self, stream):
        for x in self:
            if x is not None:
                x.record_stream(stream)


def paged_write(pages, table, starts, k, v, *, counts=None, offsets=None, times=None, k_times=None):
    """Rows of walks (prompts) to their pages: row i of walk w goes to position
    ``starts[w] + i`` (``starts`` None: i).

    ``k``, ``v``: ``[walks, length, kv_heads, dim]``, of which the first
    ``counts[w]`` rows are walk w's (None: all), or ``[rows, kv_heads, dim]`` with
    ``offsets`` (walk w has the rows ``offsets[w]`` up to ``offsets[w + 1]``).  Any
    of the three types goes to 8 bits, else the pages' own.  ``times`` (float32, of
    the rows' shape) go to ``k_times`` (``[pages, page_rows]``, contiguous).

    A walk of a negative start is left out, as are positions that have no page.
    Walks that are written at once need pages of their own there.  There is no
    gradient."""
    _operators.paged_write(pages, table, starts, k, v, counts, offsets, times, k_times)


def paged_read(pages, table, *, lens=None, length=None, offsets=None, rows=None, dtype=None,
               k_times=None):
    """Pages back to rows, as :func:`walk_attention` takes them for prompts over
    what is cached: ``k`` and ``v`` ``[walks, length, kv_heads, dim]`` of the first
    ``lens[w]`` positions of each walk, or ``[rows, kv_heads, dim]`` where walk w
    has the rows ``offsets[w]`` up to ``offsets[w + 1]``, from position 0 on; and,
    with ``k_times``, their times as a third tensor.  Rows of no walk, and of
    positions without a page, are 0.

    ``dtype``: what 8 bits are read as (bfloat16 unless given, which is exact); else
    the pages' own."""
    k, v, times = _operators.paged_read(pages, table, lens, length, offsets, rows, dtype, k_times)
    return (k, v) if times is None else (k, v, times)


def paged_attention_step(q, k, v, pages, table, lens, *, first=None, scale=None, softcap=0.0,
                         bias_table=None, buckets=None, slopes=None, times=None, k_times=None):
    """:func:`walk_attention_step` over pages: appends ``k`` and ``v``
    (``[batch, kv_heads, dim]``) at position ``lens[b]`` and returns the attention
    of ``q`` (``[batch, heads, dim]``) over positions ``first[b]`` (None: 0) to
    ``lens[b]``, the new one as the pages hold it.  The caller counts ``lens`` up.

    ``first``: for windows; what lies before is not read, and its pages may be
    another walk's by then.  More than ``lens[b]`` leaves the new event alone.
    ``table``: a row for each of the batch.  ``k_times``: ``[pages, page_rows]``,
    written at the new position.  The other arguments are
    :func:`walk_attention`'s; there is no gradient, and a result that is
    differentiated says so.

    A negative length is an idle row: output 0, nothing written.  Where there is
    no page for the new event the output is NaN, and nothing is written.  Rows of
    a batch may share pages but not the one that they write."""
    return _operators.paged_attention_step(q, k, v, pages, table, lens, first, scale, softcap,
                                           bias_table, buckets, slopes, times, k_times)


class BeamChoice(NamedTuple):
    """What :func:`beam_select` chose, ``[groups, width]``: scores (float32),
    nodes and parent beams (int64), and whether a beam has ended (bool)."""
    scores: torch.Tensor
    tokens: torch.Tensor
    parents: torch.Tensor
    ended: torch.Tensor


def beam_select(logits, scores, width, *, ended=None, end_token=None):
    """The ``width`` best continuations of each group's beams, best first.

    ``logits``: ``[groups, beams, nodes]`` of any of the three types (-inf: not a
    next node), ``scores``: float32 ``[groups, beams]``, each beam's log
    probability (-inf: no beam; a group that starts has one).  A continuation of
    beam b by node x scores ``scores[b] + log softmax(logits[b])[x]``; equal ones
    come by their beam, then by their node.  ``ended`` (bool ``[groups, beams]``):
    beams that have come to ``end_token`` continue as themselves, token
    ``end_token``.  Up to 32 beams and 32 of a width.

    A beam whose score is not finite, or whose logits hold NaN, +inf or nothing
    above -inf, has no continuations.  Where a group has fewer than ``width``: score -inf,
    parent 0, token ``end_token`` (0 without one), ended.  Exponentials are float32's
    and summed in float32, by parts of up to 4096 nodes; those sums' sum, its logarithm
    and the scores are float64, rounded at the end.  There is no gradient."""
    return BeamChoice(*_operators.beam_select(logits, scores, width, ended, end_token))


def beam_reorder(table, lens, parents, caches, *, k_times=None):
    """Makes the rows of a table, and their pages, those of chosen beams.

    Row ``g * beams + b`` of ``table`` and ``lens`` is beam b of group g; after it
    has been called, row ``g * beams + c`` of the table and lengths that it returns
    holds what beam ``parents[g, c]`` (``[groups, beams]``) held.  ``caches``: the
    :class:`Pages` of every layer, ``k_times`` as for
    :func:`paged_attention_step`.

    Beams share the full pages of their common past.  The page that is filled next,
    and those after it, go to a parent's first child; a further child takes those
    of a beam without children, with a copy of the rows: nothing else moves.  So
    each row of a group starts with pages of its own (a prompt is written to one
    row of each group, and ``parents`` 0 spreads it), and rows of a group have equal
    lengths, but for beams that have ended, which may be shorter (their children share
    their last page where a copy would take one that another beam's past or another
    child's copy lies in)."""
    return _operators.beam_reorder(table, lens, parents, list(caches), k_times)
