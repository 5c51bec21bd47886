"""Pages and beam search in float64 on the CPU, element by element."""
import math

import torch

# every value of e4m3, by its code (NaN twice)
CODES = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def eight_bits(rows):
    """Codes' values and exponents of rows [..., dim] (float64): the smallest power of two that brings
    a row's largest finite size to 448 or less, within -117 .. 120, and the nearest code, ties to the
    one of an even number; NaN where a value is not finite."""
    size = rows.abs().where(rows.isfinite(), 0.0)
    e = torch.empty(rows.shape[:-1])
    for at, top in zip(range(e.numel()), size.amax(-1).flatten().tolist()):
        n = -117
        while top > 448 * 2.0 ** n and n < 120:
            n += 1
        e.view(-1)[at] = n
    e = e.double()
    x = rows / torch.exp2(e)[..., None]
    positive = CODES[:127]  # 0 .. 448, rising
    after = torch.searchsorted(positive, x.abs().nan_to_num(0.0).contiguous()).clamp(max=126)
    below = (after - 1).clamp(min=0)
    up, down = positive[after] - x.abs(), x.abs() - positive[below]
    code = torch.where(up < down, after, torch.where(up > down, below, after - after % 2))
    value = positive[code] * torch.sign(x)
    return torch.where(rows.isfinite(), value, math.nan), e


def choice(logits, scores, width, ended=None, end=None):
    """(scores, tokens, parents, ended) of one group: logits [beams, nodes] in float64."""
    beams, nodes = logits.shape
    found = []
    for b in range(beams):
        score = float(scores[b])
        if not math.isfinite(score):
            continue
        if ended is not None and ended[b]:
            found.append((-score, b, end))
            continue
        top = logits[b].max()
        if not torch.isfinite(top) or torch.isnan(logits[b]).any():
            continue
        share = (logits[b] - top) - torch.log(torch.exp(logits[b] - top).sum())
        # the best ones of a row are among its `width` largest logits, lower nodes first
        for x in torch.sort(share, descending=True, stable=True)[1][:width].tolist():
            if share[x] > -math.inf:
                found.append((-(score + float(share[x])), b, x))
    found.sort()
    found = found[:width] + [None] * (width - len(found))
    none = (-math.inf, 0 if end is None else end, 0, True)
    rows = [none if f is None else
            (-f[0], f[2], f[1], f[2] == end or bool(ended is not None and ended[f[1]]))
            for f in found]
    return [list(x) for x in zip(*rows)]


def reorder(table, lens, parents, page_rows):
    """New rows of a table, new lengths, and copies (from page, to page, rows) of one group."""
    spare = [b for b in range(len(table)) if b not in parents]
    rows, new, copies, seen = [], [], [], set()
    for p in parents:
        full, left = divmod(max(lens[p], 0), page_rows)
        last = p
        if p in seen:
            last = spare.pop(0)
            if left and full < len(table[p]):
                copies.append((table[p][full], table[last][full], left))
        seen.add(p)
        rows.append(table[p][:full] + table[last][full:])
        new.append(lens[p])
    return rows, new, copies
