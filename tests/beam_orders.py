"""What a reordering of beams' pages has to do, and a search that uses it, in plain Python."""


def order(table, lens, parents, page_rows):
    """New rows of a group's table, new lengths, and copies (from page, to page, rows).

    A parent's first child takes its pages over.  A further child has the parent's full pages and,
    from there on, those of the next beam without children, with a copy of the parent's rows; where
    that page is part of what a beam with children holds, or takes other rows already, it has the
    parent's as well."""
    spare = [b for b in range(len(table)) if b not in parents]
    rows, copies, seen = [], [], set()
    for p in parents:
        full, left = divmod(max(lens[p], 0), page_rows)
        last, kept = p, full
        if p in seen:
            last = spare.pop(0)
            if left and full < len(table[p]):
                source, target = table[p][full], table[last][full]
                if any(table[b][full] == target and lens[b] // page_rows >= full
                       for b in parents) or any(t == target and s != source for s, t, _ in copies):
                    kept = full + 1
                else:
                    copies.append((source, target, left))
        seen.add(p)
        rows.append(table[p][:kept] + table[last][kept:])
    return rows, [lens[p] for p in parents], copies


def search(rng, orders, page_rows=4, pages=8, turns=30):
    """Random choices of parents, any of them, among beams that grow by an event a turn or have ended;
    yields (table, lens, parents) of each.  `orders` is `order` or computes the same."""
    beams = rng.choice([2, 3, 4, 5, 8])
    ids = list(range(beams * pages))
    rng.shuffle(ids)
    table = [ids[b * pages:(b + 1) * pages] for b in range(beams)]
    lens = [rng.randint(0, 2 * page_rows)] * beams
    ended = [False] * beams
    for _ in range(min(turns, page_rows * pages - lens[0])):
        lens = [n + (not e) for n, e in zip(lens, ended)]
        ended = [e or rng.random() < 0.15 for e in ended]
        some = beams if rng.random() < 0.7 else 2
        parents = [rng.randrange(some) for _ in range(beams)]
        yield table, lens, parents
        table, lens, _ = orders(table, lens, parents, page_rows)
        ended = [ended[p] for p in parents]
