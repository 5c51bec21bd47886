"""CPU checks of the reordering's formula (tests/beam_orders.py): beams keep their histories, whatever
their parents are."""
import random

from tests import beam_orders as bo

ROWS = 4
# two parents that ended early, and two longer beams that share a past and are dropped
TWO_SHORT = ([[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11], [8, 9, 14, 15]], [20, 20, 41, 41],
             [0, 0, 1, 1], 16)


def test_one_page_takes_one_childs_rows():
    rows, lens, copies = bo.order(*TWO_SHORT)
    assert copies == [(1, 9, 4)] and lens == [20] * 4
    assert rows == [[0, 1, 2, 3], [0, 9, 10, 11], [4, 5, 6, 7], [4, 5, 14, 15]]


def test_histories_are_kept():
    for seed in range(1000):
        rng = random.Random(seed)
        held, before, histories, turn = {}, None, None, 0
        for table, lens, parents in bo.search(rng, bo.order, ROWS):
            beams = range(len(table))
            if histories is None:
                before = [max(0, n - 1) for n in lens]
                histories = [[("first", b, i) for i in range(before[b])] for b in beams]
                for b in beams:
                    for i, event in enumerate(histories[b]):
                        held[table[b][i // ROWS], i % ROWS] = event
            for b in beams:  # what a step writes
                if lens[b] > before[b]:
                    histories[b].append((turn, b))
                    held[table[b][before[b] // ROWS], before[b] % ROWS] = (turn, b)
            assert [[held[table[b][i // ROWS], i % ROWS] for i in range(lens[b])]
                    for b in beams] == histories
            rows, before, copies = bo.order(table, lens, parents, ROWS)
            targets = {}
            for source, target, _ in copies:  # in any order
                assert targets.setdefault(target, source) == source
            assert not targets.keys() & {source for source, _, _ in copies}
            for source, target, left in copies:
                for i in range(left):
                    held[target, i] = held[source, i]
            histories = [list(histories[p]) for p in parents]
            assert [[held[rows[b][i // ROWS], i % ROWS] for i in range(before[b])]
                    for b in beams] == histories
            turn += 1
