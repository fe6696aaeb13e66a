"""Reservations over pages that are shared ahead of their tokens (sequences forked after a reservation): of all that want a copy of a page in one call, the last keeps it if nobody else holds
it, in whichever column; the others get copies."""
import random

import pytest
import torch

import int_flashattention_amd as ifa

pytestmark = pytest.mark.gpu


def reserve(refs, table, lens, fresh, page, pool):
    """The rule on lists, in place; pool: a number a page.  Returns what is granted."""
    free = [i for i, r in enumerate(refs) if r <= 0]
    held = list(refs)
    named = lambda i: 0 <= i < len(refs)  # noqa: E731
    spans = []
    for row, n, m in zip(table, lens, fresh):
        n, m = max(0, n), max(0, m)
        first = min(n // page, len(row))
        spans.append((n, m, first, first if m == 0 else min(-(-(n + m) // page), len(row))))
    reached = {}
    for z, (_, _, first, end) in enumerate(spans):
        for c in range(first, end):
            if named(table[z][c]) and held[table[z][c]] > 1:
                reached.setdefault(table[z][c], []).append((z, c))
    kept = {entries[-1] for i, entries in reached.items() if len(entries) == held[i]}
    granted, out, was = [], False, list(pool)
    for z, (n, m, first, end) in enumerate(spans):
        room = end
        for c in range(first, end):
            i = table[z][c]
            if named(i) and held[i] <= 1:
                continue
            if (z, c) in kept:
                if out:                        # another could not leave
                    room = c
                    break
                continue
            if not free:
                out, room = True, c
                break
            new = free.pop(0)
            refs[new] = 1
            if named(i):
                refs[i] -= 1
                pool[new] = was[i]
            table[z][c] = new
        granted.append(max(0, min(m, room * page - n)))
    return granted


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check(refs, table, lens, fresh, page):
    pool = list(range(1000, 1000 + len(refs)))
    dev = ints(refs), ints(table), ints(lens), [ints(pool)[:, None].repeat(1, 3)]
    refs, table, pool = list(refs), [list(r) for r in table], list(pool)
    granted = ifa.paged_reserve(dev[3], *dev[:3], ints(fresh), page).tolist()
    want = reserve(refs, table, lens, fresh, page, pool)
    assert granted == want
    assert (dev[1].tolist(), dev[0].tolist()) == (table, refs)
    assert dev[2].tolist() == lens and dev[3][0].tolist() == [[v] * 3 for v in pool]
    return want, table, refs


def test_sequences_forked_after_a_reservation():
    """Two that hold three pages, the second and third without a token yet: one of them gets copies, the other keeps them; with a short pool both are served."""
    for free in (3, 9):
        want, table, refs = check([2, 2, 2] + [0] * free, [[0, 1, 2], [0, 1, 2]], [5, 5], [43, 40], 16)
        assert want == [43, 40] and table == [[3, 4, 5], [0, 1, 2]] and refs[:6] == [1] * 6
    # one page too few: the first is cut short, and the second, behind the last free page, is granted nothing that had to be shared out
    want, table, refs = check([2, 2, 2, 0, 0], [[0, 1, 2], [0, 1, 2]], [5, 5], [43, 40], 16)
    assert want == [27, 0] and table == [[3, 4, 2], [0, 1, 2]] and refs == [1, 1, 2, 1, 1]


def test_holders_that_do_not_reach_the_page():
    check([3, 3] + [0] * 6, [[0, 1]] * 3, [3, 3, 3], [20, 2, 25], 16)
    check([2, 2] + [0] * 6, [[0, 1], [-1, -1], [0, 1]], [3, 0, 3], [20, 20, 0], 16)


def test_a_column_that_is_one_sequence_s_first_and_another_s_later_one():
    check([1, 2, 1, 2] + [0] * 5, [[0, 1, 3], [2, 1, 3]], [20, 3], [20, 40], 16)
    check([1, 2, 1, 2] + [0] * 5, [[0, 1, 3], [2, 1, 3]], [3, 20], [40, 20], 16)
    check([2, 2, 0, 0, 0], [[0, 1], [0, 1]], [16, 16], [3, 3], 16)             # (the first column holds no token yet)


def test_a_page_that_a_sequence_names_twice():
    check([1, 2] + [0] * 4, [[0, 1, 1]], [2], [40], 16)
    check([1, 3, 1] + [0] * 4, [[0, 1, 1], [2, -1, 1]], [2, 2], [40, 40], 16)


@pytest.mark.parametrize("width", [4, 9, 90])
@pytest.mark.parametrize("seed", range(12))
def test_random(seed, width):
    """Groups of sequences on common pages, some of their own among them, spans short and long, with and without enough pages; more sequences than one round of the books."""
    r, page = random.Random(seed * 100 + width), 16
    Z = r.choice((3, 20, 130)) if seed < 10 else 1500
    refs, table = [], []
    while len(table) < Z:
        base = [len(refs) + c for c in range(width)]
        refs += [0] * width
        for _ in range(r.choice((1, 2, 3, 8))):
            row = []
            for c in range(width):
                kind = r.random()
                if kind < 0.7:
                    row.append(base[c])
                elif kind < 0.8:
                    row.append(-1)
                else:
                    row.append(len(refs))
                    refs.append(0)
            table.append(row)
    table = table[:Z]
    refs += [0] * r.choice((0, 5, Z, Z * width))
    for row in table:
        for i in row:
            if i >= 0:
                refs[i] += 1
    lens = [r.randint(0, width * page) // r.choice((1, 1, 4)) for _ in range(Z)]
    fresh = [r.choice((0, 1, 5, 17, 40, 200, width * page)) for _ in range(Z)]
    check(refs, table, lens, fresh, page)


def test_captured_and_replayed():
    """A step of forks and reservations ahead, whose counters the call before has used: replayed on other books each time."""
    page, Z, width, pages = 16, 6, 5, 60
    refs, table, lens, fresh = ints([0] * pages), ints([[-1] * width] * Z), ints([0] * Z), ints([0] * Z)
    pool = [torch.zeros((pages, 3), dtype=torch.int32, device="cuda")]
    ifa.paged_reserve(pool, refs, table, lens, fresh, page)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        granted = ifa.paged_reserve(pool, refs, table, lens, fresh, page)
    torch.cuda.synchronize()
    r = random.Random(1)
    for _ in range(6):
        rows = [[c if r.random() < 0.8 else -1 for c in range(width)] for _ in range(Z)]
        counts = [sum(row.count(i) for row in rows) for i in range(pages)]
        n, m = [r.randint(0, 40) for _ in range(Z)], [r.choice((0, 3, 30, 60)) for _ in range(Z)]
        values = list(range(pages))
        for t, x in zip((refs, table, lens, fresh, pool[0]), (counts, rows, n, m, [[v] * 3 for v in values])):
            t.copy_(ints(x))
        graph.replay()
        junk = torch.randn(1 << 20, device="cuda").sum()
        want = reserve(counts, rows, n, m, page, values)
        assert granted.tolist() == want and table.tolist() == rows and refs.tolist() == counts and pool[0].tolist() == [[v] * 3 for v in values]
        assert junk.isfinite()
