"""The pages of a cache on the device against their definition on lists: forks, reservations, frees, compactions and copies in sequences as a server makes them."""
import pytest
import torch

import int_flashattention_amd as ifa
from pages_reference import Books, make

pytestmark = pytest.mark.gpu

SHAPES = [((16, 48), torch.int8), ((5,), torch.float32), ((7,), torch.int8), ((3, 40, 64), torch.float16)]


def device(refs, table, lens, pools):
    i32 = dict(dtype=torch.int32, device="cuda")
    return torch.tensor(refs, **i32), torch.tensor(table, **i32), torch.tensor(lens, **i32), [p.cuda() for p in pools]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pick(g, hi, n, lo=0):
    return torch.randint(lo, hi, (n,), generator=g).tolist()


@pytest.mark.parametrize("pages,Z,width,page,fill", [(1, 1, 1, 16, 1), (40, 6, 5, 16, 4), (300, 33, 9, 64, 7), (5000, 300, 12, 32, 9), (9000, 1500, 4, 16, 3)])
def test_steps(pages, Z, width, page, fill):
    g = torch.Generator().manual_seed(pages + Z)
    start = make(g, pages, Z, width, page, fill, SHAPES)
    b = Books(*start, page)
    refs, table, lens, pools = device(*start)
    for step in range(6):
        n = max(1, min(Z, 1 + 7 * step))
        ended = pick(g, Z + 2, n // 3, -2)
        keep = pick(g, width * page, len(ended), -3) if step % 2 else None
        ifa.paged_free(refs, table, lens, ints(ended), page, None if keep is None else ints(keep))
        b.free(ended, keep)
        parents, children = pick(g, Z + 1, n, -1), pick(g, Z + 1, n, -1)
        ifa.paged_fork(refs, table, lens, ints(parents), ints(children))
        b.fork(parents, children)
        b.check(refs, table, lens, pools)
        fresh = pick(g, 2 if step % 3 else 3 * page, Z, -1)
        granted = ifa.paged_reserve(pools, refs, table, lens, ints(fresh), page)
        assert granted.tolist() == b.reserve(fresh), step
        b.check(refs, table, lens, pools)
        lens += granted
        b.lens = lens.tolist()
        if step % 2:
            assert ifa.paged_compact(pools, refs, table).tolist() == b.compact()
            b.check(refs, table, lens, pools)
    assert sum(b.refs) == sum(b.named(i) for r in b.table for i in r)


def test_pages_run_out():
    """Free pages are dealt in order; tokens that find none are not granted, and the last of those that share a page does not write it while another could not leave."""
    page = 16
    start = ([3, 1, 0, 1], [[0, -1], [0, -1], [0, -1], [1, -1], [3, -1]], [5, 5, 5, 16, 10], [torch.arange(4, dtype=torch.int32)[:, None].repeat(1, 9)])
    b = Books(*start, page)
    refs, table, lens, pools = device(*start)
    fresh = [1, 1, 1, 4, 20]
    granted = ifa.paged_reserve(pools, refs, table, lens, ints(fresh), page)
    assert granted.tolist() == [1, 0, 0, 0, 6] == b.reserve(fresh)
    b.check(refs, table, lens, pools)
    assert pools[0][2].tolist() == [0] * 9


def test_a_shared_page_is_copied_once_less_than_it_is_held():
    page = 16
    start = ([4] + [0] * 9, [[0, -1]] * 4, [7] * 4, [torch.arange(10, dtype=torch.int32)[:, None].repeat(1, 5)])
    b = Books(*start, page)
    refs, table, lens, pools = device(*start)
    assert ifa.paged_reserve(pools, refs, table, lens, 1, page).tolist() == [1] * 4 == b.reserve([1] * 4)
    b.check(refs, table, lens, pools)
    assert table[:, 0].tolist() == [1, 2, 3, 0] and refs.tolist()[:4] == [1] * 4


@pytest.mark.parametrize("n", [1, 5, 64, 777])
def test_beams_are_exchanged(n):
    g = torch.Generator().manual_seed(n)
    start = make(g, 3 * n + 4, n, 3, 16, 3, [])
    b = Books(*start, 16)
    refs, table, lens, _ = device(*start)
    parents = torch.randperm(n, generator=g).tolist()
    children = list(range(n))
    ifa.paged_fork(refs, table, lens, ints(parents), ints(children))
    b.fork(parents, children)
    b.check(refs, table, lens, [])
    assert all(r in (0, 1) for r in b.refs)                                 # (an exchange: nobody holds more or less)


def test_a_sequence_listed_twice():
    start = ([1, 1, 0, 1], [[0, 3, -1], [1, -1, -1]], [20, 3], [])
    for sequences, keep in (([0, 0], None), ([0, 0, 1], [18, 3, 0]), ([0, 0], [3, 18])):
        b = Books(*start, 16)
        refs, table, lens, _ = device(*start)
        ifa.paged_free(refs, table, lens, ints(sequences), 16, None if keep is None else ints(keep))
        b.free(sequences, keep)
        b.check(refs, table, lens, [])
    b = Books(*start, 16)
    refs, table, lens, _ = device(*start)
    ifa.paged_fork(refs, table, lens, ints([1, 0, 1]), ints([0, 0, 0]))
    b.fork([1, 0, 1], [0, 0, 0])
    b.check(refs, table, lens, [])


@pytest.mark.parametrize("bytes_,offset", [(1, 0), (3, 1), (4, 4), (12, 4), (16, 0), (16384, 0), (16385, 0), (50000, 16), (40960, 8)])
def test_copy_of_any_size_and_alignment(bytes_, offset):
    """Pages of a wider tensor, so that they lie apart; what is around them stays as it was."""
    g = torch.Generator().manual_seed(bytes_)
    whole = torch.randint(-128, 128, (23, bytes_ + 32), generator=g, dtype=torch.int8)
    dev = whole.cuda()
    order = torch.randperm(23, generator=g).tolist()
    src, dst = order[:9] + [-1, 23, 5], order[9:18] + [order[18], order[19], 100]
    ifa.paged_copy([dev[:, offset:offset + bytes_]], ints(src), ints(dst))
    for s, d in zip(src[:9], dst[:9]):
        whole[d, offset:offset + bytes_] = whole[s, offset:offset + bytes_]
    assert torch.equal(dev.cpu(), whole)


def test_many_pools():
    """More than a launch holds, of several types, for every call that copies."""
    g = torch.Generator().manual_seed(3)
    shapes = [((1 + i % 5, 8), (torch.int8, torch.float32, torch.bfloat16)[i % 3]) for i in range(203)]
    start = make(g, 30, 5, 4, 16, 3, shapes)
    b = Books(*start, 16)
    refs, table, lens, pools = device(*start)
    ifa.paged_copy(pools, ints([0, 1, 2]), ints([29, 28, 27]))
    b.copy([0, 1, 2], [29, 28, 27])
    ifa.paged_fork(refs, table, lens, ints([0, 0]), ints([1, 2]))
    b.fork([0, 0], [1, 2])
    assert ifa.paged_reserve(pools, refs, table, lens, 2, 16).tolist() == b.reserve([2] * 5)
    assert ifa.paged_compact(pools, refs, table).tolist() == b.compact()
    b.check(refs, table, lens, pools)


def test_books_without_pools_and_strided_tables():
    g = torch.Generator().manual_seed(9)
    start = make(g, 100, 9, 6, 32, 4, [])
    b = Books(*start, 32)
    refs, _, lens, _ = device(*start)
    wide = torch.full((9, 11), 77, dtype=torch.int32, device="cuda")
    table = wide[:, 2:8]
    table.copy_(ints(start[1]))
    assert ifa.paged_reserve([], refs, table, lens, 40, 32).tolist() == b.reserve([40] * 9)
    ifa.paged_fork(refs, table, lens, ints([0]), ints([8]))
    b.fork([0], [8])
    assert ifa.paged_compact((), refs, table).tolist() == b.compact()
    b.check(refs, table, lens, [])
    assert (wide[:, :2] == 77).all() and (wide[:, 8:] == 77).all()


def test_nothing_to_do():
    start = ([1, 0], [[0]], [4], [torch.zeros(2, 3)])
    refs, table, lens, pools = device(*start)
    ifa.paged_free(refs, table, lens, ints([]), 16)
    ifa.paged_fork(refs, table, lens, ints([]), ints([]))
    ifa.paged_copy(pools, ints([]), ints([]))
    assert ifa.paged_reserve(pools, refs, table, lens, 0, 16).tolist() == [0]
    assert ifa.paged_reserve(pools, refs, table, lens, -5, 16).tolist() == [0]
    assert (refs.tolist(), table.tolist(), lens.tolist()) == ([1, 0], [[0]], [4])


def test_captured_steps_follow_counts_and_lengths():
    """A step captured once and replayed, other work between the replays; two graphs whose workspaces come from one pool."""
    page = 16
    g = torch.Generator().manual_seed(5)
    start = make(g, 200, 12, 8, page, 5, SHAPES)
    refs, table, lens, pools = device(*start)
    parents, children, ended, fresh = ints([0, 1, 2]), ints([3, 4, 5]), ints([7]), ints([1] * 12)
    ifa.paged_reserve(pools, refs.clone(), table.clone(), lens, fresh, page)     # (loads what the first call loads)
    side = torch.cuda.Stream()
    step, tidy = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(step, stream=side):
            ifa.paged_free(refs, table, lens, ended, page)
            ifa.paged_fork(refs, table, lens, parents, children)
            granted = ifa.paged_reserve(pools, refs, table, lens, fresh, page)
            lens += granted
        with torch.cuda.graph(tidy, stream=side, pool=step.pool()):
            index = ifa.paged_compact(pools, refs, table)
    torch.cuda.synchronize()
    b = Books(*start, page)
    for t, x in zip((refs, table, lens), start):
        t.copy_(ints(x))
    for t, x in zip(pools, start[3]):
        t.copy_(x)
    for k in range(5):
        parents.copy_(ints([k, 1, 11 - k]))
        step.replay()
        b.free([7])
        b.fork([k, 1, 11 - k], [3, 4, 5])
        want = b.reserve([1] * 12)
        assert granted.tolist() == want
        b.lens = [n + w for n, w in zip(b.lens, want)]
        junk = torch.randn(1 << 20, device="cuda").sum()
        if k % 2:
            tidy.replay()
            assert index.tolist() == b.compact()
        torch.cuda.synchronize()
        b.check(refs, table, lens, pools)
        assert junk.isfinite()


@pytest.mark.parametrize("pages", [3000, 700])
def test_prompts_of_many_columns(pages):
    """Reservations of hundreds of columns beside short ones, over entries that are named already, shared ones among them; where the pages run out, in the middle of such a span."""
    g = torch.Generator().manual_seed(pages)
    Z, width, page = 40, 170, 16
    refs, table, lens = [0] * pages, [[-1] * width for _ in range(Z)], []
    order = torch.randperm(pages, generator=g).tolist()
    for z in range(Z):
        lens.append(pick(g, 60, 1)[0] if z % 3 else 0)
        for c in range(lens[z] // page + 1):
            table[z][c] = order.pop()
        if z % 5 == 1:                         # entries ahead of the tokens, one's own and shared ones
            for c in (7, 8, 70, 130):
                table[z][c] = order[c % 3] if c % 2 == 0 else order.pop()
    for row in table:
        for i in row:
            if i >= 0:
                refs[i] += 1
    start = (refs, table, lens, [torch.arange(pages, dtype=torch.int32)[:, None].repeat(1, 5)])
    b = Books(*start, page)
    refs, table, lens, pools = device(*start)
    fresh = [(2600, 3, 1500, 0, 90, 1040, 200)[z % 7] for z in range(Z)]
    granted = ifa.paged_reserve(pools, refs, table, lens, ints(fresh), page)
    want = b.reserve(fresh)
    assert granted.tolist() == want
    assert (sum(want) < sum(fresh)) == (pages == 700) or max(fresh) > width * page - 60
    b.check(refs, table, lens, pools)


@pytest.mark.parametrize("n", [2731, 4096])
def test_the_largest_forks(n):
    """As many pairs as a call takes, to distinct children and to few of them, over and over."""
    g = torch.Generator().manual_seed(n)
    Z, width, page = 5000, 3, 16
    start = make(g, 16000, Z, width, page, 3, SHAPES[1:2])
    b = Books(*start, page)
    refs, table, lens, pools = device(*start)
    for children in (torch.randperm(Z, generator=g)[:n].tolist(), pick(g, 9, n), pick(g, Z, n)):
        parents = pick(g, Z, n)
        ifa.paged_fork(refs, table, lens, ints(parents), ints(children))
        b.fork(parents, children)
        b.check(refs, table, lens, pools)


def test_the_largest_reservation_and_pool():
    """8192 sequences, each group of eight on one last page, and a pool longer than a stretch of the books."""
    Z, page, pages = 8192, 16, 40000
    shared = list(range(pages - 1, pages - 1 - Z // 8, -1))
    refs = [0] * pages
    for i in shared:
        refs[i] = 8
    for i in range(0, 30000, 3):
        refs[i] = 1
    start = (refs, [[shared[z % (Z // 8)], -1] for z in range(Z)], [5 + z % 9 for z in range(Z)], [torch.arange(pages, dtype=torch.int32)[:, None].repeat(1, 4)])
    b = Books(*start, page)
    refs, table, lens, pools = device(*start)
    fresh = [z % 3 for z in range(Z)]
    granted = ifa.paged_reserve(pools, refs, table, lens, ints(fresh), page)
    assert granted.tolist() == b.reserve(fresh)
    b.check(refs, table, lens, pools)
    assert ifa.paged_compact(pools, refs, table).tolist() == b.compact()
    b.check(refs, table, lens, pools)


def test_refusals():
    start = ([1, 0], [[0]], [4], [torch.zeros(2, 3)])
    refs, table, lens, pools = device(*start)
    for call, error in (
            (lambda: ifa.paged_copy([], ints([0]), ints([1])), ValueError),
            (lambda: ifa.paged_copy(pools[0], ints([0]), ints([1, 0])), ValueError),
            (lambda: ifa.paged_copy([torch.zeros(4, 6, device="cuda").t()], ints([0]), ints([1])), ValueError),
            (lambda: ifa.paged_copy([pools[0], torch.zeros(3, 3, device="cuda")], ints([0]), ints([1])), ValueError),
            (lambda: ifa.paged_copy([torch.zeros(2, 3)], ints([0]), ints([1])), RuntimeError),
            (lambda: ifa.paged_copy([3], ints([0]), ints([1])), TypeError),
            (lambda: ifa.paged_copy(pools, torch.tensor([0], device="cuda"), ints([1])), ValueError),
            (lambda: ifa.paged_free(refs, table, lens, ints([0]), 24), ValueError),
            (lambda: ifa.paged_free(refs.long(), table, lens, ints([0]), 16), ValueError),
            (lambda: ifa.paged_free(refs, table, lens, ints([0]), 16, ints([0, 1])), ValueError),
            (lambda: ifa.paged_fork(refs, table, lens[:0], ints([0]), ints([0])), ValueError),
            (lambda: ifa.paged_fork(refs, table, lens, ints([0] * 4097), ints([0] * 4097)), ValueError),
            (lambda: ifa.paged_fork(refs, table, lens, ints([0]), torch.tensor([0], dtype=torch.int32)), ValueError),
            (lambda: ifa.paged_reserve([torch.zeros(3, 3, device="cuda")], refs, table, lens, 1, 16), ValueError),
            (lambda: ifa.paged_reserve(pools, refs, table, lens, ints([1, 1]), 16), ValueError),
            (lambda: ifa.paged_compact(pools, refs, table[:, :0]), ValueError)):
        with pytest.raises(error):
            call()
    assert (refs.tolist(), table.tolist(), lens.tolist()) == ([1, 0], [[0]], [4])
