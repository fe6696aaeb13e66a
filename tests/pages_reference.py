"""The pages of a cache by their definition, on Python lists: what copies, forks, reservations, frees and compactions do to counts, table, lengths and pools."""
import torch


class Books:
    def __init__(self, refs, table, lens, pools, page):
        self.refs, self.table, self.lens, self.page = list(refs), [list(r) for r in table], list(lens), page
        self.pools = [p.clone() for p in pools]

    def named(self, i):
        return 0 <= i < len(self.refs)

    def copy(self, src, dst):
        for p in self.pools:
            was = p.clone()
            for s, d in zip(src, dst):
                if self.named(s) and self.named(d):
                    p[d] = was[s]

    def free(self, sequences, keep=None):
        for i, z in enumerate(sequences):
            if not 0 <= z < len(self.table):
                continue
            kept = max(0, min(self.lens[z], keep[i] if keep is not None else 0))
            for c in range(len(self.table[z])):
                if c * self.page >= kept:
                    if self.named(self.table[z][c]):
                        self.refs[self.table[z][c]] -= 1
                    self.table[z][c] = -1
            self.lens[z] = min(self.lens[z], kept)

    def fork(self, parents, children):
        rows, lens, Z = [list(r) for r in self.table], list(self.lens), len(self.table)
        last = {c: p for p, c in zip(parents, children) if 0 <= c < Z and 0 <= p < Z}
        for c, p in last.items():
            for new in rows[p]:
                if self.named(new):
                    self.refs[new] += 1
            for old in rows[c]:
                if self.named(old):
                    self.refs[old] -= 1
            self.table[c], self.lens[c] = list(rows[p]), lens[p]

    def reserve(self, fresh):
        refs, table = list(self.refs), [list(r) for r in self.table]
        free = [i for i, r in enumerate(refs) if r <= 0]
        was = [p.clone() for p in self.pools]
        granted, waiting, out = [], {}, False
        spans = []
        for z, row in enumerate(table):
            held, m = max(0, self.lens[z]), max(0, fresh[z])
            first = min(held // self.page, len(row))
            spans.append((held, m, first, first if m == 0 else min(-(-(held + m) // self.page), len(row))))
        for z, row in enumerate(table):
            held, m, first, end = spans[z]
            room = end
            for c in range(first, end):
                i = row[c]
                if self.named(i) and not (refs[i] > 1):
                    continue
                if self.named(i) and c == first:
                    before = waiting.get(i, 0)
                    waiting[i] = before + 1
                    if refs[i] - before <= 1:
                        if out:
                            room = c
                            break
                        continue
                if not free:
                    out, room = True, c
                    # what it would have taken is still counted for those behind it
                    break
                new = free.pop(0)
                self.refs[new] = 1
                if self.named(i):
                    self.refs[i] -= 1
                    for p, o in zip(self.pools, was):
                        p[new] = o[i]
                self.table[z][c] = new
            granted.append(max(0, min(m, room * self.page - held)))
        return granted

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        src = [i for i, r in enumerate(self.refs) if r > 0 and i >= used]
        dst = [i for i, r in enumerate(self.refs) if r <= 0 and i < used]
        index = [i if r > 0 else -1 for i, r in enumerate(self.refs)]
        for s, d in zip(src, dst):
            index[s] = d
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.copy(src, dst)
        self.table = [[index[i] if self.named(i) else i for i in r] for r in self.table]
        return index

    def check(self, refs, table, lens, pools):
        assert refs.tolist() == self.refs
        assert table.tolist() == self.table
        assert lens.tolist() == self.lens
        for a, b in zip(pools, self.pools):
            assert torch.equal(a.cpu(), b)


def make(g, pages, Z, width, page, fill, shapes):
    """Sequences of up to `fill` of their columns, and pools of the given shapes and types per page."""
    order = torch.randperm(pages, generator=g).tolist()
    table, refs, lens = [], [0] * pages, []
    for _ in range(Z):
        n = int(torch.randint(0, fill * page + 1, (1,), generator=g))
        used = min(-(-n // page), len(order))
        n = min(n, used * page)
        row = [order.pop() for _ in range(used)]
        for i in row:
            refs[i] = 1
        table.append(row + [-1] * (width - used))
        lens.append(n)
    pools = [torch.randint(-100, 100, (pages, *shape), generator=g).to(dtype) for shape, dtype in shapes]
    return refs, table, lens, pools
