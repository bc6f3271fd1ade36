"""The page tables by hand, on the host: lists, one row and one page at a time."""


class Tables:
    def __init__(self, refs, table, lens, page):
        self.refs, self.table, self.lens, self.page = list(refs), [list(r) for r in table], list(lens), page
        self.width = len(self.table[0])
        self.most = min(self.width * page, 262144)

    def valid(self, i):
        return 0 <= self.lens[i] <= self.most

    def held(self, x):
        return 0 <= x < len(self.refs)

    def trim(self, keep):
        for i, k in enumerate(keep):
            k = max(k, 0)
            if self.valid(i) and k < self.lens[i]:
                for c in range(-(-k // self.page), -(-self.lens[i] // self.page)):
                    if self.held(self.table[i][c]):
                        self.refs[self.table[i][c]] -= 1
                    self.table[i][c] = -1
                self.lens[i] = k

    def fork(self, parents):
        for i, p in enumerate(parents):
            if 0 <= p < len(parents) and p != i and parents[p] < 0 and self.lens[i] == 0 and self.valid(p) and self.lens[p]:
                for c in range(-(-self.lens[p] // self.page)):
                    x = self.table[i][c] = self.table[p][c]
                    if self.held(x):
                        self.refs[x] += 1
                self.lens[i] = self.lens[p]

    def extend(self, add):
        """(granted, copies as (from, to))"""
        free = [x for x, r in enumerate(self.refs) if r <= 0]
        before, at, granted, copies, out = list(self.refs), 0, [], [], False
        for i, n in enumerate(add):
            if not self.valid(i) or n > 0 and n > self.most - self.lens[i]:
                granted.append(0)
                continue
            if n <= 0:
                granted.append(1)
                continue
            have, want = -(-self.lens[i] // self.page), -(-(self.lens[i] + n) // self.page)
            last = self.table[i][have - 1] if self.lens[i] % self.page else -1
            copy = self.held(last) and before[last] > 1
            need = want - have + copy
            if need and (out or at + need > len(free)):
                out = True
                granted.append(0)
                continue
            for c in range(have - copy, want):
                x = free[at]
                at += 1
                if c < have:
                    copies.append((last, x))
                    self.refs[last] -= 1
                self.table[i][c] = x
                self.refs[x] = 1 if self.refs[x] <= 0 else self.refs[x] + 1
            self.lens[i] += n
            granted.append(1)
        return granted, copies

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        moves = list(zip([x for x in range(n, len(self.refs)) if self.refs[x] > 0],
                         [x for x in range(n) if self.refs[x] <= 0]))
        to = dict(moves)
        for a, z in moves:
            self.refs[z], self.refs[a] = self.refs[a], 0
        for x in range(n, len(self.refs)):
            self.refs[x] = 0
        for i, row in enumerate(self.table):
            have = -(-self.lens[i] // self.page) if self.valid(i) else 0
            self.table[i] = [to.get(x, x) if c < have else -1 for c, x in enumerate(row)]
        return moves
