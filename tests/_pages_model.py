"""What the calls of esda_pages.h and esda_tree_commit do, on lists: the tests' model."""


class Model:
    """table [slots][most], refs [pages], length [slots]; rows: {(page, row): value}, what a row holds."""

    def __init__(self, table, refs, length, page_rows, rows):
        self.table, self.refs, self.length = [r[:] for r in table], refs[:], length[:]
        self.R, self.rows, self.left_out = page_rows, dict(rows), 0

    def page(self, s, k):
        most = len(self.table[s])
        return self.table[s][k] if 0 <= k < most and 0 <= self.table[s][k] < len(self.refs) else None

    def held(self, s):
        return [p for p in self.table[s] if 0 <= p < len(self.refs)]

    def free(self, slots):
        for i, s in enumerate(slots):
            if not 0 <= s < len(self.table) or s in slots[:i]:
                self.left_out += 1
                continue
            for p in self.held(s):
                self.refs[p] -= 1
            self.table[s] = [-1] * len(self.table[s])
            self.length[s] = 0

    def reserve(self, slots, rows):
        most = len(self.table[0])
        lowest = [p for p, n in enumerate(self.refs) if n == 0]
        total = 0
        for i, (s, r) in enumerate(zip(slots, rows)):
            if not 0 <= s < len(self.table) or s in slots[:i] or not 0 <= r <= most * self.R or self.length[s] < 0:
                self.left_out += 1
                continue
            lack = [k for k in range(self.length[s] // self.R, (r + self.R - 1) // self.R) if self.page(s, k) is None]
            start, total = total, total + len(lack)
            if lack and total > len(lowest):
                self.left_out += 1
                continue
            for k, p in zip(lack, lowest[start:]):
                self.table[s][k] = p
                self.refs[p] = 1

    def fork(self, src, dst, rows=None):
        R, most = self.R, len(self.table[0])
        table0, length0, held = [r[:] for r in self.table], self.length[:], []
        entries = []
        for i, (s, d) in enumerate(zip(src, dst)):
            ok = d not in dst[:i] and 0 <= s < len(table0) and 0 <= d < len(table0)
            if ok:
                r = length0[s] if rows is None else min(rows[i], length0[s])
                ok = r >= 0 and length0[s] <= most * R and \
                    all(self.page(s, k) is not None for k in range((max(r, 0) + R - 1) // R))
            if not ok:
                self.left_out += 1
                continue
            full, part = r // R, r % R
            keep = s == d and part and full == length0[s] // R
            new = table0[s][:full + bool(keep)]
            entries.append([s, d, r, new, part and not keep])
            held.append([p for p in new if s != d])
        for (s, d, r, new, _), more in zip(entries, held):
            for p in more:
                self.refs[p] += 1
            for k, p in enumerate(table0[d]):
                if 0 <= p < len(self.refs) and not (s == d and k < len(new)):
                    self.refs[p] -= 1
        copied = [table0[s][r // R] for s, d, r, new, copies in entries if copies]
        for p in copied:
            self.refs[p] += 1
        before = self.refs[:]
        lowest = [p for p, n in enumerate(before) if n == 0]
        needs = 0
        moves = []
        for s, d, r, new, copies in entries:
            self.length[d] = r
            if copies:
                tail = table0[s][r // R]
                if s == d and before[tail] == 1:
                    new.append(tail)
                    self.refs[tail] += 1  # given back below
                elif needs < len(lowest):
                    new.append(lowest[needs])
                    self.refs[lowest[needs]] = 1
                    moves.append((tail, lowest[needs], r % R))
                    needs += 1
                else:
                    self.left_out += 1
                    for p in new:
                        self.refs[p] -= 1
                    new, self.length[d] = [], 0
                self.refs[tail] -= 1
            self.table[d] = new + [-1] * (most - len(new))
        old = dict(self.rows)
        for a, b, n in moves:
            for i in range(n):
                self.rows[b, i] = old[a, i]

    def compact(self):
        live = sum(n != 0 for n in self.refs)
        movers = [p for p, n in enumerate(self.refs) if n and p >= live]
        holes = [p for p, n in enumerate(self.refs) if not n and p < live]
        to = dict(zip(movers, holes))
        old = dict(self.rows)
        for a, b in to.items():
            for i in range(self.R):
                self.rows[b, i] = old[a, i]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in r] for r in self.table]

    def commit(self, accept, count):
        old = dict(self.rows)
        for s, (path, c) in enumerate(zip(accept, count)):
            n, path = self.length[s], path[:max(c, 0)]
            ok = n >= 0 and 0 <= c <= len(accept[s]) and all(0 <= a < 64 for a in path) and \
                all(a < b for a, b in zip(path, path[1:]))
            ok = ok and all(self.page(s, (n + j) // self.R) is not None for j in path + list(range(c)))
            if not ok:
                self.left_out += 1
                continue
            for i, a in enumerate(path):
                self.rows[self.page(s, (n + i) // self.R), (n + i) % self.R] = \
                    old[self.page(s, (n + a) // self.R), (n + a) % self.R]
            self.length[s] = n + c
