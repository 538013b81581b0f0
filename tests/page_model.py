"""The page operators' definition, row by row in plain Python, on the CPU."""
import torch

BAD_BLOCK, BAD_SEQLEN, NO_PAGES, BAD_ROW = 1, 2, 8, 16


class PageModel:
    def __init__(self, k, v, table, lens):
        """`k`, `v`: lists of CPU caches; all pages free."""
        self.k, self.v = [x.clone() for x in k], [x.clone() for x in v]
        self.nb, self.bs = k[0].shape[:2]
        self.refs = [0] * self.nb
        self.table = table.clone().tolist()
        self.lens = lens.tolist()
        self.status = 0

    def width(self):
        return len(self.table[0])

    def adopt(self):
        for row, s in zip(self.table, self.lens):
            for j in range(-(-s // self.bs)):
                if row[j] != -1:
                    self.refs[row[j]] += 1

    def _copy(self, src, dst, slots):
        for c in self.k + self.v:
            c[dst, :slots] = c[src, :slots]

    def resize(self, new, window=None, sinks=0):
        bs, cap = self.bs, self.width() * self.bs
        rows = []
        for r, n in enumerate(new):
            if n < 0:
                continue
            if n > cap or not 0 <= self.lens[r] <= cap:
                self.status |= BAD_SEQLEN
                continue
            rows.append(r)
        for r in rows:
            s, n = self.lens[r], new[r]
            q0 = min(s, n)
            for j in range(-(-s // bs)):
                gone = j >= -(-n // bs)
                if window is not None:
                    toks = range(j * bs, (j + 1) * bs)
                    gone = gone or (toks[0] >= sinks and toks[-1] <= q0 - window)
                if gone and self.table[r][j] != -1:
                    self._release(self.table[r][j])
                    self.table[r][j] = -1
        free = [p for p in range(self.nb) if self.refs[p] == 0]
        needs, cows = {}, {}
        for r in rows:
            s, n = self.lens[r], new[r]
            needs[r], cows[r] = 0, False
            if n > s:
                needs[r] = -(-n // bs) - -(-s // bs)
                if s % bs:
                    e = self.table[r][s // bs]
                    if not 0 <= e < self.nb:
                        self.status |= BAD_BLOCK
                    elif self.refs[e] > 1:
                        cows[r] = True
                needs[r] += cows[r]
        total, copies = 0, []
        for r in rows:
            s, n = self.lens[r], new[r]
            first = total
            total += needs[r]
            if needs[r] and total > len(free):
                self.status |= NO_PAGES
                continue
            pages = free[first:total]
            for p in pages:
                self.refs[p] = 1
            if cows[r]:
                copies.append((self.table[r][s // bs], pages[0], s % bs))
                self.table[r][s // bs] = pages.pop(0)
            for j, p in zip(range(-(-s // bs), -(-n // bs)), pages):
                self.table[r][j] = p
            self.lens[r] = n
        for src, dst, slots in copies:
            self.refs[src] -= 1
            self._copy(src, dst, slots)

    def _release(self, page):
        if not 0 <= page < self.nb or self.refs[page] == 0:
            self.status |= BAD_BLOCK
        else:
            self.refs[page] -= 1

    def fork(self, parents, children):
        bs, rows = self.bs, len(self.lens)
        before = list(self.lens)
        taken = set()
        free = [p for p in range(self.nb) if self.refs[p] == 0]
        used = 0
        todo = []
        for p, c in zip(parents, children):
            if p < 0 or c < 0:
                continue
            if p >= rows or c >= rows or before[c] != 0 or c in taken:
                self.status |= BAD_ROW
                continue
            taken.add(c)
            todo.append((p, c))
        for p, c in todo:
            s = before[p]
            if not 0 <= s <= self.width() * bs:
                self.status |= BAD_SEQLEN
                continue
            tail = None
            if s % bs:
                src = self.table[p][s // bs]
                if not 0 <= src < self.nb:
                    self.status |= BAD_BLOCK
                    continue
                if used == len(free):
                    self.status |= NO_PAGES
                    continue
                tail = free[used]
                used += 1
                self.refs[tail] = 1
                self._copy(src, tail, s % bs)
            full = s // bs
            for e in self.table[p][:full]:
                if 0 <= e < self.nb:
                    self.refs[e] += 1
            row = self.table[p][:full] + ([tail] if tail is not None else [])
            self.table[c] = row + [-1] * (self.width() - len(row))
            self.lens[c] = s

    def compact(self):
        live = [p for p in range(self.nb) if self.refs[p]]
        n = len(live)
        holes = [p for p in range(n) if not self.refs[p]]
        movers = [p for p in live if p >= n]
        to = dict(zip(movers, holes))
        for src, dst in to.items():
            self._copy(src, dst, self.bs)
            self.refs[dst], self.refs[src] = self.refs[src], 0
        for row in self.table:
            for j, e in enumerate(row):
                if e in to:
                    row[j] = to[e]
                elif e >= n:
                    self.status |= BAD_BLOCK
        return n

    def words(self):
        out = []
        for w in range(-(-self.nb // 32)):
            x = sum(1 << i for i in range(32) if w * 32 + i < self.nb and self.refs[w * 32 + i] == 0)
            out.append(x - (1 << 32) if x >= 1 << 31 else x)
        return out


def assert_same(model, pool, table, lens, k, v, what):
    torch.cuda.synchronize()
    assert table.tolist() == model.table, f"{what}: table"
    assert lens.tolist() == model.lens, f"{what}: lengths"
    assert pool.refs.tolist() == model.refs, f"{what}: counts"
    assert pool.free_words.tolist() == model.words(), f"{what}: free bits"
    assert pool.read_status() == model.status, f"{what}: status"
    for layer, (a, b) in enumerate(zip(k + v, model.k + model.v)):
        assert torch.equal(a.cpu().view(torch.int16), b.view(torch.int16)), f"{what}: cache {layer}"
