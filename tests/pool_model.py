"""Plain model of the page pool: lists and dicts, one request after the other."""

import numpy as np


class PoolModel:
    def __init__(self, num_pages, max_reqs, columns, layout):
        self.n, self.rows, self.columns, self.layout = num_pages, max_reqs, columns, layout
        self.bp, self.per = layout.physical_block_tokens, layout.blocks_per_page
        self.refs = [0] * num_pages
        self.refs[0] = 1
        self.pages = [[] for _ in range(max_reqs)]
        self.lens = [0] * max_reqs

    def take(self, k):
        free = [p for p in range(1, self.n) if self.refs[p] == 0][:k]
        for p in free:
            self.refs[p] = 1
        return free

    def free_count(self):
        return sum(r == 0 for r in self.refs)

    def fork(self, parents, children):
        """Result list and copies (src, dst, tokens, window)."""
        start, result, copies, out, named = list(self.lens), [], [], False, set()
        for a, c in zip(parents, children):
            first = c not in named
            named.add(c)
            if not (0 <= a < self.rows and 0 <= c < self.rows and first and start[a] > 0 and start[c] == 0):
                result.append(-1)
                continue
            n = start[a]
            need = 2 if n > self.bp and n % self.bp else 1
            out = out or need > self.free_count()
            if out:
                result.append(0)
                continue
            mine = list(self.pages[a])
            fresh = self.take(need)
            for p in mine[1:len(mine) - (need == 2)]:
                self.refs[p] += 1
            copies.append((mine[0], fresh[0], min(n, self.bp), True))
            mine[0] = fresh[0]
            if need == 2:
                copies.append((mine[-1], fresh[1], n % self.bp, False))
                mine[-1] = fresh[1]
            self.pages[c], self.lens[c] = mine, n
            result.append(1)
        return result, copies

    def resize(self, rows, lens):
        limit = self.columns // self.per * self.bp
        result, named = [-1] * len(rows), set()
        first = []
        for r in rows:
            first.append(r not in named)
            named.add(r)
        for i, (r, n) in enumerate(zip(rows, lens)):
            if 0 <= r < self.rows and first[i] and n == 0:
                for p in self.pages[r]:
                    self.refs[p] -= 1
                self.pages[r], self.lens[r] = [], 0
                result[i] = 1
        out = False
        for i, (r, n) in enumerate(zip(rows, lens)):
            if 0 <= r < self.rows and first[i] and n > 0 and self.lens[r] <= n <= limit:
                need = -(-n // self.bp) - len(self.pages[r])
                out = out or need > self.free_count()
                if need and out:
                    result[i] = 0
                    continue
                self.pages[r] = self.pages[r] + self.take(need)
                self.lens[r] = n
                result[i] = 1
        return result

    def compact(self):
        """(live, to, copies); pages above the live count move into the holes below it."""
        live = [p for p in range(1, self.n) if self.refs[p]]
        holes = [p for p in range(1, len(live) + 1) if not self.refs[p]]
        movers = [p for p in live if p > len(live)]
        to = [p if self.refs[p] else -1 for p in range(self.n)]
        copies = []
        for s, d in zip(movers, holes):
            to[s] = d
            used = max([min(self.bp, n - j * self.bp) for row, n in zip(self.pages, self.lens)
                        for j, p in enumerate(row) if p == s], default=0)
            copies.append((s, d, used, any(row and row[0] == s for row in self.pages)))
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.pages = [[to[p] for p in row] for row in self.pages]
        return len(live), to, copies

    def table(self):
        t = np.zeros((self.rows, self.columns), dtype=np.int32)
        for i, row in enumerate(self.pages):
            for j, p in enumerate(row):
                t[i, j * self.per:(j + 1) * self.per] = p * self.per + np.arange(self.per)
        return t

    def copy(self, history, window, copies):
        """Apply copies to numpy stripes (bytes) in place."""
        size, lay = self.layout.stripe_page_bytes, self.layout
        h, w = history.reshape(-1, size), window.reshape(-1, size)
        for s, d, tokens, owner in copies:
            k = tokens * lay.kv_heads * lay.config.slot_bytes
            h[d, :k] = h[s, :k]
            if owner:
                w[d, :lay.window_page_bytes] = w[s, :lay.window_page_bytes]
