"""The page operators and the batched attention from their definitions, for the tests: page tables as Python lists, cache
contents as numpy arrays, attention in 64 bits."""
import numpy as np
import torch


class PageRef:
    """The tables of a KVPages and the pool contents of its layers (numpy arrays [4][capacity][row bytes] each)."""

    def __init__(self, table, lens, ref, page, pools=()):
        self.table = [list(map(int, r)) for r in table]
        self.len = [int(x) for x in lens]
        self.ref = [int(x) for x in ref]
        self.page = page
        self.pools = [np.array(p) for p in pools]

    @classmethod
    def of(cls, pages, layers=()):
        bufs = [t for kv in layers for t in (kv.k, kv.v, kv.ks, kv.vs) if t is not None]
        return cls(pages.table.cpu().tolist(), pages.len.cpu().tolist(), pages.ref.cpu().tolist(), pages.page,
                   [t.cpu().numpy() for t in bufs])

    def pages_of(self, m):
        return -(-m // self.page)

    def held(self, s):
        return min(len(self.table[s]), max(0, self.pages_of(self.len[s])))

    def _move(self, frm, to, rows):
        for p in self.pools:
            p[:, to * self.page:to * self.page + rows] = p[:, frm * self.page:frm * self.page + rows]

    def extend(self, seqs, add):
        seen, need_all = set(), 0
        for i, (s, a) in enumerate(zip(seqs, add)):
            if not 0 <= s < len(self.len) or s in seen or a < 0 or self.len[s] + a > len(self.table[s]) * self.page:
                return -(i + 1)
            seen.add(s)
        ref = list(self.ref)
        plans = []
        for s, a in zip(seqs, add):
            m = self.len[s]
            have = self.pages_of(m)
            copy = False
            if a > 0 and m % self.page:
                last = self.table[s][have - 1]
                copy = ref[last] > 1
                ref[last] -= copy
            need = self.pages_of(m + a) - have + copy
            need_all += need
            plans.append((s, a, have, copy, need))
        free = [p for p, r in enumerate(self.ref) if r <= 0]
        if need_all > len(free):
            return need_all - len(free)
        moves = []
        for s, a, have, copy, need in plans:
            m = self.len[s]
            got, free = free[:need], free[need:]
            for pg in got:
                self.ref[pg] = 1
            if copy:
                old = self.table[s][have - 1]
                self.ref[old] -= 1
                moves.append((old, got[0], m % self.page))
                self.table[s][have - 1] = got.pop(0)
            for k, pg in enumerate(got):
                self.table[s][have + k] = pg
            self.len[s] += a
        for mv in moves:
            self._move(*mv)
        return 0

    def fork(self, src, dst):
        rows = [None if s >= len(self.len) else ([], 0) if s < 0 else (self.table[s][:self.held(s)], self.len[s])
                for s in src]
        for i, d in enumerate(dst):
            if not 0 <= d < len(self.len) or rows[i] is None or d in list(dst)[i + 1:]:
                continue
            row, m = rows[i]
            for pg in row:
                self.ref[pg] += 1
            old = self.held(d)
            for e in range(old):
                self.ref[self.table[d][e]] -= 1
            for e in range(max(old, len(row))):
                self.table[d][e] = row[e] if e < len(row) else -1
            self.len[d] = m

    def trim(self, seqs, lens=None):
        for i, s in enumerate(seqs):
            if not 0 <= s < len(self.len) or s in list(seqs)[i + 1:]:
                continue
            keep = 0 if lens is None else lens[i]
            if not 0 <= keep <= self.len[s]:
                continue
            for e in range(self.pages_of(keep), self.held(s)):
                self.ref[self.table[s][e]] -= 1
                self.table[s][e] = -1
            self.len[s] = keep

    def compact(self):
        live = [p for p, r in enumerate(self.ref) if r > 0]
        n = len(live)
        holes = [p for p in range(n) if self.ref[p] <= 0]
        new = dict(zip([p for p in live if p >= n], holes))
        for frm, to in new.items():
            self._move(frm, to, self.page)
            self.ref[to], self.ref[frm] = self.ref[frm], 0
        for s in range(len(self.len)):
            for e in range(self.held(s)):
                self.table[s][e] = new.get(self.table[s][e], self.table[s][e])
        return n

    def check(self):
        """Every page is held as often as its count says."""
        want = [0] * len(self.ref)
        for s in range(len(self.len)):
            for e in range(self.held(s)):
                want[self.table[s][e]] += 1
        assert want == self.ref

    def same(self, pages, layers=()):
        got = PageRef.of(pages, layers)
        assert got.len == self.len
        assert got.table == self.table
        assert got.ref == self.ref
        for a, b in zip(got.pools, self.pools):
            assert np.array_equal(a, b)


def batch_attention(q, gate, rows, seen):
    """q, gate [T][24][256] and, per token, K / V rows (rows(t) -> [4][m][256] each, float64) of which it sees the first
    seen[t]: [T][24][256] in float64 on the CPU."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    q = q.double().cpu()
    for t, m in enumerate(seen):
        if m <= 0:
            continue
        K, V = rows(t)
        for g in range(4):
            s = q[t, 6 * g:6 * g + 6] @ K[g, :m].T / 16.0
            out[t, 6 * g:6 * g + 6] = torch.softmax(s, -1) @ V[g, :m]
    return out * torch.sigmoid(gate.double().cpu())
