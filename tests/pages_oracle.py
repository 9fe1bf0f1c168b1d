"""Plain restatements of the cache-page operators for the tests: the bookkeeping
as a sequential program, attention in 64 bits."""
import numpy as np


class Book:
    """table, n_ctx, refs and what the calls do to them, one request after another.
    moves: (from page, to page, rows) that fork and compact copy."""

    def __init__(self, n_slot, max_pages, n_pages, page):
        self.page = page
        self.table = np.full((n_slot, max_pages), -1, np.int32)
        self.n_ctx = np.zeros(n_slot, np.int32)
        self.refs = np.zeros(n_pages, np.int32)

    def _take(self):
        p = int(np.flatnonzero(self.refs == 0)[0])
        self.refs[p] = 1
        return p

    def extend(self, n_new):
        pos0 = np.full(len(self.n_ctx), -1, np.int32)
        n_free = int((self.refs == 0).sum())
        asked = 0
        for s, add in enumerate(n_new):
            if add <= 0:
                continue
            n = int(self.n_ctx[s])
            pos0[s] = -2
            if n + add > self.table.shape[1] * self.page:
                continue
            have, want = -(-n // self.page), -(-(n + add) // self.page)
            asked += want - have
            if want > have and asked > n_free:
                continue
            for k in range(have, want):
                self.table[s, k] = self._take()
            pos0[s] = n
            self.n_ctx[s] = n + add
        return pos0

    def fork(self, src, dst):
        status, moves = np.zeros(len(src), np.int32), []
        before, named = self.n_ctx.copy(), set()
        for i, (s, d) in enumerate(zip(src, dst)):
            slots = range(len(before))
            first = d not in named
            named.add(d)
            if s not in slots or d not in slots or not first or before[d] != 0:
                status[i] = 1
                continue
            n, rows = int(before[s]), int(before[s]) % self.page
            if rows and not (self.refs == 0).any():
                status[i] = 2
                continue
            whole = n // self.page
            for k in range(whole):
                self.table[d, k] = self.table[s, k]
                self.refs[self.table[s, k]] += 1
            if rows:
                self.table[d, whole] = self._take()
                moves.append((int(self.table[s, whole]), int(self.table[d, whole]), rows))
            self.n_ctx[d] = n
        return status, moves

    def free(self, slots):
        for s in slots:
            if not 0 <= s < len(self.n_ctx):
                continue
            for k in range(-(-int(self.n_ctx[s]) // self.page)):
                self.refs[self.table[s, k]] -= 1
                self.table[s, k] = -1
            self.n_ctx[s] = 0

    def compact(self):
        n_live = int((self.refs > 0).sum())
        p = np.arange(len(self.refs))
        frm, to = p[(self.refs > 0) & (p >= n_live)], p[(self.refs == 0) & (p < n_live)]
        new = p.copy()
        new[frm] = to
        self.refs[to], self.refs[frm] = self.refs[frm], 0
        held = self.table >= 0
        self.table[held] = new[self.table[held]]
        return n_live, [(int(f), int(t), self.page) for f, t in zip(frm, to)]


def attention(Q, K, V, n_new):
    """Q [T, H, 64], K, V [n, G, 64] (float64): rows t < n_new of the newest
    positions. Returns O and A = sum_j w_j |V_j|, both [n_new, H, 64]."""
    n, G = K.shape[:2]
    H = Q.shape[1]
    O, A = np.zeros((n_new, H, 64)), np.zeros((n_new, H, 64))
    for h in range(H):
        k, v = K[:, h // (H // G)], V[:, h // (H // G)]
        s = Q[:n_new, h] @ k.T / 8.0
        for t in range(n_new):
            end = n - n_new + t + 1
            if end > 0:
                w = np.exp(s[t, :end] - s[t, :end].max())
                w /= w.sum()
                O[t, h], A[t, h] = w @ v[:end], w @ np.abs(v[:end])
    return O, A
