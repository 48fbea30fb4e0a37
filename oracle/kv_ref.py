"""Oracle of the paged key / value cache, its attention and the verification of
drafted tokens -- TEST INFRASTRUCTURE ONLY.

Plain Python and numpy, request by request and token by token, from the
definitions in include/tensor_rocm.h; attention and the verification's sums in
float64. No counterpart in the reference (its paged attention kernel is never
launched, tensor_ops_cuda.cu:582-618): parity unpinned, checked against closed
forms in tests/test_oracle_kv.py."""
from __future__ import annotations

import numpy as np


class Refused(Exception):
    """The call changes nothing and is reported."""


class Cache:
    """kv [layers, 2, pages, heads, page, dim], table, lens, refs as numpy arrays."""

    def __init__(self, layers, heads, dim, page, pages, seqs, width, dtype=np.float32):
        self.kv = np.zeros((layers, 2, pages, heads, page, dim), dtype)
        self.table = np.full((seqs, width), -1, np.int32)
        self.lens = np.zeros(seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.P = page

    def _count(self, n):
        return -(-int(n) // self.P)

    def reserve(self, seq, count):
        table, lens, refs, kv = self.table.copy(), self.lens.copy(), self.refs.copy(), self.kv
        if len(set(seq)) != len(seq) or any(s < 0 or s >= len(lens) for s in seq) or any(k < 0 for k in count):
            raise Refused("bad request")
        before = self.refs
        free = [p for p in range(len(refs)) if before[p] == 0]
        copies = []
        for s, k in zip(seq, count):
            L = int(lens[s])
            if L + k > table.shape[1] * self.P:
                raise Refused("row too short")
            held = self._count(L)
            if k > 0 and L % self.P and before[table[s, held - 1]] > 1:
                if not free:
                    raise Refused("full")
                old, new = int(table[s, held - 1]), free.pop(0)
                copies.append((old, new, L % self.P))
                refs[old] -= 1
                refs[new] = 1
                table[s, held - 1] = new
            for j in range(held, self._count(L + k)):
                if not free:
                    raise Refused("full")
                table[s, j] = free.pop(0)
                refs[table[s, j]] = 1
            lens[s] = L + k
        for old, new, rows in copies:
            kv[:, :, new, :, :rows] = kv[:, :, old, :, :rows]
        self.table, self.lens, self.refs = table, lens, refs

    def write(self, layer, seq, row_start, k, v):
        """k, v [layers, rows, heads, dim]"""
        for i, s in enumerate(seq):
            n = row_start[i + 1] - row_start[i]
            for r in range(row_start[i], row_start[i + 1]):
                pos = int(self.lens[s]) - n + r - row_start[i]
                page = self.table[s, pos // self.P]
                for l in range(k.shape[0]):
                    self.kv[layer + l, 0, page, :, pos % self.P] = k[l, r]
                    self.kv[layer + l, 1, page, :, pos % self.P] = v[l, r]

    def fork(self, src, dst):
        """Returns the requests that are refused; the others are carried out."""
        refused, then = [], self.lens.copy()
        for i, (s, d) in enumerate(zip(src, dst)):
            n = len(self.lens)
            if not (0 <= s < n and 0 <= d < n) or d in src or d in dst[:i] or then[d] != 0:
                refused.append(i)
                continue
            held = self._count(self.lens[s])
            self.table[d, :held] = self.table[s, :held]
            self.lens[d] = self.lens[s]
            for p in self.table[d, :held]:
                self.refs[p] += 1
        return refused

    def drop(self, seq, count=None):
        refused = []
        for i, s in enumerate(seq):
            k = None if count is None else int(count[i])
            if not 0 <= s < len(self.lens) or s in seq[:i] or (k is not None and k < 0):
                refused.append(i)
                continue
            L = int(self.lens[s])
            left = 0 if k is None else max(0, L - k)
            for j in range(self._count(left), self._count(L)):
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = -1
            self.lens[s] = left
        return refused

    def compact(self):
        used = int((self.refs > 0).sum())
        holes = [p for p in range(used) if self.refs[p] == 0]
        for p in range(used, len(self.refs)):
            if self.refs[p] > 0:
                to = holes.pop(0)
                self.kv[:, :, to] = self.kv[:, :, p]
                self.refs[to], self.refs[p] = self.refs[p], 0
                self.table[self.table == p] = to

    def rows(self, layer, s, upto):
        """Keys and values [upto, heads, dim] of a sequence's first tokens, float64."""
        t = np.arange(upto)
        page = self.table[s, t // self.P]
        return (self.kv[layer, 0, page, :, t % self.P].astype(np.float64),
                self.kv[layer, 1, page, :, t % self.P].astype(np.float64))

    def attention(self, layer, seq, row_start, q, scale, out):
        """out (a copy of it, float64) with the rows of the requests; keys behind a
        row's place take no part, whatever they hold."""
        out = np.array(out, np.float64)
        G = q.shape[1] // self.kv.shape[3]
        for i, s in enumerate(seq):
            n = int(row_start[i + 1] - row_start[i])
            for j in range(n):
                r = row_start[i] + j
                seen = int(self.lens[s]) - n + j + 1
                if seen <= 0:
                    out[r] = 0.0
                    continue
                k, v = self.rows(layer, s, seen)
                k, v = np.repeat(k, G, 1), np.repeat(v, G, 1)
                with np.errstate(all="ignore"):
                    sc = np.einsum("hd,thd->ht", q[r].astype(np.float64), k) * scale
                    p = np.exp(sc - sc.max(1, keepdims=True))
                    out[r] = np.einsum("ht,thd->hd", p / p.sum(1, keepdims=True), v)
        return out


def verify(target, draft, ids, u, u_next, row_start):
    """(accepted, tokens, rejected); target, draft [rows, vocab] (draft None: certain)."""
    V = target.shape[1]
    accepted, rejected = [], []
    tokens = np.full(len(target), -1, np.int64)
    for i in range(len(row_start) - 1):
        a, b = int(row_start[i]), int(row_start[i + 1])
        if a == b:
            accepted.append(0)
            rejected.append(0)
            continue
        r = a
        while r < b - 1:
            x = int(ids[r])
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else np.float64(draft[r, x])
            if not np.float64(u[r]) * q < np.float64(target[r, x]):
                break
            tokens[r] = x
            r += 1
        p = target[r].astype(np.float64)
        with np.errstate(all="ignore"):
            w = p
            if r < b - 1:
                q = np.zeros(V) if draft is None else draft[r].astype(np.float64)
                if draft is None and 0 <= ids[r] < V:
                    q[ids[r]] = 1.0
                w = p - q
            w = np.where(np.isfinite(w) & (w > 0), w, 0.0)
            if r < b - 1 and w.sum() == 0:
                w = np.where(np.isfinite(p) & (p > 0), p, 0.0)
            sums = np.cumsum(w)
            over = np.flatnonzero((sums > np.float64(u_next[i]) * sums[-1]) & (w > 0))
        some = np.flatnonzero(w > 0)
        tokens[r] = over[0] if len(over) else some[-1] if len(some) else -1
        accepted.append(r - a)
        rejected.append(b - 1 - r)
    return np.array(accepted), tokens, np.array(rejected)
