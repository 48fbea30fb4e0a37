"""The paged cache on the GPU (mod_amd/csrc/kv_pages.hip, kv_attention.hip)
against oracle/kv_ref.py.

Pages, tables, lengths and counts are held to equality. Attention is held to
the float64 oracle on the scale of max |v| (its outputs are convex combinations
of v rows). With u = 2^-24 (half a step of fp32) and smax the largest |score|:
  - a score is a sum of D products; its roundings are of partial sums no larger
    than a few smax and add up as a random walk: es = 4 u sqrt(D) (smax + 1);
  - the weights' relative errors are those of the scores (twice: numerator and
    sum) plus exp's few ulp, their sums over T keys again a random walk:
    2 es + 8 u + 4 u sqrt(T);
  - fp16 queries over an fp16 cache: the weights are rounded to fp16, 2^-11 of
    each, and the output to fp16, 2^-11 of it;
  - fp32 queries over an fp16 cache: queries and weights are two fp16 parts,
    each pair off by at most 2^-22: 2^-22 of sum |q k| in a score, 2^-22 of the
    weights (fp16 outputs of any path are rounded, 2^-11)."""
import collections

import numpy as np
import pytest

from oracle import kv_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _say(m):
    print(m, flush=True)


@pytest.fixture(scope="module")
def torch(torch_dev):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from mod_amd import ops
    return ops


class Pair:
    """A cache on the GPU and its oracle, changed together."""

    def __init__(self, torch, ops, layers, heads, dim, page, pages, seqs, width, dtype="float32", fill=None):
        self.t, self.ops, self.ref = torch, ops, kv_ref.Cache(layers, heads, dim, page, pages, seqs, width,
                                                              getattr(np, dtype))
        if fill is not None:
            self.ref.kv[:] = fill
        self.kv = torch.from_numpy(self.ref.kv.copy()).cuda()
        self.kept = collections.deque(maxlen=64)
        self.table = torch.full((seqs, width), 77, dtype=torch.int32, device="cuda")
        self.lens = torch.full((seqs,), 77, dtype=torch.int32, device="cuda")
        self.refs = torch.full((pages,), 77, dtype=torch.int32, device="cuda")
        self.c = ops.KvCache(self.kv, self.table, self.lens, self.refs)
        torch.cuda.synchronize()
        ops.kv_init(self.c)

    def ints(self, v):
        return self.dev(np.array([int(x) for x in v], np.int32))

    def dev(self, a):
        t = self.t.from_numpy(np.ascontiguousarray(a)).cuda()
        # kept until the kernels that read it are done: the next ones wait for the device too
        self.kept.append(t)
        self.t.cuda.synchronize()
        return t

    def reserve(self, seq, count):
        self.ops.kv_reserve(self.c, self.ints(seq), self.ints(count), len(seq))
        self.ref.reserve(list(seq), list(count))

    def write(self, layer, seq, start, k, v):
        self.ops.kv_write(self.c, layer, k.shape[0], self.ints(seq), self.ints(start), len(seq), self.dev(k),
                          self.dev(v), k.shape[1])
        self.ref.write(layer, list(seq), start, k, v)

    def add(self, rng, seq, count, dtype=np.float32, scale=1.0):
        """Room and random tokens in all layers."""
        self.reserve(seq, count)
        start = np.concatenate([[0], np.cumsum(count)]).astype(int)
        shape = (self.ref.kv.shape[0], int(start[-1]), self.ref.kv.shape[3], self.ref.kv.shape[5])
        k, v = ((rng.standard_normal(shape) * scale).astype(dtype) for _ in range(2))
        if start[-1]:
            self.write(0, seq, start, k, v)

    def fork(self, src, dst):
        self.ops.kv_fork(self.c, self.ints(src), self.ints(dst), len(src))
        return self.ref.fork(list(src), list(dst))

    def drop(self, seq, count=None):
        self.ops.kv_drop(self.c, self.ints(seq), None if count is None else self.ints(count), len(seq))
        return self.ref.drop(list(seq), count)

    def compact(self):
        self.ops.kv_compact(self.c)
        self.ref.compact()

    def same(self):
        self.t.cuda.synchronize()
        assert np.array_equal(self.table.cpu().numpy(), self.ref.table)
        assert np.array_equal(self.lens.cpu().numpy(), self.ref.lens)
        assert np.array_equal(self.refs.cpu().numpy(), self.ref.refs)
        a, b = self.kv.cpu().numpy(), self.ref.kv
        kind = np.uint32 if b.dtype == np.float32 else np.uint16
        assert np.array_equal(a.view(kind), b.view(kind))


# ------------------------------------------------------------------- pages ---
@pytest.mark.parametrize("layers,heads,dim,page,dtype,rows", [
    (1, 1, 8, 1, "float32", np.float32),
    (2, 3, 64, 4, "float16", np.float32),
    (3, 2, 128, 16, "float32", np.float16),
    (1, 5, 72, 2, "float16", np.float16),
])
def test_random_calls(torch, ops, layers, heads, dim, page, dtype, rows):
    """Reserve, write, fork, drop and compact in any order, equal after each."""
    _say(f"pages {layers} x {heads} x {dim} page {page} {dtype}")
    rng = np.random.default_rng(page)
    p = Pair(torch, ops, layers, heads, dim, page, 45, 9, 60 // page, dtype)
    for step in range(120):
        what = rng.integers(5)
        if what <= 1:
            seq = [int(s) for s in rng.permutation(9)[:rng.integers(1, 6)]]
            count = [int(k) for k in rng.integers(0, 2 * page + 2, len(seq))]
            try:
                p.add(rng, seq, count, rows)
            except kv_ref.Refused:
                with pytest.raises(ops.RocmError):
                    ops.kv_status(p.c)
        elif what == 2:
            empty = [s for s in range(9) if p.ref.lens[s] == 0]
            full = [s for s in range(9) if p.ref.lens[s] > 0]
            if full and empty:
                n = int(rng.integers(1, len(empty) + 1))
                assert p.fork([full[int(i)] for i in rng.integers(0, len(full), n)], empty[:n]) == []
        elif what == 3:
            seq = [int(s) for s in rng.permutation(9)[:rng.integers(1, 5)]]
            if rng.random() < 0.3:
                p.drop(seq)
            else:
                p.drop(seq, [int(k) for k in rng.integers(0, 3 * page + 2, len(seq))])
        else:
            p.compact()
        p.same()
        ops.kv_status(p.c)


def test_reserve_is_all_or_nothing(torch, ops):
    rng = np.random.default_rng(3)
    p = Pair(torch, ops, 1, 1, 8, 4, 10, 6, 4)
    p.add(rng, [0, 1], [5, 8])                      # 4 of 10 pages
    p.fork([0], [2])
    for seq, count, error in [
            ([3, 4], [16, 9], "too few free pages"),        # 7 pages of 6
            ([3], [17], "too short table rows"),
            ([1], [9], "too short table rows"),
            ([3, 6], [1, 1], "does not have"),
            ([3, -1], [1, 1], "does not have"),
            ([3, 4, 3], [1, 1, 1], "twice"),
            ([3, 4], [1, -1], "does not have"),
            ([0, 2, 3, 4], [4, 4, 8, 5], "too few free pages"),   # two copies and six pages
    ]:
        _say(f"reserve {seq} {count}")
        ops.kv_reserve(p.c, p.ints(seq), p.ints(count), len(seq))
        p.same()
        with pytest.raises(ops.RocmError, match=error):
            ops.kv_status(p.c)
        ops.kv_status(p.c)                          # reported once
    p.add(rng, [0, 2, 3, 4], [4, 4, 8, 0])          # the very last pages
    p.same()
    assert not np.any(p.ref.refs == 0) or p.ref.refs[p.ref.refs == 0].size < 2
    ops.kv_reserve(p.c, p.ints([]), p.ints([]), 0)
    ops.kv_status(p.c)


def test_refused_forks_and_drops(torch, ops):
    rng = np.random.default_rng(4)
    p = Pair(torch, ops, 1, 2, 8, 2, 30, 8, 6)
    p.add(rng, [0, 1], [7, 3])
    refused = p.fork([0, 0, 1, 0, 9, 0, 1], [2, 2, 1, 8, 3, 0, 4])
    assert refused == [1, 2, 3, 4, 5]
    p.same()
    with pytest.raises(ops.RocmError, match="not empty"):
        ops.kv_status(p.c)
    assert p.fork([0, 3], [3, 5]) == [0]            # a target that is a source; an empty source is a copy of nothing
    p.same()
    with pytest.raises(ops.RocmError):
        ops.kv_status(p.c)
    assert p.drop([2, 2, -1, 4, 7], [1, 1, 1, -1, 5]) == [1, 2, 3]
    p.same()
    with pytest.raises(ops.RocmError):
        ops.kv_status(p.c)
    p.drop([0, 1, 2, 4])
    p.same()
    assert np.all(p.ref.refs == 0)
    ops.kv_status(p.c)


def test_write_leaves_the_rest(torch, ops):
    """Strided rows and layers, rows behind the last request, a layer in the middle."""
    rng = np.random.default_rng(5)
    p = Pair(torch, ops, 3, 2, 16, 4, 12, 4, 5, "float16")
    p.reserve([3, 1], [6, 0])
    p.reserve([3, 1], [3, 7])
    start = [0, 3, 8]                               # the last 3 of 9, and 5 of 7
    k, v = (rng.standard_normal((2, 11, 48)).astype(np.float32) for _ in range(2))
    k[:, 8:], v[:, 8:] = np.nan, np.nan
    ops.kv_write(p.c, 1, 2, p.ints([3, 1]), p.ints(start), 2, p.dev(k), p.dev(v), 11, row_stride=48,
                 layer_stride=11 * 48)
    p.ref.write(1, [3, 1], start, k[:, :, :32].reshape(2, 11, 2, 16), v[:, :, :32].reshape(2, 11, 2, 16))
    p.same()
    ops.kv_status(p.c)
    ops.kv_write(p.c, 0, 1, p.ints([0]), p.ints([0, 1]), 1, p.dev(k), p.dev(v), 1)     # an empty sequence
    p.same()
    with pytest.raises(ops.RocmError):
        ops.kv_status(p.c)


def test_many_pages_and_requests(torch, ops):
    """Plans that walk more pages, and more requests, than one step of the planning workgroup."""
    rng = np.random.default_rng(6)
    p = Pair(torch, ops, 1, 1, 8, 1, 40000, 4100, 40)
    seq = [int(s) for s in rng.permutation(4100)[:4096]]
    p.reserve(seq, [int(k) for k in rng.integers(0, 10, 4096)])
    p.same()
    p.drop([int(s) for s in rng.permutation(4100)[:2000]])
    p.reserve(seq[:2500], [int(k) for k in rng.integers(0, 7, 2500)])
    p.same()
    p.drop([int(s) for s in rng.permutation(4100)[:3000]])
    p.compact()
    p.same()
    ops.kv_status(p.c)


@pytest.mark.parametrize("pages", [1, 3, 1023, 1024, 1025])
def test_plans_at_their_steps(torch, ops, pages):
    """Caches of one page to a thread and of one more; every page in use, and one free."""
    rng = np.random.default_rng(pages)
    p = Pair(torch, ops, 1, 1, 8, 2, pages, 70, 600)
    p.add(rng, [0], [min(2 * pages, 1200)])
    if pages > 600:
        p.add(rng, [1], [2 * (pages - 600)])
    assert np.all(p.ref.refs == 1)
    p.compact()
    p.same()
    ops.kv_reserve(p.c, p.ints([2]), p.ints([1]), 1)
    p.same()
    with pytest.raises(ops.RocmError, match="too few free pages"):
        ops.kv_status(p.c)
    p.drop([0], [min(2 * pages, 1200) // 2])
    p.add(rng, list(range(2, 70, 5)), [2 if pages > 600 else 0] * 14)
    p.drop([0])
    p.same()
    p.compact()
    p.same()
    p.add(rng, [0], [min(2 * int((p.ref.refs == 0).sum()), 1200)])
    p.same()
    ops.kv_status(p.c)


# --------------------------------------------------------------- attention ---
def _tolerance(p, layer, seq, row_start, q, scale, x16):
    """Bound on |out - oracle| on the scale of the derivation above."""
    smax, dots, T, vmax = 0.0, 0.0, 1, 0.0
    G = q.shape[1] // p.ref.kv.shape[3]
    for i, s in enumerate(seq):
        n = int(p.ref.lens[s])
        if not n or row_start[i] == row_start[i + 1]:
            continue
        k, v = p.ref.rows(layer, s, n)
        k = np.repeat(np.where(np.isfinite(k), k, 0), G, 1)
        qs = q[row_start[i]:row_start[i + 1]].astype(np.float64)
        smax = max(smax, np.abs(np.einsum("rhd,thd->rht", qs, k)).max() * abs(scale))
        dots = max(dots, np.einsum("rhd,thd->rht", np.abs(qs), np.abs(k)).max() * abs(scale))
        T, vmax = max(T, n), max(vmax, np.abs(np.where(np.isfinite(v), v, 0)).max())
    es = 4 * U * np.sqrt(q.shape[2]) * (smax + 1)
    if p.ref.kv.dtype == np.float16 and not x16:
        es += 2.0 ** -22 * dots
    weights = 2 * es + 8 * U + 4 * U * np.sqrt(T)
    if p.ref.kv.dtype == np.float16:
        weights += 2.0 ** -11 if x16 else 2.0 ** -22
    return vmax * (weights + (2.0 ** -11 if x16 else 0.0))


def _attend(p, torch, ops, layer, seq, start, q, scale, shared, window, **kw):
    qd = p.dev(q)
    out = torch.full(q.shape, 7.0, dtype=qd.dtype, device="cuda")
    torch.cuda.synchronize()
    ops.kv_attention(p.c, layer, p.ints(seq), p.ints(start), len(seq), qd, out, q.shape[0], q.shape[1], scale,
                     shared=shared, max_rows=window, **kw)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _prefix(p, rng, n, shared, tails, scale=1.0):
    """Sequences 1 .. n that begin with the same `shared` tokens of sequence 0, and tails of their own."""
    if shared:
        p.add(rng, [0], [shared], scale=scale)
        p.fork([0] * n, list(range(1, n + 1)))
    p.add(rng, list(range(1, n + 1)), tails, scale=scale)


CASES = [
    # heads, kv heads, dim, page, shared, tails, windows, cache, queries
    (2, 1, 128, 16, 0, [1], [1], "float32", "float32"),
    (4, 2, 64, 16, 0, [33, 1, 64], [1, 1, 1], "float32", "float32"),
    (16, 8, 128, 16, 37, [5, 1, 130, 31], [1, 1, 1, 1], "float32", "float32"),
    (16, 8, 128, 16, 500, [7, 300], [1, 1], "float32", "float16"),
    (8, 8, 64, 32, 129, [40, 3, 9], [3, 1, 9], "float32", "float32"),
    (16, 8, 128, 16, 200, [5, 1, 130, 31], [1, 1, 1, 1], "float16", "float32"),
    (32, 4, 128, 64, 300, [17, 65, 2], [1, 4, 2], "float16", "float16"),
    (7, 1, 128, 1, 33, [40, 8], [5, 8], "float16", "float16"),
    (12, 2, 64, 8, 257, [1, 2, 3, 4, 5, 6, 7, 8, 9], [1, 2, 3, 4, 5, 6, 7, 8, 9], "float16", "float16"),
    (12, 2, 64, 128, 1, [700], [37], "float16", "float32"),
    (16, 2, 128, 1024, 1500, [900, 4], [20, 4], "float16", "float16"),
    (3, 3, 8, 4, 11, [6, 2], [2, 1], "float32", "float32"),
    (6, 2, 72, 2, 21, [16, 9], [3, 4], "float16", "float32"),
    (4, 1, 256, 16, 70, [35, 12], [2, 1], "float16", "float16"),
    (4, 4, 192, 16, 0, [350], [3], "float32", "float32"),
    # more columns than a tile, ragged
    (32, 4, 128, 16, 640, [9] * 40, [1 + i % 5 for i in range(40)], "float16", "float16"),
    (16, 8, 128, 16, 260, [3] * 70, [1] * 70, "float16", "float32"),
    (16, 8, 64, 16, 100, [12] * 30, [1 + i % 3 for i in range(30)], "float32", "float32"),
    # prompts: every token a query
    (4, 2, 128, 16, 0, [150, 61], [150, 61], "float16", "float16"),
    (4, 2, 64, 16, 0, [97], [97], "float32", "float32"),
]


@pytest.mark.parametrize("H,Hk,D,page,shared,tails,windows,kv,x", CASES)
def test_attention(torch, ops, H, Hk, D, page, shared, tails, windows, kv, x):
    _say(f"attention H{H}/{Hk} D{D} page {page} shared {shared} tails {tails[:4]} {kv} {x}")
    rng = np.random.default_rng(len(tails) * 1000 + shared)
    n = len(tails)
    need = -(-shared // page) + sum(1 + -(-t // page) for t in tails) + 2
    width = -(-(shared + max(tails)) // page) + 1
    # whatever the pages hold behind a sequence's end must not matter
    p = Pair(torch, ops, 2, Hk, D, page, need, n + 2, width, kv, fill=np.nan)
    _prefix(p, rng, n, shared, tails)
    p.same()
    order = [int(i) for i in rng.permutation(n)]
    seq, counts = [1 + i for i in order], [windows[i] for i in order]
    start = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    rows = int(start[-1]) + 3                       # and rows behind the last sequence
    q = rng.standard_normal((rows, H, D)).astype(x)
    scale = D ** -0.5
    ref = p.ref.attention(1, seq, start, q, scale, np.full(q.shape, 7.0))
    tol = _tolerance(p, 1, seq, start, q, scale, x == "float16")
    # all orders of the arguments that describe the same attention
    for same, hint in [(shared, max(windows)), (0, 1), (shared // 2, max(windows)), (shared, 1)]:
        got = _attend(p, torch, ops, 1, seq, start, q, scale, same, hint)
        assert np.all(got[start[-1]:] == 7.0)
        err = np.abs(got[:start[-1]].astype(np.float64) - ref[:start[-1]]).max()
        _say(f"  shared {same}: {err:.2e} of {tol:.2e}")
        assert np.isfinite(err) and err <= tol
    ops.kv_status(p.c)


@pytest.mark.parametrize("kv,x", [("float32", "float32"), ("float16", "float16"), ("float16", "float32")])
@pytest.mark.parametrize("D", [64, 128, 40])
def test_attention_masked_places(torch, ops, kv, x, D):
    """inf and NaN in keys and values that some rows of a window do not see yet:
    the rows before them are what they are without them, the rows that see them
    are not finite. A shared prefix longer than what a row sees, and rows of
    sequences with fewer tokens than queries, which see nothing."""
    _say(f"masked {kv} {x} D{D}")
    rng = np.random.default_rng(8)
    p = Pair(torch, ops, 1, 2, D, 16, 40, 6, 12, kv, fill=np.nan)
    _prefix(p, rng, 2, 70, [20, 45])
    p.add(rng, [4], [3])
    # the 4th and the 2nd token from the end of sequences 1 and 2
    for s, back, value in [(1, 4, np.nan), (2, 2, np.inf)]:
        pos = int(p.ref.lens[s]) - back
        page = int(p.ref.table[s, pos // 16])
        p.ref.kv[0, 1, page, :, pos % 16] = value
        p.ref.kv[0, 0, page, :, pos % 16] = value if back == 4 else 1.0
    p.kv.copy_(torch.from_numpy(p.ref.kv))
    q = rng.standard_normal((24, 4, D)).astype(x)
    seq, start = [1, 5, 2, 4], [0, 8, 8, 18, 23]    # 8 queries; none; 10; 5 queries of 3 tokens
    ref = p.ref.attention(0, seq, start, q, 0.3, np.full(q.shape, 7.0))
    clean = [r for r in range(23) if np.isfinite(ref[r]).all()]
    assert clean == [0, 1, 2, 3] + list(range(8, 16)) + list(range(18, 23)) and np.all(ref[18:20] == 0)
    tol = _tolerance(p, 0, seq, start, q, 0.3, x == "float16")
    for shared in (0, 33, 70):
        # (sequence 4 has a prefix of its own, and is left out where one is shared)
        got = _attend(p, torch, ops, 0, seq[:4 if not shared else 3], start[:5 if not shared else 4], q, 0.3, shared, 10)
        if shared:
            assert np.all(got[18:] == 7)
            got[18:23] = ref[18:23].astype(got.dtype)
        assert np.abs(got[clean].astype(np.float64) - ref[clean]).max() <= tol
        assert np.all(got[18:20] == 0) and np.all(got[23] == 7)
        for r in set(range(23)) - set(clean):
            assert not np.isfinite(got[r].astype(np.float64)).any()
    # a prefix that reaches into the window: rows that stand inside it see part of it only
    p.fork([1], [3])
    got = _attend(p, torch, ops, 0, [1, 3], [0, 8, 16], np.concatenate([q[:8], q[:8]]), 0.3, 90, 8)
    for half in (got[:4], got[8:12]):
        assert np.abs(half.astype(np.float64) - ref[:4]).max() <= tol
    ops.kv_status(p.c)


@pytest.mark.parametrize("D,Hk,shared,x", [(128, 2, 12301, "float16"), (128, 2, 12301, "float32"),
                                           (64, 4, 24100, "float16")])
def test_attention_long_prefix(torch, ops, D, Hk, shared, x):
    """A prefix long enough for the kernel that reads it once for 128 columns. Rows that
    stand inside it, and an infinite value that those rows do not see yet."""
    _say(f"long prefix D{D} {shared} {x}")
    rng = np.random.default_rng(13)
    n, page, H = 44, 32, 32
    tails = [1 + (7 * i) % 60 for i in range(n)]
    p = Pair(torch, ops, 1, Hk, D, page, -(-shared // page) + 3 * n + 2, n + 1, -(-shared // page) + 3, "float16",
             fill=np.nan)
    _prefix(p, rng, n, shared, tails)
    seq = [1 + int(i) for i in rng.permutation(n)]
    counts = [1 + (s % 2) for s in seq]
    counts[seq.index(1)] = 4                        # of 1 own token: three rows stand in the prefix
    start = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    q = rng.standard_normal((int(start[-1]), H, D)).astype(x)
    ref = p.ref.attention(0, seq, start, q, D ** -0.5, np.zeros(q.shape))
    tol = _tolerance(p, 0, seq, start, q, D ** -0.5, x == "float16")
    got = _attend(p, torch, ops, 0, seq, start, q, D ** -0.5, shared, 2)
    err = np.abs(got.astype(np.float64) - ref).max()
    _say(f"  {err:.2e} of {tol:.2e}")
    assert err <= tol
    pos = shared - 2                                # seen by all rows but the first one's first
    for i in range(n + 1):                          # (in a page that ends behind the prefix: one for each sequence)
        p.kv[0, 1, int(p.ref.table[i, pos // page]), :, pos % page] = np.inf
    got = _attend(p, torch, ops, 0, seq, start, q, D ** -0.5, shared, 4)
    first = int(start[seq.index(1)])
    assert np.abs(got[first].astype(np.float64) - ref[first]).max() <= tol
    for r in set(range(len(q))) - {first}:
        assert np.all(got[r] == np.inf)
    ops.kv_status(p.c)


@pytest.mark.parametrize("H,rows,kv,x", [(2, 1, "float16", "float32"), (8, 5, "float16", "float16"),
                                         (2, 2, "float32", "float32")])
def test_attention_many_requests(torch, ops, H, rows, kv, x):
    """More requests than a workgroup has threads, most of them short, some without rows."""
    _say(f"many requests H{H} {kv} {x}")
    rng = np.random.default_rng(14)
    n = 700
    p = Pair(torch, ops, 1, 1, 64, 16, 2 * n + 100, n + 1, 60, kv, fill=np.nan)
    tails = [int(t) for t in rng.integers(1, 20, n)]
    tails[5], tails[n - 2] = 400, 700
    _prefix(p, rng, n, 21, tails)
    seq = [1 + int(i) for i in rng.permutation(n)]
    start = np.concatenate([[0], np.cumsum([0 if s % 9 == 0 else rows for s in seq])]).astype(int)
    q = rng.standard_normal((int(start[-1]), H, 64)).astype(x)
    ref = p.ref.attention(0, seq, start, q, 0.125, np.zeros(q.shape))
    tol = _tolerance(p, 0, seq, start, q, 0.125, x == "float16")
    for shared in (21, 0):
        got = _attend(p, torch, ops, 0, seq, start, q, 0.125, shared, rows)
        assert np.abs(got.astype(np.float64) - ref).max() <= tol
    ops.kv_status(p.c)


@pytest.mark.parametrize("page", [1, 2])
def test_attention_many_pages_of_an_item(torch, ops, page):
    """Items of more pages than their ids fit into LDS at once: 33,000 tokens in pages of one, and in fewer."""
    tokens, Hk, G, D, rows = 33000, 16, 3, 64, 11
    pages = tokens // page + 4
    i32 = dict(dtype=torch.int32, device="cuda")
    kv = torch.full((1, 2, pages, Hk, page, D), float("nan"), dtype=torch.float16, device="cuda")
    c = ops.KvCache(kv, torch.empty(1, pages, **i32), torch.empty(1, **i32), torch.empty(pages, **i32))
    seq, start, count = torch.zeros(1, **i32), torch.tensor([0, rows], **i32), torch.tensor([tokens], **i32)
    all_rows = torch.tensor([0, tokens], **i32)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(1, tokens, Hk * D, device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn(rows, Hk * G, D, device="cuda", generator=g).half()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    ops.kv_init(c)
    ops.kv_reserve(c, seq, count, 1)
    ops.kv_write(c, 0, 1, seq, all_rows, 1, k, v, tokens)
    ops.kv_attention(c, 0, seq, start, 1, q, out, rows, Hk * G, 0.125, max_rows=rows)
    ops.kv_status(c)
    kk, vv = (t.reshape(tokens, Hk, D).double().transpose(0, 1).contiguous() for t in (k, v))
    qq = q.double().reshape(rows, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * rows, D).contiguous()
    s = torch.matmul(qq, kk.transpose(1, 2).contiguous()).reshape(Hk, G, rows, tokens) * 0.125
    late = torch.arange(tokens, device="cuda") > tokens - rows + torch.arange(rows, device="cuda")[:, None]
    w = torch.softmax(s.masked_fill(late, -torch.inf), 3).reshape(Hk, G * rows, tokens)
    ref = torch.matmul(w, vv).reshape(Hk, G, rows, D).permute(2, 0, 1, 3).reshape(rows, Hk * G, D)
    # |score| < 8: 2 es + 8 u + 4 u sqrt(33000) = 7.4e-5, and the weights' 2^-11 as a random walk is
    # less than 2^-11 itself; the output's 2^-11
    assert float((out.double() - ref).abs().max()) <= (7.4e-5 + 2.0 ** -11) * float(v.abs().max()) + 2.0 ** -11 * float(ref.abs().max())


def test_attention_large_scores(torch, ops):
    """Scores far apart and far from zero; a softmax that picks one key; queries
    beyond the fp16 range over an fp16 cache."""
    for kv, x, big in [("float32", "float32", 1e4), ("float16", "float32", 3e5), ("float16", "float16", 2e3)]:
        _say(f"large scores {kv} {x}")
        rng = np.random.default_rng(9)
        p = Pair(torch, ops, 1, 2, 128, 16, 40, 4, 20, kv)
        _prefix(p, rng, 2, 150, [30, 20])
        q = (rng.standard_normal((2, 4, 128)) * big).astype(x)
        got = _attend(p, torch, ops, 0, [1, 2], [0, 1, 2], q, 1.0, 150, 1)
        ref = p.ref.attention(0, [1, 2], [0, 1, 2], q, 1.0, np.zeros(q.shape))
        for i in range(2):
            k = np.repeat(p.ref.rows(0, i + 1, int(p.ref.lens[i + 1]))[0], 2, 1)
            scores = np.sort(np.einsum("hd,thd->ht", q[i].astype(np.float64), k), axis=1)
            # one key has all the weight (the gap to the next is far over the scores' error)
            sure = scores[:, -1] - scores[:, -2] > 40 + 2.0 ** -18 * np.abs(scores).max()
            assert sure.any()
            assert np.abs(got[i].astype(np.float64) - ref[i])[sure].max() <= 2.0 ** -10 * np.abs(ref).max()
        assert np.isfinite(got.astype(np.float64)).all()


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
def test_attention_scales(torch, ops, scale):
    """No scale (the mean over what a row sees), a negative one, a tiny and a large one."""
    for kv, x in [("float32", "float32"), ("float16", "float32"), ("float16", "float16")]:
        for D, G in [(64, 2), (128, 20)]:
            rng = np.random.default_rng(12)
            p = Pair(torch, ops, 1, 2, D, 16, 60, 5, 20, kv, fill=np.nan)
            _prefix(p, rng, 3, 150, [30, 1, 77])
            seq, start = [1, 2, 3], [0, 2, 3, 6]
            q = rng.standard_normal((6, 2 * G, D)).astype(x)
            ref = p.ref.attention(0, seq, start, q, scale, np.zeros(q.shape))
            got = _attend(p, torch, ops, 0, seq, start, q, scale, 150, 3)
            assert np.abs(got.astype(np.float64) - ref).max() <= _tolerance(p, 0, seq, start, q, scale, x == "float16")


def test_attention_strides_and_in_place(torch, ops):
    rng = np.random.default_rng(10)
    p = Pair(torch, ops, 1, 2, 64, 16, 30, 5, 10, "float16")
    _prefix(p, rng, 3, 50, [4, 9, 20])
    seq, start = [3, 1, 2], [0, 2, 3, 7]
    q = rng.standard_normal((7, 4, 64)).astype(np.float32)
    ref = p.ref.attention(0, seq, start, q, 0.125, np.zeros(q.shape))
    tol = _tolerance(p, 0, seq, start, q, 0.125, False)
    wide = np.zeros((7, 3 * 256), np.float32)       # queries inside fused projection rows
    wide[:, :256] = q.reshape(7, 256)
    wd = p.dev(wide)
    out = torch.full((7, 264), 7.0, device="cuda")
    torch.cuda.synchronize()
    ops.kv_attention(p.c, 0, p.ints(seq), p.ints(start), 3, wd, out, 7, 4, 0.125, shared=50, max_rows=4, q_stride=768,
                     out_stride=264)
    ops.kv_attention(p.c, 0, p.ints(seq), p.ints(start), 3, wd, wd, 7, 4, 0.125, shared=50, max_rows=4, q_stride=768,
                     out_stride=768)
    torch.cuda.synchronize()
    assert torch.all(out[:, 256:] == 7) and torch.all(wd[:, 256:] == 0)
    assert np.abs(out[:, :256].cpu().numpy().reshape(7, 4, 64) - ref).max() <= tol
    assert torch.equal(out[:, :256], wd[:, :256])


def test_attention_bad_ids(torch, ops):
    """Sequence ids and pages outside the cache: NaN rows and a report; the others are what they are."""
    rng = np.random.default_rng(11)
    for kv in ("float32", "float16"):
        p = Pair(torch, ops, 1, 2, 64, 16, 20, 5, 10, kv)
        _prefix(p, rng, 3, 40, [4, 40, 20])
        q = rng.standard_normal((4, 4, 64)).astype(np.float32)
        good = _attend(p, torch, ops, 0, [1, 3, 2, 1], [0, 1, 2, 3, 4], q, 0.125, 40, 1)
        got = _attend(p, torch, ops, 0, [1, 5, 2, -1], [0, 1, 2, 3, 4], q, 0.125, 40, 1)
        assert np.array_equal(got[[0, 2]], good[[0, 2]]) and np.isnan(got[[1, 3]]).all()
        with pytest.raises(ops.RocmError):
            ops.kv_status(p.c)
        for page in (20, -1, 1 << 30):
            p.table[2, 4] = page                    # a page of the second sequence's tail
            got = _attend(p, torch, ops, 0, [1, 3, 2, 1], [0, 1, 2, 3, 4], q, 0.125, 40, 1)
            assert np.array_equal(got[[0, 1, 3]], good[[0, 1, 3]]) and np.isnan(got[2]).all()
            with pytest.raises(ops.RocmError):
                ops.kv_status(p.c)


def test_attention_far_pages(torch, ops):
    """Pages beyond 2^32 bytes from the cache's beginning."""
    pages, page = 70000, 16
    kv = torch.empty((1, 2, pages, 8, page, 128), dtype=torch.float16, device="cuda")      # 4.6 GB
    table = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[-30:] = 0                                  # only the last are free
    cache = ops.KvCache(kv, table, lens, refs)
    i32 = dict(dtype=torch.int32, device="cuda")
    seq, start = torch.tensor([2, 0], **i32), torch.tensor([0, 100, 150], **i32)
    k, v = torch.randn(1, 150, 8, 128, device="cuda"), torch.randn(1, 150, 8, 128, device="cuda")
    q = torch.randn(150, 16, 128, device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    ops.kv_reserve(cache, seq, torch.tensor([100, 50], **i32), 2)
    ops.kv_write(cache, 0, 1, seq, start, 2, k, v, 150)
    ops.kv_attention(cache, 0, seq, start, 2, q, out, 150, 16, 0.09, max_rows=100)
    ops.kv_status(cache)
    assert int(table[2, 0]) == pages - 30
    for a, b in ((0, 100), (100, 150)):
        kk, vv = (x[0, a:b].half().double().repeat_interleave(2, 1).transpose(0, 1).contiguous() for x in (k, v))
        s = torch.matmul(q[a:b].double().transpose(0, 1), kk.transpose(1, 2).contiguous()) * 0.09
        s = s.masked_fill(torch.ones(b - a, b - a, device="cuda").triu(1).bool(), -torch.inf)
        ref = torch.matmul(torch.softmax(s, 2), vv).transpose(0, 1)
        # |score| < 6, sum |q k| scale < 12: 2 (4 u sqrt(128) 7 + 12 / 2^22) + 48 u + 2^-22 = 4.7e-5
        assert float((out[a:b].double() - ref).abs().max()) < 4.7e-5 * float(v.abs().max())


# -------------------------------------------------------------- as one step ---
@pytest.mark.parametrize("dtype,x", [("float32", "float32"), ("float16", "float32"), ("float16", "float16")])
def test_speculative_serving(torch, ops, dtype, x):
    """All calls as a server makes them. A prompt that all requests share; in each step every
    request's pending token and a few drafted ones join the cache, are attended to in every layer,
    verified, and those that were refused go again, by counts that never leave the device.
    Requests end and new ones begin from the prompt; the pages are compacted as it goes on."""
    rng = np.random.default_rng(21)
    layers, H, Hk, D, V, n, prompt = 2, 8, 4, 64, 3001, 6, 45
    p = Pair(torch, ops, layers, Hk, D, 16, 64, n + 3, 12, dtype, fill=np.nan)
    p.add(rng, [0], [prompt])
    live = list(range(1, n + 1))
    p.fork([0] * n, live)
    head = torch.randn(H * D, V, device="cuda")
    taken = 0
    for step in range(14):
        _say(f"step {step}")
        counts = [int(c) for c in rng.integers(1, 6, len(live))]
        start = np.concatenate([[0], np.cumsum(counts)]).astype(int)
        rows = int(start[-1])
        p.add(rng, live, counts, x)
        for layer in range(layers):
            q = rng.standard_normal((rows, H, D)).astype(x)
            ref = p.ref.attention(layer, live, start, q, D ** -0.5, np.zeros(q.shape))
            got = _attend(p, torch, ops, layer, live, start, q, D ** -0.5, prompt, 5)
            tol = _tolerance(p, layer, live, start, q, D ** -0.5, x == "float16")
            assert np.abs(got.astype(np.float64) - ref).max() <= tol
        hidden = torch.from_numpy(got).cuda().float().reshape(rows, H * D)
        target = torch.softmax(hidden @ head, 1)
        draft = torch.softmax((hidden + 0.02 * torch.randn_like(hidden)) @ head, 1)
        ids = torch.multinomial(draft, 1).reshape(rows).int()
        u, u_next = torch.rand(rows, device="cuda"), torch.rand(len(live), device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        accepted, tokens, rejected = torch.empty(len(live), **i32), torch.empty(rows, **i32), torch.empty(len(live), **i32)
        torch.cuda.synchronize()
        ops.verify_draft(target, draft, ids, u, u_next, p.ints(start), len(live), rows, V, accepted, tokens, rejected)
        ops.kv_drop(p.c, p.ints(live), rejected, len(live))
        ref = kv_ref.verify(*(t.cpu().numpy() for t in (target, draft, ids, u, u_next)), start)
        torch.cuda.synchronize()
        for a, b in zip((accepted, tokens, rejected), ref):
            assert np.array_equal(a.cpu().numpy(), b)
        assert p.ref.drop(live, [int(r) for r in ref[2]]) == []
        taken += int(np.sum(ref[0]))
        p.same()
        if step % 3 == 2:                           # two requests end, one begins
            gone = [live.pop(int(rng.integers(len(live)))) for _ in range(2)]
            p.drop(gone)
            free = next(s for s in range(1, n + 3) if p.ref.lens[s] == 0)
            p.fork([0], [free])
            live.append(free)
        if step % 4 == 3:
            p.compact()
            p.same()
    assert 0 < taken
    ops.kv_status(p.c)


class Step:
    """A step with inputs at fixed places, for graphs: every call of the cache and the verification."""

    def __init__(self, torch, ops, seed, dtype="float16"):
        self.t, self.ops = torch, ops
        rng = np.random.default_rng(seed)
        self.p = p = Pair(torch, ops, 2, 4, 64, 16, 80, 10, 20, dtype, fill=0)
        p.add(rng, [0], [70])
        p.fork([0] * 5, [1, 2, 3, 4, 5])
        self.n, self.rows, self.V = 5, 13, 4099
        g = torch.Generator(device="cuda").manual_seed(seed)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.seq, self.start = torch.tensor([3, 1, 5, 2, 4], **i32), torch.tensor([0, 3, 4, 8, 10, 13], **i32)
        self.count, self.last = torch.tensor([3, 1, 4, 2, 3], **i32), torch.tensor([9], **i32)
        self.zero = torch.tensor([0], **i32)
        self.q = torch.empty(13, 8, 64, device="cuda")
        self.k, self.v = torch.empty(2, 13, 256, device="cuda"), torch.empty(2, 13, 256, device="cuda")
        self.out = torch.empty(2, 13, 8, 64, device="cuda")
        self.target, self.draft = torch.empty(13, 4099, device="cuda"), torch.empty(13, 4099, device="cuda")
        self.u, self.u_next = torch.empty(13, device="cuda"), torch.empty(5, device="cuda")
        self.ids = torch.empty(13, **i32)
        self.accepted, self.tokens, self.rejected = torch.empty(5, **i32), torch.empty(13, **i32), torch.empty(5, **i32)
        self.g = g
        torch.cuda.synchronize()

    def fill(self):
        """New inputs (the device is waited for before and after)."""
        t = self.t
        t.cuda.synchronize()
        for a in (self.q, self.k, self.v):
            a.copy_(t.randn(a.shape, device="cuda", generator=self.g))
        logits = 3 * t.randn(self.target.shape, device="cuda", generator=self.g)
        self.target.copy_(t.softmax(logits, 1))
        self.draft.copy_(t.softmax(logits + 0.3 * t.randn(logits.shape, device="cuda", generator=self.g), 1))
        self.ids.copy_(t.multinomial(self.draft, 1, generator=self.g).reshape(13))
        for a in (self.u, self.u_next):
            a.copy_(t.rand(a.shape, device="cuda", generator=self.g))
        t.cuda.synchronize()

    def run(self, stream=None):
        o, c = self.ops, self.p.c
        o.kv_reserve(c, self.seq, self.count, 5, stream=stream)
        o.kv_write(c, 0, 2, self.seq, self.start, 5, self.k, self.v, 13, stream=stream)
        for layer in range(2):
            o.kv_attention(c, layer, self.seq, self.start, 5, self.q, self.out[layer], 13, 8, 0.125, shared=70, max_rows=4,
                           stream=stream)
        o.verify_draft(self.target, self.draft, self.ids, self.u, self.u_next, self.start, 5, 13, self.V, self.accepted,
                       self.tokens, self.rejected, stream=stream)
        o.kv_drop(c, self.seq, self.rejected, 5, stream=stream)
        o.kv_fork(c, self.seq, self.last, 1, stream=stream)     # a copy of the first request, and gone again
        o.kv_drop(c, self.last, None, 1, stream=stream)
        o.kv_compact(c, stream=stream)

    def state(self):
        self.t.cuda.synchronize()
        p = self.p
        return [a.clone() for a in (p.table, p.lens, p.refs, self.out, self.accepted, self.tokens, self.rejected)]


def _alike(torch, a, b):
    for x, y in zip(a.state(), b.state()):
        assert torch.equal(x, y)
    # a page that no sequence holds may differ
    held = a.p.refs.bool()
    assert torch.equal(a.p.kv[:, :, held], b.p.kv[:, :, held])


def test_captured_step(torch, ops):
    """A step captured by the library's own graph, its first call included, replayed with new inputs
    and eager work between, against the same steps run one call after the other."""
    from mod_amd import backend
    eager, captured = Step(torch, ops, 5), Step(torch, ops, 5)
    graph = backend.HIPGraph()
    graph.capture_begin()
    captured.run()
    graph.capture_end()
    for i in range(6):
        _say(f"replay {i}")
        for s in (eager, captured):
            s.fill()
        graph.replay()
        eager.run()
        _alike(torch, eager, captured)
        torch.randn(1 << 20, device="cuda").sum().item()
    graph.capture_begin()                           # an empty one in its place: its workspaces go back
    graph.capture_end()
    for s in (eager, captured):
        ops.kv_status(s.p.c)


def test_two_graphs_and_streams(torch, ops):
    """Two captured steps of two caches, replayed at once on two streams, against eager steps."""
    eager = [Step(torch, ops, 6), Step(torch, ops, 7)]
    captured = [Step(torch, ops, 6), Step(torch, ops, 7)]
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s, st in zip(captured, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run(stream=st)
        graphs.append(g)
    for i in range(5):
        _say(f"replay {i}")
        for s in eager + captured:
            s.fill()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        for s in eager:
            s.run()
        for a, b in zip(eager, captured):
            _alike(torch, a, b)
    for s, st in zip(eager + captured, [None, None] + streams):
        ops.kv_status(s.p.c, stream=st)
