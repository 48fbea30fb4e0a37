"""The paged cache in 4 bits on the GPU (mod_amd/csrc/kv_pages.hip,
kv_attention4.hip) against oracle/kv_ref.py.

What the cache holds after a write, and what a read gives back, are held to
equality: both are functions of single values. Attention is held to the float64
oracle on the scale of max |v|, as test_gpu_kv_cache.py derives it, with these
terms for a cache whose values are exact in fp16:
  - queries are sums of parts of 6 bits, off by at most 2^-13 (fp16) or 2^-23
    (fp32) of the largest of 32 dimensions, m_b: that times m_b sum |k| in a score;
  - fp16 queries: the weights are rounded to fp16, 2^-11 of each with the output's
    own 2^-11; fp32 queries: weights in two fp16 parts, 2^-22 of each."""
import numpy as np
import pytest

from oracle import kv_ref
from test_gpu_kv_cache import U, Pair, _attend, _prefix, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(torch_dev):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from mod_amd import ops
    return ops


class Pair4(Pair):
    """A cache of 4 bits on the GPU and its oracle; its bytes are `fill` at first."""

    def __init__(self, torch, ops, layers, heads, dim, page, pages, seqs, width, fill=255):
        super().__init__(torch, ops, layers, heads, dim // 32 * 17, page, pages, seqs, width, "uint8", fill)
        ref, self.ref = self.ref, kv_ref.Cache4(layers, heads, dim, page, pages, seqs, width)
        self.ref.kv = ref.kv
        assert self.c.c.head_dim == dim

    def add(self, rng, seq, count, dtype=np.float32, scale=1.0):
        self.reserve(seq, count)
        start = np.concatenate([[0], np.cumsum(count)]).astype(int)
        shape = (self.ref.kv.shape[0], int(start[-1]), self.ref.kv.shape[3], self.ref.D)
        k, v = ((rng.standard_normal(shape) * scale).astype(dtype) for _ in range(2))
        if start[-1]:
            self.write(0, seq, start, k, v)

    def put(self, layer, kind, s, pos, x):
        """One token's keys or values [heads, D], by the oracle."""
        self.ref.put(layer, kind, self.ref.table[s, pos // self.ref.P], pos % self.ref.P, x)

    def upload(self):
        self.kv.copy_(self.t.from_numpy(self.ref.kv))
        self.t.cuda.synchronize()

    def same(self):
        self.t.cuda.synchronize()
        assert np.array_equal(self.table.cpu().numpy(), self.ref.table)
        assert np.array_equal(self.lens.cpu().numpy(), self.ref.lens)
        assert np.array_equal(self.refs.cpu().numpy(), self.ref.refs)
        kept, want = self.ref.kv, self.ref.values()
        scales = self.ref.blocks()[1].copy()
        self.ref.kv = self.kv.cpu().numpy()
        assert np.array_equal(self.ref.blocks()[1], scales)
        assert np.array_equal(self.ref.values(), want, equal_nan=True)
        self.ref.kv = kept

    def read(self, layer, layers, seq, start, first, dtype, rows=None, row_stride=0, layer_stride=0):
        """k, v [layers, rows, width] as they come, over sevens."""
        rows = int(start[-1]) if rows is None else rows
        width = row_stride or self.ref.kv.shape[3] * self.ref.D
        each = layer_stride or rows * width
        size = max((layers - 1) * each + rows * width, 8)
        k, v = (self.t.full((size,), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        self.t.cuda.synchronize()
        self.ops.kv_read(self.c, layer, layers, self.ints(seq), self.ints(start), len(seq), k, v, rows,
                         None if first is None else self.ints(first), row_stride, layer_stride)
        self.t.cuda.synchronize()
        return k.cpu().numpy(), v.cpu().numpy()


# ----------------------------------------------------------- write and read ---
def _hard_values(rng, n):
    """Blocks of 32 with values on, just below and just above every border, under all scales."""
    y = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.5], np.float32)
    near = np.concatenate([np.nextafter(y, np.float32(0)), np.nextafter(y, np.float32(9)), y])
    x = rng.choice(near, (n, 32)) * rng.choice([-1, 1], (n, 32))
    x[:, 0] = rng.choice(np.array([3.5, 4, 5.999, 6, 6.99, np.nextafter(np.float32(7), np.float32(0)), 7, 7.5]), n)
    x = np.ldexp(x, rng.integers(-26, 16, (n, 1))).astype(np.float32)
    x[0], x[1], x[2, 5], x[3, 31], x[4, 0] = 0, 1e-42, np.inf, np.nan, -np.inf
    x[5], x[6, 3] = 3e38, -3e38
    return x


@pytest.mark.parametrize("D,Hk,page,x", [(128, 8, 16, "float32"), (64, 3, 32, "float32"), (32, 1, 16, "float16"),
                                         (96, 2, 1024, "float16"), (256, 1, 64, "float32")])
def test_every_border(torch, ops, D, Hk, page, x):
    _say(f"borders D{D} x {Hk} page {page} {x}")
    rng = np.random.default_rng(D)
    rows = 41
    p = Pair4(torch, ops, 2, Hk, D, page, 8 + 80 // page, 3, 1 + 48 // page)
    p.reserve([1], [rows])
    with np.errstate(over="ignore"):
        k, v = (_hard_values(rng, 2 * rows * Hk * D // 32).reshape(2, rows, Hk, D).astype(x) for _ in range(2))
    p.write(0, [1], [0, rows], k, v)
    p.same()
    for dtype in (torch.float32, torch.float16):
        for got, kind in zip(p.read(0, 2, [1], [0, rows], None, dtype), range(2)):
            for layer in range(2):
                want = p.ref.rows(layer, 1, rows)[kind]
                assert np.array_equal(got.reshape(2, rows, Hk, D)[layer].astype(np.float64), want, equal_nan=True)
    ops.kv_status(p.c)


@pytest.mark.parametrize("layers,heads,dim,page,rows", [(1, 1, 32, 16, np.float32), (3, 2, 128, 16, np.float16),
                                                        (2, 3, 64, 32, np.float32)])
def test_random_calls(torch, ops, layers, heads, dim, page, rows):
    """Reserve, write, fork, drop and compact in any order, equal after each, and reads between."""
    _say(f"pages {layers} x {heads} x {dim} page {page}")
    rng = np.random.default_rng(page + dim)
    p = Pair4(torch, ops, layers, heads, dim, page, 30, 9, 4)
    for step in range(70):
        what = rng.integers(6)
        if what <= 1:
            seq = [int(s) for s in rng.permutation(9)[:rng.integers(1, 6)]]
            count = [int(k) for k in rng.integers(0, page, len(seq))]
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
            p.drop(seq, None if rng.random() < 0.3 else [int(k) for k in rng.integers(0, 2 * page, len(seq))])
        elif what == 4:
            p.compact()
        else:
            seq = [int(s) for s in rng.integers(0, 9, 7)]            # some twice
            first = [int(rng.integers(0, p.ref.lens[s] + 1)) for s in seq]
            count = [int(rng.integers(0, p.ref.lens[s] - f + 1)) for s, f in zip(seq, first)]
            start = np.concatenate([[0], np.cumsum(count)]).astype(int)
            k, v = p.read(layers - 1, 1, seq, start, first, torch.float32)
            for i, s in enumerate(seq):
                for got, want in zip((k, v), p.ref.rows(layers - 1, s, first[i] + count[i])):
                    got = got[:start[-1] * heads * dim].reshape(-1, heads, dim)[start[i]:start[i + 1]]
                    assert np.array_equal(got, want[first[i]:])
        p.same()
        ops.kv_status(p.c)


@pytest.mark.parametrize("kv", ["float32", "float16", "mx4"])
@pytest.mark.parametrize("x", ["float32", "float16"])
def test_read_leaves_the_rest(torch, ops, kv, x):
    """Strided rows and layers, both ways round, rows behind the last request, a layer in the
    middle; tokens, sequences and pages that are not there become NaN rows."""
    rng = np.random.default_rng(5)
    if kv == "mx4":
        p = Pair4(torch, ops, 3, 2, 32, 16, 12, 4, 3)
    else:
        p = Pair(torch, ops, 3, 2, 32, 16, 12, 4, 3, kv)
        p.ref.D = 32
    p.reserve([3, 1], [21, 16])
    k, v = (rng.standard_normal((3, 37, 2, 32)).astype(np.float32) for _ in range(2))
    p.write(0, [3, 1], [0, 21, 37], k, v)
    dtype = getattr(torch, x)
    read = lambda *args, **kw: Pair4.read(p, *args, **kw)  # noqa: E731

    def want(layer, s, at):
        with np.errstate(over="ignore"):
            return [a[at].reshape(-1, 64).astype(x) for a in p.ref.rows(layer, s, int(p.ref.lens[s]))]
    start, first = [0, 3, 3, 7, 9], [18, 5, 9, 0]
    seq = [3, 1, 1, 3]
    rows = 12
    for row_stride, layer_stride in ((72, 12 * 72), (144, 72), (0, 0)):
        rs, ls = row_stride or 64, layer_stride or rows * 64
        got = read(1, 2, seq, start, first, dtype, rows, row_stride, layer_stride)
        for kind in range(2):
            full = np.full(got[kind].shape, 7.0, x)
            for layer in range(2):
                for i, s in enumerate(seq):
                    w = want(1 + layer, s, slice(first[i], first[i] + start[i + 1] - start[i]))[kind]
                    for j, r in enumerate(range(start[i], start[i + 1])):
                        full[layer * ls + r * rs:layer * ls + r * rs + 64] = w[j]
            assert np.array_equal(got[kind], full)
    got = read(0, 1, [1, 3], [0, 2, 5], None, dtype)                 # the last ones
    for kind in range(2):
        rows_ = np.concatenate([want(0, 1, slice(14, 16))[kind], want(0, 3, slice(18, 21))[kind]])
        assert np.array_equal(got[kind][:5 * 64].reshape(5, 64), rows_)
    ops.kv_status(p.c)
    # past the end, before the beginning, no such sequence, an empty one; the last of more than there are
    big = 2 ** 31 - 1
    for seq, start, first, there in [([1], [0, 3], [14], [0, 1]), ([1], [0, 3], [-1], [1, 2]), ([4], [0, 1], [0], []),
                                     ([-1], [0, 1], [0], []), ([0], [0, 1], [0], []), ([3], [0, 2], [big], []),
                                     ([1], [0, 18], None, list(range(2, 18)))]:
        _say(f"  read {seq} {start} {first}")
        got = read(0, 1, seq, start, first, dtype)
        n = start[-1]
        for kind in range(2):
            nan = np.isnan(got[kind][:n * 64].astype(np.float64)).reshape(n, 64)
            assert all(nan[r].all() != (r in there) for r in range(n)) and all(not nan[r].any() for r in there)
        with pytest.raises(ops.RocmError, match="does not have"):
            ops.kv_status(p.c)
    # a page outside the cache: its tokens alone
    p.table[3, 1] = 12
    got = read(0, 1, [3], [0, 21], [0], dtype)
    nan = np.isnan(got[0][:21 * 64].astype(np.float64)).reshape(21, 64)
    assert nan[16:].all() and not nan[:16].any()
    with pytest.raises(ops.RocmError, match="does not have"):
        ops.kv_status(p.c)


# --------------------------------------------------------------- attention ---
def _tolerance(p, layer, seq, row_start, q, scale, x16):
    smax, dots, T, vmax = 0.0, 0.0, 1, 0.0
    G = q.shape[1] // p.ref.kv.shape[3]
    D = q.shape[2]
    for i, s in enumerate(seq):
        n = int(p.ref.lens[s])
        if not n or row_start[i] == row_start[i + 1]:
            continue
        k, v = p.ref.rows(layer, s, n)
        k = np.repeat(np.where(np.isfinite(k), k, 0), G, 1)
        qs = q[row_start[i]:row_start[i + 1]].astype(np.float64)
        most = np.repeat(np.abs(qs).reshape(*qs.shape[:2], D // 32, 32).max(3), 32, 2)
        smax = max(smax, np.abs(np.einsum("rhd,thd->rht", qs, k)).max() * abs(scale))
        dots = max(dots, np.einsum("rhd,thd->rht", most, np.abs(k)).max() * abs(scale))
        T, vmax = max(T, n), max(vmax, np.abs(np.where(np.isfinite(v), v, 0)).max())
    es = 4 * U * np.sqrt(D) * (smax + 1) + 2.0 ** (-13 if x16 else -23) * dots
    weights = 2 * es + 8 * U + 4 * U * np.sqrt(T) + (2.0 ** -11 if x16 else 2.0 ** -22)
    return vmax * (weights + (2.0 ** -11 if x16 else 0.0))


CASES = [
    # heads, kv heads, dim, page, shared, tails, windows, queries
    (2, 1, 128, 16, 0, [1], [1], "float32"),
    (4, 2, 64, 16, 0, [33, 1, 64], [1, 1, 1], "float32"),
    (16, 8, 128, 16, 37, [5, 1, 130, 31], [1, 1, 1, 1], "float32"),
    (16, 8, 128, 16, 500, [7, 300], [1, 1], "float16"),
    (8, 8, 64, 32, 129, [40, 3, 9], [3, 1, 9], "float32"),
    (32, 4, 128, 64, 300, [17, 65, 2], [1, 4, 2], "float16"),
    (7, 1, 128, 16, 33, [40, 8], [5, 8], "float16"),
    (12, 2, 64, 16, 257, [1, 2, 3, 4, 5, 6, 7, 8, 9], [1, 2, 3, 4, 5, 6, 7, 8, 9], "float16"),
    (12, 2, 64, 128, 1, [700], [37], "float32"),
    (16, 2, 128, 1024, 1500, [900, 4], [20, 4], "float16"),
    (3, 3, 32, 16, 11, [6, 2], [2, 1], "float32"),
    (6, 2, 96, 16, 21, [16, 9], [3, 4], "float32"),
    (4, 1, 256, 16, 70, [35, 12], [2, 1], "float16"),
    (4, 4, 192, 16, 0, [350], [3], "float32"),
    # more columns than a tile, ragged
    (32, 4, 128, 16, 640, [9] * 40, [1 + i % 5 for i in range(40)], "float16"),
    (16, 8, 128, 16, 260, [3] * 70, [1] * 70, "float32"),
    (16, 8, 64, 16, 100, [12] * 30, [1 + i % 3 for i in range(30)], "float32"),
    # many heads to one kv head, and prompts: every token a query
    (40, 1, 64, 16, 0, [70, 200], [1, 1], "float16"),
    (4, 2, 128, 16, 0, [150, 61], [150, 61], "float16"),
    (4, 2, 64, 16, 0, [97], [97], "float32"),
    (6, 3, 128, 32, 45, [160], [160], "float32"),
]


@pytest.mark.parametrize("H,Hk,D,page,shared,tails,windows,x", CASES)
def test_attention(torch, ops, H, Hk, D, page, shared, tails, windows, x):
    _say(f"attention H{H}/{Hk} D{D} page {page} shared {shared} tails {tails[:4]} {x}")
    rng = np.random.default_rng(len(tails) * 1000 + shared)
    n = len(tails)
    need = -(-shared // page) + sum(1 + -(-t // page) for t in tails) + 2
    width = -(-(shared + max(tails)) // page) + 1
    # whatever the pages hold behind a sequence's end must not matter
    p = Pair4(torch, ops, 2, Hk, D, page, need, n + 2, width)
    p.ref.kv[:] = rng.choice([0, 200, 254, 255], p.ref.kv.shape)
    p.upload()
    _prefix(p, rng, n, shared, tails)
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


@pytest.mark.parametrize("x", ["float32", "float16"])
@pytest.mark.parametrize("D", [64, 128, 96])
def test_attention_masked_places(torch, ops, x, D):
    """NaN blocks in keys and values that some rows of a window do not see yet: the rows before
    them are what they are without them, the rows that see a key's are NaN, those that see a
    value's in its dimensions. Rows of sequences with fewer tokens than queries see nothing."""
    _say(f"masked {x} D{D}")
    rng = np.random.default_rng(8)
    p = Pair4(torch, ops, 1, 2, D, 16, 40, 6, 12)
    _prefix(p, rng, 2, 70, [20, 45])
    p.add(rng, [4], [3])
    # the 4th and the 2nd token from the end of sequences 1 and 2
    for s, back, kinds in [(1, 4, (0, 1)), (2, 2, (1,))]:
        for kind in kinds:
            x_ = rng.standard_normal((2, D))
            x_[:, 40] = np.nan                      # dimensions 32 .. 63
            p.put(0, kind, s, int(p.ref.lens[s]) - back, x_)
    p.upload()
    q = rng.standard_normal((24, 4, D)).astype(x)
    seq, start = [1, 5, 2, 4], [0, 8, 8, 18, 23]    # 8 queries; none; 10; 5 queries of 3 tokens
    ref = p.ref.attention(0, seq, start, q, 0.3, np.full(q.shape, 7.0))
    fine = np.isfinite(ref[:23])
    assert fine[[0, 1, 2, 3] + list(range(8, 16)) + list(range(18, 23))].all() and np.all(ref[18:20] == 0)
    assert not fine[4:8].any() and not fine[16:18, :, 32:64].any() and fine[16:18, :, :32].all()
    assert fine[16:18, :, 64:].all()
    tol = _tolerance(p, 0, seq, start, q, 0.3, x == "float16")

    def check(got, r):
        got, want, ok = got[r].astype(np.float64), ref[:23][r], fine[r]
        assert np.array_equal(np.isfinite(got), ok)
        assert np.abs(got[ok] - want[ok]).max(initial=0) <= tol
    for shared in (0, 33, 70):
        # (sequence 4 has a prefix of its own, and is left out where one is shared)
        m = 4 if not shared else 3
        got = _attend(p, torch, ops, 0, seq[:m], start[:m + 1], q, 0.3, shared, 10)
        check(got, slice(0, 23 if not shared else 18))
        assert np.all(got[23:] == 7) and (not shared or np.all(got[18:] == 7))
        assert shared or np.all(got[18:20] == 0)
    # a prefix that reaches into the window: rows that stand inside it see part of it only
    p.fork([1], [3])
    got = _attend(p, torch, ops, 0, [1, 3], [0, 8, 16], np.concatenate([q[:8], q[:8]]), 0.3, 90, 8)
    for half in (got[:8], got[8:]):
        check(half, slice(0, 8))
    ops.kv_status(p.c)


@pytest.mark.parametrize("x", ["float32", "float16"])
@pytest.mark.parametrize("D", [64, 128, 32])
def test_queries_of_any_size(torch, ops, x, D):
    """Rows of very large, very small, zero, infinite and NaN queries, dimensions of very different size in a
    block, scales of 0, below 0 and large; the output strided, over the queries, and on another stream."""
    _say(f"queries {x} D{D}")
    rng = np.random.default_rng(D)
    p = Pair4(torch, ops, 1, 2, D, 32, 9, 3, 5)
    p.add(rng, [0, 1], [37, 100], scale=3.0)
    q = rng.standard_normal((12, 6, D))
    big = 3e4 if x == "float16" else 1e30
    q[0] *= big / 4
    q[1] *= 1 / big
    q[2] = 0
    q[3, :, 5] = big
    q[4] *= 2.0 ** rng.integers(-12, 3, (6, D))
    q = q.astype(x)
    seq, start = [1, 0], [0, 9, 11]
    for scale in (D ** -0.5, -0.2, 0.0):
        ref = p.ref.attention(0, seq, start, q, scale, np.full(q.shape, 7.0))
        got = _attend(p, torch, ops, 0, seq, start, q, scale, 0, 9).astype(np.float64)
        for r in range(1, 11):                      # by rows: each has a scale of its own
            tol = _tolerance(p, 0, [seq[int(r >= 9)]], [0, 1], q[r:r + 1], scale, x == "float16")
            if r == 3:
                tol = min(tol, 10.0)
            assert np.abs(got[r] - ref[r]).max() <= tol, (scale, r)
        assert np.isfinite(got[0]).all()
    odd = q.copy()
    odd[5, 2, 7], odd[6, 1, 3] = np.inf, np.nan
    got = _attend(p, torch, ops, 0, seq, start, odd, 0.1, 0, 9)
    assert np.isnan(got[5, 2]).all() and np.isnan(got[6, 1]).all()
    bad = np.isnan(got.astype(np.float64)).all(2)
    assert bad.sum() == 2 and np.isnan(got.astype(np.float64)).sum() == 2 * D
    # q and out strided, out over q, on a stream of its own
    wide = np.full((12, 6 * D + 16), 5.0, x)
    wide[:, :6 * D] = q.reshape(12, -1)
    dev = p.dev(wide)
    stream = torch.cuda.Stream()
    ops.kv_attention(p.c, 0, p.ints(seq), p.ints(start), 2, dev, dev, 12, 6, 0.1, max_rows=9, q_stride=6 * D + 16,
                     out_stride=6 * D + 16, stream=stream)
    stream.synchronize()
    again = _attend(p, torch, ops, 0, seq, start, q, 0.1, 0, 9)
    got = dev.cpu().numpy()
    assert np.array_equal(got[:11, :6 * D].reshape(11, 6, D), again[:11]) and np.all(got[:, 6 * D:] == 5)
    assert np.array_equal(got[11], wide[11])
    ops.kv_status(p.c)


@pytest.mark.parametrize("D", [64, 128, 32])
@pytest.mark.parametrize("x", ["float32", "float16"])
def test_attention_bad_pages(torch, ops, D, x):
    """No such sequence: NaN rows. A page outside the cache: the rows that see its keys, and no others."""
    _say(f"bad pages {x} D{D}")
    rng = np.random.default_rng(3)
    p = Pair4(torch, ops, 1, 2, D, 16, 60, 5, 20)
    p.add(rng, [0, 1, 2], [300, 40, 20])
    q = rng.standard_normal((40, 4, D)).astype(x)
    seq, start = [0, 9, 1, 2], [0, 20, 23, 28, 30]
    good = _attend(p, torch, ops, 0, [0, 1, 2], [0, 20, 25, 27], np.concatenate([q[:20], q[23:30]]), 0.2, 0, 20)
    ops.kv_status(p.c)
    got = _attend(p, torch, ops, 0, seq, start, q, 0.2, 0, 20)
    assert np.isnan(got[20:23]).all() and np.all(got[30:] == 7)
    assert np.array_equal(np.concatenate([got[:20], got[23:30]]), good[:27])
    with pytest.raises(ops.RocmError, match="does not have"):
        ops.kv_status(p.c)
    for page, clean in ((18, 8), (3, 0)):          # row r of sequence 0 sees keys 0 .. 280 + r: 288 from row 8 on
        kept = int(p.table[0, page])
        for wrong in (60, -1, 2 ** 31 - 1, -2 ** 31):
            p.table[0, page] = wrong
            torch.cuda.synchronize()
            got = _attend(p, torch, ops, 0, [0, 1, 2], [0, 20, 25, 27], np.concatenate([q[:20], q[23:30]]), 0.2, 0, 20)
            assert np.array_equal(got[:clean], good[:clean]) and np.isnan(got[clean:20]).all()
            assert np.array_equal(got[20:27], good[20:27])
            with pytest.raises(ops.RocmError, match="does not have"):
                ops.kv_status(p.c)
        p.table[0, page] = kept
    # another sequence's bad page is nobody's business
    p.table[0, 18] = 60
    torch.cuda.synchronize()
    _attend(p, torch, ops, 0, [1], [0, 1], q, 0.2, 0, 1)
    ops.kv_status(p.c)
