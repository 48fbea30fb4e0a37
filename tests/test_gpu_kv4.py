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


def _masked_columns(torch, ops, D, H, rows, tokens, x):
    """Items of 32 columns: NaN blocks of values and keys, and what lies behind the end, reach the rows that see them alone;
    more rows than tokens."""
    _say(f"masked columns D{D} {rows} rows of {tokens} {x}")
    rng = np.random.default_rng(D + rows)
    p = _held(torch, ops, rng, [tokens, 70], 2, D, 16)
    codes, scales = p.ref.blocks()
    scales = scales.copy()
    for kind, pos, block in ((1, tokens - 5, 1), (0, tokens - 2, 0), (1, tokens - 1, 0)):
        scales[0, kind, p.ref.table[0, pos // 16], :, block, pos % 16] = 255
    end = p.ref.table[0, (tokens - 1) // 16]
    if tokens % 16:
        scales[0, :, end, :, :, tokens % 16:] = rng.choice([0, 200, 255], scales[0, :, end, :, :, tokens % 16:].shape)
    p.ref.kv = np.concatenate([codes.reshape(*codes.shape[:4], -1), scales.reshape(*scales.shape[:4], -1)],
                              4).reshape(p.ref.kv.shape)
    p.upload()
    q = rng.standard_normal((rows + 2, H, D)).astype(x)
    seq, start = [0, 1], [0, rows, rows + 2]
    ref = p.ref.attention(0, seq, start, q, D ** -0.5, np.zeros(q.shape))
    assert np.isnan(ref[rows - 1]).all() and np.isnan(ref[rows - 5, :, 32:64]).all() and np.isfinite(ref[rows - 5, :, :32]).all()
    tol = _tolerance(p, 0, seq, start, q, D ** -0.5, x == "float16")
    for shared in (0, 64):
        if shared:
            p.table[1] = p.table[0]                 # one prefix, and the tokens behind it
            p.ref.table[1] = p.ref.table[0]
            torch.cuda.synchronize()
            ref = p.ref.attention(0, seq, start, q, D ** -0.5, np.zeros(q.shape))
        got = _attend(p, torch, ops, 0, seq, start, q, D ** -0.5, shared, rows).astype(np.float64)
        fine = np.isfinite(ref)
        assert np.array_equal(np.isfinite(got), fine) and np.abs(got[fine] - ref[fine]).max() <= tol
    ops.kv_status(p.c)


@pytest.mark.parametrize("D,H,rows,tokens", [(128, 32, 300, 300), (64, 32, 300, 333), (64, 14, 8, 100), (128, 32, 300, 290)])
def test_attention_masked_columns(torch, ops, D, H, rows, tokens):
    _masked_columns(torch, ops, D, H, rows, tokens, "float16")


@pytest.mark.parametrize("D,H,rows,tokens", [(128, 32, 300, 300), (64, 14, 200, 213)])
def test_attention_masked_columns_fp32(torch, ops, D, H, rows, tokens):
    _masked_columns(torch, ops, D, H, rows, tokens, "float32")


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


def _bytes(rng, shape_layers, heads, dim, page, pages):
    """Bytes of a cache of normal values, as a server's would be, without the oracle's token by token."""
    ref = kv_ref.Cache4(shape_layers, heads, dim, page, pages, 1, 1)
    codes, scales = ref.blocks()
    codes[:] = rng.integers(0, 256, codes.shape)
    scales[:] = rng.integers(120, 130, scales.shape)
    return ref.kv


def _held(torch, ops, rng, lens, Hk, D, page, common=0, spare=3, order=None):
    """Sequences 0 .. n - 1 of random contents, with their first `common` pages the same."""
    need = [-(-k // page) for k in lens]
    pages = common + sum(max(0, k - common) for k in need) + spare
    p = Pair4(torch, ops, 1, Hk, D, page, pages, len(lens), max(need) + 1)
    p.ref.kv = _bytes(rng, 1, Hk, D, page, pages)
    free = [int(x) for x in rng.permutation(pages)]
    shared = [free.pop() for _ in range(common)]
    for s, (k, n) in enumerate(zip(need, lens)):
        p.ref.table[s, :k] = (shared + [free.pop() for _ in range(k - common)]) if k > common else shared[:k]
        p.ref.lens[s] = n
    for x in p.ref.table[p.ref.table >= 0]:
        p.ref.refs[x] += 1
    p.upload()
    for dev, ref in ((p.table, p.ref.table), (p.lens, p.ref.lens), (p.refs, p.ref.refs)):
        dev.copy_(torch.from_numpy(ref))
    torch.cuda.synchronize()
    return p


def _compare(p, torch, ops, seq, counts, H, D, x, rng, shared, window, most=None):
    """Attention of a batch against the oracle; `most`: of so many of its requests only."""
    start = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    q = rng.standard_normal((int(start[-1]), H, D)).astype(x)
    got = _attend(p, torch, ops, 0, seq, start, q, D ** -0.5, shared, window)
    again = _attend(p, torch, ops, 0, seq, start, q, D ** -0.5, shared, window)
    assert np.array_equal(got, again)
    for i in (range(len(seq)) if most is None else rng.permutation(len(seq))[:most]):
        rows = slice(start[i], start[i + 1])
        one = [0, counts[i]]
        ref = p.ref.attention(0, [seq[i]], one, q[rows], D ** -0.5, np.zeros(q[rows].shape))
        tol = _tolerance(p, 0, [seq[i]], one, q[rows], D ** -0.5, x == "float16")
        assert np.abs(got[rows].astype(np.float64) - ref).max(initial=0) <= tol
    ops.kv_status(p.c)
    return q, got


@pytest.mark.parametrize("n,x,D", [(64, "float16", 128), (65, "float32", 64), (256, "float16", 64), (257, "float32", 128),
                                   (700, "float16", 128)])
def test_attention_many_requests(torch, ops, n, x, D):
    """As many requests as a wave finds on its own, and one more; ragged lengths, empty requests among them, windows
    longer than announced."""
    _say(f"{n} requests {x} D{D}")
    rng = np.random.default_rng(n)
    lens = [int(k) for k in np.exp(rng.uniform(0, np.log(600), n))]
    p = _held(torch, ops, rng, lens, 2, D, 16)
    seq = [int(s) for s in rng.permutation(n)]
    counts = [int(rng.integers(0, min(4, lens[s]) + 1)) for s in seq]
    for window in (1, 4):
        _compare(p, torch, ops, seq, counts, 14, D, x, rng, 0, window, 60)


@pytest.mark.parametrize("H,Hk,D,page,x,tail,window,shared", [
    (8, 1, 128, 16, "float16", 20011, 1, 0),        # runs of one sequence, over one kv head
    (8, 1, 128, 128, "float32", 20011, 2, 0),
    (8, 4, 64, 64, "float16", 9973, 5, 0),
    (16, 2, 128, 32, "float16", 37, 3, 12320),      # a long prefix of many columns
    (16, 2, 64, 16, "float32", 700, 1, 17001),
    (24, 2, 128, 16, "float32", 3, 7, 2999),        # rows that stand inside the prefix
    (32, 4, 128, 32, "float16", 37, 3, 12320),      # items of 32 columns, for a prefix and for a prompt
    (32, 4, 128, 16, "float16", 2, 4, 17003),
    (32, 2, 128, 16, "float16", 313, 300, 0),
    (32, 2, 64, 64, "float16", 1313, 300, 0),
])
def test_attention_long(torch, ops, H, Hk, D, page, x, tail, window, shared):
    """Many tiles of a wave, more than one load of page ids holds, and runs that are joined."""
    _say(f"long H{H}/{Hk} D{D} page {page} {x} {shared} + {tail}")
    rng = np.random.default_rng(tail)
    n = 1 if not shared else 12
    lens = [shared + max(1, tail - 11 * i) for i in range(n)]
    p = _held(torch, ops, rng, lens, Hk, D, page, shared // page)
    if shared % page:                               # the prefix's last tokens lie in a page of each one's own
        codes, scales = p.ref.blocks()
        at, k = p.ref.table[:, shared // page], shared % page
        codes, scales = codes.copy(), scales.copy()
        for s in range(1, n):
            codes[:, :, at[s], :, :k] = codes[:, :, at[0], :, :k]
            scales[:, :, at[s], :, :, :k] = scales[:, :, at[0], :, :, :k]
        p.ref.kv = np.concatenate([codes.reshape(*codes.shape[:4], -1), scales.reshape(*scales.shape[:4], -1)],
                                  4).reshape(p.ref.kv.shape)
        p.upload()
    seq = [int(s) for s in rng.permutation(n)]
    counts = [min(window, lens[s]) for s in seq]
    q, got = _compare(p, torch, ops, seq, counts, H, D, x, rng, shared, window, 5)
    if shared:
        assert np.abs(_attend(p, torch, ops, 0, seq, np.concatenate([[0], np.cumsum(counts)]), q, D ** -0.5, 0, 1)
                      .astype(np.float64) - got).max() <= 2 * _tolerance(p, 0, seq[:1], [0, 1], q[:1], D ** -0.5, x == "float16")


@pytest.mark.parametrize("H,Hk,D,page,tail,window,shared", [
    (32, 2, 128, 16, 313, 300, 0),                  # prompts
    (32, 2, 64, 64, 1313, 300, 0),
    (32, 2, 128, 32, 90, 70, 6000),                 # windows behind a prefix
    (14, 2, 64, 16, 190, 150, 2999),
])
def test_attention_long_fp32(torch, ops, H, Hk, D, page, tail, window, shared):
    """Items of 32 columns of fp32 queries."""
    test_attention_long(torch, ops, H, Hk, D, page, "float32", tail, window, shared)


def test_far_pages(torch, ops):
    """Pages beyond 4 GB: the same tokens there and in a small cache, written, read and attended to."""
    rng = np.random.default_rng(11)
    Hk, D, page = 8, 128, 64
    pages = (5 << 30) // (Hk * page * 68)           # of each of k and v
    small = Pair4(torch, ops, 1, Hk, D, page, 8, 2, 8)
    far = torch.empty((1, 2, pages, Hk, page, 68), dtype=torch.uint8, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, refs = torch.full((2, 8), -1, **i32), torch.zeros(2, **i32), torch.ones(pages, **i32)
    ids = [pages - 1, pages // 2, pages - 7, 3]
    refs[ids] = 0
    c = ops.KvCache(far, table, lens, refs)
    n = 200
    small.reserve([0], [n])
    torch.cuda.synchronize()
    ops.kv_reserve(c, small.ints([0]), small.ints([n]), 1)
    torch.cuda.synchronize()
    assert sorted(table[0, :4].tolist()) == sorted(ids)
    k, v = (rng.standard_normal((1, n, Hk, D)).astype(np.float32) for _ in range(2))
    small.write(0, [0], [0, n], k, v)
    ops.kv_write(c, 0, 1, small.ints([0]), small.ints([0, n]), 1, small.dev(k), small.dev(v), n)
    small.same()
    back = small.read(0, 1, [0], [0, n], None, torch.float32)
    kb, vb = (torch.zeros(n * Hk * D, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    ops.kv_read(c, 0, 1, small.ints([0]), small.ints([0, n]), 1, kb, vb, n)
    torch.cuda.synchronize()
    assert np.array_equal(kb.cpu().numpy(), back[0]) and np.array_equal(vb.cpu().numpy(), back[1])
    for x in ("float32", "float16"):
        q = rng.standard_normal((3, 16, D)).astype(x)
        want = _attend(small, torch, ops, 0, [0], [0, 3], q, 0.1, 0, 3)
        qd = small.dev(q)
        out = torch.zeros_like(qd)
        torch.cuda.synchronize()
        ops.kv_attention(c, 0, small.ints([0]), small.ints([0, 3]), 1, qd, out, 3, 16, 0.1, max_rows=3)
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
    ops.kv_status(c)
    c.close()


def test_write_leaves_the_rest(torch, ops):
    """Strided rows and layers, rows behind the last request, a layer in the middle."""
    rng = np.random.default_rng(14)
    p = Pair4(torch, ops, 3, 2, 32, 16, 12, 4, 3, fill=0)
    p.reserve([3, 1], [21, 7])
    start = [0, 19, 24]                             # the last 19 of 21, and 5 of 7
    k, v = (rng.standard_normal((2, 27, 80)).astype(np.float32) for _ in range(2))
    k[:, 24:], v[:, 24:] = np.nan, np.nan
    for row_stride, layer_stride in ((80, 27 * 80), (160, 80)):
        a, b = ((x if layer_stride > 80 else np.ascontiguousarray(x.transpose(1, 0, 2))) for x in (k, v))
        ops.kv_write(p.c, 1, 2, p.ints([3, 1]), p.ints(start), 2, p.dev(a), p.dev(b), 27, row_stride=row_stride,
                     layer_stride=layer_stride)
        p.ref.write(1, [3, 1], start, *(x[:, :, :64].reshape(2, 27, 2, 32) for x in (k, v)))
        p.same()
        k, v = k * 3, v * 0.1
    ops.kv_status(p.c)


def test_refused_writes(torch, ops):
    """What kv_write refuses of other caches it refuses here: rows in shared pages, one sequence twice, tokens that a
    refused reserve did not make room for."""
    rng = np.random.default_rng(12)
    p = Pair4(torch, ops, 2, 2, 64, 16, 9, 6, 4)
    p.add(rng, [0], [20])
    p.fork([0], [1])
    k, v = (p.dev(rng.standard_normal((2, 8, 2, 64)).astype(np.float32)) for _ in range(2))
    ops.kv_write(p.c, 0, 2, p.ints([1]), p.ints([0, 4]), 1, k, v, 8)
    p.same()
    with pytest.raises(ops.RocmError, match="several sequences hold"):
        ops.kv_status(p.c)
    p.reserve([2, 3], [3, 3])
    ops.kv_write(p.c, 0, 2, p.ints([2, 3, 2]), p.ints([0, 3, 6, 8]), 3, k, v, 8)
    kn, vn = k.cpu().numpy(), v.cpu().numpy()
    p.ref.write(0, [2, 3], [0, 3, 6], kn, vn)
    p.same()
    with pytest.raises(ops.RocmError, match="twice"):
        ops.kv_status(p.c)
    with pytest.raises(kv_ref.Refused):
        p.ref.reserve([2, 4], [1, 200])
    ops.kv_reserve(p.c, p.ints([2, 4]), p.ints([1, 200]), 2)
    ops.kv_write(p.c, 0, 2, p.ints([2]), p.ints([0, 1]), 1, k, v, 8)
    p.same()
    with pytest.raises(ops.RocmError, match="too short table rows"):
        ops.kv_status(p.c)


def test_serving(torch, ops):
    """Prompt, forks, steps of ragged windows over two layers, drops and compaction, as a server would."""
    rng = np.random.default_rng(13)
    layers, Hk, H, D, page = 2, 2, 8, 128, 16
    p = Pair4(torch, ops, layers, Hk, D, page, 60, 9, 12)
    p.add(rng, [0], [70])
    p.fork([0] * 4, [1, 2, 3, 4])
    for step in range(6):
        seq = [int(s) for s in 1 + rng.permutation(4)]
        count = [int(k) for k in rng.integers(1, 6, 4)]
        p.reserve(seq, count)
        start = np.concatenate([[0], np.cumsum(count)]).astype(int)
        rows = int(start[-1])
        k, v = (rng.standard_normal((layers, rows, Hk, D)).astype(np.float32) for _ in range(2))
        for layer in range(layers):
            p.write(layer, seq, start, k[layer:layer + 1], v[layer:layer + 1])
            q = rng.standard_normal((rows, H, D)).astype(np.float32)
            got = _attend(p, torch, ops, layer, seq, start, q, D ** -0.5, 70, max(count))
            ref = p.ref.attention(layer, seq, start, q, D ** -0.5, np.zeros(q.shape))
            assert np.abs(got - ref).max() <= _tolerance(p, layer, seq, start, q, D ** -0.5, False)
        p.drop(seq, [int(rng.integers(0, c)) for c in count])
        if step % 2:
            p.compact()
        p.same()
    ops.kv_status(p.c)


class Step4:
    """One step of a server over a cache of 4 bits of its own: room, write, attention, read back, drop."""

    def __init__(self, torch, ops, seed):
        self.t, self.ops, self.rng = torch, ops, np.random.default_rng(seed)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.kv = torch.zeros((2, 2, 40, 2, 16, 68), dtype=torch.uint8, device="cuda")
        self.table, self.lens, self.refs = torch.full((5, 12), -1, **i32), torch.zeros(5, **i32), torch.zeros(40, **i32)
        self.c = ops.KvCache(self.kv, self.table, self.lens, self.refs)
        self.seq = torch.tensor([3, 0, 4], **i32)
        self.count, self.start = torch.tensor([2, 1, 3], **i32), torch.tensor([0, 2, 3, 6], **i32)
        self.back = torch.tensor([1, 0, 2], **i32)
        self.k, self.v = (torch.zeros((2, 6, 2, 128), device="cuda") for _ in range(2))
        self.q, self.out = (torch.zeros((6, 8, 128), device="cuda") for _ in range(2))
        self.kb, self.vb = (torch.zeros((2, 6, 2, 128), device="cuda", dtype=torch.float16) for _ in range(2))

    def fill(self, rng):
        for t in (self.k, self.v, self.q):
            t.copy_(self.t.from_numpy(rng.standard_normal(tuple(t.shape)).astype(np.float32)))

    def run(self, stream=None):
        o, c = self.ops, self.c
        o.kv_reserve(c, self.seq, self.count, 3, stream=stream)
        o.kv_write(c, 0, 2, self.seq, self.start, 3, self.k, self.v, 6, stream=stream)
        o.kv_attention(c, 1, self.seq, self.start, 3, self.q, self.out, 6, 8, 0.09, max_rows=3, stream=stream)
        o.kv_read(c, 0, 2, self.seq, self.start, 3, self.kb, self.vb, 6, stream=stream)
        o.kv_drop(c, self.seq, self.back, 3, stream=stream)

    def state(self):
        return [t.clone() for t in (self.kv, self.table, self.lens, self.refs, self.out, self.kb, self.vb)]


def _same_steps(torch, steps):
    torch.cuda.synchronize()
    first = steps[0].state()
    for s in steps[1:]:
        for a, b in zip(first, s.state()):
            assert torch.equal(a, b)


def test_captured_step(torch, ops):
    """A step captured into a graph of torch's, replayed with new inputs between eager ones on two streams."""
    eager, captured, other = (Step4(torch, ops, s) for s in (1, 1, 1))
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for s, st in zip((captured, other), streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run(st)
        graphs.append(g)
    torch.cuda.synchronize()
    for step in range(12):
        for s in (eager, captured, other):
            s.fill(np.random.default_rng(100 + step))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):          # at once, each with its own workspaces
            with torch.cuda.stream(st):
                g.replay()
        eager.run()
        _same_steps(torch, (eager, captured, other))
    assert eager.lens.tolist() == [12, 0, 0, 12, 12] and float(eager.out.abs().sum()) > 0
    for s in (eager, captured, other):
        ops.kv_status(s.c)
    graphs.clear()
