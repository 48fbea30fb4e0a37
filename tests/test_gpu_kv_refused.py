"""The paged cache where a call is refused on the device, or part of what it reads
is outside the cache: nothing but the refused request changes, and only rows that
see what is wrong are NaN. Pages, tables, lengths and counts are held to equality,
attention to the bounds derived in test_gpu_kv_cache.py."""
import numpy as np
import pytest

from oracle import kv_ref
from test_gpu_kv_cache import Pair, _attend, _prefix, _say, _tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(torch_dev):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from mod_amd import ops
    return ops


def _rows(rng, p, n):
    """Keys and values of n rows in all layers."""
    shape = (p.ref.kv.shape[0], n, p.ref.kv.shape[3], p.ref.kv.shape[5])
    return [rng.standard_normal(shape).astype(np.float32) for _ in range(2)]


def _write(p, rng, seq, count, known=True):
    """The last count[i] tokens of seq[i] written, in the oracle too where `known`."""
    start = np.concatenate([[0], np.cumsum(count)]).astype(int)
    k, v = _rows(rng, p, int(start[-1]))
    p.ops.kv_write(p.c, 0, k.shape[0], p.ints(seq), p.ints(start), len(seq), p.dev(k), p.dev(v), k.shape[1])
    if known:
        p.ref.write(0, list(seq), start, k, v)


# ------------------------------------------------------- a reserve is refused ---
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("tokens", [32, 37])
def test_refused_step_changes_nothing(torch, ops, dtype, tokens):
    """A step whose reserve finds too few pages: its writes would fall onto tokens that the sequences
    have, in pages that they share, and its drop onto tokens that they keep."""
    _say(f"refused step {dtype} {tokens}")
    rng = np.random.default_rng(tokens)
    p = Pair(torch, ops, 2, 2, 64, 16, 7, 6, 4, dtype)
    p.add(rng, [0], [tokens])
    p.fork([0, 0, 0, 0], [1, 2, 3, 4])
    seq, count = [1, 2, 3], [3, 18, 40]
    with pytest.raises(kv_ref.Refused):
        p.ref.reserve(seq, count)
    ops.kv_reserve(p.c, p.ints(seq), p.ints(count), 3)
    _write(p, rng, seq, [3, 18, 1], known=False)
    ops.kv_drop(p.c, p.ints(seq), p.ints([2, 17, 39]), 3)
    p.same()
    # a request that ends is dropped all the same, and one that is not of the refused step is served
    p.drop([3])
    p.add(rng, [4], [1])
    _write(p, rng, [1], [1], known=False)
    p.same()
    with pytest.raises(ops.RocmError, match="too few free pages"):
        ops.kv_status(p.c)
    # once that is known, or the next reserve is served, the sequences are as any other
    p.drop([2], [4])
    p.same()
    p.add(rng, [1, 2], [2, 3])
    p.drop([1], [1])
    p.same()
    ops.kv_status(p.c)


def test_next_step_is_served(torch, ops):
    """Without a status between: the step behind a refused one is served, a slot that ends and begins
    again is a new sequence, and a reserve of other sequences does not set the refused ones free."""
    rng = np.random.default_rng(2)
    p = Pair(torch, ops, 1, 2, 16, 4, 8, 6, 6)
    p.add(rng, [0, 1, 2], [6, 3, 5])                # 5 of 8 pages
    for seq, count in (([0, 1], [12, 8]), ([2, 2], [1, 1]), ([2], [-1])):
        ops.kv_reserve(p.c, p.ints(seq), p.ints(count), len(seq))
    p.add(rng, [3], [1])
    _write(p, rng, [0, 1, 2], [1, 1, 1], known=False)
    ops.kv_drop(p.c, p.ints([0, 1, 2]), p.ints([1, 2, 3]), 3)
    p.same()
    p.add(rng, [0], [3])
    p.drop([0], [1])
    p.same()
    p.drop([1])
    p.fork([0], [1])
    p.drop([1], [4])                                # a branch from an earlier token
    p.same()
    with pytest.raises(ops.RocmError):
        ops.kv_status(p.c)
    ops.kv_reserve(p.c, p.ints([2]), p.ints([400]), 1)
    ops.kv_init(p.c)
    p.ref = kv_ref.Cache(1, 2, 16, 4, 8, 6, 6)
    p.ref.kv[:] = p.kv.cpu().numpy()
    p.add(rng, [2], [5])
    p.drop([2], [2])
    p.same()
    ops.kv_status(p.c)


def test_captured_steps_until_the_pages_run_out(torch, ops):
    """Reserve, write, attention and a drop by counts in one graph, replayed until the pages run out and
    beyond: from then on nothing changes, until a sequence ends and the steps are served again."""
    rng = np.random.default_rng(3)
    p = Pair(torch, ops, 1, 2, 64, 16, 9, 5, 8, "float16")
    p.add(rng, [0], [40])
    p.fork([0, 0], [1, 2])
    seq, start, count, drop = p.ints([1, 2]), p.ints([0, 7, 12]), p.ints([7, 5]), p.ints([2, 1])
    k, v = (torch.empty(1, 12, 2 * 64, device="cuda") for _ in range(2))
    q, out = torch.randn(12, 4, 64, device="cuda"), torch.empty(12, 4, 64, device="cuda")
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        ops.kv_reserve(p.c, seq, count, 2, stream=st)
        ops.kv_write(p.c, 0, 1, seq, start, 2, k, v, 12, stream=st)
        ops.kv_attention(p.c, 0, seq, start, 2, q, out, 12, 4, 0.125, shared=40, max_rows=7, stream=st)
        ops.kv_drop(p.c, seq, drop, 2, stream=st)
    refused = 0
    for i in range(14):
        _say(f"replay {i}")
        kk, vv = (rng.standard_normal((1, 12, 2, 64)).astype(np.float32) for _ in range(2))
        k.copy_(torch.from_numpy(kk).reshape(1, 12, 128)), v.copy_(torch.from_numpy(vv).reshape(1, 12, 128))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        torch.cuda.synchronize()
        try:
            p.ref.reserve([1, 2], [7, 5])
        except kv_ref.Refused:
            refused += 1
            p.same()
            if refused == 3:                        # the two that ran out end, and begin again
                with pytest.raises(ops.RocmError, match="too few free pages"):
                    ops.kv_status(p.c, stream=st)
                p.drop([1, 2])
                p.fork([0, 0], [1, 2])
            continue
        p.ref.write(0, [1, 2], [0, 7, 12], kk, vv)
        ref = p.ref.attention(0, [1, 2], [0, 7, 12], q.cpu().numpy(), 0.125, np.zeros((12, 4, 64)))
        tol = _tolerance(p, 0, [1, 2], [0, 7, 12], q.cpu().numpy(), 0.125, False)
        assert np.abs(out.cpu().numpy() - ref).max() <= tol
        assert p.ref.drop([1, 2], [2, 1]) == []
        p.same()
    assert 3 <= refused <= 8


# -------------------------------------------------------------- shared pages ---
def test_write_into_shared_pages_is_refused(torch, ops):
    """Rows that fall into pages of another table entry: a fork without room of its own, a request that
    rewrites tokens which it shares. The rows of the same call in pages of their own are written."""
    rng = np.random.default_rng(5)
    p = Pair(torch, ops, 2, 1, 16, 4, 20, 5, 6)
    p.add(rng, [0, 3], [10, 6])
    p.fork([0], [1])
    _write(p, rng, [1], [1], known=False)           # nothing of its own yet
    p.same()
    with pytest.raises(ops.RocmError):
        ops.kv_status(p.c)
    p.reserve([1, 0], [3, 0])
    start = [0, 5, 8]                               # tokens 8 and on are in its own copy; tokens 0 .. 7 are common
    k, v = _rows(rng, p, 8)
    ops.kv_write(p.c, 0, 2, p.ints([1, 3]), p.ints(start), 2, p.dev(k), p.dev(v), 8)
    p.ref.write(0, [1], [0, 5], k[:, :5], v[:, :5])
    p.ref.write(0, [3], [0, 3], k[:, 5:], v[:, 5:])
    p.same()
    ops.kv_status(p.c)
    k, v = _rows(rng, p, 9)
    before = p.ref.kv.copy()
    ops.kv_write(p.c, 0, 2, p.ints([1, 3]), p.ints([0, 7, 9]), 2, p.dev(k), p.dev(v), 9)
    p.ref.write(0, [1], [0, 7], k[:, :7], v[:, :7])
    for t in (6, 7):                                # common tokens: left as they were
        page = int(p.ref.table[1, t // 4])
        p.ref.kv[:, :, page, :, t % 4] = before[:, :, page, :, t % 4]
    p.ref.write(0, [3], [0, 2], k[:, 7:], v[:, 7:])
    p.same()
    with pytest.raises(ops.RocmError):
        ops.kv_status(p.c)


def test_write_of_one_sequence_twice(torch, ops):
    """The first of two requests for a sequence is carried out, the other refused; one without rows is none."""
    rng = np.random.default_rng(6)
    p = Pair(torch, ops, 1, 2, 32, 4, 400, 400, 6)
    p.add(rng, list(range(300)), [4] * 300)
    seq, start = list(range(300)) + [7, 9], list(range(301)) + [301, 301]
    k, v = _rows(rng, p, 301)
    ops.kv_write(p.c, 0, 1, p.ints(seq), p.ints(start), 302, p.dev(k), p.dev(v), 301)
    p.ref.write(0, seq[:300], start[:301], k, v)
    p.same()
    with pytest.raises(ops.RocmError, match="twice"):
        ops.kv_status(p.c)
    ops.kv_write(p.c, 0, 1, p.ints([7, 9, 9]), p.ints([0, 2, 2, 5]), 3, p.dev(k), p.dev(v), 5)
    p.ref.write(0, [7, 9], [0, 2, 5], k, v)
    p.same()
    ops.kv_status(p.c)


def test_fork_of_a_bad_page(torch, ops):
    """A source whose table row holds a page outside the cache is refused, and the target stays empty."""
    rng = np.random.default_rng(7)
    p = Pair(torch, ops, 1, 1, 8, 1, 700, 6, 600)
    p.add(rng, [0, 1], [560, 3])
    for at, page in ((0, -1), (3, 700), (559, 1 << 30)):
        p.table[0, at] = page
        ops.kv_fork(p.c, p.ints([0, 1]), p.ints([2, 3]), 2)
        torch.cuda.synchronize()
        p.table[0, at] = int(p.ref.table[0, at])
        p.ref.fork([1], [3])
        p.same()
        with pytest.raises(ops.RocmError):
            ops.kv_status(p.c)
        p.drop([3])
    assert p.fork([0, 1], [2, 3]) == []
    p.same()
    ops.kv_status(p.c)


# ----------------------------------------------------------------- attention ---
@pytest.mark.parametrize("kv", ["float32", "float16"])
@pytest.mark.parametrize("D", [40, 64, 128, 256])
def test_attention_bad_id_first(torch, ops, D, kv):
    """A bad id at the head of the list, as of a slot without a request. Where nothing is shared, only its
    own rows are NaN; where something is, the rows have no prefix to read."""
    _say(f"bad id first D{D} {kv}")
    rng = np.random.default_rng(11)
    p = Pair(torch, ops, 1, 2, D, 16, 20, 5, 10, kv)
    _prefix(p, rng, 3, 40, [4, 40, 20])
    q = rng.standard_normal((4, 4, D)).astype(np.float32)
    start = [0, 1, 2, 3, 4]
    good = _attend(p, torch, ops, 0, [1, 3, 2, 1], start, q, 0.125, 0, 1)
    ops.kv_status(p.c)
    for bad in (5, -1):
        got = _attend(p, torch, ops, 0, [bad, 3, 2, 1], start, q, 0.125, 0, 1)
        assert np.isnan(got[0]).all() and np.array_equal(got[1:], good[1:])
        with pytest.raises(ops.RocmError):
            ops.kv_status(p.c)
        # a slot without rows is not looked at
        got = _attend(p, torch, ops, 0, [bad, 3, 2, 1], [1, 1, 2, 3, 4], q, 0.125, 0, 1)
        assert np.all(got[0] == 7) and np.array_equal(got[1:], good[1:])
        ops.kv_status(p.c)
        assert np.isnan(_attend(p, torch, ops, 0, [bad, 3, 2, 1], start, q, 0.125, 40, 1)).all()
        with pytest.raises(ops.RocmError):
            ops.kv_status(p.c)


@pytest.mark.parametrize("n,Hk,D,rows,kv,x", [(4096, 32, 64, 4200, "float16", "float16"),
                                              (1024, 16, 64, 5000, "float32", "float32")])
def test_attention_one_long_window_among_many(torch, ops, n, Hk, D, rows, kv, x):
    """A prompt in a batch of single tokens, with the right max_rows: n x kv heads x column tiles of the
    longest window are more items than a launch has."""
    _say(f"one long window among {n} {kv}")
    rng = np.random.default_rng(15)
    i32 = dict(dtype=torch.int32, device="cuda")
    long = n // 3
    counts = np.ones(n, int)
    counts[long] = rows
    lens = rng.integers(1, 12, n)
    lens[long] = rows + 30
    start = np.concatenate([[0], np.cumsum(counts)])
    all_rows = np.concatenate([[0], np.cumsum(lens)])
    page, total, R = 8, int(lens.sum()), int(start[-1])
    pages = int((-(-lens // page)).sum())
    k, v = (torch.randn(1, total, Hk * D, device="cuda").to(getattr(torch, kv)) for _ in range(2))
    cache = ops.KvCache(torch.empty(1, 2, pages, Hk, page, D, dtype=k.dtype, device="cuda"),
                        torch.empty(n, -(-(rows + 30) // page), **i32), torch.empty(n, **i32), torch.empty(pages, **i32))
    q = torch.randn(R, Hk, D, device="cuda").to(getattr(torch, x))
    out = torch.full_like(q, 7)
    seq, dstart = torch.arange(n, **i32), torch.from_numpy(start).to(**i32)
    dlens, dall = torch.from_numpy(lens).to(**i32), torch.from_numpy(all_rows).to(**i32)
    torch.cuda.synchronize()
    ops.kv_init(cache)
    ops.kv_reserve(cache, seq, dlens, n)
    ops.kv_write(cache, 0, 1, seq, dall, n, k, v, total)
    ops.kv_attention(cache, 0, seq, dstart, n, q, out, R, Hk, 0.125, max_rows=rows)
    ops.kv_status(cache)
    # |score| < 8 over up to 5,030 keys: 2 es + 8 u + 4 u sqrt(T), es = 4 u sqrt(64) 9
    u = 2.0 ** -24
    far = 2 * 4 * u * 8 * 9 + 8 * u + 4 * u * np.sqrt(rows + 30) + (2.0 ** -11 if x == "float16" else 0.0)
    vmax = float(v.abs().max())
    tol = vmax * (far + (2.0 ** -11 if x == "float16" else 0.0))
    for i in [0, 1, long - 1, long, long + 1, n - 1]:
        a, b, c, d = int(start[i]), int(start[i + 1]), int(all_rows[i]), int(all_rows[i + 1])
        late = torch.arange(d - c, device="cuda") > (d - c) - (b - a) + torch.arange(b - a, device="cuda")[:, None]
        for h in range(0, Hk, 5):
            kk, vv = (t[0, c:d, h * D:(h + 1) * D].double() for t in (k, v))
            s = (torch.mm(q[a:b, h].double(), kk.T.contiguous()) * 0.125).masked_fill(late, -torch.inf)
            ref = torch.mm(torch.softmax(s, 1), vv)
            assert float((out[a:b, h].double() - ref).abs().max()) <= tol
    # every other request has one row: the mean over its keys by their weights, all at once
    ones = [i for i in range(n) if i != long]
    at = torch.from_numpy(start[:-1][ones]).cuda()
    width = torch.arange(11, device="cuda")
    key = torch.from_numpy(all_rows[:-1][ones]).cuda()[:, None] + width
    dead = width >= torch.from_numpy(lens[ones]).cuda()[:, None]
    kk, vv = (t[0][key.clamp(max=total - 1)].reshape(len(ones), 11, Hk, D).double() for t in (k, v))
    s = ((kk * q[at].double()[:, None]).sum(3) * 0.125).masked_fill(dead[:, :, None], -torch.inf)
    ref = (torch.softmax(s, 1)[..., None] * vv).sum(1)
    assert float((out[at].double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("kv,x", [("float32", "float32"), ("float16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("D,window", [(64, 1), (128, 3), (128, 40), (40, 3)])
def test_attention_bad_page_of_the_prefix(torch, ops, kv, x, D, window):
    """A page outside the cache in the table row that the common tokens are read through: the rows that see
    it are NaN and it is reported; rows that stand before it are what they are, and nothing is reported
    where no row sees it."""
    _say(f"bad page of the prefix D{D} window {window} {kv} {x}")
    rng = np.random.default_rng(12)
    p = Pair(torch, ops, 1, 1, D, 16, 40, 6, 20, kv, fill=np.nan)
    _prefix(p, rng, 4, 150, [4, 60, 41, 50])
    p.drop([2, 3], [150, 186])                      # 60 and 5 tokens are left of these
    seq, counts = [1, 2, 3, 4], [min(window, 4), window, min(window, 9), window]
    start = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    q = rng.standard_normal((int(start[-1]), 4, D)).astype(x)
    ref = p.ref.attention(0, seq, start, q, 0.1, np.zeros(q.shape))
    tol = _tolerance(p, 0, seq, start, q, 0.1, x == "float16")
    limit = np.concatenate([int(p.ref.lens[s]) - n + 1 + np.arange(n) for s, n in zip(seq, counts)])
    shared = 150
    good = _attend(p, torch, ops, 0, seq, start, q, 0.1, shared, window)
    assert np.abs(good.astype(np.float64) - ref).max() <= tol
    ops.kv_status(p.c)
    for at, page in ((4, 40), (3, -1), (2, 1 << 30), (0, -5)):        # (its first token is 64, 48, 32, 0)
        was = int(p.table[1, at])
        p.table[1, at] = page
        got = _attend(p, torch, ops, 0, seq, start, q, 0.1, shared, window)
        sees = limit > 16 * at
        assert np.isnan(got[sees]).all()
        assert np.abs(got[~sees].astype(np.float64) - ref[~sees]).max(initial=0) <= tol
        with pytest.raises(ops.RocmError):
            ops.kv_status(p.c)
        # the short ones alone, behind the first one's table row, whose own rows are left out
        short = [int(start[1])] + [int(v) for v in start[1:4]]
        got = _attend(p, torch, ops, 0, seq[:3], short, q, 0.1, shared, window)
        for r in range(int(start[1]), int(start[3])):
            assert np.isnan(got[r]).all() if sees[r] else np.abs(got[r].astype(np.float64) - ref[r]).max() <= tol
        if sees[start[1]:start[3]].any():
            with pytest.raises(ops.RocmError):
                ops.kv_status(p.c)
        ops.kv_status(p.c)
        p.table[1, at] = was
