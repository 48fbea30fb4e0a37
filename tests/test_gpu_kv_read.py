"""Tokens read out of a paged cache (mod_amd/csrc/kv_pages.hip, kv_read_kernel) against
oracle/kv_ref.py: behind a refused reserve, and out of caches of every type, head
dimension and page size. A value is a function of one stored value: held to equality."""
import numpy as np
import pytest

from oracle import kv_ref
from test_gpu_kv4 import Pair4
from test_gpu_kv_cache import Pair, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(torch_dev):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from mod_amd import ops
    return ops


def _pair(torch, ops, kind, layers, heads, dim, page, pages, seqs, width):
    if kind == "mx4":
        return Pair4(torch, ops, layers, heads, dim, page, pages, seqs, width)
    p = Pair(torch, ops, layers, heads, dim, page, pages, seqs, width, kind)
    p.ref.D = dim
    return p


@pytest.mark.parametrize("kind", ["float32", "float16", "mx4"])
def test_behind_a_refused_reserve(torch, ops, kind):
    """Rows counted from the end of a sequence that is held up are NaN, and the status stays that of the reserve: until
    the status is asked, a reserve serves the sequence, or it ends."""
    _say(f"read behind a refused reserve {kind}")
    rng = np.random.default_rng(21)
    p = _pair(torch, ops, kind, 2, 2, 32, 16, 8, 5, 4)
    p.add(rng, [0, 1, 2], [20, 17, 5])

    def read(seq, start, first=None):
        got = Pair4.read(p, 0, 2, seq, start, first, torch.float32)
        return [x.reshape(2, start[-1], 64) for x in got]

    def want(s, at):
        return [[x[at].reshape(-1, 64) for x in p.ref.rows(layer, s, int(p.ref.lens[s]))] for layer in range(2)]

    def same(got, rows, s, at):
        return all(np.array_equal(got[kind][layer, rows], want(s, at)[layer][kind]) for kind in range(2) for layer in range(2))
    same_seq = lambda got: same(got, slice(3, 5), 2, slice(3, 5))  # noqa: E731

    def refuse(seq, count):
        ops.kv_reserve(p.c, p.ints(seq), p.ints(count), len(seq))
        with pytest.raises(kv_ref.Refused):
            p.ref.reserve(seq, count)
    refuse([0, 1], [3, 200])
    got = read([0, 2, 1], [0, 3, 5, 6])
    assert all(np.isnan(x[:, :3]).all() and np.isnan(x[:, 5]).all() for x in got) and same_seq(got)
    # tokens named by their place are what they are; those that the reserve did not bring are not there
    got = read([0, 1], [0, 4, 6], [18, 3])
    assert all(np.isnan(x[:, 2:4]).all() for x in got)
    assert same(got, slice(0, 2), 0, slice(18, 20)) and same(got, slice(4, 6), 1, slice(3, 5))
    with pytest.raises(ops.RocmError, match="too few free pages"):
        ops.kv_status(p.c)
    got = read([0, 1], [0, 3, 4])
    assert same(got, slice(0, 3), 0, slice(17, 20)) and same(got, slice(3, 4), 1, slice(16, 17))
    ops.kv_status(p.c)
    # a reserve that serves one of them
    refuse([0, 1], [200, 1])
    p.reserve([0], [2])
    k, v = (rng.standard_normal((2, 2, 2, 32)).astype(np.float32) for _ in range(2))
    p.write(0, [0], [0, 2], k, v)
    got = read([0, 1], [0, 4, 5])
    assert same(got, slice(0, 4), 0, slice(18, 22)) and all(np.isnan(x[:, 4]).all() for x in got)
    # and the end of the other
    p.drop([1])
    p.fork([0], [1])
    got = read([1], [0, 22])
    assert same(got, slice(0, 22), 1, slice(0, 22))
    with pytest.raises(ops.RocmError, match="too few free pages"):
        ops.kv_status(p.c)
    # a page outside the cache is still reported where its sequence is held up
    refuse([0], [200])
    p.table[0, 0] = -1
    got = read([0], [0, 3], [14])
    assert all(np.isnan(x[:, :2]).all() and not np.isnan(x[:, 2]).any() for x in got)
    with pytest.raises(ops.RocmError, match="does not have"):
        ops.kv_status(p.c)


@pytest.mark.parametrize("x", ["float32", "float16"])
@pytest.mark.parametrize("kind,heads,dim,page,layers", [
    ("float32", 1, 8, 1, 1), ("float32", 3, 40, 2, 3), ("float32", 8, 128, 16, 2), ("float32", 2, 256, 1024, 2),
    ("float16", 1, 8, 1, 2), ("float16", 5, 72, 4, 1), ("float16", 8, 128, 16, 3), ("float16", 2, 64, 32, 2),
    ("float16", 1, 256, 1024, 2), ("float32", 33, 64, 8, 2), ("mx4", 1, 32, 16, 1), ("mx4", 3, 96, 32, 3),
    ("mx4", 8, 128, 1024, 2), ("mx4", 5, 256, 16, 2), ("mx4", 33, 64, 64, 2)])
def test_every_geometry(torch, ops, kind, heads, dim, page, layers, x):
    """Head dimensions, heads and page sizes up to their limits: pieces of sequences, some twice, rows at the ends of
    pages, one layer and all of them."""
    _say(f"read {kind} {heads} x {dim} page {page} {layers} layers {x}")
    rng = np.random.default_rng(heads + dim)
    lens = [page + 3, 2 * page, 1, page]
    need = [-(-n // page) for n in lens]
    p = _pair(torch, ops, kind, layers, heads, dim, page, sum(need) + 2, 5, max(need) + 1)
    order = [3, 0, 4, 2]
    p.reserve(order, lens)
    n = sum(lens)
    k, v = ((rng.standard_normal((layers, n, heads, dim)) * 3).astype(np.float32) for _ in range(2))
    p.write(0, order, np.concatenate([[0], np.cumsum(lens)]).astype(int), k, v)
    seq, first, count = [], [], []
    for s, m in zip(order, lens):
        for a, b in ((0, m), (max(0, page - 2), m), (m - 1, m), (0, min(m, page))):
            seq.append(s)
            first.append(a if a < m else 0)
            count.append(max(0, b - first[-1]))
    pick = rng.permutation(len(seq))
    seq, first, count = ([int(a[i]) for i in pick] for a in (seq, first, count))
    start = np.concatenate([[0], np.cumsum(count)]).astype(int)
    for layer, m in ((0, layers), (layers - 1, 1)):
        got = Pair4.read(p, layer, m, seq, start, first, getattr(torch, x))
        for kind_ in range(2):
            rows = got[kind_].reshape(m, start[-1], heads, dim)
            for i, s in enumerate(seq):
                for l in range(m):
                    want = p.ref.rows(layer + l, s, first[i] + count[i])[kind_][first[i]:].astype(x)
                    assert np.array_equal(rows[l, start[i]:start[i + 1]], want)
    # the last ones
    last = [min(2, m) for m in lens]
    start = np.concatenate([[0], np.cumsum(last)]).astype(int)
    got = Pair4.read(p, 0, layers, order, start, None, getattr(torch, x))
    for kind_ in range(2):
        rows = got[kind_].reshape(layers, start[-1], heads, dim)
        for i, s in enumerate(order):
            want = p.ref.rows(0, s, lens[i])[kind_][-last[i]:].astype(x)
            assert np.array_equal(rows[0, start[i]:start[i + 1]], want)
    ops.kv_status(p.c)


@pytest.mark.parametrize("x", ["float32", "float16"])
def test_k_and_v_in_turns(torch, ops, x):
    """k and v of a row side by side, and of a layer: taken, as they share no element; half a row apart: refused."""
    rng = np.random.default_rng(9)
    p = _pair(torch, ops, "mx4", 3, 2, 32, 16, 4, 2, 2)
    p.add(rng, [1], [21])
    dtype = getattr(torch, x)
    for row_stride, layer_stride, apart in ((128, 21 * 128, 64), (64, 2 * 21 * 64, 21 * 64), (6 * 64, 128, 64)):
        both = torch.full((3 * 21 * 128,), 7.0, dtype=dtype, device="cuda")
        torch.cuda.synchronize()
        args = (p.c, 0, 3, p.ints([1]), p.ints([0, 21]), 1)
        ops.kv_read(*args, both, both[apart:], 21, row_stride=row_stride, layer_stride=layer_stride)
        torch.cuda.synchronize()
        got = both.cpu().numpy()
        for layer in range(3):
            for kind, rows in enumerate(p.ref.rows(layer, 1, 21)):
                for r in range(21):
                    at = layer * layer_stride + r * row_stride + kind * apart
                    assert np.array_equal(got[at:at + 64], rows[r].reshape(-1).astype(x))
        with pytest.raises(ops.RocmError, match="k and v overlap"):
            ops.kv_read(*args, both, both[apart - 32:], 21, row_stride=row_stride, layer_stride=layer_stride)
    ops.kv_status(p.c)
