"""Attention over a paged cache of 4 bits (mod_amd/csrc/kv_attention4.hip) on contents whose outputs are the parts of the
computation themselves (kv4_cases.py; what they see is tested in test_kv4_cases.py)."""
import numpy as np
import pytest

import kv4_cases
from oracle import kv_ref
from test_gpu_kv4 import Pair4, _masked_columns
from test_gpu_kv_cache import _attend, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(torch_dev):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from mod_amd import ops
    return ops


def _fill(c, layer, s, k, v):
    """The first tokens of sequence s, k and v [tokens, heads, D], by the oracle."""
    t = np.arange(len(k))
    page, at = c.table[s, t // c.P], t % c.P
    codes, scales = c.blocks()
    for kind, x in enumerate((k, v)):
        code, scale = kv_ref.mx4_encode(x)
        codes[layer, kind, page, :, at] = code[..., 0::2] | code[..., 1::2] << 4
        scales[layer, kind, page, :, :, at] = scale


def _upload(torch, ops, c):
    """The oracle's cache on the GPU."""
    layers, _, pages, Hk, P, _ = c.kv.shape
    p = Pair4(torch, ops, layers, Hk, c.D, P, pages, *c.table.shape)
    p.ref = c
    p.upload()
    for dev, ref in ((p.table, c.table), (p.lens, c.lens), (p.refs, c.refs)):
        dev.copy_(torch.from_numpy(ref))
    torch.cuda.synchronize()
    return p


@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("H,Hk,D,rows,x", kv4_cases.PARTS_CASES)
def test_query_parts(torch, ops, H, Hk, D, rows, x, own):
    """Every part of a query, in every dimension and head, as tails and behind a prefix."""
    _say(f"parts H{H}/{Hk} D{D} {rows} rows {x} own {own}")
    rng = np.random.default_rng(D + rows)
    c = kv4_cases.Parts(rng, D, H, Hk, rows, x, own)
    ref = kv4_cases.held(rng, [D + rows], 1, Hk, D, 16)
    _fill(ref, 0, 0, c.k, c.v)
    p = _upload(torch, ops, ref)
    for shared in (0, D, D // 2 + 5):
        got = _attend(p, torch, ops, 0, [0], [0, rows], c.q, c.scale, shared, rows).astype(np.float64)
        wrong = c.wrong(got)
        _say(f"  shared {shared}: {wrong:.2f} of the bound")
        assert np.isfinite(got).all() and wrong < 1
    ops.kv_status(p.c)


def _off(p, layer, s, rows, q, got, scale):
    """Relative error of the rows of sequence s, its last, in the 2-norm."""
    want = kv4_cases.attend(p.ref, layer, s, q, scale)
    return np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("H,Hk,D,n,rows,x", [(16, 8, 128, 600, 3, "float16"), (14, 2, 64, 900, 6, "float16"),
                                             (32, 1, 128, 320, 280, "float16"), (16, 8, 128, 600, 3, "float32"),
                                             (14, 2, 64, 900, 6, "float32"), (16, 1, 128, 200, 70, "float32")])
def test_error_of_normal_inputs(torch, ops, H, Hk, D, n, rows, x):
    """The error in the 2-norm, whose parts add up as squares. fp16: a weight's rounding and the output's, uniform within
    2^-11: 2^-11 / sqrt(3) each. fp32: a score is a running sum of exponents up to 16 (the reference is 10 below the
    largest, and follows within 5) in 5 products and 2 more roundings, 16 * 2^-24 / sqrt(3) each, of an exponent to 2; two
    parts of a weight, 2^-22. Both: a query's parts, uniform within their bound over D dimensions of keys of 1."""
    _say(f"normal H{H}/{Hk} D{D} {n} keys {x}")
    rng = np.random.default_rng(n)
    ref = kv4_cases.held(rng, [n], 1, Hk, D, 16)
    _fill(ref, 0, 0, *(rng.standard_normal((n, Hk, D)) for _ in range(2)))
    p = _upload(torch, ops, ref)
    q = rng.standard_normal((rows, H, D)).astype(x)
    scale = D ** -0.5
    most = np.abs(q.astype(np.float64)).reshape(-1, 32).max(1).max()
    parts = kv4_cases.OFF[x] * most / 3 ** 0.5 * scale * D ** 0.5
    if x == "float16":
        tol = np.sqrt(2 * (2.0 ** -11 / 3 ** 0.5) ** 2 + parts ** 2)
    else:
        tol = np.sqrt(7 * (np.log(2) * 16 * 2.0 ** -24 / 3 ** 0.5) ** 2 + 2.0 ** -44 + parts ** 2)
    off = _off(p, 0, 0, rows, q, _attend(p, torch, ops, 0, [0], [0, rows], q, scale, 0, rows), scale)
    _say(f"  {off:.2e} of {tol:.2e}")
    assert off <= tol


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ratio", [30, 300, 3000])
def test_one_large_dimension(torch, ops, D, ratio):
    """fp16 queries with one dimension much larger than the others, normal keys: the keys that it ties are told apart by
    the others. Against the roundings of the weights and of the output, which any fp16 query has, and the parts' bound:
    each of the large dimension's 31 neighbours is off by up to OFF of it, uniform, times keys of 1, in a score."""
    _say(f"one large dimension D{D} {ratio}")
    rng = np.random.default_rng(ratio)
    n, H, scale = 4096, 16, D ** -0.5
    ref = kv4_cases.held(rng, [n], 1, 1, D, 16)
    _fill(ref, 0, 0, *(rng.standard_normal((n, 1, D)) for _ in range(2)))
    p = _upload(torch, ops, ref)
    q = rng.standard_normal((4, H, D))
    q[:, :, 17] = ratio
    q = q.astype("float16")
    parts = kv4_cases.OFF["float16"] * ratio / 3 ** 0.5 * 31 ** 0.5 * scale
    sums = 8 * 2.0 ** -24 * 3 * ratio * scale / 3 ** 0.5            # (scores of up to 3 of the largest key's step)
    tol = np.sqrt(2 * (2.0 ** -11 / 3 ** 0.5) ** 2 + 2 * parts ** 2 + 2 * sums ** 2)
    off = _off(p, 0, 0, 4, q, _attend(p, torch, ops, 0, [0], [0, 4], q, scale, 0, 4), scale)
    _say(f"  {off:.2e} of {tol:.2e}")
    assert off <= tol


@pytest.mark.parametrize("H,Hk,D,page,x,shared,tail,n,window", kv4_cases.FLAT_CASES)
def test_every_key_counts(torch, ops, H, Hk, D, page, x, shared, tail, n, window):
    """Weights that are nearly the same: a tile of keys left out of any sequence, or taken twice, would show."""
    _say(f"every key H{H}/{Hk} D{D} page {page} {x} {n} x {shared} + {tail}")
    f = kv4_cases.Flat(H, Hk, D, page, x, shared, tail, n, window)
    p = _upload(torch, ops, f.c)
    want = np.zeros(f.q.shape)
    for s in f.seq:
        want[f.of(s)] = kv4_cases.attend(f.c, 0, s, f.q[f.of(s)], f.scale)
    tol = kv4_cases.flat_tolerance(x, want, f.largest)
    # (the prefix read for all of them, for none, and in part; windows longer than announced)
    for same, hint in ((shared, window), (0, window), (shared // 2, window), (shared, 1)):
        got = _attend(p, torch, ops, 0, f.seq, f.start, f.q, f.scale, same, hint).astype(np.float64)
        wrong = (np.abs(got - want) / tol).max()
        _say(f"  shared {same}, {hint} rows: {wrong:.2f} of the bound")
        assert wrong <= 1
    ops.kv_status(p.c)


@pytest.mark.parametrize("x", ["float32", "float16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("way", ["up", "down", "both"])
@pytest.mark.parametrize("H,rows", [(8, 3), (64, 150)])
def test_references_follow(torch, ops, H, rows, D, x, way):
    """Scores that climb by more than the references stay behind, fall, or do both, over runs and a prefix: values of 1
    with the signs of kv4_cases.flat, keys 0 to 6 in one dimension, 4 (fp16) or 12 (fp32) a step."""
    _say(f"references H{H} D{D} {rows} rows {x} {way}")
    rng = np.random.default_rng(D)
    n, step = 4000, 4.0 if x == "float16" else 12.0
    c = kv4_cases.held(rng, [n, n], 1, 2, D, 16, 2000)
    kv4_cases.flat(rng, c)
    level = np.arange(n) * 8 // n
    level = {"up": level, "down": 7 - level, "both": np.where(level < 4, 2 * level, 15 - 2 * level)}[way]
    for s in range(2):
        k = np.zeros((n, 2, D))
        k[:, :, 9] = kv_ref.MX4_VALUES[level][:, None]
        v = c.rows(0, s, n)[1]
        _fill(c, 0, s, k, v)
    p = _upload(torch, ops, c)
    q = np.zeros((2 * rows, H, D))
    q[:, :, 9] = np.array([1.0, -1.0, 0.5, 2.0])[np.arange(H) % 4]
    q = q.astype(x)
    want = np.concatenate([kv4_cases.attend(c, 0, s, q[rows * s:rows * (s + 1)], step) for s in range(2)])
    # scores of up to 12 steps: their sums' roundings are of exponents up to that, and 16
    largest = 12 * step
    tol = kv4_cases.flat_tolerance(x, want, largest) + 2 * 9 * 2.0 ** -24 * largest * 2
    for shared in (0, 2000, 1001):
        got = _attend(p, torch, ops, 0, [0, 1], [0, rows, 2 * rows], q, step, shared, rows).astype(np.float64)
        wrong = (np.abs(got - want) / tol).max()
        _say(f"  shared {shared}: {wrong:.2f} of the bound")
        assert wrong <= 1
    ops.kv_status(p.c)


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("x", ["float32", "float16"])
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (4, 2, 128), (16, 1, 64), (64, 1, 128), (128, 1, 64), (2, 2, 96)])
def test_one_token_picked(torch, ops, H, Hk, D, x, big):
    """Each query picks one token, whose weight is 1 and the others' 0: outputs are that token's values, of every scale
    that the cache has and every code, side by side. big: queries as large as their type holds."""
    _say(f"picked H{H}/{Hk} D{D} {x} big {big}")
    rng = np.random.default_rng(D)
    rows = 2 * D
    c = kv4_cases.held(rng, [2 * D + rows], 1, Hk, D, 16)
    codes, scales = c.blocks()
    codes[:] = rng.integers(0, 256, codes.shape)
    scales[:] = 104 + rng.permutation(scales.size).reshape(scales.shape) % 37
    v = c.rows(0, 0, 2 * D + rows)[1]
    k = np.zeros((2 * D + rows, Hk, D))
    k[np.arange(D), :, np.arange(D)] = 4.0         # 4 or -4 in a dimension of its own; the last tokens: none
    k[D + np.arange(D), :, np.arange(D)] = -4.0
    # (its keys alone: the values' scales are not what an encoder would choose)
    kept = c.kv[:, 1].copy()
    _fill(c, 0, 0, k, v)
    c.kv[:, 1] = kept
    v = c.rows(0, 0, 2 * D + rows)[1]
    p = _upload(torch, ops, c)
    which = np.stack([rng.permutation(2 * D) for _ in range(H)], 1)                  # [rows, H]
    q = np.zeros((rows, H, D))
    size = 64.0 if not big else 6e4 if x == "float16" else 1e30
    np.put_along_axis(q, (which % D)[..., None], np.where(which < D, size, -size)[..., None], 2)
    got = _attend(p, torch, ops, 0, [0], [0, rows], q.astype(x), 2.0, 0, rows).astype(np.float64)
    want = np.stack([v[which[:, h], h // (H // Hk)] for h in range(H)], 1)
    # a weight and the sum are the same number but for 2^-21; fp16: the values are its numbers
    tol = 2.0 ** -20 * np.abs(want) + (2.0 ** -11 * np.abs(want) if x == "float16" else 0)
    assert (np.abs(got - want) <= tol).all()
    ops.kv_status(p.c)


@pytest.mark.parametrize("x", ["float32", "float16"])
@pytest.mark.parametrize("H,Hk,D,rows", [(4, 2, 64, 2), (4, 2, 128, 2), (16, 1, 64, 4), (64, 1, 128, 140),
                                         (64, 1, 64, 140)])
def test_every_scale(torch, ops, H, Hk, D, rows, x):
    """Values of a whole sequence under one scale, the least to the largest that the cache has, and keys likewise, with
    queries and a factor that make ordinary scores of them: relative to that sequence's values. (fp16: an output below
    2^-14 is rounded by up to 2^-25.)"""
    _say(f"scales H{H}/{Hk} D{D} {rows} rows {x}")
    rng = np.random.default_rng(D)
    lens = [rows + 30 + int(i) for i in rng.integers(0, 40, 37)]
    c = kv4_cases.held(rng, lens, 1, Hk, D, 16)
    kv4_cases.flat(rng, c, 126)
    codes, scales = c.blocks()
    for i, n in enumerate(lens):
        pages = c.table[i, :-(-n // 16)]
        scales[0, 1, pages] = 104 + i
    p = _upload(torch, ops, c)
    seq, counts = list(range(37)), [rows] + [1 + i % 3 for i in range(36)]
    start = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    q = rng.standard_normal((int(start[-1]), H, D)).astype(x)
    scale = D ** -0.5
    most = np.abs(q).max() * 6 * 0.5 * D * scale   # a score's most
    off = kv4_cases.OFF[x] * most + (kv4_cases.PARTS[x] + 4) * 2.0 ** -24 * (most + 16 / kv4_cases.LOG2E)

    def check(got, i, want, unit):
        each = 2.0 ** -11 if x == "float16" else 2.0 ** -22
        tol = (2 * each + 4 * off) * unit + (2.0 ** -25 if x == "float16" else 0)
        assert np.isfinite(got).all() and np.abs(got - want).max() <= tol, (i, np.abs(got - want).max(), tol)
    got = _attend(p, torch, ops, 0, seq, start, q, scale, 0, rows).astype(np.float64)
    for i in seq:
        rows_ = slice(start[i], start[i + 1])
        check(got[rows_], i, kv4_cases.attend(c, 0, i, q[rows_], scale), 2.0 ** (i - 23))
    # keys: the same codes under another scale, and a factor against it
    for i in seq:
        scales[0, 0, c.table[i, :-(-lens[i] // 16)]] = 104 + i
    scales[:, 1] = 127
    p.upload()
    for i in seq:
        rows_ = slice(start[i], start[i + 1])
        factor = scale * 2.0 ** (22 - i)
        got = _attend(p, torch, ops, 0, [i], [0, counts[i]], q[rows_], factor, 0, rows).astype(np.float64)
        check(got, i, kv4_cases.attend(c, 0, i, q[rows_], factor), 1.0)
    ops.kv_status(p.c)


@pytest.mark.parametrize("D,H,rows,tokens,x", [
    (128, 32, 500, 520, "float16"), (64, 32, 500, 533, "float16"), (128, 32, 500, 490, "float32"),
    (64, 32, 500, 533, "float32"), (64, 14, 30, 100, "float32")])
def test_masked_columns(torch, ops, D, H, rows, tokens, x):
    """Enough columns for items of 32 of each type and dimension, whatever the work: NaN blocks in them and behind the end."""
    _masked_columns(torch, ops, D, H, rows, tokens, x)


@pytest.mark.parametrize("x", ["float32", "float16"])
@pytest.mark.parametrize("D,H,window", [(64, 4, 7), (128, 8, 40), (128, 64, 40), (64, 64, 40)])
def test_a_nan_anywhere(torch, ops, D, H, window, x):
    """One block of values that is NaN, in each sequence at another place: the rows that see it are NaN in its dimensions,
    and no others, whichever tile, run or prefix it lies in."""
    _say(f"NaN anywhere D{D} H{H} {window} rows {x}")
    rng = np.random.default_rng(D + H)
    n, common = 40, 90
    lens = [common + window + int(k) for k in rng.integers(0, 900, n)]
    c = kv4_cases.held(rng, lens, 1, 2, D, 16, common)
    kv4_cases.flat(rng, c)
    kv4_cases.share(c, common)
    scales = c.blocks()[1]
    # at the borders of tiles, the ends, and just before and behind what the first row sees; some in the prefix's last page
    for s, L in enumerate(lens):
        places = [L - 1, L - window, L - window + 1, L - window - 1, common, common + 5, (L - window) & -32, L & -32, L - 33,
                  common + (L - common) // 2]
        pos = max(common, min(L - 1, places[s % len(places)]))
        scales[0, 1, c.table[s, pos // 16], :, int(rng.integers(0, D // 32)), pos % 16] = 255
    p = _upload(torch, ops, c)
    seq = [int(s) for s in rng.permutation(n)]
    counts = [int(k) for k in rng.integers(1, window + 1, n)]
    start = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    q = rng.standard_normal((int(start[-1]), H, D)).astype(x)
    want = c.attention(0, seq, start, q, D ** -0.5, np.zeros(q.shape))
    fine = np.isfinite(want)
    assert 0.01 < (~fine).mean() < 0.9
    tol = kv4_cases.flat_tolerance(x, np.where(fine, want, 0), float(np.abs(q).max()) * 6 * 2.0 ** -8 * D ** 0.5)
    for shared in (0, common, 37):
        got = _attend(p, torch, ops, 0, seq, start, q, D ** -0.5, shared, window).astype(np.float64)
        assert np.array_equal(np.isfinite(got), fine)
        assert (np.abs(got - want)[fine] <= tol[fine]).all()
    ops.kv_status(p.c)
