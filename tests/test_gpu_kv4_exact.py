"""Attention over a paged cache of 4 bits (mod_amd/csrc/kv_attention4.hip) on contents whose outputs are the parts of the
computation themselves (kv4_cases.py; what they see is tested in test_kv4_cases.py)."""
import numpy as np
import pytest

import kv4_cases
from oracle import kv_ref
from test_gpu_kv4 import Pair4
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


def _fill(p, layer, s, k, v):
    """The first tokens of sequence s, k and v [tokens, heads, D], by the oracle."""
    t = np.arange(len(k))
    page, at = p.ref.table[s, t // p.ref.P], t % p.ref.P
    codes, scales = p.ref.blocks()
    for kind, x in enumerate((k, v)):
        code, scale = kv_ref.mx4_encode(x)
        codes[layer, kind, page, :, at] = code[..., 0::2] | code[..., 1::2] << 4
        scales[layer, kind, page, :, :, at] = scale


def _sequences(torch, ops, rng, lens, layers, Hk, D, page, common=0):
    """Sequences of the given lengths, in pages in any order; the first `common` tokens' pages are the same."""
    need = [-(-n // page) for n in lens]
    same = common // page
    pages = same + sum(n - same for n in need) + 3
    p = Pair4(torch, ops, layers, Hk, D, page, pages, len(lens), max(need) + 1)
    free = [int(i) for i in rng.permutation(pages)]
    first = [free.pop() for _ in range(same)]
    for s, (n, k) in enumerate(zip(lens, need)):
        p.ref.table[s, :k] = first + [free.pop() for _ in range(k - same)]
        p.ref.lens[s] = n
    np.add.at(p.ref.refs, p.ref.table[p.ref.table >= 0], 1)
    for dev, ref in ((p.table, p.ref.table), (p.lens, p.ref.lens), (p.refs, p.ref.refs)):
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
    p = _sequences(torch, ops, rng, [D + rows], 1, Hk, D, 16)
    _fill(p, 0, 0, c.k, c.v)
    p.upload()
    for shared in (0, D, D // 2 + 5):
        got = _attend(p, torch, ops, 0, [0], [0, rows], c.q, c.scale, shared, rows).astype(np.float64)
        wrong = c.wrong(got)
        _say(f"  shared {shared}: {wrong:.2f} of the bound")
        assert np.isfinite(got).all() and wrong < 1
    ops.kv_status(p.c)


def _off(p, layer, s, rows, q, got, scale):
    """Relative error of the rows of sequence s, its last, in the 2-norm."""
    want = p.ref.attention(layer, [s], [0, rows], q, scale, np.zeros(q.shape))
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
    p = _sequences(torch, ops, rng, [n], 1, Hk, D, 16)
    _fill(p, 0, 0, *(rng.standard_normal((n, Hk, D)) for _ in range(2)))
    p.upload()
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
    p = _sequences(torch, ops, rng, [n], 1, 1, D, 16)
    _fill(p, 0, 0, *(rng.standard_normal((n, 1, D)) for _ in range(2)))
    p.upload()
    q = rng.standard_normal((4, H, D))
    q[:, :, 17] = ratio
    q = q.astype("float16")
    parts = kv4_cases.OFF["float16"] * ratio / 3 ** 0.5 * 31 ** 0.5 * scale
    sums = 8 * 2.0 ** -24 * 3 * ratio * scale / 3 ** 0.5            # (scores of up to 3 of the largest key's step)
    tol = np.sqrt(2 * (2.0 ** -11 / 3 ** 0.5) ** 2 + 2 * parts ** 2 + 2 * sums ** 2)
    off = _off(p, 0, 0, 4, q, _attend(p, torch, ops, 0, [0], [0, 4], q, scale, 0, 4), scale)
    _say(f"  {off:.2e} of {tol:.2e}")
    assert off <= tol
