"""What the contents of kv4_cases.py see, by the oracle and without a GPU: each mistake that they are for is outside the
bound that the tests on the GPU hold the kernels to."""
import numpy as np
import pytest

import kv4_cases
from oracle import kv_ref


@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("H,Hk,D,rows,x", kv4_cases.PARTS_CASES)
def test_a_part_less(H, Hk, D, rows, x, own):
    rng = np.random.default_rng(D + rows)
    c = kv4_cases.Parts(rng, D, H, Hk, rows, x, own)
    for a in (c.k, c.v):
        assert np.array_equal(kv_ref.mx4_decode(*kv_ref.mx4_encode(a)), a)
    parts = kv4_cases.PARTS[x]
    assert c.wrong(c.weights(kv4_cases.split(c.q, parts, c.scale))) < 1
    assert c.wrong(c.weights(kv4_cases.split(c.q, parts - 1, c.scale))) > 1.5


def test_parts_hold_what_they_say():
    """2^-18 and 2^-23 of the largest of 32 dimensions, whatever the others are."""
    rng = np.random.default_rng(3)
    q = rng.standard_normal((4000, 64)) * 2.0 ** rng.integers(-11, 3, (4000, 64))
    for x, most in kv4_cases.OFF.items():
        y = q.astype(x).astype(np.float32) * np.float32(np.float32(0.1) * np.float32(kv4_cases.LOG2E))
        off = np.abs(kv4_cases.split(q.astype(x), kv4_cases.PARTS[x], 0.1) - y).reshape(-1, 32)
        assert (off.max(1) <= most * np.abs(y).reshape(-1, 32).max(1)).all()


@pytest.mark.parametrize("H,Hk,D,page,x,shared,tail,n,window", kv4_cases.FLAT_CASES)
def test_keys_left_out_or_taken_twice(H, Hk, D, page, x, shared, tail, n, window):
    """Any whole tile of 32 keys of the longest sequence, and of the shortest: left out, or taken twice."""
    f = kv4_cases.Flat(H, Hk, D, page, x, shared, tail, n, window)
    for s in (0, int(np.argmin(f.c.lens))):
        q, L = f.q[f.of(s)][-1:], int(f.c.lens[s])
        k, v = f.c.rows(0, s, L)
        out = kv4_cases.attend(f.c, 0, s, q, f.scale)
        tol = kv4_cases.flat_tolerance(x, out, f.largest)[0]
        sc = np.einsum("hd,thd->ht", q[0].astype(np.float64), np.repeat(k, H // Hk, 1), optimize=True) * f.scale
        assert np.abs(sc).max() < f.largest
        w = np.exp(sc) / np.exp(sc).sum(1, keepdims=True)
        for a in range(0, L - 31, 32):
            part = np.einsum("ht,thd->hd", w[:, a:a + 32], np.repeat(v[a:a + 32], H // Hk, 1))
            share = w[:, a:a + 32].sum(1)[:, None]
            if L > 32:
                assert (np.abs((out[0] - part) / (1 - share) - out[0]) > 1.1 * tol).any(), a
                assert (np.abs((out[0] + part) / (1 + share) - out[0]) > 1.1 * tol).any(), a


def test_attend_is_the_oracle():
    f = kv4_cases.Flat(8, 2, 64, 16, "float32", 37, 90, 3, 5)
    for s in range(3):
        q = f.q[f.of(s)]
        want = f.c.attention(0, [s], [0, len(q)], q, f.scale, np.zeros(q.shape))
        assert np.abs(kv4_cases.attend(f.c, 0, s, q, f.scale) - want).max() < 1e-13
    for s in (1, 2):                               # the prefix is one
        assert all(np.array_equal(a[:37], b[:37]) for a, b in zip(f.c.rows(0, s, 37), f.c.rows(0, 0, 37)))
