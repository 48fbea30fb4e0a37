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
