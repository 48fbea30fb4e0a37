"""pio_kv_read's refusal of k and v that share elements, on the host, without a GPU."""
import ctypes
import itertools

import numpy as np
import pytest

from test_oracle_kv4 import STREAM, _cache


def _read(ops, k, v, dtype, rows, layers, row_stride, layer_stride):
    return ops.lib.pio_kv_read(ctypes.byref(_cache(n_layers=layers, n_kv_heads=1, head_dim=32)), 0, layers, 64, 64, None, 1,
                               k, v, dtype, rows, row_stride, layer_stride, STREAM)


def _meets(d, width, rows, row_stride, layers, layer_stride):
    at = [r * row_stride + l * layer_stride for r in range(rows) for l in range(layers)]
    return any(abs(d + b - a) < width for a in at for b in at)


CASES = [(rows, layers, rs, ls) for rows, layers in ((1, 1), (3, 1), (1, 3), (3, 2), (4, 3))
         for rs, ls in ((32, 0), (64, 0), (72, 0), (128, 32), (384, 64), (32, 400), (104, 40))
         if ls == 0 or layers == 1 or (ls >= 32 and ((ls - 32) // rs >= rows - 1 or (rs - 32) // ls >= layers - 1))]


@pytest.mark.parametrize("rows,layers,row_stride,layer_stride", CASES)
def test_k_and_v_that_overlap(rows, layers, row_stride, layer_stride):
    """Every distance of 8 elements, either way round, against all pairs of rows: refused where two share one."""
    from mod_amd import ops
    ls = layer_stride or rows * row_stride
    span = (rows - 1) * row_stride + (layers - 1) * ls + 64
    k = 1 << 20
    refused = 0
    for d in itertools.chain(range(8, span, 8), range(-span // 8 * 8, 0, 8)):
        if _meets(d, 32, rows, row_stride, layers, ls):
            assert _read(ops, k, k + 4 * d, 0, rows, layers, row_stride, layer_stride) == ops.ERR_INVALID, d
            assert "k and v overlap" in ops.last_error()
            refused += 1
    assert refused


def test_rule_by_itself():
    """The same rule in Python, against all pairs: what is taken (k and v in turns among it) cannot be called here without
    a device."""
    rng = np.random.default_rng(1)

    def rule(d, width, rows, rs, layers, ls):
        if layers == 1:
            ls = 1 << 60
        (s1, n1), (s2, n2) = ((rs, rows), (ls, layers)) if rs <= ls else ((ls, layers), (rs, rows))
        d = abs(d)
        for k2, k1 in itertools.product(range(2), range(2)):
            off = abs(d - min(d // s2 + k2, n2 - 1) * s2)
            if abs(off - min(off // s1 + k1, n1 - 1) * s1) < width:
                return True
        return False
    taken = 0
    for rows, layers, rs, ls in CASES:
        ls = ls or rows * rs
        for d in 8 * rng.integers(-200, 200, 300):
            if d:
                meets = _meets(int(d), 32, rows, rs, layers, ls)
                assert rule(int(d), 32, rows, rs, layers, ls) == meets
                taken += not meets
    assert taken > 1000
