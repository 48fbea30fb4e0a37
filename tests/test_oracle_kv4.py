"""The oracle's cache of 4 bits (oracle/kv_ref.py) against closed forms, and the
host's checks of such a cache, without a GPU."""
import ctypes

import numpy as np
import pytest

from oracle import kv_ref


def test_every_value_comes_back():
    """Each code under each scale is its own nearest, where the block's largest fixes the scale."""
    grid = np.concatenate([kv_ref.MX4_VALUES, -kv_ref.MX4_VALUES])
    for e in range(-23, 14):
        x = np.concatenate([grid, grid]) * 2.0 ** e
        code, scale = kv_ref.mx4_encode(x)
        assert scale == [e + 127] and np.array_equal(kv_ref.mx4_decode(code, scale), x)
        assert np.array_equal(x.astype(np.float16).astype(np.float64), x)     # fp16 numbers, all of them


def test_half_a_step_and_ties():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((400, 32)) * 2.0 ** rng.integers(-14, 12, (400, 1))
    code, scale = kv_ref.mx4_encode(x)
    unit = 2.0 ** (scale.astype(np.float64) - 127)
    y, back = np.abs(x) / unit, np.abs(kv_ref.mx4_decode(code, scale)) / unit
    assert y.max() < 7 and (y.max(1) >= 3.5).all()
    step = np.where(back < 2, 0.5, np.where(back < 4, 1.0, 2.0))
    assert (np.abs(y - back) <= step / 2).all()
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] + [0.0] * 24)
    code, scale = kv_ref.mx4_encode(-ties)
    assert scale == [127] and kv_ref.mx4_decode(code, scale)[:8].tolist() == [-0.0, -1, -1, -2, -2, -4, -4, -6]


@pytest.mark.parametrize("most,byte,value", [
    (0.0, 104, 0.0), (2.0 ** -24, 104, 2.0 ** -24), (2.0 ** -25, 104, 0.0), (6.999, 127, 6.0), (7.0, 128, 8.0),
    (7 * 2.0 ** 13, 140, 6 * 2.0 ** 13), (3e38, 140, 6 * 2.0 ** 13), (np.inf, 255, np.nan), (np.nan, 255, np.nan)])
def test_scales(most, byte, value):
    x = np.zeros(64)
    x[40] = -most
    code, scale = kv_ref.mx4_encode(x)
    assert scale.tolist() == [104, byte]
    got = kv_ref.mx4_decode(code, scale)
    assert np.array_equal(got[40], -value, equal_nan=True) and np.all(got[:32] == 0)


def test_cache_holds_what_was_written():
    rng = np.random.default_rng(2)
    c = kv_ref.Cache4(2, 3, 64, 16, 9, 4, 5)
    c.reserve([2, 0], [19, 5])
    k, v = rng.standard_normal((2, 24, 3, 64)), rng.standard_normal((2, 24, 3, 64))
    c.write(0, [2, 0], [0, 19, 24], k, v)
    for s, a, n in ((2, 0, 19), (0, 19, 5)):
        for layer in range(2):
            for got, x in zip(c.rows(layer, s, n), (k, v)):
                assert np.array_equal(got, kv_ref.mx4_decode(*kv_ref.mx4_encode(x[layer, a:a + n])))
    c.fork([2], [3])
    c.reserve([3], [1])                                # a copy of the last page
    assert np.array_equal(c.rows(1, 3, 19)[0], c.rows(1, 2, 19)[0]) and c.table[3, 1] != c.table[2, 1]


# ------------------------------------------------------------- refusals ------
STREAM = None


def _cache(**change):
    from mod_amd import ops
    f = dict(kv=4096, table=4096, lens=4096, refs=4096, work=4096, kv_dtype=ops.MX4, n_layers=2, n_kv_heads=4,
             head_dim=128, page_size=16, n_pages=8, max_seqs=3, max_pages=4)
    f.update(change)
    return ops.CKvCache(**f)


@pytest.mark.parametrize("change,error", [
    (dict(head_dim=72), "head_dim"), (dict(head_dim=16), "head_dim"), (dict(head_dim=288), "head_dim"),
    (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"), (dict(kv_dtype=5), "dtype"),
    (dict(kv=4104), "aligned")])
def test_cache_refusals(change, error):
    from mod_amd import ops
    for call in (lambda c: ops.lib.pio_kv_init(c, STREAM), lambda c: ops.lib.pio_kv_compact(c, STREAM),
                 lambda c: ops.lib.pio_kv_write(c, 0, 1, 64, 64, 1, 64, 64, 0, 4, 0, 0, STREAM),
                 lambda c: ops.lib.pio_kv_read(c, 0, 1, 64, 64, None, 1, 64, 128, 0, 4, 0, 0, STREAM),
                 lambda c: ops.lib.pio_kv_attention(c, 0, 64, 64, 1, 0, 64, 64, 0, 4, 8, 0, 0, 1, 1.0, STREAM)):
        assert call(ctypes.byref(_cache(**change))) == ops.ERR_INVALID
        assert error in ops.last_error()


@pytest.mark.parametrize("change,error", [
    (dict(n=-1), "requests"), (dict(n=4097), "requests"), (dict(seq=None), "null request"), (dict(start=None), "null request"),
    (dict(seq=66), "4-byte"), (dict(start=66), "4-byte"), (dict(first=66), "4-byte"), (dict(layer=2), "layers"),
    (dict(layer=1, layers=2), "layers"), (dict(layers=-1), "layers"), (dict(layer=-1), "layers"), (dict(dtype=2), "dtype"),
    (dict(dtype=4), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 24), "rows"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(v=64), "same"), (dict(k=72), "aligned"), (dict(v=72), "aligned"),
    (dict(row_stride=500), "strides"), (dict(row_stride=516), "strides"), (dict(layer_stride=-8), "strides"),
    (dict(layer_stride=512), "overlap"), (dict(layer_stride=4 * 512 - 8), "overlap"),
    (dict(rows=1, layer_stride=504), "overlap"), (dict(row_stride=1016, layer_stride=512), "overlap"),
    (dict(rows=1, layer_stride=0, row_stride=504), "strides")])
@pytest.mark.parametrize("kind", [0, 1, 4])
def test_read_refusals(change, error, kind):
    from mod_amd import ops
    f = dict(layer=0, layers=2, seq=64, start=64, first=64, n=1, k=64, v=128, dtype=0, rows=4, row_stride=0,
             layer_stride=0)
    f.update(change)
    assert ops.lib.pio_kv_read(ctypes.byref(_cache(kv_dtype=kind)), *f.values(), STREAM) == ops.ERR_INVALID
    assert error in ops.last_error()


def test_read_of_nothing():
    """Returns before the lists or the stream are looked at."""
    from mod_amd import ops
    for change in (dict(n=0, seq=None, start=None, k=None), dict(rows=0, v=None), dict(layers=0)):
        f = dict(layer=0, layers=2, seq=64, start=64, first=None, n=1, k=64, v=128, dtype=0, rows=4, row_stride=0,
                 layer_stride=0)
        f.update(change)
        assert ops.lib.pio_kv_read(ctypes.byref(_cache()), *f.values(), STREAM) == ops.OK


def test_python_layer(monkeypatch):
    """uint8 with a last dimension of 17 / 32 is a cache of 4 bits; lists and types are looked at."""
    import torch
    from mod_amd import ops

    class Lib:
        def __getattr__(self, name):
            return lambda *args: 0

    class Fake:
        device = "cuda:0"

        def __init__(self, shape, dtype):
            self.shape, self.dtype = shape, dtype

        def data_ptr(self):
            return 4096
    monkeypatch.setattr(ops, "lib", Lib())
    rest = Fake((2, 3), "int32"), Fake((2,), "int32"), Fake((4,), "int32")
    c = ops.KvCache(Fake((1, 2, 4, 1, 16, 68), torch.uint8), *rest)
    assert (c.c.kv_dtype, c.c.head_dim, c.c.page_size) == (ops.MX4, 128, 16)
    with pytest.raises(ValueError, match="17"):
        ops.KvCache(Fake((1, 2, 4, 1, 16, 64), torch.uint8), *rest)
    f, i = torch.zeros(8), torch.zeros(4, dtype=torch.int32)
    for bad in (lambda: ops.kv_read(c, 0, 1, i.long(), i, 1, f, f, 1), lambda: ops.kv_read(c, 0, 1, i, i.long(), 1, f, f, 1),
                lambda: ops.kv_read(c, 0, 1, i, i, 1, f, f, 1, first=i.long()),
                lambda: ops.kv_read(c, 0, 1, i, i, 1, f, f.half(), 1)):
        with pytest.raises(TypeError, match="must be|differ"):
            bad()
    with pytest.raises(TypeError, match="dtype"):
        ops.kv_read(c, 0, 1, i, i, 1, f.to(torch.uint8), f.to(torch.uint8), 1)
