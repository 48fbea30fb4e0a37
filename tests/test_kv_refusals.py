"""CPU-only checks that the paged cache's and the verification's entry points
refuse what they cannot serve before any HIP call (a non-null stream value keeps
the library from creating its own; it is never used)."""
import ctypes

import pytest

STREAM = 1


def _cache(**change):
    from mod_amd import ops
    f = dict(kv=4096, table=4096, lens=4096, refs=4096, work=4096, kv_dtype=ops.F16, n_layers=2, n_kv_heads=4,
             head_dim=64, page_size=16, n_pages=10, max_seqs=3, max_pages=5)
    f.update(change)
    return ops.CKvCache(**f)


BAD_CACHES = [
    (dict(kv=None), "null pointer"), (dict(table=None), "null pointer"), (dict(lens=None), "null pointer"),
    (dict(refs=None), "null pointer"), (dict(work=None), "null pointer"), (dict(kv_dtype=2), "dtype"),
    (dict(n_layers=0), "empty"), (dict(n_kv_heads=-1), "empty"), (dict(n_pages=0), "empty"), (dict(max_seqs=0), "empty"),
    (dict(max_pages=0), "empty"), (dict(head_dim=4), "head_dim"), (dict(head_dim=68), "head_dim"),
    (dict(head_dim=264), "head_dim"), (dict(page_size=0), "page_size"), (dict(page_size=24), "page_size"),
    (dict(page_size=2048), "page_size"), (dict(kv=4104), "16-byte"), (dict(table=4098), "4-byte"),
    (dict(refs=4097), "4-byte"), (dict(n_pages=(1 << 20) + 1), "2\\^20"), (dict(max_pages=(1 << 20) + 1), "2\\^20"),
    (dict(max_pages=1 << 20, page_size=1024), "2\\^28"), (dict(max_seqs=1 << 21), "2\\^20"),
    (dict(n_kv_heads=1 << 18), "n_kv_heads"),
]


@pytest.mark.parametrize("change,error", BAD_CACHES)
def test_caches(change, error):
    from mod_amd import ops
    c = ctypes.byref(_cache(**change))
    lib = ops.lib
    for rc in (lambda: lib.pio_kv_init(c, STREAM), lambda: lib.pio_kv_status(c, STREAM),
               lambda: lib.pio_kv_reserve(c, 64, 64, 1, STREAM), lambda: lib.pio_kv_fork(c, 64, 64, 1, STREAM),
               lambda: lib.pio_kv_drop(c, 64, 64, 1, STREAM), lambda: lib.pio_kv_compact(c, STREAM),
               lambda: lib.pio_kv_write(c, 0, 1, 64, 64, 1, 64, 64, 0, 1, 0, 0, STREAM),
               lambda: lib.pio_kv_attention(c, 0, 64, 64, 1, 0, 64, 64, 0, 1, 4, 0, 0, 1, 1.0, STREAM)):
        assert rc() == ops.ERR_INVALID
        import re
        assert re.search(error, ops.last_error()), ops.last_error()


def test_null_cache():
    from mod_amd import ops
    assert ops.lib.pio_kv_work_bytes(None) == 0
    assert ops.lib.pio_kv_init(None, STREAM) == ops.ERR_INVALID and "null" in ops.last_error()
    assert ops.lib.pio_kv_work_bytes(ctypes.byref(_cache())) >= 4 * (2 + 3 + 40)


def test_requests():
    from mod_amd import ops
    c, lib = ctypes.byref(_cache()), ops.lib
    for fn in (lib.pio_kv_reserve, lib.pio_kv_fork):
        assert fn(c, 64, 64, -1, STREAM) == ops.ERR_INVALID
        assert fn(c, 64, 64, 4, STREAM) == ops.ERR_INVALID and "requests" in ops.last_error()
        assert fn(c, None, 64, 1, STREAM) == ops.ERR_INVALID and "null" in ops.last_error()
        assert fn(c, 64, None, 1, STREAM) == ops.ERR_INVALID
        assert fn(c, 66, 64, 1, STREAM) == ops.ERR_INVALID and "4-byte" in ops.last_error()
        assert fn(c, None, None, 0, STREAM) == ops.OK
    assert lib.pio_kv_drop(c, None, None, 1, STREAM) == ops.ERR_INVALID
    assert lib.pio_kv_drop(c, 64, 65, 1, STREAM) == ops.ERR_INVALID
    big = ctypes.byref(_cache(max_seqs=9000))
    assert lib.pio_kv_reserve(big, 64, 64, 4097, STREAM) == ops.ERR_INVALID


@pytest.mark.parametrize("change,error", [
    (dict(layer=2), "layers"), (dict(layer=-1), "layers"), (dict(layers=3), "layers"), (dict(layers=-1), "layers"),
    (dict(dtype=2), "dtype"), (dict(rows=-1), "rows"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(k=72), "16-byte"), (dict(row_stride=100), "strides"), (dict(row_stride=248), "strides"),
    (dict(layer_stride=-8), "strides"), (dict(layer_stride=4), "strides"), (dict(start=None), "null")])
def test_write(change, error):
    from mod_amd import ops
    f = dict(layer=0, layers=1, seq=64, start=64, n=1, k=64, v=64, dtype=0, rows=4, row_stride=0, layer_stride=0)
    f.update(change)
    assert ops.lib.pio_kv_write(ctypes.byref(_cache()), *f.values(), STREAM) == ops.ERR_INVALID
    assert error in ops.last_error()


@pytest.mark.parametrize("change,error", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(dtype=3), "dtype"), (dict(n=-1), "requests"),
    (dict(rows=-1), "rows"), (dict(shared=-1), "shared"), (dict(shared=81), "shared"), (dict(heads=0), "heads"),
    (dict(heads=6), "heads"), (dict(max_rows=0), "max_rows"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(seq=None), "null"), (dict(start=None), "null"), (dict(q=72), "16-byte"), (dict(out=8), "16-byte"),
    (dict(seq=66), "4-byte"), (dict(q_stride=500), "strides"), (dict(out_stride=504), "strides"),
    (dict(rows=1 << 29), "too many rows"), (dict(rows=1 << 23), "too many rows"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(out_stride=520), "another stride")])
def test_attention(change, error):
    from mod_amd import ops
    f = dict(layer=0, seq=64, start=64, n=1, shared=0, q=64, out=64, dtype=0, rows=4, heads=8, q_stride=0, out_stride=0,
             max_rows=1, scale=1.0)
    f.update(change)
    assert ops.lib.pio_kv_attention(ctypes.byref(_cache()), *f.values(), STREAM) == ops.ERR_INVALID
    assert error in ops.last_error()


@pytest.mark.parametrize("change,error", [
    (dict(dtype=2), "dtype"), (dict(n=-1), "requests"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=(1 << 30) + 1), "vocabulary"),
    (dict(target=None), "null"), (dict(ids=None), "null"), (dict(u=None), "null"), (dict(u_next=None), "null"),
    (dict(start=None), "null"), (dict(accepted=None), "null"), (dict(tokens=None), "null"),
    (dict(target_stride=99), "strides"), (dict(draft_stride=99), "strides"), (dict(target=66), "unaligned"),
    (dict(draft=65), "unaligned"), (dict(ids=66), "4-byte"), (dict(rejected=66), "4-byte")])
def test_verify(change, error):
    from mod_amd import ops
    f = dict(target=64, target_stride=0, draft=64, draft_stride=0, dtype=0, ids=64, u=64, u_next=64, start=64, n=1,
             rows=4, vocab=100, accepted=64, tokens=64, rejected=64)
    f.update(change)
    assert ops.lib.pio_verify_draft(*f.values(), STREAM) == ops.ERR_INVALID
    assert error in ops.last_error()


def test_python_layer():
    """KvCache takes dense int32 tables of one device on a GPU."""
    import torch
    from mod_amd import ops
    kv = torch.zeros(1, 2, 4, 1, 16, 8)
    i = dict(dtype=torch.int32)
    ok = [torch.zeros(2, 3, **i), torch.zeros(2, **i), torch.zeros(4, **i)]
    for change, error in [((kv[0], *ok), "shape"), ((kv, ok[1], *ok[1:]), "table"), ((kv, ok[0].float(), *ok[1:]), "int32"),
                          ((kv, ok[0], ok[2], ok[2]), "lens"), ((kv, ok[0], ok[1], ok[1]), "refs"),
                          ((kv.transpose(4, 5), *ok), "dense"), ((kv, *ok), "not on a GPU")]:
        with pytest.raises((ValueError, TypeError), match=error):
            ops.KvCache(*change)
    with pytest.raises(TypeError, match="dtype"):
        ops.kv_attention(None, 0, 64, 64, 1, torch.zeros(8), torch.zeros(8).half(), 1, 8, 1.0)
    with pytest.raises(TypeError, match="dtype"):
        ops.verify_draft(torch.zeros(8), torch.zeros(8).half(), 64, 64, 64, 64, 1, 1, 8, 64, 64)
