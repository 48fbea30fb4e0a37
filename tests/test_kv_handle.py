"""The paged cache's handle and the Python layer's own checks, without a GPU: a
library that notes its calls stands in for the built one."""
import pytest
import torch


class FakeLib:
    """Notes the calls of the library, and answers `status` to pio_kv_work_create."""

    def __init__(self, status=0):
        self.calls, self.status = [], status

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name,) + args)
            return {"pio_kv_work_create": self.status, "tensor_last_error": b"none"}.get(name, 0)
        return call


class FakeTensor:
    """A dense tensor on a second GPU."""
    device = "cuda:1"

    def __init__(self, shape, dtype):
        self.shape, self.dtype = shape, dtype

    def data_ptr(self):
        return 4096


def _tensors():
    return (FakeTensor((1, 2, 4, 1, 16, 8), "float16"), FakeTensor((2, 3), "int32"), FakeTensor((2,), "int32"),
            FakeTensor((4,), "int32"))


def test_workspace_is_the_handles_own(monkeypatch):
    """The workspace that calls on any stream use comes from and goes back through the pair that waits for
    the device, once, and never through the allocator's free lists, which order one stream only."""
    from mod_amd import ops
    lib = FakeLib()
    monkeypatch.setattr(ops, "lib", lib)
    c = ops.KvCache(*_tensors())
    ref = c.ref
    assert [x[0] for x in lib.calls] == ["pio_kv_work_create"] and lib.calls[0][1:] == (ref, 1)
    c.close()
    assert lib.calls[1:] == [("pio_kv_work_destroy", ref, 1)] and c.ref is None
    c.close()
    del c
    assert len(lib.calls) == 2
    c = ops.KvCache(*_tensors())
    del c
    assert [x[0] for x in lib.calls[2:]] == ["pio_kv_work_create", "pio_kv_work_destroy"]


def test_no_memory_for_the_workspace(monkeypatch):
    from mod_amd import ops
    monkeypatch.setattr(ops, "lib", FakeLib(ops.ERR_OOM))
    with pytest.raises(ops.RocmError):
        ops.KvCache(*_tensors())


def test_workspace_refusals():
    """Before any HIP call."""
    import ctypes
    from mod_amd import ops
    assert ops.lib.pio_kv_work_create(None, 0) == ops.ERR_INVALID and "null" in ops.last_error()
    c = ops.CKvCache(n_pages=0, max_seqs=3)
    assert ops.lib.pio_kv_work_create(ctypes.byref(c), 0) == ops.ERR_INVALID and "empty" in ops.last_error()
    c = ops.CKvCache(n_pages=4, max_seqs=3)
    assert ops.lib.pio_kv_work_create(ctypes.byref(c), -1) == ops.ERR_INVALID and "device" in ops.last_error()
    ops.lib.pio_kv_work_destroy(None, 0)
    ops.lib.pio_kv_work_destroy(ctypes.byref(c), 0)


def test_lists_and_types():
    """What the library reads as int32 or fp32 is that type, and k and v are of one."""
    from mod_amd import ops
    i, wrong = torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    f, half = torch.zeros(8), torch.zeros(8).half()

    class Cache:
        ref = None
    c = Cache()
    for bad in (lambda: ops.kv_reserve(c, wrong, i, 1), lambda: ops.kv_reserve(c, i, wrong, 1),
                lambda: ops.kv_fork(c, wrong, i, 1), lambda: ops.kv_fork(c, i, wrong, 1),
                lambda: ops.kv_drop(c, wrong, None, 1), lambda: ops.kv_drop(c, i, wrong, 1),
                lambda: ops.kv_write(c, 0, 1, wrong, i, 1, f, f, 1), lambda: ops.kv_write(c, 0, 1, i, wrong, 1, f, f, 1),
                lambda: ops.kv_write(c, 0, 1, i, i, 1, f, half, 1),
                lambda: ops.kv_attention(c, 0, wrong, i, 1, f, f, 1, 8, 1.0),
                lambda: ops.kv_attention(c, 0, i, wrong, 1, f, f, 1, 8, 1.0),
                lambda: ops.verify_draft(f, None, wrong, f, f, i, 1, 1, 8, i, i),
                lambda: ops.verify_draft(f, None, i, half, f, i, 1, 1, 8, i, i),
                lambda: ops.verify_draft(f, None, i, f, half, i, 1, 1, 8, i, i),
                lambda: ops.verify_draft(f, None, i, f, f, wrong, 1, 1, 8, i, i),
                lambda: ops.verify_draft(f, None, i, f, f, i, 1, 1, 8, wrong, i),
                lambda: ops.verify_draft(f, None, i, f, f, i, 1, 1, 8, i, wrong),
                lambda: ops.verify_draft(f, None, i, f, f, i, 1, 1, 8, i, i, wrong)):
        with pytest.raises(TypeError, match="must be|differ"):
            bad()
