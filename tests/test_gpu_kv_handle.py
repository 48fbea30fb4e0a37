"""The paged cache's handle on the GPU: its workspace is its own, and goes only when the device is done."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(torch_dev):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from mod_amd import ops
    return ops


def _open(torch, ops, pages=8):
    i32 = dict(dtype=torch.int32, device="cuda")
    t = (torch.zeros(1, 2, pages, 1, 4, 8, device="cuda"), torch.empty(4, 6, **i32), torch.empty(4, **i32),
         torch.empty(pages, **i32))
    c = ops.KvCache(*t)
    ops.kv_init(c)
    return c, t


def test_close_waits_for_calls_on_other_streams(torch, ops):
    i32 = dict(dtype=torch.int32, device="cuda")
    one, two = torch.tensor([1], **i32), torch.tensor([9], **i32)
    c, (kv, table, lens, refs) = _open(torch, ops)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    x = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(30):
            x = torch.mm(x, x).clamp(-1, 1)
    ops.kv_reserve(c, one, two, 1, stream=st)
    assert not st.query()
    del c
    assert st.query()
    assert table[1].tolist() == [0, 1, 2, -1, -1, -1] and int(lens[1]) == 9 and refs[:4].tolist() == [1, 1, 1, 0]


def test_workspace_is_outside_the_allocator(torch, ops):
    before = ops.pool_stats()
    c, _ = _open(torch, ops)
    assert ops.pool_stats() == before
    ops.kv_status(c)
    c.close()
    assert ops.pool_stats() == before


def test_close_while_another_stream_captures(torch, ops):
    """A handle that goes while a graph is captured leaves the capture whole."""
    c, (kv, table, lens, refs) = _open(torch, ops)
    other, _ = _open(torch, ops, 12)
    i32 = dict(dtype=torch.int32, device="cuda")
    one, three = torch.tensor([1], **i32), torch.tensor([3], **i32)
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        ops.kv_reserve(c, one, three, 1, stream=st)
        other.close()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert int(lens[1]) == 3 * (i + 1)
    ops.kv_status(c)


def test_open_while_another_stream_captures(torch, ops):
    """A handle opened while torch captures a graph on a stream of its own works, and the graph too."""
    c, (kv, table, lens, refs) = _open(torch, ops)
    i32 = dict(dtype=torch.int32, device="cuda")
    one, three = torch.tensor([1], **i32), torch.tensor([3], **i32)
    more = (torch.zeros(1, 2, 6, 1, 4, 8, device="cuda"), torch.full((4, 6), -1, **i32), torch.zeros(4, **i32),
            torch.zeros(6, **i32))
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        ops.kv_reserve(c, one, three, 1, stream=st)
        other = ops.KvCache(*more)
    for i in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert int(lens[1]) == 3 * (i + 1)
    ops.kv_reserve(other, one, three, 1)
    ops.kv_status(other)
    assert more[2].tolist() == [0, 3, 0, 0]
    ops.kv_status(c)


def test_open_in_the_captured_stream_is_refused(torch, ops):
    """The workspace is cleared by work that is waited for, which the library's own capture cannot record."""
    from mod_amd import backend
    c, t = _open(torch, ops)
    graph = backend.HIPGraph()
    torch.cuda.synchronize()
    graph.capture_begin()
    ops.kv_fork(c, t[2], t[2], 0)
    with pytest.raises(ops.RocmError, match="capturing"):
        ops.KvCache(*t)
    graph.capture_end()
    ops.kv_status(c)
