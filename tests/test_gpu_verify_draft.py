"""Verification of drafted tokens on the GPU (mod_amd/csrc/verify_draft.hip)
against oracle/kv_ref.py:verify. Results are whole numbers and have to be equal:
both sides compare and sum in 64 bits, and a difference in the order of the sums
(2^-53 of the total) reaches a boundary between two tokens in fewer than one of
10^8 of the draws here."""
import numpy as np
import pytest

from oracle import kv_ref

pytestmark = pytest.mark.gpu


def _say(m):
    print(m, flush=True)


@pytest.fixture(scope="module")
def torch(torch_dev):
    import torch
    return torch


@pytest.fixture(scope="module")
def ops(torch_dev):
    from mod_amd import ops
    return ops


def _probs(rng, rows, vocab, dtype, sharp=3.0):
    x = rng.standard_normal((rows, vocab)) * sharp
    x = np.exp(x - x.max(1, keepdims=True))
    return (x / x.sum(1, keepdims=True)).astype(dtype)


def _run(torch, ops, target, draft, ids, u, u_next, start, pad=0, rejected=True):
    n, rows, vocab = len(start) - 1, len(target), target.shape[1]

    def dev(a, wide=0):
        a = np.ascontiguousarray(a)
        if wide:
            b = np.full((a.shape[0], a.shape[1] + wide), np.nan, a.dtype)
            b[:, :a.shape[1]] = a
            a = b
        return torch.from_numpy(a).cuda()

    i32 = np.int32
    t, d = dev(target, pad), None if draft is None else dev(draft, 2 * pad)
    acc, rej = (torch.full((n + 1,), 7, dtype=torch.int32, device="cuda") for _ in range(2))
    tok = torch.full((rows + 2,), 7, dtype=torch.int32, device="cuda")
    args = [dev(np.asarray(ids, i32)), dev(np.asarray(u, np.float32)), dev(np.asarray(u_next, np.float32)),
            dev(np.asarray(start, i32))]
    torch.cuda.synchronize()
    ops.verify_draft(t, d, *args, n, rows, vocab, acc, tok, rejected=rej if rejected else None,
                     target_stride=vocab + pad if pad else 0, draft_stride=vocab + 2 * pad if pad else 0)
    torch.cuda.synchronize()
    assert int(acc[n]) == 7 and torch.all(tok[rows:] == 7) and int(rej[n]) == 7
    return acc[:n].cpu().numpy(), tok[:rows].cpu().numpy(), rej[:n].cpu().numpy()


def _check(torch, ops, target, draft, ids, u, u_next, start, **kw):
    got = _run(torch, ops, target, draft, ids, u, u_next, start, **kw)
    ref = kv_ref.verify(target, draft, ids, np.asarray(u, np.float32), np.asarray(u_next, np.float32), start)
    last = int(start[-1])
    for name, a, b in zip(("accepted", "tokens", "rejected"), got, ref):
        if name == "tokens":
            a, b = a[:last], b[:last]
        if name == "rejected" and not kw.get("rejected", True):
            continue
        assert np.array_equal(a, b), (name, a, b)
    return got


@pytest.mark.parametrize("vocab", [1, 2, 63, 257, 1000, 4099, 32003, 151936])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("certain", [False, True])
def test_against_oracle(torch, ops, vocab, dtype, certain):
    _say(f"verify vocab {vocab} {dtype.__name__} certain {certain}")
    rng = np.random.default_rng(vocab)
    n = 5 if vocab > 50000 else 40
    counts = rng.integers(0, 10, n)                 # rows of a request: drafted tokens and one more, or none
    counts[0] = 1
    start = np.concatenate([[0], np.cumsum(counts)])
    rows = int(start[-1]) + 1
    logits = rng.standard_normal((rows, vocab)) * 2
    target = np.exp(logits) / np.exp(logits).sum(1, keepdims=True)
    draft = np.exp(logits + rng.standard_normal((rows, vocab)) * 0.5)
    draft /= draft.sum(1, keepdims=True)
    ids = np.array([rng.choice(vocab, p=d) for d in draft])
    if certain:
        ids = np.where(rng.random(rows) < 0.6, target.argmax(1), ids)
    for pad in (0, 3):
        got = _check(torch, ops, target.astype(dtype), None if certain else draft.astype(dtype), ids, rng.random(rows),
                     rng.random(n), start, pad=pad)
    if vocab > 100 and not certain and n > 10:
        assert got[0].min() == 0 and got[0].max() > 1


def test_edges(torch, ops):
    """Random numbers at their ends, rows without weight, NaN and inf, ids that the vocabulary does not have."""
    rng = np.random.default_rng(1)
    V = 700
    p, q = _probs(rng, 12, V, np.float32), _probs(rng, 12, V, np.float32)
    start = [0, 2, 4, 6, 8, 10, 12]
    ids = rng.integers(0, V, 12)
    for un in (0.0, np.float32(1) - np.float32(2.0 ** -24), 1.0):
        for u in (0.0, 1.0):
            _say(f"u {u} u_next {un}")
            _check(torch, ops, p, q, ids, np.full(12, u), np.full(6, un), start)
    # all of the weight in one place: the first, the last, one in the middle; and none
    one = np.zeros((12, V), np.float32)
    for i, at in enumerate((0, V - 1, 255, 256, 400)):
        one[2 * i:2 * i + 2, at] = 1.0
    for un in (0.0, 0.5, 1.0):
        got = _check(torch, ops, one, q, ids, np.ones(12), np.full(6, un), start)
        assert list(got[1][::2][:5]) == [0, V - 1, 255, 256, 400] and got[1][10] == -1
    # target and draft alike, and a refusal all the same: drawn from the target itself
    got = _check(torch, ops, p, p, ids, np.ones(12), rng.random(6), start)
    assert np.all(got[0] == 0) and np.all(got[1][::2] >= 0)
    # an id outside the vocabulary is not accepted, whatever the random number
    bad = np.array([-1, 0, V, 0, 1 << 30, 0, -(1 << 30), 0, 5, 0, 6, 0])
    for draft in (q, None):
        got = _check(torch, ops, p, draft, bad, np.zeros(12), rng.random(6), start)
        assert np.all(got[0][:4] == 0) and np.all(got[0][4:] == 1)
    # weights that are no numbers count as 0
    odd = p.copy()
    odd[:, ::7] = np.nan
    odd[:, 3::11] = np.inf
    odd[:, 5::13] = -np.inf
    oddq = q.copy()
    oddq[:, 1::5] = np.nan
    oddq[:, 2::17] = -np.inf
    for draft in (oddq, None):
        _check(torch, ops, odd, draft, ids, rng.random(12), rng.random(6), start)
    _check(torch, ops, np.full_like(p, np.nan), q, ids, rng.random(12), rng.random(6), start)


def test_small_weights_and_ties(torch, ops):
    """Runs of equal probabilities, whose sums are exact, with a random number on a boundary:
    the token is the first whose sum is larger. fp16 subnormals. Without `rejected`."""
    V = 1 << 15
    for dtype, w in ((np.float32, 2.0 ** -15), (np.float16, 2.0 ** -15), (np.float16, 2.0 ** -24)):
        target = np.full((6, V), w, dtype)
        un = np.array([0.0, 0.25, 0.5, 2.0 ** -15, 1 - 2.0 ** -15, 1 - 2.0 ** -24])
        got = _check(torch, ops, target, None, np.zeros(6, int), np.zeros(6), un, np.arange(7), rejected=False)
        assert list(got[1]) == [0, V // 4, V // 2, 1, V - 1, V - 1]


def test_no_requests_and_no_rows(torch, ops):
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    f = torch.zeros(1, device="cuda")
    acc = torch.full((2,), 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ops.verify_draft(f, f, z, f, f, z, 0, 0, 5, acc, z)
    ops.verify_draft(None, None, None, None, f, torch.zeros(3, dtype=torch.int32, device="cuda"), 2, 0, 5, acc, None)
    torch.cuda.synchronize()
    assert torch.all(acc == 0)


def test_long_window(torch, ops):
    """More drafted tokens than a workgroup has threads."""
    rng = np.random.default_rng(2)
    V, k = 64, 700
    p = _probs(rng, k, V, np.float32)
    u = np.zeros(k)
    for stop in (0, 255, 256, 699, 10 ** 6):
        u[:] = 0.0
        if stop < k - 1:
            u[stop] = 1.0
        q = np.where(np.arange(k)[:, None] == stop, 1.0, p * 0.5).astype(np.float32)
        got = _check(torch, ops, p, q, rng.integers(0, V, k), u, rng.random(1), [0, k])
        assert got[0][0] == min(stop, k - 1)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_large_vocabulary(torch, ops, dtype):
    """More units of the vocabulary than a workgroup has threads; nothing left of the target above the draft there."""
    rng = np.random.default_rng(4)
    V = 600001
    p, q = _probs(rng, 6, V, dtype, 1.0), _probs(rng, 6, V, dtype, 1.0)
    ids = rng.integers(0, V, 6)
    for un in (0.0, 0.37, 1.0):
        _check(torch, ops, p, q, ids, np.ones(6), np.full(3, un), [0, 1, 4, 6])
    got = _check(torch, ops, p, p, ids, np.ones(6), rng.random(3), [0, 1, 4, 6])
    assert np.all(got[0] == 0) and np.all(got[1][[0, 1, 4]] >= 0)


def test_many_requests(torch, ops):
    """More requests than one dimension of a grid has."""
    rng = np.random.default_rng(5)
    n, V = 70000, 6
    counts = rng.integers(0, 3, n)
    start = np.concatenate([[0], np.cumsum(counts)])
    rows = int(start[-1])
    p, q = _probs(rng, rows, V, np.float32, 1.0), _probs(rng, rows, V, np.float32, 1.0)
    _check(torch, ops, p, q, rng.integers(0, V, rows), rng.random(rows), rng.random(n), start)
