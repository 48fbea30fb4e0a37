"""The oracle of the paged cache (oracle/kv_ref.py) against closed forms: page
counts add up after any run of calls, shared pages are copied before they are
written, attention over one key is its value, equal scores average, and the
verification draws from the target's distribution."""
import numpy as np
import pytest

from oracle import kv_ref


def _held(c):
    """Table entries that hold each page."""
    return np.bincount(c.table[c.table >= 0], minlength=len(c.refs))


def test_random_calls_keep_the_counts():
    rng = np.random.default_rng(0)
    c = kv_ref.Cache(1, 1, 8, 4, 40, 9, 12)
    mirror = {s: [] for s in range(9)}           # token values of each sequence
    next_value = 1.0
    for _ in range(300):
        what = rng.integers(4)
        if what == 0:
            seq = list(rng.permutation(9)[:rng.integers(1, 5)])
            count = [int(k) for k in rng.integers(0, 7, len(seq))]
            before = c.table.copy(), c.lens.copy(), c.refs.copy()
            try:
                c.reserve(seq, count)
            except kv_ref.Refused:
                assert all(np.array_equal(a, b) for a, b in zip(before, (c.table, c.lens, c.refs)))
                continue
            start = np.concatenate([[0], np.cumsum(count)])
            k = np.zeros((1, start[-1], 1, 8), np.float32)
            for i, s in enumerate(seq):
                for r in range(start[i], start[i + 1]):
                    k[0, r] = next_value
                    mirror[s].append(next_value)
                    next_value += 1
            c.write(0, seq, start, k, -k)
        elif what == 1:
            empty = [s for s in range(9) if not mirror[s]]
            full = [s for s in range(9) if mirror[s]]
            if empty and full:
                assert c.fork([full[0]], [empty[0]]) == []
                mirror[empty[0]] = list(mirror[full[0]])
        elif what == 2:
            s, k = int(rng.integers(9)), int(rng.integers(0, 9))
            c.drop([s], [k])
            mirror[s] = mirror[s][:max(0, len(mirror[s]) - k)]
        else:
            c.compact()
            used = int((c.refs > 0).sum())
            assert np.all(c.refs[:used] > 0) and np.all(c.refs[used:] == 0)
        assert np.array_equal(_held(c), c.refs)
        for s in range(9):
            assert c.lens[s] == len(mirror[s])
            k, v = c.rows(0, s, len(mirror[s]))
            assert np.array_equal(k[:, 0, 0], mirror[s]) and np.array_equal(v[:, 0, 0], -np.array(mirror[s]))


def test_attention_closed_forms():
    c = kv_ref.Cache(1, 2, 8, 4, 8, 2, 4)
    rng = np.random.default_rng(1)
    c.reserve([1], [6])
    kv = rng.standard_normal((2, 1, 6, 2, 8)).astype(np.float32)
    c.write(0, [1], [0, 6], kv[0], kv[1])
    q = np.zeros((6, 4, 8), np.float32)
    out = c.attention(0, [1], [0, 6], q, 1.0, np.zeros((6, 4, 8)))
    for r in range(6):           # equal scores: the mean over what the row sees
        np.testing.assert_allclose(out[r], np.repeat(kv[1, 0, :r + 1].astype(np.float64).mean(0), 2, 0), rtol=1e-12)
    c.drop([1], [6])
    c.reserve([1], [1])
    out = c.attention(0, [1], [0, 3], q[:3], 1.0, np.full((3, 4, 8), 7.0))
    assert np.all(out[:2] == 0) and np.all(out[2] != 7)      # two rows without a key


@pytest.mark.parametrize("certain", [False, True])
def test_verification_follows_the_target(certain):
    """Whatever the draft, the first token is distributed as the target says."""
    rng = np.random.default_rng(2)
    V, N = 5, 40000
    p = np.array([0.1, 0.4, 0.05, 0.25, 0.2])
    q = np.array([0.5, 0.1, 0.2, 0.0, 0.2])
    ids = np.full(N, 1) if certain else rng.choice(V, N, p=q)
    target = np.tile(p, (2 * N, 1))
    draft = None if certain else np.tile(q, (2 * N, 1))
    row_ids = np.zeros(2 * N, int)
    row_ids[::2] = ids
    acc, tok, rej = kv_ref.verify(target, draft, row_ids, rng.random(2 * N), rng.random(N), np.arange(0, 2 * N + 1, 2))
    share = np.bincount(tok[::2], minlength=V) / N
    assert np.all(np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / N))   # five standard deviations
    assert np.all(acc + rej == 1) and np.all((tok[1::2] >= 0) == (acc == 1))
