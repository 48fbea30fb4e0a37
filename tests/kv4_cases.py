"""Contents and queries for tests of the attention over a cache of 4 bits in which each part of the computation shows
in the output by itself, and what a kernel may be off by on them. numpy only: what they see is tested without a GPU."""
import numpy as np

from oracle import kv_ref

LOG2E = 1.0 / np.log(2.0)
PARTS = {"float16": 4, "float32": 5}               # of a query
# Of the largest of 32 dimensions, by the parts: it is 3.75 of its unit or more, each part leaves half a step, and those
# are 1/4 of the first unit, 1/8 of the next ones, which are 2^-4, 2^-9, 2^-14 and 2^-19 of it.
OFF = {"float16": 2.0 ** -17 / 3.75, "float32": 2.0 ** -22 / 3.75}


# ------------------------------------------------------------------ a query's parts
def _e2m3(x):
    """The nearest number of 6 bits, ties to even, saturating at 7.5."""
    a = np.abs(x)
    step = np.where(a < 2, 0.125, np.where(a < 4, 0.25, 0.5))
    return np.sign(x) * np.minimum(np.round(a / step) * step, 7.5)


def split(q, parts, scale):
    """What `parts` parts of 6 bits hold of q [.., D] * scale * log2(e): a power of two for 32 dimensions that the
    largest is below 7.5 of, and units of a 16th, then a 32nd of the one before."""
    x = q.astype(np.float32) * np.float32(np.float32(scale) * np.float32(LOG2E))
    x = x.reshape(*x.shape[:-1], -1, 32)
    first = (np.abs(x).max(-1).view(np.uint32).astype(np.int64) + 0x100000 >> 23) - 2
    rest, out = x.astype(np.float64), np.zeros(x.shape)
    for p in range(parts):
        unit = 2.0 ** (np.maximum(first - (5 * p - 1 if p else 0), 1) - 127.0)[..., None]
        part = _e2m3(rest / unit) * unit
        out, rest = out + part, rest - part
    return out.reshape(q.shape)


class Parts:
    """A sequence whose key d is 4 times the unit vector of dimension d, and its value the unit vector of another: an
    output is the softmax's weights themselves. Behind them a token of zeros for each query.
    own: all queries are 1 and n steps of 2^-k, n from 0 to 3, so that their last bits are what the weights, exp(n), hang
      on (the last dimension's is 1, and all keys have -4 there: scores are sums of small numbers); else one dimension of
      each 32, which no key has, is 2^j times the others' step, and those are -3 to 3 steps."""

    def __init__(self, rng, D, H, Hk, rows, x, own):
        self.D, self.x, self.rows = D, x, rows
        if own:
            k = 10 if x == "float16" else 16
            self.scale, most = 2.0 ** k / 4, 1.0
            q = 1.0 + rng.integers(0, 4, (rows, H, D)) * 2.0 ** -k
            q[:, :, D - 1] = 1.0
            d0 = np.array([D - 1])
        else:
            self.scale, most = 0.25, 2.0 ** (12 if x == "float16" else 17)
            q = rng.integers(-3, 4, (rows, H, D)).astype(np.float64)
            d0 = 32 * np.arange(D // 32) + (7 * np.arange(D // 32) + 5) % 32
            q[:, :, d0] = most * rng.choice([-1, 1], q[:, :, d0].shape)
        self.q = q.astype(x)
        assert np.array_equal(self.q.astype(np.float64), q)
        T = D + rows
        self.k, self.v = np.zeros((T, Hk, D)), np.zeros((T, Hk, D))
        self.to = np.stack([rng.permutation(D) for _ in range(Hk)])         # dimension of each key's value
        for h in range(Hk):
            self.k[np.arange(D), h, np.arange(D)] = 4.0
            self.k[d0, h, d0] = 0.0
            if own:
                self.k[:D - 1, h, D - 1] = -4.0
            self.v[np.arange(D), h, self.to[h]] = 1.0
        self.of = np.repeat(self.to, H // Hk, 0)                            # [H, D]
        self.used = np.setdiff1d(np.arange(D), d0)
        # of a score: what the parts drop of its one or two queries; own: roundings of those times scale * log2(e), and of
        # the products' sum, relative to the largest; roundings of sums that are no larger than 3 and 16 of an exponent
        self.own = own
        each = 4 * self.scale * most
        off = (2 * OFF[x] + 4 * 2.0 ** -24 if own else OFF[x]) * each + (PARTS[x] + 4) * 2.0 ** -24 * (3 + 16 / LOG2E)
        # of a weight (the sum is off as much); fp16: weights, their sum and the output are rounded
        self.tol = np.expm1(2 * off) + (3 * 2.0 ** -11 if x == "float16" else 3 * 2.0 ** -22)

    def weights(self, x):
        """Outputs [rows, H, D] for queries x, already times scale * log2(e)."""
        s = 4 * (x - x[:, :, -1:] if self.own else np.where(np.isin(np.arange(self.D), self.used), x, 0.0)) / LOG2E
        top = np.maximum(s.max(2, keepdims=True), 0)
        w = np.exp(s - top)
        w /= w.sum(2, keepdims=True) + (1 + np.arange(self.rows))[:, None, None] * np.exp(-top)
        out = np.zeros(x.shape)
        np.put_along_axis(out, np.broadcast_to(self.of, x.shape), w, 2)
        return out

    def exact(self):
        return self.weights(self.q.astype(np.float64) * self.scale * LOG2E)

    def wrong(self, got):
        """How many times the bound the outputs are off by."""
        want = self.exact()
        return (np.abs(got - want) / (self.tol * np.maximum(want, 1e-30))).max(initial=0, where=want > 1e-6)


PARTS_CASES = [
    # heads, kv heads, dim, rows; the last of each type run in items of 32 columns
    (4, 2, 128, 3, "float16"), (4, 2, 64, 3, "float16"), (32, 1, 128, 300, "float16"), (16, 1, 64, 4, "float16"),
    (4, 2, 128, 3, "float32"), (4, 2, 64, 3, "float32"), (16, 1, 128, 70, "float32"), (16, 1, 64, 70, "float32"),
]
