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
    (4, 2, 128, 3, "float16"), (4, 2, 64, 3, "float16"), (16, 1, 64, 4, "float16"), (32, 1, 128, 300, "float16"),
    (32, 1, 128, 400, "float16"), (32, 1, 64, 400, "float16"),
    (4, 2, 128, 3, "float32"), (4, 2, 64, 3, "float32"), (16, 1, 128, 70, "float32"), (16, 1, 64, 70, "float32"),
    (32, 1, 128, 400, "float32"), (32, 1, 64, 400, "float32"),
]


# ------------------------------------------------------------------ every key counts
def held(rng, lens, layers, Hk, D, page, common=0, spare=3):
    """A cache with sequences of the given lengths, in pages in any order; the pages of the first `common` tokens that
    these fill are the same."""
    need = [-(-n // page) for n in lens]
    same = common // page
    pages = same + sum(max(n - same, 0) for n in need) + spare
    c = kv_ref.Cache4(layers, Hk, D, page, pages, len(lens), max(need) + 1)
    free = [int(i) for i in rng.permutation(pages)]
    first = [free.pop() for _ in range(same)]
    for s, (n, k) in enumerate(zip(lens, need)):
        c.table[s, :k] = (first + [free.pop() for _ in range(max(k - same, 0))])[:k]
        c.lens[s] = n
    np.add.at(c.refs, c.table[c.table >= 0], 1)
    return c


def flat(rng, c, key=119):
    """Keys so small (under scales of 2^-8) that all weights are nearly the same, and values of 1 with signs of their own
    for every 16 rows of a page and each dimension: 32 keys that are left out, or taken twice, move some dimension of an
    output by 32 of the keys that a query sees."""
    codes, scales = c.blocks()
    codes[:, 0] = rng.integers(0, 256, codes[:, 0].shape)
    scales[:, 0], scales[:, 1] = key, 127
    sign = np.repeat(rng.integers(0, 4, (*codes[:, 1].shape[:3], c.P // 16, c.D // 2)), 16, 3).astype(np.uint8)
    codes[:, 1] = 0x22 | (sign & 1) << 3 | (sign & 2) << 6


def share(c, common):
    """The tokens of a prefix that lie in a page of each sequence's own are those of sequence 0."""
    part, at = common % c.P, common // c.P
    codes, scales = c.blocks()
    for s in range(1, len(c.lens)):
        n = min(part, int(c.lens[s]) - at * c.P)
        if n > 0:
            codes[:, :, c.table[s, at], :, :n] = codes[:, :, c.table[0, at], :, :n]
            scales[:, :, c.table[s, at], :, :, :n] = scales[:, :, c.table[0, at], :, :, :n]


def attend(c, layer, s, q, scale, times=None):
    """Outputs of q [rows, H, D], the last tokens of sequence s; times: how often each key is taken."""
    n, rows = int(c.lens[s]), len(q)
    k, v = c.rows(layer, s, n)
    times = np.ones(n) if times is None else times
    G = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape)
    hidden = np.arange(n) > np.arange(n - rows, n)[:, None]
    for h in range(k.shape[1]):
        sc = np.einsum("rgd,td->rgt", q[:, h * G:(h + 1) * G].astype(np.float64), k[:, h], optimize=True) * scale
        sc[np.broadcast_to(hidden[:, None], sc.shape)] = -np.inf
        top = sc.max(2, keepdims=True)
        w = np.exp(sc - np.where(np.isfinite(top), top, 0)) * times
        out[:, h * G:(h + 1) * G] = w @ v[:, h] / np.maximum(w.sum(2, keepdims=True), 1e-300)
    return out


def flat_tolerance(x, out, largest):
    """Of outputs of values of 1 where scores are no larger than `largest`. fp16: each weight is off by up to 2^-11 of it,
    which moves an output by that much of the weight times |v - out|; then the output is rounded. fp32: two parts of a
    weight, 2^-22. Scores, of a running sum of exponents up to 16: PARTS + 4 roundings, and what the parts drop."""
    off = (PARTS[x] + 4) * 2.0 ** -24 * 16 / LOG2E + OFF[x] * largest
    each = 2.0 ** -11 if x == "float16" else 2.0 ** -22
    return (each + 2 * off) * (1 + np.abs(out)) + each * np.abs(out)


FLAT_CASES = [
    # heads, kv heads, dim, page, queries; shared, the longest tail, how many; queries of each
    (8, 1, 128, 16, "float16", 0, 20011, 1, 1),          # runs of one sequence, over one kv head
    (8, 1, 128, 128, "float32", 0, 20011, 1, 2),
    (8, 4, 64, 64, "float16", 0, 9973, 1, 5),
    (8, 2, 64, 16, "float32", 0, 33001, 2, 1),
    (16, 2, 128, 32, "float16", 12320, 37, 12, 3),       # a long prefix
    (16, 2, 64, 16, "float32", 17001, 700, 12, 1),
    (24, 2, 128, 16, "float32", 2999, 3, 12, 7),         # rows that stand inside it
    (32, 4, 128, 32, "float16", 12320, 400, 12, 3),      # items of 32 columns
    (32, 4, 128, 16, "float16", 17003, 2, 12, 4),
    (32, 2, 128, 16, "float16", 0, 313, 1, 300),
    (32, 2, 64, 64, "float16", 0, 1313, 1, 300),
    (14, 2, 64, 16, "float16", 250, 2100, 24, 6),
    (32, 2, 128, 16, "float32", 0, 313, 1, 300),
    (32, 2, 64, 64, "float32", 0, 1313, 1, 300),
    (32, 2, 128, 32, "float32", 6000, 90, 12, 70),
    (32, 2, 64, 32, "float32", 6000, 90, 12, 70),
    (14, 2, 64, 32, "float16", 6000, 90, 40, 20),
    (32, 2, 128, 16, "float16", 0, 513, 1, 500),
    (32, 2, 64, 16, "float16", 0, 513, 1, 500),
    (32, 2, 128, 16, "float32", 0, 513, 1, 500),
    (32, 2, 64, 16, "float32", 0, 513, 1, 500),
    (8, 2, 128, 16, "float16", 0, 3000, 60, 1),          # ragged ones, cut into runs
    (8, 2, 128, 16, "float32", 0, 600, 300, 2),          # more than the waves find on their own
]


class Flat:
    def __init__(self, H, Hk, D, page, x, shared, tail, n, window):
        rng = np.random.default_rng(shared + tail)
        tails = [tail] + [max(1, int(t)) for t in np.exp(rng.uniform(np.log(max(1, tail / 40)), np.log(tail), n - 1))]
        self.c = held(rng, [shared + t for t in tails], 1, Hk, D, page, shared)
        flat(rng, self.c)
        share(self.c, shared)
        self.seq = [int(s) for s in rng.permutation(n)]
        self.counts = [min(window, int(self.c.lens[s])) if s == 0 else int(rng.integers(1, min(window, self.c.lens[s]) + 1))
                       for s in self.seq]
        self.start = np.concatenate([[0], np.cumsum(self.counts)]).astype(int)
        self.q = rng.standard_normal((int(self.start[-1]), H, D)).astype(x)
        self.scale, self.shared, self.window, self.x = D ** -0.5, shared, window, x
        # a score's most: queries times keys of up to 6 * 2^-8 in every dimension
        self.largest = float(np.abs(self.q).max()) * 6 * 2.0 ** -8 * D * self.scale

    def of(self, s):
        i = self.seq.index(s)
        return slice(self.start[i], self.start[i + 1])
