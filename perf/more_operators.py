"""Operators of a server whose paged key / value cache is held in 4 bits.

Kinds of case, each one pass through the operators as such a server calls them:

  store      keys and values of new tokens quantised as they are written into
             the cache's pages, all layers at once, and read back as the values
             that the cache now stands for
  read       tokens of sequences read out of the cache: whole sequences that
             leave the device, or stretches of them
  attention  the queries of a batch of sequences over the cache: one query a
             sequence (a decode step), a ragged window of them (drafted tokens),
             or a piece of a prompt; causal inside the window, the first
             `shared` tokens common to the batch

Where `own` is true the passes go through `mod_amd.ops`; where it is false they
are computed in elementary torch operations in 32 bits. `exact` restates each in
64 bits, sequence by sequence.

The cache: 32 neighbouring values of a token's head share a power of two, 2^e,
and each is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, times it. e is the
least with max |x| < 7 * 2^e, from -23 to 13; a value goes to the nearest, ties
to the even code. A block with an inf or a NaN reads as NaN.
  kv  uint8 [layers][k, v][pages][kv heads][page size][17 * head_dim / 32]: the
      bytes of a (page, kv head) are the codes [page size][head_dim / 2] (the
      even dimension in the low half: 3 bits of value under a sign), then e + 127
      (255: NaN) as [head_dim / 32][page size].
Beside it a table of page ids per sequence, the sequences' lengths and the number
of tables that hold each page."""
import math
import random

import torch

own = False

DEV = "cuda:0"
_TORCH = {"float32": torch.float32, "float16": torch.float16}
_BYTES = {"float32": 4, "float16": 2}
LAYER = 1              # the attention cases read the second of their two layers


def listed():
    return [
        # One token of one request, one layer: latency and nothing else.
        dict(name="store_one", kind="store", layers=1, Hk=2, D=64, page=16, n=1, context=40, new=1, x="float32"),
        # A decode step's tokens of 48 requests through all layers of the 0.6B model, whose activations are fp32.
        dict(name="store_step", kind="store", layers=28, Hk=8, D=128, page=16, n=48, context=900, new=1, x="float32"),
        # A prompt, and a few pieces of others, of an odd number of tokens.
        dict(name="store_prompt", kind="store", layers=28, Hk=8, D=128, page=32, n=3, context=60, new=1501, x="float16"),
        # The end of one sequence, one layer, for a kernel of the caller's own.
        dict(name="read_few", kind="read", layers=1, Hk=4, D=128, page=16, n=3, context=77, x="float32", whole=False),
        # Requests that leave the device for host memory, whole, in all layers.
        dict(name="read_out", kind="read", layers=28, Hk=8, D=128, page=16, n=7, context=900, x="float16", whole=True),
        # One request behind a short conversation, fp32 activations: the smallest decode step.
        dict(name="attend_one", kind="attention", n=1, shared=0, tail=301, window=1, H=16, Hk=8, D=128, page=16,
             x="float32"),
        # A chat server's decode step behind one system prompt that ends inside a page.
        dict(name="attend_chat", kind="attention", n=40, shared=1019, tail=1300, window=1, H=16, Hk=8, D=128, page=16,
             x="float32"),
        # Many long conversations that have nothing in common: the cache is read once, and that is all.
        dict(name="attend_batch", kind="attention", n=96, shared=0, tail=16000, window=1, H=32, Hk=4, D=128, page=64,
             x="float16"),
        # A few very long ones.
        dict(name="attend_long", kind="attention", n=3, shared=0, tail=120011, window=1, H=32, Hk=8, D=128, page=128,
             x="float16"),
        # Questions about one long document, drafted tokens among them.
        dict(name="attend_document", kind="attention", n=40, shared=24000, tail=700, window=3, H=32, Hk=4, D=128, page=64,
             x="float16"),
        # Windows of drafted tokens over small heads, 7 queries to a kv head.
        dict(name="attend_window", kind="attention", n=24, shared=250, tail=2100, window=6, H=14, Hk=2, D=64, page=16,
             x="float16"),
        # Pieces of two prompts behind what was read of them so far.
        dict(name="attend_prompt", kind="attention", n=2, shared=0, tail=4090, window=509, H=32, Hk=8, D=128, page=32,
             x="float16"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "store", "read"])
    if kind == "store":
        return dict(kind=kind, layers=_log(rng, 1, 28), Hk=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64]), n=_log(rng, 1, 64), context=_log(rng, 1, 600),
                    new=rng.choice([1, 1, _log(rng, 1, 64)]), x=rng.choice(["float32", "float16"]))
    if kind == "read":
        return dict(kind=kind, layers=_log(rng, 1, 28), Hk=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64]), n=_log(rng, 1, 12), context=_log(rng, 1, 700),
                    x=rng.choice(["float32", "float16"]), whole=rng.random() < 0.5)
    H, Hk, D = rng.choice([(16, 8, 128), (32, 4, 128), (32, 8, 128), (16, 16, 64), (14, 2, 64), (7, 1, 128)])
    window = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 2, 300)])
    n = _log(rng, 1, 96 if window == 1 else 24 if window <= 8 else 2)
    shared = rng.choice([0, 0, _log(rng, 1, 12000), _log(rng, 256, 12000)])
    return dict(kind=kind, n=n, shared=shared, tail=_log(rng, window, 4000), window=window, H=H, Hk=Hk, D=D,
                page=rng.choice([16, 16, 32, 64, 128]), x=rng.choice(["float32", "float16"]))


# ---------------------------------------------------------------- the plan ---
def _plan(case):
    """Lengths, tokens and pages of a case: the case's own, whatever the seed."""
    c, rng = case, random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    P, n, shared = c["page"], c["n"], c.get("shared", 0)
    if c["kind"] == "attention":
        counts = [rng.randint(1, c["window"]) for _ in range(n)]
        tails = [_log(rng, k, max(k, c["tail"])) for k in counts]
        counts[0], tails[0] = c["window"], max(c["window"], c["tail"])
        lens = [shared + t for t in tails]
    elif c["kind"] == "store":
        counts = [rng.randint(1, c["new"]) for _ in range(n)]
        counts[0] = c["new"]
        lens = [_log(rng, 1, c["context"]) + k for k in counts]
    else:
        lens = [_log(rng, 1, c["context"]) for _ in range(n)]
        lens[0] = c["context"]
        counts = list(lens) if c["whole"] else [rng.randint(1, k) for k in lens]
    first = [rng.randint(0, k - m) for k, m in zip(lens, counts)]
    whole = shared // P
    need = [-(-k // P) for k in lens]
    total = whole + sum(k - whole for k in need) + 5
    ids = list(range(total))
    rng.shuffle(ids)
    common, at, rows = ids[:whole], whole, []
    for k in need:
        rows.append(common + ids[at:at + k - whole])
        at += k - whole
    order = list(range(n + 3))
    rng.shuffle(order)
    return dict(counts=counts, lens=lens, first=first, rows=rows, pages=total, seq=order[:n], max_seqs=n + 3,
                max_pages=max(need) + 2, tail=max(lens) - shared)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# -------------------------------------------------------------- the format ---
def _views(kv, D):
    """Codes [.., page, D / 2] and scales [.., D / 32, page] of a cache's pages."""
    page = kv.shape[-2]
    flat = kv.flatten(-2)
    return flat[..., :page * D // 2].unflatten(-1, (page, D // 2)), flat[..., page * D // 2:].unflatten(-1, (D // 32, page))


_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _encode(x):
    """Codes [.., D] 0 .. 15 and scale bytes [.., D / 32] of x [.., D]."""
    x = x.float().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    m, e = torch.frexp(torch.where(fine, most, 1.0))                   # most = m * 2^e, m from 0.5 below 1
    e = (e - 3 + (m >= 0.875).int()).clamp(-23, 13)
    e = torch.where(most > 0, e, -23)
    y = torch.ldexp(torch.where(fine, x, 0.0), -e)
    a = y.abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = torch.where((y < 0) & (code > 0), code + 8, code)
    return code.flatten(-2).byte(), torch.where(fine, e + 127, 255).squeeze(-1).byte()


def _pack(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def _decode(packed, scale):
    """Values [.., D] fp32 of packed codes [.., D / 2] and scale bytes [.., D / 32]."""
    lut = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=DEV)
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).int()
    s = torch.where(scale == 255, math.nan, torch.exp2(scale.float() - 127.0))
    return (lut[code].unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _pages(kv, D, ids):
    """Tokens [.., kv heads, pages * page, D] fp32 of the pages ids [..] of one layer's k or v, in order."""
    codes, scales = _views(kv[ids], D)
    x = _decode(codes, scales.transpose(-1, -2))                       # [.., pages, Hk, page, D]
    return x.transpose(-4, -3).flatten(-3, -2)


def _fill(kv, D, normal):
    """The cache's pages filled with quantised normal values, some pages at a time."""
    layers, _, pages, heads, page, _ = kv.shape
    codes, scales = _views(kv, D)
    step = max(1, (1 << 26) // (heads * page * D))
    for layer in range(layers):
        for kind in range(2):
            for p in range(0, pages, step):
                code, scale = _encode(normal(min(step, pages - p), heads, page, D))
                codes[layer, kind, p:p + step] = _pack(code)
                scales[layer, kind, p:p + step] = scale.transpose(-1, -2)


def prepare(case, seed):
    c, plan = case, _plan(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    layers, D, P, x = c.get("layers", 2), c["D"], c["page"], _TORCH[c["x"]]
    kv = torch.zeros(layers, 2, plan["pages"], c["Hk"], P, 17 * D // 32, dtype=torch.uint8, device=DEV)
    _fill(kv, D, normal)
    table = torch.full((plan["max_seqs"], plan["max_pages"]), -1, dtype=torch.int32)
    lens = torch.zeros(plan["max_seqs"], dtype=torch.int32)
    refs = torch.zeros(plan["pages"], dtype=torch.int32)
    for q, pages, k in zip(plan["seq"], plan["rows"], plan["lens"]):
        table[q, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        lens[q] = k
        refs += torch.bincount(torch.tensor(pages, dtype=torch.int64), minlength=plan["pages"]).int()
    start = [0]
    for k in plan["counts"]:
        start.append(start[-1] + k)
    R = start[-1]
    s = dict(case=c, kv=kv, table=table.to(DEV), lens=lens.to(DEV), refs=refs.to(DEV), seq=_ints(plan["seq"]),
             row_start=_ints(start), rows=R, tail=plan["tail"],
             row_seq=torch.repeat_interleave(torch.arange(c["n"], device=DEV), torch.tensor(plan["counts"], device=DEV)))
    if c["kind"] == "attention":
        part, whole = c["shared"] % P, c["shared"] // P
        if part:       # the prefix's last tokens lie in a page of each sequence's own
            at = torch.tensor([r[whole] for r in plan["rows"]], device=DEV)
            codes, scales = _views(kv, D)
            codes[:, :, at, :, :part] = codes[:, :, at[:1], :, :part].clone()
            scales[:, :, at, :, :, :part] = scales[:, :, at[:1], :, :, :part].clone()
        s.update(q=normal(R, c["H"], D).to(x), out=torch.empty(R, c["H"], D, dtype=x, device=DEV))
    else:
        shape = (layers, R, c["Hk"], D)
        s.update(k_out=torch.empty(shape, dtype=x, device=DEV), v_out=torch.empty(shape, dtype=x, device=DEV))
        if c["kind"] == "store":
            s.update(k=normal(*shape).to(x), v=normal(*shape).to(x))
        else:
            s["first"] = _ints(plan["first"])
    if own:            # the handle that a program opens once for its cache
        from mod_amd import ops
        s["cache"] = ops.KvCache(kv, s["table"], s["lens"], s["refs"])
    return s


# --------------------------------------------------------------- one pass ----
def run(state):
    s, c = state, state["case"]
    if c["kind"] == "attention":
        (_attention_own if own else _attention_plain)(s)
        return s["out"]
    if own:
        _tokens_own(s)
    else:
        _tokens_plain(s)
    return dict(k=s["k_out"], v=s["v_out"])


def _attention_own(s):
    from mod_amd import ops
    c = s["case"]
    ops.kv_attention(s["cache"], LAYER, s["seq"], s["row_start"], c["n"], s["q"], s["out"], s["rows"], c["H"],
                     c["D"] ** -0.5, shared=c["shared"], max_rows=c["window"])


def _tokens_own(s):
    from mod_amd import ops
    c = s["case"]
    if c["kind"] == "store":
        ops.kv_write(s["cache"], 0, c["layers"], s["seq"], s["row_start"], c["n"], s["k"], s["v"], s["rows"])
    ops.kv_read(s["cache"], 0, c["layers"], s["seq"], s["row_start"], c["n"], s["k_out"], s["v_out"], s["rows"],
                first=s.get("first"))


def _tokens_plain(s):
    c = s["case"]
    P = c["page"]
    start = s["row_start"].long()
    of = s["seq"].long()[s["row_seq"]]
    first = s["lens"][s["seq"].long()].long() - (start[1:] - start[:-1]) if c["kind"] == "store" else s["first"].long()
    at = first[s["row_seq"]] + torch.arange(s["rows"], device=DEV) - start[:-1][s["row_seq"]]
    page = s["table"][of, at // P].long()
    codes, scales = _views(s["kv"], c["D"])
    for kind, name in enumerate(("k", "v")):
        if c["kind"] == "store":
            code, scale = _encode(s[name])
            codes[:, kind, page, :, at % P] = _pack(code).transpose(0, 1)
            scales[:, kind, page, :, :, at % P] = scale.transpose(0, 1)
        x = _decode(codes[:, kind, page, :, at % P], scales[:, kind, page, :, :, at % P])      # [rows, layers, Hk, D]
        s[name + "_out"].copy_(x.transpose(0, 1))


def _attention_plain(s):
    c = s["case"]
    n, Hk, G, D, P, W, shared = c["n"], c["Hk"], c["H"] // c["Hk"], c["D"], c["page"], c["window"], c["shared"]
    keys, values = s["kv"][LAYER, 0], s["kv"][LAYER, 1]
    table = s["table"][s["seq"].long()].long()
    first, count = s["row_start"][:-1].long(), (s["row_start"][1:] - s["row_start"][:-1]).long()
    # queries padded to the widest window: [n, W, Hk, G, D]
    at = (first[:, None] + torch.arange(W, device=DEV)).clamp(max=s["rows"] - 1)
    q = s["q"].float().reshape(-1, Hk, G, D)[at]
    # position that each query stands at; it sees the keys up to there
    stands = s["lens"][s["seq"].long()].long()[:, None] - count[:, None] + torch.arange(W, device=DEV)
    whole = shared // P
    # the prefix's whole pages once, [Hk, keys, D]; behind them each sequence's own, [n, Hk, keys, D]
    ids = table[0, :whole]
    kp, vp = _pages(keys, D, ids), _pages(values, D, ids)
    ids = table[:, whole:-(-(shared + s["tail"]) // P)].clamp(min=0)
    kt, vt = _pages(keys, D, ids), _pages(values, D, ids)
    t = whole * P + torch.arange(kt.shape[2], device=DEV)
    qp = q.permute(2, 0, 1, 3, 4).reshape(Hk, n * W * G, D)
    sp = torch.matmul(qp, kp.transpose(1, 2).contiguous()).reshape(Hk, n, W * G, -1).transpose(0, 1)
    qt = q.permute(0, 2, 1, 3, 4).reshape(n, Hk, W * G, D)
    st = torch.matmul(qt, kt.transpose(2, 3).contiguous())                             # [n, Hk, W * G, keys]
    seen = (t <= stands[:, :, None])[:, None, :, None, :].expand(n, 1, W, G, -1).reshape(n, 1, W * G, -1)
    scores = torch.cat([sp, st.masked_fill(~seen, -math.inf)], 3) * D ** -0.5
    weights = torch.exp(scores - scores.amax(3, keepdim=True))
    total = weights.sum(3, keepdim=True)
    wp = weights[..., :whole * P].transpose(0, 1).reshape(Hk, n * W * G, whole * P)
    o = torch.matmul(wp, vp).reshape(Hk, n, W * G, D).transpose(0, 1)
    o = (o + torch.matmul(weights[..., whole * P:], vt)) / total
    o = o.reshape(n, Hk, W, G, D).transpose(1, 2)
    row = torch.arange(s["rows"], device=DEV)
    s["out"].copy_(o[s["row_seq"], row - first[s["row_seq"]]].reshape(s["rows"], c["H"], D))


# ------------------------------------------------------------------- work ----
def work(case):
    c, plan = case, _plan(case)
    rows = sum(plan["counts"])
    token = c["Hk"] * c["D"] * 17 / 32                 # bytes of a token's keys (or values) in a layer
    if c["kind"] == "attention":
        tokens = c["shared"] + sum(k - c["shared"] for k in plan["lens"])
        seen = sum(k - m + j + 1 for k, m in zip(plan["lens"], plan["counts"]) for j in range(m))
        return dict(bytes=int(2 * tokens * token) + 2 * rows * c["H"] * c["D"] * _BYTES[c["x"]] +
                    4 * sum(map(len, plan["rows"])), flops=4 * c["H"] * c["D"] * seen)
    dense = c["Hk"] * c["D"] * _BYTES[c["x"]]
    passes = 2 if c["kind"] == "store" else 1          # written and read back, or read
    return dict(bytes=int(2 * rows * c["layers"] * passes * (token + dense)), flops=0)


# ------------------------------------------------------------------ exact ----
def _exact_tokens(block, D):
    """Values [.., page, D] in 64 bits of (page, kv head) blocks [.., page, 17 * D / 32], from the bits of each code."""
    page = block.shape[-2]
    raw = block.reshape(*block.shape[:-2], -1).long()
    byte = raw[..., :page * D // 2].reshape(*raw.shape[:-1], page, D // 2, 1)
    code = (byte >> torch.tensor([0, 4], device=DEV)).reshape(*raw.shape[:-1], page, D) & 15
    power, half = code >> 1 & 3, (code & 1).double()
    value = torch.where(power == 0, half / 2, (1 + half / 2) * 2.0 ** (power.double() - 1))
    value = value * (1 - 2 * (code >> 3).double())
    e = raw[..., page * D // 2:].reshape(*raw.shape[:-1], D // 32, page).transpose(-1, -2)
    unit = torch.where(e == 255, math.nan, 2.0 ** (e.double() - 127))
    return value * torch.repeat_interleave(unit, 32, -1)


def _exact_rounded(x, D):
    """What the cache holds of x [.., D] (finite values)."""
    x = x.double().reshape(*x.shape[:-1], D // 32, 32)
    most = x.abs().amax(-1, keepdim=True)
    e = -23 + sum((most >= 7 * 2.0 ** j).double() for j in range(-23, 13))
    y = x / 2.0 ** e
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(-6, 6)                    # ties to the even code, a multiple of two steps
    return (y * 2.0 ** e).reshape(*x.shape[:-2], D)


def exact(case, seed):
    c, s, plan = case, prepare(case, seed), _plan(case)
    D, P = c["D"], c["page"]
    if c["kind"] == "store":
        return dict(k=_exact_rounded(s["k"], D), v=_exact_rounded(s["v"], D))
    if c["kind"] == "read":
        out = ([], [])
        for pages, a, count in zip(plan["rows"], plan["first"], plan["counts"]):
            for kind in range(2):
                x = _exact_tokens(s["kv"][:, kind, torch.tensor(pages, device=DEV)], D)       # [layers, pages, Hk, P, D]
                out[kind].append(x.transpose(2, 3).reshape(c["layers"], -1, c["Hk"], D)[:, a:a + count])
        return dict(k=torch.cat(out[0], 1), v=torch.cat(out[1], 1))
    # each sequence and kv head by itself: softmax(q k^T / sqrt(D)) v over its own pages
    G, row = c["H"] // c["Hk"], 0
    out = torch.empty(s["rows"], c["H"], D, dtype=torch.float64, device=DEV)
    for pages, length, count in zip(plan["rows"], plan["lens"], plan["counts"]):
        ids = torch.tensor(pages, device=DEV)
        hidden = torch.arange(length, device=DEV) > torch.arange(length - count, length, device=DEV)[:, None]
        for h in range(c["Hk"]):
            k, v = (_exact_tokens(s["kv"][LAYER, kind, ids, h], D).reshape(-1, D)[:length] for kind in range(2))
            q = s["q"][row:row + count, h * G:(h + 1) * G].double()
            score = (q.reshape(-1, D) @ k.T.contiguous()).reshape(count, G, length) / math.sqrt(D)
            score = score.masked_fill(hidden[:, None], -math.inf)
            p = torch.exp(score - torch.logsumexp(score, 2, keepdim=True))
            out[row:row + count, h * G:(h + 1) * G] = (p.reshape(-1, length) @ v).reshape(count, G, D)
        row += count
    return out
