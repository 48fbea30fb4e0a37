"""Operators of a server that answers many requests at once from one paged cache.

Kinds of case, each one pass through an operator as such a server calls it:

  attention  the queries of a batch of sequences over a paged key / value cache
             whose first `shared` tokens all of them have in common: one query
             a sequence (a decode step) or a ragged window of them (drafted
             tokens to be verified), causal inside the window
  branch     one step over the pages themselves: the branches of the last step
             are dropped, forked again from their parents, room for their new
             tokens is reserved (a partly filled page that is shared is copied
             first), and the tokens' keys and values are written
  compact    the pages in use moved to the lowest slots, tables rewritten
  verify     drafted tokens accepted or rejected against the target's
             probabilities, and the token that follows the accepted ones drawn

Where `own` is true the passes go through `mod_amd.ops`; where it is false they
are computed in elementary torch operations, attention in 32 bits and the
verification's sums and comparisons in 64. `exact` restates each in 64 bits,
sequence by sequence.

A cache is [layers][k, v][pages][kv heads][page][head dim] beside a table of page
ids per sequence (-1 behind its last page), the sequences' lengths and the
number of tables that hold each page."""
import math
import random

import torch

own = False

DEV = "cuda:0"
_TORCH = {"float32": torch.float32, "float16": torch.float16}
_BYTES = {"float32": 4, "float16": 2}


def listed():
    return [
        # Four sequences behind a short instruction, fp32 activations and cache
        # (the decoder's own types): the smallest decode step, where latency counts.
        dict(name="attend_few", kind="attention", n=4, shared=509, tail=60, window=1, H=16, Hk=8, D=128, page=16,
             x="float32", kv="float32"),
        # A chat server's decode step: 32 sequences behind one system prompt,
        # fp32 activations over the fp16 cache; a prompt that ends inside a page.
        dict(name="attend_chat", kind="attention", n=32, shared=2039, tail=700, window=1, H=16, Hk=8, D=128, page=16,
             x="float32", kv="float16"),
        # Questions about one long document: 64 sequences behind 32,000 tokens.
        dict(name="attend_document", kind="attention", n=64, shared=32000, tail=1024, window=1, H=32, Hk=4, D=128,
             page=64, x="float16", kv="float16"),
        # Windows of 1 to 8 drafted tokens behind a shared prefix.
        dict(name="attend_window", kind="attention", n=48, shared=8200, tail=900, window=8, H=32, Hk=4, D=128, page=32,
             x="float16", kv="float16"),
        # The fp32 cache with small heads, ragged tails longer than the prefix.
        dict(name="attend_fp32", kind="attention", n=24, shared=1000, tail=3001, window=3, H=16, Hk=16, D=64, page=16,
             x="float32", kv="float32"),
        # Two branches of one request, one layer: tables and little else.
        dict(name="branch_few", kind="branch", layers=1, Hk=8, D=128, page=16, parents=1, children=2, context=41, new=5,
             x="float32", kv="float32"),
        # Four branches of each of 16 requests through all layers of the 0.6B model.
        dict(name="branch_batch", kind="branch", layers=28, Hk=8, D=128, page=16, parents=16, children=4, context=53,
             new=9, x="float32", kv="float16"),
        # A cache full of holes after half of its requests ended.
        dict(name="compact_half", kind="compact", layers=28, Hk=8, D=128, page=16, pages=168, seqs=24, live=0.5,
             kv="float16"),
        # The same with the few pages of a small cache.
        dict(name="compact_few", kind="compact", layers=2, Hk=4, D=128, page=16, pages=40, seqs=8, live=0.6,
             kv="float16"),
        # One request, four drafted tokens, the vocabulary of the Qwen3 models.
        dict(name="verify_one", kind="verify", n=1, window=4, vocab=151936, p="float32", draft=True),
        # A batch with up to eight drafted tokens each (some with none).
        dict(name="verify_batch", kind="verify", n=96, window=8, vocab=151936, p="float32", draft=True),
        # Tokens drafted without probabilities (copied from the prompt), fp16 targets.
        dict(name="verify_copied", kind="verify", n=33, window=5, vocab=32003, p="float16", draft=False),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "branch", "compact", "verify", "verify"])
    if kind == "attention":
        H, Hk, D = rng.choice([(16, 8, 128), (32, 4, 128), (32, 8, 128), (16, 16, 64), (12, 2, 64), (7, 1, 128)])
        x, kv = rng.choice([("float32", "float32"), ("float32", "float16"), ("float16", "float16"),
                            ("float16", "float16"), ("float16", "float32")])
        window = rng.choice([1, 1, 1, _log(rng, 2, 8)])
        n = _log(rng, 1, 64 if window == 1 else 16)
        shared = rng.choice([0, _log(rng, 1, 12000), _log(rng, 256, 12000)])
        return dict(kind=kind, n=n, shared=shared, tail=_log(rng, window, 1500), window=window, H=H, Hk=Hk, D=D,
                    page=rng.choice([16, 16, 32, 64, 128]), x=x, kv=kv)
    if kind == "branch":
        return dict(kind=kind, layers=_log(rng, 1, 28), Hk=rng.choice([1, 4, 8]), D=rng.choice([64, 128]),
                    page=rng.choice([16, 32]), parents=_log(rng, 1, 8), children=rng.randint(1, 4),
                    context=_log(rng, 2, 90), new=_log(rng, 1, 24), x=rng.choice(["float32", "float16"]),
                    kv=rng.choice(["float32", "float16"]))
    if kind == "compact":
        pages = _log(rng, 4, 96)
        return dict(kind=kind, layers=_log(rng, 1, 24), Hk=rng.choice([1, 4, 8]), D=rng.choice([64, 128]),
                    page=rng.choice([16, 32]), pages=pages, seqs=rng.randint(1, 17), live=rng.uniform(0.05, 0.95),
                    kv=rng.choice(["float32", "float16"]))
    return dict(kind=kind, n=_log(rng, 1, 72), window=rng.randint(0, 8), vocab=_log(rng, 50, 151936),
                p=rng.choice(["float32", "float32", "float16"]), draft=rng.random() < 0.7)


# ---------------------------------------------------------------- the plan ---
def _plan(case):
    """Lengths and pages of a case: the case's own, whatever the seed."""
    c, rng = case, random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if c["kind"] == "attention":
        counts = [rng.randint(1, c["window"]) for _ in range(c["n"])]
        tails = [_log(rng, k, max(k, c["tail"])) for k in counts]
        counts[0], tails[0] = c["window"], max(c["window"], c["tail"])
        lens = [c["shared"] + t for t in tails]
        whole, P = c["shared"] // c["page"], c["page"]
        need = [-(-n // P) for n in lens]
        total = whole + sum(k - whole for k in need) + 5
        ids = list(range(total))
        rng.shuffle(ids)
        common, at, rows = ids[:whole], whole, []
        for k in need:
            rows.append(common + ids[at:at + k - whole])
            at += k - whole
        order = list(range(c["n"] + 3))
        rng.shuffle(order)
        return dict(counts=counts, tails=tails, lens=lens, rows=rows, pages=total, seq=order[:c["n"]],
                    max_seqs=c["n"] + 3, max_pages=max(need) + 2)
    if c["kind"] == "branch":
        P, n = c["page"], c["parents"] * c["children"]
        contexts = [_log(rng, 1, c["context"]) for _ in range(c["parents"])]
        contexts[0] = c["context"]
        counts = [rng.randint(1, c["new"]) for _ in range(n)]
        counts[0] = c["new"]
        most = -(-(c["context"] + c["new"]) // P)
        held = sum(-(-k // P) for k in contexts)
        total = held + n * (1 + -(-c["new"] // P)) + 3
        ids = list(range(total))
        rng.shuffle(ids)
        rows, at = [], 0
        for k in contexts:
            rows.append(ids[at:at + -(-k // P)])
            at += -(-k // P)
        return dict(contexts=contexts, counts=counts, rows=rows, pages=total, max_seqs=c["parents"] + n,
                    max_pages=most + 1)
    if c["kind"] == "compact":
        used = max(1, min(c["pages"], round(c["pages"] * c["live"])))
        ids = rng.sample(range(c["pages"]), used)
        rows = [[] for _ in range(c["seqs"])]
        for p in ids:
            rows[rng.randrange(c["seqs"])].append(p)
        if len(rows) > 1 and rows[0]:
            rows[-1] = rows[0][:1] + rows[-1]         # a page that two tables hold
        lens = [max(0, len(r) * c["page"] - rng.randrange(c["page"])) if r else 0 for r in rows]
        return dict(rows=rows, lens=lens, pages=c["pages"], max_seqs=c["seqs"], max_pages=max(map(len, rows)) + 1)
    counts = [rng.randint(0, c["window"]) for _ in range(c["n"])]
    counts[0] = c["window"]
    return dict(counts=counts)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _tables(plan, rows):
    """Table, lengths and page counts of sequences that hold `rows`."""
    table = torch.full((plan["max_seqs"], plan["max_pages"]), -1, dtype=torch.int32)
    length = torch.zeros(plan["max_seqs"], dtype=torch.int32)
    refs = torch.zeros(plan["pages"], dtype=torch.int32)
    for i, (pages, n) in rows.items():
        table[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        length[i] = n
        refs += torch.bincount(torch.tensor(pages, dtype=torch.int64), minlength=plan["pages"]).int()
    return table.to(DEV), length.to(DEV), refs.to(DEV)


def prepare(case, seed):
    c, plan = case, _plan(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    if c["kind"] == "verify":
        start = [0]
        for k in plan["counts"]:
            start.append(start[-1] + k + 1)
        R, V = start[-1], c["vocab"]
        logits = normal(R, V) * 3.0
        target = torch.softmax(logits, 1)
        # a draft model sees the target's distribution with an error of its own
        near = torch.softmax(logits + normal(R, V) * 0.8, 1)
        ids = torch.multinomial(near, 1, generator=gen).reshape(-1).int()
        return dict(case=c, target=target.to(_TORCH[c["p"]]), ids=ids, row_start=_ints(start), rows=R, window=c["window"],
                 draft=near.to(_TORCH[c["p"]]) if c["draft"] else None,
                 u=torch.rand(R, generator=gen, device=DEV), u_next=torch.rand(c["n"], generator=gen, device=DEV),
                 accepted=torch.empty(c["n"], dtype=torch.int32, device=DEV),
                 tokens=torch.empty(R, dtype=torch.int32, device=DEV),
                 rejected=torch.empty(c["n"], dtype=torch.int32, device=DEV))
    layers = c.get("layers", 2)
    kv = normal(layers, 2, plan["pages"], c["Hk"], c["page"], c["D"]).to(_TORCH[c["kv"]])
    s = dict(case=c, kv=kv)
    if c["kind"] == "attention":
        rows = {q: (r, n) for q, r, n in zip(plan["seq"], plan["rows"], plan["lens"])}
        s["table"], s["lens"], s["refs"] = _tables(plan, rows)
        part, whole = c["shared"] % c["page"], c["shared"] // c["page"]
        if part:       # the prefix's last tokens lie in a page of each sequence's own
            own_pages = torch.tensor([r[whole] for r in plan["rows"]], device=DEV)
            kv[:, :, own_pages, :, :part] = kv[:, :, own_pages[:1], :, :part].clone()
        start = [0]
        for k in plan["counts"]:
            start.append(start[-1] + k)
        R = start[-1]
        s.update(seq=_ints(plan["seq"]), row_start=_ints(start), rows=R, q=normal(R, c["H"], c["D"]).to(_TORCH[c["x"]]),
                 row_seq=torch.repeat_interleave(torch.arange(c["n"], device=DEV), torch.tensor(plan["counts"], device=DEV)),
                 out=torch.empty(R, c["H"], c["D"], dtype=_TORCH[c["x"]], device=DEV), tail=max(plan["tails"]))
    elif c["kind"] == "branch":
        n, p = c["parents"] * c["children"], c["parents"]
        s["table"], s["lens"], s["refs"] = _tables(plan, dict(enumerate(zip(plan["rows"], plan["contexts"]))))
        start = [0]
        for k in plan["counts"]:
            start.append(start[-1] + k)
        R = start[-1]
        s.update(src=_ints([i % p for i in range(n)]), dst=_ints([p + i for i in range(n)]), counts=_ints(plan["counts"]),
                 row_start=_ints(start), rows=R,
                 row_seq=torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(plan["counts"], device=DEV)),
                 k=normal(layers, R, c["Hk"], c["D"]).to(_TORCH[c["x"]]),
                 v=normal(layers, R, c["Hk"], c["D"]).to(_TORCH[c["x"]]))
    else:
        rows = dict(enumerate(zip(plan["rows"], plan["lens"])))
        s["table"], s["lens"], s["refs"] = _tables(plan, rows)
        s.update(table_sent=s["table"].clone(), lens_sent=s["lens"].clone(), refs_sent=s["refs"].clone())
    if own:            # the handle that a program opens once for its cache, and the library's stream for torch
        from mod_amd import ops
        s["cache"] = ops.KvCache(kv, s["table"], s["lens"], s["refs"])
        s["stream"] = torch.cuda.ExternalStream(ops.lib.get_current_stream())
    return s


# --------------------------------------------------------------- one pass ----
LAYER = 1              # the attention cases read the second of their two layers


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "attention":
        return _attention_own(s) if own else _attention_plain(s)
    if c["kind"] == "verify":
        return _verify_own(s) if own else _verify_plain(s)
    if c["kind"] == "branch":
        if own:
            _branch_own(s)
        else:
            _branch_plain(s)
    elif own:
        _compact_own(s)
    else:
        _compact_plain(s)
    return dict(table=s["table"], lens=s["lens"], refs=s["refs"], kv=s["kv"])


def _attention_own(s):
    from mod_amd import ops
    c = s["case"]
    ops.kv_attention(s["cache"], LAYER, s["seq"], s["row_start"], c["n"], s["q"], s["out"], s["rows"], c["H"],
                     c["D"] ** -0.5, shared=c["shared"], max_rows=c["window"])
    return s["out"]


def _verify_own(s):
    from mod_amd import ops
    c = s["case"]
    ops.verify_draft(s["target"], s["draft"], s["ids"], s["u"], s["u_next"], s["row_start"], c["n"], s["rows"],
                     c["vocab"], s["accepted"], s["tokens"], rejected=s["rejected"])
    return dict(accepted=s["accepted"], tokens=s["tokens"], rejected=s["rejected"])


def _branch_own(s):
    from mod_amd import ops
    c, cache = s["case"], s["cache"]
    n = c["parents"] * c["children"]
    ops.kv_drop(cache, s["dst"], None, n)
    ops.kv_fork(cache, s["src"], s["dst"], n)
    ops.kv_reserve(cache, s["dst"], s["counts"], n)
    ops.kv_write(cache, 0, c["layers"], s["dst"], s["row_start"], n, s["k"], s["v"], s["rows"])


def _compact_own(s):
    from mod_amd import ops
    with torch.cuda.stream(s["stream"]):
        _send_tables(s)
    ops.kv_compact(s["cache"])


def _send_tables(s):
    """The tables as the scheduler sends them."""
    s["table"].copy_(s["table_sent"])
    s["lens"].copy_(s["lens_sent"])
    s["refs"].copy_(s["refs_sent"])


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
    t = torch.arange(shared, device=DEV)
    page = table[0, t // P]
    kp, vp = keys[page, :, t % P].float(), values[page, :, t % P].float()            # [shared, Hk, D]
    t = shared + torch.arange(s["tail"], device=DEV)
    page = table[:, (t // P).clamp(max=table.shape[1] - 1)].clamp(min=0)
    kt, vt = keys[page, :, t % P].float(), values[page, :, t % P].float()            # [n, tail, Hk, D]
    qp = q.permute(2, 0, 1, 3, 4).reshape(Hk, n * W * G, D)
    sp = torch.matmul(qp, kp.permute(1, 2, 0).contiguous()).reshape(Hk, n, W * G, shared).transpose(0, 1)
    qt = q.permute(0, 2, 1, 3, 4).reshape(n, Hk, W * G, D)
    st = torch.matmul(qt, kt.permute(0, 2, 3, 1).contiguous())                       # [n, Hk, W * G, tail]
    seen = (t <= stands[:, :, None])[:, None, :, None, :].expand(n, 1, W, G, -1).reshape(n, 1, W * G, -1)
    scores = torch.cat([sp, st.masked_fill(~seen, -math.inf)], 3) * D ** -0.5
    weights = torch.exp(scores - scores.amax(3, keepdim=True))
    total = weights.sum(3, keepdim=True)
    wp = weights[..., :shared].transpose(0, 1).reshape(Hk, n * W * G, shared)
    o = torch.matmul(wp, vp.transpose(0, 1).contiguous()).reshape(Hk, n, W * G, D).transpose(0, 1)
    o = (o + torch.matmul(weights[..., shared:], vt.transpose(1, 2).contiguous())) / total
    o = o.reshape(n, Hk, W, G, D).transpose(1, 2)
    row = torch.arange(s["rows"], device=DEV)
    s["out"].copy_(o[s["row_seq"], row - first[s["row_seq"]]].reshape(s["rows"], c["H"], D))
    return s["out"]


def _verify_plain(s):
    c = s["case"]
    V, W = c["vocab"], c["window"]
    first, count = s["row_start"][:-1].long(), (s["row_start"][1:] - s["row_start"][:-1]).long() - 1
    at = (first[:, None] + torch.arange(W + 1, device=DEV)).clamp(max=s["rows"] - 1)   # rows of each sequence
    inside = torch.arange(W + 1, device=DEV) < count[:, None]
    ids = s["ids"].long()
    p = s["target"].gather(1, ids[:, None])[:, 0].double()
    q = torch.ones_like(p) if s["draft"] is None else s["draft"].gather(1, ids[:, None])[:, 0].double()
    taken = (s["u"].double() * q < p)[at] & inside
    accepted = taken.long().cumprod(1).sum(1)
    row = first + accepted
    rejects = accepted < count
    weight = s["target"][row].double()
    if s["draft"] is None:
        less = torch.zeros_like(weight).scatter_(1, ids[row][:, None], 1.0)
    else:
        less = s["draft"][row].double()
    rest = (weight - less).clamp(min=0)
    weight = torch.where(rejects[:, None] & (rest.sum(1, keepdim=True) > 0), rest, weight)
    sums = weight.cumsum(1)
    place = (sums <= s["u_next"].double()[:, None] * sums[:, -1:]).sum(1)
    last = V - 1 - (weight > 0).flip(1).long().argmax(1)
    following = torch.minimum(place, last)
    j = torch.arange(W + 1, device=DEV)
    out = torch.where(j < accepted[:, None], ids[at], torch.where(j == accepted[:, None], following[:, None], -1))
    of = torch.repeat_interleave(torch.arange(c["n"], device=DEV), count + 1, output_size=s["rows"])
    s["tokens"].copy_(out[of, torch.arange(s["rows"], device=DEV) - first[of]])
    s["accepted"].copy_(accepted)
    s["rejected"].copy_(count - accepted)
    return dict(accepted=s["accepted"], tokens=s["tokens"], rejected=s["rejected"])


def _add_refs(refs, pages, by):
    """refs[page] += by for every page >= 0."""
    held = (pages >= 0).int() * by
    refs.index_add_(0, pages.clamp(min=0).reshape(-1).long(), held.reshape(-1))


def _branch_plain(s):
    c = s["case"]
    kv, table, lens, refs, P = s["kv"], s["table"], s["lens"], s["refs"], c["page"]
    src, dst, count = s["src"].long(), s["dst"].long(), s["counts"].long()
    # the last step's branches go
    _add_refs(refs, table[dst], -1)
    table[dst] = -1
    lens[dst] = 0
    # and are forked again
    table[dst] = table[src]
    lens[dst] = lens[src]
    _add_refs(refs, table[dst], 1)
    # pages for the new tokens, the lowest free ones in the order of the requests
    length = lens[dst].long()
    rows = table[dst].long()
    held = (length + P - 1) // P
    last = rows.gather(1, (held - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    copied = (length % P != 0) & (refs[last] > 1)
    new = (length + count + P - 1) // P - held
    need = copied.long() + new
    begin = need.cumsum(0) - need
    free = torch.sort((refs > 0).int(), stable=True).indices
    fresh = torch.where(copied, free[begin], last)
    filled = torch.arange(P, device=DEV) < (length % P)[:, None]         # the rows that the last page holds
    kv[:, :, fresh] = torch.where(filled[:, None, :, None], kv[:, :, last], kv[:, :, fresh])
    refs.index_add_(0, last, -copied.int())
    j = torch.arange(-(-c["new"] // P) + 1, device=DEV)
    page = free[(begin + copied.long())[:, None] + j]
    spare = torch.full_like(rows[:, :1], -1)
    wide = torch.cat([rows, spare], 1)                                   # the last column takes what is not used
    wide.scatter_(1, (held - 1).clamp(min=0)[:, None], fresh[:, None])
    wide.scatter_(1, torch.where(j < new[:, None], held[:, None] + j, rows.shape[1]), page)
    table[dst] = wide[:, :-1].int()
    more = torch.cat([refs, refs[:1]])
    more[torch.where(j < new[:, None], page, refs.shape[0])] = 1
    more[torch.where(copied, fresh, refs.shape[0])] = 1
    refs.copy_(more[:-1])
    lens[dst] = (length + count).int()
    # their keys and values
    row = torch.arange(s["rows"], device=DEV)
    at = length[s["row_seq"]] + row - s["row_start"][:-1].long()[s["row_seq"]]
    page = table[dst[s["row_seq"]], at // P].long()
    kv[:, 0, page, :, at % P] = s["k"].transpose(0, 1).to(kv.dtype)
    kv[:, 1, page, :, at % P] = s["v"].transpose(0, 1).to(kv.dtype)


def _compact_plain(s):
    _send_tables(s)
    kv, table, refs = s["kv"], s["table"], s["refs"]
    live = refs > 0
    index = torch.arange(refs.shape[0], device=DEV)
    inside = index < live.sum()
    src, dst = torch.nonzero(live & ~inside)[:, 0], torch.nonzero(~live & inside)[:, 0]
    kv[:, :, dst] = kv[:, :, src]
    index[src] = dst
    table.copy_(torch.where(table >= 0, index[table.clamp(min=0).long()].int(), table))
    refs[dst] = refs[src]
    refs[src] = 0


# ------------------------------------------------------------------- work ----
def work(case):
    c, plan = case, _plan(case)
    if c["kind"] == "attention":
        P, size = c["page"], _BYTES[c["kv"]]
        rows = sum(plan["counts"])
        tokens = c["shared"] + sum(plan["tails"])
        seen = sum(n - k + j + 1 for n, k in zip(plan["lens"], plan["counts"]) for j in range(k))
        return dict(bytes=2 * tokens * c["Hk"] * c["D"] * size + 2 * rows * c["H"] * c["D"] * _BYTES[c["x"]] +
                    4 * sum(map(len, plan["rows"])), flops=4 * c["H"] * c["D"] * seen)
    if c["kind"] == "verify":
        # the drafted tokens' probabilities, and of each sequence the row that its next token is drawn from
        rows = sum(plan["counts"]) + c["n"]
        row = c["vocab"] * _BYTES[c["p"]]
        both = 2 if c["draft"] else 1
        return dict(bytes=c["n"] * row * both + rows * (12 + both * _BYTES[c["p"]]), flops=3 * c["n"] * c["vocab"])
    token = 2 * c["layers"] * c["Hk"] * c["D"] * _BYTES[c["kv"]]
    tables = 4 * (plan["max_seqs"] * plan["max_pages"] + plan["pages"])
    if c["kind"] == "branch":
        P, n = c["page"], c["parents"] * c["children"]
        kept = [plan["contexts"][i % c["parents"]] for i in range(n)]
        copied = sum(k % P for k in kept)              # the tokens that a copied page holds
        written = sum(plan["counts"])
        return dict(bytes=2 * copied * token + written * token * (1 + _BYTES[c["x"]] / _BYTES[c["kv"]]) + 2 * tables,
                    flops=0)
    used = len({p for r in plan["rows"] for p in r})
    moved = len({p for r in plan["rows"] for p in r if p >= used})
    return dict(bytes=2 * moved * c["page"] * token + 2 * tables, flops=0)


# ------------------------------------------------------------------ exact ----
def exact(case, seed):
    s = prepare(case, seed)
    plan = _plan(case)
    if case["kind"] == "attention":
        return _attention_exact(s, plan)
    if case["kind"] == "verify":
        return _verify_exact(s, plan)
    return _branch_exact(s, plan) if case["kind"] == "branch" else _compact_exact(s, plan)


def _attention_exact(s, plan):
    """Each sequence by itself: softmax(q k^T / sqrt(D)) v over its own pages."""
    c = s["case"]
    P, D, G = c["page"], c["D"], c["H"] // c["Hk"]
    out, row = torch.empty(s["rows"], c["H"], D, dtype=torch.float64, device=DEV), 0
    for pages, length, count in zip(plan["rows"], plan["lens"], plan["counts"]):
        pool = s["kv"][LAYER][:, torch.tensor(pages, device=DEV)].double()          # [2, pages, Hk, P, D]
        k, v = pool.transpose(2, 3).reshape(2, len(pages) * P, c["Hk"], D)[:, :length]
        hidden = torch.arange(length, device=DEV) > torch.arange(length - count, length, device=DEV)[:, None]
        for h in range(c["Hk"]):
            q = s["q"][row:row + count, h * G:(h + 1) * G].double()                  # [count, G, D]
            score = (q.reshape(-1, D) @ k[:, h].T.contiguous()).reshape(count, G, length) / math.sqrt(D)
            score = score.masked_fill(hidden[:, None], -math.inf)
            p = torch.exp(score - torch.logsumexp(score, 2, keepdim=True))
            out[row:row + count, h * G:(h + 1) * G] = (p.reshape(-1, length) @ v[:, h].contiguous()).reshape(count, G, D)
        row += count
    return out


def _verify_exact(s, plan):
    c, start = s["case"], s["row_start"].tolist()
    ids, u, u_next = s["ids"].tolist(), s["u"].tolist(), s["u_next"].tolist()
    tokens, accepted = torch.full((s["rows"],), -1, dtype=torch.int32), []
    for i, (a, b) in enumerate(zip(start, start[1:])):
        r = a
        while r < b - 1:
            p = float(s["target"][r, ids[r]])
            q = 1.0 if s["draft"] is None else float(s["draft"][r, ids[r]])
            if not u[r] * q < p:
                break
            tokens[r] = ids[r]
            r += 1
        w = s["target"][r].double().cpu()
        if r < b - 1:
            less = torch.zeros_like(w)
            if s["draft"] is None:
                less[ids[r]] = 1.0
            else:
                less = s["draft"][r].double().cpu()
            rest = torch.relu(w - less)
            w = rest if float(rest.sum()) > 0 else w
        sums = torch.cumsum(w, 0)
        over = torch.nonzero(sums > u_next[i] * sums[-1])
        tokens[r] = int(over[0]) if len(over) else int(torch.nonzero(w > 0)[-1])
        accepted.append(r - a)
    left = [b - a - 1 - k for a, b, k in zip(start, start[1:], accepted)]
    return dict(accepted=_ints(accepted), tokens=tokens.to(DEV), rejected=_ints(left))


def _branch_exact(s, plan):
    c = s["case"]
    P, n, p = c["page"], c["parents"] * c["children"], c["parents"]
    kv = s["kv"].double()
    table, lens = s["table"].tolist(), s["lens"].tolist()
    refs = s["refs"].tolist()
    for i in range(n):                                  # forked, nothing written yet
        table[p + i], lens[p + i] = list(table[i % p]), lens[i % p]
        for page in table[p + i]:
            if page >= 0:
                refs[page] += 1
    free = [page for page, held in enumerate(refs) if not held]
    then, row = list(refs), 0
    for i, count in enumerate(plan["counts"]):
        at, length = table[p + i], lens[p + i]
        if length % P and then[at[length // P]] > 1:
            old, page = at[length // P], free.pop(0)
            kv[:, :, page, :, :length % P] = kv[:, :, old, :, :length % P]
            refs[old] -= 1
            refs[page] = 1
            at[length // P] = page
        for j in range(-(-length // P), -(-(length + count) // P)):
            at[j] = free.pop(0)
            refs[at[j]] = 1
        for t in range(length, length + count):
            for kind, x in enumerate((s["k"], s["v"])):
                kv[:, kind, at[t // P], :, t % P] = x[:, row].double()
            row += 1
        lens[p + i] = length + count
    return dict(table=_ints(table), lens=_ints(lens), refs=_ints(refs), kv=kv)


def _compact_exact(s, plan):
    kv, table, refs = s["kv"].double(), s["table"].tolist(), s["refs"].tolist()
    holes = iter([page for page, held in enumerate(refs) if not held])
    used = sum(held > 0 for held in refs)
    for page in range(used, len(refs)):
        if refs[page]:
            to = next(holes)
            kv[:, :, to] = kv[:, :, page]
            refs[to], refs[page] = refs[page], 0
            table = [[to if x == page else x for x in r] for r in table]
    return dict(table=_ints(table), lens=s["lens"], refs=_ints(refs), kv=kv)
