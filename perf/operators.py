"""The operators of a paged polar key cache, as plain cases: what they compute in elementary torch operations, and the calls that compute it here.

A page holds 128 tokens of every KV head.  A sequence's sealed pages come first: their keys are polar codes with the group's constants; the keys of
the pages behind them, its open ones, are the half-precision rows themselves.  Values are half-precision rows throughout.  `pages` [B, W] names the
physical page of every logical one (of codes, constants and values), `open_pages` [B, Wo] those of the open pages' keys, from the first open one on.
The tokens of a call are the last ones of their sequences, packed: sequence b's are rows q_start[b] .. q_start[b + 1] - 1.

Operators ("op"):
  attend  attention of a chunk of new tokens, or of one token, over the pages (`paged_attention`)
  append  norms of queries and keys for each head, their rotation by position, and the keys and values into their pages (`qk_norm_rope_append`)
  weigh   the attention weight that a chunk's queries give to each page, added to what it had (`page_weights`)
  evict   sealed pages of the least weight leave the tables (`evict_pages`)
"""
import math
import random

import torch

own = False                             # False: the plain forms, True: the framework's operators

PAGE, PAIRS, DIM = 128, 64, 128
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
HEADS = [(32, 8), (32, 32), (28, 4), (16, 8)]       # query and KV heads
BITS = [(4, 4), (4, 4), (3, 3), (4, 3)]             # radius and angle
EPS = 1e-6


def listed():
    return [
        # a chat turn's next token: one sequence, short context, 7 query heads per KV head
        dict(name="token_b1_2k", op="attend", batch=1, heads=28, kv_heads=4, tokens=2001, chunk=1, ragged=False, padded=False, sealed=True, rbits=4, tbits=4,
             dtype="bfloat16"),
        # a served batch at long context, a token each
        dict(name="token_b16_32k", op="attend", batch=16, heads=32, kv_heads=8, tokens=32768, chunk=1, ragged=False, padded=False, sealed=True, rbits=4, tbits=4,
             dtype="float16"),
        # continuous batching: sequences of all lengths, 3-bit codes
        dict(name="token_ragged_b64", op="attend", batch=64, heads=28, kv_heads=4, tokens=8192, chunk=1, ragged=True, padded=False, sealed=True, rbits=3, tbits=3,
             dtype="float16"),
        # a short turn behind a conversation, whose pages are still open (half-precision keys)
        dict(name="turn_b2_5k_open", op="attend", batch=2, heads=32, kv_heads=8, tokens=5000, chunk=37, ragged=True, padded=False, sealed=False, rbits=4, tbits=4,
             dtype="bfloat16"),
        # a batch's portions of up to 512 tokens, left-padded sequences among them
        dict(name="chunk_b8_8k", op="attend", batch=8, heads=32, kv_heads=8, tokens=8192, chunk=512, ragged=True, padded=True, sealed=True, rbits=4, tbits=4,
             dtype="bfloat16"),
        # a portion of a long document
        dict(name="chunk_b1_32k", op="attend", batch=1, heads=32, kv_heads=8, tokens=32768, chunk=2048, ragged=False, padded=False, sealed=True, rbits=4, tbits=4,
             dtype="bfloat16"),
        # the rows of a token of a served batch, and those of a long prompt
        dict(name="append_token_b16", op="append", batch=16, heads=32, kv_heads=8, tokens=4000, chunk=1, ragged=False, normed=True, dtype="bfloat16"),
        dict(name="append_prompt_b4", op="append", batch=4, heads=32, kv_heads=8, tokens=1000, chunk=4096, ragged=True, normed=True, dtype="bfloat16"),
        # what a token of each sequence attends to, and what a portion does
        dict(name="weigh_token_b8_4k", op="weigh", batch=8, heads=28, kv_heads=4, tokens=4096, chunk=1, ragged=True, sealed=True, rbits=4, tbits=4, dtype="float16"),
        dict(name="weigh_chunk_b1_16k", op="weigh", batch=1, heads=32, kv_heads=8, tokens=16384, chunk=512, ragged=False, sealed=True, rbits=4, tbits=4,
             dtype="bfloat16"),
        # a conversation's table, and those of a served batch at long context
        dict(name="evict_b1_32", op="evict", batch=1, kv_heads=8, pages=32, keep=16, ragged=False),
        dict(name="evict_b64_1k", op="evict", batch=64, kv_heads=8, pages=1024, keep=400, ragged=True),
    ]


def draw(rng):
    def spread(lo, hi):                 # even over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attend", "attend", "attend", "attend", "append", "append", "weigh", "weigh", "evict"])
    if op == "evict":
        kv_heads = rng.choice([4, 8, 32])
        pages = spread(2, 8192 // kv_heads)
        return dict(op=op, batch=spread(1, 64), kv_heads=kv_heads, pages=pages, keep=rng.randint(max(1, pages // 8), pages), ragged=rng.random() < 0.7)
    heads, kv_heads = rng.choice(HEADS)
    dtype, ragged = rng.choice(sorted(DTYPES)), rng.random() < 0.5
    if op == "append":
        batch = spread(1, 64)
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, tokens=spread(1, 8192), chunk=spread(1, 16384 * 48 // (batch * (heads + 2 * kv_heads))), ragged=ragged,
                    normed=rng.random() < 0.6, dtype=dtype)
    rbits, tbits = rng.choice(BITS)
    batch = spread(1, 64)
    cached = spread(1, min(32768, 16 * 8 * 32768 // (batch * kv_heads)))
    # (query rows times keys, and those of the plain form's scores in memory: no more than the listed largest)
    most = 16384 * 512 if op == "weigh" else 32768 * 2048
    chunk = 1 if rng.random() < 0.3 else spread(1, max(1, min(2048, most // (batch * (cached + 2048)))))
    more = dict(padded=batch > 1 and rng.random() < 0.3) if op == "attend" else {}
    return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, tokens=cached, chunk=chunk, ragged=ragged, sealed=rng.random() < 0.8, rbits=rbits, tbits=tbits,
                dtype=dtype, **more)


def _lengths(c):
    """Tokens of each sequence before the call, and in it: of the case alone."""
    r = random.Random(c["batch"] * 1000003 + c["tokens"] * 1009 + c["chunk"])
    cached, new = [c["tokens"]] * c["batch"], [c["chunk"]] * c["batch"]
    if c["ragged"]:                     # from a sixteenth on; the first sequence is the longest
        cached = [c["tokens"]] + [r.randint(-(-c["tokens"] // 16), c["tokens"]) for _ in range(c["batch"] - 1)]
        new = [c["chunk"]] + [r.randint(-(-c["chunk"] // 16), c["chunk"]) for _ in range(c["batch"] - 1)]
    return cached, new


def _sealed(c):
    return [n // PAGE if c.get("sealed") else 0 for n in _lengths(c)[0]]


def _table_lengths(c):
    """Sealed pages of each sequence of an eviction."""
    r = random.Random(c["batch"] * 1000003 + c["pages"])
    return [c["pages"]] + [r.randint(-(-c["pages"] // 16), c["pages"]) if c["ragged"] else c["pages"] for _ in range(c["batch"] - 1)]


def work(case):
    c = dict(case)
    if c["op"] == "evict":
        n = sum(_table_lengths(c))
        return {"bytes": 4 * n * (2 * c["kv_heads"] + 3), "flops": n * c["kv_heads"]}
    cached, new = _lengths(c)
    N, Nk, T = c["heads"], c["kv_heads"], sum(new)
    if c["op"] == "append":             # rows in and out, and the angles of the positions that occur
        angles = sum(new) if c["ragged"] else c["chunk"]
        return {"bytes": 2 * DIM * (T * (2 * N + 4 * Nk) + 2 * angles), "flops": T * DIM * (N + Nk) * (7 if c["normed"] else 3)}
    sealed = [PAGE * p for p in _sealed(c)]
    keys = sum(68 * s + 2 * DIM * (n + m - s) for s, n, m in zip(sealed, cached, new)) * Nk
    seen = sum(m * n + m * (m + 1) // 2 for n, m in zip(cached, new))
    if c["op"] == "weigh":
        return {"bytes": keys + T * N * (2 * DIM + 4) + 8 * Nk * sum(-(-(n + m) // PAGE) for n, m in zip(cached, new)), "flops": 2 * DIM * N * seen}
    return {"bytes": keys + 2 * DIM * Nk * sum(n + m for n, m in zip(cached, new)) + 4 * DIM * T * N, "flops": 4 * DIM * N * seen}


# ----------------------------------------------------------------------------- inputs
def _angles(positions):
    f = 5e5 ** (-torch.arange(0, DIM, 2, device="cuda", dtype=torch.float64) / DIM)
    a = positions.double()[:, None] * f
    return a.cos(), a.sin()


def _keys(g, heads, tokens, dtype):
    """[tokens, heads, 128] as a model leaves them: normal, 4 channels 8 times as large, rotated by position."""
    k = torch.randn(tokens, heads, DIM, generator=g, device="cuda")
    k[..., torch.randperm(DIM, generator=g, device="cuda")[:4]] *= 8.0
    cos, sin = (t.float()[:, None] for t in _angles(torch.arange(tokens, device="cuda")))
    a, b = k[..., :PAIRS], k[..., PAIRS:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(dtype)


def _quantize(k, rbits, tbits):
    """k [.., 128, 128] (tokens of a page, channels) -> codes [.., 128, 64] and the constants [.., 1, 64] of radius and angle: width of a bin, least."""
    x = k.float().unflatten(-1, (2, PAIRS))
    phi, r = torch.atan2(x[..., 1, :], x[..., 0, :]) % (2 * math.pi), x.square().sum(-2).sqrt()

    def bins(v, bits):
        lo, hi = v.amin(-2, keepdim=True), v.amax(-2, keepdim=True)
        step = (hi - lo) / 2 ** bits
        return ((v - lo) / step).floor().clamp_(0, 2 ** bits - 1).to(torch.uint8), step.to(k.dtype), lo.to(k.dtype)

    rho, rscale, rmn = bins(r, rbits)
    theta, tscale, tmn = bins(phi, tbits)
    return (rho << tbits) + theta, rscale, rmn, tscale, tmn


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(g, counts, width):
    """[B, width] physical pages: `counts[b]` of each, no page twice, in no order; -1 behind them.  -> table, pages in all."""
    n = sum(counts)
    every, table = torch.randperm(n, generator=g, device="cuda").int(), torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda") < _ints(counts)[:, None]] = every
    return table, n


def _prepare_evict(c, g):
    counts = _table_lengths(c)
    width = max(counts) + 2             # one or two open pages behind the sealed ones
    table, _ = _tables(g, [n + 1 + n % 2 for n in counts], width)
    w = torch.rand(c["batch"], c["kv_heads"], width, generator=g, device="cuda").pow(4) * 100
    sealed = _ints(counts)
    return dict(weights=w * (torch.arange(width, device="cuda") < sealed[:, None])[:, None], pages=table, n_sealed=sealed,
                kv_len=PAGE * sealed + torch.randint(1, PAGE, (c["batch"],), generator=g, device="cuda", dtype=torch.int32), keep=c["keep"], sinks=1,
                max_kv=PAGE * width)


def _prepare_rows(c, g):
    """Pages, tables and lengths that the other operators share."""
    dt, Nk = DTYPES[c["dtype"]], c["kv_heads"]
    cached, new = _lengths(c)
    sealed, total = _sealed(c), [a + b for a, b in zip(cached, new)]
    held = [-(-n // PAGE) for n in total]
    pages, n_pages = _tables(g, held, max(held))
    open_pages, n_open = _tables(g, [h - s for h, s in zip(held, sealed)], max(h - s for h, s in zip(held, sealed)))
    s = dict(pages=pages, open_pages=open_pages, n_sealed=_ints(sealed), kv_len=_ints(total), q_start=_ints([sum(new[:b]) for b in range(c["batch"] + 1)]),
             max_q=max(new), max_kv=max(total), rbits=c.get("rbits", 4), tbits=c.get("tbits", 4))
    if c["op"] == "append":
        s.update(keys=torch.zeros(n_open, Nk, PAGE, DIM, dtype=dt, device="cuda"), values=torch.zeros(n_pages, Nk, PAGE, DIM, dtype=dt, device="cuda"))
        return s
    values = torch.randn(n_pages, Nk, PAGE, DIM, generator=g, device="cuda", dtype=dt) if c["op"] == "attend" else torch.zeros(1, Nk, PAGE, DIM, dtype=dt, device="cuda")
    codes = torch.zeros(n_pages, Nk, PAGE, PAIRS, dtype=torch.uint8, device="cuda")
    meta = [torch.zeros(n_pages, Nk, 1, PAIRS, dtype=dt, device="cuda") for _ in range(4)]
    keys = torch.zeros(n_open, Nk, PAGE, DIM, dtype=dt, device="cuda")
    for b in range(c["batch"]):
        k = _keys(g, Nk, held[b] * PAGE, dt).unflatten(0, (held[b], PAGE)).transpose(1, 2)
        at, behind = pages[b, :sealed[b]].long(), open_pages[b, :held[b] - sealed[b]].long()
        if sealed[b]:
            for whole, part in zip([codes, *meta], _quantize(k[:sealed[b]], c["rbits"], c["tbits"])):
                whole[at] = part
        keys[behind] = k[sealed[b]:]
    return dict(s, values=values, codes=codes, rscale=meta[0], rmn=meta[1], tscale=meta[2], tmn=meta[3], keys=keys)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["op"] == "evict":
        s = _prepare_evict(c, g)
    else:
        s = _prepare_rows(c, g)
        dt, N, Nk, T, B = DTYPES[c["dtype"]], c["heads"], c["kv_heads"], int(sum(_lengths(c)[1])), c["batch"]
        if c["op"] == "append":         # one projection's output, and the tables and weights of the model
            s["qkv"] = torch.randn(T, (N + 2 * Nk) * DIM, generator=g, device="cuda").to(dt)
            s["cos"], s["sin"] = (torch.cat([t, t], -1).to(dt) for t in _angles(torch.arange(s["max_kv"] + 100, device="cuda")))
            s["q_norm"], s["k_norm"] = ((1 + 0.2 * torch.randn(DIM, generator=g, device="cuda")).to(dt) if c["normed"] else None for _ in range(2))
        else:
            s["q"] = torch.randn(T, N, DIM, generator=g, device="cuda").to(dt)
        if c["op"] == "attend":
            s["mask"] = None
            if c["padded"]:             # left padding of up to half of what is cached
                pad = (torch.rand(B, 1, generator=g, device="cuda") * s["kv_len"][:, None] / 2).int()
                s["mask"] = (torch.arange(s["max_kv"], device="cuda") >= pad).to(torch.uint8)
        if c["op"] == "weigh":          # the attention's log sums, and what the pages had
            s["weights"] = torch.rand(B, Nk, s["pages"].shape[1], generator=g, device="cuda")
            s["lse"] = _log_sums(s)
    if own:                             # what a server keeps: a layer's pages, and a step's tables
        from polarquant_amd.paged import PageBatch, PagePool
        if c["op"] == "evict":
            s["batch"] = PageBatch(None, s["kv_len"], s["n_sealed"], s["pages"], None, 1, s["max_kv"])
        else:
            s["pool"] = PagePool(s["keys"], s["values"], *(s.get(n) for n in ("codes", "rscale", "rmn", "tscale", "tmn")), rbits=s["rbits"], tbits=s["tbits"])
            s["batch"] = PageBatch(s["q_start"], s["kv_len"], s["n_sealed"], s["pages"], s["open_pages"], s["max_q"], s["max_kv"])
    return dict(s, case=c)


# ----------------------------------------------------------------------------- one pass
def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from polarquant_amd.paged import evict_pages, page_weights, paged_attention, qk_norm_rope_append
        if op == "attend":
            return paged_attention(s["q"], s["pool"], s["batch"], attention_mask=s["mask"])
        if op == "append":
            N, Nk = s["case"]["heads"], s["case"]["kv_heads"]
            q, k, v = s["qkv"].split([N * DIM, Nk * DIM, Nk * DIM], -1)
            q = qk_norm_rope_append(q, k, v, s["cos"], s["sin"], s["pool"], s["batch"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
            return {"q": q, "keys": s["keys"], "values": s["values"]}
        if op == "weigh":
            return page_weights(s["q"], s["lse"], s["pool"], s["batch"], onto=s["weights"])
        batch, weights, freed = evict_pages(s["weights"], s["batch"], s["keep"], sinks=s["sinks"])
        return {"pages": batch.pages, "n_sealed": batch.n_sealed, "kv_len": batch.kv_len, "weights": weights, "freed": freed}
    return {"attend": _attend, "append": _append, "weigh": _weigh, "evict": _evict}[op](s)


def _rows(s):
    """Of each packed row: its sequence, and its position in it."""
    starts = s["q_start"].long()
    row = torch.arange(s["q" if "q" in s else "qkv"].shape[0], device="cuda")
    b = (row[:, None] >= starts[1:]).sum(-1)
    return b, s["kv_len"].long()[b] - starts[b + 1] + row


def _all_keys(s):
    """Keys of all pages of all sequences, [B, Nk, W * 128, 128] in 32 bits."""
    W, Wo = s["pages"].shape[1], s["open_pages"].shape[1]
    logical = torch.arange(W, device="cuda")
    sealed = logical < s["n_sealed"][:, None]
    at = torch.where(sealed, s["pages"], 0).long()
    theta, rho = (s["codes"][at] & (2 ** s["tbits"] - 1)).float(), (s["codes"][at] >> s["tbits"]).float()
    phi = s["tscale"][at].float() * (theta + 0.5) + s["tmn"][at].float()
    r = s["rscale"][at].float() * (rho + 0.5) + s["rmn"][at].float()
    behind = (logical - s["n_sealed"][:, None]).clamp(0, Wo - 1).long()
    rows = s["keys"][s["open_pages"].gather(1, behind).clamp(min=0).long()].float()
    k = torch.where(sealed[:, :, None, None, None], torch.cat([r * phi.cos(), r * phi.sin()], -1), rows)
    return k.transpose(1, 2).flatten(2, 3)


def _scores(s):
    """Scores [B, Nk, heads of a KV head * max_q, keys] in 32 bits, minus infinity where there is nothing to see, and where each packed row is."""
    q, Nk, B = s["q"], s["keys"].shape[1], s["pages"].shape[0]
    k = _all_keys(s)
    b, position = _rows(s)
    t = torch.arange(q.shape[0], device="cuda") - s["q_start"].long()[b]
    wide = torch.zeros(B, s["max_q"], q.shape[1], DIM, device="cuda")
    wide[b, t] = q.float()
    last = torch.full((B, s["max_q"]), -1, device="cuda")
    last[b, t] = position
    rep = q.shape[1] // Nk
    z = wide.unflatten(2, (Nk, rep)).permute(0, 2, 3, 1, 4).flatten(2, 3) @ k.transpose(2, 3) / math.sqrt(DIM)
    key = torch.arange(k.shape[2], device="cuda")
    hidden = key > last[:, :, None]
    if s.get("mask") is not None:
        seen = torch.nn.functional.pad(s["mask"], (0, k.shape[2] - s["mask"].shape[1])) != 0
        hidden = hidden | ~seen[:, None]
    return z.unflatten(2, (rep, -1)).masked_fill_(hidden[:, None, None], -math.inf).flatten(2, 3), b, t


def _attend(s):
    z, b, t = _scores(s)
    m = z.amax(-1, keepdim=True).clamp(min=-1e30)
    w = z.sub_(m).exp_()
    total = w.sum(-1, keepdim=True)
    v = s["values"][s["pages"].clamp(min=0).long()].float().transpose(1, 2).flatten(2, 3)
    out = torch.where(total > 0, w @ v / total, 0.0)
    rep = s["q"].shape[1] // v.shape[1]
    return out.unflatten(2, (rep, -1)).permute(0, 3, 1, 2, 4)[b, t].flatten(1, 2).to(s["q"].dtype)


def _log_sums(s):
    """[T, N]: natural logarithm of each row's sum of exponentials."""
    z, b, t = _scores(s)
    rep = s["q"].shape[1] // z.shape[1]
    return z.logsumexp(-1).unflatten(2, (rep, -1)).permute(0, 3, 1, 2)[b, t].flatten(1, 2).contiguous()


def _weigh(s):
    z, b, t = _scores(s)
    B, Nk = z.shape[:2]
    lse = torch.full((B, s["max_q"], s["q"].shape[1]), math.inf, device="cuda")
    lse[b, t] = s["lse"]
    lse = lse.unflatten(2, (Nk, -1)).permute(0, 2, 3, 1).flatten(2, 3)
    w = (z - lse[..., None]).exp_().unflatten(-1, (-1, PAGE)).sum((2, 4), dtype=torch.float64)
    return (s["weights"] + w).float()


def _append(s):
    c = s["case"]
    N, Nk = c["heads"], c["kv_heads"]
    b, position = _rows(s)
    q, k, v = (t.unflatten(-1, (-1, DIM)) for t in s["qkv"].split([N * DIM, Nk * DIM, Nk * DIM], -1))
    cos, sin = s["cos"][position].float()[:, None], s["sin"][position].float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        return (x * cos + torch.cat([-x[..., PAIRS:], x[..., :PAIRS]], -1) * sin).to(v.dtype)

    logical, slot = position // PAGE, position % PAGE
    s["keys"][s["open_pages"][b, logical - s["n_sealed"].long()[b]].long(), :, slot] = turned(k, s["k_norm"])
    s["values"][s["pages"][b, logical].long(), :, slot] = v
    return {"q": turned(q, s["q_norm"]), "keys": s["keys"], "values": s["values"]}


def _evict(s):
    W, n, B = s["pages"].shape[1], s["n_sealed"].long()[:, None], s["pages"].shape[0]
    at = torch.arange(W, device="cuda").expand(B, W)
    total = s["weights"].sum(1, dtype=torch.float64).float()
    total = torch.where(at < s["sinks"], math.inf, total).masked_fill(at >= n, -math.inf)       # (what is always kept first, what is not there last)
    rank = total.sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
    stays = (rank < s["keep"]) & (at < n)
    behind = (at >= n) & (s["pages"] >= 0)
    goes = ~stays & ~behind & (at < n)
    # entries that stay, in their order, then -1
    front = lambda chosen: (~chosen).to(torch.int8).sort(dim=-1, stable=True).indices               # noqa: E731
    left, gone = (stays | behind), goes.sum(-1, keepdim=True)
    order = front(left)
    pages = torch.where(at < left.sum(-1, keepdim=True), s["pages"].gather(1, order), -1)
    kept = torch.where(at < left.sum(-1, keepdim=True), order, W)
    weights = torch.nn.functional.pad(s["weights"], (0, 1)).gather(2, kept[:, None].expand_as(s["weights"]))
    freed = torch.where(at < gone, s["pages"].gather(1, front(goes)), -1)
    gone = gone[:, 0].int()
    return {"pages": pages, "n_sealed": s["n_sealed"] - gone, "kv_len": s["kv_len"] - PAGE * gone, "weights": weights, "freed": freed}


# ----------------------------------------------------------------------------- the same in 64 bits, sequence by sequence
F64 = torch.float64


def _sequences(s, case):
    """(first row, rows, tokens, sealed pages) of each."""
    cached, new = _lengths(case)
    first = 0
    for n, m, p in zip(cached, new, _sealed(case)):
        yield first, m, n + m, p
        first += m


def _exact_keys(s, b, h, tokens, sealed):
    """[tokens, 128] of one head."""
    parts = []
    if sealed:
        at = s["pages"][b, :sealed].long()
        code = s["codes"][at, h].int()
        bins = 1 << s["tbits"]
        angle = (torch.remainder(code, bins).to(F64) + 0.5) * s["tscale"][at, h].to(F64) + s["tmn"][at, h].to(F64)
        radius = (torch.div(code, bins, rounding_mode="floor").to(F64) + 0.5) * s["rscale"][at, h].to(F64) + s["rmn"][at, h].to(F64)
        parts.append(torch.stack([radius * torch.cos(angle), radius * torch.sin(angle)], -2).reshape(-1, DIM))
    rest = -(-tokens // PAGE) - sealed
    if rest:
        parts.append(s["keys"][s["open_pages"][b, :rest].long(), h].to(F64).reshape(-1, DIM))
    return torch.cat(parts)[:tokens]


def _exact_heads(s, case):
    """Of each sequence and KV head: its indices, the scores [rows, heads, tokens] of its rows, keys that are not seen at minus infinity."""
    rep = case["heads"] // case["kv_heads"]
    for b, (first, rows, tokens, sealed) in enumerate(_sequences(s, case)):
        unseen = torch.arange(tokens, device="cuda")[None] > torch.arange(tokens - rows, tokens, device="cuda")[:, None]
        if s.get("mask") is not None:
            unseen = unseen | (s["mask"][b, :tokens] == 0)
        for h in range(case["kv_heads"]):
            q = s["q"][first:first + rows, h * rep:(h + 1) * rep].to(F64)
            z = torch.matmul(q.reshape(-1, DIM), _exact_keys(s, b, h, tokens, sealed).t().contiguous()).reshape(rows, rep, tokens) * DIM ** -0.5
            yield b, h, first, rows, tokens, z.masked_fill_(unseen[:, None], -math.inf)


def _exact_attend(s, case):
    rep, out = case["heads"] // case["kv_heads"], torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    for b, h, first, rows, tokens, z in _exact_heads(s, case):
        v = s["values"][s["pages"][b, :-(-tokens // PAGE)].long(), h].to(F64).reshape(-1, DIM)[:tokens]
        p = torch.softmax(z, -1).nan_to_num_(0.0)           # (a row that sees nothing)
        out[first:first + rows, h * rep:(h + 1) * rep] = torch.matmul(p.reshape(-1, tokens), v).reshape(rows, rep, DIM)
    return out


def _exact_weigh(s, case):
    rep, out = case["heads"] // case["kv_heads"], s["weights"].to(F64)
    for b, h, first, rows, tokens, z in _exact_heads(s, case):
        p = torch.exp(z - s["lse"][first:first + rows, h * rep:(h + 1) * rep, None].to(F64)).sum((0, 1))
        out[b, h].index_add_(0, torch.arange(tokens, device="cuda") // PAGE, p)
    return out


def _exact_append(s, case):
    N, Nk = case["heads"], case["kv_heads"]
    x = s["qkv"].to(F64).reshape(-1, N + 2 * Nk, DIM)
    keys, values, q = s["keys"].to(F64), s["values"].to(F64), torch.empty(x.shape[0], N, DIM, dtype=F64, device="cuda")
    for b, (first, rows, tokens, sealed) in enumerate(_sequences(s, case)):
        part, at = x[first:first + rows], torch.arange(tokens - rows, tokens, device="cuda")
        c, n = (s[t][at].to(F64)[:, None] for t in ("cos", "sin"))
        for heads, w, put in ((slice(0, N), s["q_norm"], "q"), (slice(N, N + Nk), s["k_norm"], "k")):
            y = part[:, heads]
            if w is not None:
                y = y / torch.sqrt(torch.mean(y * y, -1, keepdim=True) + EPS) * w.to(F64)
            lo, hi = y.chunk(2, -1)
            y = torch.cat([lo * c[..., :PAIRS] - hi * n[..., :PAIRS], hi * c[..., PAIRS:] + lo * n[..., PAIRS:]], -1)
            if put == "q":
                q[first:first + rows] = y
            else:
                keys[s["open_pages"][b, at // PAGE - sealed].long(), :, at % PAGE] = y
        values[s["pages"][b, at // PAGE].long(), :, at % PAGE] = part[:, N + Nk:]
    return {"q": q, "keys": keys, "values": values}


def _exact_evict(s, case):
    pages, weights = s["pages"].tolist(), s["weights"].cpu().to(F64)
    W, out = len(pages[0]), {"pages": [], "n_sealed": [], "kv_len": [], "weights": torch.zeros_like(weights), "freed": []}
    for b, (n, length) in enumerate(zip(s["n_sealed"].tolist(), s["kv_len"].tolist())):
        held = weights[b].sum(0).to(torch.float32).tolist()
        always = list(range(min(s["sinks"], n)))
        chosen = sorted(range(len(always), n), key=lambda j: (-held[j], j))[:max(0, s["keep"] - len(always))]
        stay = sorted(always + chosen) if n > s["keep"] else list(range(n))
        gone = [j for j in range(n) if j not in set(stay)]
        left = stay + [j for j in range(n, W) if pages[b][j] >= 0]
        out["pages"].append([pages[b][j] for j in left] + [-1] * (W - len(left)))
        out["freed"].append([pages[b][j] for j in gone] + [-1] * (W - len(gone)))
        out["weights"][b, :, :len(left)] = weights[b][:, left]
        out["n_sealed"].append(len(stay))
        out["kv_len"].append(length - PAGE * len(gone))
    return {k: v.cuda() if torch.is_tensor(v) else torch.tensor(v, dtype=torch.int32, device="cuda") for k, v in out.items()}


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    return {"attend": _exact_attend, "append": _exact_append, "weigh": _exact_weigh, "evict": _exact_evict}[c["op"]](s, c)
