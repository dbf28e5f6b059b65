"""Cases of the paged KV cache's operators: appending with the rotary embedding, attention of
single tokens and of chunks over the cache (with every row's entropy), reading a span back.

The cache holds the keys and values of sequences of different lengths in pages of ``page``
tokens.  A tier of 8 bits (int8, fp8 = e4m3) keeps one scale for each page and KV head, and
the tokens of a page that is not full yet in fp16; the fp16 tier keeps fp16 throughout.

  append  new rows of q, k and v: q and k are rotated (fp32, one rounding to fp16), k and v
          go to the cache, and the blocks that the step touched are read back in fp16;
  decode  one query token a sequence against everything cached;
  chunk   several query tokens a sequence, causal, against everything cached.

``run`` computes them in elementary torch operations (``own = False``) or by the framework's
``PagedKVCache`` (``own = True``).
"""
import math

import torch

own = False

TIERS = ("int8", "fp8", "fp16")
CODE_MAX = {"int8": 127.0, "fp8": 448.0}
_MOST = {"append": (4.4e8, 1e12), "decode": (4.4e8, 1e12), "chunk": (3e8, 4.5e11)}  # bytes, flops of a drawn case


def listed():
    def case(name, op, tier, batch, heads, kv_heads, dim, page, ctx, new):
        return {"name": name, "op": op, "tier": tier, "batch": batch, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "page": page, "ctx": ctx, "new": new}

    return [
        # a single conversation's next token: nothing but latency
        case("append 1 token", "append", "int8", 1, 32, 8, 128, 16, 500, 1),
        # one step of a serving batch: a token for each of 96 sequences
        case("append 96 x 1", "append", "fp8", 96, 32, 8, 128, 16, 1900, 1),
        # prompts of different lengths, heads of 64 (22-layer model of the benchmark)
        case("append prompts d64", "append", "fp16", 3, 32, 4, 64, 32, 0, 1111),
        # a prefill step of 16384 tokens
        case("append prompts", "append", "int8", 4, 32, 8, 128, 64, 0, 6100),
        # a single conversation's next token over a short cache: latency
        case("decode 1 x 777", "decode", "int8", 1, 32, 8, 128, 16, 776, 1),
        # a serving batch of many lengths
        case("decode 48 ragged", "decode", "int8", 48, 32, 8, 128, 64, 8000, 1),
        # fp16 tier, heads of 64
        case("decode 16 fp16 d64", "decode", "fp16", 16, 32, 4, 64, 32, 8192, 1),
        # few long documents
        case("decode 6 x long", "decode", "fp8", 6, 32, 8, 128, 128, 65000, 1),
        # verifying a few drafted tokens for a batch
        case("chunk 24 x 5", "chunk", "int8", 24, 32, 8, 128, 32, 2500, 5),
        # a short question over a cached document
        case("chunk 100 over 7000", "chunk", "fp8", 1, 32, 8, 128, 64, 7000, 100),
        # ragged prefill chunks, heads of 64
        case("chunk 5 ragged d64", "chunk", "fp16", 5, 32, 4, 64, 16, 1500, 700),
        # a prefill chunk of a long prompt
        case("chunk 2048 over 14000", "chunk", "int8", 1, 32, 8, 128, 64, 14000, 2048),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _excluded(case):
    """Sizes that no case takes."""
    starts, counts = _lengths(case)
    return 3072 in (*starts, *counts, sum(counts), case["ctx"], case["new"], case["heads"] * case["dim"],
                    case["kv_heads"] * case["dim"])


def draw(rng):
    """A case of the listed ranges: every size spread over its range, odd ones among them."""
    op = rng.choice(("append", "decode", "chunk"))
    while True:
        dim = rng.choice((64, 128, 128))
        kv_heads = rng.choice((1, 2, 4, 4, 5, 8, 8))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 4, 6, 7, 8))
        page = rng.choice((16, 32, 64, 128))
        if op == "append":
            batch = _log_int(rng, 1, 96)
            new = rng.choice((1, 1, rng.randint(2, page), _log_int(rng, 64, 6000)))
            ctx = rng.choice((0, _log_int(rng, 1, 6000)))
        elif op == "decode":
            batch, new, ctx = _log_int(rng, 1, 64), 1, _log_int(rng, 1, 65000)
        else:
            batch, new, ctx = _log_int(rng, 1, 24), _log_int(rng, 2, 2048), rng.choice((0, _log_int(rng, 1, 14000)))
        c = {"op": op, "tier": rng.choice(TIERS), "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
             "page": page, "ctx": ctx, "new": new}
        w, top = work(c), _MOST[op]
        padded = batch * heads * new * (ctx + new) if op == "chunk" else batch * kv_heads * dim * (ctx + new)
        if w["bytes"] <= top[0] and w["flops"] <= top[1] and padded <= (9e8 if op == "chunk" else 6e8) \
                and not _excluded(c):
            return c


# ------------------------------------------------------------------ what a case's sizes mean
def _lengths(case):
    """(tokens cached before the step, new tokens) of each sequence: the first has the case's
    sizes, the others fractions of them."""
    starts, counts = [], []
    for b in range(case["batch"]):
        f = 1.0 if b == 0 else 0.08 + 0.92 * ((b * 0.6180339887) % 1.0)
        g = 1.0 if b == 0 else 0.15 + 0.85 * ((b * 0.7548776662) % 1.0)
        s, n = int(case["ctx"] * f), max(1, int(case["new"] * g))
        if case["op"] == "append" and n > case["page"]:
            s -= s % case["page"]  # a long prompt's chunks begin where a page begins
        starts.append(s)
        counts.append(n)
    return starts, counts


def _spans(case):
    """Tokens of the blocks that an append touches: from the first one's first token on."""
    starts, counts = _lengths(case)
    p = case["page"]
    return [s - s % p for s in starts], [n + s % p for s, n in zip(starts, counts)]


def work(case):
    starts, counts = _lengths(case)
    hq, hk, d, p = case["heads"], case["kv_heads"], case["dim"], case["page"]
    one = 2 if case["tier"] == "fp16" else 1
    T = sum(counts)
    if case["op"] == "append":
        _, span = _spans(case)
        rows_in = T * (hq + 2 * hk) * d * 2 + T * 2 * d * 2
        stored = T * 2 * hk * d * one
        back = sum(span) * 2 * hk * d * (one + 2)
        return {"bytes": rows_in + T * hq * d * 2 + stored + back, "flops": 3 * T * (hq + hk) * d + 2 * T * 2 * hk * d}
    cached = 0
    for s, n in zip(starts, counts):
        full = (s + n) // p * p if one == 1 else 0
        cached += 2 * hk * d * (full + 2 * (s + n - full)) + 8 * hk * (full // p)
    seen = sum(n * s + n * (n + 1) // 2 for s, n in zip(starts, counts))
    return {"bytes": cached + T * hq * (4 * d + 4), "flops": 4 * hq * d * seen}


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Rows of keys and values with channels of different size, queries that make some rows
    sharp and others flat, the rotary tables of the new positions."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    starts, counts = _lengths(case)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float16)

    gain_k = torch.exp(0.5 * rand(hk, d).float())
    gain_v = torch.exp(0.4 * rand(hk, 1).float())

    def rows(gain, n):
        x = rand(n, hk, d)
        x *= gain.to(torch.float16)
        return x.view(n, hk * d)

    T = sum(counts)
    st = {"case": case, "starts": starts, "counts": counts, "scale": d ** -0.5}
    if case["op"] == "append":
        s0, _ = _spans(case)
        old = [s - z for s, z in zip(starts, s0)]  # tokens already in the first block
        st["old"] = old
        st["k_old"], st["v_old"] = rows(gain_k, sum(old)), rows(gain_v, sum(old))
        # rows as a fused q / k / v projection leaves them: one matrix, split by columns
        qkv = torch.cat([rand(T, hq * d), rows(gain_k, T), rows(gain_v, T)], dim=1)
        st["q"], st["k"], st["v"] = qkv.split([hq * d, hk * d, hk * d], dim=1)
        pos = torch.cat([torch.arange(s, s + n, device=dev) for s, n in zip(starts, counts)]).float()
        freq = 500000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float32) / d)
        ang = (pos[:, None] * freq).repeat(1, 2)
        st["cos"], st["sin"] = ang.cos().half(), ang.sin().half()
        return st
    L = sum(s + n for s, n in zip(starts, counts))
    st["k_all"], st["v_all"] = rows(gain_k, L), rows(gain_v, L)
    sharp = torch.exp2(2.0 * torch.rand(hq, 1, generator=g, device=dev) - 1.0)
    st["q"] = (rand(T, hq, d) * sharp.half()).view(T, hq * d)
    return st


def _index(lengths, width, dev):
    """Rows of a [batch, width] padded array that hold a ragged one's rows, in order."""
    return torch.cat([torch.arange(n, device=dev) + b * width for b, n in enumerate(lengths)])


def prepare(case, seed):
    st = _inputs(case, seed)
    (_own_cache if own else _plain_cache)(st)
    for name in ("k_all", "v_all", "k_old", "v_old"):  # they are in the cache now
        st.pop(name, None)
    return st


# ------------------------------------------------------------------ the framework's operators
def _own_cache(st):
    import __graft_entry__

    tko = __graft_entry__.load_package()
    c = st["case"]
    p = c["page"]
    ends = [s + n for s, n in zip(st["starts"], st["counts"])]
    cache = tko.PagedKVCache(max_seqs=c["batch"], num_pages=sum(-(-e // p) for e in ends), page_size=p,
                             kv_heads=c["kv_heads"], head_dim=c["dim"], max_pages=max(-(-e // p) for e in ends),
                             tier={"int8": tko.PrecisionTier.INT8, "fp8": tko.PrecisionTier.FP8,
                                   "fp16": tko.PrecisionTier.FP16}[c["tier"]])
    seqs = list(range(c["batch"]))
    for turn in range(max(-(-e // p) for e in ends)):  # pages handed out in turn, as lengths grow
        for b in seqs:
            if turn * p < ends[b]:
                cache.reserve(b, min(ends[b], (turn + 1) * p))
    st["cache"], st["step"] = cache, cache.step(seqs, st["starts"], st["counts"])
    if c["op"] == "append":
        s0, span = _spans(c)
        st["span"] = cache.step(seqs, s0, span)
        if sum(st["old"]):
            cache.append(st["k_old"], st["v_old"], cache.step(seqs, s0, st["old"]))
    else:
        cache.append(st["k_all"], st["v_all"], cache.step(seqs, [0] * c["batch"], ends))


def _run_own(st):
    cache, step = st["cache"], st["step"]
    if st["case"]["op"] == "append":
        q = cache.append(st["k"], st["v"], step, cos=st["cos"], sin=st["sin"], q=st["q"])
        k, v = cache.read(st["span"])
        return {"q": q, "k": k, "v": v}
    out, entropy = cache.attention(st["q"], step, st["scale"])
    return {"out": out, "entropy": entropy}


# ------------------------------------------------------------------ the plain form
def _quantise(x, tier):
    """x [..., blocks, page, kv heads, dim] fp32 -> (codes, scale of each block and head)."""
    amax = x.abs().amax(dim=(-3, -1), keepdim=True)
    s = torch.div(amax, torch.full_like(amax, CODE_MAX[tier]))
    y = torch.where(s > 0, x / s, torch.zeros_like(x))
    if tier == "int8":
        return torch.round(y).to(torch.int8), s
    return y.to(torch.float8_e4m3fn), s


def _pages_at(pages, at):
    """Pages at an index, 8-bit ones by their bytes."""
    return pages[at] if pages.dtype == torch.float16 else pages.view(torch.uint8)[at].view(pages.dtype)


def _plain_cache(st):
    """Pages of codes [page, token, kv head, dim], their scales, a table of pages, and the
    tokens of the incomplete last block (two buffers a sequence, by the block's parity)."""
    c = st["case"]
    dev = st["q"].device
    p, hk, d, B, tier = c["page"], c["kv_heads"], c["dim"], c["batch"], c["tier"]
    ends = [s + n for s, n in zip(st["starts"], st["counts"])]
    pages = [-(-e // p) for e in ends]
    width = max(pages)
    perm = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(1)).tolist()
    table = torch.zeros(B, width, dtype=torch.int64)
    for b, n in enumerate(pages):
        table[b, :n] = torch.tensor([perm.pop() for _ in range(n)])
    st["table"] = table.to(dev)
    st["start_t"], st["count_t"] = (torch.tensor(x, device=dev) for x in (st["starts"], st["counts"]))
    st["end_t"] = st["start_t"] + st["count_t"]
    kind = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "fp16": torch.float16}[tier]
    for name in ("k", "v"):
        st[name + "_pages"] = torch.zeros(sum(pages), p, hk, d, dtype=torch.float16, device=dev).to(kind)
        st[name + "_scale"] = torch.ones(sum(pages), 1, hk, 1, device=dev)
        st[name + "_open"] = torch.zeros(B, 2, p, hk, d, dtype=torch.float16, device=dev)
    parts = (st["old"], "_old") if c["op"] == "append" else (ends, "_all")
    first = [s // p for s in st["starts"]] if c["op"] == "append" else [0] * B
    at = 0
    for b, n in enumerate(parts[0]):
        for name in ("k", "v"):
            x = st[name + parts[1]][at:at + n].view(n, hk, d)
            full = n // p if tier != "fp16" else 0
            to = st["table"][b, first[b]:]
            if full:
                codes, s = _quantise(x[:full * p].float().view(full, p, hk, d), tier)
                st[name + "_pages"].view(torch.uint8)[to[:full]] = codes.view(torch.uint8)
                st[name + "_scale"][to[:full]] = s
            if tier == "fp16":
                for j in range(-(-n // p)):
                    part = x[j * p:(j + 1) * p]
                    st[name + "_pages"][to[j], :part.shape[0]] = part
            elif n > full * p:
                st[name + "_open"][b, (first[b] + full) % 2, :n - full * p] = x[full * p:]
        at += n
    if c["op"] == "append":
        s0, span = _spans(c)
        blocks = max(-(-n // p) for n in span)
        st["blocks"], st["first_t"] = blocks, torch.tensor([z // p for z in s0], device=dev)
        st["span_rows"] = _index(span, blocks * p, dev)
        offset = torch.tensor([0] + st["counts"][:-1], device=dev).cumsum(0)
        pos = st["first_t"][:, None] * p + torch.arange(blocks * p, device=dev)  # [B, blocks * page]
        st["is_new"] = (pos >= st["start_t"][:, None]) & (pos < st["end_t"][:, None])
        st["is_old"] = pos < st["start_t"][:, None]
        st["row_of"] = (offset[:, None] + pos - st["start_t"][:, None]).clamp(0, sum(st["counts"]) - 1)
    else:
        st["q_rows"] = _index(st["counts"], max(st["counts"]), dev)


def _rotate(x, cos, sin, heads, dim):
    x = x.float().view(x.shape[0], heads, dim)
    turned = torch.cat([-x[..., dim // 2:], x[..., :dim // 2]], dim=-1)
    return (x * cos.float()[:, None] + turned * sin.float()[:, None]).half()


def _run_append(st):
    c = st["case"]
    B, p, hq, hk, d, tier = c["batch"], c["page"], c["heads"], c["kv_heads"], c["dim"], c["tier"]
    nb = st["blocks"]
    q = _rotate(st["q"], st["cos"], st["sin"], hq, d).view(-1, hq * d)
    new = {"k": _rotate(st["k"], st["cos"], st["sin"], hk, d), "v": st["v"].reshape(-1, hk, d)}
    block = st["first_t"][:, None] + torch.arange(nb, device=q.device)  # [B, blocks]
    have = block * p < st["end_t"][:, None]  # blocks with tokens of the sequence
    page = st["table"].gather(1, block.clamp(max=st["table"].shape[1] - 1))
    full = have & ((block + 1) * p <= st["end_t"][:, None])
    parity = (st["first_t"] % 2)[:, None].expand(B, 1)
    out = {"q": q}
    seq = torch.arange(B, device=q.device)[:, None]
    for name in ("k", "v"):
        x = new[name][st["row_of"]]  # [B, blocks * page, kv heads, dim]
        if tier == "fp16":
            x = x.view(B, nb, p, hk, d)
            keep = st["is_new"].view(B, nb, p, 1, 1)
            pages = st[name + "_pages"]
            rows = torch.where(keep, x, pages[page])
            pages[page[have]] = rows[have]
            got = pages[page]
        else:
            before = torch.zeros_like(x)
            before[:, :p] = st[name + "_open"][seq, parity][:, 0]
            x = torch.where(st["is_new"][..., None, None], x, before)
            x = torch.where((st["is_new"] | st["is_old"])[..., None, None], x, torch.zeros_like(x))
            x = x.view(B, nb, p, hk, d)
            codes, s = _quantise(x.float(), tier)
            st[name + "_pages"].view(torch.uint8)[page[full]] = codes.view(torch.uint8)[full]
            st[name + "_scale"][page[full]] = s[full]
            last = have & ~full
            b_of, i_of = last.nonzero(as_tuple=True)
            st[name + "_open"][b_of, block[b_of, i_of] % 2] = x[b_of, i_of]
            value = (_pages_at(st[name + "_pages"], page).float() * st[name + "_scale"][page]).half()
            got = torch.where(full[..., None, None, None], value, x)
        out[name] = got.reshape(B * nb * p, hk * d)[st["span_rows"]]
    return out


def _run_attention(st):
    c = st["case"]
    B, p, hq, hk, d, tier = c["batch"], c["page"], c["heads"], c["kv_heads"], c["dim"], c["tier"]
    G, n = hq // hk, max(st["counts"])
    width = st["table"].shape[1]
    dev = st["q"].device
    q = torch.zeros(B * n, hq * d, device=dev)
    q[st["q_rows"]] = st["q"].float()
    q = q.view(B, n, hk, G, d).permute(0, 2, 1, 3, 4).reshape(B, hk, n * G, d)
    last = st["end_t"] // p  # the block that is not full
    cached = []
    for name in ("k", "v"):
        x = _pages_at(st[name + "_pages"], st["table"]).float()  # [B, width, page, kv heads, dim]
        if tier != "fp16":
            x *= st[name + "_scale"][st["table"]]
            open_ = st[name + "_open"][torch.arange(B, device=dev), last % 2].float()
            b_of = (last < width).nonzero().flatten()
            x[b_of, last[b_of]] = open_[b_of]
        cached.append(x.view(B, width * p, hk, d).permute(0, 2, 1, 3))
    k, v = cached
    x = torch.matmul(q, k.transpose(2, 3)) * st["scale"]  # [B, kv heads, n * G, tokens]
    limit = st["start_t"][:, None] + torch.arange(n, device=dev) + 1  # keys that a query sees
    limit = torch.minimum(limit, st["end_t"][:, None]).repeat_interleave(G, dim=1)
    seen = torch.arange(width * p, device=dev) < limit[:, None, :, None]
    x = torch.where(seen, x, torch.full_like(x, -torch.inf))
    x = x - x.amax(dim=-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(dim=-1, keepdim=True)
    weighted = torch.where(seen, e * x, torch.zeros_like(x)).sum(dim=-1, keepdim=True)
    entropy = torch.log(total) - weighted / total
    out = torch.matmul(e, v) / total
    out = out.view(B, hk, n, G, d).permute(0, 2, 1, 3, 4).reshape(B * n, hq * d)[st["q_rows"]]
    entropy = entropy.view(B, hk, n, G).permute(0, 2, 1, 3).reshape(B * n, hq)[st["q_rows"]]
    return {"out": out.half(), "entropy": entropy}


def run(st):
    if own:
        return _run_own(st)
    return _run_append(st) if st["case"]["op"] == "append" else _run_attention(st)


# ------------------------------------------------------------------ 64 bits
def _held(x, tier, p):
    """Rows x [n, kv heads, dim] (64 bits) of a sequence from a page's first token on, as the
    cache holds them: full pages by page and head, the rest as it is."""
    n, hk, d = x.shape
    full = n // p if tier != "fp16" else 0
    if not full:
        return x
    y = x[:full * p].view(full, p, hk, d)
    top = torch.linalg.vector_norm(y, math.inf, dim=(1, 3)).view(full, 1, hk, 1)
    # scale and quotient are fp32 numbers by definition: it says which way a tie goes
    unit = (torch.where(top > 0, top, 1.0) / CODE_MAX[tier]).float().double()
    y = (y / unit).float().double()
    # what a code steps by: 1 for integers; for e4m3 2^(e - 3) in [2^e, 2^(e + 1)), 2^-9 at the least
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3) if tier == "fp8" else 1.0
    y = torch.round(y / step) * step * unit
    return torch.cat([y.view(full * p, hk, d), x[full * p:]])


def exact(case, seed):
    st = _inputs(case, seed)
    p, hq, hk, d, tier = case["page"], case["heads"], case["kv_heads"], case["dim"], case["tier"]
    starts, counts = st["starts"], st["counts"]
    if case["op"] == "append":
        c, s = st["cos"].double()[:, None], st["sin"].double()[:, None]

        def turn(x, heads):
            x = x.double().view(-1, heads, d)
            a, b = x[..., :d // 2], x[..., d // 2:]
            lo = a * c[..., :d // 2] - b * s[..., :d // 2]
            hi = b * c[..., d // 2:] + a * s[..., d // 2:]
            return torch.cat([lo, hi], dim=-1)

        q = turn(st["q"], hq).reshape(-1, hq * d)
        # the cache takes fp16 keys: what is quantised is the rounded rotation
        k_new, v_new = turn(st["k"], hk).half().double(), st["v"].double().reshape(-1, hk, d)
        got = {"k": [], "v": []}
        at = was = 0
        for n, m in zip(counts, st["old"]):
            for name, new in (("k", k_new), ("v", v_new)):
                old = st[name + "_old"][was:was + m].double().view(m, hk, d)
                got[name].append(_held(torch.cat([old, new[at:at + n]]), tier, p).reshape(-1, hk * d))
            at, was = at + n, was + m
        return {"q": q, "k": torch.cat(got["k"]), "v": torch.cat(got["v"])}
    outs, ents = [], []
    at = row = 0
    for s, n in zip(starts, counts):
        L = s + n
        k = _held(st["k_all"][at:at + L].double().view(L, hk, d), tier, p)
        v = _held(st["v_all"][at:at + L].double().view(L, hk, d), tier, p)
        q = st["q"][row:row + n].double().view(n, hq, d)
        o = torch.empty(n, hq, d, dtype=torch.float64, device=q.device)
        e = torch.empty(n, hq, dtype=torch.float64, device=q.device)
        hidden = torch.arange(L, device=q.device)[None, :] > (s + torch.arange(n, device=q.device))[:, None]
        for h in range(hq):
            x = (q[:, h] @ k[:, h * hk // hq].T) * st["scale"]
            x.masked_fill_(hidden, -math.inf)
            w = torch.softmax(x, dim=-1)
            o[:, h] = w @ v[:, h * hk // hq]
            e[:, h] = -torch.special.xlogy(w, w).sum(dim=-1)
        outs.append(o.view(n, hq * d))
        ents.append(e)
        at, row = at + L, row + n
    return {"out": torch.cat(outs), "entropy": torch.cat(ents)}
