"""The paged KV cache (ee_paged_*, PagedKVCache) against plain implementations in 64 bits.

Tolerances, from the formats:
  * codes and scales: s = fp32(amax / top), code = rn(fp32(x / s)): the same IEEE operations in
    torch, so what ``read`` returns is compared bit for bit, fp16(code * s) included;
  * rotation: fp32 with at most three roundings (2^-24 each, of terms up to |x| + |rot|), then
    fp16: half an fp16 step of the result plus 2^-22 of the terms;
  * attention: keys and values are taken as held.  Scores are sums of exact products in fp32;
    their error 2^-22 sum |q k| scale adds to the logits.  P is rounded to fp16 relative to the
    row's reference (relative 2^-11), exp2 to 2^-21, and the output to fp16 (2^-11): together
    2^-10 + 2^-9 of sum p |v| is above all of it for logits up to about 30.  The entropy
    -sum p ln p: 2^-18 of 1 + its largest terms, i.e. of 1 + ln n + spread of the logits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TOP = {0: 127.0, 1: 448.0}


def _held(x, tier, P):
    """fp16 values [n, heads, d] -> what the cache stands for, in 64 bits (exact: code * s)."""
    n, h, d = x.shape
    full = n // P if tier != 2 else 0
    out = x.double()
    if full:
        y = x[:full * P].float().view(full, P, h, d)
        amax = y.abs().amax(dim=(1, 3), keepdim=True)
        s = torch.div(amax, torch.full_like(amax, TOP[tier]))
        z = torch.where(s > 0, torch.div(y, s), torch.zeros_like(y))
        code = torch.round(z) if tier == 0 else z.to(torch.float8_e4m3fn).float()
        out = torch.cat([(code.double() * s.double()).view(full * P, h, d), out[full * P:]])
    return out


def _rotate64(x, cos, sin, h, d):
    x, c, s = x.double().view(-1, h, d), cos.double()[:, None], sin.double()[:, None]
    rot = torch.cat([-x[..., d // 2:], x[..., :d // 2]], dim=-1)
    return x * c + rot * s, (x * c).abs() + (rot * s).abs()


def _attend64(q, k, v, start, scale):
    """One sequence: q [n, hq, d], k / v [L, hk, d] in 64 bits -> (out, entropy, sum p |v|, logit spread)."""
    n, hq, d = q.shape
    L, hk, _ = k.shape
    G = hq // hk
    x = torch.einsum("nhgd,lhd->hgnl", q.double().view(n, hk, G, d), k) * scale
    seen = torch.arange(L, device=q.device) <= start + torch.arange(n, device=q.device)[:, None]
    x = x.masked_fill(~seen, -math.inf)
    p = torch.softmax(x, dim=-1)
    o = torch.einsum("hgnl,lhd->nhgd", p, v).reshape(n, hq, d)
    a = torch.einsum("hgnl,lhd->nhgd", p, v.abs()).reshape(n, hq, d)
    ent = -torch.special.xlogy(p, p).sum(-1).permute(2, 0, 1).reshape(n, hq)
    return o, ent, a, x.masked_fill(~seen, 0).abs().max().item()


def _check(out, H, row, n, ref, hq, d):
    o, ent, a, spread = ref
    got = out[row:row + n].double().view(n, hq, d)
    assert torch.isfinite(got).all()
    worst = ((got - o).abs() - (2.0 ** -9 + 2.0 ** -10) * a - 2.0 ** -24).max().item()
    assert worst <= 0, worst
    L = 1.0 + math.log(max(2, o.shape[0] + 1e6)) + spread
    assert (H[row:row + n].double() - ent).abs().max().item() <= 2.0 ** -18 * L


def _data(g, dev, n, hk, d):
    k = torch.randn(n, hk * d, generator=g, device=dev) * torch.exp(0.5 * torch.randn(hk * d, generator=g, device=dev))
    v = torch.randn(n, hk * d, generator=g, device=dev)
    return k.half(), v.half()


def _cache(pkg, dev, ends, P, hk, d, tier, **kw):
    pages = [-(-max(e, 1) // P) for e in ends]
    return pkg.PagedKVCache(max_seqs=len(ends), num_pages=sum(pages) + 3, page_size=P, kv_heads=hk, head_dim=d,
                            max_pages=max(pages), tier=pkg.PrecisionTier(tier), device=dev, **kw)


def _ok(pkg):
    torch.cuda.synchronize()
    assert pkg._lib.device_check() == 0


@pytest.mark.parametrize("tier", [0, 1, 2])
@pytest.mark.parametrize("d,P,hk,hq", [(128, 16, 8, 32), (64, 32, 3, 9), (128, 64, 1, 1), (64, 128, 2, 10)])
@torch.no_grad()
def test_append_in_any_cut_gives_the_same_cache(pkg, cuda, tier, d, P, hk, hq):
    """The codes, scales and open rows bit for bit, from one append and from many."""
    g = torch.Generator(device=cuda).manual_seed(100 * tier + d + P)
    ends = [1, P - 1, P, P + 1, 3 * P + 5, 5 * P]
    data = [_data(g, cuda, e, hk, d) for e in ends]
    whole = _cache(pkg, cuda, ends, P, hk, d, tier)
    step = whole.step(range(len(ends)), counts=ends)
    whole.append(torch.cat([k for k, _ in data]), torch.cat([v for _, v in data]), step)
    cut = _cache(pkg, cuda, ends, P, hk, d, tier)
    sizes = [1, 2, P - 1, P, 7, 2 * P + 3]
    turn = 0
    while any(cut.lengths[b] < e for b, e in enumerate(ends)):
        at = list(cut.lengths)
        n = [min(sizes[(turn + b) % len(sizes)], e - a) for b, (e, a) in enumerate(zip(ends, at))]
        st = cut.step(range(len(ends)), counts=n)
        cut.append(torch.cat([k[a:a + m] for (k, _), a, m in zip(data, at, n)]),
                   torch.cat([v[a:a + m] for (_, v), a, m in zip(data, at, n)]), st)
        turn += 1
    got = [c.read(c.span(range(len(ends)), [0] * len(ends), ends)) for c in (whole, cut)]
    _ok(pkg)
    row = 0
    for e, (k, v) in zip(ends, data):
        for i, x in enumerate((k, v)):
            want = _held(x.view(e, hk, d), tier, P).half().view(e, hk * d)  # code * s is exact in 64 bits
            for c in got:
                assert torch.equal(c[i][row:row + e], want), (e, i)
        row += e
    # part of a span
    a = [e // 3 for e in ends]
    n = [e - x - (e > 2) for e, x in zip(ends, a)]
    k, v = cut.read(cut.span(range(len(ends)), a, n))
    full = got[1]
    at = [sum(ends[:b]) + a[b] for b in range(len(ends))]
    assert torch.equal(k, torch.cat([full[0][x:x + m] for x, m in zip(at, n)]))
    assert torch.equal(v, torch.cat([full[1][x:x + m] for x, m in zip(at, n)]))
    _ok(pkg)


@pytest.mark.parametrize("d,hk,hq", [(128, 8, 32), (64, 2, 6)])
@torch.no_grad()
def test_append_rotates_q_and_k(pkg, cuda, d, hk, hq):
    g = torch.Generator(device=cuda).manual_seed(d)
    n, P = 77, 32
    # rows of one fused projection, columns split: strides above the row's width
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g, device=cuda).half()
    q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
    ang = torch.rand(n, d, generator=g, device=cuda) * 6.3
    cos, sin = ang.cos().half(), ang.sin().half()
    c = _cache(pkg, cuda, [n], P, hk, d, 2)
    y = c.append(k, v, c.step([0], counts=[n]), cos=cos, sin=sin, q=q)
    kk, vv = c.read(c.span([0], [0], [n]))
    _ok(pkg)
    assert torch.equal(vv, v)
    for got, x, h in ((y, q, hq), (kk, k, hk)):
        want, terms = _rotate64(x, cos, sin, h, d)
        err = (got.double().view(n, h, d) - want).abs()
        step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -14))) - 10)
        assert (err - 0.5 * step - 2.0 ** -22 * terms).max().item() <= 0
    # in place, and without a table: a copy
    q2 = q.clone()
    c.append(k, v, c.step([0], starts=[0], counts=[n]), cos=cos, sin=sin, q=q2, out=q2)
    assert torch.equal(q2, y)
    z = c.append(k, v, c.step([0], starts=[0], counts=[n]), q=q)
    assert torch.equal(z, q)
    kk, _ = c.read(c.span([0], [0], [n]))
    assert torch.equal(kk, k)
    _ok(pkg)


@pytest.mark.parametrize("tier", [0, 1, 2])
@pytest.mark.parametrize("d,P,hk,hq", [(128, 16, 8, 32), (64, 32, 4, 4), (128, 64, 2, 14), (64, 128, 1, 8),
                                       (128, 32, 1, 24), (64, 16, 3, 9)])
@torch.no_grad()
def test_one_token_attention(pkg, cuda, tier, d, P, hk, hq):
    g = torch.Generator(device=cuda).manual_seed(7 * tier + d + hq)
    ends = [1, 2, P, P + 1, 15, 16, 17, 63, 64, 65, 300, 2 * P - 1, 4097]
    data = [_data(g, cuda, e, hk, d) for e in ends]
    c = _cache(pkg, cuda, ends, P, hk, d, tier)
    c.append(torch.cat([k for k, _ in data]), torch.cat([v for _, v in data]), c.step(range(len(ends)), counts=ends))
    q = (torch.randn(len(ends), hq * d, generator=g, device=cuda) * 1.5).half()
    st = c.step(range(len(ends)), starts=[e - 1 for e in ends])
    out, H = c.attention(q, st)
    again, H2 = c.attention(q, st, scale=d ** -0.5)
    _ok(pkg)
    assert torch.equal(out, again) and torch.equal(H, H2)  # the same bits every time
    for b, (e, (k, v)) in enumerate(zip(ends, data)):
        K, V = _held(k.view(e, hk, d), tier, P), _held(v.view(e, hk, d), tier, P)
        _check(out, H, b, 1, _attend64(q[b].view(1, hq, d), K, V, e - 1, d ** -0.5), hq, d)


@pytest.mark.parametrize("tier", [0, 1, 2])
@pytest.mark.parametrize("d,P,hk,hq", [(128, 16, 2, 8), (64, 32, 4, 4), (128, 64, 1, 7), (64, 128, 2, 6),
                                       (128, 128, 1, 40), (64, 64, 1, 3), (64, 16, 1, 160)])
@torch.no_grad()
def test_chunk_attention(pkg, cuda, tier, d, P, hk, hq):
    """Chunks from one token to several tiles, from position 0 and over a cache, one long one
    whose keys many CTAs share."""
    g = torch.Generator(device=cuda).manual_seed(11 * tier + d + hq)
    starts = [0, 0, 0, 1, 100, 127, 1000, 33, 9000]
    counts = [1, 5, 300, 64, 130, 129, 2, 257, 40]
    ends = [a + n for a, n in zip(starts, counts)]
    data = [_data(g, cuda, e, hk, d) for e in ends]
    c = _cache(pkg, cuda, ends, P, hk, d, tier)
    c.append(torch.cat([k for k, _ in data]), torch.cat([v for _, v in data]), c.step(range(len(ends)), counts=ends))
    q = (torch.randn(sum(counts), hq * d, generator=g, device=cuda) * 1.5).half()
    st = c.step(range(len(ends)), starts=starts, counts=counts)
    out, H = c.attention(q, st)
    again, H2 = c.attention(q, st)
    _ok(pkg)
    assert torch.equal(out, again) and torch.equal(H, H2)
    row = 0
    for a, n, e, (k, v) in zip(starts, counts, ends, data):
        K, V = _held(k.view(e, hk, d), tier, P), _held(v.view(e, hk, d), tier, P)
        _check(out, H, row, n, _attend64(q[row:row + n].view(n, hq, d), K, V, a, d ** -0.5), hq, d)
        row += n


@pytest.mark.parametrize("tier", [0, 1, 2])
@torch.no_grad()
def test_rows_that_see_nothing_and_holes(pkg, cuda, tier):
    """Sequences without new tokens, a sequence whose pages are not there (zeros), and a hole
    in the middle (skipped): the error word is set by the append alone."""
    P, hk, hq, d = 16, 2, 8, 64
    g = torch.Generator(device=cuda).manual_seed(tier)
    c = _cache(pkg, cuda, [96, 96, 96], P, hk, d, tier)
    ends = [70, 0, 64]
    data = [_data(g, cuda, e, hk, d) for e in ends]
    st = c.step([0, 1, 2], counts=ends)
    c.append(torch.cat([k for k, _ in data]), torch.cat([v for _, v in data]), st)
    _ok(pkg)
    q = torch.randn(2, hq * d, generator=g, device=cuda).half()
    st = c.step([0, 1, 2], starts=[69, 0, 63], counts=[1, 0, 1])
    before = c.attention(q, st)
    c.table[0, 2] = -1          # tokens 32 .. 47 of sequence 0
    c.table[2, :4] = 1 << 30    # no page of sequence 2 (outside the pool)
    out, H = c.attention(q, st)
    k, v = data[0]
    keep = torch.tensor([t for t in range(70) if not 32 <= t < 48], device=cuda)
    K, V = _held(k.view(70, hk, d), tier, P)[keep], _held(v.view(70, hk, d), tier, P)[keep]
    ref = _attend64(q[0].view(1, hq, d), K, V, len(keep) - 1, d ** -0.5)
    _check(out, H, 0, 1, ref, hq, d)
    _ok(pkg)
    assert not out[1].any() and not H[1].any()
    assert not torch.equal(before[0][0], out[0])
    kk, _ = c.read(c.span([0], [0], [70]))  # a hole reads as zeros
    assert not kk[32:48].any() and kk[48:64].any()
    with pytest.raises(RuntimeError, match="EE_ERR_DEVICE"):
        pkg._lib.device_check()
    c.append(k[:1], v[:1], c.step([0], starts=[40], counts=[1]))  # a token without a page
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="EE_ERR_DEVICE"):
        pkg._lib.device_check()
    # nothing at all to do
    out, H = c.attention(q[:0], c.step([1], starts=[0], counts=[0]))
    assert out.shape == (0, hq * d) and H.shape == (0, hq)
    assert c.append(k[:0], v[:0], c.step([1], counts=[0]), q=q[:0]).shape == (0, hq * d)
    _ok(pkg)


@pytest.mark.parametrize("tier", [0, 1, 2])
@pytest.mark.parametrize("n", [1, 3, 70])
@torch.no_grad()
def test_what_lies_past_the_tokens_does_not_matter(pkg, cuda, tier, n):
    """NaN and infinities in the unused part of pages and open blocks, and in other pages."""
    P, hk, hq, d, e = 32, 2, 8, 128, 150
    g = torch.Generator(device=cuda).manual_seed(tier)
    k, v = _data(g, cuda, e, hk, d)
    q = torch.randn(n, hq * d, generator=g, device=cuda).half()
    outs = []
    for fill in (0x00, 0xFF, 0x7C):
        c = pkg.PagedKVCache(max_seqs=3, num_pages=20, page_size=P, kv_heads=hk, head_dim=d, max_pages=8,
                             tier=pkg.PrecisionTier(tier), device=cuda)
        table = c.table.clone()
        c.memory.fill_(fill)  # every byte: NaN codes, NaN and infinite fp16 numbers and scales
        c.table.copy_(table)
        c.append(k, v, c.step([1], counts=[e]))
        outs.append(c.attention(q, c.step([1], starts=[e - n], counts=[n])))
    _ok(pkg)
    K, V = _held(k.view(e, hk, d), tier, P), _held(v.view(e, hk, d), tier, P)
    _check(*outs[0], 0, n, _attend64(q.view(n, hq, d), K, V, e - n, d ** -0.5), hq, d)
    for o in outs[1:]:
        assert torch.equal(o[0], outs[0][0]) and torch.equal(o[1], outs[0][1])


@pytest.mark.parametrize("tier", [0, 1, 2])
@torch.no_grad()
def test_extreme_values(pkg, cuda, tier):
    """Blocks of zeros, of fp16's largest and smallest numbers, scales that differ by many
    powers of two between blocks; a value that is not finite gives NaN, not a number."""
    P, hk, hq, d = 16, 1, 4, 64
    g = torch.Generator(device=cuda).manual_seed(3)
    e = 6 * P + 5
    k, v = _data(g, cuda, e, hk, d)
    v[:P] = 0
    k[P:2 * P] = 0
    v[2 * P:3 * P] = torch.where(v[2 * P:3 * P] > 0, 65504.0, -65504.0).half()
    v[3 * P:4 * P] = (v[3 * P:4 * P].float() * 2.0 ** -20).half()
    v[5 * P:6 * P] = (v[5 * P:6 * P].float() * 2.0 ** 6).half()
    for lo in (0, 3 * P):  # with and without the large block
        n = e - lo
        c = _cache(pkg, cuda, [n, n], P, hk, d, tier)
        c.append(torch.cat([k[lo:], k[lo:]]), torch.cat([v[lo:], v[lo:]]), c.step([0, 1], counts=[n, n]))
        q = torch.randn(2, hq * d, generator=g, device=cuda).half()
        out, H = c.attention(q, c.step([0, 1], starts=[n - 1, n - 1]))
        kk, vv = c.read(c.span([0], [0], [n]))
        _ok(pkg)
        assert torch.equal(vv, _held(v[lo:].view(n, hk, d), tier, P).half().view(n, -1))
        K, V = _held(k[lo:].view(n, hk, d), tier, P), _held(v[lo:].view(n, hk, d), tier, P)
        for b in range(2):
            _check(out, H, b, 1, _attend64(q[b].view(1, hq, d), K, V, n - 1, d ** -0.5), hq, d)
    for bad in (math.nan, math.inf):
        for x in (0, 1):
            kv = [k[3 * P:].clone(), v[3 * P:].clone()]
            kv[x][P + 3, 5] = bad
            n = e - 3 * P
            c = _cache(pkg, cuda, [n], P, hk, d, tier)
            c.append(*kv, c.step([0], counts=[n]))
            q = torch.rand(1, hq * d, generator=g, device=cuda).half()
            out, H = c.attention(q, c.step([0], starts=[n - 1]))
            _ok(pkg)
            assert not torch.isfinite(out.float().view(hq, d)).all(dim=1).any()


@pytest.mark.parametrize("tier", [0, 1])
@torch.no_grad()
def test_tokens_taken_back(pkg, cuda, tier):
    """Drafted tokens are cut off again: the cache is what it would be without them."""
    P, hk, d = 16, 2, 64
    g = torch.Generator(device=cuda).manual_seed(tier)
    k, v = _data(g, cuda, 120, hk, d)
    kd, vd = _data(g, cuda, 120, hk, d)  # the drafted tokens
    c = _cache(pkg, cuda, [120], P, hk, d, tier)
    rng = torch.Generator().manual_seed(5)
    n = 0
    while n < 100:
        draft = 1 + int(torch.randint(P, (1,), generator=rng))
        keep = int(torch.randint(draft + 1, (1,), generator=rng))
        kk, vv = torch.cat([k[n:n + keep], kd[:draft - keep]]), torch.cat([v[n:n + keep], vd[:draft - keep]])
        c.append(kk, vv, c.step([0], counts=[draft]))
        n += keep
        c.truncate(0, n)
    got = c.read(c.span([0], [0], [n]))
    _ok(pkg)
    for a, x in zip(got, (k, v)):
        assert torch.equal(a, _held(x[:n].view(n, hk, d), tier, P).half().view(n, -1))
    with pytest.raises(RuntimeError, match="can be cut"):
        c.truncate(0, 3 * P + 1)
    c.truncate(0, 3 * P)
    with pytest.raises(RuntimeError, match="can be cut"):
        c.truncate(0, 2 * P + 5)
    c.append(k[3 * P:3 * P + 20], v[3 * P:3 * P + 20], c.step([0], counts=[20]))
    c.truncate(0, 3 * P + 4)
    assert c.lengths[0] == 3 * P + 4


@torch.no_grad()
def test_pages_are_reused_and_many_sequences(pkg, cuda):
    """A pool that sequences share in turn, and a step of more sequences than a warp has lanes."""
    P, hk, hq, d, B = 16, 2, 4, 64, 201
    g = torch.Generator(device=cuda).manual_seed(1)
    c = pkg.PagedKVCache(max_seqs=B + 1, num_pages=3 * B, page_size=P, kv_heads=hk, head_dim=d, max_pages=3,
                         device=cuda)
    for turn in range(2):
        seqs = list(range(B)) if turn == 0 else list(range(B, 0, -1))
        ends = [1 + (7 * b + turn) % 48 for b in range(B)]
        k, v = _data(g, cuda, sum(ends), hk, d)
        c.append(k, v, c.step(seqs, counts=ends))
        q = torch.randn(B, hq * d, generator=g, device=cuda).half()
        out, H = c.attention(q, c.step(seqs, starts=[e - 1 for e in ends]))
        _ok(pkg)
        row = 0
        for b, e in enumerate(ends):
            K, V = _held(k[row:row + e].view(e, hk, d), 0, P), _held(v[row:row + e].view(e, hk, d), 0, P)
            _check(out, H, b, 1, _attend64(q[b].view(1, hq, d), K, V, e - 1, d ** -0.5), hq, d)
            row += e
        used = sum(-(-e // P) for e in ends)
        assert c.free_pages == 3 * B - used
        for s in seqs:
            c.release(s)
        assert c.free_pages == 3 * B
    with pytest.raises(RuntimeError, match="more than 3 pages"):
        c.reserve(0, 3 * P + 1)
    for s in range(B):
        c.reserve(s, 3 * P)
    with pytest.raises(RuntimeError, match="full"):
        c.reserve(B, 1)


@torch.no_grad()
def test_other_streams_and_graph(pkg, cuda):
    """Calls on two streams use workspaces of their own; a captured step replays."""
    P, hk, hq, d, e = 64, 8, 32, 128, 3000
    g = torch.Generator(device=cuda).manual_seed(2)
    k, v = _data(g, cuda, e, hk, d)
    c = _cache(pkg, cuda, [e], P, hk, d, 0)
    c.append(k, v, c.step([0], counts=[e]))
    st = c.step([0], starts=[e - 1])
    qs = [torch.randn(1, hq * d, generator=g, device=cuda).half() for _ in range(2)]
    want = [c.attention(q, st) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for i in (0, 1):  # workspaces made before the streams run side by side
        with torch.cuda.stream(streams[i]):
            streams[i].wait_stream(torch.cuda.default_stream())
            c.attention(qs[i], st)
    torch.cuda.synchronize()
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.attention(qs[i], st))
    torch.cuda.synchronize()
    for i in (0, 1):
        for o, H in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(H, want[i][1])
    q, out = qs[0].clone(), torch.empty_like(qs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        c.attention(q, st, out=out)
    q.copy_(qs[1])
    graph.replay()
    _ok(pkg)
    assert torch.equal(out, want[1][0])


@torch.no_grad()
def test_offsets_past_32_bits(pkg, cuda):
    """Pages whose bytes lie past 4 GB of the pool."""
    P, hk, hq, d, e = 128, 8, 8, 128, 700
    g = torch.Generator(device=cuda).manual_seed(4)
    for tier in (0, 2):
        c = pkg.PagedKVCache(max_seqs=1, num_pages=18000 if tier == 0 else 9000, page_size=P, kv_heads=hk, head_dim=d,
                             max_pages=8, tier=pkg.PrecisionTier(tier), device=cuda)
        c._free.reverse()  # the pool's last pages first
        k, v = _data(g, cuda, e, hk, d)
        c.append(k, v, c.step([0], counts=[e]))
        assert int(c.table[0, 0]) == c.num_pages - 1
        q = torch.randn(3, hq * d, generator=g, device=cuda).half()
        out, H = c.attention(q, c.step([0], starts=[e - 3], counts=[3]))
        _ok(pkg)
        K, V = _held(k.view(e, hk, d), tier, P), _held(v.view(e, hk, d), tier, P)
        _check(out, H, 0, 3, _attend64(q.view(3, hq, d), K, V, e - 3, d ** -0.5), hq, d)
        del c


@torch.no_grad()
def test_steps_that_do_not_fit_the_cache_are_left_alone(pkg, cuda):
    """Device arrays that name what the cache does not have: the error word, and no write."""
    P, hk, hq, d = 16, 1, 2, 64
    g = torch.Generator(device=cuda).manual_seed(6)
    k, v = _data(g, cuda, 8, hk, d)
    q = torch.randn(8, hq * d, generator=g, device=cuda).half()
    for i, value in ((0, 5), (0, -1), (1, -4), (1, 40), (2, 4), (3, 1), (4, 9)):
        c = pkg.PagedKVCache(max_seqs=2, num_pages=4, page_size=P, kv_heads=hk, head_dim=d, max_pages=2,
                             tier=pkg.PrecisionTier.INT8, device=cuda)
        st = c.step([0], counts=[8])  # arrays: seq, start, length, cu[0], cu[1]
        before = c.memory.clone()
        if (i, value) == (3, 1):
            value = -2
        st.arrays[i] = value
        c.append(k, v, st)
        out, H = c.attention(q, st)
        c.read(st)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="EE_ERR_DEVICE"):
            pkg._lib.device_check()
        same = c.memory == before
        assert bool(same.all())


@torch.no_grad()
def test_attention_of_earlier_positions(pkg, cuda):
    """Queries at positions before the sequence's end: its later tokens are cached and not seen."""
    P, hk, hq, d, e = 32, 2, 8, 128, 500
    g = torch.Generator(device=cuda).manual_seed(8)
    k, v = _data(g, cuda, e, hk, d)
    for tier in (0, 2):
        c = _cache(pkg, cuda, [e], P, hk, d, tier)
        c.append(k, v, c.step([0], counts=[e]))
        for start, n in ((37, 1), (63, 3), (100, 90)):
            q = torch.randn(n, hq * d, generator=g, device=cuda).half()
            out, H = c.attention(q, c.span([0], [start], [n]))
            _ok(pkg)
            K, V = _held(k.view(e, hk, d), tier, P), _held(v.view(e, hk, d), tier, P)
            _check(out, H, 0, n, _attend64(q.view(n, hq, d), K, V, start, d ** -0.5), hq, d)


@torch.no_grad()
def test_workspace_after_an_error(pkg, cuda):
    """After device_check reported, the workspace's head is zeroed before its next use."""
    P, hk, hq, d, e = 16, 2, 8, 64, 3000
    g = torch.Generator(device=cuda).manual_seed(9)
    k, v = _data(g, cuda, e, hk, d)
    c = _cache(pkg, cuda, [e], P, hk, d, 1)
    c.append(k, v, c.step([0], counts=[e]))
    q = torch.randn(1, hq * d, generator=g, device=cuda).half()
    st = c.step([0], starts=[e - 1])
    want = c.attention(q, st)
    (ws, _), = c._ws.values()
    head = pkg.load_library().ee_paged_workspace_head_bytes()
    torch.cuda.synchronize()
    assert not ws[:head].any()
    ws[:head] = 1  # as a kernel that gave up might leave it
    st.arrays[0] = 7  # no such sequence: the error word
    c.read(st)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="EE_ERR_DEVICE"):
        pkg._lib.device_check()
    st.arrays[0] = 0
    got = c.attention(q, st)
    _ok(pkg)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tier", [0, 2])
@torch.no_grad()
def test_rows_before_the_first_sequence(pkg, cuda, tier):
    """cu[0] above zero: the rows before it belong to nobody and are neither read nor written."""
    P, hk, hq, d, pad, e = 16, 2, 4, 64, 70, 45
    g = torch.Generator(device=cuda).manual_seed(10)
    k, v = _data(g, cuda, pad + e, hk, d)
    c = _cache(pkg, cuda, [e], P, hk, d, tier)
    st = pkg.PagedStep([0], [0], [pad + e], [e], cuda)
    st.arrays[3] = pad  # seq, start, length, cu[0], cu[1]
    c.reserve(0, e)
    c._upload()
    c.append(k, v, st)
    q = torch.randn(pad + e, hq * d, generator=g, device=cuda).half()
    out = torch.full((pad + e, hq * d), 7.0, dtype=torch.float16, device=cuda)
    _, H = c.attention(q, st, out=out)
    kk, vv = c.read(st)
    _ok(pkg)
    assert bool((out[:pad] == 7.0).all())
    K, V = _held(k[pad:].view(e, hk, d), tier, P), _held(v[pad:].view(e, hk, d), tier, P)
    assert torch.equal(kk[pad:], K.half().view(e, -1)) and torch.equal(vv[pad:], V.half().view(e, -1))
    _check(out, H, pad, e, _attend64(q[pad:].view(e, hq, d), K, V, 0, d ** -0.5), hq, d)
