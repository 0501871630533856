"""GPU: the paged cache of 8 bits with a scale for each block of tokens and head
(KVCache with scales [pages, blocks, heads]) against plain 64-bit forms, and its
refusals.

Tolerances (derived, per element): a rotated key is off by 2^-20 (|a| + |b|)
(tests of the 16-bit cache); a value is exact.  A scale is a power of two, so
the division is exact and one rounding follows: half a step of E4M3 (2^-4
relative, 2^-10 near zero), or 1/2 of an integer.  A scale is the one that the 64-bit
form needs, or, where the largest element's error reaches a power of two times the
type's largest, that of either side.  attend: as for the 16-bit
cache, whose bound on scores holds with one more product (the scale,
2^-24 of the score, within its 16 extra steps); with scores of any size a weight is off by
exp(2 e) - 1 (2 e where e is small); a weight times its part of the
largest scale is off by one more rounding (within the 2^-10 of sum p |v|), and the FP16 pair by
2^-40 of a weight of 1, which an element gets none of only where the heaviest tokens hold zero."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def half_step(kind, exact):
    if kind == "int8":
        return torch.full_like(exact, 0.5)
    tiny = {"bf16": 0.0, "fp16": 2.0 ** -25, "fp32": 0.0, "e4m3": 2.0 ** -10}[kind]
    return torch.finfo(DT[kind]).eps / 2 * exact.abs() + tiny


def nhd(t, layout):
    return t if layout == "nhd" else t.transpose(1, 2)


def raw(t):
    return t.view(torch.uint8)


class Cache:
    """Cache tensors of random elements, scales of `order` in memory, and the KVCache."""

    def __init__(self, g, kind, pages, page, block, heads, dim, layout="nhd", order=(0, 1, 2), spread=2):
        shape = (pages, page, heads, dim) if layout == "nhd" else (pages, heads, page, dim)
        self.kind, self.page, self.block, self.layout = kind, page, block, layout
        x = [torch.randn(shape, generator=g, device=DEV).mul_(TOP[kind] / 4).clamp_(-TOP[kind], TOP[kind]) for _ in range(2)]
        self.k, self.v = (t.round().to(torch.int8) if kind == "int8" else t.to(DT[kind]) for t in x)
        logical = (pages, page // block, heads)
        back = [order.index(i) for i in range(3)]
        self.ks, self.vs = (torch.exp2(torch.randint(-8, -8 + 2 * spread, [logical[i] for i in order], generator=g, device=DEV)
                                       .float()).permute(back) for _ in range(2))
        self.c = xg.KVCache(self.k, self.v, k_scale=self.ks, v_scale=self.vs, layout=layout)

    def stands_for(self, which):
        """FP64 [pages, page, heads, dim]."""
        t, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        x = nhd(t, self.layout).double()
        return x * s.double().repeat_interleave(self.block, 1)[..., None]


def table_of(g, lens, page, spare=2, slack=0):
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need)) + slack), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, total


# ------------------------------------------------------------------ append
def rope64(x, pos, inv, interleaved, scale=1.0):
    """(rotated, |a| + |b|) in 64 bits."""
    half = inv.numel()
    ang = pos.double()[:, None] * inv.double()
    c, s = ang.cos()[:, None] * scale, ang.sin()[:, None] * scale
    x = x.double()
    out, mag = x.clone(), torch.zeros_like(x)
    ia = torch.arange(half, device=DEV) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * scale
    return out, mag


def needed(high, top):
    """The least power of two s >= 2^-60 with high <= top s."""
    if high <= 0:
        return 2.0 ** -60
    e = math.ceil(math.log2(high / top))
    while high > top * 2.0 ** e:
        e += 1
    while high <= top * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** max(e, -60)


def check_half(cache, which, before, had, new, mag, places):
    """One half of a cache after an append: `before` and `had` are copies of its
    bytes and scales, `new` [tokens, heads, dim] what was written (with the error
    bound 2^-20 mag) at `places` [(page, place)]."""
    t, s = (cache.k, cache.ks) if which == "k" else (cache.v, cache.vs)
    top, kind, B = TOP[cache.kind], cache.kind, cache.block
    got, old = nhd(t, cache.layout), nhd(before, cache.layout).clone()
    want_s = had.clone()
    blocks = {}
    for i, (page, place) in enumerate(places):
        blocks.setdefault((page, place // B), []).append((place % B, i))
    for (page, block), items in blocks.items():
        first = min(p for p, _ in items)
        at = torch.tensor([i for _, i in items], device=DEV)
        size, err = new[at].abs(), 2.0 ** -20 * mag[at]
        size = torch.where(torch.isfinite(size), size, torch.zeros_like(size)).nan_to_num()
        most, least = (size + err).amax((0, 2)), (size - err).amax((0, 2))
        for h in range(new.shape[1]):
            scale, earlier = float(s[page, block, h]), float(had[page, block, h])
            ok = {needed(float(most[h]), top), needed(max(0.0, float(least[h])), top)}
            if first:
                ok = {max(x, earlier) for x in ok}
            assert scale in ok, (which, page, block, h, scale, ok, first)
            want_s[page, block, h] = scale
            if first and scale > earlier:  # the earlier places, rounded again
                rows = old[page, block * B:block * B + first, h].float() * (earlier / scale)
                rows = rows.round().to(torch.int8) if kind == "int8" else rows.to(DT[kind])
                raw(old)[page, block * B:block * B + first, h] = raw(rows)
            for place, i in items:
                x = new[i, h] / scale
                have = got[page, block * B + place, h].double()
                bad = (have - x.clamp(-top, top)).abs() > half_step(kind, x.clamp(-top, top)) + 2.0 ** -20 * mag[i, h] / scale
                assert not (bad & ~x.isnan()).any(), (which, page, block, place, h)
                raw(old)[page, block * B + place, h] = raw(got)[page, block * B + place, h]
    assert torch.equal(raw(got), raw(old))  # nothing else was written
    assert torch.equal(s, want_s)


def run_append(cache, table, seq, index, kn, vn, pos=None, inv=None, interleaved=False, rot_scale=1.0, q=None, q_out=None,
               want_status=0, **more):
    before = [raw(cache.k).clone().view(cache.k.dtype), raw(cache.v).clone().view(cache.v.dtype)]
    had = [cache.ks.clone(), cache.vs.clone()]
    cache.c.append(kn, vn, table, index, seq=seq, positions=pos, inv_freq=inv, rot_scale=rot_scale, interleaved=interleaved, q=q,
                   q_out=q_out, **more)
    assert cache.c.status() == want_status
    owner = seq if seq is not None else torch.arange(len(index), device=DEV)
    live = [t for t in range(len(index)) if int(owner[t]) >= 0 and int(index[t]) >= 0]
    places = [(int(table[int(owner[t]), int(index[t]) // cache.page]), int(index[t]) % cache.page) for t in live]
    keys, mag = rope64(kn, index if pos is None else pos, inv if inv is not None else torch.empty(0, device=DEV), interleaved, rot_scale)
    check_half(cache, "k", before[0], had[0], keys[live], mag[live], places)
    check_half(cache, "v", before[1], had[1], vn.double()[live], torch.zeros_like(mag[live]), places)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dim,rot,interleaved,q_heads,kv_heads", [
    (128, 128, False, 32, 8), (64, 64, True, 6, 3), (80, 32, False, 5, 5), (256, 256, True, 4, 1),
    (96, 20, True, 3, 3), (16, 6, False, 2, 1), (192, 64, False, 7, 7), (64, 0, False, 4, 2)])
@pytest.mark.parametrize("kind,cache", [("bf16", "e4m3"), ("fp16", "int8"), ("fp32", "e4m3"), ("fp32", "int8")])
def test_append_matches_64_bits(dim, rot, interleaved, q_heads, kv_heads, kind, cache):
    for layout, page, block, n in (("nhd", 16, 16, 37), ("hnd", 12, 3, 1), ("nhd", 4, 1, 9), ("hnd", 64, 64, 150)):
        g = gen(dim + n)
        S = min(n, 4)
        counts = [n // S + (i < n % S) for i in range(S)]
        first = [3 * i for i in range(S)]
        table, pages = table_of(g, [f + c for f, c in zip(first, counts)], page)
        c = Cache(g, cache, pages, page, block, kv_heads, dim, layout, order=(2, 0, 1) if n % 2 else (0, 1, 2))
        seq = [i for i in range(S) for _ in range(counts[i])]
        index = ints([first[i] + j for i in range(S) for j in range(counts[i])])
        pos = index + torch.tensor([0, 1048575, 77, 2 ** 31 - 300], dtype=torch.int64, device=DEV)[torch.tensor(seq, device=DEV)].to(torch.int32)
        if n > 3:  # padding at a sequence's end
            seq[counts[0] - 1] = -1
        seq = ints(seq)
        inv = (10000.0 ** (-torch.arange(rot // 2, device=DEV, dtype=torch.float64) / max(1, rot // 2))).float()
        qn, kn, vn = (torch.randn(n, h, dim, generator=g, device=DEV).to(DT[kind]) for h in (q_heads, kv_heads, kv_heads))
        kn[n // 2:] *= 4.0  # so that scales rise inside a block of a later call too
        q_out = torch.full_like(qn, 7.0)
        run_append(c, table, seq, index, kn, vn, pos, inv if rot else None, interleaved, 1.25, qn, q_out)
        want, mag = rope64(qn, pos, inv, interleaved, 1.25)
        live = seq >= 0
        assert ((q_out.double() - want).abs() <= half_step(kind, want) + 2.0 ** -20 * mag)[live].all()
        assert (q_out[~live] == 7.0).all()  # padding rows are left alone
        c.c.close()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("block,page", [(16, 16), (8, 32), (1, 8), (48, 48)])
def test_blocks_grow_token_by_token(kind, block, page):
    """One token a call, growing and shrinking: scales rise and stay, earlier
    elements are rounded again, a new block begins anew."""
    g = gen(block)
    S, n = 3, 70
    start = [0, 5, 31]
    table, pages = table_of(g, [s + n for s in start], page)
    c = Cache(g, kind, pages, page, block, 2, 64)
    for t in range(n):
        size = 2.0 ** float(torch.randint(-6, 7, (1,), generator=g, device=DEV))
        kn, vn = (torch.randn(S, 2, 64, generator=g, device=DEV).mul_(size).to(torch.bfloat16) for _ in range(2))
        if t % 9 == 0:
            kn[:, 0] = 0.0
        run_append(c, table, None, ints([s + t for s in start]), kn, vn)
    c.c.close()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_in_parts_equals_the_elements_rounded_again(kind):
    """A prompt in one call, and in pieces that end inside blocks: the same
    scales, and elements that differ only by the second rounding."""
    g = gen(3)
    n, H, D, page, block = 200, 3, 80, 64, 32
    table, pages = table_of(g, [n], page)
    kn, vn = (torch.randn(n, H, D, generator=g, device=DEV).to(torch.float16) for _ in range(2))
    caches = [Cache(gen(9), kind, pages, page, block, H, D) for _ in range(2)]
    seq, index = torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    caches[0].c.append(kn, vn, table, index, seq=seq)
    at = 0
    for step in (1, 30, 1, 33, 64, 5, 66):
        caches[1].c.append(kn[at:at + step], vn[at:at + step], table, index[at:at + step], seq=seq[at:at + step])
        at += step
    assert at == n and caches[0].c.status() == 0 and caches[1].c.status() == 0
    rows = table[0, torch.arange(n, device=DEV) // page].long(), torch.arange(n, device=DEV) % page
    for which in "kv":
        a, b = (x.stands_for(which)[rows] for x in caches)
        s = (caches[0].ks if which == "k" else caches[0].vs)[rows[0], rows[1] // block].double()[..., None]
        s1 = (caches[1].ks if which == "k" else caches[1].vs)[rows[0], rows[1] // block].double()[..., None]
        assert torch.equal(s, s1)
        step = half_step(kind, torch.maximum(a.abs(), b.abs()) / s) * s
        assert ((a - b).abs() <= 2 * step).all()
    for x in caches:
        x.c.close()


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_append_strides_in_place_and_sliced_cache(layout):
    g = gen(5)
    n, QH, H, D, page = 21, 4, 2, 64, 8
    table, pages = table_of(g, [n], page)
    shape = (pages, 2, page, H, D) if layout == "nhd" else (pages, 2, H, page, D)
    both = torch.zeros(shape, dtype=torch.int8, device=DEV)
    scales = torch.zeros(pages, 2, 2, H, 2, device=DEV)  # two blocks a page, strided
    c = xg.KVCache(both[:, 0], both[:, 1], k_scale=scales[:, 0, :, :, 0], v_scale=scales[:, 1, :, :, 1], layout=layout)
    for shift in (1, 8):  # odd alignment, and 16-byte pieces
        packed = torch.randn(n, (QH + 2 * H) * D + 8, generator=g, device=DEV).to(torch.bfloat16)
        q, k, v = (t.unflatten(1, (-1, D)) for t in packed[:, shift:shift + (QH + 2 * H) * D].split([QH * D, H * D, H * D], dim=1)) \
            if shift == 1 else (t.unflatten(1, (-1, D)) for t in packed[:, 8:8 + (QH + 2 * H) * D].split([QH * D, H * D, H * D], dim=1))
        before, q0 = packed.clone(), q.clone()
        index = torch.arange(n, dtype=torch.int32, device=DEV)
        inv = (10000.0 ** (-torch.arange(D // 2, device=DEV) / (D // 2))).float()
        c.append(k, v, table, index, seq=torch.zeros_like(index), inv_freq=inv, q=q)
        assert c.status() == 0
        want, mag = rope64(q0, index, inv, False)
        assert ((q.double() - want).abs() <= half_step("bf16", want) + 2.0 ** -20 * mag).all()
        assert torch.equal(packed[:, :shift], before[:, :shift]) and torch.equal(packed[:, shift + QH * D:], before[:, shift + QH * D:])
        pg, pl = table[0, index.long() // page].long(), index.long() % page
        for half, s, want in ((both[:, 0], scales[:, 0, :, :, 0], rope64(k, index, inv, False)[0]), (both[:, 1], scales[:, 1, :, :, 1], v.double())):
            unit = s[pg, pl // 4].double()[..., None]
            assert ((nhd(half, layout)[pg, pl].double() * unit - want).abs() <= (0.5 + 2.0 ** -8) * unit).all()
        assert (scales[:, 0, :, :, 1] == 0).all() and (scales[:, 1, :, :, 0] == 0).all()
    c.close()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_special_values(kind):
    g = gen(6)
    table, pages = table_of(g, [4], 4)
    c = Cache(g, kind, pages, 4, 4, 1, 16)
    x = torch.zeros(4, 1, 16, device=DEV)
    x[0, 0, :6] = torch.tensor([3.0, -1.0, float("nan"), float("inf"), -0.0, -float("inf")])
    x[1, 0, 0] = 1e-42
    x[3, 0, 15] = 440.0 if kind == "e4m3" else 126.0
    c.c.append(x, x, table, torch.arange(4, dtype=torch.int32, device=DEV), seq=torch.zeros(4, dtype=torch.int32, device=DEV))
    page, top = int(table[0, 0]), TOP[kind]
    assert float(c.ks[page, 0, 0]) == 1.0 == float(c.vs[page, 0, 0])
    got = c.v[page, :, 0].float()
    assert got[0, :2].tolist() == [3.0, -1.0] and got[0, 3:6].tolist() == [top, 0.0, -top]
    assert got[3, 15] == (448.0 if kind == "e4m3" else 126.0)  # (E4M3's steps are 32 there: 440 rounds to 448)
    if kind == "e4m3":
        assert math.isnan(got[0, 2]) and c.c.status() == 0
    else:
        assert got[0, 2] == 0 and c.c.status() == 1
    # nothing but zeros: the least scale; the largest finite number: one that holds it
    zero = torch.zeros(1, 1, 16, device=DEV)
    c.c.append(zero, zero, table, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert float(c.ks[page, 0, 0]) == 2.0 ** -60 and (c.k[page, 0].float() == 0).all()
    big = torch.full((1, 1, 16), torch.finfo(torch.float32).max, device=DEV)
    c.c.append(big, big, table, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert float(c.ks[page, 0, 0]) == 2.0 ** (120 if kind == "e4m3" else 122)
    assert float(c.k[page, 0, 0, 0].float()) == (256.0 if kind == "e4m3" else 64.0)  # (2^128 less half a step)
    c.c.close()


def test_bad_pages_and_disorder_are_reported():
    g = gen(7)
    page, block = 8, 4
    table, pages = table_of(g, [16, 16], page)
    c = Cache(g, "e4m3", pages, page, block, 2, 32)
    table[1, 1] = pages
    table[0, 1] = -5
    new = torch.randn(5, 2, 32, generator=g, device=DEV).to(torch.bfloat16)
    q = torch.randn(5, 2, 32, generator=g, device=DEV).to(torch.bfloat16)
    k0, v0, ks0 = raw(c.k).clone(), raw(c.v).clone(), c.ks.clone()
    # past the table's columns, a sequence past its rows, a bad page, a negative page, padding
    q_out = torch.full_like(q, 3.0)
    c.c.append(new, new, table, ints([16, 0, 8, 9, 2]), seq=ints([0, 2, 1, 0, -1]), q=q, q_out=q_out)
    assert c.c.status() == 1 and c.c.status() == 0
    assert torch.equal(raw(c.k), k0) and torch.equal(raw(c.v), v0) and torch.equal(c.ks, ks0) and (q_out == 3.0).all()
    # an index that goes back, one that jumps, a sequence that comes again
    for index, seq in (([1, 0, 2, 3, 4], [0, 0, 0, 0, 0]), ([0, 2, 3, 4, 5], [0] * 5), ([0, 1, 0, 2, 3], [0, 0, 1, 0, 0])):
        c.c.append(new, new, table, ints(index), seq=ints(seq), q=q.clone())
        assert c.c.status() == 1
    # padding between sequences is fine, marked by either, before or behind the tokens
    for index, seq in (([0, 1, 0, 0, 1], [0, 0, -1, 1, 1]), ([-1, 5, 6, -7, 3], [0, 0, 0, 1, 1]), ([5, 6, -1, 3, -1], [0, 0, 0, 1, 1])):
        c.c.append(new, new, table, ints(index), seq=ints(seq))
        assert c.c.status() == 0
    # but not between a sequence's tokens
    c.c.append(new, new, table, ints([5, -1, 6, 0, 1]), seq=ints([0, 0, 0, 1, 1]))
    assert c.c.status() == 1
    c.c.append(new[:0], new[:0], table, ints([]))
    assert c.c.status() == 0
    c.c.close()


# ------------------------------------------------------------------ attend
def attend64(q, k, v, lens, table, page, scale, window=0, softcap=0.0):
    """(out, lse, tolerance before rounding, lse's) in 64 bits; k, v are FP64
    [pages, page, heads, dim]."""
    S, Q, D = q.shape
    H = k.shape[2]
    out = torch.zeros(S, Q, D, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    lse = torch.full((S, Q), -math.inf, dtype=torch.float64, device=DEV)
    tol_lse = torch.zeros_like(lse)
    for i, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n == lo:
            continue
        j = torch.arange(lo, n, device=DEV)
        kk, vv = (x[table[i, j // page].long(), j % page].repeat_interleave(Q // H, 1) for x in (k, v))
        t = torch.einsum("hd,nhd->hn", q[i].double(), kk) * scale
        e = (D + 16) * 2.0 ** -24 * abs(scale) * torch.einsum("hd,nhd->hn", q[i].double().abs(), kk.abs())
        if softcap:
            t = softcap * torch.tanh(t / softcap)
        e = (e + 4 * 2.0 ** -24 * t.abs()).amax(-1)
        p = torch.softmax(t, -1)
        out[i] = torch.einsum("hn,nhd->hd", p, vv)
        # each score off by e at most: a weight lies between exp(-2 e) and exp(2 e)
        # of the exact one (its share of a sum that is off by exp(e) too)
        tol[i] = (torch.expm1(2 * e[:, None]) + 2.0 ** -10) * torch.einsum("hn,nhd->hd", p, vv.abs())
        # the FP16 pair drops less than 2^-40 of a weight of 1 (times its token's
        # part of the sixteen's scale), and the weights sum to 1 at least before
        # the division: n times 2^-40 of the largest value
        tol[i] += (n - lo) * 2.0 ** -40 * vv.abs().amax((0, 2))[:, None]
        lse[i] = torch.logsumexp(t, -1)
        tol_lse[i] = e + (n - lo) * 2.0 ** -24 + 4 * 2.0 ** -24 * lse[i].abs()
    return out, lse, tol, tol_lse


def check_attend(kind, cache, lens, page, block, Q, H, D, layout, window=0, softcap=0.0, scale=None, seed=0, wide=0, odd=False,
                 spread=2, order=(0, 1, 2)):
    g = gen(seed)
    table, pages = table_of(g, lens, page, slack=wide)
    c = Cache(g, cache, pages, page, block, H, D, layout, order=order, spread=spread)
    if odd:  # scales that are no powers of two
        for s in (c.ks, c.vs):
            s.mul_(1.0 + torch.rand(s.shape, generator=g, device=DEV))
    k64, v64 = (torch.nan_to_num(c.stands_for(x)) for x in "kv")
    # whatever lies behind a sequence's last token must not matter
    for i, n in enumerate(lens):
        if n % page:
            tail = int(table[i, n // page])
            for t in (c.k, c.v):
                rows = nhd(t, layout)[tail, n % page:]
                raw(rows)[...] = 127 if cache == "int8" else 0x7f
            for s in (c.ks, c.vs):
                s[tail, -(-(n % page) // block):] = math.nan
    q = torch.randn(len(lens), Q, D, generator=g, device=DEV).to(DT[kind])
    out, lse = torch.full_like(q, 9.0), torch.full((len(lens), Q), 9.0, device=DEV)
    scale = D ** -0.5 if scale is None else scale
    c.c.attend(q, table, ints(lens), out, lse=lse, scale=scale, window=window, softcap=softcap)
    assert c.c.status() == 0
    want, wlse, tol, tlse = attend64(q, k64, v64, lens, table, page, scale, window, softcap)
    bad = ~((out.double() - want).abs() <= half_step(kind, want) + tol)
    assert not bad.any(), (int(bad.sum()), float((out.double() - want).abs().max()))
    empty = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse), empty) and (out[empty] == 0).all()
    assert ((lse.double() - wlse).abs() <= tlse)[~empty].all()
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    c.c.attend(q, table, ints(lens), again, lse=lse2, scale=scale, window=window, softcap=softcap)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    c.c.close()
    return out, want


LENS = [[1], [0], [16], [17], [1000], [5, 0, 64, 65, 333, 1, 0], [129, 2, 777, 31]]
KINDS = [("bf16", "e4m3"), ("fp16", "e4m3"), ("bf16", "int8"), ("fp16", "int8")]


@pytest.mark.parametrize("wide", [0, 5000], ids=["cluster", "split"])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("kind,cache", KINDS)
def test_attend_lengths_and_types(lens, kind, cache, wide):
    check_attend(kind, cache, lens, 16, 16, 8, 2, 128, "nhd", seed=len(lens), wide=wide)


@pytest.mark.parametrize("Q,H,D", [(1, 1, 64), (7, 7, 80), (12, 2, 96), (32, 8, 128), (24, 1, 64), (40, 2, 256),
                                   (6, 3, 192), (9, 3, 16), (130, 2, 32), (3, 1, 144), (17, 1, 48)])
@pytest.mark.parametrize("page,block,layout,cache,wide", [
    (16, 16, "nhd", "int8", 0), (1, 1, "hnd", "e4m3", 0), (48, 16, "hnd", "e4m3", 5000), (7, 7, "nhd", "int8", 900), (64, 32, "nhd", "e4m3", 0),
    (256, 1, "hnd", "int8", 50), (24, 3, "nhd", "e4m3", 3000), (40, 8, "nhd", "int8", 0)])
def test_attend_heads_pages_and_blocks(Q, H, D, page, block, layout, cache, wide):
    check_attend("bf16", cache, [301, 1, 64], page, block, Q, H, D, layout, seed=Q + D, wide=wide, odd=D % 32 != 0, order=(2, 0, 1) if Q % 2 else (0, 1, 2))


@pytest.mark.parametrize("window", [1, 15, 16, 64, 100, 5000])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("block", [4, 16])
def test_attend_window_and_softcap(window, softcap, block):
    check_attend("bf16", "int8", [300, 64, 1, 0, 17], 16, block, 8, 4, 64, "nhd", window=window, softcap=softcap, seed=window)
    check_attend("fp16", "e4m3", [333, 16, 1, 100], 16, block, 8, 2, 128, "nhd", window=window, softcap=softcap, seed=3, wide=500)


@pytest.mark.parametrize("block", [1, 2, 16])
@pytest.mark.parametrize("cache", ["e4m3", "int8"])
def test_attend_scales_far_apart(block, cache):
    """Scales over a range of 2^20: each token's keys and values by its own."""
    check_attend("bf16", cache, [500, 77], 16, block, 8, 2, 64, "nhd", seed=block, spread=10, odd=True)
    check_attend("bf16", cache, [500, 77], 16, block, 8, 2, 64, "nhd", seed=block, spread=10, wide=700, scale=2.0 ** -14)


def test_attend_scales_at_the_ends_of_fp32():
    """Keys of 2^100 with queries of 2^-100, and values whose scales are near the
    smallest and the largest numbers."""
    g = gen(21)
    table, pages = table_of(g, [40], 16)
    c = Cache(g, "int8", pages, 16, 16, 1, 64)
    q = torch.randn(1, 4, 64, generator=g, device=DEV).to(torch.bfloat16) * 2.0 ** -100
    for k_unit, v_unit in ((2.0 ** 97, 2.0 ** 100), (2.0 ** 97, 2.0 ** -110), (2.0 ** 97, 2.0 ** -140)):
        c.ks.fill_(k_unit)
        c.vs.fill_(v_unit)
        out = torch.empty_like(q)
        c.c.attend(q, table, ints([40]), out)
        want, _, tol, _ = attend64(q, c.stands_for("k"), c.stands_for("v"), [40], table, 16, 0.125)
        # (2^-133: the smallest step of a BF16 result)
        assert ((out.double() - want).abs() <= half_step("bf16", want) + tol + 2.0 ** -134 + 40 * 2.0 ** -149).all()
    c.c.close()


@pytest.mark.parametrize("lens", [[20000], [3000, 0, 9000, 70, 1]])
def test_attend_long(lens):
    check_attend("bf16", "int8", lens, 16, 16, 16, 2, 128, "nhd", seed=3)
    check_attend("fp16", "e4m3", lens, 64, 2, 4, 4, 64, "hnd", seed=4)


def test_attend_many_sequences():
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 90, (700,), generator=g).tolist()
    check_attend("bf16", "int8", lens, 16, 16, 4, 2, 64, "nhd", seed=9)


@pytest.mark.parametrize("wide", [0, 5000])
@pytest.mark.parametrize("block", [1, 16])
@pytest.mark.parametrize("kind,cache", KINDS)
def test_attend_adds_little_to_the_outputs_rounding(kind, cache, block, wide):
    """In relative L2 the result is as near as one rounding of the exact one, 2^-15
    and a twentieth of that (tests of the 16-bit cache)."""
    out, want = check_attend(kind, cache, [777, 2500, 64], 16, block, 8, 2, 128, "nhd", seed=17, wide=wide, spread=1)
    for i in range(3):
        norm = float(want[i].norm())
        least = float((want[i].to(DT[kind]).double() - want[i]).norm()) / norm
        assert float((out[i].double() - want[i]).norm()) / norm <= 1.05 * least + 2.0 ** -15


@pytest.mark.parametrize("wide", [0, 5000])
def test_attend_nan_elements_and_scales(wide):
    g = gen(16)
    S, Q, H, D, page = 3, 4, 2, 64, 16
    lens = [60] * S
    table, pages = table_of(g, lens, page, slack=wide)
    c = Cache(g, "e4m3", pages, page, 4, H, D)
    q = torch.randn(S, Q, D, generator=g, device=DEV).to(torch.bfloat16)
    q[0, 1, 3] = float("nan")                        # every score of one head
    raw(c.k)[int(table[1, 0]), 2, 1, 5] = 0x7f       # one score of the heads of KV head 1
    c.ks[int(table[2, 1]), 1, 0] = math.nan          # four scores of the heads of KV head 0
    raw(c.v)[int(table[2, 2]), 3, 1, 9] = 0x7f       # one element of the values of KV head 1
    out, lse = torch.full_like(q, 9.0), torch.full((S, Q), 9.0, device=DEV)
    c.c.attend(q, table, ints(lens), out, lse=lse)
    nan = torch.zeros(S, Q, dtype=torch.bool, device=DEV)
    nan[0, 1] = nan[1, 2:] = nan[2, :2] = True
    assert out[nan].isnan().all() and lse[nan].isnan().all() and not lse[~nan].isnan().any()
    assert out[2, 2:, 9].isnan().all()
    rest = ~nan[..., None].expand_as(out).clone()
    rest[2, 2:, 9] = False
    k64, v64 = (torch.nan_to_num(c.stands_for(x)) for x in "kv")
    want, _, tol, _ = attend64(torch.nan_to_num(q), k64, v64, lens, table, page, D ** -0.5)
    assert ((out.double() - want).abs() <= half_step("bf16", want) + tol)[rest].all()
    c.c.close()


def test_attend_bad_lengths_and_pages_are_reported():
    g = gen(12)
    table, pages = table_of(g, [64, 64, 64, 64], 16)
    c = Cache(g, "int8", pages, 16, 8, 1, 64)
    q = torch.randn(4, 2, 64, generator=g, device=DEV).to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(4, 2, device=DEV)
    lens = ints([64, -1, 65, 64])
    table[3, 1], table[3, 2] = pages, -1  # tokens 16..47 are masked
    c.c.attend(q, table, lens, out, lse=lse)
    assert c.c.status() == 1 and c.c.status() == 0
    assert (out[1:3] == 0).all() and torch.isinf(lse[1:3]).all()
    k64, v64 = c.stands_for("k"), c.stands_for("v")
    for row, part, n in ((0, table[:1], 64), (3, table[3:, [0, 3]], 32)):
        want, _, tol, _ = attend64(q[row:row + 1], k64, v64, [n], part, 16, 0.125)
        assert ((out[row:row + 1].double() - want).abs() <= half_step("bf16", want) + tol).all()
    c.c.close()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_then_attend_in_a_graph(kind):
    """The two as a serving step uses them, captured once and replayed for
    successive tokens, against the attention over all cached tokens in 64 bits."""
    g = gen(13)
    S, Q, H, D, page, steps = 3, 4, 2, 64, 8, 21
    start = [0, 5, 16]
    table, pages = table_of(g, [s + steps for s in start], page)
    c = Cache(g, kind, pages, page, 8, H, D)
    index = ints(start)
    lens = index + 1
    inv = (10000.0 ** (-torch.arange(D // 2, device=DEV) / (D // 2))).float()
    q, kn, vn = (torch.zeros(S, h, D, dtype=torch.bfloat16, device=DEV) for h in (Q, H, H))
    out = torch.empty_like(q)

    def step():
        stream = torch.cuda.current_stream().cuda_stream
        c.c.append(kn, vn, table, index, inv_freq=inv, q=q, stream=stream)
        c.c.attend(q, table, lens, out, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    exact = [[] for _ in range(S)]
    for i in range(steps):
        for t in (q, kn, vn):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        index.copy_(torch.tensor([s + i for s in start], dtype=torch.int32))
        lens.copy_(index + 1)
        graph.replay()
        want, _, tol, _ = attend64(q, c.stands_for("k"), c.stands_for("v"), [s + i + 1 for s in start], table, page, D ** -0.5)
        assert ((out.double() - want).abs() <= half_step("bf16", want) + tol).all()
        for s in range(S):
            exact[s].append(vn[s].double().clone())
    assert c.c.status() == 0
    # what the cache holds is what was appended, to a step or two of its type
    v64 = c.stands_for("v")
    for s in range(S):
        at = torch.arange(start[s] + 8 - start[s] % 8, start[s] + steps, device=DEV)  # from the first whole block
        rows = v64[table[s, at // page].long(), at % page]
        new = torch.stack(exact[s])[at - start[s]]
        unit = c.vs[table[s, at // page].long(), at % page // 8].double()[..., None]
        assert ((rows - new).abs() <= 2 * half_step(kind, new.abs() / unit) * unit + (0 if kind == "int8" else 2.0 ** -9) * unit).all()
    c.c.close()


def test_offsets_past_32_bits():
    """Pages and scales whose offsets pass 2^32 bytes and 2^31 elements."""
    g = gen(14)
    page, D, step, pages = 16, 64, 1 << 21, 2700  # a page every 2 MB
    k, v = (torch.empty(pages * step, dtype=torch.int8, device=DEV).as_strided((pages, page, 1, D), (step, D, D, 1)) for _ in range(2))
    ks, vs = (torch.empty(pages * (step // 2), device=DEV).as_strided((pages, 2, 1), (step // 2, 1, 1)) for _ in range(2))
    c = xg.KVCache(k, v, k_scale=ks, v_scale=vs)
    table = ints([[2699, 5, 2600]])
    n = 40
    kn, vn = (torch.randn(n, 1, D, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    index = torch.arange(n, dtype=torch.int32, device=DEV)
    c.append(kn, vn, table, index, seq=torch.zeros_like(index))
    rows, place = table[0, index.long() // page].long(), index.long() % page
    k64, v64 = (t[rows, place].double() * s[rows, place // 8].double()[..., None] for t, s in ((k, ks), (v, vs)))
    for got, want, s in ((k64, kn, ks), (v64, vn, vs)):
        assert ((got - want.double()).abs() <= 0.5 * s[rows, place // 8].double()[..., None]).all()
    q = torch.randn(1, 3, D, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    c.attend(q, table, ints([n]), out)
    want, _, tol, _ = attend64(q, k64[:, None], v64[:, None], [n], torch.arange(n, device=DEV)[None], 1, 0.125)
    assert ((out.double() - want).abs() <= half_step("bf16", want) + tol).all() and c.status() == 0
    c.close()


def test_refusals():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.int8, device=DEV)
    v, s = torch.zeros_like(k), torch.ones(4, 2, 2, device=DEV)
    e = k.view(torch.uint8).view(torch.float8_e4m3fn)
    for args in ((k, v, None, None), (k, v, s, None), (k, v, None, s), (k, v, s, s.half()), (k, v, s, s[:3]), (k, v, s, s.cpu()),
                 (k, v, torch.ones(4, 3, 2, device=DEV), torch.ones(4, 3, 2, device=DEV)), (k, v, s[0, 0], s[0, 0]),
                 (k.bfloat16(), v.bfloat16(), s, s), (k, v, torch.ones(4, 0, 2, device=DEV), torch.ones(4, 0, 2, device=DEV)),
                 (k, v, s, s[:1].expand(4, 2, 2)), (k[:, :, :, :60], v[:, :, :, :60], s, s), (k, e, s, s)):
        with pytest.raises(ValueError):
            xg.KVCache(args[0], args[1], k_scale=args[2], v_scale=args[3])
    c = xg.KVCache(k, v, k_scale=s, v_scale=s.clone())
    table, idx = torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    new = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):
        c.append(new, new, table, idx, inv_freq=torch.ones(33, device=DEV))
    with pytest.raises(ValueError):
        c.append(new.to(torch.int8), new.to(torch.int8), table, idx)
    q = torch.zeros(2, 4, 64, dtype=torch.float32, device=DEV)
    with pytest.raises(ValueError):
        c.attend(q, table, idx, torch.empty_like(q))
    c.close()
    # the C entry's own checks
    d = xg.KvDesc(k.data_ptr(), v.data_ptr(), k.numel(), v.numel(), 4, 16)
    d.k_stride[:], d.v_stride[:] = (2048, 128, 64), (2048, 128, 64)
    d.kv_heads, d.head_dim, d.type = 2, 64, xg.INT8
    import ctypes
    lib, h = xg.load(), ctypes.c_void_p()

    def create(**change):
        b = xg.KvBlocks(s.data_ptr(), s.data_ptr(), s.numel() * 4, s.numel() * 4, 8)
        b.k_stride[:], b.v_stride[:] = (4, 2, 1), (4, 2, 1)
        for name, value in change.items():
            if name.endswith("stride"):
                getattr(b, name)[:] = value
            else:
                setattr(b, name, value)
        r = lib.xksv_kv_create_blocks(ctypes.byref(d), ctypes.byref(b), ctypes.byref(h))
        if h:
            lib.xksv_kv_destroy(h)
        return r

    assert create() == 0
    for bad in (dict(block=0), dict(block=5), dict(block=32), dict(k_scale=0), dict(v_scale=s.data_ptr() + 2), dict(k_bytes=60), dict(v_stride=(4, 2, 2)),
                dict(k_stride=(1 << 50, 2, 1)), dict(k_stride=(3, 2, 1))):
        assert create(**bad) == 1, bad
    assert lib.xksv_kv_create_blocks(ctypes.byref(d), None, ctypes.byref(h)) == 1
    assert lib.xksv_kv_create(ctypes.byref(d), ctypes.byref(h)) == 1  # integers have block scales
