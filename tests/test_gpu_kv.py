"""GPU: the paged key/value cache (KVCache.append, KVCache.attend) against
plain 64-bit forms, at the sizes, layouts, types and masks where they can go
wrong, and its refusals.

Tolerances (derived, per element): an output rounded once to a type is off by
at most eps / 2 relative (half the smallest subnormal near zero).  append:
the angle's cosine and sine are off by at most 2^-21 (a FP32 angle within half
an ulp of pi, 2^-23, and sincosf's 2 ulp), the two products and their sum by
3 * 2^-24, so a rotated value is off by 2^-20 (|a| + |b|) before rounding.
attend: a FP32 score is off by e = (dim + 16) 2^-24 scale sum |q k| + 4 * 2^-24 |t|,
a weight by 2 e relative, its rounding for the tensor cores by 2^-11, sums of
n terms by n 2^-24 at most (n <= 1000s here: within the 2^-11), so the output
by (2 e + 2^-10) sum p |v| before rounding."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
TINY = {"bf16": 0.0, "fp16": 2.0 ** -25, "fp32": 0.0, "e4m3": 2.0 ** -10}


def half_step(kind, exact):
    return torch.finfo(DT[kind]).eps / 2 * exact.abs() + TINY[kind]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make_cache(g, kind, pages, page, heads, dim, layout, fill=None):
    """Cache tensors of N(0, 1) values (or bytes `fill`), KVCache, and FP64
    [pages, page, heads, dim] views of what they stand for."""
    shape = (pages, page, heads, dim) if layout == "nhd" else (pages, heads, page, dim)
    k, v = (torch.randn(shape, generator=g, device=DEV).mul_(30 if kind == "e4m3" else 1).to(DT[kind]) for _ in range(2))
    ks = vs = None
    if kind == "e4m3":
        ks, vs = (torch.rand(heads, generator=g, device=DEV) * 0.05 + 0.01 for _ in range(2))
    return k, v, ks, vs, xg.KVCache(k, v, k_scale=ks, v_scale=vs, layout=layout)


def rows64(c, scale, layout):
    r = c.double() if layout == "nhd" else c.double().permute(0, 2, 1, 3)
    return r if scale is None else r * scale.double()[:, None]


def table_of(g, lens, page, spare=2, slack=0):
    """A page table of shuffled pages over a pool with `spare` unused ones;
    entries behind a sequence's pages are out of range."""
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
    out, mag = x.clone(), x.abs()
    ia = torch.arange(half, device=DEV) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * scale
    return out, mag


@pytest.mark.parametrize("dim,rot,interleaved,q_heads,kv_heads", [
    (128, 128, False, 32, 8), (64, 64, True, 6, 3), (80, 32, False, 5, 5), (256, 256, True, 4, 1),
    (96, 20, True, 3, 3), (16, 6, False, 2, 1), (192, 64, False, 7, 7), (64, 0, False, 4, 2)])
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "bf16"), ("bf16", "e4m3"), ("fp32", "e4m3")])
def test_append_matches_64_bits(dim, rot, interleaved, q_heads, kv_heads, kind, cache):
    for layout, page, n in (("nhd", 16, 37), ("hnd", 5, 1), ("nhd", 1, 9)):
        g = gen(dim + n)
        S = min(n, 4)
        counts = [n // S + (i < n % S) for i in range(S)]
        first = [3 * i for i in range(S)]
        table, pages = table_of(g, [f + c for f, c in zip(first, counts)], page)
        k, v, ks, vs, c = make_cache(g, cache, pages, page, kv_heads, dim, layout)
        k0, v0 = rows64(k, None, layout), rows64(v, None, layout)
        seq = torch.tensor([i for i in range(S) for _ in range(counts[i])], dtype=torch.int32, device=DEV)
        index = torch.tensor([first[i] + j for i in range(S) for j in range(counts[i])], dtype=torch.int32, device=DEV)
        # positions far out, where an FP32 angle would be off by radians
        pos = index + torch.tensor([0, 1048575, 77, 2 ** 31 - 200], dtype=torch.int64, device=DEV)[seq.long()].to(torch.int32)
        if n > 3:
            seq[2] = -1  # padding
        inv = (10000.0 ** (-torch.arange(rot // 2, device=DEV, dtype=torch.float64) / max(1, rot // 2))).float()
        qn, kn, vn = (torch.randn(n, h, dim, generator=g, device=DEV).to(DT[kind]) for h in (q_heads, kv_heads, kv_heads))
        q_out = torch.full_like(qn, 7.0)
        c.append(kn, vn, table, index, seq=seq, positions=pos, inv_freq=inv if rot else None, rot_scale=1.25,
                 interleaved=interleaved, q=qn, q_out=q_out)
        assert c.status() == 0
        want, mag = rope64(qn, pos, inv, interleaved, 1.25)
        live = (seq >= 0).nonzero()[:, 0]
        err = (q_out.double() - want).abs()
        assert (err <= half_step(kind, want) + 2.0 ** -20 * mag)[live].all()
        assert (q_out[seq < 0] == 7.0).all()  # padding rows are left alone
        want, mag = rope64(kn, pos, inv, interleaved, 1.25)
        got_k, got_v = rows64(k, None, layout), rows64(v, None, layout)
        pg = table[seq[live].long(), index[live].long() // page].long()
        pl = index[live].long() % page
        for got, old, val, m, s in ((got_k, k0, want, mag, ks), (got_v, v0, vn.double(), torch.zeros_like(mag), vs)):
            val, m = val[live], m[live]
            if s is not None:
                val, m = val / s.double()[:, None], m / s.double()[:, None] + val.abs() * 2.0 ** -4  # + the division
                val = val.clamp(-448, 448)
            bad = (got[pg, pl] - val).abs() > half_step(cache, val) + 2.0 ** -20 * m
            assert not bad.any()
            old[pg, pl] = got[pg, pl]
            assert torch.equal(got, old)  # nothing else was written
        c.close()


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_append_strides_in_place_and_sliced_cache(layout):
    """q, k and v as slices of one packed buffer whose rows are of odd
    alignment, q rotated in place, and a cache whose k and v are two halves of one tensor."""
    g = gen(5)
    n, QH, H, D, page = 11, 4, 2, 64, 8
    table, pages = table_of(g, [n], page)
    shape = (pages, 2, page, H, D) if layout == "nhd" else (pages, 2, H, page, D)
    both = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    c = xg.KVCache(both[:, 0], both[:, 1], layout=layout)
    packed = torch.randn(n, (QH + 2 * H) * D + 3, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = (t.unflatten(1, (-1, D)) for t in packed[:, 1:1 + (QH + 2 * H) * D].split([QH * D, H * D, H * D], dim=1))
    before = packed.clone()
    q0 = q.clone()
    index = torch.arange(n, dtype=torch.int32, device=DEV)
    inv = (10000.0 ** (-torch.arange(D // 2, device=DEV) / (D // 2))).float()
    c.append(k, v, table, index, seq=torch.zeros_like(index), inv_freq=inv, q=q)
    assert c.status() == 0
    want, mag = rope64(q0, index, inv, False)
    assert ((q.double() - want).abs() <= half_step("bf16", want) + 2.0 ** -20 * mag).all()
    assert torch.equal(packed[:, 0], before[:, 0]) and torch.equal(packed[:, 1 + QH * D:], before[:, 1 + QH * D:])
    want, mag = rope64(k, index, inv, False)
    pg, pl = table[0, index.long() // page].long(), index.long() % page
    got = rows64(both[:, 0], None, layout)[pg, pl]
    assert ((got - want).abs() <= half_step("bf16", want) + 2.0 ** -20 * mag).all()
    assert torch.equal(rows64(both[:, 1], None, layout)[pg, pl], v.double())
    c.close()


def test_append_special_values_saturate_and_stay():
    """E4M3: values beyond 448 scales saturate, NaN stays NaN, zero keeps."""
    g = gen(6)
    table, pages = table_of(g, [1], 4)
    k, v, ks, vs, c = make_cache(g, "e4m3", pages, 4, 1, 16, "nhd")
    x = torch.zeros(1, 1, 16, device=DEV)
    x[0, 0, :5] = torch.tensor([1e30, -1e30, float("nan"), float("inf"), -0.0])
    c.append(x, x, table, torch.zeros(1, dtype=torch.int32, device=DEV))
    got = v[int(table[0, 0]), 0, 0].float().tolist()
    assert got[0] == 448 and got[1] == -448 and math.isnan(got[2]) and got[3] == 448 and got[5:] == [0.0] * 11
    assert torch.equal(k.view(torch.uint8)[int(table[0, 0]), 0], v.view(torch.uint8)[int(table[0, 0]), 0])
    c.close()


def test_append_bad_pages_are_skipped_and_reported():
    g = gen(7)
    table, pages = table_of(g, [8, 8], 4)
    k, v, _, _, c = make_cache(g, "bf16", pages, 4, 2, 32, "nhd")
    new = torch.randn(5, 2, 32, generator=g, device=DEV).to(torch.bfloat16)
    table[1, 1] = pages  # one page past the cache
    # places: fine, past the table's columns, a sequence past its rows, a bad page, a negative page
    table[0, 1] = -5
    seq = torch.tensor([0, 0, 2, 1, 0], dtype=torch.int32, device=DEV)
    index = torch.tensor([1, 8, 0, 4, 7], dtype=torch.int32, device=DEV)
    k0, v0 = k.clone(), v.clone()
    q = torch.randn(5, 2, 32, generator=g, device=DEV).to(torch.bfloat16)
    q_out = torch.full_like(q, 3.0)
    c.append(new, new, table, index, seq=seq, q=q, q_out=q_out)
    assert c.status() == 1 and c.status() == 0
    k0[int(table[0, 0]), 1] = new[0]
    v0[int(table[0, 0]), 1] = new[0]
    assert torch.equal(k, k0) and torch.equal(v, v0)
    assert torch.equal(q_out[0], q[0]) and (q_out[1:] == 3.0).all()
    c.append(new[:0], new[:0], table, index[:0])  # no tokens: nothing happens
    assert c.status() == 0
    c.close()


# ------------------------------------------------------------------ attend
def attend64(q, k, v, lens, table, page, scale, window=0, softcap=0.0):
    """(out, lse, tolerance before rounding) in 64 bits; k, v are FP64
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
        tol[i] = (2 * e[:, None] + 2.0 ** -10) * torch.einsum("hn,nhd->hd", p, vv.abs())
        lse[i] = torch.logsumexp(t, -1)
        tol_lse[i] = e + (n - lo) * 2.0 ** -24 + 4 * 2.0 ** -24 * lse[i].abs()
    return out, lse, tol, tol_lse


def check_attend(kind, cache, lens, page, Q, H, D, layout, window=0, softcap=0.0, scale=None, seed=0, q_mag=1.0,
                 wide=0):
    g = gen(seed)
    table, pages = table_of(g, lens, page)
    if wide:  # a table of `wide` more columns, unused
        table = torch.cat([table, torch.full((len(lens), wide), -1, dtype=torch.int32, device=DEV)], 1)
    k, v, ks, vs, c = make_cache(g, cache, pages, page, H, D, layout)
    # whatever lies behind a sequence's last token must not matter
    for i, n in enumerate(lens):
        if n % page:
            tail = int(table[i, n // page])
            for t in (k, v):
                (t[tail, n % page:] if layout == "nhd" else t[tail, :, n % page:]).fill_(float("nan"))
    q = (torch.randn(len(lens), Q, D, generator=g, device=DEV) * q_mag).to(DT[kind])
    out, lse = torch.full_like(q, 9.0), torch.full((len(lens), Q), 9.0, device=DEV)
    scale = D ** -0.5 if scale is None else scale
    c.attend(q, table, torch.tensor(lens, dtype=torch.int32, device=DEV), out, lse=lse, scale=scale, window=window,
             softcap=softcap)
    assert c.status() == 0
    k64, v64 = (torch.nan_to_num(rows64(t, s, layout)) for t, s in ((k, ks), (v, vs)))
    want, wlse, tol, tlse = attend64(q, k64, v64, lens, table, page, scale, window, softcap)
    bad = ~((out.double() - want).abs() <= half_step(kind, want) + tol)
    assert not bad.any(), (int(bad.sum()), float((out.double() - want).abs().max()))
    empty = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse), empty) and (out[empty] == 0).all()
    assert ((lse.double() - wlse).abs() <= tlse)[~empty].all()
    c.close()


LENS = [[1], [0], [16], [17], [1000], [5, 0, 64, 65, 333, 1, 0], [129, 2, 777, 31]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")])
def test_attend_lengths_and_types(lens, kind, cache):
    check_attend(kind, cache, lens, 16, 8, 2, 128, "nhd", seed=len(lens))


@pytest.mark.parametrize("Q,H,D", [(1, 1, 64), (7, 7, 80), (12, 2, 96), (32, 8, 128), (24, 1, 64), (40, 2, 256),
                                   (6, 3, 192), (9, 3, 16), (130, 2, 32), (3, 1, 144), (17, 1, 48)])
@pytest.mark.parametrize("page,layout,cache", [(16, "nhd", "bf16"), (1, "hnd", "e4m3"), (48, "hnd", "bf16"), (7, "nhd", "e4m3"),
                                               (256, "nhd", "bf16")])
def test_attend_heads_and_pages(Q, H, D, page, layout, cache):
    check_attend("bf16", cache, [301, 1, 64], page, Q, H, D, layout, seed=Q + D)


# The same with tables of room for many more tokens: these calls split the
# work over all warps and join in a second kernel.
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")])
def test_attend_in_a_long_table(lens, kind, cache):
    check_attend(kind, cache, lens, 16, 8, 2, 128, "nhd", seed=len(lens), wide=5000)


@pytest.mark.parametrize("Q,H,D", [(1, 1, 64), (7, 7, 80), (12, 2, 96), (32, 8, 128), (24, 1, 64), (40, 2, 256),
                                   (6, 3, 192), (9, 3, 16), (130, 2, 32), (3, 1, 144), (17, 1, 48)])
@pytest.mark.parametrize("page,layout,cache", [(16, "nhd", "bf16"), (1, "hnd", "e4m3"), (48, "hnd", "bf16"), (7, "nhd", "e4m3")])
def test_attend_heads_and_pages_in_a_long_table(Q, H, D, page, layout, cache):
    check_attend("bf16", cache, [301, 1, 64], page, Q, H, D, layout, seed=Q + D, wide=5000)


@pytest.mark.parametrize("window,softcap", [(1, 0.0), (15, 20.0), (64, 0.0), (5000, 20.0)])
def test_attend_window_and_softcap_in_a_long_table(window, softcap):
    check_attend("bf16", "bf16", [333, 16, 1, 100], 16, 8, 2, 128, "nhd", window=window, softcap=softcap, seed=3, wide=500)


@pytest.mark.parametrize("window", [1, 15, 16, 64, 100, 5000])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_attend_window_and_softcap(window, softcap):
    check_attend("bf16", "bf16", [300, 64, 1, 0, 17], 16, 8, 4, 64, "nhd", window=window, softcap=softcap, seed=window)


def test_attend_large_scores_and_negative_scale():
    """Scores in the thousands: the running maximum keeps the exponentials in
    range; a negative scale prefers the other end."""
    for scale in (4.0, -4.0):
        check_attend("bf16", "bf16", [500, 33], 16, 4, 2, 64, "nhd", scale=scale, q_mag=8.0)


@pytest.mark.parametrize("lens", [[20000], [3000, 0, 9000, 70, 1]])
def test_attend_long(lens):
    """Lengths that are split and joined."""
    check_attend("bf16", "bf16", lens, 16, 16, 2, 128, "nhd", seed=3)
    check_attend("fp16", "e4m3", lens, 64, 4, 4, 64, "hnd", seed=4)


def test_attend_many_sequences():
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 90, (700,), generator=g).tolist()
    check_attend("bf16", "bf16", lens, 16, 4, 2, 64, "nhd", seed=9)


def test_attend_strides_and_repeats():
    """q and out as slices of wider buffers; the same call twice gives the same bits."""
    g = gen(11)
    lens = [700, 45, 0]
    table, pages = table_of(g, lens, 16, slack=3)
    k, v, _, _, c = make_cache(g, "bf16", pages, 16, 2, 64, "nhd")
    wide = torch.randn(3, 9, 71, generator=g, device=DEV).to(torch.bfloat16)
    q = wide[:, 1:7, 3:67]
    buf = torch.full((6, 3, 70), 5.0, dtype=torch.bfloat16, device=DEV)
    out = buf.transpose(0, 1)[..., 2:66]
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    c.attend(q, table, n, out)
    want, _, tol, _ = attend64(q, k.double(), v.double(), lens, table, 16, 0.125)
    assert ((out.double() - want).abs() <= half_step("bf16", want) + tol).all()
    first = buf.clone()
    assert (first[..., :2] == 5).all() and (first[..., 66:] == 5).all()
    for _ in range(3):
        c.attend(q, table, n, out)
        assert torch.equal(buf, first)
    assert c.status() == 0
    c.close()


def test_attend_bad_lengths_and_pages_are_reported():
    g = gen(12)
    table, pages = table_of(g, [64, 64, 64, 64], 16)
    k, v, _, _, c = make_cache(g, "bf16", pages, 16, 1, 64, "nhd")
    q = torch.randn(4, 2, 64, generator=g, device=DEV).to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(4, 2, device=DEV)
    lens = torch.tensor([64, -1, 65, 64], dtype=torch.int32, device=DEV)
    table[3, 1], table[3, 2] = pages, -1  # tokens 16..47 are masked
    c.attend(q, table, lens, out, lse=lse)
    assert c.status() == 1 and c.status() == 0
    assert (out[1:3] == 0).all() and torch.isinf(lse[1:3]).all()
    want, _, tol, _ = attend64(q[:1], k.double(), v.double(), [64], table, 16, 0.125)
    assert ((out[:1].double() - want).abs() <= half_step("bf16", want) + tol).all()
    pages3 = table[3:, [0, 3]]
    want, _, tol, _ = attend64(q[3:], k.double(), v.double(), [32], pages3, 16, 0.125)
    assert ((out[3:].double() - want).abs() <= half_step("bf16", want) + tol).all()
    table[3] = -1  # every page is bad: the row is empty
    c.attend(q, table, lens, out, lse=lse)
    assert c.status() == 1 and (out[3] == 0).all() and torch.isinf(lse[3]).all()
    c.close()


def test_append_then_attend_in_a_graph():
    """The two as a serving step uses them, captured once and replayed for
    successive tokens, against the attention over all tokens in 64 bits."""
    g = gen(13)
    S, Q, H, D, page, steps = 3, 4, 2, 64, 8, 21
    start = [0, 5, 16]
    table, pages = table_of(g, [s + steps for s in start], page)
    k, v, _, _, c = make_cache(g, "bf16", pages, page, H, D, "nhd")
    index = torch.tensor(start, dtype=torch.int32, device=DEV)
    lens = index + 1
    inv = (10000.0 ** (-torch.arange(D // 2, device=DEV) / (D // 2))).float()
    q, kn, vn = (torch.zeros(S, h, D, dtype=torch.bfloat16, device=DEV) for h in (Q, H, H))
    out = torch.empty_like(q)

    def step():
        stream = torch.cuda.current_stream().cuda_stream
        c.append(kn, vn, table, index, inv_freq=inv, q=q, stream=stream)
        c.attend(q, table, lens, out, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        for t in (q, kn, vn):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        index.copy_(torch.tensor([s + i for s in start], dtype=torch.int32))
        lens.copy_(index + 1)
        q0 = q.clone()
        graph.replay()
        turned, mag = rope64(q0, index, inv, False)
        assert ((q.double() - turned).abs() <= half_step("bf16", turned) + 2.0 ** -20 * mag).all()
        want, _, tol, _ = attend64(q, k.double(), v.double(), [s + i + 1 for s in start], table, page, D ** -0.5)
        assert ((out.double() - want).abs() <= half_step("bf16", want) + tol).all()
    assert c.status() == 0
    c.close()


def test_offsets_past_32_bits():
    """Pages whose offsets pass 2^32 bytes and 2^31 elements: append and attend
    at the far end of a 5.6 GB buffer."""
    g = gen(14)
    page, D, step, pages = 16, 64, 1 << 20, 2700  # a page every 2 MB
    k, v = (torch.empty(pages * step, dtype=torch.bfloat16, device=DEV).as_strided((pages, page, 1, D), (step, D, D, 1))
            for _ in range(2))
    c = xg.KVCache(k, v)
    table = torch.tensor([[2699, 5, 2600]], dtype=torch.int32, device=DEV)
    n = 40
    kn, vn = (torch.randn(n, 1, D, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    index = torch.arange(n, dtype=torch.int32, device=DEV)
    c.append(kn, vn, table, index, seq=torch.zeros_like(index))
    rows = table[0, index.long() // page].long()
    assert torch.equal(k[rows, index.long() % page], kn) and torch.equal(v[rows, index.long() % page], vn)
    q = torch.randn(1, 3, D, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    c.attend(q, table, torch.tensor([n], dtype=torch.int32, device=DEV), out)
    want, _, tol, _ = attend64(q, kn.double()[:, None], vn.double()[:, None], [n], torch.arange(n, device=DEV)[None], 1, 0.125)
    assert ((out.double() - want).abs() <= half_step("bf16", want) + tol).all() and c.status() == 0
    c.close()


def test_calls_on_several_streams():
    """Two sequences' attention at once on two streams, a call for the default
    stream made inside a side stream, and a caller's own workspace."""
    g = gen(15)
    table, pages = table_of(g, [5000, 3000], 16)
    k, v, _, _, c = make_cache(g, "bf16", pages, 16, 2, 64, "nhd")
    q = torch.randn(2, 8, 64, generator=g, device=DEV).to(torch.bfloat16)
    lens = torch.tensor([5000, 3000], dtype=torch.int32, device=DEV)
    want, _, tol, _ = attend64(q, k.double(), v.double(), [5000, 3000], table, 16, 0.125)
    torch.cuda.synchronize()
    outs = [torch.zeros(1, 8, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                c.attend(q[i:i + 1], table[i:i + 1], lens[i:i + 1], outs[i], stream=side.cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        assert ((outs[i].double() - want[i:i + 1]).abs() <= (half_step("bf16", want) + tol)[i:i + 1]).all()
    out = torch.zeros_like(q)
    ws = torch.empty(c.attend_workspace(2, 8, table.shape[1]), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(sides[0]):
        c.attend(q, table, lens, out)  # the legacy default stream
        torch.cuda.default_stream().synchronize()
        first = out.clone()
        c.attend(q, table, lens, out, workspace=ws, stream=sides[0].cuda_stream)
    torch.cuda.synchronize()
    assert ((out.double() - want).abs() <= half_step("bf16", want) + tol).all() and torch.equal(out, first)
    with pytest.raises(RuntimeError):
        c.attend(q, table, lens, out, workspace=ws[:256])
    assert c.status() == 0
    c.close()


def test_refusals():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    with pytest.raises(ValueError):
        xg.KVCache(k, v.half())
    with pytest.raises(ValueError):
        xg.KVCache(k[..., :60], v[..., :60])  # a row of 120 bytes
    with pytest.raises(ValueError):
        xg.KVCache(k.float(), v.float())
    with pytest.raises(ValueError):
        xg.KVCache(k[:1].expand(4, 16, 2, 64), v)  # pages overlap
    with pytest.raises(ValueError):
        xg.KVCache(k.flatten()[4:4 + 3 * 2048].view(3, 16, 2, 64), v[:3])  # 8-byte aligned
    with pytest.raises(ValueError):
        xg.KVCache(k, v, k_scale=torch.ones(2, device=DEV))  # scales of a 16-bit cache
    with pytest.raises(ValueError):
        xg.KVCache(torch.zeros(1, 1, 1, 264, dtype=torch.bfloat16, device=DEV),
                   torch.zeros(1, 1, 1, 264, dtype=torch.bfloat16, device=DEV))
    c = xg.KVCache(k, v)
    table = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    idx = torch.zeros(2, dtype=torch.int32, device=DEV)
    new = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    inv = torch.ones(33, device=DEV)
    with pytest.raises(RuntimeError):
        c.append(new, new, table, idx, inv_freq=inv)  # rotates 66 of 64 dims
    with pytest.raises(ValueError):
        c.append(new, new.half(), table, idx)
    with pytest.raises(ValueError):
        c.append(new[:, :1], new[:, :1], table, idx)
    with pytest.raises(ValueError):
        c.append(new, new, table, idx.long())
    with pytest.raises(ValueError):
        c.append(new, new, table, idx.cpu())
    with pytest.raises(RuntimeError):
        c.append(new, new, table, idx, q=new, q_out=new[:1].expand(2, 2, 64))  # rows of q_out overlap
    q = torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):
        c.attend(q, table, idx, torch.empty_like(q))  # 3 query heads over 2
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError):
        c.attend(q, table, idx, torch.empty_like(q))  # FP16 over a BF16 cache
    q = q.bfloat16()
    with pytest.raises(ValueError):
        c.attend(q, table[:1], idx, torch.empty_like(q))
    with pytest.raises(ValueError):
        c.attend(q, table, idx, torch.empty_like(q), window=-1)
    with pytest.raises(RuntimeError):
        c.attend(q, table, idx, torch.empty_like(q), softcap=-1.0)
    c.attend(q[:0], table, idx[:0], torch.empty_like(q[:0]))  # no sequences: nothing happens
    assert c.status() == 0
    c.close()


# ------------------------------------------------- special scores, precision
# how a unit's blocks are worked off: by a cluster of CTAs, split over all
# warps and joined, or (many short sequences) by one warp alone
WAYS = {"cluster": (3, 60, 0), "split": (3, 60, 5000), "alone": (900, 40, 5000)}


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3")])
def test_attend_nan_and_infinite_scores(way, kind, cache):
    """A score that is NaN or +infinity makes its head's row and lse NaN; scores of -infinity only
    are an empty row; neither touches another row."""
    S, n, wide = WAYS[way]
    g = gen(16)
    Q, H, D, page = 4, 2, 64, 16
    lens = [n] * S
    table, pages = table_of(g, lens, page, slack=wide)
    k, v, ks, vs, c = make_cache(g, cache, pages, page, H, D, "nhd")
    q = torch.randn(S, Q, D, generator=g, device=DEV).to(DT[kind])
    q[0, 1, 3] = float("nan")           # every score of one head
    k[int(table[1, 0]), 2, 1, 5] = float("nan")  # one score of the heads of KV head 1
    if cache != "e4m3":
        q[2] = q[2].abs() + 0.5
        for p in table[2, :-(-n // page)].tolist():
            k[p, :, 0] = -float("inf")  # every score of KV head 0
        q[1, :2, 7] = 0.5
        k[int(table[1, 0]), 3, 0, 7] = float("inf")  # one score of its heads
    out, lse = torch.full_like(q, 9.0), torch.full((S, Q), 9.0, device=DEV)
    c.attend(q, table, torch.tensor(lens, dtype=torch.int32, device=DEV), out, lse=lse)
    assert c.status() == 0
    nan = torch.zeros(S, Q, dtype=torch.bool, device=DEV)
    nan[0, 1] = nan[1, 2:] = True
    empty = torch.zeros_like(nan)
    if cache != "e4m3":
        empty[2, :2] = nan[1, :2] = True
    assert torch.isnan(out[nan]).all() and torch.isnan(lse[nan]).all()
    assert (out[empty] == 0).all() and (lse[empty] == -math.inf).all()
    k64, v64 = (torch.nan_to_num(rows64(t, s, "nhd"), posinf=0.0, neginf=0.0) for t, s in ((k, ks), (v, vs)))
    want, wlse, tol, tlse = attend64(torch.nan_to_num(q), k64, v64, lens, table, page, D ** -0.5)
    rest = ~(nan | empty)
    assert ((out.double() - want).abs() <= half_step(kind, want) + tol)[rest].all()
    assert ((lse.double() - wlse).abs() <= tlse)[rest].all()
    c.close()


@pytest.mark.parametrize("wide", [0, 5000])
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")])
def test_attend_adds_little_to_the_outputs_rounding(kind, cache, wide):
    """In relative L2 the result is as near as one rounding of the exact one,
    and 2^-15 and a twentieth of that for what comes before it: weights in two
    16-bit parts are off by 2^-17 relative at most, scores by 2^-20;
    independent errors of the terms p v of a sum whose terms have random signs
    add up as the terms themselves do."""
    g = gen(17)
    lens, Q, H, D, page = [777, 2500, 64], 8, 2, 128, 16
    table, pages = table_of(g, lens, page, slack=wide)
    k, v, ks, vs, c = make_cache(g, cache, pages, page, H, D, "nhd")
    q = torch.randn(3, Q, D, generator=g, device=DEV).to(DT[kind])
    out = torch.empty_like(q)
    c.attend(q, table, torch.tensor(lens, dtype=torch.int32, device=DEV), out)
    assert c.status() == 0
    want, _, _, _ = attend64(q, rows64(k, ks, "nhd"), rows64(v, vs, "nhd"), lens, table, page, D ** -0.5)
    for i in range(3):
        norm = float(want[i].norm())
        least = float((want[i].to(DT[kind]).double() - want[i]).norm()) / norm
        assert float((out[i].double() - want[i]).norm()) / norm <= 1.05 * least + 2.0 ** -15
    c.close()
