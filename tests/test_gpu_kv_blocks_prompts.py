"""GPU: appends of more than 512 tokens to a cache with block scales, where keys and
values go by runs of tokens through a kernel of their own, against 64-bit forms;
unaligned ones, which keep to the element-by-element kernel, too.

Tolerances are those of test_gpu_kv_blocks.py: a rotated key is off by 2^-20 (|a| + |b|), a
scale is the one that the 64-bit form needs (or that of either side, where the largest element's
error reaches a border), and one rounding follows."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402
from test_gpu_kv_blocks import DEV, DT, TOP, Cache, gen, half_step, ints, nhd, raw, rope64, table_of  # noqa: E402


def needed(high, top):
    """The least power of two s >= 2^-60 with high <= top s, elementwise."""
    e = torch.ceil(torch.log2(high.clamp(min=2.0 ** -200) / top))
    e = torch.where(high > top * torch.exp2(e), e + 1, e)
    e = torch.where(high <= top * torch.exp2(e - 1), e - 1, e)
    return torch.exp2(e.clamp(min=-60.0))


def check_half(c, which, before, had, x, err, page, place):
    """One half of the cache after an append of x [tokens, heads, dim] (off by err) to
    (page, place): scales, elements, the blocks' earlier elements, and all that is left as it was."""
    t, s = (c.k, c.ks) if which == "k" else (c.v, c.vs)
    top, B, blocks = TOP[c.kind], c.block, c.page // c.block
    got, old = nhd(t, c.layout).contiguous(), nhd(before, c.layout).contiguous()
    H, D = x.shape[1:]
    ids, at = torch.unique(page * blocks + place // B, return_inverse=True)
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    slot = at[:, None].expand(-1, H)
    most, least = (torch.zeros(len(ids), H, dtype=torch.float64, device=DEV).scatter_reduce(0, slot, (size + sign * err).clamp(min=0).amax(-1), "amax")
                   for sign in (1, -1))
    first = torch.full((len(ids),), B, dtype=torch.int64, device=DEV).scatter_reduce(0, at, place % B, "amin")
    now, was = (z.reshape(-1, H)[ids].double() for z in (s.contiguous(), had.contiguous()))
    begun = (first == 0)[:, None]
    ok = torch.zeros_like(now, dtype=torch.bool)
    for high in (most, least):
        ok |= now == torch.where(begun, needed(high, top), torch.maximum(needed(high, top), was))
    assert ok.all(), (which, int((~ok).sum()), now[~ok][:4], was[~ok][:4], most[~ok][:4])
    rest = had.contiguous().reshape(-1, H).clone()
    rest[ids] = s.contiguous().reshape(-1, H)[ids]
    assert torch.equal(rest, s.contiguous().reshape(-1, H))  # no other scale was written
    # the new elements
    unit = now[at][..., None]
    want = (x / unit).clamp(-top, top)
    have = got[page, place].double()
    nan = x.isnan()
    bad = ~((have - want).abs() <= half_step(c.kind, want) + err / unit) & ~nan
    assert not bad.any(), (which, int(bad.sum()), bad.nonzero()[:3], have[bad][:3], want[bad][:3])
    assert (have[nan].isnan() if c.kind == "e4m3" else have[nan] == 0).all()
    # the blocks' earlier places, rounded again where the scale has risen; all else as it was
    expect = old.reshape(-1, B, H, D).clone()
    earlier = (torch.arange(B, device=DEV)[None] < first[:, None])[..., None, None] & ((now > was) & ~begun)[:, None, :, None]
    ratio = torch.where(now > was, was / now, torch.ones_like(now)).float()[:, None, :, None]
    again = expect[ids].float() * ratio
    again = again.round().to(torch.int8) if c.kind == "int8" else again.to(t.dtype)
    raw(expect)[ids] = torch.where(earlier, raw(again), raw(expect)[ids])
    expect = expect.reshape(got.shape)
    raw(expect)[page, place] = raw(got)[page, place]
    assert torch.equal(raw(got), raw(expect)), which


def run(c, table, seq, index, k, v, q=None, q_out=None, pos=None, inv=None, interleaved=False, rot_scale=1.0, status=0, skipped=()):
    before = [raw(t).clone().view(t.dtype) for t in (c.k, c.v)]
    had = [c.ks.clone(), c.vs.clone()]
    q0 = None if q is None else q.clone()
    o0 = None if q is None else (q if q_out is None else q_out).clone()
    k0, v0 = k.clone(), v.clone()
    c.c.append(k, v, table, index, seq=seq, positions=pos, inv_freq=inv, rot_scale=rot_scale, interleaved=interleaved, q=q, q_out=q_out)
    assert c.c.status() == status
    assert torch.equal(k.float().nan_to_num(7.0), k0.float().nan_to_num(7.0)) and torch.equal(v.float().nan_to_num(7.0), v0.float().nan_to_num(7.0))
    live = (seq >= 0) & (index >= 0)
    live[list(skipped)] = False
    at = live.nonzero()[:, 0]
    page, place = table[seq[at].long(), index[at].long() // c.page].long(), index[at].long() % c.page
    angle = index if pos is None else pos
    freq = torch.empty(0, device=DEV) if inv is None else inv
    keys, mag = rope64(k0, angle, freq, interleaved, rot_scale)
    check_half(c, "k", before[0], had[0], keys[at], 2.0 ** -20 * mag[at], page, place)
    check_half(c, "v", before[1], had[1], v0.double()[at], torch.zeros_like(mag[at]), page, place)
    if q is not None:
        want, mag = rope64(q0, angle, freq, interleaved, rot_scale)
        have = (q if q_out is None else q_out)
        kind = {torch.bfloat16: "bf16", torch.float16: "fp16", torch.float32: "fp32"}[q.dtype]
        assert ((have.double() - want).abs() <= half_step(kind, want) + 2.0 ** -20 * mag)[at].all()
        assert torch.equal(have[~live], o0[~live])


def layout_of(g, counts, first, page, padding):
    """(seq, index, table, pages): the sequences' tokens one after another, of random numbering,
    with padding behind some of them, marked by either."""
    order = torch.randperm(len(counts), generator=torch.Generator().manual_seed(len(counts))).tolist()
    table, pages = table_of(g, [f + n for f, n in zip(first, counts)], page)
    seq, index = [], []
    for i in order:
        seq += [i] * counts[i]
        index += range(first[i], first[i] + counts[i])
        if padding and i % 3 == 0:
            seq += [-1, i if i % 2 else -5, -1]
            index += [4, -1, -2147483648]
    return ints(seq), ints(index), table, pages


SHAPES = [(128, 128, False, 32, 8), (128, 64, False, 4, 1), (64, 64, True, 6, 3), (80, 80, False, 5, 5), (80, 32, False, 20, 20), (256, 256, True, 4, 1),
          (96, 48, False, 3, 3), (16, 0, False, 2, 17), (16, 16, False, 2, 2), (192, 24, True, 7, 7), (144, 144, False, 9, 9)]


@pytest.mark.parametrize("dim,rot,interleaved,q_heads,kv_heads", SHAPES)
@pytest.mark.parametrize("kind,cache", [("bf16", "e4m3"), ("fp16", "int8"), ("fp32", "e4m3"), ("fp32", "int8"), ("bf16", "int8")])
def test_prompts_match_64_bits(dim, rot, interleaved, q_heads, kv_heads, kind, cache):
    for layout, page, block, counts in (("nhd", 16, 16, [600]), ("hnd", 48, 24, [1, 300, 17, 400, 5]), ("nhd", 8, 1, [520, 3]), ("hnd", 256, 256, [700, 1, 90]),
                                        ("nhd", 128, 64, [65, 64, 63, 200, 300]), ("nhd", 12, 4, [2] * 300)):
        g = gen(dim + page)
        first = [(5 * i) % 37 for i in range(len(counts))]
        seq, index, table, pages = layout_of(g, counts, first, page, True)
        n = len(seq)
        assert n > 512
        c = Cache(g, cache, pages, page, block, kv_heads, dim, layout, order=(2, 0, 1) if block % 16 else (0, 1, 2))
        inv = (10000.0 ** (-torch.arange(rot // 2, device=DEV, dtype=torch.float64) / max(1, rot // 2))).float()
        pos = index + 1048575 if page == 16 else None
        q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV).to(DT[kind]) for h in (q_heads, kv_heads, kv_heads))
        size = torch.exp2(torch.randint(-7, 8, (n, 1, 1), generator=g, device=DEV).float()).to(DT[kind])
        k, v = k * size, v * size.flip(0)
        v[::5] = 0
        run(c, table, seq, index, k, v, q, torch.full_like(q, 7.0) if page > 16 else None, pos, inv if rot else None, interleaved, 1.25)
        c.c.close()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("block,page", [(16, 16), (64, 64), (32, 128), (256, 256), (1, 4), (48, 48)])
def test_calls_that_end_and_go_on_inside_blocks(block, page, kind):
    """Prompts in several calls, growing and shrinking: scales rise and stay, the
    elements of earlier calls are rounded again."""
    g = gen(block)
    S, counts = 2, (523, 600, 1001, 530)
    start = [3, 21]
    table, pages = table_of(g, [s + sum(counts) for s in start], page)
    c = Cache(g, kind, pages, page, block, 3, 64)
    inv = (10000.0 ** (-torch.arange(32, device=DEV) / 32)).float()
    for i, n in enumerate(counts):
        seq = torch.arange(S, dtype=torch.int32, device=DEV).repeat_interleave(n)
        index = torch.cat([torch.arange(s, s + n, dtype=torch.int32, device=DEV) for s in start])
        size = 2.0 ** (0, 6, -4, 9)[i]
        k, v = ((torch.randn(S * n, 3, 64, generator=g, device=DEV) * size).to(torch.bfloat16) for _ in range(2))
        run(c, table, seq, index, k, v, inv=inv)
        start = [s + n for s in start]
    c.c.close()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("shift", [8, 1])  # 16-byte pieces, and odd alignment (the element-by-element kernel, several runs a CTA)
@pytest.mark.parametrize("block,page", [(16, 16), (4, 32), (128, 128)])
def test_sliced_inputs_with_queries_in_place(block, page, shift, kind):
    g = gen(block + shift)
    QH, H, D, counts = 4, 2, 64, [700, 1, 64, 130]
    seq, index, table, pages = layout_of(g, counts, [0, 9, 16, 3], page, True)
    n = len(seq)
    c = Cache(g, kind, pages, page, block, H, D)
    packed = torch.randn(n, (QH + 2 * H) * D + 16, generator=g, device=DEV).to(torch.bfloat16)
    rows = packed[:, shift:shift + (QH + 2 * H) * D]
    q, k, v = (t.unflatten(1, (-1, D)) for t in rows.split([QH * D, H * D, H * D], dim=1))
    before = packed.clone()
    inv = (10000.0 ** (-torch.arange(D // 2, device=DEV) / (D // 2))).float()
    run(c, table, seq, index, k, v, q, None, None, inv)
    assert torch.equal(packed[:, :shift], before[:, :shift]) and torch.equal(packed[:, shift + QH * D:], before[:, shift + QH * D:])
    c.c.close()


@pytest.mark.parametrize("dim,rot", [(80, 40), (64, 20), (32, 6)])  # rotated halves that fill no pieces
def test_odd_rotations(dim, rot):
    g = gen(rot)
    seq, index, table, pages = layout_of(g, [600, 33], [0, 7], 16, True)
    n = len(seq)
    c = Cache(g, "e4m3", pages, 16, 8, 3, dim)
    inv = (10000.0 ** (-torch.arange(rot // 2, device=DEV) / (rot // 2))).float()
    q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV).to(torch.float16) for h in (6, 3, 3))
    run(c, table, seq, index, k, v, q, torch.full_like(q, 7.0), None, inv)
    c.c.close()


@pytest.mark.parametrize("typ", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("block,page", [(16, 16), (64, 64)])
def test_special_values(block, page, kind, typ):
    """NaN, infinities, zeros, subnormal and the largest numbers, alone in their blocks and
    among others; a block of nothing else."""
    g = gen(3)
    n, H, D = 640, 9, 64
    table, pages = table_of(g, [n], page)
    c = Cache(g, kind, pages, page, block, H, D)
    k, v = (torch.randn(n, H, D, generator=g, device=DEV).to(DT[typ]) for _ in range(2))
    big, tiny = torch.finfo(DT[typ]).max, torch.finfo(DT[typ]).smallest_normal / 4
    for t in (k, v):
        t[5, 0, 3] = float("nan")
        t[70, 1, 0], t[71, 1, 63] = float("inf"), -float("inf")
        t[100, 2, 9] = big
        t[192:256, 3] = 0.0
        t[256:320, 4] = float("nan")
        t[320:384, 5] = float("inf")
        t[384:448, 6] = tiny
        t[448:512, 7] = -big
        t[600, 8, 60], t[601, 8, 1] = float("nan"), -float("inf")
    seq, index = torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    run(c, table, seq, index, k, v, status=1 if kind == "int8" else 0)
    # again from inside a block, over what is there
    at = slice(3, None)
    run(c, table, seq[at], index[at], k[at], v[at], status=1 if kind == "int8" else 0)
    c.c.close()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_bad_pages_are_skipped_and_reported(kind):
    g = gen(4)
    page, block, n = 32, 8, 300
    table, pages = table_of(g, [n, n, n], page)
    c = Cache(g, kind, pages, page, block, 2, 64)
    table[1, 2], table[2, 0], table[0, 9] = pages, -4, 2 ** 31 - 1
    seq, index = ints([0] * n + [1] * n + [2] * n + [7] * 20), torch.cat([torch.arange(n, dtype=torch.int32, device=DEV)] * 3 + [ints(range(20))])
    k, v, q = (torch.randn(len(seq), h, 64, generator=g, device=DEV).to(torch.bfloat16) for h in (2, 2, 4))
    skipped = list(range(288, 300)) + list(range(n + 64, n + 96)) + list(range(2 * n, 2 * n + 32)) + list(range(3 * n, 3 * n + 20))
    run(c, table, seq, index, k, v, q, status=1, skipped=skipped)
    # past the table's columns
    seq, index = seq[:600], torch.arange(20, 620, dtype=torch.int32, device=DEV)
    table[0, 9] = 3
    run(c, table, seq * 0, index, k[:600], v[:600], status=1, skipped=range(300, 600))
    c.c.close()


def test_disorder_is_reported():
    """An index that goes back, one that jumps, a sequence that comes again, at the start, inside
    and at the end of a call; the blocks of other sequences are as they should be."""
    g = gen(5)
    page, block, n = 16, 8, 900
    table, pages = table_of(g, [700, 700], page)
    c = Cache(g, "e4m3", pages, page, block, 2, 64)
    k, v = (torch.randn(n, 2, 64, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    good = torch.cat([torch.arange(600, dtype=torch.int32, device=DEV), torch.arange(300, dtype=torch.int32, device=DEV)])
    seq = ints([0] * 600 + [1] * 300)
    run(c, table, seq, good, k, v)
    for where in (1, 40, 599):
        for other in (where - 1, where + 2):  # back (or the same place), and a jump
            index = good.clone()
            index[where:600] += other - where
            c.c.append(k, v, table, index, seq=seq)
            assert c.c.status() == 1, (where, other)
            check_half_of_sequence(c, table, k, v, 1, 600, 300)
    again = seq.clone()
    again[880:] = 0
    index = good.clone()
    index[880:] = torch.arange(650, 670, dtype=torch.int32, device=DEV)
    c.c.append(k, v, table, index, seq=again)
    assert c.c.status() == 1
    # with padding between sequences, but not among one's tokens
    index = good.clone()
    index[300] = -1
    c.c.append(k, v, table, index, seq=seq)
    assert c.c.status() == 1
    c.c.close()


def check_half_of_sequence(c, table, k, v, s, at, n):
    """Sequence s, appended from its first place on by tokens at .. at + n."""
    j = torch.arange(n, device=DEV)
    page, place = table[s, j // c.page].long(), j % c.page
    for x, t, scale in ((k, c.k, c.ks), (v, c.v, c.vs)):
        x = x[at:at + n].double()
        unit = scale[page, place // c.block].double()[..., None]
        high = torch.zeros(-(-n // c.block), x.shape[1], dtype=torch.float64, device=DEV)
        high = high.scatter_reduce(0, (j // c.block)[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
        assert torch.equal(unit[..., 0], needed(high, TOP[c.kind])[j // c.block])
        assert ((nhd(t, c.layout)[page, place].double() - x / unit).abs() <= half_step(c.kind, x / unit)).all()


@pytest.mark.parametrize("block", [4, 16])
def test_as_many_sequences_as_tokens(block):
    """A decode step of more than 512 sequences, with and without `seq`."""
    g = gen(block)
    S = 700
    lens = torch.randint(1, 60, (S,), generator=torch.Generator().manual_seed(1)).tolist()
    table, pages = table_of(g, lens, 16)
    index = ints([x - 1 for x in lens])
    seq = torch.arange(S, dtype=torch.int32, device=DEV)
    k, v, q = (torch.randn(S, h, 128, generator=g, device=DEV).to(torch.bfloat16) for h in (4, 4, 8))
    inv = (10000.0 ** (-torch.arange(64, device=DEV) / 64)).float()
    caches = [Cache(gen(9), "int8", pages, 16, block, 4, 128) for _ in range(2)]
    run(caches[0], table, seq, index, k, v, q.clone(), None, None, inv)
    caches[1].c.append(k, v, table, index, inv_freq=inv)
    assert caches[1].c.status() == 0
    for name in ("k", "v", "ks", "vs"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))
    for c in caches:
        c.c.close()


@pytest.mark.parametrize("n", [512, 513])
def test_both_kernels_give_the_same(n):
    """The two sides of the rule on tokens, each with aligned and unaligned input: the
    same bits."""
    g = gen(6)
    page, H, D = 32, 5, 128
    table, pages = table_of(g, [n], page)
    wide = torch.randn(n, 2, H, D + 8, generator=g, device=DEV).to(torch.bfloat16)
    odd = wide[..., 1:D + 1].contiguous()
    holder = torch.empty(2 * n * H * D + 1, dtype=torch.bfloat16, device=DEV)
    seq, index = torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    caches = [Cache(gen(9), "e4m3", pages, page, 16, H, D) for _ in range(2)]
    for c, at in zip(caches, (0, 1)):
        x = holder[at:at + odd.numel()].view(odd.shape)
        x.copy_(odd)
        c.c.append(x[:, 0], x[:, 1], table, index, seq=seq)
        assert c.c.status() == 0
    for name in ("k", "v", "ks", "vs"):
        assert torch.equal(raw(getattr(caches[0], name)), raw(getattr(caches[1], name)))
    for c in caches:
        c.c.close()


def test_prompts_in_a_graph():
    g = gen(7)
    n, H, D, page = 800, 4, 64, 16
    table, pages = table_of(g, [n], page)
    c = Cache(g, "int8", pages, page, 8, H, D)
    seq, index = torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    inv = (10000.0 ** (-torch.arange(D // 2, device=DEV) / (D // 2))).float()
    q, k, v = (torch.zeros(n, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(3))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.c.append(k, v, table, index, seq=seq, inv_freq=inv, q=q, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        q0 = q.clone()
        other = Cache(gen(1), "int8", pages, page, 8, H, D)
        graph.replay()
        other.c.append(k, v, table, index, seq=seq, inv_freq=inv, q=q0)
        used = table[0].long()
        torch.cuda.synchronize()
        assert torch.equal(q, q0)
        for name in ("k", "v", "ks", "vs"):
            assert torch.equal(getattr(c, name)[used], getattr(other, name)[used])
        other.c.close()
    assert c.c.status() == 0
    c.c.close()


@pytest.mark.parametrize("block", [4, 16])
def test_more_sequences_without_seq_than_the_first_kernel_takes(block):
    g = gen(block)
    S = 2500
    lens = torch.randint(1, 20, (S,), generator=torch.Generator().manual_seed(1)).tolist()
    table, pages = table_of(g, lens, 16)
    k, v = (torch.randn(S, 2, 64, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(S, 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    inv = (10000.0 ** (-torch.arange(32, device=DEV) / 32)).float()
    c = Cache(g, "int8", pages, 16, block, 2, 64)
    before, had, q0 = [raw(t).clone().view(t.dtype) for t in (c.k, c.v)], [c.ks.clone(), c.vs.clone()], q.clone()
    index = ints([x - 1 for x in lens])
    c.c.append(k, v, table, index, inv_freq=inv, q=q)
    assert c.c.status() == 0
    at = torch.arange(S, device=DEV)
    page, place = table[at, index.long() // 16].long(), index.long() % 16
    keys, mag = rope64(k, index, inv, False)
    check_half(c, "k", before[0], had[0], keys, 2.0 ** -20 * mag, page, place)
    check_half(c, "v", before[1], had[1], v.double(), torch.zeros_like(mag), page, place)
    want, mag = rope64(q0, index, inv, False)
    assert ((q.double() - want).abs() <= half_step("bf16", want) + 2.0 ** -20 * mag).all()
    c.c.close()


def test_a_sequence_that_comes_again_is_found_wherever_it_was():
    """Among one-token sequences in any order: next but one, in the same tile, in the same CTA's
    tokens, and far behind; padding of the same number does not count."""
    g = gen(8)
    n, page = 2100, 16
    table, pages = table_of(g, [16] * (n + 3), page)
    c = Cache(g, "int8", pages, page, 8, 1, 16)
    k, v = (torch.randn(n, 1, 16, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    for order in (torch.arange(n), torch.randperm(n, generator=torch.Generator().manual_seed(2)), torch.arange(n).flip(0)):
        seq, index = order.to(torch.int32).to(DEV), torch.full((n,), 8, dtype=torch.int32, device=DEV)
        c.c.append(k, v, table, index, seq=seq)
        assert c.c.status() == 0
        for first, then in ((0, 2), (5, 7), (15, 17), (16, 31), (0, n - 1), (700, 1801), (n - 3, n - 1), (31, 33), (1023, 2047)):
            again, places = seq.clone(), index.clone()
            again[then] = again[first]
            places[then] = 0  # (another block: what is stored is defined)
            c.c.append(k, v, table, places, seq=again)
            assert c.c.status() == 1, (first, then)
            places[first] = -1
            c.c.append(k, v, table, places, seq=again)
            assert c.c.status() == 0, (first, then)
    c.c.close()
