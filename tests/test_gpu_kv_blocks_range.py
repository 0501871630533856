"""GPU: attention over block scales of any size (KVCache.attend), up to values that the
result's type just holds, and far apart within a sequence.  The 64-bit form and its
tolerances are those of test_gpu_kv_blocks.py: sums are in units of the largest scale, a
power of two, so that no product or sum of them leaves FP32's range, and what falls
below 2^-126 of that scale is far below the bound's 2^-40 of the largest value."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv_blocks import DEV, DT, TOP, Cache, attend64, gen, half_step, ints, nhd, table_of  # noqa: E402


def attended(c, q, table, lens, tiny=0.0, **how):
    out, lse = torch.full_like(q, 9.0), torch.empty(q.shape[:2], device=DEV)
    c.c.attend(q, table, ints(lens), out, lse=lse, **how)
    assert c.c.status() == 0
    want, wlse, tol, tlse = attend64(q, c.stands_for("k"), c.stands_for("v"), lens, table, c.page, q.shape[2] ** -0.5, **how)
    kind = "bf16" if q.dtype == torch.bfloat16 else "fp16"
    bad = ~((out.double() - want).abs() <= half_step(kind, want) + tol + tiny)
    assert not bad.any(), (int(bad.sum()), float(out[bad][0]), float(want[bad][0]))
    some = ~torch.isinf(wlse)
    assert ((lse.double() - wlse).abs() <= tlse)[some].all()
    return out, want


@pytest.mark.parametrize("wide", [0, 5000], ids=["cluster", "split"])
@pytest.mark.parametrize("block", [16, 4])
@pytest.mark.parametrize("kind,top", [("int8", 120), ("e4m3", 118)])  # 127 2^120 and 448 2^118 are below 2^127
@pytest.mark.parametrize("Q,H,D", [(8, 2, 128), (5, 5, 80), (24, 2, 64), (16, 1, 256)])
def test_values_up_to_the_largest(Q, H, D, kind, top, block, wide):
    g = gen(D)
    lens = [777, 1, 64, 300]
    table, pages = table_of(g, lens, 16, slack=wide)
    c = Cache(g, kind, pages, 16, block, H, D)
    q = torch.randn(len(lens), Q, D, generator=g, device=DEV).to(torch.bfloat16)
    for e in (top, 113, 100):
        c.vs.fill_(2.0 ** e)
        out, _ = attended(c, q, table, lens)
        assert torch.isfinite(out).all()
    # any elements: the largest that there are
    c.vs.fill_(2.0 ** top)
    raw = torch.full_like(nhd(c.v, c.layout), TOP[kind]) if kind == "int8" else torch.full(c.v.shape, TOP[kind], device=DEV).to(c.v.dtype)
    c.v.view(torch.uint8).copy_(raw.view(torch.uint8))
    out, want = attended(c, q, table, lens)
    assert torch.isfinite(out).all() and float(want.abs().max()) > 2.0 ** 126
    c.c.close()


@pytest.mark.parametrize("wide", [0, 9000], ids=["cluster", "split"])
@pytest.mark.parametrize("block", [16, 8, 1])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_value_scales_from_the_least_to_the_largest(kind, block, wide):
    """Each block and head its own scale between 2^-60 and 2^118, in any order; and rising or
    falling along the sequence."""
    g = gen(block)
    lens = [500, 33, 2000]
    table, pages = table_of(g, lens, 16, slack=wide)
    c = Cache(g, kind, pages, 16, block, 2, 64)
    q = torch.randn(3, 8, 64, generator=g, device=DEV).to(torch.bfloat16)
    c.vs.copy_(torch.exp2(torch.randint(-60, 119, c.vs.shape, generator=g, device=DEV).float()))
    attended(c, q, table, lens)
    attended(c, q, table, lens, window=40)
    for falling in (False, True):
        for i, n in enumerate(lens):
            e = torch.linspace(-60, 118, -(-n // 16), device=DEV).round()
            e = e.flip(0) if falling else e
            c.vs[table[i, :len(e)].long()] = torch.exp2(e)[:, None, None]
        attended(c, q, table, lens)
    # the last block alone is large, and small with the rest zeros
    c.vs.fill_(2.0 ** -60)
    c.vs[table[2, 124].long()] = 2.0 ** 118
    attended(c, q, table, lens)
    c.c.close()


@pytest.mark.parametrize("wide", [0, 9000], ids=["cluster", "split"])
@pytest.mark.parametrize("e", [-60, -100, -126, -133])
def test_small_value_scales(e, wide):
    """Scales down to the smallest numbers; the result's own smallest step is 2^-133."""
    g = gen(5)
    lens = [400, 17]
    table, pages = table_of(g, lens, 16, slack=wide)
    c = Cache(g, "int8", pages, 16, 16, 2, 64)
    q = torch.randn(2, 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    c.vs.fill_(2.0 ** e)
    attended(c, q, table, lens, tiny=2.0 ** -134 + 400 * 2.0 ** -149)
    c.c.close()


def test_many_values_of_the_largest_size():
    """20000 tokens, whose plain sum is 2^141."""
    g = gen(6)
    table, pages = table_of(g, [20000], 64)
    c = Cache(g, "int8", pages, 64, 16, 1, 64)
    c.vs.fill_(2.0 ** 120)
    c.v.fill_(127)
    q = torch.randn(1, 4, 64, generator=g, device=DEV).to(torch.bfloat16) * 0.01
    out, want = attended(c, q, table, [20000])
    assert torch.isfinite(out).all() and float(want.min()) > 2.0 ** 126
    c.c.close()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_of_the_largest_numbers_then_attend(kind):
    g = gen(7)
    n = 40
    table, pages = table_of(g, [n], 16)
    c = Cache(g, kind, pages, 16, 16, 1, 64)
    x = (torch.rand(n, 1, 64, generator=g, device=DEV) * 2 - 1) * 2.0 ** 126
    index = torch.arange(n, dtype=torch.int32, device=DEV)
    c.c.append((x * 2.0 ** -120), x, table, index, seq=torch.zeros_like(index))
    q = torch.randn(1, 4, 64, generator=g, device=DEV).to(torch.bfloat16) * 2.0 ** -6
    out, want = attended(c, q, table, [n])
    assert torch.isfinite(out).all() and float(want.abs().max()) > 2.0 ** 122
    c.c.close()


def test_a_neighbour_without_weight_costs_what_its_scale_says():
    """A token that holds all the weight next to one without any whose scale is 2^r as
    large: off by 2^-40 of the largest scale of the sixteen times its elements, and by
    the FP16 pair's 2^-22 of itself."""
    g = gen(8)
    D = 64
    c = Cache(g, "int8", 2, 16, 1, 1, D)
    table = ints([[0]])
    c.ks.fill_(2.0 ** -3)
    c.k.fill_(0)
    c.k[0, 0], c.k[0, 1] = 127, -127
    q = torch.full((1, 2, D), 1.0, device=DEV, dtype=torch.bfloat16)  # scores of 127 and -127: the other's weight is below 2^-300
    for r in (0, 10, 20, 30, 38):
        c.vs.fill_(1.0)
        c.vs[0, 1] = 2.0 ** r
        out = torch.empty_like(q)
        c.c.attend(q, table, ints([2]), out)
        v = c.v[0, 0, 0].double()
        bound = half_step("bf16", v) + 2.0 ** (r - 40) * v.abs() + 2.0 ** -22 * v.abs()
        assert ((out[0].double() - v).abs() <= bound).all(), r
    c.c.close()
