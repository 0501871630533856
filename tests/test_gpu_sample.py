"""GPU: sampling (xksv_gpu.sample) against a plain form in 64 bits, at the sizes,
types, ties and settings where it can go wrong, and its refusals.

Tolerances: weights and sums are FP64 on both sides, added in different orders:
a sum of n weights of 2 ulp is off by (n + 2) 2^-52 relative at most, below 2^-31
for 2^21 tokens.  A token or a count whose border is nearer than MARGIN = 2^-30
to the sum that decides it may fall to either side; all others are exact.  The
FP32 log of a share is off by half a step, 2^-24 relative, and MARGIN."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MARGIN = 2.0 ** -30


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def plain(z, u, heat=1.0, k=0, p=1.0, m=0.0):
    """(token, kept, logprob, sure) of one row: `sure` is False where a border
    lies within MARGIN of what decides it."""
    z = np.asarray(z, np.float64)
    heat, p, m, u = (float(np.float32(x)) for x in (heat, p, m, u))
    if np.isnan(z).any() or not np.isfinite(z.max(initial=-np.inf)):
        return -1, 0, math.nan, True
    some = np.flatnonzero(z > -np.inf)
    order = some[np.argsort(-z[some], kind="stable")]
    if heat == 0.0:
        k, heat = 1, 1.0
    if k > 0:
        order = order[:k]
    w = np.exp((z[order] - z[order[0]]) / heat)
    total, sure = math.fsum(w), True
    n = len(w)
    if p < 1.0:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int(np.count_nonzero(before < p * total)))
        sure &= bool((np.abs(before[1:] - p * total) > MARGIN * total).all())
    low = max(math.exp(-700.0), min(m, 1.0) if m > 0 else 0.0)
    sure &= bool(((np.abs(w - low) > MARGIN * low) | (w == 1.0)).all())  # (exp(0) is exact)
    n = max(1, min(n, int(np.count_nonzero(w >= low))))
    order, w = order[:n], w[:n]
    at = np.argsort(order)
    up = np.cumsum(w[at])
    i = min(int(np.searchsorted(up, u * up[-1], side="right")), n - 1)
    sure &= bool((np.abs(up[:-1] - u * up[-1]) > MARGIN * up[-1]).all())
    return int(order[at[i]]), n, math.log(w[at[i]] / up[-1]), sure


def check(logits, u, least_sure=0.9, **how):
    """The call's tokens, counts and logs against the plain form's, row by row."""
    rows = logits.shape[0]
    kept = torch.full((rows,), -7, dtype=torch.int32, device=DEV)
    logprob = torch.full((rows,), 7.0, device=DEV)
    tokens = xg.sample(logits, u, kept=kept, logprob=logprob, **how)
    torch.cuda.synchronize()
    at = {n: v.tolist() if torch.is_tensor(v) else [v] * rows for n, v in how.items()}
    z, us = logits.double().cpu().numpy(), u.tolist()
    names = dict(temperature="heat", top_k="k", top_p="p", min_p="m")
    sure = 0
    for r in range(rows):
        token, n, log, ok = plain(z[r], us[r], **{names[x]: at[x][r] for x in how})
        sure += ok
        if not ok:
            continue
        assert (int(tokens[r]), int(kept[r])) == (token, n), (r, us[r], {x: at[x][r] for x in how})
        got = float(logprob[r])
        assert got == log or math.isnan(got) and math.isnan(log) or abs(got - log) <= 2.0 ** -24 * abs(log) + MARGIN, (r, got, log)
    assert sure >= least_sure * rows
    return tokens


def logits_of(seed, rows, vocab, kind, slope=1.0, extra=0):
    z = torch.rand((rows, vocab + extra), generator=gen(seed), device=DEV).clamp_(min=1e-12).log_().mul_(-slope)
    return z.sub_(4.0).to(DT[kind])[:, extra:]


def unit(seed, rows):
    return torch.rand(rows, generator=gen(seed), device=DEV)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 255, 1000, 4097, 32003])
def test_small_and_odd_vocabularies(vocab, kind):
    z = logits_of(vocab, 5, vocab, kind, extra=vocab % 8)
    u = unit(vocab + 1, 5)
    check(z, u)
    check(z, u, temperature=0.6, top_k=3)
    check(z, u, temperature=1.3, top_p=0.8)
    check(z, u, top_k=20, top_p=0.9, min_p=0.05)
    check(z, u, temperature=0.0)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 3, 40, 150])
def test_large_vocabulary_each_row_its_settings(rows, kind):
    rng = np.random.default_rng(rows)
    pick = lambda v, t: torch.from_numpy(rng.choice(np.array(v, t), rows)).to(DEV)
    z = logits_of(rows, rows, 128256, kind, slope=0.9)
    check(z, unit(rows, rows), temperature=pick([0, 0.3, 0.7, 1, 1.5], np.float32), top_k=pick([-1, 0, 1, 2, 50, 1000, 5000, 200000], np.int32),
          top_p=pick([1, 1.5, 0.5, 0.9, 0.99, 0.0], np.float32), min_p=pick([0, -1, 0.02, 0.3, 1, 2], np.float32))


@pytest.mark.parametrize("how", [dict(), dict(top_k=100000), dict(top_p=0.97), dict(top_k=60000, top_p=0.9), dict(min_p=1e-4),
                                 dict(temperature=50.0, top_p=0.5), dict(temperature=0.05, top_k=100), dict(temperature=1e6, top_p=0.3)],
                         ids=lambda h: "-".join(h) or "none")
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_many_kept_tokens(kind, how):
    check(logits_of(5, 4, 151936, kind, slope=0.4), unit(6, 4), **how)


@pytest.mark.parametrize("how", [dict(), dict(top_k=1500), dict(top_k=5), dict(top_p=0.5), dict(top_p=0.31, top_k=30000),
                                 dict(min_p=1.0), dict(top_k=1024), dict(top_k=1025)], ids=lambda h: "-".join(f"{k}{v}" for k, v in h.items()) or "none")
@pytest.mark.parametrize("values", [1, 2, 5])
def test_ties_go_to_the_lowest_index(values, how):
    # 40001 tokens of one, two or five different logits, 0 and -0 among them
    level = torch.tensor([0.0, -0.0, 0.5, -0.25, 1.0], device=DEV)
    at = torch.randint(0, values, (3, 40001), generator=gen(values), device=DEV)
    check(level[at].to(torch.bfloat16), unit(3, 3), **how)


def test_more_ties_around_zero_than_the_candidate_list_holds():
    # logits so near zero that their bits spread over the whole range of keys
    z = torch.randn((2, 50000), generator=gen(1), device=DEV) * 1e-3
    z[:, ::3] = 0.0
    z[:, 1::3] *= 1e-30
    for how in (dict(top_p=0.5), dict(top_k=25000), dict(top_p=0.2, top_k=30000), dict(temperature=0.001, top_p=0.9)):
        check(z, unit(2, 2), **how)


def test_masked_tokens():
    z = logits_of(8, 6, 32000, "fp32")
    keep = torch.rand(z.shape, generator=gen(9), device=DEV) < 0.001
    keep[:, 77] = True
    for fill in (-math.inf, torch.finfo(torch.float32).min, -1e9):
        m = torch.where(keep, z, torch.full_like(z, fill))
        for how in (dict(), dict(top_k=10), dict(top_k=5000), dict(top_p=0.9), dict(top_k=20000, top_p=0.95), dict(temperature=0.0)):
            check(m, unit(10, 6), **how)
    one = torch.full((2, 32000), -math.inf, device=DEV)
    one[0, 31999] = -3.0
    one[1, 0] = 1e30
    check(one, unit(11, 2))
    check(one, unit(11, 2), top_k=4, top_p=0.5)


def test_rows_without_a_distribution():
    z = logits_of(1, 6, 5000, "fp16")
    z[0] = -math.inf
    z[1, 4999] = math.nan
    z[2, 3] = math.inf
    z[3, 0] = math.nan
    z[3, 1] = math.inf
    for how in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.5)):
        got = check(z, unit(2, 6), least_sure=0.0 if how else 0.9, **how)
        assert got[:4].tolist() == [-1, -1, -1, -1] and (got[4:] >= 0).all()
    heat = torch.tensor([-1.0, math.nan, math.inf, 1e-7, 1e7, 1.0], device=DEV)
    z = logits_of(1, 6, 5000, "fp16")
    kept, logprob = torch.empty(6, dtype=torch.int32, device=DEV), torch.empty(6, device=DEV)
    got = xg.sample(z, unit(2, 6), temperature=heat, kept=kept, logprob=logprob)
    assert got[:5].tolist() == [-1] * 5 and got[5] >= 0 and kept[:5].tolist() == [0] * 5 and logprob[:5].isnan().all()
    u = unit(2, 6)
    u[0] = math.nan
    assert xg.sample(z, u)[0] == -1
    bad = torch.full((6,), math.nan, device=DEV)
    assert (xg.sample(z, unit(2, 6), top_p=bad) == -1).all() and (xg.sample(z, unit(2, 6), min_p=bad) == -1).all()


@pytest.mark.parametrize("u", [0.0, -1.0, 1.0, 7.0, 1.0 - 2.0 ** -24])
def test_ends_of_the_draw(u):
    z = logits_of(3, 4, 9001, "fp32")
    z[:, 0] = -math.inf
    z[:, -1] = -math.inf
    us = torch.full((4,), u, device=DEV)
    for how in (dict(), dict(top_k=50)):
        got = xg.sample(z, us, **how)
        for r in range(4):
            some = z[r].topk(how.get("top_k", 8999)).indices
            if u <= 0:
                assert got[r] == some.min()
            elif u >= 1:
                assert got[r] == some.max()
    check(z, us.clamp(0, 1), least_sure=0.0)


def test_frequencies():
    # 2^17 draws among eight tokens: each count within 6 standard deviations
    z = torch.tensor([0.0, 1.0, 2.0, -math.inf, 0.5, -1.0, 2.0, 1.5], device=DEV)
    n = 1 << 17
    got = xg.sample(z.expand(n, 8), unit(1, n), temperature=0.8)
    p = torch.softmax(z.double() / 0.8, 0)
    count = torch.bincount(got, minlength=8).double()
    assert ((count - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_vocabulary_larger_than_shared_memory(kind):
    vocab = 1000003
    z = logits_of(4, 2, vocab, kind, slope=0.5, extra=3)
    for how in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.9), dict(top_k=300000)):
        check(z, unit(5, 2), **how)


def test_same_call_same_tokens_and_neighbours_untouched():
    z = logits_of(12, 33, 50257, "bf16", slope=0.7)
    u = unit(13, 33)
    box = torch.full((35,), 99, dtype=torch.int64, device=DEV)
    a = xg.sample(z, u, tokens=box[1:34], top_p=0.93).clone()
    assert box[0] == 99 and box[34] == 99
    for _ in range(5):
        assert torch.equal(xg.sample(z, u, top_p=0.93), a)
    # a row's token does not depend on the rows beside it (nor on how a row is
    # split over CTAs, but for sums that lie next to a border)
    one = torch.cat([xg.sample(z[r:r + 1], u[r:r + 1], top_p=0.93) for r in range(33)])
    sure = [plain(z[r].double().cpu().numpy(), float(u[r]), p=0.93)[3] for r in range(33)]
    assert all(x == y for x, y, ok in zip(a.tolist(), one.tolist(), sure) if ok)


def test_streams_and_graphs():
    z, u = logits_of(14, 8, 32000, "bf16"), unit(15, 8)
    want = xg.sample(z, u, top_k=50, temperature=0.9)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = xg.sample(z, u, top_k=50, temperature=0.9, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.zeros(8, dtype=torch.int64, device=DEV)
    with torch.cuda.graph(graph):
        xg.sample(z, u, tokens=out, top_k=50, temperature=0.9, stream=torch.cuda.current_stream().cuda_stream)
    for seed in (16, 17):
        z.copy_(logits_of(seed, 8, 32000, "bf16"))
        u.copy_(unit(seed, 8))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, xg.sample(z, u, top_k=50, temperature=0.9))


def test_refusals():
    z, u = logits_of(1, 4, 100, "fp32"), unit(1, 4)
    for bad in (dict(logits=z.double()), dict(logits=z.t()), dict(logits=z[0]), dict(logits=z.cpu()), dict(u=u[:3]), dict(u=u.double()),
                dict(u=u.cpu()), dict(tokens=torch.empty(4, dtype=torch.int32, device=DEV)), dict(kept=torch.empty(4, device=DEV)),
                dict(logprob=torch.empty(3, device=DEV)), dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:2]),
                dict(min_p=torch.empty(8, device=DEV)[::2]), dict(u=None)):
        with pytest.raises((ValueError, AttributeError)):
            xg.sample(**{**dict(logits=z, u=u), **bad})
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=1e-8), dict(temperature=math.inf), dict(top_p=math.nan),
                dict(min_p=math.nan), dict(logits=torch.empty((1, (1 << 22) + 1), dtype=torch.bfloat16, device=DEV), u=u[:1]),
                dict(logits=torch.empty((4, 0), device=DEV))):
        with pytest.raises(RuntimeError):
            xg.sample(**{**dict(logits=z, u=u), **bad})
    assert xg.sample(z[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("vocab,rows", [(40009, 3), (40009, 170), (901, 20)])
@pytest.mark.parametrize("centre,scale,heat", [(0.0, 3.0, 1.0), (0.0, 3e-4, 1e-3), (0.0, 1e-3, 1.0), (0.0, 0.02, 0.01), (-80.0, 20.0, 30.0),
                                               (300.0, 100.0, 50.0), (-1000.0, 3.0, 1.0), (0.0, 1e30, 1.0), (0.0, 2e5, 1e5), (5.0, 1e-30, 1.0)])
def test_nucleus_of_bf16_logits_of_any_magnitude(centre, scale, heat, vocab, rows):
    # logits near zero, far from it and on both sides; zeros and masked tokens among them
    z = torch.randn((rows, vocab), generator=gen(rows), device=DEV) * scale + centre
    z[:, 5::11] = -math.inf
    z[:, 3::13] *= 0.0
    z[1::2, 0::17] = torch.finfo(torch.bfloat16).min
    z = z.to(torch.bfloat16)
    u = unit(rows + 1, rows)
    zero = torch.exp(-z.float().amax(1) / heat)  # as much as a logit of zero, relative to the largest
    share = torch.tensor([0.02, 0.3, 0.6, 0.9, 0.999, 0.5], device=DEV).repeat(rows // 6 + 1)[:rows]
    check(z, u, temperature=heat, top_p=share)
    check(z, u, temperature=heat, top_p=share, min_p=0.02)
    check(z, u, temperature=heat, top_p=share, min_p=torch.where(zero < 1, zero, 0.5))


def test_nucleus_border_among_equal_logits_is_an_index():
    # BF16, 40001 tokens of seven logits: whichever CTA holds the border's last token, also at its ends
    level = torch.tensor([2.0, 1.0, 0.5, 0.0, -0.5, -1.0, -3.0], device=DEV)
    z = level[torch.randint(0, 7, (1, 40001), generator=gen(4), device=DEV)].to(torch.bfloat16).expand(64, -1)
    share = torch.linspace(0.01, 0.999, 64, device=DEV)
    check(z, unit(5, 64), top_p=share)
    check(z[:8], torch.ones(8, device=DEV) - 2.0 ** -24, top_p=share[::8].contiguous())  # the last kept token
    # (0.01 in FP32 is 2.2e-10 short of 400 tokens of 40000, which is nearer than MARGIN: one row of the four is not sure)
    check(torch.zeros((4, 40000), device=DEV, dtype=torch.bfloat16), unit(6, 4), least_sure=0.75, top_p=share[::16].contiguous())


@pytest.mark.parametrize("bad", [dict(temperature=1e300), dict(top_k=2.5), dict(top_p="0.9"), dict(min_p=None), dict(top_k=None)], ids=str)
def test_settings_that_are_no_numbers_of_their_type(bad):
    # (1e300 is FP32's infinity, which the library refuses; the others are refused ahead of it)
    with pytest.raises(RuntimeError if bad.get("temperature") else ValueError):
        xg.sample(logits_of(1, 4, 100, "fp32"), unit(1, 4), **bad)
    assert (xg.sample(logits_of(1, 4, 100, "fp32"), unit(1, 4), top_k=10 ** 12) >= 0).all()
