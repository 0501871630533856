"""GPU: sampling where sums of the same weights in another order fall on both sides of
top-p's border.  The rows are made in 80-bit arithmetic."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402
from test_gpu_sample import DT, check, gen, unit  # noqa: E402

DEV = "cuda:0"


def halves(rng, first=20400, second=20556):
    """FP32 logits whose nearest `first` tokens (of a distance below 2^-15) weigh half
    of all, but for some 1e-11: the tokens beyond them are near -0.008, and two far ones
    bring their sum to that of the first."""
    near = -np.exp2(rng.uniform(-31, -15, first)).astype(np.float32)
    near[0] = 0.0
    far = -rng.uniform(0.0068, 0.0090, second).astype(np.float32)
    exp = lambda z: np.exp(z.astype(np.longdouble))
    goal = exp(near).sum() + np.longdouble(rng.uniform(-1e-11, 1e-11))
    # all of the far ones by one shift, a little short; then what is missing as two small weights
    far = (far + np.float32(np.log((goal - np.longdouble(2e-5)) / exp(far).sum()))).astype(np.float32)
    rest = exp(far).sum()
    for spare in (1e-9, 0.0):
        one = np.float32(np.log(goal - rest))
        while rest + exp(one) > goal - np.longdouble(spare):
            one = np.nextafter(one, np.float32(-np.inf))
        far, rest = np.append(far, one), rest + exp(one)
    z = np.concatenate([near, far])
    rng.shuffle(z)
    return z


def test_nucleus_whose_parts_fall_short_of_their_whole():
    """Each row's nucleus is its first 20400 tokens, or one more or less: sums of 40958
    weights in 64 bits are off by far less than a weight."""
    rng = np.random.default_rng(11)
    rows, first = 96, 20400
    z = np.stack([halves(rng) for _ in range(rows)])
    u = torch.from_numpy(rng.random(rows, np.float32)).to(DEV)
    kept, logprob = torch.empty(rows, dtype=torch.int32, device=DEV), torch.empty(rows, device=DEV)
    tokens = xg.sample(torch.from_numpy(z).to(DEV), u, top_p=0.5, kept=kept, logprob=logprob)
    count = kept.cpu().numpy()
    assert (np.abs(count - first) <= 1).all(), count[np.abs(count - first) > 1]
    # a kept token's weight lies within 2^-15 of 1, their sum within 0.06 of 20400, and
    # a token more or less is 2^-14.3 of it: a share is 1 / 20400 to 2^-13.5.  Tokens are
    # drawn by index, of almost equal weights: the n-th where n / 20400 passes u, or one next to it
    assert (np.abs(logprob.cpu().numpy() + math.log(first)) <= 2.0 ** -13.5).all()
    for r in range(rows):
        at = np.flatnonzero(z[r] > -2.0 ** -14)
        assert len(at) == first
        token = int(tokens[r])
        assert abs(int(np.searchsorted(at, token)) - float(u[r]) * first) <= 3, r


@pytest.mark.parametrize("kind", ["fp16", "fp32"])
@pytest.mark.parametrize("values", [1, 2, 5, 300])
@pytest.mark.parametrize("rows,vocab", [(3, 40001), (300, 9001), (2, 128256)])
def test_more_tokens_near_the_largest_than_candidates(rows, vocab, values, kind):
    """Flat and heavily tied rows: thousands of tokens lie as near as the guess of few, so
    that the border is found among all of them, by index where it is one logit's."""
    level = torch.cat([torch.zeros(1, device=DEV), -torch.rand(values - 1, generator=gen(values), device=DEV) * 2])
    z = level[torch.randint(0, values, (rows, vocab), generator=gen(rows), device=DEV)].to(DT[kind])
    for how in (dict(top_p=0.9), dict(top_p=0.31), dict(top_p=0.0625, temperature=0.5), dict(top_p=0.97, min_p=0.3)):
        # (equal logits weigh 1 each, and 0.0625 of 128256 tokens is 8016: the border lies on
        # a sum, which no row of them is sure of; those sums are exact on both sides)
        border = values == 1 and (how["top_p"] * vocab).is_integer()
        check(z, unit(rows + 1, rows), least_sure=0.0 if border else 0.9, **how)
        if border:
            kept = torch.empty(rows, dtype=torch.int32, device=DEV)
            xg.sample(z, unit(rows + 1, rows), kept=kept, **how)
            assert (kept == int(how["top_p"] * vocab)).all()


@pytest.mark.parametrize("kind,rows,vocab", [("fp32", 600, 128256), ("bf16", 600, 256000)])
def test_many_rows_that_their_ctas_do_not_hold(kind, rows, vocab):
    z = torch.rand((rows, vocab), generator=gen(rows), device=DEV).clamp_(min=1e-12).log_().mul_(-0.9).to(DT[kind])
    u, some = unit(1, rows), slice(0, rows, 67)
    for how in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.95), dict(top_k=20000)):
        kept = torch.empty(rows, dtype=torch.int32, device=DEV)
        tokens = xg.sample(z, u, kept=kept, **how)
        assert torch.equal(check(z[some].contiguous(), u[some].contiguous(), **how), tokens[some])
        assert ((tokens >= 0) & (tokens < vocab)).all() and (kept > 0).all()
