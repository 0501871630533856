"""GPU: sampling where sums of the same weights in another order fall on both sides of
top-p's border.  The rows are made in 80-bit arithmetic."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402

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
