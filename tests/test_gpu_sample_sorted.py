"""GPU: sampling among more candidates than a CTA has threads, which its first CTA
sorts several a thread, twice: by logit, and the kept ones by index.  The plain form,
its margins and the tolerances are those of test_gpu_sample.py; a call repeated gives
the same bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402
from test_gpu_sample import DEV, DT, check, gen, logits_of, unit  # noqa: E402


def repeated(z, u, times, **how):
    rows, vocab = z.shape
    want = check(z, u, **how)
    kept, logprob = torch.empty(rows, dtype=torch.int32, device=DEV), torch.empty(rows, device=DEV)
    xg.sample(z, u, kept=kept, logprob=logprob, **how)
    wrong = torch.zeros((), dtype=torch.int64, device=DEV)
    k, l = torch.empty_like(kept), torch.empty_like(logprob)
    for _ in range(times):
        got = xg.sample(z, u, kept=k, logprob=l, **how)
        wrong += ((got != want) | (k != kept) | (l != logprob) | (got < 0) | (got >= vocab)).sum()
    assert int(wrong) == 0
    return kept


@pytest.mark.parametrize("kind,rows", [("bf16", 300), ("fp32", 148)])
@pytest.mark.parametrize("how", [dict(), dict(top_p=0.95), dict(min_p=0.01)], ids=lambda h: "-".join(h) or "all")
def test_top_k_above_a_ctas_threads(how, kind, rows):
    k = torch.linspace(513, 1536, rows, device=DEV).to(torch.int32)
    kept = repeated(logits_of(rows, rows, 32003, kind, slope=0.6), unit(1, rows), 300, top_k=k, **how)
    assert int(kept.max()) > 512


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
def test_nucleus_above_a_ctas_threads(kind):
    # up to 1800 likely tokens, in runs of eight that the first guess sees as one: about as many candidates
    rows, vocab = 200, 32000
    z = torch.rand((rows, vocab), generator=gen(2), device=DEV).clamp_(min=1e-12).log_().mul_(3.0).sub_(6.0)
    run = torch.rand((rows, vocab // 8), generator=gen(3), device=DEV).argsort(1)
    near = run < torch.linspace(90, 225, rows, device=DEV)[:, None]
    likely = -torch.rand((rows, vocab), generator=gen(4), device=DEV)
    z = torch.where(near.repeat_interleave(8, 1), likely, z).to(DT[kind])
    kept = repeated(z, unit(5, rows), 300, top_p=0.9)
    assert int((kept > 512).sum()) > rows // 2 and int(kept.max()) <= 2048
