"""GPU: sessions with 8-bit blocks and sampled continuations, against the model's
own Transformers forward (the models, archives and tolerances of
test_gpu_serve.py)."""
import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu

import xksv_runtime as rt  # noqa: E402
import xksv_serve as serve  # noqa: E402
from test_gpu_serve import DEV, archive, close  # noqa: E402


@pytest.mark.parametrize("name", ["llama", "qwen2", "mistral"])
@pytest.mark.parametrize("kv,block", [("e4m3-blocks", None), ("int8-blocks", None), ("int8-blocks", 2), ("e4m3-blocks", 1)])
def test_session_with_block_scales_matches_transformers(tmp_path, name, kv, block):
    """An 8-bit cache rounds keys and values by 2^-4 more (E4M3; integers by half a
    step of 1/64 of a block's largest), as the per-head E4M3 cache does: its tolerance."""
    path = archive(tmp_path, name)
    ref, _, _ = rt.load_archive(path, DEV)
    s = serve.load_session(path, DEV, pages=64, page_size=8, max_seqs=4, kv_dtype=kv, kv_block=block)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 256, (n,), generator=g) for n in (1, 40, 17)]
    ids = [p.to(DEV) for p in prompts]
    with torch.no_grad():
        seqs, logits = s.prefill(prompts)
        for step in range(12):
            want = torch.stack([ref(x[None]).logits[0, -1] for x in ids])
            assert close(logits, want, 1e-1), step
            order = [0, 1, 2] if step % 3 else [2, 0]
            token = want.argmax(-1)
            if len(order) < 3:
                part = s.step([seqs[i] for i in order], token[torch.tensor(order, device=DEV)])
                rest = s.step([seqs[1]], token[1:2])
                logits = torch.stack([part[1], rest[0], part[0]])
            else:
                logits = s.step(seqs, token)
            ids = [torch.cat((x, t[None])) for x, t in zip(ids, token)]
    s._check()
    s.release(seqs)
    assert len(s.free_pages) == 64 and not s.length
    s.close()


def test_pages_are_taken_again_with_their_old_scales(tmp_path):
    """A sequence on pages that another one left: its blocks begin anew."""
    path = archive(tmp_path, "llama")
    s = serve.load_session(path, DEV, pages=6, page_size=8, max_seqs=2, kv_dtype="int8-blocks")
    prompt = [3, 200, 77, 9, 14, 250, 1, 1, 8, 90, 33]
    first = s.generate([prompt], 12)
    for c in s.caches:
        c.k_scale.fill_(2.0 ** 40)
        c.v_scale.fill_(2.0 ** 40)
    assert s.generate([prompt], 12) == first
    s.close()


def test_sampled_continuations(tmp_path):
    path = archive(tmp_path, "llama")
    s = serve.load_session(path, DEV, pages=80, page_size=16, max_seqs=4)
    gen = lambda seed: torch.Generator(device=DEV).manual_seed(seed)
    prompts = [[5, 9, 200], [77] * 20, [1, 2, 3, 4]]
    greedy = s.generate(prompts, 10)
    # one candidate, or a temperature of 0 for one prompt: the greedy continuation
    assert s.generate(prompts, 10, temperature=1.5, top_k=1, generator=gen(1)) == greedy
    mixed = s.generate(prompts, 10, temperature=[0.0, 2.0, 0.0], generator=gen(1))
    assert mixed[0] == greedy[0] and mixed[2] == greedy[2] and mixed[1] != greedy[1]
    # the generator decides
    a, b, c = (s.generate(prompts, 10, temperature=2.0, top_p=0.99, generator=gen(i)) for i in (7, 7, 8))
    assert a == b and a != c and [len(x) for x in a] == [10, 10, 10]
    # every token is among the top_k of its place, as a session without sampling sees it
    out = s.generate(prompts, 6, temperature=3.0, top_k=[5, 9, 2], generator=gen(3))
    for prompt, got, k in zip(prompts, out, (5, 9, 2)):
        seqs, logits = s.prefill([prompt])
        for t in got:
            row = logits[0].float()
            assert row[t] >= row.topk(k).values[-1] - 3e-2 * 2 * row.norm() / 16
            logits = s.step(seqs, [t])
        s.release(seqs)
    # a prompt that ends leaves the others' settings with their rows
    stop = mixed[1][2]
    cut = s.generate(prompts, 10, eos=stop, temperature=[0.0, 2.0, 0.0], generator=gen(1))
    assert cut[0] == greedy[0][:greedy[0].index(stop) + 1] if stop in greedy[0] else cut[0] == greedy[0]
    assert len(s.free_pages) == 80 and not s.length
    s.close()


def test_refusals(tmp_path):
    path = archive(tmp_path, "llama")
    for bad in (dict(kv_dtype="int4"), dict(kv_dtype="e4m3", kv_block=8), dict(kv_dtype="int8-blocks", kv_block=3),
                dict(kv_dtype="int8-blocks", kv_block=0)):
        with pytest.raises(rt.ArchiveError):
            serve.load_session(path, DEV, pages=4, page_size=16, max_seqs=2, **bad)
    s = serve.load_session(path, DEV, pages=4, page_size=16, max_seqs=2)
    with pytest.raises(rt.ArchiveError, match="values of top_k"):
        s.generate([[1], [2]], 3, temperature=1.0, top_k=[1])
    with pytest.raises(rt.ArchiveError, match="range"):
        s.generate([[1], [2]], 3, temperature=[1.0, -1.0])
    with pytest.raises(RuntimeError):
        s.generate([[1]], 3, temperature=-1.0)
    assert len(s.free_pages) == 4 and len(s.free_seqs) == 2
    s.close()
