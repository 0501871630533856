"""GPU: what a session says of errors and settings (models and archives of
test_gpu_serve.py)."""
import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu

import xksv_runtime as rt  # noqa: E402
import xksv_serve as serve  # noqa: E402
from test_gpu_serve import DEV, archive  # noqa: E402


def test_an_error_is_reported_once(tmp_path):
    """A NaN key, which integers do not hold, is an error of every layer's cache: the
    call that met it fails, others go on."""
    s = serve.load_session(archive(tmp_path, "llama"), DEV, pages=8, page_size=8, max_seqs=2, kv_dtype="int8-blocks")
    good = s.generate([[1, 2, 3]], 4)
    with torch.no_grad():
        s.core.embed_tokens.weight[5] = float("nan")
    with pytest.raises(rt.ArchiveError, match="^paged cache"):
        s.prefill([[1, 5, 3]])
    assert s.generate([[1, 2, 3]], 4) == good
    assert len(s.free_pages) == 8 and len(s.free_seqs) == 2
    s.close()


@pytest.mark.parametrize("kv,said", [("int8-blocks", "NaN"), ("e4m3-blocks", None), ("bf16", None)])
def test_a_nan_key_is_named(tmp_path, kv, said):
    """Integers hold no NaN: the append reports it, and the session says so.  The other
    caches keep it, and the logits are NaN."""
    s = serve.load_session(archive(tmp_path, "llama"), DEV, pages=8, page_size=8, max_seqs=2, kv_dtype=kv)
    good = s.generate([[1, 2, 3]], 4)
    with torch.no_grad():
        s.core.embed_tokens.weight[5] = float("nan")
    if said:
        with pytest.raises(rt.ArchiveError, match=said):
            s.prefill([[1, 5, 3]])
    else:
        seqs, logits = s.prefill([[1, 5, 3]])
        assert logits.isnan().all()
        s.release(seqs)
    # it is reported once, and others go on
    assert s.generate([[1, 2, 3]], 4) == good
    assert len(s.free_pages) == 8 and len(s.free_seqs) == 2
    s.close()


@pytest.mark.parametrize("kv,said", [("int8-blocks", "NaN .*, or a page or place outside"), ("e4m3-blocks", "^paged cache: a page or place outside"),
                                     ("bf16", "^paged cache: a page or place outside")])
def test_an_error_names_its_possible_causes(tmp_path, kv, said):
    s = serve.load_session(archive(tmp_path, "llama"), DEV, pages=8, page_size=8, max_seqs=2, kv_dtype=kv)
    s.caches[1].status = lambda stream=0: 1  # (as after an error)
    with pytest.raises(rt.ArchiveError, match=said):
        s.prefill([[1, 2, 3]])
    assert len(s.free_pages) == 8 and len(s.free_seqs) == 2
    s.close()


def test_settings_of_one_value_are_numbers(tmp_path):
    """A tensor or an array without dimensions is a number; of more than one dimension it
    is refused."""
    import numpy as np
    s = serve.load_session(archive(tmp_path, "llama"), DEV, pages=40, page_size=8, max_seqs=4)
    gen = lambda: torch.Generator(device=DEV).manual_seed(3)
    prompts = [[1, 2, 3], [4] * 9]
    want = s.generate(prompts, 6, temperature=0.75, top_k=20, top_p=0.5, min_p=0.25, generator=gen())
    for one in (torch.tensor, np.array, lambda v: torch.tensor(v, device=DEV)):
        assert s.generate(prompts, 6, temperature=one(0.75), top_k=one(20), top_p=one(0.5), min_p=one(0.25), generator=gen()) == want
    assert s.generate(prompts, 6, temperature=torch.tensor(0.0)) == s.generate(prompts, 6)
    for bad in (dict(temperature=torch.ones(2, 1)), dict(top_p=[[0.5], [0.5]]), dict(temperature="warm"), dict(top_k=[1.5, "a"])):
        with pytest.raises((rt.ArchiveError, ValueError)):
            s.generate(prompts, 2, **{"temperature": 1.0, **bad})
    assert len(s.free_pages) == 40 and len(s.free_seqs) == 4
    s.close()


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_torchs_default_dtype_does_not_matter(tmp_path, default):
    path = archive(tmp_path, "llama")
    how = dict(temperature=1.5, top_p=0.9)

    def run():
        s = serve.load_session(path, DEV, pages=40, page_size=8, max_seqs=4, kv_dtype="int8-blocks")
        out = s.generate([[1, 2, 3], [4] * 9], 6, **how, generator=torch.Generator(device=DEV).manual_seed(3))
        s.close()
        return out

    want, before = run(), torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        assert run() == want
    finally:
        torch.set_default_dtype(before)
