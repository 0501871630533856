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
