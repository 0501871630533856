"""GPU: serving on compressed weights -- archives compiled here, loaded with
fused layers, prompts and steps through the paged cache -- against the model's
own Transformers forward on decoded weights; fused layers with bias and the
fused feed-forward layer against torch in 64 bits.

A session's logits differ from the Transformers forward's by BF16 roundings at
other places (the fused epilogues round once where Transformers rounds after
every operation): two roundings of 2^-8 per layer operation, about eight such operations a
layer, in relative L2 at most (they add in quadrature): 2^-8 * sqrt(2 * 8 * layers + 8) < 3e-2
for the two layers here."""
import json

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu

import xksv_compile as xc  # noqa: E402
import xksv_gpu as xg  # noqa: E402
import xksv_runtime as rt  # noqa: E402
import xksv_serve as serve  # noqa: E402
from golden.make_archives import write_safetensors  # noqa: E402

DEV = "cuda:0"
BASE = {"hidden_size": 128, "intermediate_size": 352, "num_hidden_layers": 2, "num_attention_heads": 8,
        "num_key_value_heads": 2, "vocab_size": 256, "max_position_embeddings": 512, "rms_norm_eps": 1e-5,
        "tie_word_embeddings": False, "torch_dtype": "bfloat16"}
CONFIGS = {
    "llama": dict(BASE, architectures=["LlamaForCausalLM"], model_type="llama", hidden_act="silu", rope_theta=10000.0),
    "llama-gelu": dict(BASE, architectures=["LlamaForCausalLM"], model_type="llama", hidden_act="gelu_pytorch_tanh",
                       mlp_bias=True, attention_bias=True, rope_theta=500000.0),
    "qwen2": dict(BASE, architectures=["Qwen2ForCausalLM"], model_type="qwen2", hidden_act="silu", rope_theta=10000.0),
    "mistral": dict(BASE, architectures=["MistralForCausalLM"], model_type="mistral", hidden_act="silu",
                    rope_theta=10000.0, sliding_window=24, head_dim=32),
}


def archive(tmp_path, name, codec="dfloat11"):
    """An archive of a seeded model of CONFIGS[name]."""
    from transformers import AutoConfig, AutoModelForCausalLM
    src = tmp_path / name
    src.mkdir()
    (src / "config.json").write_text(json.dumps(CONFIGS[name]))
    model = AutoModelForCausalLM.from_config(AutoConfig.from_pretrained(src))
    g = torch.Generator().manual_seed(1)
    tensors = []
    for n, t in model.state_dict().items():
        v = torch.randn(t.shape, generator=g) * (0.3 if n.endswith("bias") else 0.08)
        v = torch.ones(t.shape) if n.endswith("norm.weight") else v
        v = v.to(torch.bfloat16)
        tensors.append((n, "BF16", list(t.shape), v.view(torch.uint8).numpy().tobytes()))
    write_safetensors(src / "model.safetensors", tensors)
    return xc.compile_checkpoint(src, tmp_path / f"{name}.xksv", codec)


def close(a, b, tol=3e-2):
    return float((a.float() - b.float()).norm() / b.float().norm()) < tol


@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_session_matches_transformers(tmp_path, name, kv):
    path = archive(tmp_path, name)
    ref, _, _ = rt.load_archive(path, DEV)
    s = serve.load_session(path, DEV, pages=64, page_size=8, max_seqs=4, kv_dtype=kv)
    assert all(hasattr(l.self_attn.q_proj, "xksv_fused") and hasattr(l.mlp, "xksv_fused_mlp") for l in s.layers)
    # an 8-bit cache rounds keys and values by 2^-4 more
    tol = 3e-2 if kv == "bf16" else 1e-1
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 256, (n,), generator=g) for n in (1, 40, 17)]
    ids = [p.to(DEV) for p in prompts]
    with torch.no_grad():
        seqs, logits = s.prefill(prompts)
        for step in range(12):
            want = torch.stack([ref(x[None]).logits[0, -1] for x in ids])
            assert close(logits, want, tol), step
            # a step of all, then of some, in another order
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


def test_generate_is_the_greedy_continuation(tmp_path):
    """Every generated token is among the best of the Transformers logits at its
    place (within the logits' own tolerance)."""
    path = archive(tmp_path, "llama")
    ref, _, _ = rt.load_archive(path, DEV)
    s = serve.load_session(path, DEV, pages=40, page_size=16, max_seqs=3)
    prompts = [[5, 9, 200], [77] * 20]
    out = s.generate(prompts, 10)
    assert [len(o) for o in out] == [10, 10] and len(s.free_pages) == 40
    for p, o in zip(prompts, out):
        with torch.no_grad():
            logits = ref(torch.tensor([p + o], device=DEV)).logits[0].float()
        for k, t in enumerate(o):
            row = logits[len(p) + k - 1]
            assert row.max() - row[t] <= 3e-2 * 2 * row.norm()
    assert s.generate([[5, 9, 200]], 10, eos=out[0][3])[0] == out[0][:out[0].index(out[0][3]) + 1]
    s.close()


def test_session_refusals(tmp_path):
    path = archive(tmp_path, "llama")
    s = serve.load_session(path, DEV, pages=4, page_size=16, max_seqs=2, max_tokens=48)
    for bad, match in (([torch.zeros(0, dtype=torch.long)], "empty"), ([[1]] * 3, "too many"), ([[1] * 49], "exceeds"),
                       ([[1] * 33, [1] * 33], "full"), ([], "empty"), ([[1, 256]], "vocabulary"), ([[-1]], "vocabulary")):
        with pytest.raises(rt.ArchiveError, match=match):
            s.prefill(bad)
        assert len(s.free_pages) == 4 and len(s.free_seqs) == 2
    seqs, _ = s.prefill([[1] * 48, [2] * 15])
    s.step(seqs[1:], [3])
    for bad, match in ((seqs[:1], "exceeds"), (seqs[1:], "full"), ([seqs[1], seqs[1]], "repeated"), ([], "no sequence"),
                       ([9], "unknown")):
        with pytest.raises(rt.ArchiveError, match=match):
            s.step(bad, [1] * len(bad))
    for bad, match in (([1, 2], "one token"), ([256], "vocabulary")):
        with pytest.raises(rt.ArchiveError, match=match):
            s.step(seqs[1:], bad)
    assert s.length[seqs[1]] == 16  # refused steps add nothing
    s.release(seqs[:1])
    assert s.step(seqs[1:], [4]).shape == (1, 256)
    with pytest.raises(rt.ArchiveError, match="dtype"):
        serve.PagedSession(s.model, 4, kv_dtype="int8")
    s.close()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch", [1, 2, 9, 150])
def test_fused_weight_epilogue(tmp_path, dtype, batch):
    """FusedWeight's epilogue for BF16 activations (one linear call) and others."""
    path = archive(tmp_path, "llama-gelu")
    a = rt.ResidentArchive(path, DEV)
    a.verify()
    name = "model.layers.0.mlp.up_proj"
    fw, W, bias = a.fused(name + ".weight"), a.tensor(name + ".weight").double(), a.tensor(name + ".bias")
    g = torch.Generator(device=DEV).manual_seed(batch)
    x, mul, res = (torch.randn(batch, n, generator=g, device=DEV).to(dtype) for n in (128, 352, 352))
    y = fw(x, bias=bias, act="gelu", mul=mul, residual=res)
    z = x.to(torch.bfloat16).double() @ W.t() if batch >= 4 else x.double() @ W.t()
    want = torch.nn.functional.gelu(z + bias.double()) * mul.double() + res.double()
    assert y.dtype == dtype and y.shape == (batch, 352)
    # half a step of the type, and FP32 sums of 128 products
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -16 * (1 + mul.double().abs()) * (1 + z.abs())
    assert ((y.double() - want).abs() <= tol).all()
    # operands of any strides and shape: transposed, expanded, FP16 factors
    xt = x.t().contiguous().t()
    again = fw(xt, bias=bias.half(), act="gelu", mul=mul.t().contiguous().t(), residual=res)
    assert ((again.double() - want).abs() <= tol + 2.0 ** -10).all()
    same = fw(x[:1].expand(batch, -1))
    assert ((same - fw(x[:1])).abs() <= 2.0 ** -7 * (1 + same.abs())).all()
    cube = fw(x[:, None, None], residual=res[:, None, None])
    assert cube.shape == (batch, 1, 1, 352)
    fw.close()


@pytest.mark.parametrize("at", ["layer", "head"])
def test_a_step_that_raises_leaves_the_sequences_as_they_were(tmp_path, at):
    """A step that fails in its second layer, or behind the last one, and is made
    again gives the logits of a session that never failed; pages taken for it are
    free again.  (The cache holds large values at first, so that a place left
    unwritten would show.)"""
    path = archive(tmp_path, "llama")
    a = serve.load_session(path, DEV, pages=24, page_size=8, max_seqs=2)
    b = serve.PagedSession(a.model, 24, page_size=8, max_seqs=2)
    for s in (a, b):
        s.kv.fill_(8.0)
    prompts, tokens = [list(range(16)), [7, 9, 11]], [3, 4]  # the first one's next token needs a new page
    seqs, _ = a.prefill(prompts)
    other, _ = b.prefill(prompts)
    module = a.layers[1].mlp if at == "layer" else a.model.lm_head
    whole, (lengths, pages) = module.forward, (dict(a.length), list(a.free_pages))
    owned = {s: list(p) for s, p in a.owned.items()}

    def fails(*args, **kwargs):
        raise MemoryError("no room")

    module.forward = fails
    for _ in range(2):
        with pytest.raises(MemoryError):
            a.step(seqs, tokens)
        assert a.length == lengths and a.owned == owned and a.free_pages == pages
    module.forward = whole
    want = b.step(other, tokens)
    assert close(a.step(seqs, tokens), want, 1e-2)
    assert a.length == {s: n + 1 for s, n in lengths.items()} and len(a.free_pages) == len(pages) - 1
    assert close(a.step(seqs, tokens), b.step(other, tokens), 1e-2)
    a._check()
    a.close()
    b.close()


def test_fused_weight_takes_more_tokens_than_one_call(tmp_path):
    """2^20 tokens and more, which one linear call refuses, on a weight of 256 x
    128: the first, the last and the tokens around the parts' borders."""
    path = archive(tmp_path, "llama")
    a = rt.ResidentArchive(path, DEV)
    a.verify()
    name = "lm_head.weight"
    fw, W = a.fused(name), a.tensor(name).double()
    n = (1 << 20) + 3
    g = torch.Generator(device=DEV).manual_seed(5)
    x, res = (torch.randn(n, c, generator=g, device=DEV, dtype=torch.bfloat16) for c in (128, 256))
    y = fw(x, act="relu", residual=res)
    at = torch.tensor([0, (1 << 19) - 1, 1 << 19, (1 << 20) - 1, 1 << 20, n - 1], device=DEV)
    want = torch.relu(x[at].double() @ W.t()) + res[at].double()
    # half a step of BF16, and a FP32 sum of 128 products and the residual
    tol = 129 * 2.0 ** -24 * (x[at].double().abs() @ W.abs().t()) + 2.0 ** -23 * (want.abs() + res[at].double().abs())
    assert ((y[at].double() - want).abs() <= 2.0 ** -8 * want.abs() + tol).all()
    fw.close()


def test_hooks_of_fused_modules_run(tmp_path):
    """Forward hooks of every layer that a session calls run, once a step, and
    what a hook returns is used."""
    path = archive(tmp_path, "llama-gelu")
    s = serve.load_session(path, DEV, pages=8, page_size=8, max_seqs=1)
    seen = []
    for layer in s.layers:
        for name, m in layer.named_modules():
            if name.rsplit(".", 1)[-1] in ("q_proj", "k_proj", "v_proj", "o_proj", "mlp", "gate_proj", "up_proj", "down_proj"):
                m.register_forward_hook(lambda m, args, out, name=name: seen.append(name))
    seqs, want = s.prefill([[1, 2, 3]])
    assert len(seen) == 8 * len(s.layers) and len(set(seen)) == 8
    seen.clear()
    s.step(seqs, [4])
    assert len(seen) == 8 * len(s.layers) and len(set(seen)) == 8
    s.release(seqs)
    handle = s.layers[1].mlp.gate_proj.register_forward_hook(lambda m, args, out: torch.zeros_like(out))
    seqs, other = s.prefill([[1, 2, 3]])
    assert not close(other, want)
    s.release(seqs)
    handle.remove()
    assert close(s.prefill([[1, 2, 3]])[1], want)
    s.close()


def test_scales_of_layers_and_heads(tmp_path):
    """Keys of large biases (qwen2) in an 8-bit cache: with a scale per layer,
    kind and head each stored element is its value rounded once (2^-4 relative,
    and the BF16 key's own 2^-8), where the default saturates at 28."""
    path = archive(tmp_path, "qwen2")
    s = serve.load_session(path, DEV, pages=4, page_size=8, max_seqs=1)
    with torch.no_grad():
        for layer in s.layers:
            layer.self_attn.k_proj.bias.mul_(200)
    prompt = [list(range(20))]
    s.prefill(prompt)
    exact = s.kv.double()  # BF16 [layers, 2, pages, page_size, heads, dim]
    top = exact.abs().amax((2, 3, 5))
    assert float(top[0, 0].min()) > 28 and (top[0, :, 0] != top[0, :, 1]).all()  # each head a scale of its own

    def stored(scale):
        e = serve.PagedSession(s.model, 4, page_size=8, max_seqs=1, kv_dtype="e4m3", **scale)
        e.prefill(prompt)
        rows = torch.stack([torch.stack([c.view(torch.uint8).view(torch.float8_e4m3fn).double() * f.double()[:, None]
                                         for c, f in ((x.k, x.k_scale), (x.v, x.v_scale))]) for x in e.caches])
        e._check()
        e.close()
        return rows

    # (the second layer's input already holds the first one's roundings)
    got, want, step = stored(dict(kv_scale=top.float() / 400))[0], exact[0], top[0] / 400
    assert ((got - want).abs() <= (2.0 ** -4 + 2.0 ** -7) * want.abs() + 2.0 ** -10 * step[:, None, None, :, None]).all()
    assert float(stored({})[0, 0].abs().max()) == 28.0
    for bad, match in ((torch.ones(3, device=DEV), "shape"), (0.0, "above zero"), (float("nan"), "above zero")):
        with pytest.raises(rt.ArchiveError, match=match):
            serve.PagedSession(s.model, 4, kv_dtype="e4m3", kv_scale=bad)
    s.close()


def test_ids_on_the_device_outside_the_vocabulary(tmp_path):
    """They give rows of NaN and change no other sequence."""
    path = archive(tmp_path, "llama")
    a = serve.load_session(path, DEV, pages=8, page_size=8, max_seqs=3)
    b = serve.PagedSession(a.model, 8, page_size=8, max_seqs=3)
    prompts = [[1, 2], [3, 4, 5], [6]]
    seqs, _ = a.prefill(prompts)
    other, _ = b.prefill(prompts)
    got = a.step(seqs, torch.tensor([256, 7, -1], device=DEV))
    want = b.step(other, torch.tensor([255, 7, 0], device=DEV))
    assert torch.isnan(got[0]).all() and torch.isnan(got[2]).all() and torch.isfinite(want).all()
    assert close(got[1:2], want[1:2], 1e-2)
    a._check()
    a.close()
    b.close()
