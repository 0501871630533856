"""Serving on compressed weights: a decoder model loaded from an archive, its
key/value cache in pages, one call per token step.

``load_session(path, device, ...)`` loads an archive with fused layers
(xksv_runtime.load_archive) and opens a ``PagedSession`` on the model.  The
session keeps every layer's keys and values in one paged buffer (BF16, or
float8 with a scale per head), gives sequences pages from a free list, and
runs the model's modules itself:

    session = xksv_serve.load_session("model.xksv", "cuda:0", pages=4096)
    seqs, logits = session.prefill([ids_a, ids_b])      # prompts of any lengths
    logits = session.step(seqs, logits.argmax(-1))      # one token each
    session.release(seqs)

A step's layer is: the input norm, the q / k / v products (with their biases),
the append with its rotation (KVCache.append), the attention over the cache
(KVCache.attend), the output product with the residual in its epilogue, and
the feed-forward layer likewise (xksv_runtime.FusedMLP).  Prompts attend among
their own tokens (torch), on the keys as the cache holds them.

No counterpart in the reference, whose generation leaves the cache to
Transformers (python/runtime.py:289-330).
"""
import xksv_gpu
from xksv_runtime import fail, load_archive

MODEL_TYPES = ("llama", "mistral", "qwen2")


def load_session(path, device, verify=True, part_index=True, **session):
    """load_archive(fused_gemv=True, fused_mlp=True) and a PagedSession on it;
    the further keyword arguments are PagedSession's."""
    model, tokenizer, archive = load_archive(path, device, verify=verify, fused_gemv=True, fused_mlp=True,
                                             part_index=part_index)
    s = PagedSession(model, device=archive.device, **session)
    s.tokenizer, s.archive = tokenizer, archive
    return s


class PagedSession:
    """A decoder model (Llama layout: q_proj, k_proj, v_proj, o_proj, a gated
    feed-forward layer, two norms a layer) over a paged cache of `pages` pages
    of `page_size` tokens.  `max_tokens` bounds one sequence (default: the
    model's positions).  kv_dtype "bf16" keeps the model's BF16; "e4m3" halves
    the cache: an element stands for its value times `kv_scale`, a number or a
    tensor that broadcasts to [layers, 2 (keys, values), KV heads].  Keys and
    values beyond 448 kv_scale (28 by default) saturate there, unreported:
    models with large key or value biases need scales of their own."""

    def __init__(self, model, pages, page_size=16, max_tokens=None, max_seqs=256, kv_dtype="bf16", kv_scale=1.0 / 16,
                 device=None):
        import torch
        config = model.config
        if config.model_type not in MODEL_TYPES:
            fail(f"paged sessions serve {', '.join(MODEL_TYPES)} models, not {config.model_type}")
        if kv_dtype not in ("bf16", "e4m3"):
            fail(f"unknown cache dtype {kv_dtype}")
        self.model, self.core, self.config = model, model.model, config
        self.layers = list(self.core.layers)
        self.device = torch.device(device or next(model.parameters()).device)
        rope = self.core.rotary_emb
        if rope.rope_type == "dynamic" or rope.rope_type == "longrope":
            fail(f"rotation of type {rope.rope_type} changes with the length")
        self.inv_freq = rope.inv_freq.to(self.device, torch.float32).contiguous()
        self.rot_scale = float(rope.attention_scaling)
        self.heads, self.kv_heads = config.num_attention_heads, config.num_key_value_heads
        self.dim = getattr(config, "head_dim", None) or config.hidden_size // self.heads
        self.windows = [self._window(i) for i in range(len(self.layers))]
        self.page_size, self.max_tokens = page_size, max_tokens or config.max_position_embeddings
        store = torch.bfloat16 if kv_dtype == "bf16" else torch.float8_e4m3fn
        shape = (len(self.layers), 2, pages, page_size, self.kv_heads, self.dim)
        self.kv = torch.zeros(shape, dtype=torch.uint8 if kv_dtype == "e4m3" else store, device=self.device).view(store)
        scales = [(None, None)] * len(self.layers)
        if kv_dtype == "e4m3":
            scale = torch.as_tensor(kv_scale, dtype=torch.float32, device=self.device)
            shape = (len(self.layers), 2, self.kv_heads)
            try:
                scales = scale.expand(shape).contiguous()
            except RuntimeError:
                fail(f"kv_scale of shape {list(scale.shape)} for {list(shape)} [layers, 2, heads]")
            if not bool(((scales > 0) & torch.isfinite(scales)).all()):
                fail("kv_scale is above zero and finite")
        self.caches = [xksv_gpu.KVCache(l[0], l[1], k_scale=s[0], v_scale=s[1]) for l, s in zip(self.kv, scales)]
        self.table = torch.full((max_seqs, -(-self.max_tokens // page_size)), -1, dtype=torch.int32, device=self.device)
        self.free_pages = list(range(pages))[::-1]
        self.free_seqs = list(range(max_seqs))[::-1]
        self.length = {}  # sequence -> its tokens
        self.owned = {}   # sequence -> its pages

    def _window(self, layer):
        """A layer's sliding window, 0 for none."""
        types = getattr(self.config, "layer_types", None)
        window = getattr(self.config, "sliding_window", None)
        sliding = types[layer] == "sliding_attention" if types else getattr(self.config, "use_sliding_window", True)
        return int(window) if window and sliding else 0

    # ---- pages
    def _grow(self, needs):
        """Gives each sequence pages for its new length, all or none."""
        import torch
        want = {s: -(-n // self.page_size) - len(self.owned[s]) for s, n in needs.items()}
        for s, n in needs.items():
            if n > self.max_tokens:
                fail(f"sequence of {n} tokens exceeds {self.max_tokens}")
        if sum(want.values()) > len(self.free_pages):
            fail("paged cache is full")
        rows, cols, pages = [], [], []
        for s, k in want.items():
            for _ in range(k):
                page = self.free_pages.pop()
                rows.append(s)
                cols.append(len(self.owned[s]))
                pages.append(page)
                self.owned[s].append(page)
        if pages:
            at = torch.tensor([rows, cols], device=self.device)
            self.table[at[0], at[1]] = torch.tensor(pages, dtype=torch.int32, device=self.device)
        self.length.update(needs)

    def _held(self, seqs):
        """What _shrink takes the sequences back to."""
        return {s: (self.length[s], len(self.owned[s])) for s in seqs}

    def _shrink(self, held):
        for s, (length, pages) in held.items():
            self.free_pages.extend(reversed(self.owned[s][pages:]))
            del self.owned[s][pages:]
            self.length[s] = length

    def release(self, seqs):
        """Ends sequences; their pages become free."""
        for s in seqs:
            self.free_pages.extend(self.owned.pop(s))
            del self.length[s]
            self.free_seqs.append(s)

    # ---- layers
    def _project(self, layer, h):
        """Rows of q, k and v heads of one layer's normed input."""
        a = layer.self_attn
        x = layer.input_layernorm(h)
        return (m(x).unflatten(-1, (n, self.dim)) for m, n in ((a.q_proj, self.heads), (a.k_proj, self.kv_heads),
                                                               (a.v_proj, self.kv_heads)))

    def _finish(self, layer, h, attended):
        """The output product, the feed-forward layer and their residuals."""
        o = layer.self_attn.o_proj
        x = attended.flatten(-2)
        h = o(x, residual=h) if hasattr(o, "xksv_fused") else h + o(x)
        x = layer.post_attention_layernorm(h)
        return layer.mlp(x, residual=h) if hasattr(layer.mlp, "xksv_fused_mlp") else h + layer.mlp(x)

    def _check(self):
        stream = self._stream()
        if any(c.status(stream) for c in self.caches):
            fail("paged cache: a page or place outside the cache")

    def _stream(self):
        import torch
        return torch.cuda.current_stream(self.device).cuda_stream

    def prefill(self, prompts):
        """Begins a sequence per prompt (1-D token ids of any length above 0);
        returns (sequences, the logits [n, vocabulary] after each prompt)."""
        import torch
        prompts = [torch.as_tensor(p).reshape(-1) for p in prompts]
        if not prompts or any(p.numel() == 0 for p in prompts):
            fail("empty prompt")
        for p in prompts:  # (an id outside the vocabulary would fault the embedding)
            low, high = p.aminmax()
            if low < 0 or high >= self.config.vocab_size:
                fail("token id outside the vocabulary")
        prompts = [p.to(self.device) for p in prompts]
        if len(prompts) > len(self.free_seqs):
            fail("too many sequences")
        seqs = [self.free_seqs.pop() for _ in prompts]
        for s in seqs:
            self.owned[s], self.length[s] = [], 0
        try:
            self._grow({s: p.numel() for s, p in zip(seqs, prompts)})
            return seqs, self._prefill(seqs, prompts)
        except BaseException:
            self.release(seqs)
            raise

    def _prefill(self, seqs, prompts):
        import torch
        counts = [p.numel() for p in prompts]
        place = torch.cat([torch.arange(n, device=self.device) for n in counts])
        owner = torch.repeat_interleave(torch.tensor(seqs, device=self.device), torch.tensor(counts, device=self.device))
        index, seq = place.to(torch.int32), owner.to(torch.int32)
        page, slot = self.table[owner, place // self.page_size].long(), place % self.page_size
        with torch.no_grad(), torch.cuda.device(self.device):
            h = self.core.embed_tokens(torch.cat(prompts))
            for layer, cache, window in zip(self.layers, self.caches, self.windows):
                q, k, v = self._project(layer, h)
                cache.append(k, v, self.table, index, seq=seq, inv_freq=self.inv_freq, rot_scale=self.rot_scale, q=q,
                             stream=self._stream())
                # the keys and values as later steps will read them
                k, v = (self._cached(c, s, page, slot, q.dtype) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
                out = torch.empty_like(q)
                at = 0
                for n in counts:
                    out[at:at + n] = self._causal(q[at:at + n], k[at:at + n], v[at:at + n], window)
                    at += n
                h = self._finish(layer, h, out)
            last = torch.tensor(counts, device=self.device).cumsum(0) - 1
            logits = self.model.lm_head(self.core.norm(h[last]))
        self._check()
        return logits

    def _cached(self, c, scale, page, slot, dtype):
        import torch
        if c.dtype == dtype:
            return c[page, slot]
        rows = c.view(torch.uint8)[page, slot].view(c.dtype).float()
        return (rows * scale[:, None]).to(dtype)

    def _causal(self, q, k, v, window):
        import torch
        import torch.nn.functional as F
        n = q.shape[0]
        q, k, v = (t.transpose(0, 1)[None] for t in (q, k, v))
        mask = None
        if window and window < n:
            i = torch.arange(n, device=self.device)
            mask = (i[None] <= i[:, None]) & (i[None] > i[:, None] - window)
        out = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, is_causal=mask is None, enable_gqa=True)
        return out[0].transpose(0, 1)

    def step(self, seqs, tokens):
        """One more token of each sequence (`tokens` [n]); returns the logits [n,
        vocabulary] after it.  Ids outside the vocabulary are refused; ids on
        the device are not waited for: there such a row's logits are NaN.  A
        step that raises leaves the sequences as they were."""
        import torch
        if len(set(seqs)) != len(seqs) or any(s not in self.length for s in seqs):
            fail("step: unknown or repeated sequence")
        if not len(seqs):
            fail("step: no sequence")
        tokens = torch.as_tensor(tokens).reshape(-1)
        if tokens.numel() != len(seqs):
            fail("step: one token per sequence")
        if not tokens.is_cuda and (tokens.min() < 0 or tokens.max() >= self.config.vocab_size):
            fail("token id outside the vocabulary")
        held = self._held(seqs)
        try:
            self._grow({s: self.length[s] + 1 for s in seqs})
            return self._step(seqs, tokens)
        except BaseException:  # some layers hold the token's keys, others do not
            self._shrink(held)
            raise

    def _step(self, seqs, tokens):
        import torch
        with torch.no_grad(), torch.cuda.device(self.device):
            rows = torch.tensor(seqs, device=self.device)
            lens = torch.tensor([self.length[s] for s in seqs], dtype=torch.int32, device=self.device)
            table, index = self.table[rows], lens - 1
            ids = tokens.to(self.device)
            inside = ids.clamp(0, self.config.vocab_size - 1)  # (another id would fault the embedding)
            h = self.core.embed_tokens(inside)
            stream = self._stream()
            for layer, cache, window in zip(self.layers, self.caches, self.windows):
                q, k, v = self._project(layer, h)
                cache.append(k, v, table, index, inv_freq=self.inv_freq, rot_scale=self.rot_scale, q=q, stream=stream)
                out = torch.empty_like(q)
                cache.attend(q, table, lens, out, window=window, stream=stream)
                h = self._finish(layer, h, out)
            logits = self.model.lm_head(self.core.norm(h))
            return logits.masked_fill_((ids != inside)[:, None], float("nan")) if tokens.is_cuda else logits

    def generate(self, prompts, max_new_tokens, eos=None):
        """Greedy continuations of the prompts: a list of token lists, each ended
        by `eos` or max_new_tokens."""
        import torch
        seqs, logits = self.prefill(prompts)
        out = [[] for _ in seqs]
        live = list(range(len(seqs)))
        try:
            for k in range(max_new_tokens):
                token = logits.argmax(-1)
                ids = token.tolist()
                for i, t in zip(live, ids):
                    out[i].append(t)
                keep = [j for j, t in enumerate(ids) if t != eos]
                live = [live[j] for j in keep]
                if not live or k + 1 == max_new_tokens:
                    break
                logits = self.step([seqs[i] for i in live], token[torch.tensor(keep, device=self.device)])
            self._check()
        finally:
            self.release(seqs)
        return out

    def close(self):
        for c in self.caches:
            c.close()
