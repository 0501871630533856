"""Measured cases of the 8-bit cache with block scales, and of sampling.

A served token step of a model whose keys and values are held in 8 bits with a
scale for each block of tokens and head:

* ``append``  position rotation of new queries and keys, and the append of keys
  and values to the pages, each block's scale raised where the new tokens need
  it (``xksv_gpu.KVCache.append`` on a cache with block scales);
* ``attend``  attention of one new token per sequence over those pages
  (``xksv_gpu.KVCache.attend``);
* ``sample``  the next token of each row of logits by temperature, top-k,
  top-p and min-p from a given random number (``xksv_gpu.sample``).

``run`` computes them through the framework where ``own`` is true, and with
elementary torch operations where it is false: in 32 bits, and the weights of
``sample``, whose sums decide between neighbouring tokens, in 64.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn,
         "int8": torch.int8}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
# the largest element of a block, in units of its scale
TOP = {"e4m3": 448.0, "int8": 127.0}
# a block's scale is a power of two, not below this one
LEAST = -60


def listed():
    return [
        # ---- append: "block" is the tokens of a page that share a scale ----
        # one sequence's new token into a block that others began
        dict(name="append-token-e4m3", op="append", tokens=1, seqs=1, pads=0, q_heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, far=30000, page=16, block=16, layout="nhd", type="bf16", cache="e4m3"),
        # a padded decode batch: every token raises or keeps its own block
        dict(name="append-batch-int8", op="append", tokens=200, seqs=200, pads=11, q_heads=28, kv_heads=4, dim=128,
             rot=128, interleaved=False, far=100000, page=32, block=8, layout="hnd", type="bf16", cache="int8"),
        # prompts of uneven lengths, part of each head rotated in pairs
        dict(name="append-prompts-interleaved", op="append", tokens=3001, seqs=7, pads=0, q_heads=20, kv_heads=20,
             dim=80, rot=32, interleaved=True, far=500, page=48, block=24, layout="nhd", type="fp16", cache="e4m3"),
        # a full prefill chunk
        dict(name="append-prefill-16384", op="append", tokens=16384, seqs=5, pads=0, q_heads=32, kv_heads=8, dim=128,
             rot=128, interleaved=False, far=8000, page=64, block=16, layout="nhd", type="bf16", cache="e4m3"),
        # ---- attend ---------------------------------------------------------
        # one short conversation: latency
        dict(name="attend-one-short", op="attend", seqs=1, length=777, ragged=False, empty=0, q_heads=32, kv_heads=8,
             dim=128, page=16, block=16, layout="nhd", type="bf16", cache="e4m3", window=0, softcap=0.0),
        # one very long document: the split over its length
        dict(name="attend-one-long", op="attend", seqs=1, length=131071, ragged=False, empty=0, q_heads=32,
             kv_heads=8, dim=128, page=16, block=16, layout="nhd", type="bf16", cache="e4m3", window=0, softcap=0.0),
        # a decode batch of uneven lengths with free slots, a scale per token
        dict(name="attend-batch-token-scales", op="attend", seqs=130, length=6000, ragged=True, empty=9, q_heads=28,
             kv_heads=4, dim=128, page=32, block=1, layout="hnd", type="fp16", cache="e4m3", window=0, softcap=0.0),
        # the largest batch: uneven lengths to 16384, integers
        dict(name="attend-batch-long-int8", op="attend", seqs=64, length=16384, ragged=True, empty=0, q_heads=32,
             kv_heads=8, dim=128, page=64, block=64, layout="nhd", type="bf16", cache="int8", window=0, softcap=0.0),
        # ---- sample: "slope" is how steeply a row's largest logits fall -----
        # one conversation's next token
        dict(name="sample-token-32000", op="sample", rows=1, vocab=32000, type="bf16", extra=0, slope=1.2, banned=0.0,
             mixed=False, temperature=0.7, top_k=40, top_p=0.95, min_p=0.0),
        # one row of a large vocabulary, most of it inside the nucleus
        dict(name="sample-token-128256-flat", op="sample", rows=1, vocab=128256, type="fp32", extra=0, slope=0.6,
             banned=0.0, mixed=False, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0),
        # an odd vocabulary in a wider buffer, tokens that a grammar forbids,
        # each row with its own settings
        dict(name="sample-batch-odd", op="sample", rows=77, vocab=32003, type="fp16", extra=5, slope=1.0, banned=0.3,
             mixed=True, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
        # a full decode batch, each row with its own settings
        dict(name="sample-batch-256", op="sample", rows=256, vocab=128256, type="bf16", extra=0, slope=1.0, banned=0.0,
             mixed=True, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "sample"])
    if op == "sample":
        vocab = _log(rng, 1000, 262144)
        rows = max(1, min(_log(rng, 1, 512), 256 * 128256 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, type=rng.choice(["bf16", "fp16", "fp32"]),
                    extra=rng.choice([0, 0, 8, 13]), slope=round(rng.uniform(0.4, 1.6), 3),
                    banned=rng.choice([0.0, 0.0, 0.1, 0.9]), mixed=rng.random() < 0.5,
                    temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]), top_k=rng.choice([0, 0, 1, 20, 50, 1000]),
                    top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.98]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]))
    dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 12])
    page = rng.choice([1, 8, 16, 16, 24, 64, 256])
    block = rng.choice([b for b in (1, 2, 4, 8, 16, 16, 24, 32, 64, 128) if page % b == 0])
    case = dict(op=op, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, block=block,
                layout=rng.choice(["nhd", "hnd"]), type=rng.choice(["bf16", "bf16", "fp16"]),
                cache=rng.choice(["e4m3", "int8"]))
    if op == "append":
        cap = 16384 * 48 * 128 // ((q_heads + 2 * kv_heads) * dim)
        # prompts of a few sequences, or one new token each of many
        if rng.random() < 0.5:
            tokens = min(_log(rng, 1, 16384), cap)
            seqs = min(tokens, _log(rng, 1, 64))
        else:
            tokens = seqs = _log(rng, 1, 256)
        case.update(tokens=tokens, seqs=seqs, pads=rng.randrange(0, 1 + seqs // 8) if tokens == seqs else 0,
                    rot=dim if rng.random() < 0.6 else dim // 2, interleaved=rng.random() < 0.4,
                    far=_log(rng, 1, 1000000))
        if page > 64:
            case.update(page=64, block=min(64, block))
        return case
    cap = 64 * 16384 * 8 * 128 // 2 // (kv_heads * dim)
    length = min(_log(rng, 1, 131072), cap)
    seqs = max(1, min(_log(rng, 1, 256), cap // length))
    case.update(seqs=seqs, length=length, ragged=rng.random() < 0.6, empty=rng.randrange(0, 1 + seqs // 8),
                window=_log(rng, 1, length) if rng.random() < 0.2 else 0,
                softcap=30.0 if rng.random() < 0.2 else 0.0)
    return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _as_int(a):
    return torch.from_numpy(a.astype(np.int32)).cuda()


def _pages(gen, lens, page, pool=1):
    """A page table over a pool of pages, in random order; unused entries -1."""
    need = [-(-int(n) // page) for n in lens]
    total, width = max(pool, sum(need)), max(1, max(need))
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, device="cuda", dtype=torch.int32)
    used = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[used] = order[:int(used.sum())]
    return table, total


def _cache(gen, case, pages):
    """Keys and values in units of their scales, and the scales [pages, blocks,
    heads]: powers of two around what a normal variable needs."""
    H, D, P = case["kv_heads"], case["dim"], case["page"]
    shape = (pages, P, H, D) if case["layout"] == "nhd" else (pages, H, P, D)
    top = TOP[case["cache"]]

    def elements():
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).mul_(top / 4).clamp_(-top, top)
        return x.round_().to(torch.int8) if case["cache"] == "int8" else x.to(torch.float8_e4m3fn)

    def scales():
        e = torch.randint(-2, 2, (pages, P // case["block"], H), generator=gen, device="cuda")
        return torch.exp2(e + math.floor(math.log2(4 / top)))

    return elements(), elements(), scales(), scales()


def _append_inputs(case, seed):
    g = _gen(seed)
    rng = np.random.default_rng(seed)
    T, S, D = case["tokens"], case["seqs"], case["dim"]
    # each sequence's share of the tokens, its first new place, and the
    # position of that place (the cache begins at the sequence's far end)
    cuts = np.sort(rng.permutation(T - 1)[:S - 1] + 1) if S > 1 else np.zeros(0, np.int64)
    counts = np.diff(np.concatenate([[0], cuts, [T]]))
    first = rng.integers(0, case["page"] + 1, S)
    far = rng.integers(0, case["far"] + 1, S)
    seq = np.repeat(np.arange(S), counts)
    index = first[seq] + np.concatenate([np.arange(c) for c in counts])
    positions = far[seq] + index
    seq[rng.permutation(T)[:case["pads"]]] = -1
    table, total = _pages(g, first + counts, case["page"], T // case["page"] + 2 * S + 1)
    k_cache, v_cache, ks, vs = _cache(g, case, total)
    kind = TYPES[case["type"]]
    q, k, v = (_randn(g, (T, h, D), kind) for h in (case["q_heads"], case["kv_heads"], case["kv_heads"]))
    inv = 1.0 / (500000.0 ** (torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"]))
    return dict(q=q, k=k, v=v, table=table, k_cache=k_cache, v_cache=v_cache, ks=ks, vs=vs, seq=_as_int(seq),
                index=_as_int(index), positions=_as_int(positions), inv_freq=inv.float(), q_out=torch.zeros_like(q))


def _attend_inputs(case, seed):
    g = _gen(seed)
    rng = np.random.default_rng(seed)
    n, top = case["seqs"], case["length"]
    lens = rng.integers(1, top + 1, n) if case["ragged"] else np.full(n, top)
    if case["ragged"]:
        lens[rng.integers(0, n)] = top
    lens[rng.permutation(n)[:case["empty"]]] = 0
    table, total = _pages(g, lens, case["page"])
    k_cache, v_cache, ks, vs = _cache(g, case, total)
    q = _randn(g, (n, case["q_heads"], case["dim"]), TYPES[case["type"]])
    return dict(q=q, table=table, k_cache=k_cache, v_cache=v_cache, ks=ks, vs=vs, lens=_as_int(lens), host_lens=lens,
                scale=case["dim"] ** -0.5, out=torch.empty_like(q),
                lse=torch.empty(q.shape[:2], device="cuda", dtype=torch.float32))


def _sample_inputs(case, seed):
    g = _gen(seed)
    rng = np.random.default_rng(seed)
    R, V = case["rows"], case["vocab"]
    # the n-th largest of V values of -slope log(uniform) lies about slope
    # log(n) below the largest, as a language model's logits do
    z = torch.rand((R, V + case["extra"]), generator=g, device="cuda").clamp_(min=1e-12).log_().mul_(-case["slope"])
    if case["banned"]:
        z[torch.rand(z.shape, generator=g, device="cuda") < case["banned"]] = -math.inf
        z[:, seed % V] = 0.0  # (one token at least is allowed)
    logits = z.sub_(8.0).to(TYPES[case["type"]])[:, :V]
    how = dict(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
    if case["mixed"]:
        pick = lambda v, t: torch.from_numpy(rng.choice(np.array(v, t), R)).cuda()
        how = dict(temperature=pick([0.0, 0.4, 0.7, 1.0, 1.0, 1.2], np.float32), top_k=pick([0, 0, 1, 20, 64, 1000], np.int32),
                   top_p=pick([1.0, 1.0, 0.6, 0.9, 0.95], np.float32), min_p=pick([0.0, 0.0, 0.02, 0.1], np.float32))
    return dict(logits=logits, u=torch.rand(R, generator=g, device="cuda"), how=how,
                tokens=torch.empty(R, device="cuda", dtype=torch.int64), kept=torch.empty(R, device="cuda", dtype=torch.int32),
                logprob=torch.empty(R, device="cuda"))


INPUTS = {"append": _append_inputs, "attend": _attend_inputs, "sample": _sample_inputs}


def prepare(case, seed):
    s = INPUTS[case["op"]](case, seed)
    s["case"] = case
    if own:
        path = str(Path.cwd() / "xks-vectorforge_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import xksv_gpu
        s["xg"] = xksv_gpu
        if case["op"] != "sample":
            s["cache"] = xksv_gpu.KVCache(s["k_cache"], s["v_cache"], k_scale=s["ks"], v_scale=s["vs"],
                                          layout=case["layout"])
    return s


# --------------------------------------------------------------- own calls
def _own(s):
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "sample":
        s["xg"].sample(s["logits"], s["u"], s["tokens"], kept=s["kept"], logprob=s["logprob"], stream=stream, **s["how"])
        return s["tokens"], s["kept"], s["logprob"]
    if case["op"] == "append":
        s["cache"].append(s["k"], s["v"], s["table"], s["index"], seq=s["seq"], positions=s["positions"],
                          inv_freq=s["inv_freq"], interleaved=case["interleaved"], q=s["q"], q_out=s["q_out"],
                          stream=stream)
        return _appended(s)
    s["cache"].attend(s["q"], s["table"], s["lens"], s["out"], lse=s["lse"], scale=s["scale"],
                      window=case["window"], softcap=case["softcap"], stream=stream)
    return s["out"], s["lse"]


def _appended(s):
    """The queries and the whole cache; integers as the numbers they are."""
    k, v = ((c.half() if c.dtype == torch.int8 else c) for c in (s["k_cache"], s["v_cache"]))
    return s["q_out"], k, v, s["ks"], s["vs"]


# -------------------------------------------------------------- plain form
def _rows(cache, layout):
    """[pages, page_size, heads, dim] view of a cache of either layout."""
    return cache if layout == "nhd" else cache.permute(0, 2, 1, 3)


def _bytes(cache):
    """The same elements in a type that can be indexed."""
    return cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache


def _rotate(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _held(x, kind):
    """FP32 numbers in units of their scale as the cache holds them."""
    top = TOP[kind]
    return x.clamp(-top, top).to(torch.float8_e4m3fn) if kind == "e4m3" else x.round().clamp(-top, top).to(torch.int8)


def _needed(high, kind):
    """The least power of two that holds blocks whose largest element is `high`."""
    m, e = torch.frexp(high / TOP[kind])
    e = torch.where(m == 0.5, e - 1, e)
    # (the quotient is rounded: a power of two too small is put right)
    e = torch.where(high > TOP[kind] * torch.exp2(e.double()), e + 1, e)
    return torch.exp2(torch.where(high > 0, e, torch.full_like(e, LEAST)).clamp(min=LEAST).float())


def _plain_append(s):
    case = s["case"]
    P, B, H, D, kind = case["page"], case["block"], case["kv_heads"], case["dim"], case["cache"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    live = s["seq"] >= 0
    q = _rotate(s["q"].float(), cos, sin, case["rot"], case["interleaved"])
    s["q_out"].copy_(torch.where(live[:, None, None], q, s["q_out"].float()))
    k = _rotate(s["k"].float(), cos, sin, case["rot"], case["interleaved"])
    # padding tokens repeat the first live token
    src = torch.where(live, torch.arange(len(live), device="cuda"), torch.argmax(live.to(torch.int32)))
    index = s["index"].long()[src]
    page, place = s["table"][s["seq"].long()[src], index // P].long(), index % P
    block = page * (P // B) + place // B
    blocks = s["ks"].shape[0] * (P // B)
    # each block's first new place, B where there is none
    begin = torch.full((blocks,), B, device="cuda", dtype=torch.int64).scatter_reduce(0, block, place % B, "amin")
    # places before the first new one, in blocks that have both
    older = (torch.arange(B, device="cuda")[None] < begin[:, None]) & (begin < B)[:, None]
    older = older.view(-1, P, 1, 1)
    for cache, scale, rows in ((s["k_cache"], s["ks"], k[src]), (s["v_cache"], s["vs"], s["v"].float()[src])):
        high = torch.zeros(blocks, H, device="cuda").scatter_reduce(0, block[:, None].expand(-1, H), rows.abs().amax(-1), "amax")
        had = scale.view(blocks, H)
        want = torch.maximum(_needed(high, kind), torch.where((begin > 0)[:, None], had, torch.zeros_like(had)))
        want = torch.where((begin < B)[:, None], want, had)
        spread = lambda t: t.view(-1, P // B, 1, H).expand(-1, -1, B, -1).reshape(-1, P, H, 1)
        # the elements a block held before, in units of its new scale
        held = _rows(cache, case["layout"])
        moved = _held(held.float() * spread(had / want), kind)
        mixed = torch.where(older & spread(want > had), _bytes(moved), _bytes(held))
        mixed[page, place] = _bytes(_held(rows / want[block][..., None], kind))
        _bytes(held).copy_(mixed)
        scale.copy_(want.view(scale.shape))
    return _appended(s)


def _plain_attend(s):
    case = s["case"]
    H, P, B = case["kv_heads"], case["page"], case["block"]
    n, top = s["q"].shape[0], case["length"]
    at = s["table"].long().clamp(min=0)

    def rows(cache, scale):  # [seqs, heads, tokens, dim]
        x = _bytes(_rows(cache, case["layout"]))[at].view(cache.dtype).float()
        x = x * scale[at].repeat_interleave(B, 2)[..., None]
        return x.flatten(1, 2)[:, :top].transpose(1, 2)

    q = s["q"].float().view(n, H, -1, case["dim"])
    score = (q @ rows(s["k_cache"], s["ks"]).transpose(2, 3)) * s["scale"]
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    j, length = torch.arange(score.shape[-1], device="cuda"), s["lens"][:, None]
    seen = j < length
    if case["window"]:
        seen &= j >= length - case["window"]
    score = torch.where(seen[:, None, None, :], score, torch.full_like(score, -math.inf))
    high = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = torch.exp(score - high)
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen[:, None, :, None], rows(s["v_cache"], s["vs"]), torch.zeros((), device="cuda"))
    o = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    s["out"].copy_(o.view(s["out"].shape))
    s["lse"].copy_(torch.where(total > 0, high + torch.log(total), torch.full_like(total, -math.inf)).view(s["lse"].shape))
    return s["out"], s["lse"]


def _column(v, rows):
    return v.double()[:, None] if torch.is_tensor(v) else torch.full((rows, 1), float(v), device="cuda", dtype=torch.float64)


def _plain_sample(s):
    z = s["logits"].float()
    R, V = z.shape
    heat, top_k, top_p, min_p = (_column(s["how"][n], R) for n in ("temperature", "top_k", "top_p", "min_p"))
    # scalars are 32-bit numbers, as a tensor of settings holds them
    heat, top_p, min_p = heat.float().double(), top_p.float().double(), min_p.float().double()
    greedy = heat == 0
    # tokens by logit, equal ones by index
    fall, order = torch.sort(z, dim=-1, descending=True, stable=True)
    w = torch.exp((fall.double() - fall[:, :1].double()) / torch.where(greedy, torch.ones_like(heat), heat))
    rank = torch.arange(V, device="cuda")[None]
    keep = (rank < torch.where(greedy, torch.ones_like(top_k), top_k)) | ((top_k <= 0) & ~greedy)
    w = torch.where(keep, w, torch.zeros_like(w))
    total = w.sum(-1, keepdim=True)
    ahead = torch.cat((torch.zeros_like(total), torch.cumsum(w, -1)[:, :-1]), -1)
    keep &= (ahead < top_p * total) | (top_p >= 1) | (rank == 0)
    keep &= (w >= min_p) & (w > 0)
    w = torch.where(keep, w, torch.zeros_like(w))
    # the draw goes through the kept tokens by index
    flat = torch.zeros_like(w).scatter_(1, order, w)
    up = torch.cumsum(flat, -1)
    past = (up > s["u"].double()[:, None] * up[:, -1:]) & (flat > 0)
    last = V - 1 - torch.argmax((flat > 0).flip(-1).to(torch.int8), -1)
    s["tokens"].copy_(torch.where(past.any(-1), torch.argmax(past.to(torch.int8), -1), last))
    s["kept"].copy_(keep.sum(-1))
    s["logprob"].copy_(torch.log(flat.gather(1, s["tokens"][:, None]) / up[:, -1:])[:, 0])
    return s["tokens"], s["kept"], s["logprob"]


PLAIN = {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- the work
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # each logit less the largest, its weight, and the sum
        return {"bytes": float(n * SIZES[case["type"]] + 20 * case["rows"]), "flops": 3.0 * n}
    D, H, Q, e = case["dim"], case["kv_heads"], case["q_heads"], SIZES[case["type"]]
    if case["op"] == "append":
        T = case["tokens"] - case["pads"]
        scales = 8 * H * -(-T // case["block"])
        return {"bytes": float(T * D * (2 * Q * e + 2 * H * (e + 1)) + scales + 12 * case["tokens"]),
                "flops": 3.0 * T * (Q + H) * case["rot"]}
    mean = (case["length"] + 1) / 2 if case["ragged"] else case["length"]
    if case["window"]:
        mean = min(mean, case["window"])
    seen = mean * (case["seqs"] - case["empty"])
    return {"bytes": float(seen * 2 * H * (D + 4 / case["block"]) + 2 * case["seqs"] * Q * D * e),
            "flops": 4.0 * seen * Q * D}


# ------------------------------------------- the definitions, in 64 bits
def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    T, rot, P, B, kind = case["tokens"], case["rot"], case["page"], case["block"], case["cache"]
    # each pair is a complex number, turned by exp(i angle)
    turn = torch.polar(torch.ones(T, rot // 2, device="cuda", dtype=torch.float64),
                       s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]

    def turned(x):
        y = x.double()
        head = y[..., :rot]
        pair = head.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        got = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        y[..., :rot] = (got if case["interleaved"] else got.transpose(-1, -2)).flatten(-2)
        return y

    live = torch.nonzero(s["seq"] >= 0)[:, 0]
    q_out = torch.zeros_like(s["q"], dtype=torch.float64)
    q_out[live] = turned(s["q"])[live]
    where = s["index"].long()[live]
    page, place = s["table"].long()[s["seq"].long()[live], where // P], where % P
    caches, scales = [], []
    for cache, scale, rows in ((s["k_cache"], s["ks"], turned(s["k"])), (s["v_cache"], s["vs"], s["v"].double())):
        c = (cache if case["layout"] == "nhd" else cache.transpose(1, 2)).double().unflatten(1, (P // B, B))
        new = torch.full_like(c, math.nan)
        new[page, place // B, place % B] = rows[live]
        touched = new[..., 0, 0].isnan().logical_not()  # [pages, blocks, places]
        begin = torch.where(touched.any(-1), touched.to(torch.int8).argmax(-1), B)
        high = new.abs().nan_to_num(nan=0.0).amax((2, 4))
        need = torch.exp2(torch.log2(high / TOP[kind]).ceil().clamp(min=LEAST))
        old = scale.double()
        now = torch.where((begin > 0)[..., None], torch.maximum(need, old), need)
        now = torch.where((begin < B)[..., None], now, old)
        before = torch.arange(B, device="cuda") < begin[..., None]
        before &= (begin < B)[..., None]
        c = torch.where(before[..., None, None], c * (old / now)[:, :, None, :, None], c)
        c = torch.where(touched[..., None, None], new / now[:, :, None, :, None], c).flatten(1, 2)
        caches.append(c if case["layout"] == "nhd" else c.transpose(1, 2).contiguous())
        scales.append(now)
    return q_out, caches[0], caches[1], scales[0], scales[1]


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    H, G, P, B = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["page"], case["block"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    lse = torch.full(s["lse"].shape, -math.inf, device="cuda", dtype=torch.float64)
    for i, n in enumerate(s["host_lens"]):
        n = int(n)
        if not n:
            continue
        j = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        page, place = s["table"][i].long()[j // P], j % P
        for h in range(H):
            k, v = ((c.view(torch.uint8)[page, place, h] if case["layout"] == "nhd" else c.view(torch.uint8)[page, h, place])
                    .view(c.dtype).double() * scale[page, place // B, h].double()[:, None]
                    for c, scale in ((s["k_cache"], s["ks"]), (s["v_cache"], s["vs"])))
            heads = slice(h * G, (h + 1) * G)
            t = s["q"][i, heads].double() @ k.T * s["scale"]
            if case["softcap"]:
                t = torch.tanh(t / case["softcap"]) * case["softcap"]
            lse[i, heads] = torch.logsumexp(t, -1)
            out[i, heads] = torch.softmax(t, -1) @ v
    return out, lse


def _exact_sample(case, seed):
    s = _sample_inputs(case, seed)
    R = case["rows"]
    z = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    how = {n: v.double().cpu().numpy() if torch.is_tensor(v) else np.full(R, v, np.float64) for n, v in s["how"].items()}
    tokens, kept, logprob = np.zeros(R, np.int64), np.zeros(R, np.int32), np.zeros(R)
    for r in range(R):
        heat, k, p, low = (np.float64(np.float32(how[n][r])) for n in ("temperature", "top_k", "top_p", "min_p"))
        some = np.flatnonzero(z[r] > -np.inf)
        order = some[np.lexsort((some, -z[r, some]))]
        if heat == 0:
            k, heat = 1, 1.0
        if k > 0:
            order = order[:int(k)]
        w = np.exp((z[r, order] - z[r, order[0]]) / heat)
        n = len(w)
        if p < 1:
            # the shortest run of the most likely that holds the share p
            n = max(1, int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1)
        n = min(n, len(w), int(np.count_nonzero(w >= low)))
        order, w = order[:n], w[:n]
        by = np.argsort(order)
        up = np.cumsum(w[by])
        at = min(int(np.searchsorted(up, u[r] * up[-1], side="right")), n - 1)
        tokens[r], kept[r], logprob[r] = order[by[at]], n, math.log(w[by[at]] / up[-1])
    return torch.from_numpy(tokens), torch.from_numpy(kept), torch.from_numpy(logprob)


EXACT = {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}


def exact(case, seed):
    return EXACT[case["op"]](case, seed)
