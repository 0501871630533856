"""Measured cases of the operators around compressed linear layers.

Three operators make the serving token step of a model whose weights stay
compressed in HBM:

* ``linear``  the product with compressed weights, with bias, activation,
  gating factor and residual in its epilogue (``xksv_gpu.Plan.linear``);
* ``append``  position rotation of new queries and keys, and the append of
  keys and values to a paged cache (``xksv_gpu.KVCache.append``);
* ``attend``  attention of one new token per sequence over that cache
  (``xksv_gpu.KVCache.attend``).

``run`` computes them through the framework where ``own`` is true, and with
elementary torch operations in 32 bits where it is false.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0
# bytes a weight of N(0, s) values takes as a compressed slab: the sign and
# mantissa byte, and the exponent's entropy of about 2.6 bits
SLAB_BYTES = 1.33


def listed():
    return [
        # ---- linear: "codec" is the archive's (serial blocks are indexed) --
        # one token through an attention output projection, residual added
        dict(name="linear-token-4096", op="linear", codec="serial", rows=4096, cols=4096, batch=1, bias=False,
             act="none", mul=False, residual=True, out="bf16", extra=0),
        # 16 requests' tokens through a gated layer's up projection: bias,
        # and the product with the activated gate
        dict(name="linear-batch16-gated", op="linear", codec="serial", rows=14336, cols=4096, batch=16, bias=True,
             act="none", mul=True, residual=False, out="bf16", extra=0),
        # a short prompt through a layer of odd sizes whose blocks are of the
        # parallel codec, rows of x inside a wider buffer, FP32 out
        dict(name="linear-ragged-parallel", op="linear", codec="parallel", rows=2040, cols=1848, batch=77, bias=True,
             act="gelu_tanh", mul=False, residual=True, out="fp32", extra=24),
        # a chunk of prompt tokens through a down projection
        dict(name="linear-prompt-2048", op="linear", codec="serial", rows=4096, cols=14336, batch=2048, bias=False,
             act="silu", mul=False, residual=True, out="bf16", extra=0),
        # ---- append ---------------------------------------------------------
        # one sequence's new token
        dict(name="append-token", op="append", tokens=1, seqs=1, pads=0, q_heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, far=30000, page=16, layout="nhd", type="bf16", cache="bf16"),
        # a padded decode batch into an 8-bit cache
        dict(name="append-batch-e4m3", op="append", tokens=200, seqs=200, pads=11, q_heads=32, kv_heads=8, dim=128,
             rot=128, interleaved=False, far=100000, page=32, layout="hnd", type="bf16", cache="e4m3"),
        # prompts of uneven lengths, part of each head rotated in pairs
        dict(name="append-prompts-interleaved", op="append", tokens=3001, seqs=7, pads=0, q_heads=20, kv_heads=20,
             dim=80, rot=32, interleaved=True, far=500, page=48, layout="nhd", type="fp16", cache="fp16"),
        # a full prefill chunk
        dict(name="append-prefill-16384", op="append", tokens=16384, seqs=5, pads=0, q_heads=32, kv_heads=8, dim=128,
             rot=128, interleaved=False, far=8000, page=64, layout="nhd", type="bf16", cache="bf16"),
        # ---- attend ---------------------------------------------------------
        # one short conversation: latency
        dict(name="attend-one-short", op="attend", seqs=1, length=777, ragged=False, empty=0, q_heads=32, kv_heads=8,
             dim=128, page=16, layout="nhd", type="bf16", cache="bf16", window=0, softcap=0.0),
        # one very long document: the split over its length
        dict(name="attend-one-long", op="attend", seqs=1, length=131071, ragged=False, empty=0, q_heads=32,
             kv_heads=8, dim=128, page=16, layout="nhd", type="bf16", cache="bf16", window=0, softcap=0.0),
        # a decode batch of uneven lengths with free slots, 8-bit cache
        dict(name="attend-batch-e4m3", op="attend", seqs=130, length=6000, ragged=True, empty=9, q_heads=28,
             kv_heads=4, dim=128, page=32, layout="hnd", type="bf16", cache="e4m3", window=0, softcap=0.0),
        # the largest batch: uneven lengths to 16384
        dict(name="attend-batch-long", op="attend", seqs=64, length=16384, ragged=True, empty=0, q_heads=32,
             kv_heads=8, dim=128, page=16, layout="nhd", type="bf16", cache="bf16", window=0, softcap=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "append", "attend"])
    if op == "linear":
        cols = _log(rng, 32, 1792) * 8
        rows = _log(rng, 256, 16384)
        if rng.random() < 0.7:
            rows = -(-rows // 16) * 16
            cols = -(-cols // 16) * 16
        while rows * cols > 4096 * 14336:
            rows = rows // 32 * 16
        return dict(op=op, codec=rng.choice(["serial", "serial", "parallel"]), rows=rows, cols=cols,
                    batch=min(_log(rng, 1, 4096), 4096 * 14336 * 2048 // (rows * cols)), bias=rng.random() < 0.5,
                    act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), mul=rng.random() < 0.3,
                    residual=rng.random() < 0.5, out=rng.choice(["bf16", "bf16", "fp32"]),
                    extra=rng.choice([0, 0, 8, 40]))
    dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 12])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    case = dict(op=op, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=rng.choice([1, 8, 16, 16, 24, 64, 256]),
                layout=rng.choice(["nhd", "hnd"]), type=kind, cache=rng.choice([kind, kind, "e4m3"]))
    if op == "append":
        cap = 16384 * 48 * 128 // ((q_heads + 2 * kv_heads) * dim)
        # prompts of a few sequences, or one new token each of many
        if rng.random() < 0.5:
            tokens = min(_log(rng, 1, 16384), cap)
            seqs = min(tokens, _log(rng, 1, 64))
        else:
            tokens = seqs = _log(rng, 1, 256)
        case.update(tokens=tokens, seqs=seqs, pads=rng.randrange(0, 1 + tokens // 8), page=min(64, case["page"]),
                    rot=dim if rng.random() < 0.6 else dim // 2, interleaved=rng.random() < 0.4,
                    far=_log(rng, 1, 1000000))
        return case
    cap = 64 * 8192 * 8 * 128 * 2 // (kv_heads * dim * (1 if case["cache"] == "e4m3" else 2))
    length = min(_log(rng, 1, 131072), cap)
    seqs = max(1, min(_log(rng, 1, 256), cap // length))
    case.update(seqs=seqs, length=length, ragged=rng.random() < 0.6, empty=rng.randrange(0, 1 + seqs // 8),
                window=_log(rng, 1, length) if rng.random() < 0.2 else 0,
                softcap=30.0 if rng.random() < 0.2 else 0.0)
    return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _lens(case, seed):
    """Lengths of the cached sequences, on the host."""
    rng = np.random.default_rng(seed)
    n, top = case["seqs"], case["length"]
    lens = rng.integers(1, top + 1, n) if case["ragged"] else np.full(n, top)
    if case["ragged"]:
        lens[rng.integers(0, n)] = top
    if case["empty"]:
        lens[rng.permutation(n)[:case["empty"]]] = 0
    return lens.astype(np.int64)


def _linear_inputs(case, seed):
    g = _gen(seed)
    R, C, B = case["rows"], case["cols"], case["batch"]
    out = TYPES[case["out"]]
    w = _randn(g, (R, C), torch.bfloat16, 0.02)
    x = _randn(g, (B, C + case["extra"]), torch.bfloat16)[:, :C]
    return dict(w=w, x=x, bias=_randn(g, (R,), torch.bfloat16, 0.5) if case["bias"] else None,
                mul=_randn(g, (B, R), torch.bfloat16) if case["mul"] else None,
                residual=_randn(g, (B, R), out) if case["residual"] else None,
                y=torch.empty(B, R, device="cuda", dtype=out))


def _pages(gen, lens, page, pool):
    """A page table over a pool of pages, in random order; unused entries -1."""
    need = [-(-int(n) // page) for n in lens]
    total, width = max(pool, sum(need)), max(1, max(need))
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, device="cuda", dtype=torch.int32)
    counts = torch.tensor(need, device="cuda")
    used = torch.arange(width, device="cuda")[None, :] < counts[:, None]
    table[used] = order[:int(used.sum())]
    return table, total


def _cache(gen, case, pages):
    """Keys and values of the cache's type and layout, and the heads' scales."""
    H, D, P, kind = case["kv_heads"], case["dim"], case["page"], case["cache"]
    shape = (pages, P, H, D) if case["layout"] == "nhd" else (pages, H, P, D)
    if kind == "e4m3":
        ks = torch.rand(H, generator=gen, device="cuda") * 0.02 + 0.01
        vs = torch.rand(H, generator=gen, device="cuda") * 0.02 + 0.01
        k, v = (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16).mul_(64.0)
                .clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn) for _ in range(2))
        return k, v, ks, vs
    k, v = (torch.randn(shape, generator=gen, device="cuda", dtype=TYPES[kind]) for _ in range(2))
    return k, v, None, None


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
    local = np.concatenate([np.arange(c) for c in counts])
    index = first[seq] + local
    positions = far[seq] + index
    pads = rng.permutation(T)[:case["pads"]]
    seq[pads] = -1
    table, total = _pages(g, first + counts, case["page"], T // case["page"] + 2 * S + 1)
    k_cache, v_cache, ks, vs = _cache(g, case, total)
    kind = TYPES[case["type"]]
    q, k, v = (_randn(g, (T, h, D), kind) for h in (case["q_heads"], case["kv_heads"], case["kv_heads"]))
    inv = 1.0 / (500000.0 ** (torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"]))
    as_int = lambda a: torch.from_numpy(a.astype(np.int32)).cuda()
    return dict(q=q, k=k, v=v, table=table, k_cache=k_cache, v_cache=v_cache, ks=ks, vs=vs, seq=as_int(seq),
                index=as_int(index), positions=as_int(positions), inv_freq=inv.float(), q_out=torch.zeros_like(q))


def _attend_inputs(case, seed):
    g = _gen(seed)
    lens = _lens(case, seed)
    table, total = _pages(g, lens, case["page"], 1)
    k_cache, v_cache, ks, vs = _cache(g, case, total)
    kind = TYPES[case["type"]]
    q = _randn(g, (case["seqs"], case["q_heads"], case["dim"]), kind)
    return dict(q=q, table=table, k_cache=k_cache, v_cache=v_cache, ks=ks, vs=vs,
                lens=torch.from_numpy(lens.astype(np.int32)).cuda(), host_lens=lens,
                scale=case["dim"] ** -0.5, out=torch.empty_like(q),
                lse=torch.empty(q.shape[:2], device="cuda", dtype=torch.float32))


INPUTS = {"linear": _linear_inputs, "append": _append_inputs, "attend": _attend_inputs}


class _Payload:
    """A weight's slabs as the GPU encoder lays them out in device memory."""

    def __init__(self, xksv_gpu, w, codec):
        stream = torch.cuda.current_stream().cuda_stream
        self.xg = xksv_gpu
        self.ptr, self.size, slabs = xksv_gpu.cuda_pack_tensor(w.data_ptr(), w.shape[0], w.shape[1], codec,
                                                               stream=stream)
        row = w.shape[1] * 2
        for s in slabs:
            s["dst_offset"] //= row
            s["rows"], s["cols"] = s["rows"] or s["src_size"] // row, w.shape[1]
        self.plan = xksv_gpu.Plan(slabs)
        if self.plan.index(self.ptr, stream, payload_bytes=self.size):
            raise RuntimeError("the encoded weight could not be indexed")

    def __del__(self):
        self.plan.close()
        self.xg.free_device(self.ptr)


def prepare(case, seed):
    s = INPUTS[case["op"]](case, seed)
    s["case"] = case
    if own:
        path = str(Path.cwd() / "xks-vectorforge_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import xksv_gpu
        if case["op"] == "linear":
            codec = xksv_gpu.CODEC_TILE16 if case["codec"] == "serial" else xksv_gpu.CODEC_PARALLEL32
            s["payload"] = _Payload(xksv_gpu, s["w"], codec)
            s["w"] = None  # the weight stays compressed
        else:
            s["cache"] = xksv_gpu.KVCache(s["k_cache"], s["v_cache"], k_scale=s["ks"], v_scale=s["vs"],
                                          layout=case["layout"])
    return s


# --------------------------------------------------------------- own calls
def _own(s):
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "linear":
        p = s["payload"]
        p.plan.linear(p.ptr, s["x"], s["y"], bias=s["bias"], act=case["act"], mul=s["mul"], residual=s["residual"],
                      payload_bytes=p.size, stream=stream)
        return s["y"]
    if case["op"] == "append":
        s["cache"].append(s["k"], s["v"], s["table"], s["index"], seq=s["seq"], positions=s["positions"],
                          inv_freq=s["inv_freq"], interleaved=case["interleaved"], q=s["q"], q_out=s["q_out"],
                          stream=stream)
        return s["q_out"], s["k_cache"], s["v_cache"]
    s["cache"].attend(s["q"], s["table"], s["lens"], s["out"], lse=s["lse"], scale=s["scale"],
                      window=case["window"], softcap=case["softcap"], stream=stream)
    return s["out"], s["lse"]


# -------------------------------------------------------------- plain form
def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_linear(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    z = _act(z, s["case"]["act"])
    if s["mul"] is not None:
        z = z * s["mul"].float()
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(s["y"].dtype)


def _rows(cache, layout):
    """[pages, page_size, heads, dim] view of a cache of either layout."""
    return cache if layout == "nhd" else cache.permute(0, 2, 1, 3)


def _rotate(x, cos, sin, rot, interleaved):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_append(s):
    case = s["case"]
    page = case["page"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    live = s["seq"] >= 0
    q = _rotate(s["q"].float(), cos, sin, case["rot"], case["interleaved"])
    s["q_out"].copy_(torch.where(live[:, None, None], q, s["q_out"].float()))
    k, v = _rotate(s["k"].float(), cos, sin, case["rot"], case["interleaved"]), s["v"].float()
    if case["cache"] == "e4m3":
        k = (k / s["ks"][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        v = (v / s["vs"][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    # padding tokens go to a spare row behind the live ones: the first live
    # token's place, written with that token's values once more
    lead = torch.argmax(live.to(torch.int32))
    src = torch.where(live, torch.arange(len(live), device="cuda"), lead)
    index = s["index"].long()[src]
    pages = s["table"][s["seq"].long()[src], index // page].long()
    for cache, rows in ((s["k_cache"], k), (s["v_cache"], v)):
        # a float8 cache is written through its bytes
        new = rows[src].to(cache.dtype)
        raw = torch.uint8 if cache.element_size() == 1 else cache.dtype
        _rows(cache.view(raw), case["layout"])[pages, index % page] = new.view(raw)
    return s["q_out"], s["k_cache"], s["v_cache"]


def _plain_attend(s):
    case = s["case"]
    H, D, page = case["kv_heads"], case["dim"], case["page"]
    k_rows, v_rows = _rows(s["k_cache"], case["layout"]), _rows(s["v_cache"], case["layout"])
    lens = s["host_lens"]
    q = s["q"].float().view(len(lens), H, -1, D)
    n = 0
    while n < len(lens):
        # as many sequences at a time as 2^28 gathered elements hold
        m, top = n, 1
        while m < len(lens) and (m == n or (m + 1 - n) * max(top, int(lens[m])) * H * D <= 1 << 28):
            top = max(top, int(lens[m]))
            m += 1
        at = s["table"][n:m, :-(-top // page)].long().clamp_(min=0)
        raw = [r if r.element_size() > 1 else r.view(torch.uint8) for r in (k_rows, v_rows)]
        k, v = (r[at].flatten(1, 2)[:, :top].view(c.dtype).float() for r, c in zip(raw, (k_rows, v_rows)))
        if case["cache"] == "e4m3":
            k, v = k * s["ks"][:, None], v * s["vs"][:, None]
        score = (q[n:m] @ k.permute(0, 2, 3, 1)) * s["scale"]
        if case["softcap"]:
            score = case["softcap"] * torch.tanh(score / case["softcap"])
        j, length = torch.arange(top, device="cuda"), s["lens"][n:m, None]
        seen = j < length
        if case["window"]:
            seen &= j >= length - case["window"]
        seen = seen[:, None, None, :]
        score = torch.where(seen, score, torch.full_like(score, -math.inf))
        high = score.amax(-1, keepdim=True).clamp_(min=-1e30)
        p = torch.exp(score - high)
        total = p.sum(-1, keepdim=True)
        v = torch.where(seen[:, 0, 0, :, None, None], v, torch.zeros_like(v))
        o = (p @ v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
        s["out"][n:m] = o.reshape(m - n, -1, D).to(s["out"].dtype)
        s["lse"][n:m] = torch.where(total > 0, high + torch.log(total), torch.full_like(total, -math.inf)).reshape(m - n, -1)
        n = m
    return s["out"], s["lse"]


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the work
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
    if case["op"] == "linear":
        R, C, B, o = case["rows"], case["cols"], case["batch"], size[case["out"]]
        n = SLAB_BYTES * R * C + 2 * B * C + o * B * R + 2 * R * case["bias"] + 2 * B * R * case["mul"]
        return {"bytes": n + o * B * R * case["residual"], "flops": 2.0 * R * C * B}
    D, H, Q, e, c = case["dim"], case["kv_heads"], case["q_heads"], size[case["type"]], size[case["cache"]]
    if case["op"] == "append":
        T = case["tokens"] - case["pads"]
        return {"bytes": float(T * D * (2 * Q * e + 2 * H * (e + c)) + 12 * case["tokens"]),
                "flops": 3.0 * T * (Q + H) * case["rot"]}
    mean = (case["length"] + 1) / 2 if case["ragged"] else case["length"]
    if case["window"]:
        mean = min(mean, case["window"])
    seen = mean * (case["seqs"] - case["empty"])
    return {"bytes": float(seen * 2 * H * D * c + 2 * case["seqs"] * Q * D * e), "flops": 4.0 * seen * Q * D}


# ------------------------------------------- the definitions, in 64 bits
def _exact_linear(case, seed):
    s = _linear_inputs(case, seed)
    z = torch.einsum("bc,rc->br", s["x"].double(), s["w"].double())
    if case["bias"]:
        z += s["bias"].double()
    if case["act"] == "relu":
        z = z.clamp(min=0)
    elif case["act"] == "silu":
        z = z * torch.sigmoid(z)
    elif case["act"] == "gelu":
        z = z * torch.special.ndtr(z)
    elif case["act"] == "gelu_tanh":
        # (1 + tanh u) / 2 is the logistic function of 2 u
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if case["mul"]:
        z *= s["mul"].double()
    if case["residual"]:
        z += s["residual"].double()
    return z


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    T, rot, page = case["tokens"], case["rot"], case["page"]
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
    slot = s["table"].long()[s["seq"].long()[live], where // page] * page + where % page
    caches = []
    for name, rows, scale in (("k_cache", turned(s["k"]), s["ks"]), ("v_cache", s["v"].double(), s["vs"])):
        c = s[name].double()
        if scale is not None:
            rows = (rows / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        at = (slot // page, slot % page) if case["layout"] == "nhd" else (slot // page, slice(None), slot % page)
        c[at] = rows[live]
        caches.append(c)
    return q_out, caches[0], caches[1]


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    H, G = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    lse = torch.full(s["lse"].shape, -math.inf, device="cuda", dtype=torch.float64)
    for i, n in enumerate(s["host_lens"]):
        n = int(n)
        if not n:
            continue
        lo = max(0, n - case["window"]) if case["window"] else 0
        j = torch.arange(lo, n, device="cuda")
        page, place = s["table"][i].long()[j // case["page"]], j % case["page"]
        for h in range(H):
            k, v = ((c[page, place, h] if case["layout"] == "nhd" else c[page, h, place]).double()
                    for c in (b.view(torch.uint8) if b.element_size() == 1 else b for b in (s["k_cache"], s["v_cache"])))
            if case["cache"] == "e4m3":
                k, v = ((c[page, place, h] if case["layout"] == "nhd" else c[page, h, place]).view(torch.float8_e4m3fn).double()
                        for c in (s["k_cache"].view(torch.uint8), s["v_cache"].view(torch.uint8)))
                k, v = k * s["ks"][h].double(), v * s["vs"][h].double()
            heads = slice(h * G, (h + 1) * G)
            t = s["q"][i, heads].double() @ k.T * s["scale"]
            if case["softcap"]:
                t = torch.tanh(t / case["softcap"]) * case["softcap"]
            lse[i, heads] = torch.logsumexp(t, -1)
            out[i, heads] = torch.softmax(t, -1) @ v
    return out, lse


def exact(case, seed):
    return {"linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, seed)
