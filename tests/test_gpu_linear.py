"""GPU: the linear layer on compressed weights (Plan.linear) against the plain
form in 64 bits, over codecs, batches on every route, epilogues, strides and
plans of several weights, and its refusals.

Tolerance (derived, per element): z is a sum of C exact products (BF16 times
BF16) and a bias, added in FP32 in some order: off by at most (C + 1) 2^-24
sum |w x| + 2^-23 |bias|; an activation changes that by at most 1.13 times and
adds its own 8 ulp, 2^-21 (|z| + 1); the factor multiplies both; residual and
output add an ulp each; y is rounded once, by half a step of its type."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402
from helpers import bf16_to_f32, words_for  # noqa: E402

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def pack(mats, seed, lead=3):
    """Slabs of each (rows, cols, y row, x offset, codec) weight, at odd byte
    offsets; returns the payload on the device, entries and weights."""
    rng = np.random.default_rng(seed)
    payload, entries, ws = bytearray(b"\0" * lead), [], []
    for R, C, y0, xo, codec in mats:
        w = words_for("normal002", R * C, rng).reshape(R, C)
        ws.append((torch.from_numpy(bf16_to_f32(w)).to(DEV), y0, xo))
        for r0 in range(0, R, 16):
            rows = w[r0:r0 + 16].astype("<u2")
            blob = rows.tobytes() if codec == xg.CODEC_RAW else xg.host_pack(rows.tobytes(), len(rows), C, codec)
            entries.append(dict(src_offset=len(payload), src_size=len(blob), rows=len(rows), cols=C,
                                dst_offset=y0 + r0, x_offset=xo, codec=codec))
            payload += blob
    return torch.frombuffer(payload, dtype=torch.uint8).to(DEV), entries, ws


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def expected(ws, x, yn, bias, act, mul, residual):
    """(y, tolerance before rounding, covered columns)."""
    B = x.shape[0]
    z, tol = (torch.zeros(B, yn, dtype=torch.float64, device=DEV) for _ in range(2))
    cover = torch.zeros(yn, dtype=torch.bool, device=DEV)
    for w, y0, xo in ws:
        R, C = w.shape
        xs, wd = x[:, xo:xo + C].double(), w.double()
        z[:, y0:y0 + R] = xs @ wd.t()
        tol[:, y0:y0 + R] = (C + 1) * 2.0 ** -24 * (xs.abs() @ wd.abs().t())
        cover[y0:y0 + R] = True
    if bias is not None:
        z, tol = z + bias.double(), tol + 2.0 ** -23 * bias.double().abs()
    y = act64(z, act)
    if act != "none":
        tol = 1.13 * tol + 2.0 ** -21 * (z.abs() + 1)
    if mul is not None:
        y, tol = y * mul.double(), tol * mul.double().abs() + 2.0 ** -23 * (y * mul.double()).abs()
    if residual is not None:
        y, tol = y + residual.double(), tol + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, tol + 2.0 ** -23 * y.abs(), cover


def check(plan, payload, ws, xn, yn, batch, out="bf16", bias=None, act="none", mul=None, residual=None, x_pad=0,
          seed=0, rounds=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x = rnd(batch, xn + x_pad).to(torch.bfloat16)[:, :xn]
    b = rnd(yn).to(DT[bias]) if bias else None
    m = rnd(batch, yn + 5).to(DT[mul])[:, 2:2 + yn] if mul else None
    r = rnd(batch, yn).to(DT[residual]) if residual else None
    for _ in range(rounds):
        y = torch.full((batch, yn + 3), 77.0, device=DEV, dtype=DT[out])[:, :yn]
        plan.linear(payload, x, y, bias=b, act=act, mul=m, residual=r)
        assert plan.status() == 0
        want, tol, cover = expected(ws, x, yn, b, act, m, r)
        got = y.double()
        err = (got - want).abs()
        ok = err <= torch.finfo(DT[out]).eps / 2 * want.abs() + tol
        assert ok[:, cover].all(), (batch, float(err[:, cover].max()))
        assert (got[:, ~cover] == 77).all()
        assert (y.as_strided((batch, 3), (yn + 3, 1), y.storage_offset() + yn) == 77).all()


SERIAL, PARALLEL, RAW = 1, 2, 0
# one weight; several with a gap between their rows and columns; odd shapes
PLANS = {
    "serial": [(160, 512, 0, 0, SERIAL)],
    "serial-many": [(512, 256, 0, 0, SERIAL), (48, 256, 560, 0, SERIAL), (64, 1024, 512 + 128, 256, SERIAL)],
    "serial-tail": [(40, 512, 3, 0, SERIAL)],
    "parallel": [(96, 512, 0, 0, PARALLEL)],
    "raw": [(64, 264, 0, 0, RAW)],
    "mixed": [(32, 256, 0, 8, SERIAL), (20, 256, 32, 8, PARALLEL), (16, 256, 60, 8, RAW), (33, 1000, 100, 0, RAW)],
    "odd-cols": [(37, 250, 0, 0, SERIAL), (20, 77, 40, 3, PARALLEL)],
}


def build(name, seed=1):
    payload, entries, ws = pack(PLANS[name], seed)
    xn = max(xo + C for _, C, _, xo, _ in PLANS[name])
    yn = max(y0 + R for R, _, y0, _, _ in PLANS[name])
    return payload, entries, ws, xn, yn


@pytest.mark.parametrize("name", PLANS)
@pytest.mark.parametrize("batch", [1, 2, 3, 4, 7, 16, 33, 128, 129, 300])
def test_linear_matches_64_bits(name, batch):
    payload, entries, ws, xn, yn = build(name)
    plan = xg.Plan(entries)
    for indexed in (False, True):
        if indexed:
            assert plan.index(payload) == 0
        check(plan, payload, ws, xn, yn, batch, seed=batch)
        check(plan, payload, ws, xn, yn, batch, out="fp32", bias="bf16", act="silu", mul="bf16", residual="fp32",
              x_pad=3, seed=batch + 1)
    plan.close()


@pytest.mark.parametrize("name", ["serial", "serial-many"])
@pytest.mark.parametrize("route", [xg.GEMM_FUSED, xg.GEMM_SCRATCH])
@pytest.mark.parametrize("batch", [4, 64, 65, 100, 128])
def test_linear_routes_that_a_caller_picks(name, route, batch):
    payload, entries, ws, xn, yn = build(name)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0
    auto = plan.linear_workspace(batch)
    plan.set_gemm_route(route)
    check(plan, payload, ws, xn, yn, batch, bias="fp32", act="gelu", residual="bf16", seed=batch)
    # the default decodes on its own past 64 tokens
    assert (plan.linear_workspace(batch) == auto) or (route == xg.GEMM_FUSED) == (batch > 64)
    plan.close()


@pytest.mark.parametrize("act", list(xg.ACTS))
@pytest.mark.parametrize("batch", [1, 3, 20, 200])
def test_linear_epilogues(act, batch):
    payload, entries, ws, xn, yn = build("serial-many", 2)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0
    for out in ("bf16", "fp32"):
        for bias, mul, residual in (("fp32", None, "bf16"), (None, "fp32", None), ("bf16", "bf16", "bf16")):
            check(plan, payload, ws, xn, yn, batch, out=out, bias=bias, act=act, mul=mul, residual=residual,
                  x_pad=8, seed=batch)
    plan.close()


@pytest.mark.parametrize("batch", [1, 2, 16, 256, 1000])
def test_linear_larger_weight(batch):
    """Several slab groups and splits of the columns over CTAs."""
    rng = np.random.default_rng(3)
    R, C = 1040, 4112
    w = words_for("student3", R * C, rng).reshape(R, C)
    words = np.ascontiguousarray(w.astype("<u2"))  # held while its address is in use
    pay, slabs = xg.host_pack_tensor(words.ctypes.data, R * C * 2, R, C, SERIAL)
    for s in slabs:
        s["dst_offset"] //= 2 * C
        s["rows"], s["cols"] = s["rows"] or s["src_size"] // (2 * C), C
    payload = torch.from_numpy(pay).to(DEV)
    ws = [(torch.from_numpy(bf16_to_f32(w)).to(DEV), 0, 0)]
    plan = xg.Plan(slabs)
    assert plan.index(payload) == 0
    check(plan, payload, ws, C, R, batch, bias="bf16", act="gelu", residual="bf16", seed=batch, rounds=2)
    plan.close()


@pytest.mark.parametrize("batch", [1, 16, 70, 300])
@pytest.mark.parametrize("cols", [520, 8200])
def test_linear_fp32_sums_stay_fp32(batch, cols):
    """An FP32 result's relative error does not grow with the columns.  The
    tensor cores cut each addition towards zero by at most the last place of
    the running sum, 2^-23 (2^-24 on average), 32 additions of 16 columns to an
    accumulator: 32 * 2^-24 of the result's norm, with what is added in FP32
    behind it far below."""
    payload, entries, ws = pack([(64, cols, 0, 0, xg.CODEC_PARALLEL32), (64, cols, 64, 0, xg.CODEC_TILE16)], 5)
    plan = xg.Plan(entries)
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(batch, cols, generator=g, device=DEV).bfloat16()
    y = torch.empty(batch, 128, device=DEV)
    plan.linear(payload, x, y)
    torch.cuda.synchronize()
    assert plan.status() == 0
    want = x.double() @ torch.cat([w for w, _, _ in ws]).double().t()
    assert float((y - want).norm() / want.norm()) <= 32 * 2.0 ** -24


@pytest.mark.parametrize("batch", [1, 3, 16, 200])
def test_linear_in_place_and_special_values(batch):
    """The residual and the factor may be y itself; infinities and NaN in one
    token's x stay in that token's row."""
    payload, entries, ws, xn, yn = build("serial", 4)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0
    g = torch.Generator(device=DEV).manual_seed(batch)
    x = torch.randn(batch, xn, generator=g, device=DEV).to(torch.bfloat16)
    y0 = torch.randn(batch, yn, generator=g, device=DEV).to(torch.bfloat16)
    for kw in (dict(residual=None), dict(mul=None)):
        y = y0.clone()
        kw = {k: y for k in kw}
        plan.linear(payload, x, y, act="relu", **kw)
        ref = {k: y0 for k in kw}
        want, tol, _ = expected(ws, x, yn, None, "relu", ref.get("mul"), ref.get("residual"))
        assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + tol).all()
    x[0, 5], x[-1, 9] = float("inf"), float("nan")
    y = torch.zeros(batch, yn, dtype=torch.bfloat16, device=DEV)
    plan.linear(payload, x, y)
    assert torch.isnan(y[-1]).all()
    assert not torch.isfinite(y[0]).any()
    if batch > 2:
        want, tol, _ = expected(ws, x[1:-1], yn, None, "none", None, None)
        assert ((y[1:-1].double() - want).abs() <= 2.0 ** -8 * want.abs() + tol).all()
    assert plan.status() == 0
    plan.close()


@pytest.mark.parametrize("batch", [1, 16, 160])
def test_linear_captured_on_another_stream(batch):
    """A chain of two layers captured into a graph on a side stream and replayed on new inputs."""
    pa, ea, wa = pack([(256, 128, 0, 0, SERIAL)], 5)
    pb, eb, wb = pack([(128, 256, 0, 0, SERIAL)], 6)
    up, down = xg.Plan(ea), xg.Plan(eb)
    assert up.index(pa) == 0 and down.index(pb) == 0
    x = torch.zeros(batch, 128, dtype=torch.bfloat16, device=DEV)
    h = torch.zeros(batch, 256, dtype=torch.bfloat16, device=DEV)
    y = torch.zeros(batch, 128, dtype=torch.bfloat16, device=DEV)

    def run():
        st = torch.cuda.current_stream().cuda_stream
        up.linear(pa, x, h, act="silu", stream=st)
        down.linear(pb, h, y, residual=x, stream=st)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(3):
        x.copy_(torch.randn(batch, 128, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        graph.replay()
        want, tol, _ = expected(wa, x, 256, None, "silu", None, None)
        assert ((h.double() - want).abs() <= 2.0 ** -8 * want.abs() + tol).all()
        want, tol, _ = expected(wb, h, 128, None, "none", None, x)
        assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + tol).all()
    assert up.status() == 0 and down.status() == 0
    up.close()
    down.close()


def test_linear_reports_bad_stream():
    payload, entries, ws, xn, yn = build("serial", 7)
    plan = xg.Plan(entries)
    payload[entries[0]["src_offset"] + 8] ^= 1  # its bit count
    for batch in (1, 200):
        y = torch.zeros(batch, yn, dtype=torch.bfloat16, device=DEV)
        plan.linear(payload, torch.zeros(batch, xn, dtype=torch.bfloat16, device=DEV), y)
        assert plan.status() == 1
    plan.close()


def test_linear_refusals():
    payload, entries, ws, xn, yn = build("serial", 8)
    plan = xg.Plan(entries)
    x, y = torch.zeros(2, xn, dtype=torch.bfloat16, device=DEV), torch.zeros(2, yn, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        plan.linear(payload, x.float(), y)
    with pytest.raises(ValueError):
        plan.linear(payload, x, y.half())
    with pytest.raises(ValueError):
        plan.linear(payload, x, y, act="tanh")
    with pytest.raises(ValueError):
        plan.linear(payload, x, y, bias=y[0, :-1])
    with pytest.raises(ValueError):
        plan.linear(payload, x, y, residual=y[:1])
    with pytest.raises(ValueError):
        plan.linear(payload, x, y.cpu())
    with pytest.raises(RuntimeError):
        plan.linear(payload, x[:, :-8], y)  # x too narrow
    with pytest.raises(RuntimeError):
        plan.linear(payload, x, y[:, :-1])  # y too narrow
    with pytest.raises(RuntimeError):
        plan.linear(payload, x, y[:1].expand(2, yn))  # rows of y overlap
    with pytest.raises(RuntimeError):
        plan.linear(payload[:-1], x, y)  # payload too short
    with pytest.raises(RuntimeError):
        plan.linear(payload, x, y, workspace=torch.zeros(256, dtype=torch.uint8, device=DEV))
    plan.linear(payload, x[:0], y[:0])  # no tokens: nothing happens
    plan.close()
    two = xg.Plan(entries + [dict(entries[0], dst_offset=8)])  # rows covered twice
    with pytest.raises(RuntimeError):
        two.linear(payload, x, y)
    two.close()


@pytest.mark.parametrize("batch", [4, 16, 64])
def test_linear_fp32_sums_stay_fp32_where_a_cta_holds_all_columns(batch):
    """The fused route: more groups of slabs than SMs (each reads other columns
    of x), so that a CTA adds all 8192 columns of its groups.  Weights and x are
    above zero, so what is cut off adds up: each addition cuts less than the
    running sum's last place, 2^-23 of it, 32 additions of 16 columns to an
    accumulator; the 16 accumulators of 512 columns are added in FP32, half a
    last place each, 16 * 2^-24 (one accumulator for all columns: 512 * 2^-24
    on average)."""
    cols, n = 8192, 160
    rng = np.random.default_rng(23)
    payload, entries, ws = bytearray(), [], []
    for i in range(n):
        w = (words_for("normal002", 16 * cols, rng) & 0x7FFF).astype("<u2")
        blob = xg.host_pack(w.tobytes(), 16, cols, SERIAL)
        entries.append(dict(src_offset=len(payload), src_size=len(blob), rows=16, cols=cols, dst_offset=16 * i,
                            x_offset=16 * i, codec=SERIAL))
        payload += blob
        ws.append(bf16_to_f32(w).reshape(16, cols))
    payload = torch.frombuffer(payload, dtype=torch.uint8).to(DEV)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0 and plan.fused_ready(payload)
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.rand(batch, cols + 16 * n, generator=g, device=DEV).bfloat16()
    want = torch.cat([x[:, 16 * i:16 * i + cols].double() @ torch.from_numpy(w).to(DEV).double().t()
                      for i, w in enumerate(ws)], 1)
    y = torch.empty(batch, 16 * n, device=DEV)
    plan.linear(payload, x, y)
    assert plan.status() == 0
    assert float((y - want).norm() / want.norm()) <= 32 * 2.0 ** -23 + 16 * 2.0 ** -24
    plan.close()


def plan_of(R, C, seed, kind="normal002"):
    """An indexed plan of one serial weight: (payload, plan, FP32 weight)."""
    w = words_for(kind, R * C, np.random.default_rng(seed)).reshape(R, C)
    words = np.ascontiguousarray(w.astype("<u2"))
    pay, slabs = xg.host_pack_tensor(words.ctypes.data, R * C * 2, R, C, SERIAL)
    for s in slabs:
        s["dst_offset"] //= 2 * C
        s["rows"], s["cols"] = s["rows"] or s["src_size"] // (2 * C), C
    return torch.from_numpy(pay).to(DEV), xg.Plan(slabs), torch.from_numpy(bf16_to_f32(w)).to(DEV)


@pytest.mark.parametrize("batch", [1, 4, 16, 64, 65])
def test_workspace_asked_for_before_an_index_serves_after_it(batch):
    payload, plan, w = plan_of(1024, 4096, 21)
    ws = torch.empty(plan.linear_workspace(batch), dtype=torch.uint8, device=DEV)
    x = torch.randn(batch, 4096, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).bfloat16()
    for step in range(3):
        if step == 1:
            assert plan.index(payload) == 0
        elif step == 2:
            plan.set_gemm_route(xg.GEMM_FUSED)
        for out in (torch.bfloat16, torch.float32):
            y = torch.empty(batch, 1024, device=DEV, dtype=out)
            plan.linear(payload, x, y, workspace=ws)
            want, tol, _ = expected([(w, 0, 0)], x, 1024, None, "none", None, None)
            assert ((y.double() - want).abs() <= torch.finfo(out).eps / 2 * want.abs() + tol).all()
    assert plan.status() == 0
    plan.close()


def test_calls_reserve_what_their_route_uses():
    """One token through an indexed weight reserves no decoded copy of it."""
    payload, plan, w = plan_of(1024, 4096, 22)
    assert plan.index(payload) == 0
    x = torch.ones(64, 4096, dtype=torch.bfloat16, device=DEV)
    y = torch.empty(64, 1024, dtype=torch.bfloat16, device=DEV)

    def taken(batch):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        plan.linear(payload, x[:batch], y[:batch])
        return torch.cuda.max_memory_allocated() - before

    assert taken(1) <= 4096 and taken(3) <= 4096
    assert taken(4) < 8 << 20  # the segments' sums of 16 tokens; the decoded weight is 8 MB
    other = payload.clone()  # another payload than the indexed one is decoded first
    want = y[:1].clone()
    plan.linear(payload, x[:1], want)
    plan.linear(other, x[:1], y[:1])
    assert ((y[0].double() - want[0].double()).abs() <= 2.0 ** -8 * want[0].double().abs() + 2.0 ** -12).all()
    assert plan.status() == 0
    plan.close()
