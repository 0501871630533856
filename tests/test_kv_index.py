"""CPU: the paged cache's index arithmetic (csrc/kv_index.h) as plain C++ on
the host -- pages outside the cache, tokens outside the table, lengths and
windows at their edges -- and the binding's argument checks."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "xks-vectorforge_b200" / "csrc"


def run_cpp(tmp_path, body):
    src = tmp_path / "t.cpp"
    src.write_text('#include "kv_index.h"\n#include <cassert>\n#include <cstdio>\n#include <vector>\n'
                   "using namespace xksv;\nint main() {\n" + body + "\n return 0;\n}\n")
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-I", str(CSRC), str(src), "-o",
                    str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_page_lookup_stays_inside_the_table(tmp_path):
    run_cpp(tmp_path, """
  // 3 sequences by 4 pages, rows 5 apart; the last row holds 4 entries only
  std::vector<int32_t> t(2 * 5 + 4, 0);
  t[0] = 7; t[3] = 9; t[5] = -1; t[10 + 3] = 8; t[10] = 2147483647;
  auto at = [&](int64_t s, int32_t i) {
    const KvPlace p = kv_place(t.data(), 3, 4, 5, 9, 16, s, i);
    assert(p.place == (p.page < 0 ? 0u : uint32_t(i) % 16));
    return p.page;
  };
  assert(at(0, 0) == 7 && at(0, 15) == 7 && at(0, 16) == 0);
  assert(at(0, 63) == -1);            // page 9 of a cache of 9 pages
  assert(at(1, 3) == -1);             // page -1
  assert(at(2, 63) == 8);             // the table's last entry
  assert(at(2, 64) == -1);            // behind it
  assert(at(2, 0) == -1);             // a page number of 2^31 - 1
  assert(at(3, 0) == -1 && at(-1, 0) == -1 && at(0, -1) == -1);
  assert(at(0, 2147483647) == -1 && at(int64_t(1) << 40, 0) == -1);
""")


def test_span_of_lengths_and_windows(tmp_path):
    run_cpp(tmp_path, """
  auto is = [](KvSpan s, int64_t f, int64_t l, bool ok) { return s.first == f && s.length == l && s.ok == ok; };
  assert(is(kv_span(0, 4, 16, 0), 0, 0, true));
  assert(is(kv_span(64, 4, 16, 0), 0, 64, true));
  assert(is(kv_span(65, 4, 16, 0), 0, 0, false));
  assert(is(kv_span(-1, 4, 16, 0), 0, 0, false));
  assert(is(kv_span(64, 4, 16, 1), 63, 64, true));
  assert(is(kv_span(64, 4, 16, 64), 0, 64, true));
  assert(is(kv_span(64, 4, 16, 63), 1, 64, true));
  assert(is(kv_span(64, 4, 16, ~uint64_t(0)), 0, 64, true));
  assert(is(kv_span(0, 4, 16, 1), 0, 0, true));
""")


def test_split_covers_every_block_once(tmp_path):
    """Workers' block ranges tile all blocks; every unit is either written by
    one worker or joined from exactly the slots its workers left."""
    run_cpp(tmp_path, """
  uint64_t seed = 1;
  auto rnd = [&](uint64_t n) { seed = seed * 6364136223846793005ull + 1442695040888963407ull; return (seed >> 33) % n; };
  for (int round = 0; round < 60; ++round) {
    const uint64_t units = 1 + rnd(round % 3 ? 9 : 300), warps = 1 + rnd(round % 2 ? 1184 : 40);
    std::vector<uint64_t> u0{0};
    for (uint64_t u = 0; u < units; ++u) u0.push_back(u0.back() + 1 + rnd(rnd(4) ? 5 : 900));
    const uint64_t total = u0.back();
    const KvShare sh = kv_share(total, uint32_t(warps));
    const uint64_t workers = sh.workers;
    assert(workers == (warps < total ? warps : total));
    std::vector<int> seen(2 * workers, 0), done(units, 0);
    struct Join { uint64_t u, i; uint32_t parts; };
    std::vector<Join> joins;
    std::vector<uint64_t> slot_unit(2 * workers, ~0ull);
    for (uint64_t i = 0, u = 0; i < workers; ++i) {
      const uint64_t a = kv_start(sh, i), b = kv_start(sh, i + 1);
      assert(a < b && (i + 1 < workers || b == total) && (i || a == 0));
      for (uint64_t t = a; t < b; ++t) assert(kv_owner(sh, t) == i);
      while (u0[u + 1] <= a) ++u;
      for (uint64_t v = u; v < units && u0[v] < b; ++v) {
        const KvPiece p = kv_piece(sh, i, a, b, u0[v], u0[v + 1]);
        if (p.slot < 0) { assert(!done[v]); done[v] = 1; continue; }
        assert(uint64_t(p.slot) < 2 * workers && !seen[p.slot]);
        seen[p.slot] = 1; slot_unit[p.slot] = v;
        if (p.parts) { assert(p.parts >= 2 && p.slot == int64_t(2 * i + 1)); joins.push_back({v, i, p.parts}); }
      }
    }
    for (size_t x = 0; x < joins.size(); ++x)
      for (size_t y = x + 1; y < joins.size() && joins[y].i / 8 == joins[x].i / 8; ++y)
        assert(joins[x].parts <= 8 || joins[y].parts <= 8);
    for (auto& j : joins) {
      assert(!done[j.u]);
      done[j.u] = 1;
      for (uint32_t k = 0; k < j.parts; ++k) {
        const uint64_t slot = k ? 2 * (j.i + k) : 2 * j.i + 1;
        assert(slot < 2 * workers && slot_unit[slot] == j.u);
        slot_unit[slot] = ~0ull;
      }
    }
    for (uint64_t u = 0; u < units; ++u) assert(done[u]);
    for (uint64_t x : slot_unit) assert(x == ~0ull);
  }
  assert(kv_blocks(kv_span(0, 4, 16, 0), 16) == 0 && kv_blocks(kv_span(17, 4, 16, 0), 16) == 2);
  assert(kv_blocks(kv_span(64, 4, 16, 1), 16) == 1 && kv_blocks(kv_span(-3, 4, 16, 1), 16) == 0);
  assert(kv_blocks(kv_span(49, 4, 16, 2), 16) == 2 && kv_blocks(kv_span(49, 4, 16, 49), 32) == 2);
""")


def test_binding_refuses_before_the_library():
    torch = pytest.importorskip("torch")
    import xksv_gpu as xg
    k = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        xg.KVCache(k, k.clone())
    with pytest.raises(ValueError, match="layout"):
        xg.KVCache(k, k.clone(), layout="dhn")
    xg._torch_types()
    dev = -1  # get_device() of a CPU tensor
    x = torch.zeros(4, 8)
    assert xg._matrix(x, 4, 8, "x", dev) == (x.data_ptr(), 8)
    assert xg._matrix(x[:, :6], 4, 6, "x", dev) == (x.data_ptr(), 8)
    for bad in (x.t(), x[0], x[:, ::2], x[:3]):
        with pytest.raises(ValueError):
            xg._matrix(bad, 4, 8, "x", dev)
    with pytest.raises(ValueError, match="dtype"):
        xg._type(x.double(), (xg.BF16,), "x")
    h = torch.zeros(3, 2, 64)
    assert xg._heads(h.transpose(0, 1), 2, 3, 64, "h", dev)[1:] == (64, 128)
    with pytest.raises(ValueError, match="contiguous"):
        xg._heads(h[..., ::2], 3, 2, 32, "h", dev)
    with pytest.raises(ValueError):
        xg._ints(torch.zeros(4, dtype=torch.int64), 4, "index", dev)
    with pytest.raises(ValueError):
        xg._ints(torch.zeros(8, dtype=torch.int32)[::2], 4, "index", dev)
    with pytest.raises(ValueError):
        xg._table(torch.zeros(4, 4, dtype=torch.int32).t(), dev)


def test_argument_blocks_match_the_header(tmp_path):
    """The packed argument blocks have the C structs' sizes and field offsets."""
    import xksv_gpu as xg
    fields = {
        "xksv_linear_args": (xg.LINEAR_ARGS, "x x_cols x_stride y y_cols y_stride batch bias mul mul_stride residual "
                             "residual_stride y_type bias_type mul_type residual_type act flags"),
        "xksv_kv_append_args": (xg.KV_APPEND_ARGS, "q k v q_out q_stride[0] q_stride[1] k_stride[0] k_stride[1] v_stride[0] "
                                "v_stride[1] q_out_stride[0] q_out_stride[1] tokens table table_rows table_cols table_stride "
                                "seq index positions inv_freq rot_scale rot_dim q_heads type flags"),
        "xksv_kv_attend_args": (xg.KV_ATTEND_ARGS, "q out lse q_stride[0] q_stride[1] out_stride[0] out_stride[1] seqs table "
                                "table_cols table_stride lens scale softcap window q_heads type"),
    }
    src = tmp_path / "f.cpp"
    lines = ['#include "xksv_cuda.h"', "#include <cstddef>", "#include <cstdio>", "int main() {"]
    for name, (_, names) in fields.items():
        lines += [f'std::printf("%zu\\n", offsetof({name}, {n}));' for n in names.split()]
        lines.append(f'std::printf("%zu\\n", sizeof({name}));')
    src.write_text("\n".join(lines) + "\n}\n")
    exe = tmp_path / "f"
    subprocess.run(["g++", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = iter(int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split())
    for name, (packed, names) in fields.items():
        n = len(names.split())
        # a block whose k-th field alone is 1 (or 1.0) differs from zeros at that field's offset
        zero = packed.pack(*[0] * n)
        for k in range(n):
            one = packed.pack(*[int(k == i) for i in range(n)])
            at = next(i for i in range(len(zero)) if one[i] != zero[i])
            want = next(got)
            assert want <= at < want + 4, (name, names.split()[k])
        assert packed.size == next(got), name


def test_null_arguments_are_refused():
    import build as b
    b.build()
    import xksv_gpu as xg
    lib = xg.load()
    assert lib.xksv_kv_create(None, None) == 1
    assert lib.xksv_kv_append(None, None, None) == 1
    assert lib.xksv_kv_attend(None, None, None, 0, None) == 1
    assert lib.xksv_kv_status(None, None) == 1
    assert lib.xksv_kv_attend_workspace(None, 1, 1, 1) == 0
    assert lib.xksv_plan_linear(None, None, 0, None, None, 0, None) == 1
    assert lib.xksv_plan_linear_workspace(None, 4) == 0
    lib.xksv_kv_destroy(None)


def test_plan_calls_without_a_plan():
    import build as b
    b.build()
    import xksv_gpu as xg
    lib = xg.load()
    assert lib.xksv_plan_linear_workspace_for(None, None, 4, xg.BF16) == 0
    assert lib.xksv_plan_set_parts(None, 0) == 1
    assert lib.xksv_plan_device(None) == -1
