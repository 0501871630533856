"""CPU: the index arithmetic of appends to a cache with block scales
(csrc/kv_index.h) as plain C++ on the host."""
from test_kv_index import run_cpp


def test_runs_end_with_blocks_sequences_and_disorder(tmp_path):
    run_cpp(tmp_path, """
  //                     0  1  2  3  4  5  6   7  8  9 10
  const int32_t seq[] = {0, 0, 0, 0, 1, 1, -1, 1, 2, 2, 2};
  const int32_t idx[] = {2, 3, 4, 5, 6, 8, 9, 10, 7, 6, 2147483647};
  std::vector<bool> want4 = {false, true, false, true, false, false, false, false, false, false, false};
  for (uint64_t t = 0; t < 11; ++t) {
    assert(kv_follows(seq, idx, t, 4) == want4[t]);
    assert(!kv_follows(nullptr, idx, t, 4));
    assert(!kv_follows(seq, idx, t, 1));
  }
  assert(kv_follows(seq, idx, 2, 16));
  const int32_t one[] = {0, 0}, low[] = {-1, 0}, far[] = {2147483647, -2147483647 - 1};
  assert(!kv_follows(one, low, 1, 4));
  assert(!kv_follows(one, far, 1, 4));
""")


def test_least_scale_that_holds_a_number(tmp_path):
    run_cpp(tmp_path, """
  auto e = [](float x, bool i) { uint32_t b; __builtin_memcpy(&b, &x, 4); return kv_scale_exponent(b, i); };
  assert(e(448.f, false) == 0 && e(448.00003f, false) == 1 && e(224.f, false) == -1 && e(0.4375f, false) == -10);
  assert(e(127.f, true) == 0 && e(127.00001f, true) == 1 && e(63.5f, true) == -1 && e(1.f, true) == -6);
  assert(e(0.f, false) == -60 && e(0.f, true) == -60 && e(1e-44f, true) == -60 && e(1e-30f, false) == -60);
  assert(e(3.4028235e38f, false) == 120 && e(3.4028235e38f, true) == 122);
  for (int k = -40; k < 100; ++k)
    for (float m : {1.f, 1.25f, 1.75f, 1.7500001f, 1.984375f, 1.9843751f, 1.9999999f})
      for (bool i : {false, true}) {
        const double x = double(m) * __builtin_ldexp(1.0, k), top = i ? 127 : 448;
        const int s = e(float(x), i);
        assert(x <= top * __builtin_ldexp(1.0, s) && x > top * __builtin_ldexp(1.0, s - 1));
      }
""")
