// Attention of one new token per sequence over the paged cache: how a call's
// work is planned, and its kernels (kv_attend_kernel.cuh) for 16-bit caches and E4M3 with a
// scale per head.
#include "kv_attend_kernel.cuh"

namespace xksv {

// Where the units' clusters fit the GPU at once and the table's room is at most
// kShort tokens, a cluster takes a unit, else all warps share all blocks and a
// second kernel joins.  8 KV heads of 128 in BF16, clusters against that: one
// sequence of 777 tokens 7.6 and 10.2 us, of 4000 14.6 and 15.9; two of 4000
// 16.7 and 17.2; six of 777 11.0 and 15.8.  Past one wave the clusters lose:
// eight uneven sequences to 777 15.0 and 12.1, 64 of them 81 and 28.
constexpr uint64_t kShort = 4096;

AttendPlan kv_attend_plan(const xksv_kv_desc& c, const xksv_kv_blocks& b, uint64_t seqs, uint32_t q_heads, uint64_t table_cols, int sms) {
  AttendPlan pl{};
  const uint32_t group = q_heads / c.kv_heads;
  pl.chunks = (group + 15) / 16;
  pl.heads = (group + pl.chunks - 1) / pl.chunks;
  pl.pad_dim = uint32_t(pad_dim(c.head_dim));
  pl.page_shift = pl.block_shift = -1;
  for (int k = 0; k < 31; ++k)
    if (c.page_size == 1ull << k) pl.page_shift = k;
  uint32_t block = 16, per_sm = 1;
  if (b.block) {
    for (int k = 0; k < 31; ++k)
      if (b.block == 1ull << k) pl.block_shift = k;
    pl.even = b.block % 16 == 0;
    pl.heads <= 8 ? shape_of<ELE4M3Blocks, 1>(pl.pad_dim, &block, &per_sm) : shape_of<ELE4M3Blocks, 2>(pl.pad_dim, &block, &per_sm);
  } else if (c.type == XKSV_E4M3) {
    pl.heads <= 8 ? shape_of<ELE4M3, 1>(pl.pad_dim, &block, &per_sm) : shape_of<ELE4M3, 2>(pl.pad_dim, &block, &per_sm);
  } else {
    pl.heads <= 8 ? shape_of<EL16, 1>(pl.pad_dim, &block, &per_sm) : shape_of<EL16, 2>(pl.pad_dim, &block, &per_sm);
  }
  // no more workers than blocks of the longest sequences the table can hold
  const uint64_t longest = table_cols * c.page_size / block + 1;
  const uint64_t blocks = seqs * c.kv_heads * pl.chunks;
  const uint64_t most = uint64_t(sms) * per_sm * kWarps;
  pl.warps = uint32_t(blocks >= most || longest >= most ? most : std::min<uint64_t>(most, blocks * longest));
  // sums, maximum and weight of each head; with block scales its sums' unit
  pl.slot_floats = (uint64_t(pl.heads) * (pl.pad_dim + (b.block ? 3 : 2)) + 31) / 32 * 32;
  pl.joins_off = 2 * pl.warps * pl.slot_floats * sizeof(float);
  pl.bytes = pl.joins_off + pl.warps * sizeof(int4);
  if (blocks * kCluster <= uint64_t(sms) * per_sm && table_cols * c.page_size <= kShort) {
    pl.clusters = uint32_t(blocks);
    pl.bytes = 0;
  }
  return pl;
}

cudaError_t launch_kv_attend(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  if (p.b.block) return launch_kv_attend_blocks(p, pl, st);
  if (p.c.type == XKSV_E4M3) return launch_dim<false, ELE4M3>(p, pl, st);
  return p.c.type == XKSV_BF16 ? launch_dim<true, EL16>(p, pl, st) : launch_dim<false, EL16>(p, pl, st);
}

}  // namespace xksv
