// Index arithmetic of the paged key/value cache, shared by its kernels and
// by host code (compiles as plain C++).
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define XKSV_HD __host__ __device__ __forceinline__
#else
#define XKSV_HD inline
#endif

namespace xksv {

// Where token `index` of sequence `seq` lives, from a page table of `rows`
// sequences by `cols` pages whose rows are `stride` entries apart; page -1
// when the token lies outside the table or its page outside the cache.  The
// table is read only inside its bounds.  Indexes are below 2^31: 32-bit division.
struct KvPlace {
  int32_t page;
  uint32_t place;
};
XKSV_HD KvPlace kv_place(const int32_t* table, uint64_t rows, uint64_t cols, uint64_t stride, uint64_t pages,
                         uint32_t page_size, int64_t seq, int32_t index) {
  if (seq < 0 || uint64_t(seq) >= rows || index < 0) return KvPlace{-1, 0};
  const uint32_t col = uint32_t(index) / page_size;
  if (col >= cols) return KvPlace{-1, 0};
  const int32_t page = table[uint64_t(seq) * stride + col];
  return page < 0 || uint64_t(page) >= pages ? KvPlace{-1, 0} : KvPlace{page, uint32_t(index) - col * page_size};
}

// Whether token t (above 0) goes on with the one before it in the same block of
// `block` tokens: of the same sequence, its place one higher.  Without `seq`
// every token is a sequence of its own.
XKSV_HD bool kv_follows(const int32_t* seq, const int32_t* index, uint64_t t, uint32_t block) {
  return seq && t > 0 && seq[t] >= 0 && seq[t] == seq[t - 1] && index[t - 1] >= 0 && index[t - 1] < index[t] &&
         index[t] - index[t - 1] == 1 && uint32_t(index[t]) % block != 0;
}

// The exponent of the least power of two 2^e, e >= -60, with high <= 448 * 2^e
// (E4M3) or high <= 127 * 2^e; from the bits of a finite FP32 number >= 0.
XKSV_HD int kv_scale_exponent(uint32_t high, bool integer) {
  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  const int e = int(high >> 23) - 127 - (integer ? 6 : 8) + ((high & 0x7fffffu) > (integer ? 0x7e0000u : 0x600000u) ? 1 : 0);
  return e < -60 ? -60 : e;
}

// Cached tokens that a new token attends to: [first, length).  A length
// outside [0, cols * page_size] is an error and attends to nothing.
struct KvSpan {
  int64_t first, length;
  bool ok;
};
XKSV_HD KvSpan kv_span(int64_t length, uint64_t cols, uint64_t page_size, uint64_t window) {
  if (length < 0 || uint64_t(length) > cols * page_size) return KvSpan{0, 0, false};
  const int64_t first = window && uint64_t(length) > window ? length - int64_t(window) : 0;
  return KvSpan{first, length, true};
}

// ------------------------------------------------------ the attention's split
// A unit is one (sequence, KV head, chunk of query heads); its cached tokens
// are cut into blocks at multiples of the block's size (so that a block lies
// in as few pages as it can); an empty unit has none.
XKSV_HD uint64_t kv_blocks(KvSpan s, uint32_t tokens) {
  return s.length > s.first ? uint64_t(s.length + tokens - 1) / tokens - uint64_t(s.first) / tokens : 0;
}
// All units' blocks in order, `total` of them, are shared evenly among
// workers = min(warps, total): worker i takes blocks [start(i), start(i + 1)),
// quot or quot + 1 of them.
struct KvShare {
  uint64_t total, quot;
  uint32_t workers, more;  // the first `more` workers take quot + 1
};
XKSV_HD KvShare kv_share(uint64_t total, uint32_t warps) {
  const uint32_t w = total < warps ? uint32_t(total) : warps;
  const uint64_t q = w ? total / w : 0;
  return KvShare{total, q, w, uint32_t(total - q * w)};
}
XKSV_HD uint64_t kv_start(const KvShare& s, uint32_t worker) {
  return worker * s.quot + (worker < s.more ? worker : s.more);
}
// The worker that holds a block.
XKSV_HD uint32_t kv_owner(const KvShare& s, uint64_t block) {
  const uint64_t head = s.more * (s.quot + 1);
  return block < head ? uint32_t(block / (s.quot + 1)) : s.more + uint32_t((block - head) / s.quot);
}
// What worker `i`, holding blocks [a, b), does with its piece of the unit of
// blocks [u0, u1): writes the output (slot -1) or leaves the piece in a slot
// for the join.  A worker leaves at most two pieces: one of a unit begun
// before its blocks (slot 2 i), one of a unit that goes on behind them (slot
// 2 i + 1).  parts > 0 on the unit's first piece: the join reads that one and
// the slots 2 (i + 1), .. , 2 (i + parts - 1).  Among n workers in a row
// one at most begins a unit of more than n parts.
struct KvPiece {
  int64_t slot;
  uint32_t parts;
};
XKSV_HD KvPiece kv_piece(const KvShare& s, uint32_t i, uint64_t a, uint64_t b, uint64_t u0, uint64_t u1) {
  if (u0 >= a && u1 <= b) return KvPiece{-1, 0};
  if (u0 < a) return KvPiece{2 * int64_t(i), 0};
  return KvPiece{2 * int64_t(i) + 1, kv_owner(s, u1 - 1) - i + 1};
}

}  // namespace xksv
