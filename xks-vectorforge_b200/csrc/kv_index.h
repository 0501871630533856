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

// Page that holds token `index` of sequence `seq`, read from a page table of
// `rows` sequences by `cols` pages whose rows are `stride` entries apart; -1
// when the token lies outside the table or its page outside the cache.  The
// table is read only inside its bounds.
XKSV_HD int64_t kv_page(const int32_t* table, uint64_t rows, uint64_t cols, uint64_t stride, uint64_t pages,
                        uint64_t page_size, int64_t seq, int64_t index) {
  if (seq < 0 || uint64_t(seq) >= rows || index < 0) return -1;
  const uint64_t col = uint64_t(index) / page_size;
  if (col >= cols) return -1;
  const int64_t page = table[uint64_t(seq) * stride + col];
  return page < 0 || uint64_t(page) >= pages ? -1 : page;
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

}  // namespace xksv
