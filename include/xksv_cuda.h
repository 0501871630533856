/*
 * xksv_cuda.h -- C ABI of the B200 slab decoder (libxksv_cuda.so).
 *
 * Part 1 keeps the reference's GPU entry points: same names, signatures,
 * argument meaning and return codes, so ctypes callers of the reference
 * library (python/runtime.py:40-44, 251-255; python/tune.py:16-19) load this
 * library unchanged through XKSV_CUDA_LIBRARY.  `input` is a HOST pointer to
 * one encoded slab; `output`, `x` are DEVICE pointers on the current device.
 * Each call is synchronous and returns 0 on success, 1 on any failure
 * (null pointer, bad header or size, invalid codebook or bit stream, CUDA
 * error).  Outputs are written only through device kernels of this library.
 *
 * Part 2 adds a device-resident batched interface (no counterpart in the
 * reference): a plan describes many slabs of one payload buffer already in
 * device memory; decode / GEMV / GEMM are enqueued on a caller stream
 * without host synchronisation, and errors are collected in a device status
 * word read back by xksv_plan_status().
 *
 * Parts 7 and 8 serve a model whose weights stay compressed (no counterpart
 * in the reference): a linear layer on a plan's weights with its epilogue,
 * and a paged key/value cache with the attention that reads it.
 */
#ifndef XKSV_CUDA_H
#define XKSV_CUDA_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------- Part 1: reference-compatible entry points ------------- */

/* Serial-codec ("bf16-huffman-tile16") slab -> BF16 row-major [rows, cols]
 * at output.  Replaces reference cuda/decode.cu:85-87 (validation :47-66). */
int xksv_cuda_decode(const void* input, size_t size, size_t rows, size_t cols, void* output);

/* Serial-codec slab fused with y = W x: x is FP32 [cols], output FP32 [rows]
 * (overwritten).  Replaces reference cuda/decode.cu:89-92. */
int xksv_cuda_gemv(const void* input, size_t size, size_t rows, size_t cols, const float* x,
                   float* output);

/* Serial-codec slab fused with Y = W X: x is FP32 row-major [cols, batch],
 * output FP32 row-major [rows, batch] (overwritten).  Replaces reference
 * cuda/decode.cu:94-98. */
int xksv_cuda_gemm(const void* input, size_t size, size_t rows, size_t cols, size_t batch,
                   const float* x, float* output);

/* Parallel-codec ("bf16-huffman-parallel32", XKSP2) slab -> BF16 row-major
 * [rows, cols] (dimensions read from the slab header).  Replaces reference
 * cuda/parallel.cu:68-70 (validation :33-53). */
int xksv_cuda_decode_parallel(const void* input, size_t n, void* output);

/* Parallel-codec slab fused with y = W x, x FP32 [cols], output FP32 [rows]
 * (overwritten).  Replaces reference cuda/parallel.cu:71-74. */
int xksv_cuda_gemv_parallel(const void* input, size_t n, const float* x, float* output);

/* ---------------- Part 2: batched, device-resident interface ------------ */

enum {
  XKSV_CODEC_RAW = 0,        /* block stores the source bytes unchanged */
  XKSV_CODEC_TILE16 = 1,     /* "bf16-huffman-tile16" (serial codec) */
  XKSV_CODEC_PARALLEL32 = 2  /* "bf16-huffman-parallel32" (XKSP2) */
};

/* One archive block, as listed in the archive index (src/compile.cpp:459-470):
 * where its bytes sit in the payload buffer, its slab shape, and where its
 * result goes.  For decode, dst_offset is a byte offset into the output.
 * For GEMV/GEMM, dst_offset is the first output row and x_offset the element
 * offset of this slab's column 0 inside x (so one plan can serve several
 * weight matrices).  Raw blocks used by GEMV/GEMM must give rows and cols
 * (BF16 row-major data); raw blocks used by decode only need src_size. */
typedef struct xksv_slab {
  uint64_t src_offset;
  uint64_t src_size;
  uint64_t rows;
  uint64_t cols;
  uint64_t dst_offset;
  uint64_t x_offset;
  uint32_t codec;
  uint32_t flags; /* must be 0 */
} xksv_slab;

typedef struct xksv_plan xksv_plan;

/* Validates the host table, copies it to the current device and groups it by
 * codec.  Returns 0 and a plan, or 1.  The plan records the extents its
 * table needs: payload bytes (largest src_offset + src_size), decoded bytes
 * (largest dst_offset + rows * cols * 2, or + src_size for raw blocks), X rows
 * (largest x_offset + cols) and Y rows (largest dst_offset + rows).  Every call
 * below is given the size of each device buffer it reads or writes and
 * returns 1 without launching anything when a slab lies outside one: a bad
 * table entry never reaches a kernel as an out-of-bounds access. */
int xksv_plan_create(const xksv_slab* slabs, size_t n, xksv_plan** plan);
void xksv_plan_destroy(xksv_plan* plan);

/* Enqueues decode of every slab of the plan from d_payload (device,
 * payload_size bytes) into d_out (device, out_size bytes) on `stream` (a
 * cudaStream_t; NULL = legacy default stream).  Returns 1 for launch errors
 * and, without launching, when a slab lies outside either buffer or when
 * d_out or a coded slab's dst_offset is odd (BF16 words need 2-byte
 * alignment); stream errors are found by xksv_plan_status(). */
int xksv_plan_decode(const xksv_plan* plan, const void* d_payload, size_t payload_size, void* d_out,
                     size_t out_size, void* stream);

/* The same decode from a HOST payload (pinned memory for overlap): the first
 * payload_size bytes at h_payload are copied into d_payload (device, at least
 * as large) in 8 pieces on a plan-owned stream while the slabs of each piece
 * that has landed are decoded on `stream`, so the copy and the decode
 * overlap.  The copies wait for work already enqueued on `stream`.  Needs
 * each codec's slabs in increasing payload order (an archive's block order;
 * otherwise, and for a plan indexed on d_payload, it copies once and then
 * decodes).  Returns 1 as xksv_plan_decode does (a slab past payload_size or
 * past out_size included).  No reference counterpart (the reference stages
 * one slab per blocking call, cuda/decode.cu:47-83). */
int xksv_plan_decode_host(const xksv_plan* plan, const void* h_payload, size_t payload_size,
                          void* d_payload, void* d_out, size_t out_size, void* stream);

/* Enqueues Y[dst_offset + r, b] = sum_c W[r, c] * X[x_offset + c, b] for every
 * slab, X FP32 row-major [x_rows, batch] and Y FP32 row-major [y_rows, batch]
 * (rows of Y not covered by a slab are left untouched).  Returns 1 without
 * launching when a slab lies outside the payload, X or Y. */
int xksv_plan_gemm(const xksv_plan* plan, const void* d_payload, size_t payload_size, const float* d_x,
                   size_t x_rows, float* d_y, size_t y_rows, size_t batch, void* stream);

/* The tensor-core path (batch >= 4) decodes the plan's weights into a BF16
 * scratch before its GEMM; by default each plan allocates its own on first
 * use and keeps it, i.e. a decoded copy of its weights.  Plans whose calls
 * are serialised on one stream can share one caller-owned scratch instead:
 * xksv_plan_scratch_bytes gives the bytes a plan needs (0 when it has no
 * tensor-core path) and xksv_plan_set_scratch lends it a device buffer of at
 * least that size, 256-byte aligned (the plan's own scratch, if any, is
 * freed; NULL returns to an own scratch).  Returns 1 for a buffer too small
 * or misaligned.  The caller keeps the buffer alive while the plan uses it. */
size_t xksv_plan_scratch_bytes(const xksv_plan* plan);
int xksv_plan_set_scratch(xksv_plan* plan, void* d_scratch, size_t bytes);

/* Tensor-core routing of xksv_plan_gemm for 4 <= batch <= 128 on a plan
 * indexed for the payload (xksv_plan_index) whose slabs are all 16-row
 * serial-codec slabs: XKSV_GEMM_FUSED decodes each tile row straight into
 * the shared-memory operand stages of the tensor-core MMAs (one kernel, no
 * decoded weight written to memory); XKSV_GEMM_SCRATCH decodes into the BF16
 * scratch and runs the tensor-core GEMM on it (also the route for larger
 * batches and other plans); XKSV_GEMM_AUTO (the default) picks the fused
 * kernel wherever it applies.  Returns 1 for an unknown route. */
enum { XKSV_GEMM_AUTO = 0, XKSV_GEMM_SCRATCH = 1, XKSV_GEMM_FUSED = 2 };
int xksv_plan_set_gemm_route(xksv_plan* plan, int route);
/* 1 when the fused route applies to this plan and payload (after
 * xksv_plan_index), else 0. */
int xksv_plan_fused_ready(const xksv_plan* plan, const void* d_payload);

/* Synchronises `stream`, returns 0 when no slab reported an error since the
 * last call (then clears the word), else 1. */
int xksv_plan_status(const xksv_plan* plan, void* stream);

/* Number of kernel launches the last xksv_plan_decode / xksv_plan_gemm call
 * enqueued (for accounting in benchmarks). */
int xksv_plan_launches(const xksv_plan* plan);

/* Builds the plan's tile index for resident weights: one decode pass over
 * the plan's 16-row serial-codec slabs with cols % 16 == 0 records the bit
 * offsets at which every 16x16 tile's codes and its row 8 start (8 bytes per
 * tile) and each slab's decode tables (5920 bytes per slab), all kept on the
 * device with the plan.  Afterwards xksv_plan_gemm and xksv_plan_decode with
 * the same d_payload pointer decode those slabs tile-parallel (one or two
 * threads per tile) instead of re-synchronising each slab's single bit
 * stream on every call.
 * Serial-codec slabs of other shapes up to 16 rows get an index for decoding
 * (xksv_plan_decode, and layers that decode first).  Of the plan's
 * parallel-codec slabs, when they are too few to fill the GPU with one warp
 * each and the largest has 16384 elements or more, it records where parts of
 * their substreams begin (4 bytes per 32 or more codes) and their decode
 * tables (10 KB a slab), so that a decode shares each slab among several
 * warps.  Of the compressed weight that is 29 % for 2048 x 2048, 13 % for
 * 4096 x 4096 and 4 % for 4096 x 14336; xksv_plan_set_parts(plan, 0) leaves it
 * off.
 * The index describes the payload's contents at this call: rebuild it if they
 * change.  No reference counterpart (the reference decodes every slab from
 * its first bit, cuda/decode.cu:12-45); it is an acceleration structure on
 * the side, the slab format is unchanged.  Synchronises `stream`; 0 on
 * success, 1 on a bad slab or CUDA error (no index is kept then).  Calls on
 * one plan must not overlap, and a former index is freed: graphs captured
 * with it are not replayed after this call. */
int xksv_plan_index(xksv_plan* plan, const void* d_payload, size_t payload_size, void* stream);

/* Whether the plan's next xksv_plan_index records parts of parallel-codec
 * slabs (nonzero, the default) or not (0).  Returns 1 for NULL. */
int xksv_plan_set_parts(xksv_plan* plan, int on);


/* ---------------- Part 3: archive-side encoder (host CPU) --------------- */
/* The compile step that produces slabs for the decoder; byte-identical to the
 * reference's xksv_pack (codec XKSV_CODEC_TILE16, src/c_api.cpp:18-28) and
 * xksv_pack_parallel (XKSV_CODEC_PARALLEL32, src/c_api.cpp:44-65): same
 * argument checks, 0 on success and 1 on failure (the reference returns -1),
 * output malloc'd and released with xksv_host_free. */
int xksv_host_pack(const void* data, size_t n, size_t rows, size_t cols, int codec, void** out,
                   size_t* out_size);
void xksv_host_free(void* p);

/* Splits a row-major BF16 [rows, cols] tensor into the compiler's slabs
 * (whole rows, at most 16 rows and 1 MiB each: src/compile.cpp:449-479),
 * encodes them on `threads` host threads (0 = all cores), keeps an encoding
 * only when smaller than the raw bytes (src/compile.cpp:268-275), and returns
 * the concatenated payload plus one xksv_slab per slab (dst_offset =
 * dst_base + the slab's byte offset in the tensor).  Both outputs are
 * malloc'd; release them with xksv_host_free. */
int xksv_host_pack_tensor(const void* data, size_t nbytes, size_t rows, size_t cols, int codec,
                          int threads, uint64_t dst_base, void** payload, size_t* payload_size,
                          xksv_slab** table, size_t* nslabs);

/* GPU encoder: the slabs of xksv_host_pack_tensor, byte-identical, built on
 * the current device from a row-major BF16 [rows, cols] tensor in device
 * memory (histograms, Huffman lengths with the reference's tie order,
 * canonical codes and bit packing in kernels; src/compile.cpp:247-285,
 * 449-479, src/c_api.cpp:18-28, 44-65, src/codec.cpp:32-58).  *d_payload is
 * device memory allocated by the library (release with xksv_cuda_free), the
 * slab table host memory as for xksv_host_pack_tensor.  Synchronises
 * `stream`; 0 on success, 1 on bad arguments, a CUDA error, or a code longer
 * than 32 bits (not produced for the compiler's <= 1 MiB slabs). */
int xksv_cuda_pack_tensor(const void* d_data, size_t rows, size_t cols, int codec, uint64_t dst_base,
                          void** d_payload, size_t* payload_size, xksv_slab** table, size_t* nslabs,
                          void* stream);
void xksv_cuda_free(void* d_ptr);

/* ---------------- Part 4: decode without device allocation -------------- */
/* No counterpart in the reference.  For callers that cannot let a library
 * allocate device memory -- a server that has reserved the whole GPU for its
 * own allocator, or code that cannot afford cudaMalloc's implicit
 * device-wide synchronisation.  Decodes the n slabs of `slabs` (host array,
 * same fields as for xksv_plan_create) from d_payload into d_out (both device
 * buffers owned by the caller) on `stream`, then waits for the stream and
 * returns 0 on success, 1 on a bad table entry (a slab outside the
 * payload_size bytes at d_payload or the out_size bytes at d_out included,
 * found before any launch), a launch error or a slab that fails to decode,
 * and 2 when n exceeds XKSV_NOALLOC_MAX_SLABS.
 * Besides the caller's buffers it uses only a fixed scratch array compiled
 * into the library (the slab table and a status word, about 192 KiB on every
 * GPU that loads the library, kept until the process exits).  The first call
 * on a device looks that array up (cudaGetSymbolAddress) and keeps its
 * address: make it before any stream capture, and make no call on a device
 * after a cudaDeviceReset of it (the address is stale then).  All calls
 * share the array: calls that overlap on the GPU race, so issue them one at
 * a time. */
#define XKSV_NOALLOC_MAX_SLABS 4096
int xksv_cuda_decode_noalloc(const xksv_slab* slabs, size_t n, const void* d_payload, size_t payload_size,
                             void* d_out, size_t out_size, void* stream);

/* Fused variant: no separate collective.  The indexed GEMV kernel writes its
 * output rows into this rank's block of its own gathered buffer; the grid's
 * last CTA copies the block into every other rank's buffer (CUDA IPC peer
 * mappings, stores over NVLink), fences once and raises this rank's flag on
 * every rank; a one-warp kernel on each rank then waits (bounded, about a
 * second; an error bit in the plan's status word after that) until all
 * ranks' flags reach this call.  Plain peer stores only, no multicast.  The
 * gathered buffers alternate between two halves on successive calls, so a
 * result stays valid until the call after next on any rank. */
#define XKSV_TP_IPC_BYTES 64
typedef struct xksv_tp_fused xksv_tp_fused;

/* Allocates this rank's gathered buffers (2 x nranks * max_rows_shard *
 * max_batch floats, max_batch <= 4) and flags on the current device and
 * returns its IPC handle (XKSV_TP_IPC_BYTES) for the other ranks.  0 or 1. */
int xksv_tp_fused_create(int nranks, int rank, size_t max_rows_shard, size_t max_batch, xksv_tp_fused** ctx,
                         void* ipc_handle);
/* Opens the peers' buffers: handles = every rank's handle, in rank order. */
int xksv_tp_fused_open(xksv_tp_fused* ctx, const void* handles);
/* Enqueues the fused GEMV/GEMM (batch <= max_batch) of this rank's plan,
 * which must hold only 16-row serial-codec slabs with a tile index for
 * d_payload (xksv_plan_index) and write no row at or past rows_shard.  X is
 * FP32 [x_rows, batch].  The gathered Y [nranks * rows_shard, batch] (rank
 * order) is copied to d_y_full when it is not NULL, and its address in the
 * context's buffers is stored to *d_gathered when that is not NULL.
 * Collective: every rank makes the same calls in the same order.  1 for bad
 * arguments (a slab outside the payload, X or the rank's rows included) or
 * launch errors. */
int xksv_tp_fused_gemm(xksv_tp_fused* ctx, const xksv_plan* plan, const void* d_payload, size_t payload_size,
                       const float* d_x, size_t x_rows, size_t rows_shard, size_t batch, float* d_y_full,
                       float** d_gathered, void* stream);
void xksv_tp_fused_destroy(xksv_tp_fused* ctx);

/* ---------------- Part 6: SHA-256 of decoded bytes on the GPU ----------- */
/* The archive index stores the SHA-256 of every block's and tensor's decoded
 * BF16 bytes (reference src/compile.cpp:255, 483; checked after decoding in
 * src/verify.cpp:262-273 on the CPU).  These compute FIPS 180-4 SHA-256 on
 * the device, so decoded weights are verified without copying them back.
 * No reference counterpart.  Enqueued on `stream`; 0 on success, 1 on bad
 * arguments or a CUDA error. */

/* n ranges of device memory at d_base: ranges[2i] = byte offset,
 * ranges[2i + 1] = length (a HOST array); 32-byte digests to d_digests
 * (device, n * 32 bytes). */
int xksv_cuda_sha256(const uint64_t* ranges, size_t n, const void* d_base, void* d_digests, void* stream);

/* Digest i (slab order of xksv_plan_create) = SHA-256 of slab i's decoded
 * bytes in d_out (out_size bytes): [dst_offset, dst_offset + rows * cols * 2),
 * or src_size bytes for a raw slab. */
int xksv_plan_sha256(const xksv_plan* plan, const void* d_out, size_t out_size, void* d_digests, void* stream);

/* ---------------- Part 5: tensor-parallel fused GEMV / GEMM ------------- */
/* One process per GPU; each rank's plan holds the slabs of its own rows
 * [g*R/G, (g+1)*R/G) of W with dst_offset rebased to the shard's first row.
 * No reference counterpart (the reference has no multi-GPU path); the NCCL
 * library is opened at run time (libnccl.so.2, reusing an already loaded
 * copy), so these return 1 when it is absent. */
#define XKSV_TP_ID_BYTES 128

/* A fresh NCCL unique id (XKSV_TP_ID_BYTES bytes) for xksv_tp_comm_create:
 * made by one rank and sent to the others by the caller. 0 or 1. */
int xksv_tp_unique_id(void* id);

/* Collective over nranks processes: creates this rank's communicator on the
 * current CUDA device.  0 or 1. */
int xksv_tp_comm_create(const void* id, int nranks, int rank, void** comm);
void xksv_tp_comm_destroy(void* comm);

/* Enqueues on `stream`: d_y_shard[rows_shard, batch] = W_shard X (the fused
 * plan GEMM, X FP32 [x_rows, batch]), then one all-gather of every rank's
 * shard into d_y_full[nranks * rows_shard, batch] (rank order = row order;
 * all ranks pass the same rows_shard).  Returns 1 for launch errors and,
 * without launching, for a slab outside the payload, X or the shard's rows;
 * slab errors are read with xksv_plan_status. */
int xksv_tp_gemm(const xksv_plan* plan, const void* d_payload, size_t payload_size, const float* d_x,
                 size_t x_rows, float* d_y_shard, size_t rows_shard, float* d_y_full, size_t batch, void* comm,
                 void* stream);

/* ---------------- Part 7: linear layer on compressed weights ------------ */
/* No reference counterpart (the reference's GEMV takes one FP32 column and
 * leaves bias, activation and residual to the caller, python/runtime.py:
 * 264-284).  Element types of activations and caches: */
enum { XKSV_BF16 = 1, XKSV_FP16 = 2, XKSV_FP32 = 3, XKSV_E4M3 = 4, XKSV_INT8 = 5 };
enum { XKSV_ACT_NONE = 0, XKSV_ACT_RELU = 1, XKSV_ACT_SILU = 2, XKSV_ACT_GELU = 3, XKSV_ACT_GELU_TANH = 4 };

/* For every token b and every row r of Y that a slab covers:
 *   z = sum_c W[r, c] x[b, x_offset + c] + bias[r]
 *   y[b, r] = act(z) * mul[b, r] + residual[b, r]
 * Rows of Y are y's columns (dst_offset + r of the slab, below y_cols);
 * columns of Y that no slab covers are left as they were.  x is BF16
 * [batch, x_cols], y BF16 or FP32 [batch, y_cols]; consecutive tokens are
 * x_stride, y_stride, mul_stride and residual_stride elements apart (at
 * least the columns; 2- or 4-byte aligned rows will do).  bias [y_cols], mul and
 * residual [batch, y_cols] are BF16 or FP32, NULL when absent.  residual and
 * mul may be y itself (same type and stride); no other buffers overlap y.
 * GELU is z Phi(z); GELU_TANH its tanh form; SILU z / (1 + exp(-z)).  Sums,
 * bias, activation, product and residual are FP32, rounded once into y. */
typedef struct xksv_linear_args {
  const void* x;
  uint64_t x_cols, x_stride;
  void* y;
  uint64_t y_cols, y_stride;
  uint64_t batch;
  const void* bias;
  const void* mul;
  uint64_t mul_stride;
  const void* residual;
  uint64_t residual_stride;
  uint32_t y_type, bias_type, mul_type, residual_type; /* XKSV_BF16 or XKSV_FP32; ignored for NULL */
  uint32_t act;                                        /* XKSV_ACT_* */
  uint32_t flags;                                      /* must be 0 */
} xksv_linear_args;

/* Enqueues the layer on `stream`, on the device the plan was created on.
 * d_workspace is caller-owned device memory, 256-byte aligned, its contents
 * free before and after; calls that may overlap need their own (and their own
 * plan: one call in flight per plan).  xksv_plan_linear_workspace(plan, batch)
 * bytes serve every call of that batch, whatever the payload and the result's
 * type, before and after xksv_plan_index and xksv_plan_set_gemm_route (some
 * route decodes the weight there); xksv_plan_linear_workspace_for gives what a
 * call on d_payload takes as the plan stands, often far less: ask again after
 * either of the two.  Allocates nothing, so it can be captured into a graph.  A
 * tile index (xksv_plan_index) speeds it up as it does xksv_plan_gemm, and
 * xksv_plan_set_gemm_route selects the route of 4 to 128 tokens here too
 * (XKSV_GEMM_AUTO: fused up to 64 tokens; past them, and for other plans of
 * columns in multiples of 8, the weight is decoded into the workspace, 2 bytes
 * an element).  Returns 1 without launching for 2^20 tokens or more, a slab
 * outside the payload, x or y, two slabs covering the same row of Y, a raw slab
 * that is not rows x cols, unknown types or activations, or a workspace too
 * small; batch 0 does nothing.  Slab errors are read with xksv_plan_status.  As in
 * xksv_plan_gemm, batches that share a row between several CTAs add in an
 * order that may differ between runs (the last bits of the FP32 sums). */
size_t xksv_plan_linear_workspace(const xksv_plan* plan, size_t batch);
size_t xksv_plan_linear_workspace_for(const xksv_plan* plan, const void* d_payload, size_t batch, uint32_t y_type);
/* The device the plan was created on (-1 for NULL). */
int xksv_plan_device(const xksv_plan* plan);
int xksv_plan_linear(const xksv_plan* plan, const void* d_payload, size_t payload_size,
                     const xksv_linear_args* args, void* d_workspace, size_t workspace_bytes, void* stream);

/* ---------------- Part 8: paged key/value cache ------------------------- */
/* No reference counterpart.  The cache is two caller-owned device buffers of
 * pages; a page holds page_size tokens of every KV head.  Element (page p,
 * token t, head h, dim d) of k is k[p * k_stride[0] + t * k_stride[1] +
 * h * k_stride[2] + d], likewise v: strides in elements, so pages may be
 * [page_size, heads, dim] or [heads, page_size, dim] or slices of a larger
 * buffer.  type is XKSV_BF16, XKSV_FP16 or XKSV_E4M3; an E4M3 element stands
 * for its value times k_scale[h] / v_scale[h] (device FP32 [kv_heads]; NULL:
 * 1).  A sequence's tokens live in the pages its row of the page table lists:
 * token j in page table[j / page_size] at place j % page_size. */
typedef struct xksv_kv_desc {
  void* k;
  void* v;
  uint64_t k_bytes, v_bytes; /* buffer sizes */
  uint64_t pages, page_size;
  uint64_t k_stride[3], v_stride[3]; /* page, token, head */
  const float* k_scale;
  const float* v_scale;
  uint32_t kv_heads, head_dim, type, flags; /* flags must be 0 */
} xksv_kv_desc;
typedef struct xksv_kv xksv_kv;

/* Describes a cache on the current device.  Returns 1 for null or
 * misaligned buffers (16 bytes), strides that are no multiple of 16 bytes,
 * that leave the buffer or let two elements overlap, a head_dim above 256 or
 * whose row is no multiple of 16 bytes, and scales with a 16-bit type.
 * Every call below runs on this device, whichever is current. */
int xksv_kv_create(const xksv_kv_desc* desc, xksv_kv** kv);

/* A cache of 8-bit elements with a scale for each block of tokens and head:
 * type is XKSV_E4M3 or XKSV_INT8 (two's complement, -127 .. 127), k_scale and v_scale of the
 * desc are NULL, and an element of place t and head h of a page stands for its
 * value times the FP32 number scale[page * stride[0] + t / block * stride[1] +
 * h * stride[2]] (strides in elements; `block` divides page_size).  No scale
 * needs to be known beforehand: xksv_kv_append sets them.  The tokens of one
 * call that go to one block make each head's scale the least power of two 2^e, e >= -60,
 * that holds their largest finite element (448 or 127 times the scale), or
 * leave the block's scale as it is where that is larger and the block's first
 * new token is not its first place; where the scale rises, the
 * elements of the block's places before are rounded to it again.  A call that writes a block's
 * first place begins the block anew; its places behind the new tokens hold
 * nothing.  In such a call the tokens of one sequence stand next to each
 * other, their index rising by one (padding may stand between sequences): a call that breaks
 * this, or two sequences that write to one block, leave the
 * elements of the blocks concerned undefined; the former is reported by
 * xksv_kv_status.  NaN becomes E4M3's NaN, or an integer zero, reported by
 * xksv_kv_status.  Infinite elements saturate.  xksv_kv_attend takes any
 * positive finite scales.  Returns 1 as xksv_kv_create does, and for scales that
 * leave their buffers or overlap. */
typedef struct xksv_kv_blocks {
  float* k_scale;
  float* v_scale;
  uint64_t k_bytes, v_bytes; /* buffer sizes */
  uint64_t block;
  uint64_t k_stride[3], v_stride[3]; /* page, block, head */
} xksv_kv_blocks;
int xksv_kv_create_blocks(const xksv_kv_desc* desc, const xksv_kv_blocks* blocks, xksv_kv** kv);
void xksv_kv_destroy(xksv_kv* kv);
/* Synchronises `stream`; 0 when no call reported an error since the last one
 * (then clears the word), else 1: a page outside the cache, a sequence or a
 * place outside the page table, a length above the table's; with block scales
 * also a sequence's tokens out of order, and NaN for an integer. */
int xksv_kv_status(const xksv_kv* kv, void* stream);

/* New tokens into the cache.  Token t is token index[t] of sequence seq[t]
 * (NULL: sequence t) and its rotation position is positions[t] (NULL:
 * index[t]).  Keys and queries are rotated: for the pairs (a, b) of the first
 * rot_dim dims -- (i, i + rot_dim / 2), or (2i, 2i + 1) with
 * XKSV_KV_INTERLEAVED -- and the angle positions[t] * inv_freq[i],
 *   (a, b) -> rot_scale * (a cos - b sin, b cos + a sin),
 * angles exact to FP32 after reduction at any position; rot_dim 0 rotates
 * nothing.  Values are stored as they are.  A stored element is rounded once
 * (E4M3: divided by the head's scale, saturated at 448, NaN kept).  q [tokens,
 * q_heads, head_dim] rotated goes to q_out (may be q itself with the same strides);
 * both NULL when there is none.  Strides in elements: [0] token, [1] head;
 * the last dimension is contiguous; any alignment of the type will do.
 * A token whose seq or index is negative is padding: nothing of it is read or
 * written.  A token outside the table or whose page is outside the cache is
 * skipped too and reported by xksv_kv_status.  Two tokens of one call with
 * the same place leave either one's elements there. */
#define XKSV_KV_INTERLEAVED 1u
typedef struct xksv_kv_append_args {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  uint64_t q_stride[2], k_stride[2], v_stride[2], q_out_stride[2];
  uint64_t tokens;
  const int32_t* table; /* [table_rows, table_cols], rows table_stride apart */
  uint64_t table_rows, table_cols, table_stride;
  const int32_t* seq;
  const int32_t* index;
  const int32_t* positions;
  const float* inv_freq; /* device FP32 [rot_dim / 2] */
  float rot_scale;
  uint32_t rot_dim, q_heads;
  uint32_t type;  /* of q, k, v and q_out: XKSV_BF16, XKSV_FP16 or XKSV_FP32 */
  uint32_t flags; /* XKSV_KV_INTERLEAVED or 0 */
} xksv_kv_append_args;
int xksv_kv_append(const xksv_kv* kv, const xksv_kv_append_args* args, void* stream);

/* Attention of one new token per sequence: with L = lens[s] cached tokens
 * (the new one included, its key appended first), query head h of KV head
 * g = h / (q_heads / kv_heads), and j over the last `window` of the L tokens
 * (0: all of them),
 *   t_j = scale * q[s, h] . K[j, g]   (softcap c > 0: c * tanh(t_j / c))
 *   out[s, h] = sum_j softmax(t)_j V[j, g],   lse[s, h] = log sum_j exp(t_j).
 * No score above -infinity (L = 0 among them): zeros and -infinity; a score
 * that is NaN or +infinity: NaN in both; an infinite element of an attended
 * value: infinity or NaN there. Tokens behind L, and the rest of
 * their pages, are not read. q and out are [seqs, q_heads, head_dim] of
 * `type`, strides in elements ([0] sequence, [1] head), the last dimension
 * contiguous; type is the cache's, or BF16 or FP16 over an 8-bit cache. lse is
 * FP32 [seqs, q_heads] contiguous, or NULL. Scores, softmax statistics and
 * sums are FP32, a weight enters its product within 2^-17 of itself (8-bit and FP16
 * caches: 2^-23, or 2^-40 of the largest weight where that is more; with block scales
 * its product with its value's scale within 2^-23, or 2^-40 of the largest weight
 * times the largest scale among the sixteen tokens of the same j / 16; scales below
 * 2^-125 of the sequence's largest may count as zero; scale * q . k without the key's
 * scale is an FP32 number too, infinite beyond those). A length that is negative or above table_cols * page_size
 * gives zeros and -infinity, a page outside the cache counts as masked; both
 * are reported by xksv_kv_status. d_workspace: as for xksv_plan_linear, of at
 * least xksv_kv_attend_workspace(kv, seqs, q_heads, table_cols) bytes (0 for
 * few sequences of short tables: NULL will do). The work is split over the
 * tokens and joined in a fixed order: the same call gives the same bits. */
typedef struct xksv_kv_attend_args {
  const void* q;
  void* out;
  float* lse;
  uint64_t q_stride[2], out_stride[2];
  uint64_t seqs;
  const int32_t* table; /* [seqs, table_cols], rows table_stride apart */
  uint64_t table_cols, table_stride;
  const int32_t* lens;
  float scale, softcap;
  uint64_t window;
  uint32_t q_heads, type;
} xksv_kv_attend_args;
size_t xksv_kv_attend_workspace(const xksv_kv* kv, size_t seqs, size_t q_heads, size_t table_cols);
int xksv_kv_attend(const xksv_kv* kv, const xksv_kv_attend_args* args, void* d_workspace, size_t workspace_bytes,
                   void* stream);

/* ---------------- Part 9: sampling -------------------------------------- */
/* No reference counterpart.  Draws one token for each row of logits [rows,
 * vocab] (contiguous rows, `stride` elements apart, 0 for one and the same; any
 * alignment of the type).
 * With the row's tokens ordered by logit z, equal ones by index, and w =
 * exp((z - largest z) / temperature), a token is kept when
 *   - fewer than top_k tokens are before it (top_k <= 0: all),
 *   - the weights before it sum to less than top_p times the sum of those that
 *     top_k keeps (top_p >= 1: all; the first is always kept), and
 *   - w >= min_p (min_p <= 0: all; above 1 as 1) and w >= exp(-700).
 * The token is the first, by index, whose kept weights up to and including its
 * own sum to more than u[row] times all kept ones (u below 0 as 0; u >= 1: the
 * last kept).
 * Temperature 0 takes the first token of the order, else it lies in
 * [1e-6, 1e6].  Weights and sums are FP64 in a fixed order.  Tokens at -infinity
 * are never kept.  A row with a NaN, without a logit above -infinity or with
 * one at infinity, or with a temperature outside these or a NaN among its
 * settings gives token -1, kept 0 and logprob NaN.
 * tokens is int64 [rows]; kept (int32 [rows], NULL or the number of kept
 * tokens) and logprob (FP32 [rows], NULL or the log of the token's share of
 * the kept weights).  temperature, top_k, top_p and min_p are [rows] on the
 * device, or NULL for the `_all` number.  Runs on CUDA device `device`,
 * whichever is current; no workspace.  Returns 1 without launching for bad
 * arguments: more than XKSV_SAMPLE_MAX_VOCAB tokens or 2^24 rows, misaligned
 * pointers, a temperature_all outside its range, a NaN. */
#define XKSV_SAMPLE_MAX_VOCAB (1u << 22)
typedef struct xksv_sample_args {
  const void* logits;
  uint64_t rows, vocab, stride;
  const float* u;
  int64_t* tokens;
  int32_t* kept;
  float* logprob;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int32_t top_k_all;
  float top_p_all, min_p_all;
  uint32_t type;   /* XKSV_BF16, XKSV_FP16 or XKSV_FP32 */
  int32_t device;
  uint32_t flags;  /* must be 0 */
} xksv_sample_args;
int xksv_sample(const xksv_sample_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* XKSV_CUDA_H */
