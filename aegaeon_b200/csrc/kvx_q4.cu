// Entry points of the 4-bit paged KV cache (include/kvx.h, kvx_q4_*): checks of
// arguments on the host, then one or two kernel launches on the caller's stream.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/kvx.h"
#include "kvx_q4_attention.cuh"
#include "kvx_q4_extend.cuh"
#include "kvx_q4_rows.cuh"

namespace kvx {
void record_error(const std::string& msg);  // kvx_runtime.cu

namespace q4 {
namespace {

int fail(int code, const std::string& msg) {
  record_error(msg);
  return code;
}

int cuda_fail(const char* what, cudaError_t e) {
  return fail(KVX_ERR_CUDA, std::string(what) + ": " + cudaGetErrorName(e) + " (" +
                                cudaGetErrorString(e) + ")");
}

bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Geometry of a cache from the arguments of an entry point.
int cache_of(const void* key_pages, const void* value_pages, int64_t stride, int64_t num_blocks, int64_t kv_heads, int64_t block_size,
             int64_t head_dim, Cache* out) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(KVX_ERR_INVALID_ARGUMENT, "head_dim must be 64, 128 or 256");
  if (block_size < 16 || block_size % 16 || block_size > 4096)
    return fail(KVX_ERR_INVALID_ARGUMENT, "block_size must be a multiple of 16, at most 4096");
  if (kv_heads < 1 || kv_heads > 1024)
    return fail(KVX_ERR_INVALID_ARGUMENT, "kv_heads must be in [1, 1024]");
  if (num_blocks < 0 || num_blocks > INT32_MAX)
    return fail(KVX_ERR_INVALID_ARGUMENT, "num_blocks must be in [0, 2^31)");
  const int64_t head_bytes = block_size * (head_dim / 2 + 4);
  if (num_blocks > 0) {
    if (!key_pages || !value_pages) return fail(KVX_ERR_INVALID_ARGUMENT, "null cache pages");
    if (!aligned(key_pages, 16) || !aligned(value_pages, 16) || stride % 16)
      return fail(KVX_ERR_INVALID_ARGUMENT,
                  "cache pages and the stride between them must be multiples of 16 bytes");
    if (stride < kv_heads * head_bytes)
      return fail(KVX_ERR_INVALID_ARGUMENT, "page stride below the size of a page");
    if (stride > INT64_MAX / num_blocks)
      return fail(KVX_ERR_INVALID_ARGUMENT, "pages beyond the address space");
  }
  out->pages[0] = static_cast<uint8_t*>(const_cast<void*>(key_pages));
  out->pages[1] = static_cast<uint8_t*>(const_cast<void*>(value_pages));
  out->stride = stride;
  out->num_blocks = num_blocks;
  out->kv_heads = int(kv_heads);
  out->block_size = int(block_size);
  out->head_bytes = int(head_bytes);
  return KVX_OK;
}

int64_t element_size(int dtype) { return dtype == kFp32 ? 4 : 2; }

bool rows_vec(const Rows& r, int dtype) {
  const int64_t e = element_size(dtype);
  return aligned(r.base, 16) && r.token_stride * e % 16 == 0 && r.head_stride * e % 16 == 0;
}

template <typename T, int D>
void launch_rows(bool write, bool vec, const RowArgs& a, unsigned grid, cudaStream_t s) {
  if (write) {
    if (vec) q4_write<T, D, true><<<grid, kRowThreads, 0, s>>>(a);
    else q4_write<T, D, false><<<grid, kRowThreads, 0, s>>>(a);
  } else {
    if (vec) q4_read<T, D, true><<<grid, kRowThreads, 0, s>>>(a);
    else q4_read<T, D, false><<<grid, kRowThreads, 0, s>>>(a);
  }
}

template <typename T>
void launch_rows(bool write, bool vec, int head_dim, const RowArgs& a, unsigned grid,
                 cudaStream_t s) {
  if (head_dim == 64) launch_rows<T, 64>(write, vec, a, grid, s);
  else if (head_dim == 128) launch_rows<T, 128>(write, vec, a, grid, s);
  else launch_rows<T, 256>(write, vec, a, grid, s);
}

int run_rows(bool write, RowArgs& a, int dtype, int64_t num_tokens, int64_t head_dim,
             void* stream) {
  if (dtype != kBf16 && dtype != kFp16 && dtype != kFp32)
    return fail(KVX_ERR_INVALID_ARGUMENT, "unknown dtype");
  if (num_tokens < 0) return fail(KVX_ERR_INVALID_ARGUMENT, "negative token count");
  if (num_tokens == 0) return KVX_OK;
  if (!a.rows[0].base || !a.rows[1].base || !a.slots)
    return fail(KVX_ERR_INVALID_ARGUMENT, "null argument");
  for (const Rows& r : a.rows)
    if (!aligned(r.base, element_size(dtype)))
      return fail(KVX_ERR_INVALID_ARGUMENT, "rows are not aligned to their type");
  if (!aligned(a.slots, 8))
    return fail(KVX_ERR_INVALID_ARGUMENT, "slots are not aligned to their type");
  if (num_tokens > INT32_MAX / a.cache.kv_heads)
    return fail(KVX_ERR_INVALID_ARGUMENT, "too many tokens in one call");
  const int64_t num_rows = num_tokens * a.cache.kv_heads;
  a.num_rows = uint32_t(num_rows);
  a.by_heads = Divisor::of(uint32_t(a.cache.kv_heads));
  a.by_block = Divisor::of(uint32_t(a.cache.block_size));
  const int64_t per_block = kRowThreads / (head_dim / 16);
  const int64_t grid = (num_rows + per_block - 1) / per_block;
  const bool vec = rows_vec(a.rows[0], dtype) && rows_vec(a.rows[1], dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == kBf16) launch_rows<__nv_bfloat16>(write, vec, int(head_dim), a, unsigned(grid), s);
  else if (dtype == kFp16) launch_rows<__half>(write, vec, int(head_dim), a, unsigned(grid), s);
  else launch_rows<float>(write, vec, int(head_dim), a, unsigned(grid), s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KVX_OK : cuda_fail(write ? "q4_write" : "q4_read", e);
}

// ---- attention -----------------------------------------------------------------

// Query rows of a tile: the smallest of 8, 16, 32 that holds a sequence's rows
// (the row count pads to it), at most 16 where D = 256 fills the registers.
int tile_rows(int64_t rows, int64_t head_dim) {
  if (rows <= 8) return 8;
  if (rows <= 16 || head_dim == 256) return 16;
  return 32;
}

// CTAs that are resident on the device at once.
int resident(int rows, int64_t head_dim, int sms) {
  return ctas_per_sm(int(head_dim), rows) * sms;
}

int sm_count(int* sms, int* device) {
  cudaError_t e = cudaGetDevice(device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *device);
  return e == cudaSuccess ? KVX_OK : cuda_fail("cudaDeviceGetAttribute", e);
}

// Items up to which the join takes a block for each row: 18 or more warps share
// an item then, and the rows' blocks still fit the device in a wave or two.
constexpr int64_t kJoinByItem = 64;

uint64_t workspace_of(int rows, int64_t head_dim, int sms) {
  const uint64_t shares = uint64_t(kWarps) * resident(rows, head_dim, sms);
  return 2 * shares * rows * (4 * head_dim + 8) + shares * sizeof(Joint);
}

template <typename T, int D, int NT>
int launch_attention(const AttnArgs& a, int grid, int64_t items, double bound,
                     int device, cudaStream_t s) {
  constexpr int shared = Shape<D>::kShared;
  static std::atomic<uint64_t> allowed{0};  // devices that know the shared-memory size
  cudaError_t e = cudaSuccess;
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(q4_attend<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             shared);
    if (e != cudaSuccess) return cuda_fail("cudaFuncSetAttribute", e);
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  q4_attend<T, D, NT><<<grid, kThreads, shared, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail("q4_attend", e);
  if (bound <= 1) return KVX_OK;  // one share has the whole of every item
  // The join's launch overlaps the attention.
  const int shares = grid * kWarps;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.joint_by_item ? items * 8 * NT
                                              : (shares + kJoinWarps - 1) / kJoinWarps));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = a.joint_by_item ? cudaLaunchKernelEx(&cfg, q4_join<T, D, NT, true>, a, shares)
                      : cudaLaunchKernelEx(&cfg, q4_join<T, D, NT, false>, a, shares);
  return e == cudaSuccess ? KVX_OK : cuda_fail("q4_join", e);
}

template <typename T>
int launch_attention(const AttnArgs& a, int64_t head_dim, int rows, int grid, int64_t items,
                     double bound, int device, cudaStream_t s) {
  if (head_dim == 64) {
    if (rows == 8) return launch_attention<T, 64, 1>(a, grid, items, bound, device, s);
    if (rows == 16) return launch_attention<T, 64, 2>(a, grid, items, bound, device, s);
    return launch_attention<T, 64, 4>(a, grid, items, bound, device, s);
  }
  if (head_dim == 128) {
    if (rows == 8) return launch_attention<T, 128, 1>(a, grid, items, bound, device, s);
    if (rows == 16) return launch_attention<T, 128, 2>(a, grid, items, bound, device, s);
    return launch_attention<T, 128, 4>(a, grid, items, bound, device, s);
  }
  if (rows == 8) return launch_attention<T, 256, 1>(a, grid, items, bound, device, s);
  return launch_attention<T, 256, 2>(a, grid, items, bound, device, s);
}

template <typename T, int D>
int launch_extend(const AttnArgs& a, int64_t tiles, int device, cudaStream_t s) {
  constexpr int shared = ExtendShape<D>::kShared;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = cudaSuccess;
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(q4_extend<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
    if (e != cudaSuccess) return cuda_fail("cudaFuncSetAttribute", e);
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  q4_extend<T, D><<<unsigned(tiles * a.cache.kv_heads), kExtendThreads, shared, s>>>(a, int(tiles));
  e = cudaGetLastError();
  return e == cudaSuccess ? KVX_OK : cuda_fail("q4_extend", e);
}

template <typename T>
int launch_extend(const AttnArgs& a, int64_t head_dim, int64_t tiles, int device, cudaStream_t s) {
  return head_dim == 64 ? launch_extend<T, 64>(a, tiles, device, s)
                        : launch_extend<T, 128>(a, tiles, device, s);
}

}  // namespace

// The device status word of this part (kvx_device_status reads all of them).
int q4_device_status(int reset, int* value) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_q4_status, sizeof(int));
  if (e == cudaSuccess && reset && *value) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_q4_status, &zero, sizeof(int));
  }
  return e == cudaSuccess ? KVX_OK : cuda_fail("q4 status", e);
}

}  // namespace q4
}  // namespace kvx

using namespace kvx;
using namespace kvx::q4;

extern "C" {

int kvx_q4_write(const void* key, const void* value, int dtype, int64_t num_tokens,
                 int64_t key_token_stride, int64_t key_head_stride, int64_t value_token_stride,
                 int64_t value_head_stride, const int64_t* slots, void* key_pages,
                 void* value_pages, int64_t page_stride, int64_t num_blocks, int64_t kv_heads,
                 int64_t block_size, int64_t head_dim, void* stream) {
  record_error("");
  RowArgs a{};
  int rc = cache_of(key_pages, value_pages, page_stride, num_blocks, kv_heads, block_size,
                    head_dim, &a.cache);
  if (rc) return rc;
  a.rows[0] = Rows{const_cast<void*>(key), key_token_stride, key_head_stride};
  a.rows[1] = Rows{const_cast<void*>(value), value_token_stride, value_head_stride};
  a.slots = slots;
  return run_rows(true, a, dtype, num_tokens, head_dim, stream);
}

int kvx_q4_read(const void* key_pages, const void* value_pages, int64_t page_stride,
                int64_t num_blocks, int64_t kv_heads, int64_t block_size, int64_t head_dim,
                const int64_t* slots, int64_t num_tokens,
                void* key, void* value, int dtype, int64_t key_token_stride,
                int64_t key_head_stride, int64_t value_token_stride, int64_t value_head_stride,
                void* stream) {
  record_error("");
  RowArgs a{};
  int rc = cache_of(key_pages, value_pages, page_stride, num_blocks, kv_heads, block_size,
                    head_dim, &a.cache);
  if (rc) return rc;
  a.rows[0] = Rows{key, key_token_stride, key_head_stride};
  a.rows[1] = Rows{value, value_token_stride, value_head_stride};
  a.slots = slots;
  return run_rows(false, a, dtype, num_tokens, head_dim, stream);
}

int kvx_q4_attention_workspace(int64_t head_dim, int64_t rows_per_sequence, uint64_t* bytes_out) {
  record_error("");
  if (!bytes_out) return fail(KVX_ERR_INVALID_ARGUMENT, "null bytes_out");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(KVX_ERR_INVALID_ARGUMENT, "head_dim must be 64, 128 or 256");
  int sms = 0, device = 0;
  const int rc = sm_count(&sms, &device);
  if (rc) return rc;
  *bytes_out = workspace_of(tile_rows(rows_per_sequence, head_dim), head_dim, sms);
  return KVX_OK;
}

int kvx_q4_attention(const void* query, int64_t query_token_stride, int64_t query_head_stride,
                     void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse,
                     int dtype, int64_t num_tokens, int64_t num_heads, const void* key_pages,
                     const void* value_pages, int64_t page_stride, int64_t num_blocks,
                     int64_t kv_heads, int64_t block_size, int64_t head_dim,
                     const int32_t* block_tables, int64_t table_stride, int64_t table_width,
                     const int32_t* seq_lens, const int32_t* query_starts, int64_t batch,
                     double scale, int64_t window, int64_t sinks, void* workspace,
                     uint64_t workspace_bytes, void* stream) {
  record_error("");
  AttnArgs a{};
  int rc = cache_of(key_pages, value_pages, page_stride, num_blocks, kv_heads, block_size,
                    head_dim, &a.cache);
  if (rc) return rc;
  if (dtype != kBf16 && dtype != kFp16)
    return fail(KVX_ERR_INVALID_ARGUMENT, "queries must be bf16 or fp16");
  if (num_tokens < 0 || batch < 0 || table_width < 0)
    return fail(KVX_ERR_INVALID_ARGUMENT, "negative count");
  if (num_heads < 1 || num_heads % kv_heads)
    return fail(KVX_ERR_INVALID_ARGUMENT, "query heads must be a multiple of kv_heads");
  if (window < 0 || sinks < 0)
    return fail(KVX_ERR_INVALID_ARGUMENT, "window and sinks must not be negative");
  if (!std::isfinite(scale)) return fail(KVX_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (num_tokens == 0 || batch == 0) return KVX_OK;
  if (!query || !out || !seq_lens || (!block_tables && table_width > 0))
    return fail(KVX_ERR_INVALID_ARGUMENT, "null argument");
  if (!aligned(query, 2) || !aligned(out, 2) || !aligned(workspace, 16) || !aligned(lse, 4) ||
      !aligned(block_tables, 4) || !aligned(seq_lens, 4) || !aligned(query_starts, 4))
    return fail(KVX_ERR_INVALID_ARGUMENT, "an argument is not aligned to its type");
  const int64_t group = num_heads / kv_heads;
  if (!query_starts && num_tokens % batch)
    return fail(KVX_ERR_LENGTH_MISMATCH,
                "without query_starts every sequence has the same number of query tokens");
  constexpr int64_t kMost = 1ll << 30;  // each first, so that no product passes 64 bits
  if (num_tokens >= kMost || group >= kMost || num_tokens * group >= kMost || batch >= kMost ||
      table_width >= kMost || table_width * block_size >= kMost)
    return fail(KVX_ERR_INVALID_ARGUMENT, "request too large for one call");
  const int64_t queries = query_starts ? num_tokens : num_tokens / batch;
  const int rows = tile_rows(queries * group, head_dim);
  int sms = 0, device = 0;
  rc = sm_count(&sms, &device);
  if (rc) return rc;
  if (!workspace || workspace_bytes < workspace_of(rows, head_dim, sms))
    return fail(KVX_ERR_INVALID_ARGUMENT,
                "workspace smaller than kvx_q4_attention_workspace() says");
  a.query = query;
  a.q_token = query_token_stride;
  a.q_head = query_head_stride;
  a.q_vec = aligned(query, 16) && query_token_stride % 8 == 0 && query_head_stride % 8 == 0;
  a.out = out;
  a.o_token = out_token_stride;
  a.o_head = out_head_stride;
  a.o_vec = aligned(out, 8) && out_token_stride % 4 == 0 && out_head_stride % 4 == 0;
  a.o_vec16 = aligned(out, 16) && out_token_stride % 8 == 0 && out_head_stride % 8 == 0;
  a.lse = lse;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.table_width = int(table_width);
  a.lens = seq_lens;
  a.starts = query_starts;
  a.batch = int(batch);
  a.queries = int(queries);
  a.num_tokens = int(num_tokens);
  a.group = int(group);
  const double scale_log2 = std::fabs(scale) * 1.4426950408889634;
  a.scale_log2 = float(std::min(scale_log2, 3.4e38));
  a.scale_part = float(std::frexp(scale_log2, &a.scale_exp));
  a.sign = scale < 0 ? -1.f : 1.f;
  a.window = window == 0 || window > kNoWindow ? kNoWindow : int(window);
  a.sinks = a.window == kNoWindow ? 0 : int(std::min<int64_t>(sinks, kNoWindow));
  a.upp = int(block_size / 16);
  a.upp_shift = -1;
  for (int i = 0; i < 9; ++i)
    if (a.upp == 1 << i) a.upp_shift = i;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Many rows: whole tiles of 128 rows on the tensor cores, where there are enough
  // of them for half the SMs (they do not share a sequence's cache).
  if (queries * group > 32 && head_dim <= 128 &&
      num_tokens * group / kTileRows * kv_heads >= sms / 2) {
    const int64_t most = query_starts
                             ? num_tokens * group / kExtendRows + batch
                             : batch * ((queries * group + kExtendRows - 1) / kExtendRows);
    if (most * kv_heads > INT32_MAX)
      return fail(KVX_ERR_INVALID_ARGUMENT, "request too large for one call");
    return dtype == kBf16 ? launch_extend<__nv_bfloat16>(a, head_dim, most, device, s)
                          : launch_extend<__half>(a, head_dim, most, device, s);
  }
  // CTAs: those that are resident at once, or fewer where even the longest
  // sequences that the tables can hold have too few units for their warps.
  const int64_t tiles = query_starts ? num_tokens * group / rows + batch
                                     : batch * ((queries * group + rows - 1) / rows);
  const int64_t units = std::max<int64_t>(table_width * a.upp, 1);
  const int64_t items = tiles * kv_heads;
  int64_t grid = resident(rows, head_dim, sms);
  const double bound = double(items) * double((units + kPiece - 1) / kPiece);
  if (bound < double(grid * kWarps)) grid = (int64_t(bound) + kWarps - 1) / kWarps;
  const int64_t pieces = 2ll * kWarps * resident(rows, head_dim, sms) * rows;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + pieces * head_dim);
  a.joints = reinterpret_cast<Joint*>(a.part_ml + pieces);
  a.joint_by_item = !query_starts && items <= kJoinByItem;
  return dtype == kBf16
             ? launch_attention<__nv_bfloat16>(a, head_dim, rows, int(grid), items, bound, device, s)
             : launch_attention<__half>(a, head_dim, rows, int(grid), items, bound, device, s);
}

}  // extern "C"
