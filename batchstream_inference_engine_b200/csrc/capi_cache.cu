// C ABI of the operators that keep a conversation's cache bounded: attention over
// a sliding window with sink tokens, rotary embedding with the K/V append from
// frequencies, and block copies (declared in include/batchstream_b200.h).
//
// Validation, messages and launch rules as in capi.cu: a malformed call is an
// error code plus a message, launches go on the caller's stream, nothing here
// allocates device memory.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/batchstream_b200.h"
#include "decode.cuh"
#include "window.cuh"

namespace bsb {
// capi.cu: messages, launch count, SMs of the current device, tensor maps and
// record sizes of the decode kernels.
void set_last_error(const char* message);
void add_kernel_launches(int n);
int sm_count(int* sms);
int pool_tensor_map(CUtensorMap* map, const void* base, int64_t rows, int64_t head_dim);
int query_tensor_map(CUtensorMap* map, const void* base, int64_t tokens, int64_t token_stride,
                     int64_t heads, int64_t head_dim, int64_t box_heads, int64_t box_tokens);
int32_t decode_record_stride(int64_t groups, int64_t head_dim);
int launch_rotary_append(const void* qkv, int64_t qkv_stride, bool bf16, const double* freq,
                         int32_t rotary_dim, bool interleaved, double amp, const int32_t* pos,
                         const int32_t* slots, int32_t ntok, int32_t H, int32_t Hkv, int32_t D,
                         void* q_out, void* k_pool, void* v_pool, bool pool_bf16,
                         int64_t pool_slots, bool vec, uint32_t* status, cudaStream_t stream);
int launch_copy_blocks(void* k_pool, void* v_pool, const int32_t* src, const int32_t* dst,
                       int32_t n, int32_t num_blocks, int64_t rows, int64_t block_bytes, int align,
                       int sms, uint32_t* status, cudaStream_t stream);
}  // namespace bsb

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  bsb::set_last_error(buf);
  return code;
}

int cuda_fail(int e, const char* what) {
  return fail(BS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(static_cast<cudaError_t>(e)));
}

#define BS_CHECK(cond, ...)                                \
  do {                                                     \
    if (!(cond)) return fail(BS_ERR_INVALID, __VA_ARGS__); \
  } while (0)

constexpr int64_t kInt32Max = 2147483647ll;
constexpr int64_t kMaxHeadDim = 256;
constexpr int64_t kMaxGroups = 16;
// Context lengths, windows and sink counts: sums of two stay within int32.
constexpr int64_t kMaxContext = 1ll << 30;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int dtype_size(int32_t dtype) { return dtype == BS_BF16 ? 2 : 4; }

// a * b, or -1 when it does not fit (both non-negative).
int64_t product(int64_t a, int64_t b) {
  int64_t out = 0;
  return __builtin_mul_overflow(a, b, &out) ? -1 : out;
}

// The sizes of a window attention call.
struct WindowShape {
  int64_t rows, tokens, max_query_len;  // sequences; query tokens
  bool chunks;                          // chunks of tokens (else one token per row)
  int64_t heads, kv_heads, head_dim, block_size, max_blocks, window, sinks;
  int32_t dtype;
};

int check_window_shape(const WindowShape& s) {
  BS_CHECK(s.dtype == BS_BF16 || s.dtype == BS_F32, "dtype must be bfloat16 or float32");
  BS_CHECK(s.rows >= 0 && s.rows <= kInt32Max && s.tokens >= 0 && s.tokens <= kInt32Max,
           "row or token count out of range");
  BS_CHECK(s.max_query_len >= 0 && s.max_query_len <= kInt32Max, "max_query_len out of range");
  BS_CHECK(s.kv_heads > 0 && s.heads > 0 && s.heads % s.kv_heads == 0,
           "heads must equal kv_heads * groups");
  BS_CHECK(s.head_dim > 0 && s.block_size > 0 && s.max_blocks > 0, "sizes must be positive");
  BS_CHECK(s.window >= 1, "window must be at least 1");
  BS_CHECK(s.sinks >= 0, "sinks must be non-negative");
  if (s.head_dim > kMaxHeadDim || s.heads / s.kv_heads > kMaxGroups || s.kv_heads > kInt32Max) {
    return fail(BS_ERR_UNSUPPORTED, "head_dim <= %lld and groups <= %lld are supported",
                static_cast<long long>(kMaxHeadDim), static_cast<long long>(kMaxGroups));
  }
  const int64_t context = product(s.max_blocks, s.block_size);
  if (context < 0 || context > kMaxContext) {
    return fail(BS_ERR_UNSUPPORTED, "a table row covers more than 2^30 tokens");
  }
  return BS_OK;
}

// Key ranges of the CUDA-core kernel: about four CTAs per SM in all, none of
// fewer than 128 keys (one group a warp).
constexpr int64_t kMaxSimtSplits = 64;
constexpr int64_t kMinSimtKeys = 128;

// Whether the ranges of a tile are a cluster whose CTAs join through distributed shared
// memory, instead of leaving records for a second kernel: while they take no more waves.
// A cluster's CTAs start and end together, so fewer of them run at once (410 CTAs in
// clusters of 5, 384 of 8, where 444 fit), and those without keys stay; records cost the
// second kernel.  Measured, clusters / records in us, 444 at once; fp32, 7 heads of 64:
// 384 CTAs (8 a cluster; 1 wave, 1) 16.0 / 24.1, 392 (2, 1) 28.1 / 24.1, 448 (2, 2) 29.5 /
// 34.7, 410 (5; 1, 1) 16.2 / 20.5, 420 (2, 1) 26.7 / 20.5; 296 at once, 16 heads of 64:
// 384 (8; 2, 2) 49.0 / 62.7, 560 (3, 2) 72.0 / 63.2, 390 (3, of which one without keys; 2,
// 1) 49.8 / 33.1; heads of 128: 512 (2, 2) 67.5 / 93.9, 560 (3, 2) 97.3 / 95.5.
bool simt_clusters_win(int64_t items, int64_t busy, int64_t clusters, int64_t resident) {
  return clusters > 0 && (items + clusters - 1) / clusters <= (busy + resident - 1) / resident;
}

// How the CUDA-core kernel runs a call.
struct SimtPlan {
  int64_t tile_tokens, qtiles, items, splits, rec_stride, bytes;
  bool clustered;
};

int plan_simt(const WindowShape& s, SimtPlan* p) {
  int sms = 0;
  if (int rc = bsb::sm_count(&sms)) return rc;
  const int64_t groups = s.heads / s.kv_heads;
  p->tile_tokens = s.chunks ? std::max<int64_t>(1, bsb::kWindowSimtRows / groups) : 1;
  p->qtiles = s.chunks ? (s.max_query_len + p->tile_tokens - 1) / p->tile_tokens : 1;
  p->items = product(product(s.rows, p->qtiles), s.kv_heads);
  if (p->items < 0 || p->items > kInt32Max) {
    return fail(BS_ERR_UNSUPPORTED, "too many query tiles");
  }
  const int64_t keys = std::min(s.max_blocks * s.block_size,
                                std::min(s.window, kMaxContext) + std::min(s.sinks, kMaxContext) +
                                    p->tile_tokens - 1);
  const int64_t want = p->items > 0 ? (4ll * sms + p->items - 1) / p->items : 1;
  p->splits = std::max<int64_t>(
      1, std::min(std::min(want, kMaxSimtSplits), (keys + kMinSimtKeys - 1) / kMinSimtKeys));
  if (p->items * p->splits > kInt32Max) p->splits = 1;
  p->clustered = false;
  if (p->splits > 1 && p->splits <= bsb::kMaxWindowCluster) {
    const bool bf16 = s.dtype == BS_BF16, wide = p->tile_tokens * groups > 8;
    const int head_dim = static_cast<int>(s.head_dim), cluster = static_cast<int>(p->splits);
    const int ctas = bsb::window_simt_at_once(bf16, wide, head_dim, 1);
    const int clusters = bsb::window_simt_at_once(bf16, wide, head_dim, cluster);
    if (ctas <= 0 || clusters < 0) {
      return fail(BS_ERR_CUDA, "occupancy query for window attention failed (%d, %d)", ctas,
                  clusters);
    }
    const int64_t per = bsb::window_range(static_cast<int32_t>(keys), cluster);
    const int64_t busy = p->items * ((keys + per - 1) / per);
    p->clustered = simt_clusters_win(p->items, busy, clusters, static_cast<int64_t>(sms) * ctas);
  }
  const int64_t gm = p->tile_tokens * groups <= 8 ? 8 : bsb::kWindowSimtRows;
  p->rec_stride = gm * s.head_dim + 2 * gm;
  p->bytes = p->splits > 1 && !p->clustered ? p->items * p->splits * p->rec_stride * 4 : 0;
  return BS_OK;
}

// Shapes the tensor-core kernels take (with 16-byte aligned pools and queries, and
// outputs that their stores can address; see mma_pointers).
bool mma_shape(const WindowShape& s) {
  return s.dtype == BS_BF16 && s.block_size % 16 == 0 && (s.head_dim == 64 || s.head_dim == 128);
}

// How the tensor-core decode runs a call: a cluster of segment_ctas CTAs per
// (sequence, kv head); or (segment_ctas 0) persistent CTAs over the batch's units,
// with two partial records and one merge task each.
struct MmaDecodePlan {
  int64_t segment_ctas, grid, rec_stride, tasks_offset, bytes;
};

constexpr int64_t kMaxSegmentCtas = 8;

// Whether clusters of c CTAs take the segments, the longest of `most` units, instead
// of spans over the batch.  Clusters start and end sooner (no scan of the batch, no
// merge launch), spans share ragged work out evenly.  Measured, clusters / spans in us,
// lengths log-uniform up to four windows; d64, 14 + 2 heads: one sequence, window 1024:
// 4.1 / 7.5; 32 (c = 6), 4096 (11 units a warp): 16.0 / 22.0, 16384 (43): 38.8 / 26.0; 64
// (c = 3), 1024 (6): 12.5 / 15.6, 2048 (11): 17.9 / 16.5; 200 (c = 1), 512 (8.5): 14.4 /
// 15.6, 1024 (17): 23.0 / 17.5; d128, 28 + 4 heads, 32 (c = 2), 1024 (8.4): 16.6 / 19.4,
// 2048 (16): 25.4 / 21.2.
bool clusters_win(int64_t c, int64_t most) { return most <= c * 4 * (c >= 4 ? 16 : 9); }

int plan_mma_decode(const WindowShape& s, MmaDecodePlan* p) {
  int sms = 0, dev = 0;
  if (int rc = bsb::sm_count(&sms)) return rc;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  const int64_t groups = s.heads / s.kv_heads;
  // Resident CTAs per SM by device, [head_dim 128][more than 8 heads a group].
  static std::atomic<int> per_sm[64][2][2];
  std::atomic<int>* known = dev < 64 ? &per_sm[dev][s.head_dim == 128][groups > 8] : nullptr;
  int ctas = known != nullptr ? known->load() : 0;
  if (ctas == 0) {
    ctas = bsb::window_decode_mma_ctas_per_sm(static_cast<int>(s.head_dim),
                                              static_cast<int>(groups));
    if (ctas <= 0) return fail(BS_ERR_CUDA, "occupancy query for window decode failed (%d)", ctas);
    if (known != nullptr) known->store(ctas);
  }
  // Units the batch can hold: a window of n tokens touches n / 16 + 1 of them.
  // Fewer than one unit a warp would only add records to merge.
  const int64_t unit = bsb::kWindowUnit;
  const int64_t seen = (std::min(s.window, kMaxContext) + unit - 1) / unit + 1 +
                       (std::min(s.sinks, kMaxContext) + unit - 1) / unit;
  const int64_t most = std::min(seen, s.max_blocks * s.block_size / unit);
  const int64_t resident = static_cast<int64_t>(sms) * ctas, segments = s.rows * s.kv_heads;
  p->segment_ctas = 0;
  if (segments > 0 && segments <= resident) {
    const int64_t c = std::min({kMaxSegmentCtas, std::max<int64_t>(resident / segments, 1),
                                std::max<int64_t>((most + 3) / 4, 1)});
    if (clusters_win(c, most)) {
      p->segment_ctas = c;
      p->grid = segments * c;
      p->rec_stride = p->tasks_offset = p->bytes = 0;
      return BS_OK;
    }
  }
  const int64_t units = s.rows * s.kv_heads * most;
  p->grid = std::max<int64_t>(1, std::min(resident, (units + 3) / 4));
  p->rec_stride = bsb::decode_record_stride(groups, s.head_dim);
  p->tasks_offset = (2 * p->grid * p->rec_stride * 4 + 255) / 256 * 256;
  p->bytes = p->tasks_offset + p->grid * static_cast<int64_t>(sizeof(bsb::MergeTask));
  return BS_OK;
}

// How the tensor-core prefill runs a call: one CTA per 128-row query tile, kv head and
// range of key steps.
struct MmaChunkPlan {
  int64_t tile_tokens, qtiles, items, splits, ml_offset, bytes;
};

constexpr int64_t kMaxRecordBytes = 64ll << 20;

int plan_mma_chunks(const WindowShape& s, MmaChunkPlan* p) {
  int sms = 0;
  if (int rc = bsb::sm_count(&sms)) return rc;
  const int64_t groups = s.heads / s.kv_heads;
  p->tile_tokens = bsb::kWindowTileRows / groups;
  p->qtiles = (s.max_query_len + p->tile_tokens - 1) / p->tile_tokens;
  p->items = product(product(s.rows, p->qtiles), s.kv_heads);
  if (p->items < 0 || p->items > kInt32Max / bsb::kMaxWindowRanges / 8) {
    return fail(BS_ERR_UNSUPPORTED, "too many query tiles");
  }
  // Tiles that can hold tokens (the others of a padded launch exit at once); two CTAs
  // run on an SM, so ranges are cut only as far as one wave of them goes.  Cut as far as
  // two waves / one, us: 4 chunks of 300, d64 (136 tiles), window 1024: 25.5 / 19.1, 4096:
  // 28.1 / 27.1; 8 of 200 (192): 28.4 / 19.0; 4 of 300, d128 (272), 1024: 42.7 / 24.6, 4096:
  // 49.7 / 41.5.
  const int64_t busy = std::max<int64_t>(
      1, std::min(s.rows * p->qtiles,
                  (s.tokens + p->tile_tokens - 1) / p->tile_tokens + s.rows) * s.kv_heads);
  const int64_t keys = std::min(s.max_blocks * s.block_size,
                                std::min(s.window, kMaxContext) + std::min(s.sinks, kMaxContext) +
                                    p->tile_tokens + 32);
  const int64_t most = keys / (bsb::kWindowStepKeys * bsb::kMinWindowSteps);
  const int64_t record = bsb::kWindowTileRows * (s.head_dim + 2) * 4;
  p->splits = std::max<int64_t>(
      1, std::min(std::min<int64_t>(2ll * sms / busy, bsb::kMaxWindowRanges), most));
  while (p->splits > 1 && p->items * p->splits * record > kMaxRecordBytes) --p->splits;
  p->ml_offset = p->items * p->splits * bsb::kWindowTileRows * s.head_dim;
  p->bytes = p->splits > 1 ? p->items * p->splits * record : 0;
  return BS_OK;
}

// Scratch of a call: the largest of the kernels its shape may run on.
int window_workspace(const WindowShape& s, uint64_t* bytes_out) {
  BS_CHECK(bytes_out != nullptr, "bytes_out is null");
  if (int rc = check_window_shape(s)) return rc;
  SimtPlan p;
  if (int rc = plan_simt(s, &p)) return rc;
  int64_t need = p.bytes;
  if (mma_shape(s) && s.chunks) {
    MmaChunkPlan m;
    if (int rc = plan_mma_chunks(s, &m)) return rc;
    need = std::max(need, m.bytes);
  } else if (mma_shape(s)) {
    MmaDecodePlan m;
    if (int rc = plan_mma_decode(s, &m)) return rc;
    need = std::max(need, m.bytes);
  }
  *bytes_out = static_cast<uint64_t>(need);
  return BS_OK;
}

// Everything of a call but its shape.
struct WindowCall {
  const void* query;
  int64_t q_stride;
  const int32_t* cu_q;
  const int32_t* context_lens;
  const int32_t* seq_rows;
  const void* key_pool;
  const void* value_pool;
  const int32_t* block_tables;
  int64_t table_stride, table_rows, num_blocks;
  double scaling;
  void* output;
  int64_t o_stride;
  void* workspace;
  uint64_t workspace_bytes;
  uint32_t* status;
  void* stream;
};

int check_workspace(const WindowCall& c, int64_t need) {
  if (need > 0 && (c.workspace == nullptr || c.workspace_bytes < static_cast<uint64_t>(need))) {
    return fail(BS_ERR_WORKSPACE, "workspace of %llu bytes is smaller than the %lld needed",
                static_cast<unsigned long long>(c.workspace_bytes), static_cast<long long>(need));
  }
  BS_CHECK(aligned16(c.workspace), "workspace must be 16-byte aligned");
  return BS_OK;
}

// Pointers and strides the tensor-core kernels can take: TMA and bulk copies of
// pools and query rows, 16-byte output rows.
bool mma_pointers(const WindowCall& c) {
  return aligned16(c.query) && aligned16(c.key_pool) && aligned16(c.value_pool) &&
         aligned16(c.output) && c.q_stride % 8 == 0 && c.o_stride % 8 == 0;
}

int run_mma_decode(const WindowShape& s, const WindowCall& c) {
  MmaDecodePlan p;
  if (int rc = plan_mma_decode(s, &p)) return rc;
  if (int rc = check_workspace(c, p.bytes)) return rc;
  CUtensorMap kmap, vmap;
  const int64_t rows = s.kv_heads * c.num_blocks * s.block_size;
  if (int rc = bsb::pool_tensor_map(&kmap, c.key_pool, rows, s.head_dim)) return rc;
  if (int rc = bsb::pool_tensor_map(&vmap, c.value_pool, rows, s.head_dim)) return rc;
  bsb::DecodeArgs a{};
  a.q = c.query;
  a.q_stride_seq = c.q_stride;
  a.out = c.output;
  a.o_stride_seq = c.o_stride;
  a.k_pool = c.key_pool;
  a.v_pool = c.value_pool;
  a.block_tables = c.block_tables;
  a.bt_stride = c.table_stride;
  a.bt_rows = static_cast<int32_t>(c.table_rows);
  a.seq_rows = c.seq_rows;
  a.context_lens = c.context_lens;
  a.num_seqs = static_cast<int32_t>(s.rows);
  a.num_heads = static_cast<int32_t>(s.heads);
  a.num_kv_heads = static_cast<int32_t>(s.kv_heads);
  a.groups = static_cast<int32_t>(s.heads / s.kv_heads);
  a.head_dim = static_cast<int32_t>(s.head_dim);
  a.block_size = static_cast<int32_t>(s.block_size);
  a.num_blocks = static_cast<int32_t>(c.num_blocks);
  a.max_blocks = static_cast<int32_t>(s.max_blocks);
  a.scale = static_cast<float>(c.scaling);
  uint8_t* ws = static_cast<uint8_t*>(c.workspace);
  a.partials = reinterpret_cast<float*>(ws);
  a.rec_stride = static_cast<int32_t>(p.rec_stride);
  a.tasks = p.segment_ctas > 0 ? nullptr
                               : reinterpret_cast<bsb::MergeTask*>(ws + p.tasks_offset);
  a.segment_ctas = static_cast<int32_t>(p.segment_ctas);
  a.status = c.status;
  a.window = static_cast<int32_t>(std::min(s.window, kMaxContext));
  a.sinks = static_cast<int32_t>(std::min(s.sinks, kMaxContext));
  a.block_units = static_cast<int32_t>(s.block_size / bsb::kWindowUnit);
  bsb::apply_wait_probe(a);
  const int rc = bsb::launch_window_decode_mma(a, kmap, vmap, static_cast<int>(p.grid),
                                               static_cast<cudaStream_t>(c.stream));
  if (rc != 0) return cuda_fail(rc, "window decode launch");
  bsb::add_kernel_launches(p.segment_ctas > 0 ? 1 : 2);  // the decode and its merge pass
  return BS_OK;
}

int run_mma_chunks(const WindowShape& s, const WindowCall& c, bsb::WindowArgs& a) {
  MmaChunkPlan p;
  if (int rc = plan_mma_chunks(s, &p)) return rc;
  if (int rc = check_workspace(c, p.bytes)) return rc;
  CUtensorMap qmap, kmap, vmap;
  const int64_t rows = s.kv_heads * c.num_blocks * s.block_size;
  const int64_t groups = s.heads / s.kv_heads;
  if (int rc = bsb::query_tensor_map(&qmap, c.query, s.tokens, c.q_stride, s.heads, s.head_dim,
                                     groups, p.tile_tokens)) {
    return rc;
  }
  if (int rc = bsb::pool_tensor_map(&kmap, c.key_pool, rows, s.head_dim)) return rc;
  if (int rc = bsb::pool_tensor_map(&vmap, c.value_pool, rows, s.head_dim)) return rc;
  a.tile_tokens = static_cast<int32_t>(p.tile_tokens);
  a.qtiles = static_cast<int32_t>(p.qtiles);
  a.splits = static_cast<int32_t>(p.splits);
  a.records = static_cast<float*>(c.workspace);
  a.rec_stride_ml = p.ml_offset;
  const int rc = bsb::launch_window_prefill(a, qmap, kmap, vmap,
                                            static_cast<cudaStream_t>(c.stream));
  if (rc != 0) return cuda_fail(rc, "window prefill launch");
  bsb::add_kernel_launches(p.splits > 1 ? 2 : 1);
  return BS_OK;
}

int run_window(const WindowShape& s, const WindowCall& c) {
  if (int rc = check_window_shape(s)) return rc;
  BS_CHECK(s.max_blocks <= c.table_stride, "max_blocks_per_seq must be in [1, table_stride]");
  BS_CHECK(c.table_rows > 0 && c.table_rows <= kInt32Max, "table_rows out of range");
  BS_CHECK(c.num_blocks > 0, "sizes must be positive");
  BS_CHECK(c.q_stride >= s.heads * s.head_dim && c.o_stride >= s.heads * s.head_dim,
           "token strides must cover heads * head_dim");
  const int64_t pool_rows = product(product(s.kv_heads, c.num_blocks), s.block_size);
  if (pool_rows < 0 || pool_rows > kInt32Max) {
    return fail(BS_ERR_UNSUPPORTED, "pool has more than 2^31 rows");
  }
  if (s.rows == 0 || s.tokens == 0) return BS_OK;
  BS_CHECK(!s.chunks || s.max_query_len > 0, "max_query_len must be positive");
  BS_CHECK(c.query && c.key_pool && c.value_pool && c.block_tables && c.context_lens &&
               c.output && (!s.chunks || c.cu_q),
           "null pointer argument");
  const bool mma = mma_shape(s) && mma_pointers(c);
  if (mma && !s.chunks) return run_mma_decode(s, c);
  bsb::WindowArgs a{};
  a.q = c.query;
  a.q_stride = c.q_stride;
  a.out = c.output;
  a.o_stride = c.o_stride;
  a.k_pool = c.key_pool;
  a.v_pool = c.value_pool;
  a.block_tables = c.block_tables;
  a.bt_stride = c.table_stride;
  a.bt_rows = static_cast<int32_t>(c.table_rows);
  a.max_blocks = static_cast<int32_t>(s.max_blocks);
  a.seq_rows = c.seq_rows;
  a.context_lens = c.context_lens;
  a.cu_q = s.chunks ? c.cu_q : nullptr;
  a.num_rows = static_cast<int32_t>(s.rows);
  a.num_tokens = static_cast<int32_t>(s.tokens);
  a.max_query_len = static_cast<int32_t>(s.max_query_len);
  a.num_heads = static_cast<int32_t>(s.heads);
  a.num_kv_heads = static_cast<int32_t>(s.kv_heads);
  a.groups = static_cast<int32_t>(s.heads / s.kv_heads);
  a.head_dim = static_cast<int32_t>(s.head_dim);
  a.block_size = static_cast<int32_t>(s.block_size);
  a.num_blocks = static_cast<int32_t>(c.num_blocks);
  a.window = static_cast<int32_t>(std::min(s.window, kMaxContext));
  a.sinks = static_cast<int32_t>(std::min(s.sinks, kMaxContext));
  a.scale = static_cast<float>(c.scaling);
  a.status = c.status;
  // The tensor-core prefill compares scores before it scales them: it needs a
  // magnitude to scale by.
  if (mma && a.scale != 0.f && std::isfinite(a.scale)) return run_mma_chunks(s, c, a);

  SimtPlan p;
  if (int rc = plan_simt(s, &p)) return rc;
  if (int rc = check_workspace(c, p.bytes)) return rc;
  a.tile_tokens = static_cast<int32_t>(p.tile_tokens);
  a.qtiles = static_cast<int32_t>(p.qtiles);
  a.splits = static_cast<int32_t>(p.splits);
  a.clustered = p.clustered ? 1 : 0;
  a.records = static_cast<float*>(c.workspace);
  a.rec_stride = static_cast<int32_t>(p.rec_stride);
  const bool vec = (s.head_dim * dtype_size(s.dtype)) % 16 == 0 && aligned16(c.key_pool) &&
                   aligned16(c.value_pool);
  const int rc = bsb::launch_window_simt(a, s.dtype == BS_BF16, vec,
                                         static_cast<cudaStream_t>(c.stream));
  if (rc != 0) return cuda_fail(rc, "window attention launch");
  bsb::add_kernel_launches(p.splits > 1 && !p.clustered ? 2 : 1);
  return BS_OK;
}

}  // namespace

extern "C" {

int bs_window_attention_batched_workspace_bytes(int64_t num_seqs, int64_t num_heads,
                                                int64_t num_kv_heads, int64_t head_dim,
                                                int64_t block_size, int64_t max_blocks_per_seq,
                                                int32_t dtype, int64_t window, int64_t sinks,
                                                uint64_t* bytes_out) {
  const WindowShape s{num_seqs, num_seqs,   1,          false,
                      num_heads, num_kv_heads, head_dim, block_size,
                      max_blocks_per_seq, window, sinks, dtype};
  return window_workspace(s, bytes_out);
}

int bs_window_prefill_attention_workspace_bytes(int64_t num_tokens, int64_t num_rows,
                                                int64_t max_query_len, int64_t num_heads,
                                                int64_t num_kv_heads, int64_t head_dim,
                                                int64_t block_size, int64_t max_blocks_per_seq,
                                                int32_t dtype, int64_t window, int64_t sinks,
                                                uint64_t* bytes_out) {
  // (A chunk cannot hold more than all tokens; a negative bound stays to be refused.)
  const WindowShape s{num_rows, num_tokens, std::min(max_query_len, num_tokens), true,
                      num_heads, num_kv_heads, head_dim, block_size,
                      max_blocks_per_seq, window, sinks, dtype};
  return window_workspace(s, bytes_out);
}

int bs_window_attention_batched(const void* query, int64_t query_seq_stride, const void* key_pool,
                                const void* value_pool, const int32_t* block_tables,
                                int64_t table_stride, int64_t table_rows, const int32_t* seq_rows,
                                const int32_t* context_lens, int64_t num_seqs, int64_t num_heads,
                                int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                int64_t num_blocks, int64_t max_blocks_per_seq, int32_t dtype,
                                double scaling, int64_t window, int64_t sinks, void* output,
                                int64_t output_seq_stride, void* workspace,
                                uint64_t workspace_bytes, uint32_t* status, void* stream) {
  const WindowShape s{num_seqs, num_seqs,   1,          false,
                      num_heads, num_kv_heads, head_dim, block_size,
                      max_blocks_per_seq, window, sinks, dtype};
  const WindowCall c{query,        query_seq_stride, nullptr,    context_lens, seq_rows,
                     key_pool,     value_pool,       block_tables, table_stride, table_rows,
                     num_blocks,   scaling,          output,     output_seq_stride, workspace,
                     workspace_bytes, status,        stream};
  return run_window(s, c);
}

int bs_window_prefill_attention(const void* query, int64_t query_token_stride, const int32_t* cu_q,
                                int64_t num_rows, int64_t num_tokens, int64_t max_query_len,
                                const int32_t* context_lens, const int32_t* seq_rows,
                                const void* key_pool, const void* value_pool,
                                const int32_t* block_tables, int64_t table_stride,
                                int64_t table_rows, int64_t max_blocks_per_seq, int64_t num_heads,
                                int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                int64_t num_blocks, int32_t dtype, double scaling, int64_t window,
                                int64_t sinks, void* output, int64_t output_token_stride,
                                void* workspace, uint64_t workspace_bytes, uint32_t* status,
                                void* stream) {
  const WindowShape s{num_rows, num_tokens, std::min(max_query_len, num_tokens), true,
                      num_heads, num_kv_heads, head_dim, block_size,
                      max_blocks_per_seq, window, sinks, dtype};
  const WindowCall c{query,        query_token_stride, cu_q,      context_lens, seq_rows,
                     key_pool,     value_pool,       block_tables, table_stride, table_rows,
                     num_blocks,   scaling,          output,     output_token_stride, workspace,
                     workspace_bytes, status,        stream};
  return run_window(s, c);
}

int bs_rotary_append(const void* qkv, int64_t qkv_row_stride, int32_t dtype,
                     const double* frequencies, int64_t rotary_dim, int32_t interleaved,
                     double amplitude, const int32_t* positions, const int32_t* slot_mapping,
                     int64_t num_tokens, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                     void* query_out, void* key_pool, void* value_pool, int32_t pool_dtype,
                     int64_t num_blocks, int64_t block_size, uint32_t* status, void* stream) {
  BS_CHECK(dtype == BS_BF16 || dtype == BS_F32, "dtype must be bfloat16 or float32");
  BS_CHECK(pool_dtype == BS_BF16 || pool_dtype == BS_F32, "pool dtype must be bf16 or fp32");
  BS_CHECK(num_tokens >= 0 && num_tokens <= kInt32Max, "num_tokens out of range");
  BS_CHECK(num_heads > 0 && num_kv_heads > 0 && head_dim > 0, "sizes must be positive");
  BS_CHECK(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
           "rotary_dim must be even and in [2, head_dim]");
  BS_CHECK(std::isfinite(amplitude), "amplitude must be finite");
  BS_CHECK(num_blocks > 0 && block_size > 0, "sizes must be positive");
  if (head_dim > 1024 || num_heads > 65536 || num_kv_heads > 65536) {
    return fail(BS_ERR_UNSUPPORTED, "head_dim <= 1024 and at most 65536 heads are supported");
  }
  BS_CHECK(qkv_row_stride >= (num_heads + 2 * num_kv_heads) * head_dim,
           "qkv rows must hold q, k and v");
  const int64_t slots = product(num_blocks, block_size);
  if (slots < 0 || slots > kInt32Max) return fail(BS_ERR_UNSUPPORTED, "pool too large");
  if (num_tokens == 0) return BS_OK;
  BS_CHECK(qkv && frequencies && positions && slot_mapping && query_out && key_pool && value_pool,
           "null pointer argument");
  const bool vec = head_dim % 8 == 0 && rotary_dim % (interleaved ? 8 : 16) == 0 &&
                   qkv_row_stride % 8 == 0 && aligned16(qkv) && aligned16(query_out) &&
                   aligned16(key_pool) && aligned16(value_pool);
  const int rc = bsb::launch_rotary_append(
      qkv, qkv_row_stride, dtype == BS_BF16, frequencies, static_cast<int32_t>(rotary_dim),
      interleaved != 0, amplitude, positions, slot_mapping, static_cast<int32_t>(num_tokens),
      static_cast<int32_t>(num_heads), static_cast<int32_t>(num_kv_heads),
      static_cast<int32_t>(head_dim), query_out, key_pool, value_pool, pool_dtype == BS_BF16,
      slots, vec, status, static_cast<cudaStream_t>(stream));
  if (rc != 0) return cuda_fail(rc, "rotary_append launch");
  bsb::add_kernel_launches(1);
  return BS_OK;
}

int bs_copy_blocks(void* key_pool, void* value_pool, int32_t pool_dtype, int64_t num_layers,
                   int64_t num_kv_heads, int64_t num_blocks, int64_t block_size, int64_t head_dim,
                   const int32_t* src, const int32_t* dst, int64_t num_pairs, uint32_t* status,
                   void* stream) {
  BS_CHECK(pool_dtype == BS_BF16 || pool_dtype == BS_F32, "pool dtype must be bf16 or fp32");
  BS_CHECK(num_layers > 0 && num_kv_heads > 0 && num_blocks > 0 && block_size > 0 && head_dim > 0,
           "sizes must be positive");
  BS_CHECK(num_blocks <= kInt32Max, "num_blocks out of range");
  BS_CHECK(num_pairs >= 0 && num_pairs <= kInt32Max, "num_pairs out of range");
  const int64_t rows = product(num_layers, num_kv_heads);
  const int64_t block_bytes = product(product(block_size, head_dim), dtype_size(pool_dtype));
  if (rows < 0 || block_bytes < 0 || product(product(rows, num_blocks), block_bytes) < 0) {
    return fail(BS_ERR_UNSUPPORTED, "pool too large");
  }
  if (num_pairs == 0) return BS_OK;
  BS_CHECK(key_pool && value_pool && src && dst, "null pointer argument");
  int sms = 0;
  if (int rc = bsb::sm_count(&sms)) return rc;
  const uint64_t bits = reinterpret_cast<uintptr_t>(key_pool) |
                        reinterpret_cast<uintptr_t>(value_pool) |
                        static_cast<uint64_t>(block_bytes);
  const int align = bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 2;
  const int rc = bsb::launch_copy_blocks(key_pool, value_pool, src, dst,
                                         static_cast<int32_t>(num_pairs),
                                         static_cast<int32_t>(num_blocks), rows, block_bytes, align,
                                         sms, status, static_cast<cudaStream_t>(stream));
  if (rc != 0) return cuda_fail(rc, "copy_blocks launch");
  bsb::add_kernel_launches(1);
  return BS_OK;
}

}  // extern "C"
