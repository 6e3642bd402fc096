// Sliding-window paged attention with sink tokens: arguments and work layout
// shared by its kernels and the C ABI (capi_cache.cu).
//
// The query token at position p of a sequence sees key j when
//     j <= p  and  (j < sinks  or  j > p - window),
// so a tile of consecutive tokens at positions p0 .. p1 reads the keys
//     [0, sink_n)  and  [lo, p1],   lo = max(0, p0 - window + 1),
//                                   sink_n = min(sinks, lo)
// and nothing in between: those blocks may have been freed (their table entries
// are not looked at).  Scores stay in fp32 (the full-context kernels round them
// to bf16 twice because the reference op they replace does; this operator has no
// such counterpart).
#pragma once

#include "common.cuh"

namespace bsb {

struct WindowArgs {
  const void* q;  // [T, H, D], heads of a token contiguous
  int64_t q_stride;  // elements between query tokens
  void* out;
  int64_t o_stride;
  const void* k_pool;  // [Hkv, NB, bs, D] contiguous
  const void* v_pool;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t bt_rows, max_blocks;
  const int32_t* seq_rows;      // optional row of each sequence in block_tables
  const int32_t* context_lens;  // [R] tokens of each sequence, the new ones included
  const int32_t* cu_q;          // [R + 1] query token offsets; null: one token per sequence
  int32_t num_rows, num_tokens, max_query_len;
  int32_t num_heads, num_kv_heads, groups, head_dim, block_size, num_blocks;
  int32_t window, sinks;
  float scale;
  // Query tiles of tile_tokens tokens per sequence (1 without cu_q).
  int32_t tile_tokens, qtiles;
  // A tile's keys are cut into up to `splits` ranges, one CTA each; with more
  // than one, a CTA leaves a record (O unnormalised, then row maxima in base 2
  // and row sums) that a second kernel merges in range order.
  int32_t splits;
  // CUDA cores: the ranges' CTAs are a cluster and join through distributed shared memory
  // instead (no records, no second kernel).
  int32_t clustered;
  float* records;
  int32_t rec_stride;
  // Tensor-core chunks: the (maximum, sum) pairs of every record row start this
  // many floats after the O rows.
  int64_t rec_stride_ml;
  uint32_t* status;
};

// What one query tile reads.
struct WindowTile {
  int32_t tok0;    // first query token (row of q and out)
  int32_t ntok;    // query tokens of the tile
  int32_t pos0;    // position of the first one
  int32_t row;     // block-table row
  int32_t lo;      // first key of the window range
  int32_t sink_n;  // sink keys ahead of it
  int32_t count;   // keys the tile reads: sink_n + pos0 + ntok - lo
};

// Tile `tile` of sequence r.  False when it holds no work: past the chunk's
// end, a padding row (context length 0: nothing read, its output left as it
// was), or an invalid row, reported when `report`.
__device__ __forceinline__ bool window_tile(const WindowArgs& a, int32_t r, int32_t tile,
                                            WindowTile& w, bool report) {
  const int32_t ctx = __ldg(a.context_lens + r);
  int32_t tok0 = r, n = 1;
  if (a.cu_q != nullptr) {
    tok0 = __ldg(a.cu_q + r);
    n = __ldg(a.cu_q + r + 1) - tok0;
  }
  if (ctx == 0 || n == 0) return false;
  w.row = a.seq_rows != nullptr ? __ldg(a.seq_rows + r) : r;
  if (w.row < 0 || w.row >= a.bt_rows) {
    if (report) set_status(a.status, kStatusBadRow);
    return false;
  }
  // max_blocks * block_size fits in int32 (host).
  if (n < 0 || n > a.max_query_len || tok0 < 0 || tok0 > a.num_tokens - n || ctx < n ||
      ctx > a.max_blocks * a.block_size) {
    if (report) set_status(a.status, kStatusBadLength);
    return false;
  }
  const int32_t first = tile * a.tile_tokens;
  if (first >= n) return false;
  w.tok0 = tok0 + first;
  w.ntok = min(a.tile_tokens, n - first);
  w.pos0 = ctx - n + first;
  w.lo = max(0, w.pos0 - a.window + 1);
  w.sink_n = min(a.sinks, w.lo);
  w.count = w.sink_n + w.pos0 + w.ntok - w.lo;
  return true;
}

// Position of the v-th key a tile reads.
__device__ __forceinline__ int32_t window_key(const WindowTile& w, int32_t v) {
  return v < w.sink_n ? v : w.lo + (v - w.sink_n);
}

// Keys of one of `splits` ranges of a tile with `count` keys: a multiple of
// 128, so that the ranges begin where the kernel's key steps do.
__host__ __device__ __forceinline__ int32_t window_range(int32_t count, int32_t splits) {
  return ((count + splits - 1) / splits + 127) / 128 * 128;
}

// Query rows (tokens x heads of one kv head) of a tile of the CUDA-core kernel.
constexpr int kWindowSimtRows = 16;
constexpr int kMaxWindowCluster = 8;  // CTAs of a cluster

// Tensor-core chunks: rows of a query tile, the fewest steps of 64 keys in a range
// and the most ranges.
constexpr int kWindowTileRows = 128;
constexpr int kWindowStepKeys = 64;
// Shorter ranges join more than they share.  us with 2 / 4 / 8 steps a range, and uncut:
// one chunk of 33, d64, window 1024: 11.6 / 12.0 / 14.4 / 16.9; of 300: 11.6 / 10.4 / 10.3 /
// 10.3; four of 64: 14.6 / 13.6 / 15.3 / 17.7; one of 300, d128: 18.1 / 13.2 / 13.3 / 13.4,
// window 8192: 19.6 / 20.8 / 16.5 / 16.5.
constexpr int kMinWindowSteps = 4;
constexpr int kMaxWindowRanges = 8;

int launch_window_prefill(const WindowArgs& a, const CUtensorMap& qmap, const CUtensorMap& kmap,
                          const CUtensorMap& vmap, cudaStream_t stream);
// What runs at once of the CUDA-core kernel: CTAs per SM (cluster 1), or clusters of so many
// CTAs on the device (negative: a CUDA error); wide: more than 8 query rows a tile.
int window_simt_at_once(bool bf16, bool wide, int head_dim, int cluster);
int launch_window_simt(const WindowArgs& a, bool bf16, bool vec, cudaStream_t stream);

}  // namespace bsb
