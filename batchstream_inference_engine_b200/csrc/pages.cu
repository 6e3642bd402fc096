// Block copies of the paged cache: block src[i] of every layer and kv head, K and
// V, to block dst[i], all pairs in one launch (forks copy a parent's last partial
// block, compaction moves blocks to lower ids).
//
// The pairs happen at once: a destination named by two pairs, or read by another
// pair, would make the result depend on their order, so such a pair is skipped and
// reported.  Every CTA looks its own destination up in the pair list (n entries
// from L2, against the 2 * layers * kv heads blocks it copies).
#include "common.cuh"

namespace bsb {
namespace {

constexpr int kThreads = 256;

struct CopyArgs {
  uint8_t* k_pool;  // [layers * kv heads, num_blocks] blocks of block_bytes
  uint8_t* v_pool;
  const int32_t* src;
  const int32_t* dst;
  int32_t n, num_blocks;
  int64_t rows;  // layers * kv heads
  int64_t block_bytes;
  int32_t slices;  // CTAs per pair
  uint32_t* status;
};

template <typename V>
__global__ void __launch_bounds__(kThreads) copy_blocks_kernel(const CopyArgs a) {
  pdl_trigger();
  pdl_wait();
  const int32_t i = static_cast<int32_t>(blockIdx.x / a.slices);
  const int32_t slice = static_cast<int32_t>(blockIdx.x % a.slices);
  const int32_t s = a.src[i], d = a.dst[i];
  if (s < 0 || d < 0 || s == d) return;  // padding, or nothing to do
  if (s >= a.num_blocks || d >= a.num_blocks) {
    if (threadIdx.x == 0) set_status(a.status, kStatusBadBlock);
    return;
  }
  int clash = 0;
  for (int32_t j = threadIdx.x; j < a.n; j += kThreads) {
    const int32_t sj = a.src[j], dj = a.dst[j];
    // Pairs that pad (a negative end) claim nothing; a pair j onto itself reads.
    if (j != i && sj >= 0 && dj >= 0 && (dj == d || sj == d)) clash = 1;
  }
  if (__syncthreads_or(clash)) {
    if (threadIdx.x == 0) set_status(a.status, kStatusBadCopy);
    return;
  }
  const int64_t vecs = a.block_bytes / static_cast<int64_t>(sizeof(V));
  for (int64_t row = slice; row < 2 * a.rows; row += a.slices) {
    uint8_t* pool = row < a.rows ? a.k_pool : a.v_pool;
    const int64_t base = (row < a.rows ? row : row - a.rows) * a.num_blocks;
    const V* from = reinterpret_cast<const V*>(pool + (base + s) * a.block_bytes);
    V* to = reinterpret_cast<V*>(pool + (base + d) * a.block_bytes);
    for (int64_t x = threadIdx.x; x < vecs; x += kThreads) to[x] = from[x];
  }
}

}  // namespace

int launch_copy_blocks(void* k_pool, void* v_pool, const int32_t* src, const int32_t* dst,
                       int32_t n, int32_t num_blocks, int64_t rows, int64_t block_bytes, bool vec,
                       int sms, uint32_t* status, cudaStream_t stream) {
  // About eight CTAs per SM over all pairs, at most one per (K or V, layer, head).
  int64_t slices = (static_cast<int64_t>(sms) * 8 + n - 1) / n;
  if (slices > 2 * rows) slices = 2 * rows;
  if (slices * n > 0x7fffffff) return static_cast<int>(cudaErrorInvalidConfiguration);
  const CopyArgs a{static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), src, dst, n,
                   num_blocks, rows, block_bytes, static_cast<int32_t>(slices), status};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(slices * n));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = vec ? copy_blocks_kernel<uint4> : copy_blocks_kernel<uint16_t>;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, a));
}

}  // namespace bsb
