// Verification of drafted tokens against the target model's distribution, from given
// random numbers (speculative sampling: Leviathan et al., "Fast Inference from Transformers
// via Speculative Decoding", 2023).
//
// With p_r = softmax(logits_r / T) the target's distribution at row r of a sequence, x its
// draft and q the distribution that x was drawn from (certain where there is none):
//     x is accepted  if  u_r q(x) < p_r(x),
// and at the first row that is not, or behind the last draft, one more token is drawn, with
// the weights max(p - q, 0) (p without x where x was certain; p itself where nothing is
// left), or p behind the last draft: the first j at which the running sum of the weights
// exceeds u times their sum, u of the sequence's last row.  T = 0 takes the largest logit.
//
// draft_stats_kernel reads every logit once: a CTA holds a piece of a row in registers and
// leaves its maximum, the sum of its exponentials and the first index of the maximum.
// draft_verify_kernel, a cluster per sequence, joins them, finds the row that ends the
// step and draws from it alone, in fp64: the sums run over the whole vocabulary, and where
// its tokens weigh 1e-5 each, an error of 1e-7 in the sum ahead of one moves one draw in a
// hundred to its neighbour.
#include "common.cuh"
#include "drafts.cuh"

namespace bsb {
namespace {

constexpr float kLog2eF = 1.4426950408889634f;
constexpr int kStatThreads = 256;
constexpr int kThreads = 512, kWarps = kThreads / 32;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Whether (value a, index i) comes ahead of (b, j) as the maximum: a NaN counts as the
// largest, equal values go to the lowest index.
__device__ __forceinline__ bool ahead(float a, int32_t i, float b, int32_t j) {
  const bool na = a != a, nb = b != b;
  if (na || nb) return na && (!nb || i < j);
  return a > b || (a == b && i < j);
}

// 1 / T as a factor of base-2 exponents; 0 stands for taking the largest logit.
__device__ __forceinline__ bool samples(float temperature) {
  return temperature > 0.f && temperature < INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kStatThreads) draft_stats_kernel(const DraftArgs a) {
  constexpr int VE = 16 / sizeof(T);  // elements of a 16-byte load
  constexpr int LOADS = kDraftPiece / (kStatThreads * VE);
  __shared__ float s_max[kStatThreads / 32], s_sum[kStatThreads / 32], s_temp;
  __shared__ int32_t s_arg[kStatThreads / 32], s_seq;
  pdl_wait();
  pdl_trigger();
  const int32_t row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_seq = -1;
  __syncthreads();
  // The row's 16-byte pieces, as memory is aligned: element j is `shift` + j of them.
  const T* logits = static_cast<const T*>(a.logits) + row * a.logits_stride;
  const int32_t shift = static_cast<int32_t>((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(T));
  const int32_t first = piece * kDraftPiece - shift;
  float v[LOADS][VE];
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    const int32_t j = first + (k * kStatThreads + tid) * VE;
    if (j >= 0 && j + VE <= a.vocab) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(logits + j));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < VE; ++i) v[k][i] = to_float(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        v[k][i] = j + i >= 0 && j + i < a.vocab ? to_float(logits[j + i]) : -INFINITY;
      }
    }
  }
  for (int32_t b = tid; b < a.num_seqs; b += kStatThreads) {
    if (a.cu_rows[b] <= row && row < a.cu_rows[b + 1]) {
      s_seq = b;
      s_temp = a.temperature != nullptr ? a.temperature[b] : a.temperature_all;
    }
  }
  // The first maximum.
  float top = -INFINITY;
  int32_t arg = 0x7fffffff;
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const int32_t j = first + (k * kStatThreads + tid) * VE + i;
      if (j >= 0 && j < a.vocab && ahead(v[k][i], j, top, arg)) {
        top = v[k][i];
        arg = j;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t2 = __shfl_xor_sync(0xffffffffu, top, o);
    const int32_t a2 = __shfl_xor_sync(0xffffffffu, arg, o);
    if (ahead(t2, a2, top, arg)) {
      top = t2;
      arg = a2;
    }
  }
  if (lane == 0) {
    s_max[warp] = top;
    s_arg[warp] = arg;
  }
  __syncthreads();
  if (s_seq < 0) {  // a row of no sequence
    if (piece == 0 && tid == 0) a.tokens[row] = -1;
    return;
  }
#pragma unroll
  for (int w = 0; w < kStatThreads / 32; ++w) {
    if (ahead(s_max[w], s_arg[w], top, arg)) {
      top = s_max[w];
      arg = s_arg[w];
    }
  }
  float sum = 0.f;
  if (samples(s_temp) && top > -INFINITY && top < INFINITY) {
    const float scale = fminf(kLog2eF / s_temp, 3e38f);
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
#pragma unroll
      for (int i = 0; i < VE; ++i) sum += fast_exp2((v[k][i] - top) * scale);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kStatThreads / 32; ++w) sum += s_sum[w];
  }
  if (tid == 0) {
    a.records[static_cast<int64_t>(row) * a.pieces + piece] =
        make_float4(top, sum, __int_as_float(arg), 0.f);
  }
}

// A row's statistics from its pieces': the lanes of a warp take them in turn.
struct RowStats {
  float top, sum;  // largest logit; sum of exp((l - top) / T)
  int32_t arg;
};

__device__ __forceinline__ RowStats join_row(const DraftArgs& a, int32_t row, float temperature,
                                             int lane) {
  const float4* rec = a.records + static_cast<int64_t>(row) * a.pieces;
  RowStats s{-INFINITY, 0.f, 0x7fffffff};
  for (int32_t c = lane; c < a.pieces; c += 32) {
    const float4 r = __ldcg(rec + c);
    const int32_t arg = __float_as_int(r.z);
    if (ahead(r.x, arg, s.top, s.arg)) {
      s.top = r.x;
      s.arg = arg;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t2 = __shfl_xor_sync(0xffffffffu, s.top, o);
    const int32_t a2 = __shfl_xor_sync(0xffffffffu, s.arg, o);
    if (ahead(t2, a2, s.top, s.arg)) {
      s.top = t2;
      s.arg = a2;
    }
  }
  if (samples(temperature) && s.top > -INFINITY && s.top < INFINITY) {
    const float scale = fminf(kLog2eF / temperature, 3e38f);
    for (int32_t c = lane; c < a.pieces; c += 32) {
      const float4 r = __ldcg(rec + c);
      if (r.y > 0.f) s.sum += r.y * fast_exp2((r.x - s.top) * scale);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, o);
  }
  return s;
}

__device__ __forceinline__ double cluster_load64(const double* p, uint32_t rank) {
  uint32_t addr;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

// Inclusive sums of the CTA's threads, in thread order.  All threads call it.
__device__ __forceinline__ double block_scan(double v, double (&totals)[kWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  __syncthreads();  // the last use of totals
  if (lane == 31) totals[warp] = v;
  __syncthreads();
  double before = 0.0;
  for (int w = 0; w < warp; ++w) before += totals[w];
  return before + v;
}

template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads) draft_verify_kernel(const DraftArgs a) {
  __shared__ int32_t s_first, s_arg;
  __shared__ float s_top;
  __shared__ double s_totals[kWarps], s_incl[kThreads], s_part;
  pdl_wait();
  const int32_t b = blockIdx.x / a.ranks, rank = blockIdx.x % a.ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t r0 = a.cu_rows[b], r1 = a.cu_rows[b + 1];
  if (r0 < 0 || r1 < r0 || r1 > a.num_rows) {
    if (rank == 0 && tid == 0) {
      set_status(a.status, kStatusBadLength);
      a.accepted[b] = 0;
    }
    return;
  }
  const int32_t n = r1 - r0;
  if (n == 0) {  // padding
    if (rank == 0 && tid == 0) a.accepted[b] = 0;
    return;
  }
  const float temperature = a.temperature != nullptr ? a.temperature[b] : a.temperature_all;
  const bool sampled = samples(temperature);
  const double inv_t = sampled ? 1.0 / static_cast<double>(temperature) : 0.0;
  const T* logits = static_cast<const T*>(a.logits);
  const Q* probs = static_cast<const Q*>(a.draft_probs);
  if (tid == 0) s_first = n - 1;
  __syncthreads();
  // The first draft that is not accepted.
  for (int32_t i = warp; i < n - 1; i += kWarps) {
    const int32_t r = r0 + i, x = a.draft_tokens[r];
    const RowStats s = join_row(a, r, temperature, lane);
    if (lane == 0) {
      bool take = false;
      if (x < 0 || x >= a.vocab) {
        set_status(a.status, kStatusBadIndex);
      } else if (!sampled) {
        take = x == s.arg;
      } else if (s.top > -INFINITY && s.top < INFINITY) {
        const double l = static_cast<double>(to_float(logits[r * a.logits_stride + x]));
        const double p = exp((l - static_cast<double>(s.top)) * inv_t) / static_cast<double>(s.sum);
        const double q =
            probs != nullptr ? static_cast<double>(to_float(probs[r * a.probs_stride + x])) : 1.0;
        take = static_cast<double>(a.uniforms[r]) * q < p;
      }
      if (!take) atomicMin(&s_first, i);
    }
  }
  __syncthreads();
  const int32_t taken = s_first, row = r0 + taken;
  if (warp == 0) {
    const RowStats s = join_row(a, row, temperature, lane);
    if (lane == 0) {
      s_top = s.top;
      s_arg = s.arg;
    }
  }
  if (rank == 0) {
    for (int32_t i = tid; i < n; i += kThreads) {
      if (i != taken) a.tokens[r0 + i] = i < taken ? a.draft_tokens[r0 + i] : -1;
    }
    if (tid == 0) {
      a.accepted[b] = taken;
      if (!sampled && temperature != 0.f) set_status(a.status, kStatusBadValue);
    }
  }
  __syncthreads();
  const float top = s_top;
  const bool weighable = top > -INFINITY && top < INFINITY;
  if (!sampled || !weighable) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = s_arg;
      if (sampled) set_status(a.status, kStatusBadValue);
    }
    return;
  }

  // The draw: this CTA's share of the vocabulary, a run of it to each thread.
  const T* lrow = logits + row * a.logits_stride;
  const bool rejected = taken < n - 1;
  const int32_t x = rejected ? a.draft_tokens[row] : -1;
  const bool certain = rejected && probs == nullptr;
  const Q* qrow = rejected && !certain ? probs + row * a.probs_stride : nullptr;
  const int32_t share = (a.vocab + a.ranks - 1) / a.ranks, run = (share + kThreads - 1) / kThreads;
  const int32_t end = min(a.vocab, (rank + 1) * share);
  const int32_t j0 = min(end, rank * share + tid * run), j1 = min(end, j0 + run);
  const double top64 = static_cast<double>(top);
  auto weight = [&](int32_t j) -> double {  // of p, not normalised
    const float l = to_float(lrow[j]);
    return l == -INFINITY || (certain && j == x) ? 0.0 : exp((static_cast<double>(l) - top64) * inv_t);
  };
  double inv_z = 0.0;
  auto rest = [&](int32_t j) -> double {  // of p - q
    const double d = weight(j) * inv_z - static_cast<double>(to_float(qrow[j]));
    return d > 0.0 ? d : 0.0;
  };
  // Sums of the CTAs ahead and of all, from this CTA's inclusive sums.
  auto join = [&](double mine, double& before, double& all) {
    const double incl = block_scan(mine, s_totals);
    s_incl[tid] = incl;
    if (tid == kThreads - 1) s_part = incl;
    if (a.ranks > 1) {
      cluster_sync();
    } else {
      __syncthreads();
    }
    before = all = 0.0;
    for (int32_t k = 0; k < a.ranks; ++k) {
      if (k == rank) before = all;
      all += a.ranks > 1 ? cluster_load64(&s_part, k) : s_part;
    }
    if (a.ranks > 1) cluster_sync();  // s_part may be written again
  };
  double sum = 0.0, before, all;
  for (int32_t j = j0; j < j1; ++j) sum += weight(j);
  join(sum, before, all);
  bool use_rest = false;
  if (qrow != nullptr) {
    inv_z = 1.0 / all;
    const double p_sum = sum, p_before = before, p_all = all;
    sum = 0.0;
    for (int32_t j = j0; j < j1; ++j) sum += rest(j);
    join(sum, before, all);
    use_rest = all > 0.0;
    if (!use_rest) {  // nothing is left: p itself
      before = p_before;
      all = p_all;
      const double incl = block_scan(p_sum, s_totals);
      s_incl[tid] = incl;
      __syncthreads();
    }
  }
  if (!(all > 0.0)) {  // a certain draft that has all the weight
    if (rank == 0 && tid == 0) a.tokens[row] = x;
    return;
  }
  double target = static_cast<double>(a.uniforms[r1 - 1]) * all;
  if (!(target < all)) target = all * (1.0 - 1.1102230246251565e-16);
  if (target < 0.0) target = 0.0;
  // The thread whose run holds the token; its warp walks the run.
  const double ahead_of = before + (tid > 0 ? s_incl[tid - 1] : 0.0);
  const bool holds = ahead_of <= target && target < before + s_incl[tid];
  const uint32_t who = __ballot_sync(0xffffffffu, holds);
  if (who == 0) return;
  const int src = __ffs(who) - 1;
  const int32_t k0 = __shfl_sync(0xffffffffu, j0, src), k1 = __shfl_sync(0xffffffffu, j1, src);
  double base = __shfl_sync(0xffffffffu, ahead_of, src);
  int32_t last = -1;  // last token of any weight, should the run's sums fall short
  for (int32_t k = k0; k < k1; k += 32) {
    const int32_t j = k + lane;
    const double own = j < k1 ? (use_rest ? rest(j) : weight(j)) : 0.0;
    double incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, own > 0.0 && base + incl > target);
    if (over != 0) {
      last = k + __ffs(over) - 1;
      break;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, own > 0.0);
    if (some != 0) last = k + 31 - __clz(some);
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) a.tokens[row] = last;
}

template <typename T, typename Q>
int launch(const DraftArgs& a, cudaStream_t stream) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.num_rows) * static_cast<unsigned>(a.pieces));
  cfg.blockDim = dim3(kStatThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaSuccess;
  if (a.num_rows > 0) e = cudaLaunchKernelEx(&cfg, draft_stats_kernel<T>, a);
  if (e != cudaSuccess || a.num_seqs == 0) return static_cast<int>(e);
  cfg.gridDim = dim3(static_cast<unsigned>(a.num_seqs) * static_cast<unsigned>(a.ranks));
  cfg.blockDim = dim3(kThreads);
  if (a.ranks > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return static_cast<int>(cudaLaunchKernelEx(&cfg, draft_verify_kernel<T, Q>, a));
}

}  // namespace

int launch_verify_drafts(const DraftArgs& a, bool bf16, bool probs_bf16, cudaStream_t stream) {
  if (bf16) {
    return probs_bf16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, stream)
                      : launch<__nv_bfloat16, float>(a, stream);
  }
  return probs_bf16 ? launch<float, __nv_bfloat16>(a, stream) : launch<float, float>(a, stream);
}

}  // namespace bsb
