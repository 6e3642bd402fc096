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
// leaves its maximum, the sum of its exponentials and the first index of the maximum.  That
// sum, of the acceptance, is fp32: where 2^17 tokens weigh 2^-17 each, an exponent is off by
// 3.5 * 2^-24 of 17 (the difference, log2(e) / T, their product), ex2 by 2^-22 and the sums by
// some 30 roundings: 2^-17 of the sum at most.  In fp64 a pass over every row would cost what
// one of the draw's costs over a row of each sequence.
//
// draft_verify_kernel, a cluster per sequence, joins them, finds the row that ends the
// step and draws from it alone, in fp64: the sums run over the whole vocabulary, and where
// its tokens weigh 1e-5 each, an error of 1e-7 in the sum ahead of one moves one draw in a
// hundred to its neighbour.  Each warp sums a range of the row in blocks of 256 tokens and
// keeps the sums of up to 64 parts of it, so that the draw walks one part again.
//
// 64 sequences with four drafts each from a small model, 151936 bf16 logits: 73 us (floor 15),
// 28 of them the first pass, 3.5 TB/s, bound by the latency of CTAs that each load one piece, then
// work on it (2.4 of 4 instructions a clock and SM, DRAM 42% busy); the rest is the draw, two passes
// over a row's weights, some 20 instructions a token, on 128 of 148 SMs with 16 warps each: latency
// again (2.4 of 4, fp64 units 28% busy).  One sequence: 13 us; 200 ragged ones, 32003 fp32
// logits: 55 (floor 16).  Not kept: 768 or 1024 threads a
// drawing CTA, four or eight CTAs an SM in the first pass (within 3%).
#include "common.cuh"
#include "drafts.cuh"

namespace bsb {
namespace {

constexpr float kLog2eF = 1.4426950408889634f;
constexpr int kStatThreads = 256;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBlock = 256;  // tokens a warp weighs at a time
constexpr int kParts = 64;   // of a warp's range, most
constexpr int kKept = 32;    // rows of a sequence whose maximum is kept

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Whether (value a, index i) comes ahead of (b, j) as the maximum: a NaN counts as the
// largest, equal values go to the lowest index.
__device__ __forceinline__ bool ahead(float a, int32_t i, float b, int32_t j) {
  const bool na = a != a, nb = b != b;
  if (na || nb) return na && (!nb || i < j);
  return a > b || (a == b && i < j);
}

// Whether a temperature weighs tokens: from the smallest normal number on (log2(e) / T is then
// finite in fp32).  0 and those below take the largest logit.
__device__ __forceinline__ bool samples(float temperature) {
  return temperature >= 1.17549435e-38f && temperature < INFINITY;
}

// N elements of a row as they lie in memory, in 32-bit words.
template <typename T, int N>
struct Raw {
  static constexpr int PER = 4 / sizeof(T), WORDS = N / PER;
  uint32_t w[WORDS];
  __device__ __forceinline__ float at(int i) const {
    if constexpr (PER == 1) return __uint_as_float(w[i]);
    return __uint_as_float(i % 2 == 0 ? w[i / 2] << 16 : w[i / 2] & 0xffff0000u);
  }
  __device__ __forceinline__ void load(const T* p) {  // on 16 bytes
#pragma unroll
    for (int k = 0; k < WORDS; k += 4) {
      const uint4 v = coherent_load(reinterpret_cast<const uint4*>(p) + k / 4);
      w[k] = v.x;
      w[k + 1] = v.y;
      w[k + 2] = v.z;
      w[k + 3] = v.w;
    }
  }
  // Elements j .. j + N - 1 of a row, `out` where the row does not go or at `skip`.
  __device__ __forceinline__ void load(const T* row, int32_t j, int32_t end, float out,
                                       int32_t skip = -1) {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      float e[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int32_t at = j + k * PER + i;
        e[i] = at >= 0 && at < end && at != skip ? to_float(row[at]) : out;
      }
      if constexpr (PER == 1) {
        w[k] = __float_as_uint(e[0]);
      } else {
        w[k] = (__float_as_uint(e[0]) >> 16) | (__float_as_uint(e[1]) & 0xffff0000u);
      }
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kStatThreads, 6) draft_stats_kernel(const DraftArgs a) {
  constexpr int VE = 16 / sizeof(T);  // elements of a 16-byte load
  constexpr int LOADS = draft_piece<T>() / (kStatThreads * VE);
  __shared__ float s_max[kStatThreads / 32], s_sum[kStatThreads / 32], s_temp;
  __shared__ int32_t s_arg[kStatThreads / 32], s_seq;
  pdl_wait();
  pdl_trigger();
  const int32_t row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_seq = -1;
  // The row's 16-byte units, as memory is aligned: element j is `shift` + j of them.
  const T* logits = static_cast<const T*>(a.logits) + row * a.logits_stride;
  const int32_t shift = static_cast<int32_t>((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(T));
  const int32_t first = piece * draft_piece<T>() - shift + tid * VE;
  Raw<T, VE> v[LOADS];
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    const int32_t j = first + k * kStatThreads * VE;
    if (j >= 0 && j + VE <= a.vocab) {
      v[k].load(logits + j);
    } else {
      v[k].load(logits, j, a.vocab, -INFINITY);
    }
  }
  __syncthreads();
  for (int32_t b = tid; b < a.num_seqs; b += kStatThreads) {
    if (a.cu_rows[b] <= row && row < a.cu_rows[b + 1]) {
      s_seq = b;
      s_temp = a.temperature != nullptr ? a.temperature[b] : a.temperature_all;
    }
  }
  // The maximum (fmaxf passes over NaN, which the sum finds).
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
#pragma unroll
    for (int i = 0; i < VE; i += 2) top = fmaxf(top, fmaxf(v[k].at(i), v[k].at(i + 1)));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_max[warp] = top;
  __syncthreads();
  if (s_seq < 0) {  // a row of no sequence
    if (piece == 0 && tid == 0) a.tokens[row] = -1;
    return;
  }
#pragma unroll
  for (int w = 0; w < kStatThreads / 32; ++w) top = fmaxf(top, s_max[w]);
  // The sum of exponentials where it is wanted, else only whether there is a NaN.
  const bool finite = top > -INFINITY && top < INFINITY, weigh = samples(s_temp) && finite;
  float sum = 0.f;
  if (weigh) {
    const float scale = kLog2eF / s_temp;
    const float2 scale2 = make_float2(scale, scale), minus_top = make_float2(-top, -top);
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
#pragma unroll
      for (int i = 0; i < VE; i += 2) {
        const float2 z =
            __fmul2_rn(__fadd2_rn(make_float2(v[k].at(i), v[k].at(i + 1)), minus_top), scale2);
        sums = __fadd2_rn(sums, make_float2(fast_exp2(z.x), fast_exp2(z.y)));
      }
    }
    sum = sums.x + sums.y;
  } else {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        if (v[k].at(i) != v[k].at(i)) sum = __int_as_float(0x7fffffff);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kStatThreads / 32; ++w) sum += s_sum[w];
  // The first index of the maximum, NaN before all else, where the row may be decided by it.
  const bool has_nan = sum != sum;
  int32_t arg = 0x7fffffff;
  if (!weigh || has_nan) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int32_t j = first + k * kStatThreads * VE + i;
        const float e = v[k].at(i);
        if ((has_nan ? e != e : e == top) && j >= 0 && j < a.vocab) arg = min(arg, j);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) arg = min(arg, __shfl_xor_sync(0xffffffffu, arg, o));
    if (lane == 0) s_arg[warp] = arg;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStatThreads / 32; ++w) arg = min(arg, s_arg[w]);
    if (has_nan) top = __int_as_float(0x7fffffff);
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
  const float4 none = make_float4(-INFINITY, 0.f, __int_as_float(0x7fffffff), 0.f);
  const float4 mine = lane < a.pieces ? __ldcg(rec + lane) : none;  // all there is, for most
  RowStats s{mine.x, 0.f, __float_as_int(mine.z)};
  for (int32_t c = lane + 32; c < a.pieces; c += 32) {
    const float4 r = __ldcg(rec + c);
    if (ahead(r.x, __float_as_int(r.z), s.top, s.arg)) {
      s.top = r.x;
      s.arg = __float_as_int(r.z);
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
    const float scale = kLog2eF / temperature;
    if (mine.y > 0.f) s.sum = mine.y * fast_exp2((mine.x - s.top) * scale);
    for (int32_t c = lane + 32; c < a.pieces; c += 32) {
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

// The double of a float that is 0 or a positive normal number (of 0: 2^-127; infinities and NaN
// become large numbers).  Whole-number instructions: the fp64 units are what bounds the draw.
__device__ __forceinline__ double widen(float v) {
  const uint32_t u = __float_as_uint(v);
  return __hiloint2double(static_cast<int32_t>((u >> 3) + (896u << 20)),
                          static_cast<int32_t>(u << 29));
}

// Weights exp((l - top) / T) of logits of type L: 2^(k / 64) from a table times the series of
// e^(r ln 2 / 64) for the rest, |r| <= 1/2, whose next term is below 2^-44 of it.  The
// constants live in registers (as immediates each takes two moves at every use).
template <typename L>
struct Weigher {
  // Distances and T in units of 2^-66 where T is small: 0, which widen takes for 2^-127, then is
  // below 2^-60 of T, and subnormal differences are normal numbers.
  static constexpr bool kSmallUnits = sizeof(L) == 2;
  const double* table;
  float units;
  double per_t, round, c4, c3, c2, c1;
  __device__ __forceinline__ Weigher(const double* t, float temperature) : table(t) {
    constexpr double kC = 0.010830424696249145;  // ln 2 / 64
    units = kSmallUnits && temperature < 8.6736174e-19f /* 2^-60 */ ? 7.378697629e19f : 1.f;
    per_t = -64.0 * 1.4426950408889634 / (static_cast<double>(temperature) * units);
    round = 6755399441055744.0;  // 1.5 * 2^52: a sum's low bits are the nearest whole number
    c4 = kC * kC * kC * kC / 24.0;
    c3 = kC * kC * kC / 6.0;
    c2 = kC * kC / 2.0;
    c1 = kC;
    asm volatile("" : "+d"(round), "+d"(c4), "+d"(c3), "+d"(c2), "+d"(c1));
  }
  __device__ __forceinline__ double exact_distance(float top, float l) const {
    return (static_cast<double>(top) - static_cast<double>(l)) * units;
  }
  // Of bf16 logits the fp32 difference is exact, but for logits 2^16 times smaller than the
  // largest: off by 2^-24 of that one at most, which moves the weights of the few that there are by
  // less than the sums can show.
  __device__ __forceinline__ double distance(float top, float l) const {
    return kSmallUnits ? widen((top - l) * units) : exact_distance(top, l);
  }
  __device__ __forceinline__ double operator()(double d) const {
    const double t = fma(d, per_t, round);
    const int32_t k = __double2loint(t);
    const double r = fma(d, per_t, round - t);
    const double e = fma(fma(fma(fma(r, c4, c3), r, c2), r, c1), r, 1.0) * table[k & 63];
    return __hiloint2double(__double2hiint(e) + ((k >> 6) << 20), __double2loint(e));
  }
};

template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads, 1) draft_verify_kernel(const DraftArgs a) {
  __shared__ int32_t s_first, s_arg[kKept];
  __shared__ float s_top[kKept];
  __shared__ double s_exp2[64], s_parts[kWarps][kParts], s_warps[kWarps], s_all;
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
  if (tid < 64) s_exp2[tid] = exp2(tid / 64.0);
  const Weigher<T> weight(s_exp2, sampled ? temperature : 1.f);
  // From this distance on the weight is 0 (2^-1000).
  const float most = sampled ? 1000.f * 0.69314718f * temperature : 0.f;
  const T* logits = static_cast<const T*>(a.logits);
  const Q* probs = static_cast<const Q*>(a.draft_probs);
  if (tid == 0) s_first = n - 1;
  __syncthreads();
  // The first draft that is not accepted; and what its row, or the last, ends with.
  for (int32_t i = warp; i < n; i += kWarps) {
    const int32_t r = r0 + i, x = a.draft_tokens[r];
    const bool draft = i < n - 1, known = x >= 0 && x < a.vocab;
    float l = 0.f, q = 1.f, u = 0.f;
    if (draft && known && sampled) {
      l = to_float(logits[r * a.logits_stride + x]);
      if (probs != nullptr) q = to_float(probs[r * a.probs_stride + x]);
      u = a.uniforms[r];
    }
    const RowStats s = join_row(a, r, temperature, lane);
    if (lane == 0 && i < kKept) {
      s_top[i] = s.top;
      s_arg[i] = s.arg;
    }
    if (lane == 0 && draft) {
      bool take = false;
      if (!known) {
        set_status(a.status, kStatusBadIndex);
      } else if (!sampled) {
        take = x == s.arg;
      } else if (s.top > -INFINITY && s.top < INFINITY && s.top - l < most) {
        const double p = weight(weight.exact_distance(s.top, l)) / static_cast<double>(s.sum);
        take = static_cast<double>(u) * static_cast<double>(q) < p;
      }
      if (!take) atomicMin(&s_first, i);
    }
  }
  __syncthreads();
  const int32_t taken = s_first, row = r0 + taken;
  if (taken >= kKept) {
    if (warp == 0) {
      const RowStats s = join_row(a, row, temperature, lane);
      if (lane == 0) {
        s_top[0] = s.top;
        s_arg[0] = s.arg;
      }
    }
    __syncthreads();
  }
  const float top = s_top[taken < kKept ? taken : 0];
  const int32_t arg = s_arg[taken < kKept ? taken : 0];
  if (rank == 0) {
    for (int32_t i = tid; i < n; i += kThreads) {
      if (i != taken) a.tokens[r0 + i] = i < taken ? a.draft_tokens[r0 + i] : -1;
    }
    if (tid == 0) {
      a.accepted[b] = taken;
      if (!(temperature >= 0.f && temperature < INFINITY)) set_status(a.status, kStatusBadValue);
    }
  }
  const bool weighable = top > -INFINITY && top < INFINITY;
  if (!sampled || !weighable) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = arg;
      if (sampled) set_status(a.status, kStatusBadValue);
    }
    return;
  }

  // The draw: this CTA's share of the vocabulary, a range of it to each warp, lanes along it.
  const T* lrow = logits + row * a.logits_stride;
  const bool rejected = taken < n - 1;
  const int32_t x = rejected ? a.draft_tokens[row] : -1;
  const bool certain = rejected && probs == nullptr;
  const Q* qrow = rejected && !certain ? probs + row * a.probs_stride : nullptr;
  // 16-byte loads of 8 tokens a lane: blocks begin where the row's 16-byte units do, `shift`
  // tokens ahead of it, if the draft probabilities' units are the same.
  const int32_t shift = static_cast<int32_t>((reinterpret_cast<uintptr_t>(lrow) & 15u) / sizeof(T));
  const bool wide = qrow == nullptr || ((reinterpret_cast<uintptr_t>(qrow) - shift * sizeof(Q)) & 15u) == 0;
  const int32_t blocks = (a.vocab + shift + kBlock - 1) / kBlock;  // of the row
  const int32_t all_warps = a.ranks * kWarps, me = rank * kWarps + warp;
  const int32_t b0 = static_cast<int32_t>(static_cast<int64_t>(blocks) * me / all_warps);
  const int32_t b1 = static_cast<int32_t>(static_cast<int64_t>(blocks) * (me + 1) / all_warps);
  const int32_t per = (b1 - b0 + kParts - 1) / kParts;  // blocks of a part
  double inv_z = 0.0;
  // A block's logits and draft probabilities, a lane's 8 tokens; their weights.
  struct Block {
    Raw<T, 8> l;
    Raw<Q, 8> q;
  };
  auto fetch = [&](int32_t block, bool rest, Block& b) {
    const int32_t j0 = block * kBlock - shift, j = j0 + lane * 8;
    if (wide && j0 >= 0 && j0 + kBlock <= a.vocab && !(certain && x >= j0 && x < j0 + kBlock)) {
      b.l.load(lrow + j);
      if (rest) b.q.load(qrow + j);
    } else {
      b.l.load(lrow, j, a.vocab, -INFINITY, certain ? x : -1);
      if (rest) b.q.load(qrow, j, a.vocab, 0.f);
    }
  };
  auto weigh = [&](const Block& b, bool rest, double (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float l = b.l.at(i);
      bool keep = top - l < most;
      w[i] = weight(weight.distance(top, l));
      if (rest) {  // where p is above q (of the high word: neither negative nor NaN)
        w[i] = fma(w[i], inv_z, -widen(fabsf(b.q.at(i))));
        keep = keep && static_cast<uint32_t>(__double2hiint(w[i])) < 0x7ff00000u;
      }
      w[i] = __hiloint2double(keep ? __double2hiint(w[i]) : 0, keep ? __double2loint(w[i]) : 0);
    }
  };
  // Sums of the weights of this warp's parts and of its range; then of the ranges ahead of it,
  // of those ahead of the next, and of all (each range ends exactly where the next begins:
  // the sums are formed in the same order).
  auto add_up = [&](bool rest, double& before, double& before_next, double& all) {
    double range = 0.0;
    Block ahead_block;
    if (b0 < b1) fetch(b0, rest, ahead_block);
    for (int32_t p = 0, block = b0; block < b1; ++p) {
      double sum = 0.0;
      for (const int32_t end = min(block + per, b1); block < end; ++block) {
        const Block now = ahead_block;
        if (block + 1 < b1) fetch(block + 1, rest, ahead_block);
        double w[8];
        weigh(now, rest, w);
        sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      range += sum;
      if (lane == 0) s_parts[warp][p] = sum;
    }
    if (lane == 0) s_warps[warp] = range;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int w = 0; w < kWarps; ++w) t += s_warps[w];
      s_all = t;
    }
    if (a.ranks > 1) {
      cluster_sync();
    } else {
      __syncthreads();
    }
    double ctas = 0.0, warps = 0.0;
    all = 0.0;
    for (int32_t k = 0; k < a.ranks; ++k) {
      if (k == rank) ctas = all;
      all += a.ranks > 1 ? cluster_load64(&s_all, k) : s_all;
    }
    for (int w = 0; w < warp; ++w) warps += s_warps[w];
    before = ctas + warps;
    before_next = ctas + (warps + s_warps[warp]);
    if (a.ranks > 1) {
      cluster_sync();  // the sums may be written again
    } else {
      __syncthreads();
    }
  };
  double before, before_next, all;
  bool rest = qrow != nullptr;
  add_up(false, before, before_next, all);
  if (rest) {
    inv_z = 1.0 / all;
    add_up(true, before, before_next, all);
    rest = all > 0.0;
    if (!rest) add_up(false, before, before_next, all);  // nothing is left: p itself
  }
  if (!(all > 0.0)) {  // a certain draft that has all the weight
    if (rank == 0 && tid == 0) a.tokens[row] = x;
    return;
  }
  double target = static_cast<double>(a.uniforms[r1 - 1]) * all;
  if (!(target < all)) target = all * (1.0 - 1.1102230246251565e-16);
  if (target < 0.0) target = 0.0;
  // The warp whose range holds the token: every range ends where the next begins.
  if (!(before <= target && target < before_next)) return;
  // Its part.
  double sums[kParts / 32], incl[kParts / 32], carry = 0.0;
  int32_t part = -1, last = -1;
#pragma unroll
  for (int k = 0; k < kParts / 32; ++k) {
    const int32_t p = 32 * k + lane;
    sums[k] = p * per < b1 - b0 ? s_parts[warp][p] : 0.0;
    incl[k] = sums[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, incl[k], o);
      if (lane >= o) incl[k] += v;
    }
    incl[k] += carry;
    carry = __shfl_sync(0xffffffffu, incl[k], 31);
    const uint32_t some = __ballot_sync(0xffffffffu, sums[k] > 0.0);
    const uint32_t over = __ballot_sync(0xffffffffu, sums[k] > 0.0 && before + incl[k] > target);
    if (part < 0 && over != 0) part = 32 * k + __ffs(over) - 1;
    if (some != 0) last = 32 * k + 31 - __clz(some);
  }
  if (part < 0) part = last;  // (the parts' sums fell short of the range's)
  double ahead_of = before;
#pragma unroll
  for (int k = 0; k < kParts / 32; ++k) {
    const double v = __shfl_sync(0xffffffffu, incl[k] - sums[k], part & 31);
    if (part / 32 == k) ahead_of += v;
  }
  int32_t token = -1;  // the last of any weight, should the part's sums fall short
  for (int32_t block = b0 + part * per, end = min(block + per, b1); block < end; ++block) {
    Block now;
    fetch(block, rest, now);
    double w[8], own = 0.0;
    weigh(now, rest, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) own += w[i];
    double sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    // A lane's tokens: the first past the target, and the last of any weight.
    double run = ahead_of + (sum - own);
    int32_t hit = -1, some = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      run += w[i];
      if (w[i] > 0.0) {
        some = i;
        if (hit < 0 && run > target) hit = i;
      }
    }
    const uint32_t over = __ballot_sync(0xffffffffu, hit >= 0);
    if (over != 0) {
      if (lane == __ffs(over) - 1) a.tokens[row] = block * kBlock - shift + lane * 8 + hit;
      return;
    }
    const uint32_t any = __ballot_sync(0xffffffffu, some >= 0);
    if (any != 0) {
      const int src = 31 - __clz(any);
      token = block * kBlock - shift + src * 8 + __shfl_sync(0xffffffffu, some, src);
    }
    ahead_of += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) a.tokens[row] = token;
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
