// Rotary embedding of q and k with the K/V append, for every rotary form the
// table-driven rope_append does not cover: half or interleaved pairs, part of the
// head, and frequencies scaled for long contexts.
//
// Pair i of the first rotary_dim dims of a head, at position p, turns by the angle
// p * freq[i]:
//     x' = amp * (x cos - y sin),   y' = amp * (y cos + x sin)
// with (x, y) = dims (i, i + rotary_dim / 2), or (2i, 2i + 1) when interleaved.
// The other dims of q and k, and v, are copied.  The products stay in fp32 and
// are rounded once, to the output's type.
//
// The angle needs 64 bits: at position 10^6 the fp32 product of position and
// frequency is off by up to 0.06 rad.  So the turn count p * freq / 2 pi is
// computed, and its whole turns dropped, in fp64; what is left is below half a
// turn.  One CTA per token computes the rotary_dim / 2 pairs of cos and sin once,
// in shared memory, for all its heads.
//
// Bound by memory, and for few tokens by the launch: 4096 tokens of 28 + 2 * 4 heads of
// 128 (75.5 MB read and written, 64 rotary dims) take 13.1 us with the rows in L2 and
// 16.9 without, one token 2.3 us in a graph.  All 64-bit functions instead of fp32 ones
// for bf16 outputs, one element a thread: 51 us.  Loading four units a thread before
// storing any (16.8 us, where one takes 12.4) or the row ahead of the positions (13.0) was
// slower with the rows in L2: the CTAs of an SM hide each other's latency already.
#include "common.cuh"

namespace bsb {
namespace {

constexpr int kThreads = 128;
constexpr double kTurnsPerRad = 0.15915494309189533577;  // 1 / (2 pi)

template <typename T>
__device__ __forceinline__ float rot_in(T v);
template <>
__device__ __forceinline__ float rot_in<float>(float v) { return v; }
template <>
__device__ __forceinline__ float rot_in<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T rot_out(float v);
template <>
__device__ __forceinline__ float rot_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 rot_out<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

struct RotaryArgs {
  const void* qkv;  // rows [q heads | k heads | v heads] of D
  int64_t qkv_stride;
  const double* freq;  // [rotary_dim / 2]
  const int32_t* pos;
  const int32_t* slots;
  int32_t ntok, H, Hkv, D, rotary_dim;
  double amp;
  void* q_out;  // [T, H, D]
  void* k_pool;
  void* v_pool;
  int64_t pool_slots;
  uint32_t* status;
};

// Cos and sin of 2 pi turns for an fp64 turn count, |turns| <= 1/2.  fp32 outputs
// take the fp64 functions (rounding the angle to fp32 alone would cost them 1.6
// half steps); for bf16 rows, 2^16 times coarser, the fp32 ones do (off by 2^-22 at most;
// their k in a fp32 pool too: its digits beyond 2^-8 are not the model's).
__device__ __forceinline__ float2 cos_sin(double turns, double amp, float) {
  double s, c;
  sincospi(2.0 * turns, &s, &c);
  return make_float2(static_cast<float>(c * amp), static_cast<float>(s * amp));
}
__device__ __forceinline__ float2 cos_sin(double turns, double amp, __nv_bfloat16) {
  float s, c;
  sincospif(static_cast<float>(2.0 * turns), &s, &c);
  return make_float2(c * static_cast<float>(amp), s * static_cast<float>(amp));
}

// A token's position and slot, and its cos / sin pairs in shared memory.
struct Token {
  int32_t slot;
  bool rotate, append;  // q and k are rotated; k and v have a slot
};

template <typename T>
__device__ __forceinline__ Token begin_token(const RotaryArgs& a, int32_t t, float2* turn) {
  const int32_t p = a.pos[t];
  Token tok;
  tok.slot = a.slots[t];
  const bool bad_slot = tok.slot >= a.pool_slots;
  tok.rotate = p >= 0;
  tok.append = tok.slot >= 0 && !bad_slot;
  if (threadIdx.x == 0) {
    if (p < 0) set_status(a.status, kStatusBadPosition);
    if (bad_slot) set_status(a.status, kStatusBadSlot);
  }
  if (tok.rotate) {
    for (int32_t i = threadIdx.x; i < (a.rotary_dim >> 1); i += kThreads) {
      const double turns = static_cast<double>(p) * a.freq[i] * kTurnsPerRad;
      turn[i] = cos_sin(turns - rint(turns), a.amp, T());
    }
  }
  __syncthreads();
  return tok;
}

// One pair: (x, y) turned by the angle of cs.
__device__ __forceinline__ void turn_pair(float& x, float& y, float2 cs) {
  const float u = fmaf(x, cs.x, -(y * cs.y));
  y = fmaf(y, cs.x, x * cs.y);
  x = u;
}

// 16-byte rows: a thread takes 8 dims at a time (both halves' 8 for the half
// layout, so that a pair never leaves its thread).  A token's units are the rotated
// ones of every q and k head, then the copied ones, then v's.
template <typename T, typename Tpool, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_append_vec_kernel(const RotaryArgs a) {
  extern __shared__ float2 turn[];
  pdl_wait();
  pdl_trigger();
  const int32_t t = blockIdx.x;
  const Token tok = begin_token<T>(a, t, turn);
  const T* row = static_cast<const T*>(a.qkv) + t * a.qkv_stride;
  T* q_row = static_cast<T*>(a.q_out) + static_cast<int64_t>(t) * a.H * a.D;
  Tpool* k_row = static_cast<Tpool*>(a.k_pool) + static_cast<int64_t>(tok.slot) * a.D;
  Tpool* v_row = static_cast<Tpool*>(a.v_pool) + static_cast<int64_t>(tok.slot) * a.D;
  const int64_t head_stride = a.pool_slots * a.D;
  const int32_t half = a.rotary_dim >> 1;
  const int32_t turned = INTER ? a.rotary_dim >> 3 : half >> 3;  // units per head
  const int32_t copied = (a.D - a.rotary_dim) >> 3;
  const int32_t n_turned = (a.H + a.Hkv) * turned, n_copied = (a.H + a.Hkv) * copied;
  const int32_t units = n_turned + n_copied + a.Hkv * (a.D >> 3);
  for (int32_t u = threadIdx.x; u < units; u += kThreads) {
    if (u < n_turned) {
      const int32_t hh = u / turned, d = (u - hh * turned) * 8;
      if (!tok.rotate || (hh >= a.H && !tok.append)) continue;
      const T* src = row + hh * a.D + d;
      float x[8], y[8];
      load8(src, x);
      if constexpr (INTER) {
#pragma unroll
        for (int j = 0; j < 4; ++j) turn_pair(x[2 * j], x[2 * j + 1], turn[(d >> 1) + j]);
      } else {
        load8(src + half, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) turn_pair(x[j], y[j], turn[d + j]);
      }
      if (hh < a.H) {
        store8(q_row + hh * a.D + d, x);
        if constexpr (!INTER) store8(q_row + hh * a.D + d + half, y);
      } else {
        Tpool* dst = k_row + (hh - a.H) * head_stride + d;
        store8(dst, x);
        if constexpr (!INTER) store8(dst + half, y);
      }
    } else {
      const bool is_v = u >= n_turned + n_copied;
      const int32_t e = is_v ? u - n_turned - n_copied : u - n_turned;
      const int32_t per = is_v ? a.D >> 3 : copied;
      const int32_t i = e / per;
      const int32_t d = (e - i * per) * 8 + (is_v ? 0 : a.rotary_dim);
      const int32_t hh = is_v ? a.H + a.Hkv + i : i;
      if ((!is_v && !tok.rotate) || (hh >= a.H && !tok.append)) continue;
      float x[8];
      load8(row + hh * a.D + d, x);
      if (hh < a.H) {
        store8(q_row + hh * a.D + d, x);
      } else {
        store8((is_v ? v_row : k_row) + (hh - a.H - (is_v ? a.Hkv : 0)) * head_stride + d, x);
      }
    }
  }
}

// Any size and alignment, one element at a time.
template <typename T, typename Tpool, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_append_kernel(const RotaryArgs a) {
  extern __shared__ float2 turn[];
  pdl_wait();
  pdl_trigger();
  const int32_t t = blockIdx.x;
  const int32_t half = a.rotary_dim >> 1;
  const Token tok = begin_token<T>(a, t, turn);
  const T* row = static_cast<const T*>(a.qkv) + t * a.qkv_stride;
  const int32_t heads = a.H + 2 * a.Hkv;
  for (int32_t e = threadIdx.x; e < heads * a.D; e += kThreads) {
    const int32_t hh = e / a.D, d = e - hh * a.D;
    const bool is_q = hh < a.H, is_v = hh >= a.H + a.Hkv;
    if (!is_q && !tok.append) continue;
    if (!is_v && !tok.rotate) continue;
    float v = rot_in<T>(row[e]);
    if (!is_v && d < a.rotary_dim) {
      const int32_t i = INTER ? d >> 1 : (d < half ? d : d - half);
      const bool second = INTER ? (d & 1) != 0 : d >= half;
      const int32_t other = INTER ? (d ^ 1) : (second ? d - half : d + half);
      const float y = rot_in<T>(row[hh * a.D + other]);
      float x0 = second ? y : v, y0 = second ? v : y;
      turn_pair(x0, y0, turn[i]);
      v = second ? y0 : x0;
    }
    if (is_q) {
      static_cast<T*>(a.q_out)[static_cast<int64_t>(t) * a.H * a.D + e] = rot_out<T>(v);
    } else {
      const int32_t kvh = hh - a.H - (is_v ? a.Hkv : 0);
      Tpool* pool = static_cast<Tpool*>(is_v ? a.v_pool : a.k_pool);
      pool[(kvh * a.pool_slots + tok.slot) * a.D + d] = rot_out<Tpool>(v);
    }
  }
}

template <typename T, typename Tpool>
int launch_rotary_t(const RotaryArgs& a, bool interleaved, bool vec, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.ntok);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(float2) * (a.rotary_dim / 2);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = vec ? (interleaved ? rotary_append_vec_kernel<T, Tpool, true>
                                   : rotary_append_vec_kernel<T, Tpool, false>)
                    : (interleaved ? rotary_append_kernel<T, Tpool, true>
                                   : rotary_append_kernel<T, Tpool, false>);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, a));
}

}  // namespace

int launch_rotary_append(const void* qkv, int64_t qkv_stride, bool bf16, const double* freq,
                         int32_t rotary_dim, bool interleaved, double amp, const int32_t* pos,
                         const int32_t* slots, int32_t ntok, int32_t H, int32_t Hkv, int32_t D,
                         void* q_out, void* k_pool, void* v_pool, bool pool_bf16,
                         int64_t pool_slots, bool vec, uint32_t* status, cudaStream_t stream) {
  const RotaryArgs a{qkv,  qkv_stride, freq, pos,   slots,  ntok,   H,          Hkv,   D,
                     rotary_dim, amp,  q_out, k_pool, v_pool, pool_slots, status};
  if (bf16 && pool_bf16) {
    return launch_rotary_t<__nv_bfloat16, __nv_bfloat16>(a, interleaved, vec, stream);
  }
  if (bf16) return launch_rotary_t<__nv_bfloat16, float>(a, interleaved, vec, stream);
  if (pool_bf16) return launch_rotary_t<float, __nv_bfloat16>(a, interleaved, vec, stream);
  return launch_rotary_t<float, float>(a, interleaved, vec, stream);
}

}  // namespace bsb
