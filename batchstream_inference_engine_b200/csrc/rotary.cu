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

template <typename T, typename Tpool, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_append_kernel(const RotaryArgs a) {
  extern __shared__ float2 turn[];  // [rotary_dim / 2] (cos, sin) times amp
  pdl_trigger();
  pdl_wait();
  const int32_t t = blockIdx.x;
  const int32_t half = a.rotary_dim >> 1;
  const int32_t p = a.pos[t];
  const int32_t slot = a.slots[t];
  const bool bad_pos = p < 0, bad_slot = slot >= a.pool_slots;
  if (threadIdx.x == 0) {
    if (bad_pos) set_status(a.status, kStatusBadPosition);
    if (bad_slot) set_status(a.status, kStatusBadSlot);
  }
  if (!bad_pos) {
    for (int32_t i = threadIdx.x; i < half; i += kThreads) {
      const double turns = static_cast<double>(p) * a.freq[i] * kTurnsPerRad;
      double s, c;
      sincospi(2.0 * (turns - rint(turns)), &s, &c);
      turn[i] = make_float2(static_cast<float>(c * a.amp), static_cast<float>(s * a.amp));
    }
  }
  __syncthreads();
  const T* row = static_cast<const T*>(a.qkv) + t * a.qkv_stride;
  const int32_t heads = a.H + 2 * a.Hkv;
  for (int32_t e = threadIdx.x; e < heads * a.D; e += kThreads) {
    const int32_t hh = e / a.D, d = e - hh * a.D;
    const bool is_q = hh < a.H, is_v = hh >= a.H + a.Hkv;
    if (!is_q && (slot < 0 || bad_slot)) continue;
    if (!is_v && bad_pos) continue;
    float v = rot_in<T>(row[e]);
    if (!is_v && d < a.rotary_dim) {
      const int32_t i = INTER ? d >> 1 : (d < half ? d : d - half);
      const bool second = INTER ? (d & 1) != 0 : d >= half;
      const int32_t other = INTER ? (d ^ 1) : (second ? d - half : d + half);
      const float y = rot_in<T>(row[hh * a.D + other]);
      const float2 cs = turn[i];
      v = second ? fmaf(v, cs.x, y * cs.y) : fmaf(v, cs.x, -(y * cs.y));
    }
    if (is_q) {
      static_cast<T*>(a.q_out)[static_cast<int64_t>(t) * a.H * a.D + e] = rot_out<T>(v);
    } else {
      const int32_t kvh = hh - a.H - (is_v ? a.Hkv : 0);
      Tpool* pool = static_cast<Tpool*>(is_v ? a.v_pool : a.k_pool);
      pool[(kvh * a.pool_slots + slot) * a.D + d] = rot_out<Tpool>(v);
    }
  }
}

template <typename T, typename Tpool>
int launch_rotary_t(const RotaryArgs& a, bool interleaved, cudaStream_t stream) {
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
  auto kernel = interleaved ? rotary_append_kernel<T, Tpool, true>
                            : rotary_append_kernel<T, Tpool, false>;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, a));
}

}  // namespace

int launch_rotary_append(const void* qkv, int64_t qkv_stride, bool bf16, const double* freq,
                         int32_t rotary_dim, bool interleaved, double amp, const int32_t* pos,
                         const int32_t* slots, int32_t ntok, int32_t H, int32_t Hkv, int32_t D,
                         void* q_out, void* k_pool, void* v_pool, bool pool_bf16,
                         int64_t pool_slots, uint32_t* status, cudaStream_t stream) {
  const RotaryArgs a{qkv,  qkv_stride, freq, pos,   slots,  ntok,   H,          Hkv,   D,
                     rotary_dim, amp,  q_out, k_pool, v_pool, pool_slots, status};
  if (bf16 && pool_bf16) {
    return launch_rotary_t<__nv_bfloat16, __nv_bfloat16>(a, interleaved, stream);
  }
  if (bf16) return launch_rotary_t<__nv_bfloat16, float>(a, interleaved, stream);
  if (pool_bf16) return launch_rotary_t<float, __nv_bfloat16>(a, interleaved, stream);
  return launch_rotary_t<float, float>(a, interleaved, stream);
}

}  // namespace bsb
