// The 4-bit cache's append (rotary embedding of q and k, K and V quantised into their
// slots) and its inverse, reading rows back as bf16.
//
// The rotary embedding is rotary.cu's; what is quantised is the rotated key itself, not its
// bf16 rounding, and in fp64: where an element lies between two codes, an error of 2^-22 in
// its angle (the fp32 functions') would flip one code in some 10^5, by a whole step.
//
// A thread takes 8 dims at a time, four of them a group, which finds its extremes with
// shuffles.  One CTA per token.
#include "int4.cuh"

namespace bsb {
namespace {

constexpr int kThreads = 128;
constexpr double kTurnsPerRad = 0.15915494309189533577;  // 1 / (2 pi)
// Groups whose largest element is below kTiny are zeros; at kHuge and above (and where an
// element is not finite) they are zeros and reported.
constexpr float kTiny = 7.8886090522101181e-31f;  // 2^-100
constexpr float kHuge = 1.3292279957849159e36f;   // 2^120

struct AppendArgs {
  const void* qkv;  // rows [q heads | k heads | v heads] of D
  int64_t qkv_stride;
  const double* freq;  // [rotary_dim / 2]
  const int32_t* pos;
  const int32_t* slots;
  int32_t H, Hkv, D, rotary_dim;
  double amp;
  void* q_out;  // [T, H, D]
  uint8_t* k_pool;
  uint8_t* v_pool;
  int32_t num_blocks, block_size;
  uint32_t* status;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Dims d .. d + 7 of a head and their partners' values: x, and y of the same pairs.  The
// sign of the sine's term: -1 for a pair's first dim, 1 for its second, 0 past the rotary
// dims.
template <typename T, bool INTER, bool VEC>
__device__ __forceinline__ void load_pairs(const AppendArgs& a, const T* head, int32_t d,
                                           float (&x)[8], float (&y)[8]) {
  const int32_t half = a.rotary_dim >> 1;
  if constexpr (VEC) {
    load8(head + d, x);
    if constexpr (INTER) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = x[j ^ 1];
    } else if (d < a.rotary_dim) {
      load8(head + (d < half ? d + half : d - half), y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int32_t e = d + j;
      x[j] = to_float(head[e]);
      y[j] = 0.f;
      if (e < a.rotary_dim) y[j] = to_float(head[INTER ? e ^ 1 : e < half ? e + half : e - half]);
    }
  }
}

// Pair index of dim e, and whether it is the pair's second dim.
template <bool INTER>
__device__ __forceinline__ int32_t pair_of(int32_t e, int32_t half, bool& second) {
  second = INTER ? (e & 1) != 0 : e >= half;
  return INTER ? e >> 1 : second ? e - half : e;
}

// 8 elements of a group that this thread and its three neighbours hold: writes the group's
// share of codes and, on its first thread, the scale.  All 32 lanes call it.  Exact borders:
// the fp32 quotient's code is corrected by the remainder x - s n, which is exact.
template <typename V>
__device__ __forceinline__ void quantise(const V (&x)[8], bool mine, int quad, uint32_t* codes,
                                         uint16_t* scale, uint32_t* status) {
  // Largest elements of either side, rounded up to fp32 (which the 4-bit rounding up does not
  // notice); NaN as infinity.
  float hi = 0.f, lo = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float up, down;
    if constexpr (sizeof(V) == 8) {
      up = __double2float_ru(x[j]);
      down = __double2float_ru(-x[j]);
    } else {
      up = x[j];
      down = -x[j];
    }
    if (!(x[j] == x[j])) up = down = INFINITY;
    hi = fmaxf(hi, up);
    lo = fmaxf(lo, down);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fmaxf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  const float top = fmaxf(hi, lo);
  float s = 0.f;
  if (top >= kHuge) {  // (infinity too)
    if (mine && quad == 0) set_status(status, kStatusBadValue);
  } else if (top >= kTiny) {
    s = __uint_as_float((__float_as_uint(top * 0.125f) + 0xfffffu) & 0xfff00000u);
    if (lo < hi) s = -s;
  }
  const float inv = s == 0.f ? 0.f : 1.f / s, limit = fabsf(s) * 0.5f;
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float n = s == 0.f ? 0.f : rintf(static_cast<float>(x[j]) * inv);
    const V rest = s == 0.f ? V(0) : fma(V(-n), V(s), x[j]);
    const V far = rest < V(0) ? -rest : rest;
    const bool odd = (static_cast<int>(n) & 1) != 0;
    if (far > V(limit) || (far == V(limit) && odd)) n += (rest < V(0)) == (s < 0.f) ? 1.f : -1.f;
    const int code = max(0, min(15, static_cast<int>(n) + 8));
    word |= static_cast<uint32_t>(code) << (4 * ((j >> 1) + 4 * (j & 1)));
  }
  if (!mine) return;
  *codes = word;
  if (quad == 0) *scale = static_cast<uint16_t>(__float_as_uint(s) >> 16);
}

template <typename T, bool INTER, bool VEC>
__global__ void __launch_bounds__(kThreads) int4_append_kernel(const AppendArgs a) {
  extern __shared__ double2 turn[];  // cos, sin of the pairs, times amp
  pdl_wait();
  pdl_trigger();
  const int32_t t = blockIdx.x;
  const int32_t slot = a.slots[t], p = a.rotary_dim > 0 ? a.pos[t] : 0;
  const bool bad_slot = slot >= a.num_blocks * a.block_size;  // fits in int32 (host)
  const bool rotate = p >= 0, append = slot >= 0 && !bad_slot;
  if (threadIdx.x == 0) {
    if (p < 0) set_status(a.status, kStatusBadPosition);
    if (bad_slot) set_status(a.status, kStatusBadSlot);
  }
  const int32_t half = a.rotary_dim >> 1;
  if (rotate) {
    for (int32_t i = threadIdx.x; i < half; i += kThreads) {
      const double turns = static_cast<double>(p) * a.freq[i] * kTurnsPerRad;
      double s, c;
      sincospi(2.0 * (turns - rint(turns)), &s, &c);
      turn[i] = make_double2(c * a.amp, s * a.amp);
    }
  }
  __syncthreads();
  const T* row = static_cast<const T*>(a.qkv) + t * a.qkv_stride;
  const int32_t D = a.D, per = D >> 3;  // units of 8 dims a head

  if (rotate) {
    T* q_row = static_cast<T*>(a.q_out) + static_cast<int64_t>(t) * a.H * D;
    for (int32_t u = threadIdx.x; u < a.H * per; u += kThreads) {
      const int32_t h = u / per, d = (u - h * per) * 8;
      float x[8], y[8];
      load_pairs<T, INTER, VEC>(a, row + h * D, d, x, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (d + j < a.rotary_dim) {
          bool second;
          const double2 cs = turn[pair_of<INTER>(d + j, half, second)];
          const float c = static_cast<float>(cs.x), s = static_cast<float>(cs.y);
          y[j] = second ? fmaf(x[j], c, y[j] * s) : fmaf(x[j], c, -(y[j] * s));
        } else {
          y[j] = x[j];
        }
      }
      if constexpr (VEC) {
        store8(q_row + h * D + d, y);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) store(q_row + h * D + d + j, y[j]);
      }
    }
  }
  if (!append) return;

  const int32_t blk = slot / a.block_size, off = slot - blk * a.block_size;
  const int64_t block_bytes = static_cast<int64_t>(a.block_size) * int4_row_bytes(D);
  const int32_t units = 2 * a.Hkv * per;  // k heads, then v heads
  for (int32_t u0 = threadIdx.x & ~31; u0 < units; u0 += kThreads) {
    const int32_t u = min(u0 + static_cast<int32_t>(threadIdx.x & 31), units - 1);
    const int32_t hh = u / per, d = (u - hh * per) * 8;
    const bool is_v = hh >= a.Hkv;
    const bool mine = u0 + static_cast<int32_t>(threadIdx.x & 31) < units && (is_v || rotate);
    const T* head = row + (a.H + hh) * D;
    float x[8], y[8];
    load_pairs<T, INTER, VEC>(a, head, d, x, y);
    uint8_t* block = (is_v ? a.v_pool : a.k_pool) +
                     (static_cast<int64_t>(is_v ? hh - a.Hkv : hh) * a.num_blocks + blk) * block_bytes;
    uint32_t* codes =
        reinterpret_cast<uint32_t*>(block + off * int4_code_bytes(D) + (d >> 1));
    uint16_t* scale = reinterpret_cast<uint16_t*>(block + a.block_size * int4_code_bytes(D) +
                                                  off * int4_scale_bytes(D)) + d / kInt4Group;
    double v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = static_cast<double>(x[j]);
      if (!is_v && rotate && d + j < a.rotary_dim) {
        bool second;
        const double2 cs = turn[pair_of<INTER>(d + j, half, second)];
        const double w = static_cast<double>(y[j]) * cs.y;
        v[j] = second ? fma(v[j], cs.x, w) : fma(v[j], cs.x, -w);
      }
    }
    quantise(v, mine, threadIdx.x & 3, codes, scale, a.status);
  }
}

struct ReadArgs {
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const int32_t* slots;
  int64_t ntok;
  int32_t Hkv, D, num_blocks, block_size;
  __nv_bfloat16* k_out;  // [T, Hkv, D]
  __nv_bfloat16* v_out;
  uint32_t* status;
};

// One thread per 8 dims of a row; rows without a slot are zeros.
__global__ void __launch_bounds__(256) int4_read_kernel(const ReadArgs a) {
  pdl_wait();
  pdl_trigger();
  const int32_t per = a.D >> 3;
  const int64_t n = a.ntok * a.Hkv * per;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t r = i / per;
    const int32_t d = static_cast<int32_t>(i - r * per) * 8;
    const int64_t t = r / a.Hkv;
    const int32_t h = static_cast<int32_t>(r - t * a.Hkv);
    const int32_t slot = a.slots[t];
    const bool bad = slot >= a.num_blocks * a.block_size;
    if (bad && h == 0 && d == 0) set_status(a.status, kStatusBadSlot);
    const int32_t at = slot < 0 || bad ? 0 : slot;
    const int32_t blk = at / a.block_size, off = at - blk * a.block_size;
    const int64_t block = (static_cast<int64_t>(h) * a.num_blocks + blk) * a.block_size *
                          int4_row_bytes(a.D);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const uint8_t* src = (part == 0 ? a.k_pool : a.v_pool) + block;
      uint32_t v[4] = {0u, 0u, 0u, 0u};
      if (slot >= 0 && !bad) {
        const uint32_t w =
            *reinterpret_cast<const uint32_t*>(src + off * int4_code_bytes(a.D) + (d >> 1));
        const uint32_t s = reinterpret_cast<const uint16_t*>(
            src + a.block_size * int4_code_bytes(a.D) + off * int4_scale_bytes(a.D))[d / kInt4Group];
        const uint32_t scale = s | (s << 16);
        int4_values(w, scale, int4_shift(scale), v);
      }
      *reinterpret_cast<uint4*>((part == 0 ? a.k_out : a.v_out) + r * a.D + d) =
          make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

template <typename T>
int launch_append_t(const AppendArgs& a, int32_t ntok, bool interleaved, bool vec,
                    cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ntok);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(double2) * (a.rotary_dim / 2);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = vec ? (interleaved ? int4_append_kernel<T, true, true>
                                   : int4_append_kernel<T, false, true>)
                    : (interleaved ? int4_append_kernel<T, true, false>
                                   : int4_append_kernel<T, false, false>);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, a));
}

}  // namespace

int launch_int4_append(const void* qkv, int64_t qkv_stride, bool bf16, const double* freq,
                       int32_t rotary_dim, bool interleaved, double amp, const int32_t* pos,
                       const int32_t* slots, int32_t ntok, int32_t H, int32_t Hkv, int32_t D,
                       void* q_out, void* k_pool, void* v_pool, int32_t num_blocks,
                       int32_t block_size, bool vec, uint32_t* status, cudaStream_t stream) {
  const AppendArgs a{qkv,   qkv_stride, freq,  pos,   slots,
                     H,     Hkv,        D,     rotary_dim, amp,
                     q_out, static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool),
                     num_blocks, block_size, status};
  return bf16 ? launch_append_t<__nv_bfloat16>(a, ntok, interleaved, vec, stream)
              : launch_append_t<float>(a, ntok, interleaved, vec, stream);
}

int launch_int4_read(const void* k_pool, const void* v_pool, const int32_t* slots, int64_t ntok,
                     int32_t Hkv, int32_t D, int32_t num_blocks, int32_t block_size, void* k_out,
                     void* v_out, int sms, uint32_t* status, cudaStream_t stream) {
  const ReadArgs a{static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), slots,
                   ntok, Hkv, D, num_blocks, block_size, static_cast<__nv_bfloat16*>(k_out),
                   static_cast<__nv_bfloat16*>(v_out), status};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  const int64_t units = ntok * Hkv * (D >> 3), want = (units + 255) / 256;
  cfg.gridDim = dim3(static_cast<unsigned>(want < 8ll * sms ? want : 8ll * sms));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, int4_read_kernel, a));
}

}  // namespace bsb
