// The 4-bit cache's append (rotary embedding of q and k, K and V quantised into their
// slots) and its inverse, reading rows back as bf16.
//
// The rotary embedding is rotary.cu's; what is quantised is the rotated key itself, not its
// bf16 rounding, and in fp64: where an element lies between two codes, an error of 2^-22 in
// its angle (the fp32 functions') would flip one code in some 10^5, by a whole step.
//
// A thread takes 8 dims at a time, four of them a group, which finds its extremes with
// shuffles.  One CTA per token.
//
// 4096 tokens, 28 + 2 x 4 heads of 128, all turned: 24 us, then a read of all rows (6), 2.9
// TB/s of what the append reads and writes.  What bounds it is latency: the position, the
// slot, the row, the angles' fp64 sine and cosine and the group's extremes follow one
// another (2.0 instructions a clock and SM).  96 or 64
// threads a CTA take the same, 192 2 us more, 288 12.
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

// Cos and sin of a token's pairs, times amp, as fp64 and rounded to fp32.
struct Turns {
  double2* exact;
  float2* rounded;
};

// Dims d .. d + 7 of a head turned by the angles of their pairs: F is double (keys) or float
// (queries).  VEC: the 8 dims lie on 16 bytes and are all a pair's first dims, all its second
// (half layout), or whole pairs, or all past the rotary dims.
template <typename T, bool INTER, bool VEC, typename F, typename F2>
__device__ __forceinline__ void turned(const AppendArgs& a, const T* head, int32_t d,
                                       const F2* turn, F (&out)[8]) {
  const int32_t half = a.rotary_dim >> 1;
  float x[8], y[8];
  if constexpr (VEC) {
    load8(head + d, x);
    if (d >= a.rotary_dim) {
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = static_cast<F>(x[j]);
      return;
    }
    if constexpr (INTER) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const F2 cs = turn[(d + j) >> 1];
        const F u = static_cast<F>(x[j]), v = static_cast<F>(x[j + 1]);
        out[j] = fma(u, cs.x, -(v * cs.y));
        out[j + 1] = fma(v, cs.x, u * cs.y);
      }
    } else {
      const bool second = d >= half;
      load8(head + (second ? d - half : d + half), y);
      const F2* cs = turn + (second ? d - half : d);
      const F sign = second ? F(1) : F(-1);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        out[j] = fma(static_cast<F>(x[j]), cs[j].x, sign * (static_cast<F>(y[j]) * cs[j].y));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int32_t e = d + j;
      const F u = static_cast<F>(to_float(head[e]));
      if (e >= a.rotary_dim) {
        out[j] = u;
        continue;
      }
      const bool second = INTER ? (e & 1) != 0 : e >= half;
      const F v = static_cast<F>(to_float(head[INTER ? e ^ 1 : second ? e - half : e + half]));
      const F2 cs = turn[INTER ? e >> 1 : second ? e - half : e];
      const F w = v * cs.y;
      out[j] = fma(u, cs.x, second ? w : -w);
    }
  }
}

// The magnitude of v rounded up to fp32.
__device__ __forceinline__ float magnitude(float v) { return fabsf(v); }
__device__ __forceinline__ float magnitude(double v) { return __double2float_ru(fabs(v)); }
__device__ __forceinline__ bool negative(float v) { return __float_as_int(v) < 0; }
__device__ __forceinline__ bool negative(double v) { return __double2hiint(v) < 0; }

// 8 elements of a group that this thread and its three neighbours hold: writes the group's
// share of codes and, on its first thread, the scale.  All 32 lanes call it.  Exact borders:
// the fp32 quotient's code is corrected by the remainder x - s n, which is exact.
template <typename F>
__device__ __forceinline__ void quantise(const F (&x)[8], bool mine, int quad, uint32_t* codes,
                                         uint16_t* scale, uint32_t* status) {
  // Largest elements of either side, rounded up to fp32 (which the 4-bit rounding up does not
  // notice) and compared by their bits, in which NaN is the largest.  Where those are equal, or
  // at a limit, the elements themselves are compared.
  float size[8];
  uint32_t hi = 0, lo = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    size[j] = magnitude(x[j]);
    const uint32_t bits = __float_as_uint(size[j]);
    if (negative(x[j])) {
      lo = max(lo, bits);
    } else {
      hi = max(hi, bits);
    }
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = max(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  const uint32_t top = max(hi, lo), huge = __float_as_uint(kHuge), tiny = __float_as_uint(kTiny);
  bool too_large = top >= huge, held = top >= tiny, mirrored = lo < hi;
  if constexpr (sizeof(F) == 8) {
    if (__any_sync(0xffffffffu, hi == lo || top == huge || top == tiny)) {
      double above = 0.0, below = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (negative(x[j])) {
          below = fmax(below, -x[j]);
        } else {
          above = fmax(above, x[j]);
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        above = fmax(above, __shfl_xor_sync(0xffffffffu, above, o));
        below = fmax(below, __shfl_xor_sync(0xffffffffu, below, o));
      }
      const double most = fmax(above, below);
      too_large = top > huge || most >= kHuge;  // (NaN is in `top` alone)
      held = most >= kTiny;
      mirrored = below < above;
    }
  }
  float s = 0.f;
  if (too_large) {  // (infinity and NaN too)
    if (mine && quad == 0) set_status(status, kStatusBadValue);
  } else if (held) {
    s = __uint_as_float((__float_as_uint(__uint_as_float(top) * 0.125f) + 0xfffffu) & 0xfff00000u);
    if (mirrored) s = -s;
  }
  if (!mine) return;
  uint32_t word = 0x88888888u;  // zeros
  if (s != 0.f) {
    float inv;  // (near enough: the remainder tells)
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fabsf(s)));
    const float limit = fabsf(s) * 0.5f;
    word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // Of magnitudes; the sign comes last.  A sum with 1.5 * 2^23 has the nearest whole number
      // in its low bits.
      const float near = fmaf(size[j], inv, 12582912.f);
      int m = __float_as_int(near) - 0x4b400000;
      const F rest = fma(F(12582912.f - near), F(fabsf(s)), x[j] < F(0) ? -x[j] : x[j]);
      const F far = rest < F(0) ? -rest : rest;
      if (far > F(limit) || (far == F(limit) && (m & 1) != 0)) m += rest < F(0) ? -1 : 1;
      const int code = (negative(x[j]) != (s < 0.f) ? -m : m) + 8;
      word |= static_cast<uint32_t>(min(15, code)) << (4 * ((j >> 1) + 4 * (j & 1)));
    }
  }
  *codes = word;
  if (quad == 0) *scale = static_cast<uint16_t>(__float_as_uint(s) >> 16);
}

// DIM: head_dim, or 0 for any.
template <typename T, bool INTER, bool VEC, int DIM>
__global__ void __launch_bounds__(kThreads) int4_append_kernel(const AppendArgs a) {
  extern __shared__ double2 shared_turns[];
  pdl_wait();
  pdl_trigger();
  const int32_t t = blockIdx.x;
  const T* row = static_cast<const T*>(a.qkv) + t * a.qkv_stride;
  const int32_t D = DIM > 0 ? DIM : a.D, per = D >> 3;  // units of 8 dims a head
  // The token's row will be wanted once its angles are there.
  for (int64_t at = threadIdx.x * 128ll; at < (a.H + 2 * a.Hkv) * D * static_cast<int64_t>(sizeof(T));
       at += kThreads * 128) {
    asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const char*>(row) + at));
  }
  const int32_t half = a.rotary_dim >> 1;
  const Turns turn{shared_turns, reinterpret_cast<float2*>(shared_turns + half)};
  const int32_t slot = a.slots[t], p = a.rotary_dim > 0 ? a.pos[t] : 0;
  const bool bad_slot = slot >= a.num_blocks * a.block_size;  // fits in int32 (host)
  const bool rotate = p >= 0, append = slot >= 0 && !bad_slot;
  if (threadIdx.x == 0) {
    if (p < 0) set_status(a.status, kStatusBadPosition);
    if (bad_slot) set_status(a.status, kStatusBadSlot);
  }
  if (rotate) {
    for (int32_t i = threadIdx.x; i < half; i += kThreads) {
      const double turns = static_cast<double>(p) * a.freq[i] * kTurnsPerRad;
      double s, c;
      sincospi(2.0 * (turns - rint(turns)), &s, &c);
      c *= a.amp;
      s *= a.amp;
      turn.exact[i] = make_double2(c, s);
      turn.rounded[i] = make_float2(static_cast<float>(c), static_cast<float>(s));
    }
  }
  const int32_t at = append ? slot : 0, blk = at / a.block_size, off = at - blk * a.block_size;
  const int64_t block_bytes = static_cast<int64_t>(a.block_size) * int4_row_bytes(D);
  const int32_t units = a.Hkv * per;
  auto store_heads = [&](bool keys) {
    const T* heads = row + (a.H + (keys ? 0 : a.Hkv)) * D;
    uint8_t* pool = keys ? a.k_pool : a.v_pool;
    // Values from the last warp down: they are there before the angles, which the first warps
    // work on.
    const int32_t first = keys ? threadIdx.x & ~31 : kThreads - 32 - (threadIdx.x & ~31);
    for (int32_t u0 = first; u0 < units; u0 += kThreads) {
      const int32_t own = u0 + static_cast<int32_t>(threadIdx.x & 31), u = min(own, units - 1);
      const int32_t hh = u / per, d = (u - hh * per) * 8;
      uint8_t* block = pool + (static_cast<int64_t>(hh) * a.num_blocks + blk) * block_bytes;
      uint32_t* codes = reinterpret_cast<uint32_t*>(block + off * int4_code_bytes(D) + (d >> 1));
      uint16_t* scale = reinterpret_cast<uint16_t*>(block + a.block_size * int4_code_bytes(D) +
                                                    off * int4_scale_bytes(D)) + d / kInt4Group;
      const int quad = threadIdx.x & 3;
      if (keys && a.rotary_dim > 0) {
        double v[8];
        turned<T, INTER, VEC>(a, heads + hh * D, d, turn.exact, v);
        quantise(v, own < units && rotate, quad, codes, scale, a.status);
      } else {
        float v[8];
        if constexpr (VEC) {
          load8(heads + hh * D + d, v);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = to_float(heads[hh * D + d + j]);
        }
        quantise(v, own < units, quad, codes, scale, a.status);
      }
    }
  };
  if (append) store_heads(false);
  __syncthreads();
  if (append) store_heads(true);
  if (rotate) {
    T* q_row = static_cast<T*>(a.q_out) + static_cast<int64_t>(t) * a.H * D;
    // (From the last thread down: the first have the keys.)
    const int32_t me = kThreads - 1 - static_cast<int32_t>(threadIdx.x);
    if constexpr (VEC && !INTER) {
      // 8 pairs at a time: dims d and those half the rotary dims on; then the dims behind.
      const int32_t pairs = half >> 3, rest = (D - a.rotary_dim) >> 3;
      for (int32_t u = me; u < a.H * pairs; u += kThreads) {
        const int32_t h = u / pairs, d = (u - h * pairs) * 8;
        const T* src = row + h * D + d;
        T* dst = q_row + h * D + d;
        float x[8], y[8];
        load8(src, x);
        load8(src + half, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 cs = turn.rounded[d + j];
          const float v = fmaf(x[j], cs.x, -(y[j] * cs.y));
          y[j] = fmaf(y[j], cs.x, x[j] * cs.y);
          x[j] = v;
        }
        store8(dst, x);
        store8(dst + half, y);
      }
      for (int32_t u = me; u < a.H * rest; u += kThreads) {
        const int32_t h = u / rest, e = h * D + a.rotary_dim + (u - h * rest) * 8;
        float x[8];
        load8(row + e, x);
        store8(q_row + e, x);
      }
    } else {
      for (int32_t u = me; u < a.H * per; u += kThreads) {
        const int32_t h = u / per, d = (u - h * per) * 8;
        float y[8];
        turned<T, INTER, VEC>(a, row + h * D, d, turn.rounded, y);
        if constexpr (VEC) {
          store8(q_row + h * D + d, y);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) store(q_row + h * D + d + j, y[j]);
        }
      }
    }
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
  cfg.dynamicSmemBytes = (sizeof(double2) + sizeof(float2)) * (a.rotary_dim / 2);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = int4_append_kernel<T, false, false, 0>;
  if (!vec) {
    if (interleaved) kernel = int4_append_kernel<T, true, false, 0>;
  } else if (a.D == 64) {
    kernel = interleaved ? int4_append_kernel<T, true, true, 64> : int4_append_kernel<T, false, true, 64>;
  } else if (a.D == 128) {
    kernel = interleaved ? int4_append_kernel<T, true, true, 128> : int4_append_kernel<T, false, true, 128>;
  } else {
    kernel = interleaved ? int4_append_kernel<T, true, true, 0> : int4_append_kernel<T, false, true, 0>;
  }
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
