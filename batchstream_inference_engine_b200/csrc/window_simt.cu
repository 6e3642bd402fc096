// Sliding-window paged attention on the CUDA cores: fp32 pools and every shape
// the tensor-core kernels do not take (any block size, head_dim <= 256, up to 16
// query heads per kv head), for single tokens and for prompt chunks.
//
// One CTA per (query tile, kv head, key range); the tile is one token, or as many
// tokens of a chunk as fill 16 rows with their query heads, so each key row is
// read once for all of them.  Each warp takes every fourth group of 32 keys: lane
// j looks up key j of the group, the warp starts asynchronous 16-byte copies of the
// group's K rows, then of its V rows, into shared memory (so a group costs the
// latency of its table entries and one of its rows, whatever their number), lane j
// computes key j's scores against the query rows (fp32 in shared memory, read as
// broadcasts), the running softmax of a row comes from warp reductions, and the V
// rows are weighted with lanes along head_dim.  No barrier until the four warps'
// states are combined at the end.  Rows of more than 256 bytes copy V over K once the
// scores are there: both would leave room for one CTA on an SM (fp32, d128, 200
// sequences, window 2000: 140 us with both, 117 so; 47 sequences, window 900: 31 and
// 33).  24 fp32 sequences of up to 4096 tokens, d64, window 777: 12.1 us, a chain of
// table entry, rows, scores, V and join with too few keys to hide it (one warp lane
// loading its own key row instead: 68 us).  The ranges of a tile are a cluster that
// joins through distributed shared memory while clusters take no more waves than single
// CTAs would; else they leave records for a second kernel, which costs some 4 us.  Rows that are not whole 16-byte pieces are read one element at a time.
//
// Over 4-bit pools a group's codes are turned into floats on their way to shared memory, K's,
// then V's in their place: an element costs some three instructions there, next to its four
// to eight products.  Loads of eight rows' pieces are issued together and scores read 16 bytes:
// 24 fp32 sequences of 1 to 4096 tokens, d64, whole context: 47 us (one element at a time: 68);
// with 16 heads a group 94 (227).
//
// A weight of zero skips its V row, so NaN or infinities in a key that a row does
// not see never reach that row.
#include <mutex>
#include <type_traits>
#include <vector>

#include "int4.cuh"
#include "window.cuh"

namespace bsb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2eW = 1.4426950408889634f;

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T of_float(float v);
template <>
__device__ __forceinline__ float of_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 of_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// 16 bytes of a row as floats.
__device__ __forceinline__ void widen16(const float* p, float (&out)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  out[0] = v.x; out[1] = v.y; out[2] = v.z; out[3] = v.w;
}
__device__ __forceinline__ void widen16(const __nv_bfloat16* p, float (&out)[8]) { load8(p, out); }

__device__ __forceinline__ void copy16_async(void* smem_dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem_dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory of one warp: 32 K rows, then 32 V rows or the V rows in their place; at
// the end its state, GM rows of head_dim floats.  Lanes read K rows in parallel, so a
// pad of 16 bytes (one float in the element-wise form, which holds K as floats and
// leaves V in the pool) moves consecutive rows to different banks.  Rows of 4-bit pools
// are floats, V in K's place.
template <typename T, int GM, int DPL, bool VEC, bool Q4>
struct Layout {
  static constexpr bool kVOverK = DPL * 32 * sizeof(T) > 256;
  __host__ __device__ static int k_row(int D) {
    return Q4 ? D * 4 + 16 : VEC ? D * static_cast<int>(sizeof(T)) + 16 : (D + 1) * 4;
  }
  __host__ __device__ static int v_row(int D) {
    return kVOverK ? k_row(D) : D * static_cast<int>(sizeof(T));
  }
  __host__ __device__ static int v_offset(int D) { return kVOverK ? 0 : 32 * k_row(D); }
  __host__ __device__ static int warp_bytes(int D) {
    const int rows = VEC ? v_offset(D) + 32 * v_row(D) : 32 * k_row(D), state = GM * D * 4;
    return ((rows > state ? rows : state) + 15) / 16 * 16;
  }
  __host__ __device__ static int q_bytes(int D) { return (GM * D * 4 + 15) / 16 * 16; }
  // Query rows | warps | probabilities [warp][32][GM] | maxima, sums [warp][GM].
  __host__ __device__ static int total(int D) {
    return q_bytes(D) + kWarps * (warp_bytes(D) + 32 * GM * 4 + 2 * GM * 4);
  }
};

// Linear CTA index -> (sequence, query tile, kv head).
__device__ __forceinline__ void window_item(const WindowArgs& a, int64_t item, int32_t& r,
                                            int32_t& tile, int32_t& h) {
  h = static_cast<int32_t>(item % a.num_kv_heads);
  item /= a.num_kv_heads;
  tile = static_cast<int32_t>(item % a.qtiles);
  r = static_cast<int32_t>(item / a.qtiles);
}

// GM: query rows held per CTA; DPL: head dims per lane; VEC: 16-byte K rows; FULL:
// head_dim is exactly 32 DPL (its loops then have compile-time bounds); Q4: 4-bit pools.
template <typename T, int GM, int DPL, bool VEC, bool FULL, bool Q4>
__global__ void __launch_bounds__(kThreads) window_simt_kernel(const WindowArgs a) {
  static_assert(!Q4 || !VEC, "4-bit rows are held as floats");
  using L_ = Layout<T, GM, DPL, VEC, Q4>;
  extern __shared__ __align__(16) uint8_t wsm[];
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t split = blockIdx.x % a.splits;
  const int64_t item = blockIdx.x / a.splits;
  int32_t r, tile, h;
  window_item(a, item, r, tile, h);
  WindowTile w;
  if (!window_tile(a, r, tile, w, tid == 0 && tile == 0 && h == 0 && split == 0)) return;
  const int32_t per = window_range(w.count, a.splits);
  // (A cluster's CTA without keys stays: it joins, and the others read its empty part.)
  if (!a.clustered && static_cast<int64_t>(split) * per >= w.count) return;
  const int32_t begin =
      static_cast<int32_t>(min(static_cast<int64_t>(split) * per, static_cast<int64_t>(w.count)));
  const int32_t end = w.count - begin < per ? w.count : begin + per;

  const int G = a.groups, D = FULL ? 32 * DPL : a.head_dim, bs = a.block_size;
  const int rows = w.ntok * G;  // <= GM (host)
  float* sQ = reinterpret_cast<float*>(wsm);
  uint8_t* states = wsm + L_::q_bytes(D);
  const int warp_bytes = L_::warp_bytes(D), k_row = L_::k_row(D), v_row = L_::v_row(D);
  uint8_t* sK = states + warp * warp_bytes;
  uint8_t* sV = sK + L_::v_offset(D);
  float* probs = reinterpret_cast<float*>(states + kWarps * warp_bytes);
  float* sP = probs + warp * 32 * GM;
  float* sM = probs + kWarps * 32 * GM;
  float* sL = sM + kWarps * GM;

  // Query rows: row t * G + g is head g of the kv head's group, token t.
  const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(w.tok0) * a.q_stride +
               static_cast<int64_t>(h) * G * D;
  for (int e = tid; e < rows * D; e += kThreads) {
    const int t = e / (G * D);
    sQ[e] = to_float<T>(q[static_cast<int64_t>(t) * a.q_stride + (e - t * G * D)]);
  }
  __syncthreads();

  const int64_t head_off = static_cast<int64_t>(h) * a.num_blocks * bs * D;
  const T* kh = static_cast<const T*>(a.k_pool) + head_off;
  const T* vh = static_cast<const T*>(a.v_pool) + head_off;
  const int32_t* table = a.block_tables + static_cast<int64_t>(w.row) * a.bt_stride;
  const float zscale = a.scale * kLog2eW;

  float m[GM], l[GM], o[GM][DPL];
#pragma unroll
  for (int i = 0; i < GM; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int k = 0; k < DPL; ++k) o[i][k] = 0.f;
  }

  for (int32_t base = begin + warp * 32; base < end; base += kThreads) {
    // Lane j's key of the group: its position and its row's offset (-1: none).
    const int32_t v = base + lane;
    int32_t pos = 0;
    int64_t off = -1, scales = 0;  // Q4: bytes, of the row's codes and scales
    if (v < end) {
      pos = window_key(w, v);
      const int32_t blk = __ldg(table + pos / bs);
      if (blk >= 0 && blk < a.num_blocks) {
        if constexpr (Q4) {
          off = (static_cast<int64_t>(h) * a.num_blocks + blk) * bs * int4_row_bytes(D);
          scales = off + static_cast<int64_t>(bs) * int4_code_bytes(D) +
                   (pos % bs) * int4_scale_bytes(D);
          off += (pos % bs) * int4_code_bytes(D);
        } else {
          off = (static_cast<int64_t>(blk) * bs + pos % bs) * D;
        }
      } else {
        set_status(a.status, kStatusBadBlock);
      }
    }
    constexpr int kElems = 16 / sizeof(T);
    // Copies of 16 bytes, consecutive lanes along a row; rows of no key stay as they
    // are (their scores and weights are never used).
    auto copy_rows = [&](int first, int last) {  // 0: K, 1: V
      const int per_row = D / kElems;
      for (int part = first; part <= last; ++part) {
        const T* from = part == 0 ? kh : vh;
        uint8_t* to = part == 0 ? sK : sV;
        const int stride = part == 0 ? k_row : v_row;
#pragma unroll 4
        for (int it = 0; it < per_row; ++it) {
          const int idx = it * 32 + lane;
          const int key = idx / per_row, c = idx - key * per_row;
          const int64_t ko = __shfl_sync(0xffffffffu, off, key);
          if (ko >= 0) copy16_async(to + key * stride + c * 16, from + ko + c * kElems);
        }
        copy_commit();
      }
    };
    // A pool's rows as floats, a lane taking 8 dims at a time, of 4 or 8 rows at once.
    auto widen_rows = [&](const void* pool) {
      const int per_row = D >> 3;  // a multiple of 4
      const uint8_t* bytes = static_cast<const uint8_t*>(pool);
      constexpr int kAtOnce = FULL && DPL > 1 ? 8 : 4;
      for (int it = 0; it < per_row; it += kAtOnce) {
        uint32_t words[kAtOnce];
        uint16_t scale[kAtOnce];
        int to[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int idx = (it + k) * 32 + lane;
          const int key = idx / per_row, c = idx - key * per_row;
          const int64_t ko = __shfl_sync(0xffffffffu, off, key);
          const int64_t so = __shfl_sync(0xffffffffu, scales, key);
          to[k] = ko < 0 ? -1 : key * k_row + 32 * c;
          if (ko < 0) continue;
          words[k] = coherent_load(reinterpret_cast<const uint32_t*>(bytes + ko) + c);
          scale[k] = coherent_load(reinterpret_cast<const uint16_t*>(bytes + so) + (c >> 2));
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          if (to[k] < 0) continue;
          float f[8];
          int4_floats(words[k], int4_scale_float(scale[k]), f);
          float4* dst = reinterpret_cast<float4*>(sK + to[k]);
          dst[0] = make_float4(f[0], f[1], f[2], f[3]);
          dst[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
      }
    };
    if constexpr (Q4) {
      widen_rows(a.k_pool);
    } else if constexpr (VEC) {
      copy_rows(0, L_::kVOverK ? 0 : 1);
      copy_wait<L_::kVOverK ? 0 : 1>();
    } else {
      for (int key = 0; key < 32; ++key) {
        const int64_t ko = __shfl_sync(0xffffffffu, off, key);
        if (ko < 0) continue;
        float* dst = reinterpret_cast<float*>(sK + key * k_row);
        for (int d = lane; d < D; d += 32) dst[d] = to_float<T>(kh[ko + d]);
      }
    }
    __syncwarp();
    float s[GM];
#pragma unroll
    for (int i = 0; i < GM; ++i) s[i] = 0.f;
    if constexpr (VEC || Q4) {
      using Held = std::conditional_t<Q4, float, T>;
      constexpr int kHeld = 16 / sizeof(Held);
      const Held* krow = reinterpret_cast<const Held*>(sK + lane * k_row);
#pragma unroll 4
      for (int d = 0; d < D; d += kHeld) {
        float k[kHeld];
        widen16(krow + d, k);
#pragma unroll
        for (int i = 0; i < GM; ++i) {
          if (i < rows) {
#pragma unroll
            for (int x = 0; x < kHeld; x += 4) {
              const float4 q4 = *reinterpret_cast<const float4*>(sQ + i * D + d + x);
              s[i] = fmaf(q4.x, k[x], fmaf(q4.y, k[x + 1],
                                           fmaf(q4.z, k[x + 2], fmaf(q4.w, k[x + 3], s[i]))));
            }
          }
        }
      }
    } else {
      const float* krow = reinterpret_cast<const float*>(sK + lane * k_row);
      for (int d = 0; d < D; ++d) {
        const float kv = krow[d];
#pragma unroll
        for (int i = 0; i < GM; ++i) {
          if (i < rows) s[i] = fmaf(sQ[i * D + d], kv, s[i]);
        }
      }
    }
    if constexpr (VEC && L_::kVOverK) {
      __syncwarp();  // every lane has read its K row
      copy_rows(1, 1);
    }
    if constexpr (Q4) {
      __syncwarp();  // every lane has read its K row
      widen_rows(a.v_pool);
    }
#pragma unroll
    for (int i = 0; i < GM; ++i) {
      if (i >= rows) {
        sP[lane * GM + i] = 0.f;
        continue;
      }
      const int32_t qpos = w.pos0 + i / G;
      const bool seen = off >= 0 && pos <= qpos && (pos < a.sinks || pos > qpos - a.window);
      const float z = seen ? s[i] * zscale : -INFINITY;
      float mx = z;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mnew = fmaxf(m[i], mx);
      const float mb = mnew == -INFINITY ? 0.f : mnew;  // no key of this row yet
      const float corr = fast_exp2(m[i] - mb);
      const float p = seen ? fast_exp2(z - mb) : 0.f;
      m[i] = mnew;
      l[i] = l[i] * corr + p;  // this lane's part of the sum
#pragma unroll
      for (int k = 0; k < DPL; ++k) o[i][k] *= corr;
      sP[lane * GM + i] = p;
    }
    if constexpr (VEC) copy_wait<0>();
    __syncwarp();
    const uint32_t held = __ballot_sync(0xffffffffu, off >= 0);  // keys with a row
    const int nkeys = min(32, end - base);
#pragma unroll 4
    for (int j = 0; j < nkeys; ++j) {
      if (!((held >> j) & 1u)) continue;
      const int64_t vo = VEC || Q4 ? 0 : __shfl_sync(0xffffffffu, off, j);
      float vv[DPL];
#pragma unroll
      for (int k = 0; k < DPL; ++k) {
        const int d = lane + 32 * k;
        if constexpr (Q4) {
          vv[k] = d < D ? reinterpret_cast<const float*>(sK + j * k_row)[d] : 0.f;
        } else if constexpr (VEC) {
          vv[k] = FULL || d < D ? to_float<T>(reinterpret_cast<const T*>(sV + j * v_row)[d]) : 0.f;
        } else {
          vv[k] = FULL || d < D ? to_float<T>(vh[vo + d]) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < GM; i += 4) {
        if (i >= rows) continue;
        // Rows past the tile's hold zeros.
        const float4 p4 = *reinterpret_cast<const float4*>(sP + j * GM + i);
        const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (p[x] != 0.f) {
#pragma unroll
            for (int k = 0; k < DPL; ++k) o[i + x][k] = fmaf(p[x], vv[k], o[i + x][k]);
          }
        }
      }
    }
    __syncwarp();  // the next group overwrites sK and sP
  }

  // Each warp's state over its own K and V rows.
  float* state = reinterpret_cast<float*>(sK);
#pragma unroll
  for (int i = 0; i < GM; ++i) {
    if (i >= rows) continue;
    float lr = l[i];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) lr += __shfl_xor_sync(0xffffffffu, lr, x);
    if (lane == 0) {
      sM[warp * GM + i] = m[i];
      sL[warp * GM + i] = lr;
    }
#pragma unroll
    for (int k = 0; k < DPL; ++k) {
      const int d = lane + 32 * k;
      if (d < D) state[i * D + d] = o[i][k];
    }
  }
  __syncthreads();
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(w.tok0) * a.o_stride +
           static_cast<int64_t>(h) * G * D;
  // A cluster's CTA leaves its part where the query rows were, its maxima and sums where
  // the weights were.
  float* rec = a.clustered ? sQ : a.splits > 1 ? a.records + static_cast<int64_t>(blockIdx.x) * a.rec_stride : nullptr;
  for (int e = tid; e < rows * D; e += kThreads) {
    const int i = e / D;
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) M = fmaxf(M, sM[x * GM + i]);
    const float mb = M == -INFINITY ? 0.f : M;
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float f = fast_exp2(sM[x * GM + i] - mb);
      L += sL[x * GM + i] * f;
      O += reinterpret_cast<const float*>(states + x * warp_bytes)[e] * f;
    }
    if (rec != nullptr) {
      rec[e] = O;
      if (e - i * D == 0) {
        float* ml = a.clustered ? probs : rec + GM * D;
        ml[i] = M;
        ml[GM + i] = L;
      }
    } else {
      const int t = e / (G * D);
      out[static_cast<int64_t>(t) * a.o_stride + (e - t * G * D)] = of_float<T>(O / L);
    }
  }
  if (!a.clustered) return;
  // Every CTA joins a share of the elements, in range order; all reads of a join are
  // issued before the first is used.
  cluster_sync();
  for (int e = split * kThreads + tid; e < rows * D; e += a.splits * kThreads) {
    const int i = e / D;
    float ms[kMaxWindowCluster], ls[kMaxWindowCluster], os[kMaxWindowCluster], M = -INFINITY;
#pragma unroll
    for (int x = 0; x < kMaxWindowCluster; ++x) {
      ms[x] = x < a.splits ? cluster_load(probs, i, x) : -INFINITY;
      ls[x] = x < a.splits ? cluster_load(probs, GM + i, x) : 0.f;
      os[x] = x < a.splits ? cluster_load(sQ, e, x) : 0.f;
    }
#pragma unroll
    for (int x = 0; x < kMaxWindowCluster; ++x) M = fmaxf(M, ms[x]);
    const float mb = M == -INFINITY ? 0.f : M;
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int x = 0; x < kMaxWindowCluster; ++x) {
      const float f = fast_exp2(ms[x] - mb);
      L += ls[x] * f;
      O += os[x] * f;
    }
    const int t = e / (G * D);
    out[static_cast<int64_t>(t) * a.o_stride + (e - t * G * D)] = of_float<T>(O / L);
  }
  cluster_sync();  // the others may still read this CTA's shared memory
}

// Joins the records of a tile's key ranges, in range order.
template <typename T, int GM>
__global__ void __launch_bounds__(kThreads) window_simt_merge_kernel(const WindowArgs a) {
  pdl_wait();
  int32_t r, tile, h;
  window_item(a, blockIdx.x, r, tile, h);
  WindowTile w;
  if (!window_tile(a, r, tile, w, false)) return;
  const int G = a.groups, D = a.head_dim;
  const int32_t per = window_range(w.count, a.splits);
  const int n = (w.count + per - 1) / per;
  const float* rec = a.records + static_cast<int64_t>(blockIdx.x) * a.splits * a.rec_stride;
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(w.tok0) * a.o_stride +
           static_cast<int64_t>(h) * G * D;
  for (int e = threadIdx.x; e < w.ntok * G * D; e += kThreads) {
    const int i = e / D;
    float M = -INFINITY;
    for (int s = 0; s < n; ++s) {
      M = fmaxf(M, rec[static_cast<int64_t>(s) * a.rec_stride + GM * D + i]);
    }
    const float mb = M == -INFINITY ? 0.f : M;
    float L = 0.f, O = 0.f;
    for (int s = 0; s < n; ++s) {
      const float* p = rec + static_cast<int64_t>(s) * a.rec_stride;
      const float f = fast_exp2(p[GM * D + i] - mb);
      L += p[GM * D + GM + i] * f;
      O += p[e] * f;
    }
    const int t = e / (G * D);
    out[static_cast<int64_t>(t) * a.o_stride + (e - t * G * D)] = of_float<T>(O / L);
  }
}

// Shared memory for an instance's largest head_dim.
template <typename T, int GM, int DPL, bool VEC, bool FULL, bool Q4>
cudaError_t allow_smem() {
  static unsigned long long configured = 0;  // one bit per device
  return once_per_device(&configured, [] {
    return cudaFuncSetAttribute(window_simt_kernel<T, GM, DPL, VEC, FULL, Q4>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Layout<T, GM, DPL, VEC, Q4>::total(DPL * 32));
  });
}

template <typename T, int GM, int DPL, bool VEC, bool FULL, bool Q4 = false>
int launch_one(const WindowArgs& a, cudaStream_t stream) {
  using L_ = Layout<T, GM, DPL, VEC, Q4>;
  const int smem = L_::total(a.head_dim);
  auto kernel = window_simt_kernel<T, GM, DPL, VEC, FULL, Q4>;
  const cudaError_t e = allow_smem<T, GM, DPL, VEC, FULL, Q4>();
  if (e != cudaSuccess) return static_cast<int>(e);
  const int64_t items = static_cast<int64_t>(a.num_rows) * a.qtiles * a.num_kv_heads;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * a.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.clustered) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  const int rc = static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, a));
  if (rc != 0 || a.splits == 1 || a.clustered) return rc;
  cfg.gridDim = dim3(static_cast<unsigned>(items));
  cfg.dynamicSmemBytes = 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, window_simt_merge_kernel<T, GM>, a));
}

template <typename T, int GM, int DPL, bool VEC>
int launch_full(const WindowArgs& a, cudaStream_t stream) {
  if (VEC && a.head_dim == 32 * DPL) return launch_one<T, GM, DPL, VEC, VEC>(a, stream);
  return launch_one<T, GM, DPL, VEC, false>(a, stream);
}

template <typename T, int GM>
int launch_q4(const WindowArgs& a, cudaStream_t stream) {
  if (a.head_dim == 32) return launch_one<T, GM, 1, false, true, true>(a, stream);
  if (a.head_dim == 64) return launch_one<T, GM, 2, false, true, true>(a, stream);
  if (a.head_dim == 128) return launch_one<T, GM, 4, false, true, true>(a, stream);
  if (a.head_dim < 128) return launch_one<T, GM, 4, false, false, true>(a, stream);
  return launch_one<T, GM, 8, false, false, true>(a, stream);
}

template <typename T, int GM, bool VEC>
int launch_dims(const WindowArgs& a, cudaStream_t stream) {
  if (a.head_dim <= 32) return launch_full<T, GM, 1, VEC>(a, stream);
  if (a.head_dim <= 64) return launch_full<T, GM, 2, VEC>(a, stream);
  if (a.head_dim <= 128) return launch_full<T, GM, 4, VEC>(a, stream);
  return launch_full<T, GM, 8, VEC>(a, stream);
}

template <typename T>
int launch_rows(const WindowArgs& a, bool vec, cudaStream_t stream) {
  const bool wide = a.tile_tokens * a.groups > 8;
  if (a.int4) return wide ? launch_q4<T, kWindowSimtRows>(a, stream) : launch_q4<T, 8>(a, stream);
  if (!wide) {
    return vec ? launch_dims<T, 8, true>(a, stream) : launch_dims<T, 8, false>(a, stream);
  }
  return vec ? launch_dims<T, kWindowSimtRows, true>(a, stream)
             : launch_dims<T, kWindowSimtRows, false>(a, stream);
}

// What the device runs at once of an instance: CTAs per SM (cluster 1), or clusters of
// `cluster` CTAs on the whole device; or a CUDA error, negative.  Asked for once per
// device and size.
template <typename T, int GM, int DPL, bool VEC, bool FULL, bool Q4 = false>
int at_once(int D, int cluster) {
  struct Known {
    int device, D, cluster, count;
  };
  static std::mutex mutex;
  static std::vector<Known> known;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return -static_cast<int>(e);
  std::lock_guard<std::mutex> lock(mutex);
  for (const Known& k : known) {
    if (k.device == dev && k.D == D && k.cluster == cluster) return k.count;
  }
  using L_ = Layout<T, GM, DPL, VEC, Q4>;
  auto kernel = window_simt_kernel<T, GM, DPL, VEC, FULL, Q4>;
  e = allow_smem<T, GM, DPL, VEC, FULL, Q4>();
  int count = 0;
  if (e == cudaSuccess && cluster == 1) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&count, kernel, kThreads, L_::total(D));
  } else if (e == cudaSuccess) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = L_::total(D);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&count, kernel, &cfg);
  }
  if (e != cudaSuccess) return -static_cast<int>(e);
  known.push_back({dev, D, cluster, count});
  return count;
}

// As the launch chooses, with aligned pools.
template <typename T, int GM, int DPL>
int at_once_full(int D, int cluster, bool int4) {
  if (int4) {
    if constexpr (DPL >= 4) {
      if (D != 128) return at_once<T, GM, DPL, false, false, true>(D, cluster);
    }
    if constexpr (DPL <= 4) return at_once<T, GM, DPL, false, true, true>(D, cluster);
  }
  if (D * sizeof(T) % 16 != 0) return at_once<T, GM, DPL, false, false>(D, cluster);
  return D == 32 * DPL ? at_once<T, GM, DPL, true, true>(D, cluster)
                       : at_once<T, GM, DPL, true, false>(D, cluster);
}

template <typename T, int GM>
int at_once_dims(int D, int cluster, bool int4) {
  return D <= 32 ? at_once_full<T, GM, 1>(D, cluster, int4)
         : D <= 64 ? at_once_full<T, GM, 2>(D, cluster, int4)
         : D <= 128 ? at_once_full<T, GM, 4>(D, cluster, int4)
                    : at_once_full<T, GM, 8>(D, cluster, int4);
}

}  // namespace

int window_simt_at_once(bool bf16, bool int4, bool wide, int head_dim, int cluster) {
  return bf16 ? (wide ? at_once_dims<__nv_bfloat16, kWindowSimtRows>(head_dim, cluster, int4)
                      : at_once_dims<__nv_bfloat16, 8>(head_dim, cluster, int4))
              : (wide ? at_once_dims<float, kWindowSimtRows>(head_dim, cluster, int4)
                      : at_once_dims<float, 8>(head_dim, cluster, int4));
}

int launch_window_simt(const WindowArgs& a, bool bf16, bool vec, cudaStream_t stream) {
  return bf16 ? launch_rows<__nv_bfloat16>(a, vec, stream) : launch_rows<float>(a, vec, stream);
}

}  // namespace bsb
