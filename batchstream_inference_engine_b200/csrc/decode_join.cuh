// Split-K decode: how the parts of a segment that several warps, or several CTAs, have
// worked on come together.  Shared by the tensor-core kernels over bf16 and 4-bit pools.
//
// C is the kernel's configuration: W warps with S stages of STAGE_BYTES each at the start of
// shared memory, then W slots of SLOT0_BYTES; GROWS query rows, of one token or, for short
// chunks (CHUNK), several.  A warp leaves a part (O
// unnormalised [G][D], then row maxima in base 2 and row sums) in its slot 0, its last part
// in slot 1, which lies over its stages.
#pragma once

#include "decode.cuh"

namespace bsb {

constexpr int kMaxRanks = 8;  // CTAs of a cluster

// Whose parts the slots hold (seq < 0: none).
template <int W>
struct WarpSlots {
  int32_t seq[W][2], kvh[W][2], nb[W][2];
  int64_t unit[W][2];
};

template <typename C>
__device__ __forceinline__ float* warp_slot(uint8_t* smem, int w, int k) {
  return reinterpret_cast<float*>(k == 0 ? smem + C::W * C::S * C::STAGE_BYTES + w * C::SLOT0_BYTES
                                         : smem + w * C::S * C::STAGE_BYTES);
}

// The end of a cluster's segment (DecodeArgs::segment_ctas): every warp with units has
// left its part (O, maxima, sums) in its slot 0.  The CTA joins its warps' parts, all
// threads at once, then the cluster's CTAs each join a share of the elements over all
// CTAs' parts, in rank order.  Every read of a join is issued before the first is used:
// one trip through distributed shared memory costs some 250 ns.  A part without a finite
// score has the maximum -inf and weighs 0, but is not left out: if its scores are NaN,
// so are its O and sums, and 0 * NaN brings that to the output.
template <typename C, int D>
__device__ __forceinline__ void join_segment(const DecodeArgs& a, uint8_t* smem,
                                             const WarpSlots<C::W>& slots, int32_t seq,
                                             int32_t kvh, int32_t ranks) {
  constexpr int W = C::W, kThreads = W * 32;
  __shared__ float part_ml[2 * C::GROWS];
  float* part = reinterpret_cast<float*>(smem);  // over the stages, whose copies are done
  const int tid = threadIdx.x, G = a.groups;
  const OutRows<C::CHUNK> to(a, seq, kvh);
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out);
  __syncthreads();
  bool parked = ranks > 1;  // or one warp has written the output
#pragma unroll
  for (int w = 0; w < W; ++w) parked |= slots.seq[w][0] >= 0;
  if (!parked) return;
  for (int e = tid; e < G * D; e += kThreads) {
    const int r = e / D;
    float m[W], l[W], o[W], M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* slot = warp_slot<C>(smem, w, 0);
      const bool has = slots.seq[w][0] >= 0;
      m[w] = has ? slot[G * D + r] : -INFINITY;
      l[w] = has ? slot[G * D + G + r] : 0.f;
      o[w] = has ? slot[e] : 0.f;
      M = fmaxf(M, m[w]);
    }
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = fast_exp2(m[w] - base);
      L += f * l[w];
      O += f * o[w];
    }
    if (ranks == 1) {
      if (!C::CHUNK || r < to.rows) out[to.row(r, D) + e - r * D] = __float2bfloat16_rn(O / L);
    } else {
      part[e] = O;
      if (e % D == 0) {
        part_ml[r] = M;
        part_ml[C::GROWS + r] = L;
      }
    }
  }
  if (ranks == 1) return;
  cluster_sync();
  const int rank = blockIdx.x % a.segment_ctas;
  for (int e = rank * kThreads + tid; e < G * D; e += ranks * kThreads) {
    const int r = e / D;
    float m[kMaxRanks], l[kMaxRanks], o[kMaxRanks], M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxRanks; ++k) {
      m[k] = k < ranks ? cluster_load(part_ml, r, k) : -INFINITY;
      l[k] = k < ranks ? cluster_load(part_ml, C::GROWS + r, k) : 0.f;
      o[k] = k < ranks ? cluster_load(part, e, k) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kMaxRanks; ++k) M = fmaxf(M, m[k]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxRanks; ++k) {
      const float f = fast_exp2(m[k] - base);
      L += f * l[k];
      O += f * o[k];
    }
    if (!C::CHUNK || r < to.rows) out[to.row(r, D) + e - r * D] = __float2bfloat16_rn(O / L);
  }
  cluster_sync();  // the others may still read this CTA's shared memory
}

// A CTA's end (spans over the batch): a segment cut between warps is a chain: the last
// portion of the warp where it starts, the only portion of warps inside it, the first
// portion of the warp where it ends.  The chain's tail (no later non-empty warp continues
// the segment) folds the earlier slots into its own and finishes the segment: writes the
// output, or hands a segment that other CTAs hold parts of to
// cut(seq, kvh, seg_unit, nb, part), which the warp calls together.
template <typename C, int D, typename CutFn>
__device__ __forceinline__ void fold_slots(const DecodeArgs& a, uint8_t* smem, const Span& sp,
                                           int64_t spanw, const WarpSlots<C::W>& slots,
                                           CutFn&& cut) {
  constexpr int W = C::W;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.groups;
  __syncthreads();
  auto warp_empty = [&](int w) {
    return sp.r0 + spanw * (w + 1) / W == sp.r0 + spanw * w / W;
  };
  auto holds = [&](int w, int k, int32_t seq, int32_t kvh) {
    return slots.seq[w][k] == seq && slots.kvh[w][k] == kvh;
  };
  for (int k = 0; k < 2; ++k) {
    const int32_t seq = slots.seq[warp][k];
    if (seq < 0) continue;
    const int32_t kvh = slots.kvh[warp][k];
    bool tail = true;
    if (k == 1 || slots.seq[warp][1] < 0) {
      for (int w2 = warp + 1; w2 < W; ++w2) {
        if (warp_empty(w2)) continue;
        tail = !holds(w2, 0, seq, kvh);
        break;
      }
    }
    if (!tail) continue;
    float* mine = warp_slot<C>(smem, warp, k);
    for (int w2 = warp - 1; w2 >= 0; --w2) {
      if (warp_empty(w2)) continue;
      const int k2 = holds(w2, 1, seq, kvh) ? 1 : (holds(w2, 0, seq, kvh) ? 0 : -1);
      if (k2 < 0) break;
      const float* other = warp_slot<C>(smem, w2, k2);
      // Row factors once (lane r < G), then one FMA pair per element; a row
      // spans D >= 64 elements, so elements e = lane + 32j share row (32j) / D.
      float fa = 0.f, fb = 0.f;
      if (lane < G) {
        const float ma = mine[G * D + lane], mb = other[G * D + lane];
        const float M = fmaxf(ma, mb);
        const float base = M == -INFINITY ? 0.f : M;  // neither has a finite score
        fa = fast_exp2(ma - base);
        fb = fast_exp2(mb - base);
        mine[G * D + G + lane] = mine[G * D + G + lane] * fa + other[G * D + G + lane] * fb;
        mine[G * D + lane] = M;
      }
      // Compile-time bounds (rows padded to GROWS): the loads of all elements
      // issue back to back instead of one dependent step at a time.
#pragma unroll
      for (int j = 0; j < C::GROWS * D / 32; ++j) {
        const int r = (32 * j) / D;
        const float a0 = __shfl_sync(0xffffffffu, fa, r);
        const float b0 = __shfl_sync(0xffffffffu, fb, r);
        const int e = lane + 32 * j;
        if (r < G) mine[e] = mine[e] * a0 + other[e] * b0;
      }
      __syncwarp();
      if (k2 == 1) break;  // the chain starts in that warp
    }
    const int64_t seg_unit = slots.unit[warp][k];
    const int32_t nb = slots.nb[warp][k];
    if (seg_unit >= sp.r0 && seg_unit + nb <= sp.r1) {
      const OutRows<C::CHUNK> to(a, seq, kvh);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out);
      const float inv_l = lane < G ? 1.f / mine[G * D + G + lane] : 0.f;
#pragma unroll
      for (int j = 0; j < C::GROWS * D / 32; ++j) {
        const int r = (32 * j) / D;
        const float inv = __shfl_sync(0xffffffffu, inv_l, r);
        const int e = lane + 32 * j;
        if (r < to.rows) out[to.row(r, D) + e - r * D] = __float2bfloat16_rn(mine[e] * inv);
      }
    } else {
      cut(seq, kvh, seg_unit, nb, mine);
    }
  }
}

// Leaves a CTA's record of a segment that is cut across CTAs; the CTA that holds the
// segment's last unit lists it in `task`.
template <typename C, int D>
__device__ __forceinline__ void record_cut(const DecodeArgs& a, const Span& sp, int32_t seq,
                                           int32_t kvh, int64_t seg_unit, int32_t nb,
                                           const float* part, MergeTask& task) {
  const int lane = threadIdx.x & 31, G = a.groups;
  warp_store_record_fixed<C::GROWS, D>(a, sp, seg_unit, part, part + G * D, part + G * D + G, lane);
  if (lane == 0 && seg_unit < sp.r0 && seg_unit + nb <= sp.r1) {
    task.seg_unit = seg_unit;
    task.q = sp.q;
    task.rem = sp.rem;
    task.seq = seq;
    task.kvh = kvh;
    task.nb = nb;
    task.valid = 1;
  }
}

}  // namespace bsb
