// Tensor-core split-K decode attention over 4-bit pools (int4.cuh): bf16 queries, head_dim
// 64 or 128, block sizes that are multiples of 16, up to 16 query heads per kv head; the
// whole context, or a sliding window with sink tokens.
//
// The batch's units of 16 tokens are shared out as in decode_mma.cu: equal spans over the
// batch, or clusters per segment for few segments, with the same joins (decode_join.cuh).  A
// warp works through its span on its own, in steps of up to UNITS units of one segment; its
// lanes copy a step's codes and scales into a ring of S stages (cp.async, 16 bytes a lane),
// with the table entries of the step after it already on their way.
//
// The codes never pass through shared memory as bf16: they become the products' operands in
// registers, in the order in which the products take them,
//     S = Q K^T    Q the rows (16, the group's heads), K's codes the columns' operand: a lane
//                  takes the same quarter of the dims of one key per 8 keys, whatever their
//                  groups, and the query's fragments are laid out alike;
//     O^T = V^T P^T    V^T the rows' operand: one ldmatrix.trans brings a lane the codes of 4
//                  dims for two neighbouring keys in one register, so a shift and a mask leave
//                  the pair of one dim; P^T is S's accumulator as it is.
// A register of two values costs a shift (three of four), a mask and a fused multiply-add, 11
// instructions for 8 elements; all else together is less.  Stages are swizzled so that
// neither operand's loads meet in a bank.
#include "decode_join.cuh"
#include "int4.cuh"

namespace bsb {
namespace {

enum : int32_t { kFirst = 1, kLast = 2, kWhole = 4, kSlot1 = 8, kCount = 16 };  // units from bit 4

template <int D, bool G16>
struct Cfg {
  static constexpr int W = 4;      // warps per CTA
  static constexpr int S = 2;      // stages per warp
  static constexpr int UNITS = 2;  // units of a step
  static constexpr int MIN_CTAS = 3;
  static constexpr int GROWS = G16 ? 16 : 8;
  static constexpr int CODE_BYTES = kWindowUnit * D / 2;  // of a unit, K or V
  static constexpr int SCALE_BYTES = kWindowUnit * D / 16;
  static constexpr int Q_BYTES = GROWS * D * 2;
  // K codes | V codes | K scales | V scales, each of all units; the query.
  static constexpr int V_OFF = UNITS * CODE_BYTES;
  static constexpr int KS_OFF = 2 * UNITS * CODE_BYTES;
  static constexpr int VS_OFF = KS_OFF + UNITS * SCALE_BYTES;
  static constexpr int Q_OFF = VS_OFF + UNITS * SCALE_BYTES;
  static constexpr int STAGE_BYTES = Q_OFF + Q_BYTES;
  static constexpr int SLOT_FLOATS = GROWS * D + 2 * GROWS;
  static constexpr int SLOT0_BYTES = (SLOT_FLOATS * 4 + 127) / 128 * 128;
  static constexpr int SMEM_BYTES = W * S * STAGE_BYTES + W * SLOT0_BYTES;
  static_assert(STAGE_BYTES % 128 == 0, "stages stay 128-byte aligned");
  static_assert(SLOT_FLOATS * 4 <= S * STAGE_BYTES, "slot 1 must fit in the stages");
};

// What a stage holds.
template <int UNITS>
struct StepMeta {
  int32_t seq, kvh, nb, flags;
  int64_t seg_unit;
  int32_t map[UNITS];  // visible tokens of each unit
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int D, bool G16>
__global__ void __launch_bounds__(128, (Cfg<D, G16>::MIN_CTAS)) decode_int4_kernel(const DecodeArgs a) {
  using C = Cfg<D, G16>;
  constexpr int W = C::W, S = C::S, UNITS = C::UNITS;
  constexpr int NG = D / kInt4Group;  // groups of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ StepMeta<UNITS> meta[W][S];
  __shared__ ScanSmem scan;
  __shared__ WarpStarts starts;
  __shared__ WarpSlots<W> slots;
  __shared__ MergeTask task;  // the cut segment this CTA finishes

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* wst = smem + warp * S * C::STAGE_BYTES;
  if (tid < W * 2) slots.seq[tid / 2][tid % 2] = -1;
  if (tid == 0) task.valid = 0;
  pdl_wait();
  pdl_trigger();
  constexpr int kScratchInts = W * S * C::STAGE_BYTES / 4;
  int32_t own_seq = 0, own_kvh = 0, own_units = 0, ranks = 1;  // the cluster's segment
  const bool clustered = a.segment_ctas > 0;
  const Span sp =
      clustered ? segment_span<W>(a, starts, own_seq, own_kvh, own_units, ranks)
      : 2 * a.num_seqs <= kScratchInts
          ? compute_warp_spans_smem<W, true>(a, scan, starts, reinterpret_cast<int32_t*>(smem))
          : compute_warp_spans<W, true>(a, scan, starts);  // both sync the inits
  if (clustered && own_units == 0) return;  // no part in a segment
  if (sp.r0 >= sp.r1 && !clustered) {
    if (tid == 0) a.tasks[blockIdx.x].valid = 0;
    return;
  }

  const int G = a.groups;
  const int64_t Hkv = a.num_kv_heads;
  const int64_t spanw = sp.r1 - sp.r0;
  const int64_t wr0 = sp.r0 + spanw * warp / W;
  const int64_t wr1 = sp.r0 + spanw * (warp + 1) / W;

  // ---------------------------------------------------------------- issue cursor
  // The next step: its sequence, kv head and first unit.  All lanes keep identical copies.
  int32_t ci = starts.seq[warp];
  int64_t cprefix = starts.prefix[warp];
  int32_t clen = 0, crow = 0, cnb = 0, ch = 0, cb = 0;
  int32_t nxt_len = 0, nxt_row = 0;
  int64_t cu = wr0;
  WindowUnits cw{};
  if (wr1 > wr0) {
    cnb = units_of<true>(a, starts.len[warp], starts.row[warp], clen, crow);
    cw = window_units(a, clen);
    const int64_t rel = wr0 - cprefix * Hkv;
    ch = static_cast<int32_t>(rel / cnb);
    cb = static_cast<int32_t>(rel % cnb);
    nxt_len = starts.nlen[warp];
    nxt_row = starts.nrow[warp];
  }
  const int64_t block_bytes = static_cast<int64_t>(a.block_size) * int4_row_bytes(D);
  const int32_t scales_at = a.block_size * int4_code_bytes(D);  // of a block

  // The step prepared last: lane u < UNITS has unit u's token unit and table entry.
  int32_t step_units = 0, step_tu = 0, step_blk = -1;
  auto prepare = [&]() {
    step_units = static_cast<int32_t>(min(static_cast<int64_t>(min(UNITS, cnb - cb)), wr1 - cu));
    if (step_units <= 0) {
      step_units = 0;
      return;
    }
    if (lane < step_units) {
      const int32_t x = cb + lane;
      step_tu = x < cw.sink_units ? x : x - cw.sink_units + cw.first_unit;
      step_blk = __ldg(a.block_tables + static_cast<int64_t>(crow) * a.bt_stride +
                       (a.block_units == 1 ? step_tu : step_tu / a.block_units));
    }
  };
  // Starts the prepared step's copies into a stage and prepares the one after.
  auto issue = [&](int stage) {
    if (step_units == 0) return;
    const int32_t n = step_units;
    const uint32_t dst = smem_u32(wst + stage * C::STAGE_BYTES);
    const int64_t seg_unit = cprefix * Hkv + static_cast<int64_t>(ch) * cnb;
    const bool first = cu == wr0 || cb == 0;
    StepMeta<UNITS>& m = meta[warp][stage];
    if (lane == 0) {
      const bool last = cu + n == wr1 || cb + n == cnb;
      const bool whole = seg_unit >= wr0 && seg_unit + cnb <= wr1 && !(clustered && ranks > 1);
      m.seq = ci;
      m.kvh = ch;
      m.nb = cnb;
      m.seg_unit = seg_unit;
      m.flags = (first ? kFirst : 0) | (last ? kLast : 0) | (whole ? kWhole : 0) |
                (seg_unit > wr0 ? kSlot1 : 0) | n * kCount;
    }
    if (lane < n) {
      const bool valid = step_blk >= 0 && step_blk < a.num_blocks;
      if (!valid) set_status(a.status, kStatusBadBlock);
      const int32_t tok0 = step_tu * kWindowUnit, lo = clen - a.window;
      auto below = [](int32_t c) {  // map of a unit's first c tokens
        return c >= kWindowUnit ? 0xffff : c <= 0 ? 0 : (1 << c) - 1;
      };
      m.map[lane] = valid ? below(clen - tok0) & (~below(lo - tok0) | below(a.sinks - tok0)) : 0;
      if (!valid) step_blk = -1;
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int32_t blk = __shfl_sync(0xffffffffu, step_blk, u);
      const int32_t tu = __shfl_sync(0xffffffffu, step_tu, u);
      if (u >= n || blk < 0) continue;
      const int32_t tok = a.block_units == 1 ? 0 : tu % a.block_units * kWindowUnit;
      const int64_t block =
          (static_cast<int64_t>(ch) * a.num_blocks + blk) * block_bytes;
      const uint8_t* k = static_cast<const uint8_t*>(a.k_pool) + block;
      const uint8_t* v = static_cast<const uint8_t*>(a.v_pool) + block;
      // 16-byte piece c of row r lies at piece c ^ f(r) of its row: 8 rows of one piece, and 8
      // neighbouring pieces, are then in different banks.
#pragma unroll
      for (int i = 0; i < C::CODE_BYTES / 512; ++i) {
        const int id = lane + 32 * i;
        const int r = id / (D / 32), c = id % (D / 32);
        const uint32_t at = r * (D / 2) + ((D == 128 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1)) << 4);
        const int32_t from = tok * int4_code_bytes(D) + id * 16;
        copy16(dst + u * C::CODE_BYTES + at, k + from);
        copy16(dst + C::V_OFF + u * C::CODE_BYTES + at, v + from);
      }
      constexpr int kPieces = C::SCALE_BYTES / 16;
      if (lane < 2 * kPieces) {
        const int c = lane % kPieces;
        copy16(dst + (lane < kPieces ? C::KS_OFF : C::VS_OFF) + u * C::SCALE_BYTES + c * 16,
               (lane < kPieces ? k : v) + scales_at + tok * int4_scale_bytes(D) + c * 16);
      }
    }
    if (first) {
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) +
                               static_cast<int64_t>(ci) * a.q_stride_seq +
                               static_cast<int64_t>(ch) * G * D;
      for (int e = lane; e < G * D / 8; e += 32) copy16(dst + C::Q_OFF + e * 16, q + e * 8);
    }
    // On to the next step.
    cu += n;
    cb += n;
    if (cu < wr1 && cb == cnb) {
      cb = 0;
      if (++ch == Hkv) {
        ch = 0;
        cprefix += cnb;
        ++ci;
        cnb = ci < a.num_seqs ? units_of<true>(a, nxt_len, nxt_row, clen, crow) : 1;
        while (cnb == 0) {  // empty or invalid sequences own no units
          ++ci;
          cnb = ci < a.num_seqs ? seq_units<true>(a, ci, clen, crow, false) : 1;
        }
        cw = window_units(a, max(clen, 0));
        if (ci + 1 < a.num_seqs) {
          nxt_len = __ldg(a.context_lens + ci + 1);
          nxt_row = a.seq_rows != nullptr ? __ldg(a.seq_rows + ci + 1) : ci + 1;
        }
      }
    }
    prepare();
  };

  prepare();
#pragma unroll
  for (int s = 0; s < S; ++s) {
    issue(s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // ---------------------------------------------------------------- compute
  const int g = lane >> 2, t = lane & 3;
  constexpr int WORDS = D / 32;  // words of codes a lane takes of a key
  uint32_t qa[WORDS][4], qb[G16 ? WORDS : 1][4];  // query rows g, g + 8
  float o[NG][2][4], o2[G16 ? NG : 1][2][4];      // O^T of query columns 0 .. 7, 8 .. 15
  float m2[2] = {-INFINITY, -INFINITY}, lsum[2] = {0.f, 0.f};
  const float zscale = a.scale * kLog2e;
  int32_t left = static_cast<int32_t>(wr1 - wr0);

  for (int stage = 0; left > 0; stage = stage + 1 == S ? 0 : stage + 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    __syncwarp();
    const StepMeta<UNITS>& mt = meta[warp][stage];
    const int32_t flags = mt.flags, n = flags / kCount;
    const uint8_t* st = wst + stage * C::STAGE_BYTES;
    const uint32_t base = smem_u32(st);
    left -= n;
    if (flags & kFirst) {
      m2[0] = m2[1] = -INFINITY;
      lsum[0] = lsum[1] = 0.f;
#pragma unroll
      for (int q = 0; q < NG; ++q) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[q][j][e] = 0.f;
            if (G16) o2[q][j][e] = 0.f;
          }
        }
      }
      // Lane t's dims: a quarter of the row's.
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        const uint4* src = reinterpret_cast<const uint4*>(st + C::Q_OFF) + t * WORDS + w;
        const uint4 x = g < G ? src[g * (D / 8)] : zero;
        qa[w][0] = x.x; qa[w][1] = x.y; qa[w][2] = x.z; qa[w][3] = x.w;
        if (G16) {
          const uint4 y = g + 8 < G ? src[(g + 8) * (D / 8)] : zero;
          qb[w][0] = y.x; qb[w][1] = y.y; qb[w][2] = y.z; qb[w][3] = y.w;
        }
      }
    }
    // S = Q K^T, 8 keys at a time.
    float s[2 * UNITS][4];
    bool all = true;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float(&acc)[4] = s[2 * u + j];
        acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
        if (u >= n) continue;
        const int r = 8 * j + g;
        const uint32_t row = base + u * C::CODE_BYTES + r * (D / 2);
        uint32_t w[WORDS], group;
        if constexpr (D == 128) {
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(row + ((t ^ ((r >> 1) & 3)) << 4)));
          group = t;
        } else {
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                       : "=r"(w[0]), "=r"(w[1])
                       : "r"(row + (((t >> 1) ^ ((r >> 2) & 1)) << 4) + (t & 1) * 8));
          group = t >> 1;
        }
        const uint32_t bits = *reinterpret_cast<const uint16_t*>(
            st + C::KS_OFF + u * C::SCALE_BYTES + (r * NG + group) * 2);
        const uint32_t scale = bits | (bits << 16), shift = int4_shift(scale);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          uint32_t v[4];
          int4_values(w[i], scale, shift, v);
          const uint32_t a0[4] = {qa[i][0], G16 ? qb[G16 ? i : 0][0] : 0u, qa[i][1],
                                  G16 ? qb[G16 ? i : 0][1] : 0u};
          const uint32_t a1[4] = {qa[i][2], G16 ? qb[G16 ? i : 0][2] : 0u, qa[i][3],
                                  G16 ? qb[G16 ? i : 0][3] : 0u};
          mma_bf16_16816(acc, a0, v[0], v[1]);
          mma_bf16_16816(acc, a1, v[2], v[3]);
        }
      }
      all = all && u < n && mt.map[u] == 0xffff;
    }
    // Scores in base 2; unseen tokens -inf.
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int x = 0; x < 2 * UNITS; ++x) {
      const int32_t map = all ? 0xffff : x / 2 < n ? mt.map[x / 2] : 0;
#pragma unroll
      for (int e = 0; e < (G16 ? 4 : 2); ++e) {
        float v = __fmul_rn(s[x][e], zscale);
        if (!all && !((map >> (8 * (x & 1) + 2 * t + (e & 1))) & 1)) v = -INFINITY;
        s[x][e] = v;
        mx[e >> 1] = fmaxf(mx[e >> 1], v);
      }
    }
    float corr[2] = {1.f, 1.f};
#pragma unroll
    for (int hr = 0; hr < (G16 ? 2 : 1); ++hr) {
      float m = mx[hr];
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const float mtop = fmaxf(m2[hr], m);
      const float mnew = mtop == -INFINITY ? 0.f : mtop;  // no token yet (no -inf - -inf)
      corr[hr] = fast_exp2(m2[hr] - mnew);
      m2[hr] = mtop;
      float ps = 0.f;
#pragma unroll
      for (int x = 0; x < 2 * UNITS; ++x) {
        const float p0 = fast_exp2(s[x][2 * hr] - mnew), p1 = fast_exp2(s[x][2 * hr + 1] - mnew);
        s[x][2 * hr] = p0;
        s[x][2 * hr + 1] = p1;
        ps += p0 + p1;
      }
      lsum[hr] = lsum[hr] * corr[hr] + ps;
    }
    // The rows' factors belong to this lane's columns 2t, 2t + 1.
    if (__any_sync(0xffffffffu, corr[0] != 1.f || (G16 && corr[1] != 1.f))) {
#pragma unroll
      for (int hr = 0; hr < (G16 ? 2 : 1); ++hr) {
        const float f0 = __shfl_sync(0xffffffffu, corr[hr], 8 * t);
        const float f1 = __shfl_sync(0xffffffffu, corr[hr], 8 * t + 4);
#pragma unroll
        for (int q = 0; q < NG; ++q) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float(&acc)[4] = hr == 0 ? o[q][j] : o2[G16 ? q : 0][j];
            acc[0] *= f0;
            acc[1] *= f1;
            acc[2] *= f0;
            acc[3] *= f1;
          }
        }
      }
    }
    // O^T += V^T P^T, 16 keys at a time.
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (u >= n) continue;
      const uint32_t p0 = pack_bf16x2(s[2 * u][0], s[2 * u][1]);
      const uint32_t p1 = pack_bf16x2(s[2 * u + 1][0], s[2 * u + 1][1]);
      const uint32_t p2 = G16 ? pack_bf16x2(s[2 * u][2], s[2 * u][3]) : 0u;
      const uint32_t p3 = G16 ? pack_bf16x2(s[2 * u + 1][2], s[2 * u + 1][3]) : 0u;
      // Scales of keys 2t, 2t + 1 and 2t + 8, 2t + 9, pairs of groups in a register.
      const uint32_t* sv =
          reinterpret_cast<const uint32_t*>(st + C::VS_OFF + u * C::SCALE_BYTES);
      uint32_t keep_lo = 0xffffffffu, keep_hi = 0xffffffffu;
      if (!all) {  // scales of unseen tokens become 0: their codes may be stale, scales NaN
        const int32_t map = mt.map[u];
        auto pair = [&](int tok) {
          return (((map >> tok) & 1) ? 0x0000ffffu : 0u) |
                 (((map >> (tok + 1)) & 1) ? 0xffff0000u : 0u);
        };
        keep_lo = pair(2 * t);
        keep_hi = pair(2 * t + 8);
      }
      uint32_t sc[4][NG / 2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = 2 * t + (k & 1) + 8 * (k >> 1);
#pragma unroll
        for (int i = 0; i < NG / 2; ++i) sc[k][i] = sv[key * (NG / 2) + i];
      }
      const int r = 8 * ((lane >> 3) & 1) + (lane & 7);
#pragma unroll
      for (int q0 = 0; q0 < NG; q0 += 2) {
        const int q = q0 + (lane >> 4);  // the group whose row this lane points at
        const uint32_t piece = D == 128 ? q ^ ((r >> 1) & 3) : q ^ ((r >> 2) & 1);
        uint32_t c[4];
        ldmatrix_x4_trans(base + C::V_OFF + u * C::CODE_BYTES + r * (D / 2) + (piece << 4), c[0],
                          c[1], c[2], c[3]);
#pragma unroll
        for (int qq = 0; qq < 2; ++qq) {
          const uint32_t sel = qq == 0 ? 0x5410 : 0x7632;
          const uint32_t s_lo = __byte_perm(sc[0][q0 / 2], sc[1][q0 / 2], sel) & keep_lo;
          const uint32_t s_hi = __byte_perm(sc[2][q0 / 2], sc[3][q0 / 2], sel) & keep_hi;
          uint32_t lo[4], hi[4];  // dim i of the lane's four, keys (2t, 2t + 1), (2t + 8, 2t + 9)
          int4_values(c[2 * qq], s_lo, int4_shift(s_lo), lo);
          int4_values(c[2 * qq + 1], s_hi, int4_shift(s_hi), hi);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t av[4] = {lo[2 * j], lo[2 * j + 1], hi[2 * j], hi[2 * j + 1]};
            mma_bf16_16816(o[q0 + qq][j], av, p0, p1);
            if (G16) mma_bf16_16816(o2[G16 ? q0 + qq : 0][j], av, p2, p3);
          }
        }
      }
    }
    // The stage has been read: refill it with the step S positions ahead.
    __syncwarp();
    const int32_t seq = mt.seq, kvh = mt.kvh, nb = mt.nb;
    const int64_t seg_unit = mt.seg_unit;
    __syncwarp();
    issue(stage);
    asm volatile("cp.async.commit_group;" ::: "memory");

    if (flags & kLast) {
      float lrow[2];
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        float l = lsum[hr];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        lrow[hr] = l;
      }
      const bool whole = (flags & kWhole) != 0;
      const int slot_of = (flags & kSlot1) ? 1 : 0;
      float* slot = warp_slot<C>(smem, warp, slot_of);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) +
                           static_cast<int64_t>(seq) * a.o_stride_seq +
                           static_cast<int64_t>(kvh) * G * D;
      // Neighbouring lanes (g, g ^ 1) hold the dims 2k and 2k + 1: each takes both dims of one
      // of the two query rows.
      const int odd = g & 1;
#pragma unroll
      for (int hr = 0; hr < (G16 ? 2 : 1); ++hr) {
        const int row = 8 * hr + 2 * t + odd;
        const float inv = whole ? 1.f / __shfl_sync(0xffffffffu, lrow[hr], 8 * t + 4 * odd) : 1.f;
#pragma unroll
        for (int q = 0; q < NG; ++q) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float(&acc)[4] = hr == 0 ? o[q][i / 2] : o2[G16 ? q : 0][i / 2];
            const float x0 = acc[2 * (i & 1)], x1 = acc[2 * (i & 1) + 1];  // rows 2t, 2t + 1
            const float got = __shfl_xor_sync(0xffffffffu, odd ? x0 : x1, 4);
            const float lo = (odd ? got : x0) * inv, hi = (odd ? x1 : got) * inv;
            const int dim = 32 * q + 8 * (g >> 1) + 2 * i;
            if (row < G) {
              if (whole) {
                *reinterpret_cast<uint32_t*>(out + row * D + dim) = pack_bf16x2(lo, hi);
              } else {
                *reinterpret_cast<float2*>(slot + row * D + dim) = make_float2(lo, hi);
              }
            }
          }
        }
        if (!whole && t == 0 && 8 * hr + g < G) {
          slot[G * D + 8 * hr + g] = m2[hr];
          slot[G * D + G + 8 * hr + g] = lrow[hr];
        }
      }
      if (!whole && lane == 0) {
        slots.seq[warp][slot_of] = seq;
        slots.kvh[warp][slot_of] = kvh;
        slots.nb[warp][slot_of] = nb;
        slots.unit[warp][slot_of] = seg_unit;
      }
      __syncwarp();
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  if (clustered) {
    join_segment<C, D>(a, smem, slots, own_seq, own_kvh, ranks);
    return;
  }
  fold_slots<C, D>(a, smem, sp, spanw, slots, [&](int32_t seq, int32_t kvh, int64_t seg_unit,
                                                  int32_t nb, const float* part) {
    record_cut<C, D>(a, sp, seq, kvh, seg_unit, nb, part, task);
  });
  __syncthreads();
  if (tid == 0) a.tasks[blockIdx.x] = task;
}

template <int D, bool G16>
cudaError_t allow_smem() {
  static unsigned long long configured = 0;  // one bit per device
  return once_per_device(&configured, [] {
    return cudaFuncSetAttribute(decode_int4_kernel<D, G16>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Cfg<D, G16>::SMEM_BYTES);
  });
}

template <int D, bool G16>
int launch_one(const DecodeArgs& a, int grid, cudaStream_t stream) {
  using C = Cfg<D, G16>;
  cudaError_t e = allow_smem<D, G16>();
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(C::W * 32);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.segment_ctas > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.segment_ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return static_cast<int>(cudaLaunchKernelEx(&cfg, decode_int4_kernel<D, G16>, a));
}

template <int D, bool G16>
int occupancy_one() {
  using C = Cfg<D, G16>;
  int n = 0;
  cudaError_t e = allow_smem<D, G16>();
  if (e == cudaSuccess) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, decode_int4_kernel<D, G16>, C::W * 32,
                                                      C::SMEM_BYTES);
  }
  return e != cudaSuccess ? -static_cast<int>(e) : n;
}

}  // namespace

int launch_decode_int4(const DecodeArgs& a, int grid, cudaStream_t stream) {
  const bool g16 = a.groups > 8;
  int rc;
  if (a.head_dim == 64) {
    rc = g16 ? launch_one<64, true>(a, grid, stream) : launch_one<64, false>(a, grid, stream);
  } else {
    rc = g16 ? launch_one<128, true>(a, grid, stream) : launch_one<128, false>(a, grid, stream);
  }
  if (rc != 0 || a.tasks == nullptr) return rc;
  return launch_decode_merge(a, grid, stream);
}

int decode_int4_ctas_per_sm(int head_dim, int groups) {
  const bool g16 = groups > 8;
  if (head_dim == 64) return g16 ? occupancy_one<64, true>() : occupancy_one<64, false>();
  return g16 ? occupancy_one<128, true>() : occupancy_one<128, false>();
}

}  // namespace bsb
