// Tensor-core split-K decode attention over 4-bit pools (int4.cuh): bf16 queries, head_dim
// 64 or 128, block sizes that are multiples of 16, up to 16 query heads per kv head; the
// whole context, or a sliding window with sink tokens.
//
// The batch's units of 16 tokens are shared out as in decode_mma.cu: equal spans over the
// batch, or clusters per segment for few segments, with the same joins (decode_join.cuh).  A
// warp works through its span on its own, a unit at a time; its lanes copy a unit's codes and
// scales into a ring of S stages (cp.async, 16 bytes a lane), with the table entries of up to
// 32 units in a register of each lane and those of the next already on their way.
//
// The codes never pass through shared memory as bf16: they become the products' operands in
// registers, in the order in which the products take them,
//     S^T = K Q^T    K the rows' operand (16 keys): a lane takes the same quarter of the dims
//                    of two keys, whatever their groups, and the query's fragments are laid
//                    out alike;
//     O^T = V^T P^T  V^T the rows' operand: one ldmatrix.trans brings a lane the codes of 4
//                    dims for two neighbouring keys in one register, so a shift and a mask
//                    leave the pair of one dim; P^T is S^T, its 8 x 8 tiles transposed.
// So no row of either product is padding for up to 8 heads, and the softmax's factors belong
// to O's columns as they are.  A register of two values costs a shift (three of four), a mask
// and a fused multiply-add, 11 instructions for 8 elements; all else together is less.  Stages
// are swizzled so that neither operand's loads meet in a bank.
//
// Scores are weighed against a maximum that moves only when one is more than 2^8 above it
// (then all lanes find the new one and O is scaled): most units need no reduction.
//
// Weights are rounded to bf16, the products' type (2^-9 of each; their sum takes them
// unrounded); scores, maxima, sums and O are fp32.
//
// Chunks of up to 16 rows, tokens times heads, run here as well (CHUNK): a chunk is a sequence
// whose rows are its tokens' heads; only units that some token does not see whole are masked
// row by row.  chunk_rows_kernel lists them ahead.
//
// 256 sequences of 512 to 32768 tokens (log-uniform), 28 + 4 heads of 128, 1.05 GB of codes and
// scales: 280 us, 3.8 TB/s, 57% of a plain copy's rate.  What bounds it is latency inside a
// warp: codes, operands, scores, weights and second product follow one another, 340
// instructions for 16 tokens of 128 dims, half of them what turns codes into operands, and
// three warps a scheduler issue 2.2 of 4 a clock and SM (DRAM 40% busy).  64 sequences of 1 to
// 16384, 14 + 2 heads of 64: 24 us (floor 1.9): launch, search of the spans, table entries,
// codes and joins follow one another for 5.9 units a warp (10426 on 444 CTAs), and the
// merge behind them.  One sequence of 77: 5.4 us.  The pools as bf16 (window attention's
// decode): 43 us for 64 of 1 to 8192 at d64, 37 here; at d128 111 and 68.
// Not kept: a join by all threads of CTAs that hold one segment only (the same time).
#include <type_traits>

#include "decode_join.cuh"
#include "int4.cuh"
#include "window.cuh"

namespace bsb {
namespace {

// Of a step (4 bits): there is one; a portion's first or last one; it has all its units and
// their tokens are all visible.
enum : uint32_t { kFirst = 1, kLast = 2, kFull = 4, kStep = 8 };
// Of a portion: the segment is all the warp's; it goes to slot 1.
enum : int32_t { kWhole = 1, kSlot1 = 2 };
constexpr float kSlack = 8.f;  // how far above the maximum a score may be, base 2
constexpr float kNoScore = -3.402823466e38f;  // the maximum before any score: no finite one is below

// NQ tiles of 8 query rows, one or two; CHUNK_: rows of several tokens.
template <int D, int NQ, bool CHUNK_>
struct Cfg {
  static constexpr bool CHUNK = CHUNK_;
  static constexpr int W = 4;                    // warps per CTA
  static constexpr int U = 2;                    // units of a step (with one: 72 for 66, 289 for 268 us)
  static constexpr int S = D == 64 ? 4 : 3;      // stages per warp, a step each
  // CTAs per SM.  us with one more / these / one fewer, 256 sequences of 2048, d64, one tile of
  // rows: 49 / 45 / --, two: 55 / 53 / --; d128, one: (spills) / 96 / 98, two: -- / 121 / 123.
  static constexpr int MIN_CTAS = 4 - NQ;
  static constexpr int GROWS = 8 * NQ;
  static constexpr int CODE_BYTES = kWindowUnit * D / 2;  // of a unit, K or V
  static constexpr int SCALE_BYTES = kWindowUnit * D / 16;
  // A unit in a stage: K codes | V codes | K scales | V scales.
  static constexpr int KS_OFF = 2 * CODE_BYTES;
  static constexpr int VS_OFF = KS_OFF + SCALE_BYTES;
  static constexpr int UNIT_BYTES = VS_OFF + SCALE_BYTES;
  static constexpr int STAGE_BYTES = U * UNIT_BYTES;
  static constexpr int SLOT_FLOATS = GROWS * D + 2 * GROWS;
  static constexpr int SLOT0_BYTES = (SLOT_FLOATS * 4 + 127) / 128 * 128;
  static constexpr int SMEM_BYTES = W * S * STAGE_BYTES + W * SLOT0_BYTES;
  static_assert(STAGE_BYTES % 128 == 0, "stages stay 128-byte aligned");
  static_assert(SLOT_FLOATS * 4 <= S * STAGE_BYTES, "slot 1 must fit in the stages");
  static_assert(S <= 8, "a stage has 4 bits of the flags");
};

// Whose a run of units is.
struct Owner {
  int32_t seq, kvh, nb, flags;
  int64_t seg_unit;
};

// Of chunks also: its length, first query token and tokens.
struct ChunkOwner : Owner {
  int32_t len, tok0, tokens;
};

// What a stage holds: the visible tokens of a step that does not show them all (16 bits a
// unit), and whose it is of a portion's first and last ones.
struct StepMeta {
  uint32_t map;
  Owner owner;
};
struct ChunkMeta {
  uint32_t map;
  int32_t first[2];  // positions of the units' first tokens
  ChunkOwner owner;
};

// Up to 32 consecutive units of a segment, one per lane.
struct Run {
  int32_t n;
  uint32_t flags;  // kFirst, kLast: a portion's first, its last units
  int32_t blk;       // this lane's: block-table entry, unit of its block, visible tokens
  int32_t in_block, map;
  int32_t first;  // chunks: position of its first token
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// The 8 x 8 tile of 16-bit elements that a warp holds, a row to four lanes, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// D = A * B, as mma_bf16_16816.
__device__ __forceinline__ void mma_zero_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

template <int D, int NQ, bool CHUNK>
__global__ void __launch_bounds__(128, (Cfg<D, NQ, CHUNK>::MIN_CTAS))
    decode_int4_kernel(const DecodeArgs a) {
  using C = Cfg<D, NQ, CHUNK>;
  using Whose = std::conditional_t<CHUNK, ChunkOwner, Owner>;
  using Meta = std::conditional_t<CHUNK, ChunkMeta, StepMeta>;
  constexpr int W = C::W, S = C::S, U = C::U;
  constexpr int NG = D / kInt4Group;  // groups of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Meta meta[W][S];
  __shared__ Whose owners[W][2];  // of the current run and the one behind it
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

  const int G = a.groups, heads = CHUNK ? a.chunk_heads : G;
  const int64_t Hkv = a.num_kv_heads;
  const int64_t spanw = sp.r1 - sp.r0;
  const int64_t wr0 = sp.r0 + spanw * warp / W;
  const int64_t wr1 = sp.r0 + spanw * (warp + 1) / W;

  // ---------------------------------------------------------------- fetch cursor
  // The next run's sequence, kv head and first unit.  All lanes keep identical copies.
  int32_t ci = starts.seq[warp];
  int64_t cprefix = starts.prefix[warp];
  int32_t clen = 0, crow = 0, cnb = 0, ch = 0, cb = 0;
  int32_t nxt_len = 0, nxt_row = 0;
  int32_t togo = static_cast<int32_t>(wr1 - wr0);  // units that are not in a run yet
  bool begins = true;                              // the next run is its portion's first
  int parity = 0;
  if (togo > 0) {
    cnb = units_of<true>(a, starts.len[warp], starts.row[warp], clen, crow);
    const int64_t rel = wr0 - cprefix * Hkv;
    ch = static_cast<int32_t>(rel / cnb);
    cb = static_cast<int32_t>(rel % cnb);
    nxt_len = starts.nlen[warp];
    nxt_row = starts.nrow[warp];
  }
  // Loads the next run's table entries and moves the cursor past it.
  auto fetch = [&]() {
    Run r{};
    r.n = min(min(32, cnb - cb), togo);
    if (r.n <= 0) {
      r.n = 0;
      return r;
    }
    const WindowUnits cw = window_units(a, clen);
    const int32_t x = cb + lane;
    const int32_t tu = x < cw.sink_units ? x : x - cw.sink_units + cw.first_unit;
    r.blk = -1;
    if (lane < r.n) {
      const int32_t ent = a.block_units == 1 ? tu : tu / a.block_units;
      r.in_block = tu - ent * a.block_units;
      r.blk = __ldg(a.block_tables + static_cast<int64_t>(crow) * a.bt_stride + ent);
    }
    const int32_t tok0 = tu * kWindowUnit;
    int2 tokens{};
    if constexpr (CHUNK) tokens = coherent_load(a.chunk_rows + ci);
    // What the last token sees, or any of them.
    const int32_t lo = CHUNK ? clen - a.chunk_window - (tokens.y - 1) : clen - a.window;
    auto below = [](int32_t c) {  // map of a unit's first c tokens
      return c >= kWindowUnit ? 0xffff : c <= 0 ? 0 : (1 << c) - 1;
    };
    r.map = below(clen - tok0) & (~below(lo - tok0) | below(a.sinks - tok0));
    if constexpr (CHUNK) {  // (bit 16: all of them see all of it)
      r.first = tok0;
      if (tok0 + kWindowUnit <= clen - (tokens.y - 1) &&
          (tok0 >= clen - a.chunk_window || tok0 + kWindowUnit <= a.sinks)) {
        r.map |= 0x10000;
      }
    }
    togo -= r.n;
    cb += r.n;
    const bool ends = togo == 0 || cb == cnb;
    r.flags = (begins ? kFirst : 0u) | (ends ? kLast : 0u);
    if (lane == 0) {
      const int64_t seg_unit = cprefix * Hkv + static_cast<int64_t>(ch) * cnb;
      Whose& w = owners[warp][parity];
      w.seq = ci;
      w.kvh = ch;
      w.nb = cnb;
      w.seg_unit = seg_unit;
      w.flags = (seg_unit >= wr0 && seg_unit + cnb <= wr1 && !(clustered && ranks > 1) ? kWhole : 0) |
                (seg_unit > wr0 ? kSlot1 : 0);
      if constexpr (CHUNK) {
        w.len = clen;
        w.tok0 = tokens.x;
        w.tokens = tokens.y;
      }
    }
    parity ^= 1;
    begins = ends;
    if (togo > 0 && cb == cnb) {
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
        if (ci + 1 < a.num_seqs) {
          nxt_len = coherent_load(a.context_lens + ci + 1);
          nxt_row = a.seq_rows != nullptr ? coherent_load(a.seq_rows + ci + 1) : ci + 1;
        }
      }
    }
    return r;
  };

  // ---------------------------------------------------------------- issue
  const int32_t block_bytes = a.block_size * int4_row_bytes(D);  // fits (host)
  const int32_t scales_at = a.block_size * int4_code_bytes(D);   // of a block
  const int64_t head_bytes = static_cast<int64_t>(a.num_blocks) * block_bytes;
  // This lane's pieces of a unit: where they are in a block and in a stage.  16-byte piece c
  // of row r lies at piece c ^ f(r) of its row: 8 rows of one piece, and 8 neighbouring
  // pieces, are then in different banks.
  const int lr = lane / (D / 32), lc = lane % (D / 32);
  const uint32_t piece_at =
      lr * (D / 2) + ((D == 128 ? lc ^ ((lr >> 1) & 3) : lc ^ ((lr >> 2) & 1)) << 4);
  constexpr int kScalePieces = C::SCALE_BYTES / 16;
  const uint8_t* const k_codes = static_cast<const uint8_t*>(a.k_pool) + lane * 16;
  const uint8_t* const v_codes = static_cast<const uint8_t*>(a.v_pool) + lane * 16;
  const uint8_t* const scales = static_cast<const uint8_t*>(lane < kScalePieces ? a.k_pool : a.v_pool) +
                                scales_at + (lane % kScalePieces) * 16;  // K's lanes, V's lanes

  Run cur = fetch(), nxt{};
  int32_t idx = 0;     // next unit of the current run: it and the one behind it are a step
  uint32_t full = 0;   // its units whose tokens are all visible
  int64_t head_at = 0;
  const Whose* owner = nullptr;
  auto begin_run = [&]() {
    if (cur.n == 0) return;
    const bool valid = cur.blk >= 0 && cur.blk < a.num_blocks;
    // (Units that the window of a longer group would reach may have no block any more.)
    if (lane < cur.n && !valid && (!CHUNK || cur.map != 0)) set_status(a.status, kStatusBadBlock);
    if (!valid) cur.blk = cur.map = 0;  // any block will do: none of its tokens counts
    full = __ballot_sync(0xffffffffu, lane < cur.n && cur.map == (CHUNK ? 0x1ffff : 0xffff));
    owner = &owners[warp][parity ^ 1];
    const int32_t kvh = owner->kvh;
    head_at = kvh * head_bytes;
    if (cur.flags & kFirst) {  // the query will be wanted: into L1
      int32_t first = owner->seq, tokens = 1;
      if constexpr (CHUNK) {
        first = owner->tok0;
        tokens = owner->tokens;
      }
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + first * a.q_stride_seq +
                               static_cast<int64_t>(kvh) * heads * D + lane * 64;
      for (int32_t j = 0; j < tokens; ++j) {
        if (lane * 64 < heads * D) {
          asm volatile("prefetch.global.L1 [%0];" ::"l"(q + j * a.q_stride_seq));
        }
      }
    }
    idx = 0;
    nxt = fetch();
  };
  __syncwarp();
  begin_run();
  // Starts the next step's copies into the stage at `dst` and returns its flags.
  auto issue = [&](uint32_t dst, int stage) -> uint32_t {
    uint32_t flags = 0;
    if (cur.n != 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int from = min(idx + u, cur.n - 1);  // (a step past the end repeats the last unit)
        const int32_t blk = __shfl_sync(0xffffffffu, cur.blk, from);
        int64_t at = head_at + static_cast<int64_t>(blk) * block_bytes, scales_from = at;
        if (a.block_units != 1) {
          const int32_t tok = __shfl_sync(0xffffffffu, cur.in_block, from) * kWindowUnit;
          at += tok * int4_code_bytes(D);
          scales_from += tok * int4_scale_bytes(D);
        }
        const uint8_t* k = k_codes + at;
        const uint8_t* v = v_codes + at;
        const uint32_t to = dst + u * C::UNIT_BYTES;
#pragma unroll
        for (int i = 0; i < C::CODE_BYTES / 512; ++i) {  // (8 rows on: the same swizzle)
          copy16(to + piece_at + i * 512, k + i * 512);
          copy16(to + piece_at + C::CODE_BYTES + i * 512, v + i * 512);
        }
        if (lane < 2 * kScalePieces) copy16(to + lane * 16 + C::KS_OFF, scales + scales_from);
      }
      const uint32_t every = (1u << U) - 1u;
      flags = kStep | (((full >> idx) & every) == every ? kFull : 0u);
      if (idx == 0) flags |= cur.flags & kFirst;
      if (idx + U >= cur.n) flags |= cur.flags & kLast;
      if (flags != (kStep | kFull)) {
        uint32_t seen = __shfl_sync(0xffffffffu, cur.map, idx);
        const uint32_t second = __shfl_sync(0xffffffffu, cur.map, idx + 1);
        if constexpr (CHUNK) seen &= 0xffffu;
        if (idx + 1 < cur.n) seen |= second << 16;
        int32_t first[2];
        if constexpr (CHUNK) {
          first[0] = __shfl_sync(0xffffffffu, cur.first, idx);
          first[1] = __shfl_sync(0xffffffffu, cur.first, idx + 1);
        }
        if (lane == 0) {
          Meta& m = meta[warp][stage];
          m.map = seen;
          if (CHUNK || (flags & (kFirst | kLast))) m.owner = *owner;
          if constexpr (CHUNK) {
            m.first[0] = first[0];
            m.first[1] = first[1];
          }
        }
        __syncwarp();  // the owner has been read
      }
      idx += U;
      if (idx >= cur.n) {
        cur = nxt;
        begin_run();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return flags;
  };

  // ---------------------------------------------------------------- compute
  const int g = lane >> 2, t = lane & 3;
  constexpr int WORDS = D / 32;     // words of codes a lane takes of a key
  uint32_t qf[NQ][WORDS][4];        // query rows g, g + 8: lane t's quarter of the dims
  float o[NQ][NG][2][4];            // O^T, columns 2t, 2t + 1 (+ 8)
  float m2[NQ][2], lsum[NQ][2];     // of the same columns
  const float zscale = a.scale * kLog2e;
  const uint32_t ring = smem_u32(wst);
  uint32_t queue = 0;  // flags of the steps in the stages, the oldest in the lowest bits
  // Of a unit's part of a stage, this lane's: K codes, K scale, V codes (as ldmatrix wants
  // them), V scales.
  const uint32_t k_at = g * (D / 2) + (D == 128 ? (t ^ ((g >> 1) & 3)) << 4
                                                : (((t >> 1) ^ ((g >> 2) & 1)) << 4) + (t & 1) * 8);
  const uint32_t ks_at = C::KS_OFF + (g * NG + (D == 128 ? t : t >> 1)) * 2;
  const int vr = 8 * ((lane >> 3) & 1) + (lane & 7);
  const uint32_t v_at = C::CODE_BYTES + vr * (D / 2) +
                        (((lane >> 4) ^ (D == 128 ? (vr >> 1) & 3 : (vr >> 2) & 1)) << 4);
  const uint32_t vs_at = C::VS_OFF + 2 * t * (NG * 2);

  // The first S turns only fill the stages.
  int stage = 0;
#pragma unroll 1
  for (int it = -S;; it = min(it + 1, 0)) {
    const uint32_t base = ring + stage * C::STAGE_BYTES;
    if (it >= 0) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
      __syncwarp();
      const uint32_t flags = queue & 15u;
      if (flags == 0) break;
      const Meta& mt = meta[warp][stage];
      float bias[U][2];  // of keys g, g + 8 of each unit: -inf where the token is not seen
#pragma unroll
      for (int u = 0; u < U; ++u) bias[u][0] = bias[u][1] = 0.f;
      if (flags != (kStep | kFull)) {
        if (flags & kFirst) {
          int32_t first = mt.owner.seq, rows = G;
          if constexpr (CHUNK) {
            first = mt.owner.tok0;
            rows = mt.owner.tokens * heads;
          }
          const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) +
                                   first * a.q_stride_seq +
                                   static_cast<int64_t>(mt.owner.kvh) * heads * D + t * (D / 4);
#pragma unroll
          for (int h = 0; h < NQ; ++h) {
            m2[h][0] = m2[h][1] = kNoScore;
            lsum[h][0] = lsum[h][1] = 0.f;
#pragma unroll
            for (int x = 0; x < NG; ++x) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[h][x][j][e] = 0.f;
              }
            }
            const int32_t row = g + 8 * h, token = CHUNK ? row / heads : 0;
            const __nv_bfloat16* from =
                q + token * (CHUNK ? a.q_stride_seq : 0) + (row - token * heads) * D;
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
              uint4 x = make_uint4(0u, 0u, 0u, 0u);
              if (row < rows) x = *reinterpret_cast<const uint4*>(from + w * 8);
              qf[h][w][0] = x.x;
              qf[h][w][1] = x.y;
              qf[h][w][2] = x.z;
              qf[h][w][3] = x.w;
            }
          }
        }
        if (!(flags & kFull)) {
          // Unseen tokens: their codes may be stale, their scales NaN; with scales of 0 they
          // are 0.
          const uint32_t seen = mt.map;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            uint16_t* scale = reinterpret_cast<uint16_t*>(wst + stage * C::STAGE_BYTES +
                                                          u * C::UNIT_BYTES + C::KS_OFF);
            for (int e = lane; e < 2 * kWindowUnit * NG; e += 32) {
              if (!((seen >> (16 * u + e / NG % kWindowUnit)) & 1)) scale[e] = 0;
            }
            if (!((seen >> (16 * u + g)) & 1)) bias[u][0] = -INFINITY;
            if (!((seen >> (16 * u + g + 8)) & 1)) bias[u][1] = -INFINITY;
          }
          __syncwarp();
        }
      }
      // S^T = K Q^T: keys g and g + 8 of each unit, in two chains.
      float s[U][NQ][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t unit = base + u * C::UNIT_BYTES;
        uint32_t kw[2][WORDS], ks[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t from = unit + k_at + r * 8 * (D / 2);  // (key g + 8 has key g's swizzle)
          if constexpr (D == 128) {
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(kw[r][0]), "=r"(kw[r][1]), "=r"(kw[r][2]), "=r"(kw[r][3])
                         : "r"(from));
          } else {
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                         : "=r"(kw[r][0]), "=r"(kw[r][1])
                         : "r"(from));
          }
          uint16_t bits;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(unit + ks_at + r * 8 * NG * 2));
          ks[r] = __byte_perm(bits, 0, 0x1010);
        }
        float s2[NQ][4];
        const uint32_t shift[2] = {int4_shift(ks[0]), int4_shift(ks[1])};
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          uint32_t x[4], y[4];
          int4_values(kw[0][i], ks[0], shift[0], x);
          int4_values(kw[1][i], ks[1], shift[1], y);
          const uint32_t k0[4] = {x[0], y[0], x[1], y[1]}, k1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
          for (int h = 0; h < NQ; ++h) {
            if (i == 0) {
              mma_zero_16816(s[u][h], k0, qf[h][i][0], qf[h][i][1]);
              mma_zero_16816(s2[h], k1, qf[h][i][2], qf[h][i][3]);
            } else {
              mma_bf16_16816(s[u][h], k0, qf[h][i][0], qf[h][i][1]);
              mma_bf16_16816(s2[h], k1, qf[h][i][2], qf[h][i][3]);
            }
          }
        }
        // Scores in base 2 of keys g (e 0, 1) and g + 8 (e 2, 3).  (The product is rounded
        // before the maximum is taken from it: huge scores that are equal stay equal.)
#pragma unroll
        for (int h = 0; h < NQ; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[u][h][e] = __fmaf_rn(s[u][h][e] + s2[h][e], zscale, bias[u][e >> 1]);
          }
        }
      }
      if constexpr (CHUNK) {
        if (!(flags & kFull)) {  // the rows' own limits
#pragma unroll
          for (int h = 0; h < NQ; ++h) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int32_t at = mt.owner.len - mt.owner.tokens + (8 * h + 2 * t + c) / heads;
#pragma unroll
              for (int k = 0; k < 2 * U; ++k) {
                const int32_t key = mt.first[k / 2] + g + 8 * (k % 2);
                if (key > at || (key >= a.sinks && key <= at - a.chunk_window)) {
                  s[k / 2][h][c + 2 * (k % 2)] = -INFINITY;
                }
              }
            }
          }
        }
      }
      float above = -INFINITY;
#pragma unroll
      for (int h = 0; h < NQ; ++h) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          above = fmaxf(above, fmaxf(fmaxf(s[u][h][0], s[u][h][2]) - m2[h][0],
                                     fmaxf(s[u][h][1], s[u][h][3]) - m2[h][1]));
        }
      }
      if (__any_sync(0xffffffffu, above > kSlack)) {
#pragma unroll
        for (int h = 0; h < NQ; ++h) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = m2[h][c];
#pragma unroll
            for (int u = 0; u < U; ++u) m = fmaxf(m, fmaxf(s[u][h][c], s[u][h][c + 2]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const float corr = fast_exp2(m2[h][c] - m);
            m2[h][c] = m;
            lsum[h][c] *= corr;
#pragma unroll
            for (int x = 0; x < NG; ++x) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                o[h][x][j][c] *= corr;
                o[h][x][j][c + 2] *= corr;
              }
            }
          }
        }
      }
      // O^T += V^T P^T.
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t unit = base + u * C::UNIT_BYTES;
        // The codes of V; the scales of keys 2t, 2t + 1 and 2t + 8, 2t + 9, pairs of groups in
        // a register.
        uint32_t sc[4][NG / 2], vc[NG / 2][4];
#pragma unroll
        for (int q = 0; q < NG / 2; ++q) {  // (pieces 2 and 3 are 0 and 1 with one bit turned)
          ldmatrix_x4_trans(unit + (v_at ^ (32 * q)), vc[q][0], vc[q][1], vc[q][2], vc[q][3]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t from = unit + vs_at + ((k & 1) + 8 * (k >> 1)) * (NG * 2);
          if constexpr (NG == 4) {
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                         : "=r"(sc[k][0]), "=r"(sc[k][1])
                         : "r"(from));
          } else {
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(sc[k][0]) : "r"(from));
          }
        }
        uint32_t p[NQ][2];  // P^T: query column g, keys 2t, 2t + 1 and 2t + 8, 2t + 9
#pragma unroll
        for (int h = 0; h < NQ; ++h) {
          float e[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            e[c] = fast_exp2(s[u][h][c] - m2[h][c]);
            e[c + 2] = fast_exp2(s[u][h][c + 2] - m2[h][c]);
            lsum[h][c] += e[c] + e[c + 2];
          }
          p[h][0] = transpose_8x8(pack_bf16x2(e[0], e[1]));
          p[h][1] = transpose_8x8(pack_bf16x2(e[2], e[3]));
        }
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const uint32_t sel = q % 2 == 0 ? 0x5410 : 0x7632;
          const uint32_t s_lo = __byte_perm(sc[0][q / 2], sc[1][q / 2], sel);
          const uint32_t s_hi = __byte_perm(sc[2][q / 2], sc[3][q / 2], sel);
          uint32_t lo[4], hi[4];  // dim i of the lane's four, keys (2t, 2t + 1), (2t + 8, 2t + 9)
          int4_values(vc[q / 2][2 * (q % 2)], s_lo, int4_shift(s_lo), lo);
          int4_values(vc[q / 2][2 * (q % 2) + 1], s_hi, int4_shift(s_hi), hi);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t av[4] = {lo[2 * j], lo[2 * j + 1], hi[2 * j], hi[2 * j + 1]};
#pragma unroll
            for (int h = 0; h < NQ; ++h) mma_bf16_16816(o[h][q][j], av, p[h][0], p[h][1]);
          }
        }
      }

      if (flags & kLast) {
        const int32_t seq = mt.owner.seq, kvh = mt.owner.kvh;
        const bool whole = (mt.owner.flags & kWhole) != 0;
        const int slot_of = (mt.owner.flags & kSlot1) ? 1 : 0;
        float* slot = warp_slot<C>(smem, warp, slot_of);
        const OutRows<CHUNK> to(a, seq, kvh);
        if (lane == 0 && !whole) {
          slots.seq[warp][slot_of] = seq;
          slots.kvh[warp][slot_of] = kvh;
          slots.nb[warp][slot_of] = mt.owner.nb;
          slots.unit[warp][slot_of] = mt.owner.seg_unit;
        }
        __syncwarp();  // (slot 1 lies over the stages: their last reads are done)
        // Neighbouring lanes (g, g ^ 1) hold the dims 2k and 2k + 1: each takes both dims of one
        // of the two query rows.
        const int odd = g & 1;
#pragma unroll
        for (int h = 0; h < NQ; ++h) {
          float l[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            l[c] = lsum[h][c];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
          }
          const int row = 8 * h + 2 * t + odd;
          const float inv = whole ? 1.f / (odd ? l[1] : l[0]) : 1.f;
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + to.row(row, D);
#pragma unroll
          for (int q = 0; q < NG; ++q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float(&acc)[4] = o[h][q][i / 2];
              const float x0 = acc[2 * (i & 1)], x1 = acc[2 * (i & 1) + 1];  // rows 2t, 2t + 1
              const float got = __shfl_xor_sync(0xffffffffu, odd ? x0 : x1, 4);
              const float lo = (odd ? got : x0) * inv, hi = (odd ? x1 : got) * inv;
              const int dim = 32 * q + 8 * (g >> 1) + 2 * i;
              if (whole && row < to.rows) {
                *reinterpret_cast<uint32_t*>(out + dim) = pack_bf16x2(lo, hi);
              } else if (!whole && row < G) {
                *reinterpret_cast<float2*>(slot + row * D + dim) = make_float2(lo, hi);
              }
            }
          }
          if (!whole && g < 2 && row < G) {  // (g is odd here where the row is)
            slot[G * D + row] = odd ? m2[h][1] : m2[h][0];
            slot[G * D + G + row] = odd ? l[1] : l[0];
          }
        }
      }
    }
    // The stage has been read: refill it with the step S positions ahead.
    __syncwarp();
    queue = (queue >> 4) | (issue(base, stage) << (4 * (S - 1)));
    stage = stage + 1 == S ? 0 : stage + 1;
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

template <int D, int NQ, bool CHUNK>
cudaError_t allow_smem() {
  static unsigned long long configured = 0;  // one bit per device
  return once_per_device(&configured, [] {
    return cudaFuncSetAttribute(decode_int4_kernel<D, NQ, CHUNK>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Cfg<D, NQ, CHUNK>::SMEM_BYTES);
  });
}

template <int D, int NQ, bool CHUNK>
int launch_one(const DecodeArgs& a, int grid, cudaStream_t stream) {
  using C = Cfg<D, NQ, CHUNK>;
  cudaError_t e = allow_smem<D, NQ, CHUNK>();
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
  return static_cast<int>(cudaLaunchKernelEx(&cfg, decode_int4_kernel<D, NQ, CHUNK>, a));
}

template <int D, int NQ, bool CHUNK>
int occupancy_one() {
  using C = Cfg<D, NQ, CHUNK>;
  int n = 0;
  cudaError_t e = allow_smem<D, NQ, CHUNK>();
  if (e == cudaSuccess) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, decode_int4_kernel<D, NQ, CHUNK>, C::W * 32,
                                                      C::SMEM_BYTES);
  }
  return e != cudaSuccess ? -static_cast<int>(e) : n;
}

template <int D, bool CHUNK>
int occupancy_rows(int rows) {
  return rows > 8 ? occupancy_one<D, 2, CHUNK>() : occupancy_one<D, 1, CHUNK>();
}

// Joins, behind the decode kernel, the records of the segments that are cut across CTAs: one
// CTA for each of its CTAs (`tasks`).  A warp takes a row's maximum, weights and sum, then the
// threads share the records out, a 16-byte piece of the rows each, kBatch loads at a time.
constexpr int kMergeThreads = 256;
template <int D, bool CHUNK>
__global__ void __launch_bounds__(kMergeThreads, 3) merge_int4_kernel(const DecodeArgs a) {
  constexpr int kBatch = 8, kWarps = kMergeThreads / 32;
  extern __shared__ float weights[];  // [records][rows]
  __shared__ float inverse[kShortChunkRows];
  __shared__ float4 sums[kMergeThreads];
  pdl_wait();
  const MergeTask t = a.tasks[blockIdx.x];
  if (!t.valid) return;
  const int G = a.groups, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t first = span_owner(t.seg_unit, t.q, t.rem);
  const int n = static_cast<int>(span_owner(t.seg_unit + t.nb - 1, t.q, t.rem) - first + 1);
  // (Behind its first CTA the segment is what a span begins with.)
  const float* rec0 = a.partials + record_index(first, t.seg_unit, t.q, t.rem) * a.rec_stride;
  const float* rest = a.partials + first * 2 * a.rec_stride;
  auto record = [&](int c) { return c == 0 ? rec0 : rest + static_cast<int64_t>(2 * c) * a.rec_stride; };
  const int pieces = G * D / 4, width = (pieces + 31) / 32 * 32;
  const int sets = width >= kMergeThreads ? 1 : kMergeThreads / width;
  const int set = tid / width, own = tid - set * width;  // (set >= sets: no part)
  float4 v[kBatch];
  auto fetch = [&](int piece, int c0) {  // pieces of the set's next records
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = c0 + u * sets;
      if (c < n) v[u] = __ldcg(reinterpret_cast<const float4*>(record(c)) + piece);
    }
  };
  if (set < sets && own < pieces) fetch(own, set);  // with the maxima and sums: one trip
  for (int r = warp; r < G; r += kWarps) {
    float m = -INFINITY, l = 0.f;
    for (int c = lane; c < n; c += 32) {
      const float x = __ldcg(record(c) + G * D + r);
      weights[c * G + r] = x;
      m = fmaxf(m, x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int c = lane; c < n; c += 32) {
      const float w = fast_exp2(weights[c * G + r] - m);
      weights[c * G + r] = w;
      l += w * __ldcg(record(c) + G * D + G + r);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) inverse[r] = 1.f / l;
  }
  __syncthreads();
  const OutRows<CHUNK> to(a, t.seq, t.kvh);
  for (int p0 = 0; p0 < pieces; p0 += kMergeThreads) {  // (more than one turn: one set)
    const int piece = p0 + own, r = piece * 4 / D;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (set < sets && piece < pieces) {
      for (int c0 = set; c0 < n; c0 += kBatch * sets) {
        if (p0 != 0 || c0 != set) fetch(piece, c0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int c = c0 + u * sets;
          if (c < n) {
            const float w = weights[c * G + r];
            acc.x += w * v[u].x;
            acc.y += w * v[u].y;
            acc.z += w * v[u].z;
            acc.w += w * v[u].w;
          }
        }
      }
    }
    if (sets > 1) {
      sums[tid] = acc;
      __syncthreads();
      if (set == 0) {
        for (int k = 1; k < sets; ++k) {
          const float4 x = sums[k * width + own];
          acc.x += x.x;
          acc.y += x.y;
          acc.z += x.z;
          acc.w += x.w;
        }
      }
    }
    if (set == 0 && piece < pieces && r < to.rows) {
      const float inv = inverse[r];
      const uint2 o = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv),
                                 pack_bf16x2(acc.z * inv, acc.w * inv));
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + to.row(r, D) + piece * 4 -
                                r * D) = o;
    }
  }
}

template <int D, bool CHUNK>
int launch_merge(const DecodeArgs& a, int grid, cudaStream_t stream) {
  // Room for the weights of 16 rows and 700 CTAs; the grids hold at most four an SM.
  constexpr int kMaxSmem = 45 * 1024;
  static unsigned long long configured = 0;  // one bit per device
  cudaError_t e = once_per_device(&configured, [] {
    return cudaFuncSetAttribute(merge_int4_kernel<D, CHUNK>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  });
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(grid) * a.groups * sizeof(float);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, merge_int4_kernel<D, CHUNK>, a));
}

// Short chunks as sequences of the kernel above; without tokens, of length 0.
__global__ void __launch_bounds__(128) chunk_rows_kernel(const WindowArgs a, int2* rows,
                                                         int32_t* lens, int32_t* table_rows) {
  pdl_wait();
  pdl_trigger();
  const int32_t b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= a.num_rows) return;
  WindowTile w{};
  const bool any = window_tile(a, b, 0, w, true);
  rows[b] = any ? make_int2(w.tok0, w.ntok) : make_int2(0, 0);
  lens[b] = any ? w.pos0 + w.ntok : 0;
  table_rows[b] = any ? w.row : 0;
}

template <int D, bool CHUNK>
int launch_rows(const DecodeArgs& a, int grid, cudaStream_t stream) {
  const int rc = a.groups > 8 ? launch_one<D, 2, CHUNK>(a, grid, stream)
                              : launch_one<D, 1, CHUNK>(a, grid, stream);
  return rc != 0 || a.tasks == nullptr ? rc : launch_merge<D, CHUNK>(a, grid, stream);
}

}  // namespace

int launch_decode_int4(const DecodeArgs& a, int grid, cudaStream_t stream) {
  if (a.chunk_rows != nullptr) {
    return a.head_dim == 64 ? launch_rows<64, true>(a, grid, stream)
                            : launch_rows<128, true>(a, grid, stream);
  }
  return a.head_dim == 64 ? launch_rows<64, false>(a, grid, stream)
                          : launch_rows<128, false>(a, grid, stream);
}

int decode_int4_ctas_per_sm(int head_dim, int rows, bool chunks) {
  if (chunks) return head_dim == 64 ? occupancy_rows<64, true>(rows) : occupancy_rows<128, true>(rows);
  return head_dim == 64 ? occupancy_rows<64, false>(rows) : occupancy_rows<128, false>(rows);
}

int launch_chunk_rows(const WindowArgs& a, int2* rows, int32_t* lens, int32_t* table_rows,
                      cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.num_rows + 127) / 128);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, chunk_rows_kernel, a, rows, lens, table_rows));
}

}  // namespace bsb
