// Sliding-window paged attention of prompt chunks on the 5th-generation tensor
// cores (tcgen05 + TMEM): bf16, head_dim 64 or 128, block sizes that are multiples
// of 16, up to 16 query heads per kv head.
//
// Query rows are packed: a CTA's tile of 128 rows is 128 / G consecutive tokens times
// the G query heads of one kv head, so every K and V row that it loads serves the whole
// group, and the keys it reads beyond its window are those of a few tokens (18 at G = 7)
// instead of 128.
//
// The keys a CTA reads are 16-token units: the sink units, then the window's from
// the first token any row sees to the last row's own.  A step is 4 units, each one
// TMA box per K, V and 64 dims through the block table, so sink units and window
// units share a step and nothing between them is touched.
//
// Roles (8 warps, two CTAs per SM):
//   * softmax (warps 0-3), one thread per query row: S from TMEM, mask on border steps
//     only, base-2 online softmax in fp32 whose maximum moves only when it grows by more
//     than 2^8 (then O is rescaled in TMEM), P rounded to bf16 (the tensor cores' input)
//     over the first half of S's columns;
//   * MMA (warp 4): step t is O += P V of step t - 2 (P from TMEM), then S = Q K^T of
//     step t over that P's columns (one thread's products execute in order), then one
//     commit.  S has two buffers, so the scores of the next step are there when the
//     softmax of this one ends;
//   * loaders, of Q and K (warp 5) and of V (warp 6): a TMA box is only 16 rows, and
//     issuing one takes a warp some 35 cycles;
//   * guard (warp 7): on border steps it zeroes the V rows that no row of the CTA
//     sees (never-loaded or stale memory, which 0 * NaN would let through), and the
//     non-finite elements of the others, whose keys it lists: rows that do see such a
//     key get its non-finite values added at the end, rows that do not stay clean.
//
// A step of one tile takes 512 clocks of the special-function units (16 exponentials a
// clock and SM) and 256 (head_dim 64) or 512 (128) of the tensor cores, but a softmax
// warp needs some 1500 from scores to scores: its loads, maxima, exponentials and
// stores follow one another.  Two CTAs to an SM overlap them, and one's start and end with the other's
// steps.  Two tiles in one CTA over the same keys read half as much from L2, but start
// and end together: 8 chunks of 512, d64, 14 heads, window 1024: 45.7 us so, 36.9 with
// a tile each; 6 ragged chunks of 100 to 2048, d128, 28 heads, window 4096: 268 and
// 243 us.  As it is: 37.1 us, and 237 us with the keys in L2 (1015 TFLOP/s, 61% of what a
// plain matrix product reaches), 279 without (52%).  Two stages of d128 are all that fits;
// a third is worth 1%.  The d64 case has 464 tiles for 296 places: SMs are busy for 83% of
// its time.
// Tried and slower: exponentials by the maximum of the steps before, checked afterwards
// (more registers for a wait that the other CTA hides: 39.3 against 39.9 us, 254 and 257,
// and slower for long chunks); two threads a row, 32 keys each, that swap their maxima
// (what a step costs whatever its keys is paid twice: 40.5 against 36.7, 269 and 243).
//
// A call with fewer CTAs than two per SM cuts each tile's steps into ranges, whose
// records window_prefill_merge_kernel joins in range order.
//
// Over 4-bit pools (Q4) warps 5 to 7 write the operands that TMA would bring: each takes
// every third half tile of 32 keys, of K of one step, then of V of the step before, a lane
// 32 dims of a token at a time, whose codes and scale it loaded two half tiles ahead (three: 3%
// slower, four: 8%).  What no row of the CTA sees gets a scale of 0; appended values are finite, so
// there is nothing to guard.  Two tiles share a CTA's K and V where a chunk has rows for both
// (16 warps, of which 7 write).
// 6 ragged chunks of 100 to 2048 behind up to 16384, d128, 28 heads: 798 us = 866 TFLOP/s, 53% of
// what a plain matrix product reaches; over bf16 pools 631.  Without the softmax 620, without the
// conversion 740: a step's latency and the writers' instructions both bound it (1.9 a clock and SM,
// tensor pipe 47%).  8 chunks of 512, d64: 78 us (bf16 70).  64 chunks of 5 behind up to 8192, d64:
// 67 us; without softmax and conversion 68 where this was 74, without the loads 55: a step of 64
// keys costs its round of barriers however few of its rows hold tokens.
//
// Waits are bounded and their outcome made warp-uniform before warp-collective
// instructions; the loaders and the MMA warp drain what they started before TMEM is
// freed, also on the error path.
#include "int4.cuh"
#include "tcgen05.cuh"
#include "window.cuh"

namespace bsb {
namespace {

constexpr int kRows = 128;  // query rows of a tile (TMEM lanes)
constexpr int kKeys = 64;   // keys of a step
constexpr int kUnit = 16;   // tokens per unit (one TMA box)
constexpr int kUnits = kKeys / kUnit;
constexpr int kRing = 8;  // step barriers (>= K stages, >= V stages)
constexpr uint32_t kTileCols = 256;  // TMEM columns of a tile: two S/P buffers, O
constexpr float kLog2eP = 1.4426950408889634f;
constexpr float kRescaleSlack = 8.f;
constexpr float kFarMaximum = 1073741824.f;  // 2^30
constexpr int kMaxBad = 64;  // listed keys with non-finite V (more: all are looked at)

// TILES query tiles share a CTA's K and V: one (two CTAs per SM, 8 warps each) or, over
// 4-bit pools, two (one CTA per SM, 16 warps).
template <int D, int TILES>
struct Cfg {
  static constexpr int ROWS = TILES * kRows;
  static constexpr int MMA_WARP = 4 * TILES, LOAD_K_WARP = MMA_WARP + 1;
  static constexpr int LOAD_V_WARP = MMA_WARP + 2, GUARD_WARP = MMA_WARP + 3;
  static constexpr int THREADS = 256 * TILES, MIN_CTAS = 3 - TILES;
  static constexpr int WRITERS = THREADS / 32 - LOAD_K_WARP;  // of K and V from 4-bit pools
  static constexpr int HALVES = D / 64;
  // Stages of K and V: the CTAs of an SM share its 227 KiB.
  static constexpr int KS = TILES == 2 ? (D == 64 ? 6 : 4) : (D == 64 ? 5 : 2);
  static constexpr int VS = KS;
  static constexpr int Q_HALF_BYTES = ROWS * 128;  // 64 dims of the rows
  static constexpr int Q_BYTES = HALVES * Q_HALF_BYTES;
  static constexpr int HALF_BYTES = kKeys * 128;
  static constexpr int STAGE_BYTES = HALVES * HALF_BYTES;
  static constexpr int SMEM_BYTES = Q_BYTES + (KS + VS) * STAGE_BYTES;
  static constexpr uint32_t O_COL = 2 * kKeys;  // behind the two S/P buffers
  static_assert(O_COL + D <= kTileCols, "TMEM columns");
  static_assert(KS <= kRing && VS <= kRing, "a step waiter could fall a whole ring behind");
};

// The units a tile reads.
struct Steps {
  int32_t sink_units, first_unit, units;
  int32_t pos0, pos1;  // first and last position of its tokens
};

__device__ __forceinline__ Steps steps_of(const WindowArgs& a, const WindowTile& w) {
  Steps s;
  s.first_unit = w.lo / kUnit;
  s.sink_units = min((a.sinks + kUnit - 1) / kUnit, s.first_unit);
  s.pos0 = w.pos0;
  s.pos1 = w.pos0 + w.ntok - 1;
  s.units = s.sink_units + s.pos1 / kUnit - s.first_unit + 1;
  return s;
}

__device__ __forceinline__ int32_t step_count(const Steps& s) {
  return (s.units + kUnits - 1) / kUnits;
}

// First position of unit x of the range.
__device__ __forceinline__ int32_t unit_pos(const Steps& s, int32_t x) {
  return (x < s.sink_units ? x : x - s.sink_units + s.first_unit) * kUnit;
}

// Whether some row of the tile does not see some key of step j.
__device__ __forceinline__ bool step_masked(const WindowArgs& a, const Steps& s, int32_t j) {
  const int32_t u0 = j * kUnits, u1 = u0 + kUnits - 1;
  if (u1 >= s.units || unit_pos(s, u1) + kUnit - 1 > s.pos0) return true;
  if (u0 < s.sink_units && a.sinks < min(u1 + 1, s.sink_units) * kUnit) return true;
  // The step's first window unit against the last row's window.
  return u1 >= s.sink_units && unit_pos(s, max(u0, s.sink_units)) <= s.pos1 - a.window;
}

// Steps [lo, hi] that need no mask (every row sees every key): behind the
// sinks, the units from the first that all windows hold whole to the last that ends at
// or before the first row.
__device__ __forceinline__ void plain_steps(const WindowArgs& a, const Steps& s, int32_t& lo,
                                            int32_t& hi) {
  const int32_t out = s.pos1 - a.window;  // the last position that some row does not see
  const int32_t whole = out < 0 ? 0 : out / kUnit + 1;
  lo = (s.sink_units + max(whole - s.first_unit, 0) + kUnits - 1) / kUnits;
  hi = (s.sink_units + (s.pos0 + 1) / kUnit - s.first_unit) / kUnits - 1;
}

__device__ __forceinline__ bool sees(const WindowArgs& a, int32_t qpos, int32_t pos) {
  return pos <= qpos && (pos < a.sinks || pos > qpos - a.window);
}

// Ranges a tile with `steps` steps is cut into.
__device__ __forceinline__ int32_t step_ranges(int32_t steps, int32_t splits) {
  const int32_t most = (steps + kMinWindowSteps - 1) / kMinWindowSteps;
  return most < splits ? most : splits;
}

// Linear item -> (sequence, tile, kv head), which also numbers the records.
__device__ __forceinline__ void tile_of(const WindowArgs& a, int32_t item, int32_t& r,
                                        int32_t& tile, int32_t& h) {
  h = item % a.num_kv_heads;
  item /= a.num_kv_heads;
  r = item % a.num_rows;
  tile = a.qtiles - 1 - item / a.num_rows;
}

// Most sequences that every CTA ranks (one a thread).
constexpr int kMaxRanked = 256;

// The sequence, tile and kv head of launch index b: the sequences with the most
// steps first, a sequence's last tiles, which see the most keys, ahead of its others.
// A step range is the whole of a CTA's time, so the long ones must not start last.
// All threads call it; `steps` and `pick` are shared memory.
__device__ __forceinline__ void ranked_tile(const WindowArgs& a, int32_t b, int32_t (&steps)[kMaxRanked],
                                            int32_t& pick, int32_t& r, int32_t& tile, int32_t& h) {
  h = b % a.num_kv_heads;
  b /= a.num_kv_heads;
  tile = a.qtiles - 1 - b % a.qtiles;
  r = b / a.qtiles;
  if (a.num_rows == 1 || a.num_rows > kMaxRanked) return;
  const int t = threadIdx.x;
  int32_t mine = 0;
  if (t < a.num_rows) {
    const int32_t tokens = coherent_load(a.cu_q + t + 1) - coherent_load(a.cu_q + t);
    // Keys that the chunk's last tile reads, near enough for an order.
    if (tokens > 0) mine = min(coherent_load(a.context_lens + t), a.window + a.tile_tokens);
    steps[t] = mine;
  }
  __syncthreads();
  if (t < a.num_rows) {
    int32_t rank = 0;
    for (int32_t i = 0; i < a.num_rows; ++i) {
      rank += steps[i] > mine || (steps[i] == mine && i < t) ? 1 : 0;
    }
    if (rank == r) pick = t;  // the ranks are a permutation of the rows
  }
  __syncthreads();
  r = pick;
}

// a * 0 + c on bf16 pairs.
__device__ __forceinline__ uint32_t fma_zero_bf16x2(uint32_t a, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0u), "r"(c));
  return d;
}

template <int D, bool Q4, int TILES>
__global__ void __launch_bounds__((Cfg<D, TILES>::THREADS), (Cfg<D, TILES>::MIN_CTAS))
    window_prefill_kernel(const __grid_constant__ CUtensorMap qmap,
                          const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, const WindowArgs a) {
  static_assert(Q4 || TILES == 1, "the loaders and the guard are for one tile");
  using C = Cfg<D, TILES>;
  constexpr int kMmaWarp = C::MMA_WARP, kLoadKWarp = C::LOAD_K_WARP;
  constexpr int kLoadVWarp = C::LOAD_V_WARP, kGuardWarp = C::GUARD_WARP;
  extern __shared__ __align__(1024) uint8_t smem[];  // 128-byte swizzle atoms
  __shared__ uint64_t q_full, k_full[C::KS], v_full[C::VS], v_ok[C::VS], step_done[TILES][kRing],
      p_full[TILES][2], mma_done;
  __shared__ uint32_t tmem_base;
  __shared__ int32_t bad_count, bad_pos[kMaxBad];

  uint8_t* const sQ = smem;
  auto sK = [&](int st) { return smem + C::Q_BYTES + st * C::STAGE_BYTES; };
  auto sV = [&](int st) { return smem + C::Q_BYTES + (C::KS + st) * C::STAGE_BYTES; };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_wait();
  const int32_t split = blockIdx.x % a.splits;
  __shared__ int32_t ranked[kMaxRanked], picked;
  int32_t r, tile, h;
  ranked_tile(a, blockIdx.x / a.splits, ranked, picked, r, tile, h);
  // The item of its records (tile_of).
  const int32_t item = ((a.qtiles - 1 - tile) * a.num_rows + r) * a.num_kv_heads + h;
  WindowTile w;
  if (!window_tile(a, r, tile, w, tid == 0 && tile == 0 && h == 0 && split == 0)) return;
  const Steps sd = steps_of(a, w);
  const int32_t all = step_count(sd);
  const int32_t ranges = step_ranges(all, a.splits);
  if (split >= ranges) return;
  const int32_t j0 = split * all / ranges;
  const int32_t n = (split + 1) * all / ranges - j0;  // steps of this CTA

  if (tid == 0) {
    mbar_init(&q_full, 1);
    // (4-bit: an arrival for each half tile written.)
    for (int s = 0; s < C::KS; ++s) mbar_init(&k_full[s], Q4 ? 2 : 1);
    for (int s = 0; s < C::VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_ok[s], Q4 ? 2 : 1);
    }
    for (int x = 0; x < TILES; ++x) {
      for (int s = 0; s < kRing; ++s) mbar_init(&step_done[x][s], 1);
      for (int b = 0; b < 2; ++b) mbar_init(&p_full[x][b], kRows);
    }
    mbar_init(&mma_done, 1);
    fence_barrier_init();
    bad_count = 0;
  }
  if (warp == 0) {
    __syncwarp();  // thread 0 comes from the barriers' setup
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_base)),
                 "r"(TILES * kTileCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  auto wait_all = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0;
  };
  // Step u of a tile is done: P V of step u - 2 and S of step u (of the tiles before it too:
  // they are issued first).  Waiters take the steps in order and are never kRing behind (see
  // the ring sizes).
  auto wait_step = [&](int u, int of = TILES - 1) {
    return wait_all(&step_done[of][u % kRing], (u / kRing) & 1);
  };

  if (Q4 && warp >= kLoadKWarp) {
    // ---------------------------------------------------------------- 4-bit K and V
    if (warp == kLoadKWarp) {
      if (lane == 0) {
        const uint32_t rows = static_cast<uint32_t>(a.tile_tokens * a.groups);
        mbar_arrive_expect_tx(&q_full, C::HALVES * rows * 128u);
        for (int hf = 0; hf < C::HALVES; ++hf) {
          tma_load_3d(sQ + hf * C::Q_HALF_BYTES, &qmap, &q_full, hf * 64, h * a.groups, w.tok0);
        }
      }
      __syncwarp();
    }
    constexpr int NG = D / kInt4Group, ROWS = 32 / NG, PARTS = kUnit / ROWS;  // rows a load
    constexpr int kWriters = C::WRITERS;
    const int32_t* table = a.block_tables + static_cast<int64_t>(w.row) * a.bt_stride;
    const int32_t block_units = a.block_size / kUnit;
    const int32_t block_bytes = a.block_size * int4_row_bytes(D);  // fits (host)
    // This lane's token (of ROWS) and dims.  Neighbouring lanes have neighbouring tokens: their
    // 16-byte pieces of a step's row of 64 dims, at `piece` ^ k, are then in different banks.
    const int row = lane % ROWS, group = lane / ROWS;
    const uint32_t piece = ((group & 1) * 4) ^ (row & 7);
    const uint32_t ring = smem_u32(sK(0)) + (group >> 1) * C::HALF_BYTES + row * 128;
    const int64_t head_at = static_cast<int64_t>(h) * a.num_blocks * block_bytes +
                            row * int4_code_bytes(D) + group * 16;
    const uint8_t* const k_codes = static_cast<const uint8_t*>(a.k_pool) + head_at;
    const uint8_t* const v_codes = static_cast<const uint8_t*>(a.v_pool) + head_at;
    const int32_t to_scales = a.block_size * int4_code_bytes(D) + row * int4_scale_bytes(D) +
                              group * 2 - row * int4_code_bytes(D) - group * 16;
    // Half tiles of 32 keys in the order K(0), V(-1), K(1), V(0), K(2), V(1), ..: half
    // tile i is half i & 1 of K(i / 4) or, with bit 1, of V(i / 4 - 1).
    auto step_of = [&](int32_t i) { return (i >> 2) - ((i >> 1) & 1); };
    auto token_unit = [&](int32_t x) {  // of unit x of the range
      return x < sd.sink_units ? x : x - sd.sink_units + sd.first_unit;
    };
    // Table entries of units 32 q .. 32 q + 31 of the CTA's steps, a lane each, for an even and
    // an odd q (-1: past the range).  Window q + 1 is loaded when K is 16 units into window q, which
    // V, at most 8 behind it, has entered by then.
    const int32_t unit0 = j0 * kUnits, units = min(n * kUnits, sd.units - unit0);
    int32_t even = -1, odd = -1, windows = 0;
    auto load_entries = [&]() {
      const int32_t x = 32 * windows + lane;
      int32_t blk = -1;
      if (x < units) {
        const int32_t tu = token_unit(unit0 + x);
        blk = __ldg(table + (block_units == 1 ? tu : tu / block_units));
      }
      if (windows++ & 1) {
        odd = blk;
      } else {
        even = blk;
      }
    };
    load_entries();
    load_entries();
    struct Codes {
      uint4 words[2][PARTS];
      uint32_t scale[2][PARTS];
    };
    int32_t plain_lo, plain_hi;
    plain_steps(a, sd, plain_lo, plain_hi);
    auto load = [&](int32_t i, Codes& c) {
      const int32_t j = step_of(i), x0 = j * kUnits + 2 * (i & 1);
      if (j < 0 || x0 >= n * kUnits) return;
      const bool is_v = (i & 2) != 0;
      if (x0 + 16 >= 32 * windows) load_entries();
      const int32_t win = (x0 & 32) != 0 ? odd : even;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int32_t blk = __shfl_sync(0xffffffffu, win, (x0 + e) & 31);
        if (static_cast<uint32_t>(blk) >= static_cast<uint32_t>(a.num_blocks)) {
          if (lane == 0 && !is_v && x0 + e < units) set_status(a.status, kStatusBadBlock);
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            c.words[e][p] = make_uint4(0u, 0u, 0u, 0u);
            c.scale[e][p] = 0u;
          }
          continue;
        }
        const uint8_t* codes = (is_v ? v_codes : k_codes) + static_cast<int64_t>(blk) * block_bytes;
        const uint8_t* scales = codes + to_scales;
        if (block_units != 1) {
          const int32_t first = token_unit(unit0 + x0 + e) % block_units * kUnit;
          codes += first * int4_code_bytes(D);
          scales += first * int4_scale_bytes(D);
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          c.words[e][p] =
              coherent_load(reinterpret_cast<const uint4*>(codes + p * ROWS * int4_code_bytes(D)));
          c.scale[e][p] = coherent_load(
              reinterpret_cast<const uint16_t*>(scales + p * ROWS * int4_scale_bytes(D)));
        }
      }
    };
    // Codes are loaded kAhead of this warp's half tiles ahead.
    constexpr int kAhead = 2;
    Codes codes[kAhead];
    int32_t i = warp - kLoadKWarp;
#pragma unroll
    for (int x = 0; x < kAhead; ++x) load(i + x * kWriters, codes[x]);
    bool ok = true;
    auto turn = [&](Codes& c) {
      const bool is_v = (i & 2) != 0;
      const int32_t j = step_of(i);
      if (j >= 0 && j < n) {
        // Step j - KS has read the K stage, step j - VS + 2 the V stage.
        if (j >= (is_v ? C::VS : C::KS)) ok = wait_step(is_v ? j - C::VS + 2 : j - C::KS);
        if (!ok) return;
        const int stage = is_v ? j % C::VS : j % C::KS;
        if (j0 + j < plain_lo || j0 + j > plain_hi) {
          // Rows that nobody sees may hold anything: their values are 0.  (Here, not where the
          // codes are loaded, which would wait for them.)
          const int32_t x0 = (j0 + j) * kUnits + 2 * (i & 1);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int32_t pos = token_unit(x0 + e) * kUnit + row;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
              const int32_t at = pos + p * ROWS;
              if (at > sd.pos1 || (at >= a.sinks && at < w.lo)) c.scale[e][p] = 0u;
            }
          }
        }
        const uint32_t to = ring + ((is_v ? C::KS : 0) + stage) * C::STAGE_BYTES + (i & 1) * 32 * 128;
        uint32_t at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) at[k] = to + ((piece ^ k) << 4);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            const uint32_t words[4] = {c.words[e][p].x, c.words[e][p].y, c.words[e][p].z,
                                       c.words[e][p].w};
            const uint32_t scale = __byte_perm(c.scale[e][p], 0, 0x1010);
            const uint32_t shift = int4_shift(scale);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t v[4];
              int4_values(words[k], scale, shift, v);
              asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(
                               at[k] + (e * kUnit + p * ROWS) * 128),
                           "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                           : "memory");
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(is_v ? &v_ok[stage] : &k_full[stage]);
      }
      i += kWriters;
      load(i + (kAhead - 1) * kWriters, c);
    };
    const int32_t end = 4 * (n + 1);
    while (ok && i < end) {
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        if (ok && i < end) turn(codes[x]);
      }
    }
    const bool drained = warp != kLoadKWarp || wait_all(&q_full, 0);
    if ((!ok || !drained) && lane == 0) set_status(a.status, kStatusWaitTimeout);
  } else if (warp == kLoadKWarp || warp == kLoadVWarp) {
    // ---------------------------------------------------------------- loaders
    const bool is_k = warp == kLoadKWarp;
    const CUtensorMap* map = is_k ? &kmap : &vmap;
    const int stages = is_k ? C::KS : C::VS;
    uint8_t* ring = is_k ? sK(0) : sV(0);
    uint64_t* full = is_k ? k_full : v_full;
    const int32_t* table = a.block_tables + static_cast<int64_t>(w.row) * a.bt_stride;
    const int32_t block_units = a.block_size / kUnit;
    const int unit = lane % kUnits, half = lane / kUnits;  // this lane's box of a step
    uint8_t* box = ring + half * C::HALF_BYTES + unit * 2048;
    const int32_t head_row = h * a.num_blocks * a.block_size;
    // Pool row of this lane's unit of step j (-1: past the range or invalid).
    auto fetch = [&](int32_t j) -> int32_t {
      const int32_t x = (j0 + j) * kUnits + unit;
      if (j >= n || x >= sd.units || half >= C::HALVES) return -1;
      const int32_t tu = x < sd.sink_units ? x : x - sd.sink_units + sd.first_unit;
      const int32_t ent = block_units == 1 ? tu : tu / block_units;
      const int32_t blk = __ldg(table + ent);
      if (blk < 0 || blk >= a.num_blocks) {
        if (is_k && half == 0) set_status(a.status, kStatusBadBlock);
        return -1;
      }
      return head_row + blk * a.block_size + (tu - ent * block_units) * kUnit;
    };
    int32_t y = fetch(0), y_next = fetch(1);
    if (is_k && lane == 0) {
      const uint32_t rows = static_cast<uint32_t>(a.tile_tokens * a.groups);
      mbar_arrive_expect_tx(&q_full, C::HALVES * rows * 128u);
      for (int hf = 0; hf < C::HALVES; ++hf) {
        tma_load_3d(sQ + hf * C::Q_HALF_BYTES, &qmap, &q_full, hf * 64, h * a.groups, w.tok0);
      }
    }
    __syncwarp();
    // Step j - KS has read the K stage, step j - VS + 2 the V stage.
    const int32_t lag = is_k ? 0 : 2;
    bool ok = true;
    int32_t loads = 0;
    int stage = 0;
    for (int32_t j = 0; j < n; ++j) {
      if (j >= stages) ok = wait_step(j - stages + lag);
      if (!ok) break;
      const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, y >= 0));
      if (lane == 0) mbar_arrive_expect_tx(full + stage, boxes * 2048u);
      __syncwarp();
      if (y >= 0) tma_load_2d(box + stage * C::STAGE_BYTES, map, full + stage, half * 64, y);
      loads = j + 1;
      if (++stage == stages) stage = 0;
      y = y_next;
      y_next = fetch(j + 2);
    }
    // Drain: every load has landed before the CTA leaves its shared memory.
    bool drained = !is_k || wait_all(&q_full, 0);
    for (int32_t j = max(0, loads - stages); j < loads; ++j) {
      drained = wait_all(full + j % stages, (j / stages) & 1) && drained;
    }
    if ((!ok || !drained) && lane == 0) set_status(a.status, kStatusWaitTimeout);
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t kIdescS = umma_idesc(128, kKeys, 0, 0);
    constexpr uint32_t kIdescO = umma_idesc(128, D, 0, 1);
    constexpr uint32_t kQHalf = C::Q_HALF_BYTES >> 4;
    constexpr uint32_t kStageStep = C::STAGE_BYTES >> 4, kHalf = C::HALF_BYTES >> 4;
    const uint64_t desc_q = umma_desc(smem_u32(sQ), 16, 1024);
    const uint32_t hi = static_cast<uint32_t>(desc_q >> 32);  // of every operand
    const uint32_t q_lo = static_cast<uint32_t>(desc_q);
    const uint32_t k_lo = static_cast<uint32_t>(umma_desc(smem_u32(sK(0)), 16, 1024));
    // V: dims contiguous (MN-major): 64-dim halves HALF_BYTES apart, 8 keys 1024.
    const uint32_t v_lo =
        static_cast<uint32_t>(umma_desc(smem_u32(sV(0)), C::HALF_BYTES, 1024));
    const uint32_t mine = elect_lane();  // issues every product
    bool ok = wait_all(&q_full, 0);
    // Ring positions and phases are carried along: this warp's own instructions, products
    // apart, must stay well below a step's time.
    int ks = 0, vs = 0;
    uint32_t k_phase = 0, v_phase = 0;
    for (int32_t u = 0; u < n + 2 && ok; ++u) {
      const int b = u & 1;
      const bool pv = u > 1, qk = u < n;
      // P last: K and V are there long before it.
      if (qk) ok = wait_all(&k_full[ks], k_phase);
      if (pv) ok = ok && wait_all(&v_ok[vs], v_phase);
      if (!ok) break;
#pragma unroll
      for (int x = 0; x < TILES; ++x) {
        if (pv) ok = wait_all(&p_full[x][b], ((u >> 1) & 1) ^ 1);  // of step u - 2
        if (!ok) break;
        tc_fence_after();
        const uint32_t cols = tmem + x * kTileCols, s_col = cols + b * kKeys;
        if (pv) {
          const uint32_t v0 = v_lo + vs * kStageStep;
          unroll<kKeys / 16>([&](auto k) {
            // P: 8 columns per 16 keys; V: 16 rows of 128 bytes.
            umma_f16_ts_elect<8 * k, 128 * k>(mine, cols + C::O_COL, s_col, v0, hi, kIdescO,
                                              k > 0 || u > 2 ? 1u : 0u);
          });
        }
        if (qk) {
          const uint32_t q0 = q_lo + x * (kRows * 128 >> 4), k0 = k_lo + ks * kStageStep;
          unroll<D / 16>([&](auto k) {
            // 32 bytes a slice of 16 dims.
            umma_f16_elect<(k / 4) * kQHalf + 2 * (k % 4), (k / 4) * kHalf + 2 * (k % 4)>(
                mine, s_col, q0, k0, hi, kIdescS, k > 0 ? 1u : 0u);
          });
        }
        umma_commit_elect(mine, &step_done[x][u % kRing]);
      }
      if (!ok) break;
      if (++ks == C::KS) {
        ks = 0;
        k_phase ^= 1u;
      }
      if (pv && ++vs == C::VS) {
        vs = 0;
        v_phase ^= 1u;
      }
    }
    __syncwarp();
    umma_commit_elect(mine, &mma_done);
    const bool drained = wait_all(&mma_done, 0);
    if ((!ok || !drained) && lane == 0) set_status(a.status, kStatusWaitTimeout);
  } else if (warp == kGuardWarp) {
    // ---------------------------------------------------------------- guard
    bool ok = true;
    for (int32_t j = 0; j < n; ++j) {
      const int vs = j % C::VS;
      ok = wait_all(&v_full[vs], (j / C::VS) & 1);
      if (!ok) break;
      if (step_masked(a, sd, j0 + j)) {
        auto position = [&](int row) {  // of the key of a V row
          return unit_pos(sd, (j0 + j) * kUnits + row / kUnit) + row % kUnit;
        };
        // Rows that no query row sees become zero (lane = row, then four rows at a
        // time, eight lanes along each).
        for (int g = 0; g < kKeys / 32; ++g) {
          const int row = g * 32 + lane;
          const int32_t pos = position(row);
          const bool live = (j0 + j) * kUnits + row / kUnit < sd.units && pos <= sd.pos1 &&
                            (pos < a.sinks || pos >= w.lo);
          const uint32_t dead = __ballot_sync(0xffffffffu, !live);
          for (int q = 0; q < 8; ++q) {
            if (!((dead >> (4 * q + (lane >> 3))) & 1u)) continue;
            uint8_t* p = sV(vs) + (g * 32 + 4 * q + (lane >> 3)) * 128 + (lane & 7) * 16;
            for (int hf = 0; hf < C::HALVES; ++hf) {
              *reinterpret_cast<uint4*>(p + hf * C::HALF_BYTES) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          __syncwarp();
        }
        // x * 0 is 0 or, for infinities and NaN, NaN, and stays NaN in the sum.
        uint32_t sum = 0;
#pragma unroll 8
        for (int c = 0; c < C::STAGE_BYTES / 512; ++c) {
          const uint4 v = *reinterpret_cast<const uint4*>(sV(vs) + (c * 32 + lane) * 16);
          sum = fma_zero_bf16x2(v.x, sum);
          sum = fma_zero_bf16x2(v.y, sum);
          sum = fma_zero_bf16x2(v.z, sum);
          sum = fma_zero_bf16x2(v.w, sum);
        }
        if (__any_sync(0xffffffffu, sum != 0u)) {
          // Lane = (row of a group of 4, 16-byte column of a 128-byte row).
          for (int g = 0; g < kKeys / 4; ++g) {
            const int row = g * 4 + (lane >> 3), col = lane & 7;
            bool bad = false;
            for (int hf = 0; hf < C::HALVES; ++hf) {
              uint4* p =
                  reinterpret_cast<uint4*>(sV(vs) + hf * C::HALF_BYTES + row * 128 + col * 16);
              uint4 v = *p;
              uint32_t* e = reinterpret_cast<uint32_t*>(&v);
              bool hit = false;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                // All exponent bits set: infinity or NaN.
                uint32_t keep = 0xffffffffu;
                if ((e[i] & 0x7f80u) == 0x7f80u) keep &= 0xffff0000u;
                if ((e[i] & 0x7f800000u) == 0x7f800000u) keep &= 0x0000ffffu;
                hit |= keep != 0xffffffffu;
                e[i] &= keep;
              }
              if (hit) *p = v;
              bad |= hit;
            }
            const uint32_t any = __ballot_sync(0xffffffffu, bad);
            if (col == 0 && ((any >> (lane & ~7)) & 0xffu) != 0) {
              const int32_t at = atomicAdd(&bad_count, 1);
              if (at < kMaxBad) bad_pos[at] = position(row);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_ok[vs]);
      __syncwarp();
    }
    if (!ok && lane == 0) set_status(a.status, kStatusWaitTimeout);
  } else {
    // ---------------------------------------------------------------- softmax
    const int row = tid, own = warp / 4;  // row of the CTA's tiles; its tile
    const int32_t tok = row / a.groups, g = row - tok * a.groups;
    const bool live = tok < w.ntok;
    const int32_t qpos = w.pos0 + tok;
    const uint32_t lane_base = (static_cast<uint32_t>(warp % 4 * 32) << 16) + own * kTileCols;
    const uint32_t o_addr = tmem + lane_base + C::O_COL;
    const float zscale = fabsf(a.scale) * kLog2eP;
    // Exponents are scale * score - scale * raw_used, the largest score used so far.  That
    // product is rounded and the fused step takes it from the exact one, which shifts all
    // of a row's exponents alike, by up to 2^-24 of the product: harmless until 2^shift
    // overflows.  From 2^30 on rows scale by the power of two below, which is exact:
    // scores that differ at all are then 2^5 or more apart, so only the keys at the
    // maximum count, as they do with the scale itself.
    float raw_used = -INFINITY, zs = zscale, l_run = 0.f;
    auto scale_of = [&](float top) {
      return fabsf(top * zscale) < kFarMaximum || top == -INFINITY  // (-inf: no key yet)
                 ? zscale : __uint_as_float(__float_as_uint(zscale) & 0x7f800000u);
    };
    int32_t plain_lo, plain_hi;
    plain_steps(a, sd, plain_lo, plain_hi);
    const bool any_live = __any_sync(0xffffffffu, live);
    bool ok = true;
    for (int32_t u = 0; u < n; ++u) {
      ok = wait_step(u, own);
      if (!ok) break;
      if (!any_live) {  // nothing reads what comes of these rows
        mbar_arrive(&p_full[own][u & 1]);
        continue;
      }
      tc_fence_after();
      const uint32_t s_addr = tmem + lane_base + (u & 1) * kKeys;
      // Visible tokens of the step's units, 16 bits each (border steps only).
      const bool border =
          (j0 + u < plain_lo || j0 + u > plain_hi) && step_masked(a, sd, j0 + u);
      uint32_t maps[2];
      if (border) {
        auto below = [](int32_t c) -> uint32_t {  // map of the first c tokens
          return c >= kUnit ? 0xffffu : c <= 0 ? 0u : (1u << c) - 1u;
        };
#pragma unroll
        for (int un = 0; un < kUnits; ++un) {
          const int32_t ux = (j0 + u) * kUnits + un;
          const int32_t p0 = unit_pos(sd, ux);
          uint32_t map = below(qpos - p0 + 1) &
                         (~below(qpos - a.window + 1 - p0) | below(a.sinks - p0));
          if (ux >= sd.units || !live) map = 0;
          maps[un / 2] = un % 2 ? maps[un / 2] | (map << 16) : map;
        }
        __syncwarp();  // ahead of .aligned loads
      }
      uint32_t v[2][32];
      tmem_ld32(s_addr, v[0]);
      tmem_ld32(s_addr + 32, v[1]);
      tmem_wait_ld();
      tmem_settle(v[0]);
      tmem_settle(v[1]);
      if (a.scale < 0.f) {  // turned around: the rest works with the scale's magnitude
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i / 32][i % 32] ^= 0x80000000u;
      }
      if (border) {  // unseen keys become -inf
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          if (!((maps[i / 32] >> (i % 32)) & 1u)) v[i / 32][i % 32] = 0xff800000u;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 32; ++i) {  // three-input maxima
        mx[i & 3] = fmaxf(fmaxf(mx[i & 3], __uint_as_float(v[0][i])), __uint_as_float(v[1][i]));
      }
      const float raw = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grow = live && __fmul_rn(raw, zscale) > __fmul_rn(raw_used, zscale) + kRescaleSlack;
      if (u == 0) {
        raw_used = raw;
        zs = scale_of(raw);
      } else if (__any_sync(0xffffffffu, grow)) {
        // O may be rescaled once P V of the step before is done; rows that did not
        // grow keep theirs (factor 1).
        ok = wait_step(u + 1, own);
        if (!ok) break;
        tc_fence_after();
        const float corr = grow ? fast_exp2(__fmul_rn(raw_used, zscale) - __fmul_rn(raw, zscale)) : 1.f;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          tmem_ld32(o_addr + c0, o);
          tmem_wait_ld();
          tmem_settle(o);
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
          tmem_st32(o_addr + c0, o);
        }
        l_run *= corr;
        raw_used = grow ? raw : raw_used;
        zs = scale_of(raw_used);
      }
      const float m_base = raw_used == -INFINITY ? 0.f : raw_used * zs;  // no -inf - -inf
      const float2 zs2 = make_float2(zs, zs), mm = make_float2(-m_base, -m_base);
      float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                       make_float2(0.f, 0.f)};
      uint32_t p[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 e = __ffma2_rn(make_float2(__uint_as_float(v[i / 16][2 * (i % 16)]),
                                                __uint_as_float(v[i / 16][2 * (i % 16) + 1])),
                                    zs2, mm);
        const float2 pe = make_float2(fast_exp2(e.x), fast_exp2(e.y));
        sum[i & 3] = __fadd2_rn(sum[i & 3], pe);
        p[i] = pack_bf16x2(pe.x, pe.y);
      }
      tmem_st32(s_addr, p);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[own][u & 1]);
      l_run += ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) +
               ((sum[2].x + sum[2].y) + (sum[3].x + sum[3].y));
    }
    // The last P V is done (the steps in order, as everywhere).
    if (ok) ok = wait_step(n, own) && wait_step(n + 1, own);
    if (!ok) {
      if (lane == 0) set_status(a.status, kStatusWaitTimeout);
    } else {
      tc_fence_after();
      const bool split_up = ranges > 1;
      // Listed keys are complete: the guard arrived for every V that was used.
      const int32_t bad = bad_count;
      const float scale = split_up ? 1.f : 1.f / l_run;
      const int32_t* table = a.block_tables + static_cast<int64_t>(w.row) * a.bt_stride;
      const int64_t rec_row = (static_cast<int64_t>(item) * a.splits + split) * C::ROWS + row;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(o_addr + c0, v);
        tmem_wait_ld();
        tmem_settle(v);
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * scale);
        if (bad > 0 && live) {
          const int32_t count = bad <= kMaxBad ? bad : n * kKeys;
          for (int32_t b = 0; b < count; ++b) {
            int32_t pos;
            if (bad <= kMaxBad) {
              pos = bad_pos[b];
            } else {
              const int32_t ux = j0 * kUnits + b / kUnit;
              if (ux >= sd.units) break;
              pos = unit_pos(sd, ux) + b % kUnit;
            }
            if (!sees(a, qpos, pos)) continue;
            const int32_t blk = __ldg(table + pos / a.block_size);
            if (blk < 0 || blk >= a.num_blocks) continue;
            const __nv_bfloat16* src =
                static_cast<const __nv_bfloat16*>(a.v_pool) +
                ((static_cast<int64_t>(h) * a.num_blocks + blk) * a.block_size +
                 pos % a.block_size) * D + c0;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float e = __bfloat162float(src[c]);
              if (!isfinite(e)) v[c] = __float_as_uint(__uint_as_float(v[c]) + e);
            }
          }
        }
        if (!live) {
          // Holds no token: nothing to store.
        } else if (split_up) {
          float* dst = a.records + rec_row * D + c0;
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            *reinterpret_cast<uint4*>(dst + c) = make_uint4(v[c], v[c + 1], v[c + 2], v[c + 3]);
          }
        } else {
          __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) +
                               static_cast<int64_t>(w.tok0 + tok) * a.o_stride +
                               static_cast<int64_t>(h * a.groups + g) * D + c0;
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            uint4 o;
            o.x = pack_bf16x2(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
            o.y = pack_bf16x2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
            o.z = pack_bf16x2(__uint_as_float(v[c + 4]), __uint_as_float(v[c + 5]));
            o.w = pack_bf16x2(__uint_as_float(v[c + 6]), __uint_as_float(v[c + 7]));
            *reinterpret_cast<uint4*>(dst + c) = o;
          }
        }
        __syncwarp();  // rows without a token, and those that see a listed key, part above
      }
      if (split_up && live) {
        float* ml = a.records + a.rec_stride_ml + rec_row * 2;
        *reinterpret_cast<float2*>(ml) = make_float2(raw_used * zscale, l_run);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(TILES * kTileCols));
  }
}

// Joins the records of a tile's step ranges, in range order: eight threads a
// row, D / 8 columns each.
constexpr int kMergeThreads = 256;
constexpr int kMergeRows = kMergeThreads / 8;

template <int D>
__global__ void __launch_bounds__(kMergeThreads) window_prefill_merge_kernel(const WindowArgs a) {
  pdl_wait();
  const int parts = a.tile_rows / kMergeRows;  // CTAs per tile
  const int32_t item = blockIdx.x / parts;
  int32_t r, tile, h;
  tile_of(a, item, r, tile, h);
  WindowTile w;
  if (!window_tile(a, r, tile, w, false)) return;
  const int32_t row = (blockIdx.x % parts) * kMergeRows + threadIdx.x / 8;
  const int32_t tok = row / a.groups, g = row - tok * a.groups;
  if (tok >= w.ntok) return;
  const Steps sd = steps_of(a, w);
  const int32_t ranges = step_ranges(step_count(sd), a.splits);
  if (ranges <= 1) return;  // written by the kernel itself
  const int32_t c = (threadIdx.x % 8) * (D / 8);
  const int64_t rec0 = static_cast<int64_t>(item) * a.splits * a.tile_rows + row;
  const float* ml = a.records + a.rec_stride_ml;
  float M = -INFINITY;
  for (int32_t s = 0; s < ranges; ++s) M = fmaxf(M, ml[(rec0 + s * a.tile_rows) * 2]);
  const float base = M == -INFINITY ? 0.f : M;
  float L = 0.f, acc[D / 8];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int32_t s = 0; s < ranges; ++s) {
    const float2 p = *reinterpret_cast<const float2*>(ml + (rec0 + s * a.tile_rows) * 2);
    // A range without a finite score of this row weighs 0 (NaN scores: 0 * NaN).
    const float f = fast_exp2(p.x - base);
    L += f * p.y;
    const float4* o = reinterpret_cast<const float4*>(a.records + (rec0 + s * a.tile_rows) * D + c);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const float4 v = o[i];
      acc[4 * i] += f * v.x;
      acc[4 * i + 1] += f * v.y;
      acc[4 * i + 2] += f * v.z;
      acc[4 * i + 3] += f * v.w;
    }
  }
  const float inv = 1.f / L;
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) +
                       static_cast<int64_t>(w.tok0 + tok) * a.o_stride +
                       static_cast<int64_t>(h * a.groups + g) * D + c;
#pragma unroll
  for (int i = 0; i < D / 8; i += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = acc[i + k] * inv;
    store8(dst + i, v);
  }
}

template <int D, bool Q4, int TILES>
int launch_d(const WindowArgs& a, const CUtensorMap& qmap, const CUtensorMap& kmap,
             const CUtensorMap& vmap, cudaStream_t stream) {
  using C = Cfg<D, TILES>;
  static unsigned long long configured = 0;  // one bit per device
  cudaError_t e = once_per_device(&configured, [] {
    return cudaFuncSetAttribute(window_prefill_kernel<D, Q4, TILES>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
  });
  if (e != cudaSuccess) return static_cast<int>(e);
  const int64_t items = static_cast<int64_t>(a.num_rows) * a.qtiles * a.num_kv_heads;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * a.splits));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, window_prefill_kernel<D, Q4, TILES>, qmap, kmap, vmap, a);
  if (e != cudaSuccess || a.splits == 1) return static_cast<int>(e);
  cfg.gridDim = dim3(static_cast<unsigned>(items * (C::ROWS / kMergeRows)));
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, window_prefill_merge_kernel<D>, a));
}

}  // namespace

int launch_window_prefill(const WindowArgs& a, const CUtensorMap& qmap, const CUtensorMap& kmap,
                          const CUtensorMap& vmap, cudaStream_t stream) {
  if (a.int4 && a.tile_rows == 2 * kRows) {  // (kmap and vmap are not used)
    return a.head_dim == 64 ? launch_d<64, true, 2>(a, qmap, kmap, vmap, stream)
                            : launch_d<128, true, 2>(a, qmap, kmap, vmap, stream);
  }
  if (a.int4) {
    return a.head_dim == 64 ? launch_d<64, true, 1>(a, qmap, kmap, vmap, stream)
                            : launch_d<128, true, 1>(a, qmap, kmap, vmap, stream);
  }
  return a.head_dim == 64 ? launch_d<64, false, 1>(a, qmap, kmap, vmap, stream)
                          : launch_d<128, false, 1>(a, qmap, kmap, vmap, stream);
}

}  // namespace bsb
