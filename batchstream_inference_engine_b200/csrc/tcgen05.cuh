// tcgen05 (5th-generation tensor core) helpers: descriptors, MMA, commits, TMEM
// accesses, and the 3-D tiled load of query tiles.  Thin wrappers over one PTX
// instruction each.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace bsb {

__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  // sm100 shared-memory matrix descriptor: start, leading and stride byte
  // offsets in 16-byte units, version 1, 128-byte swizzle.
  uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// Instruction descriptor of kind::f16: bf16 A and B, f32 accumulator.
__host__ __device__ constexpr uint32_t umma_idesc(int m, int n, int a_mn_major, int b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn_major) << 15) |
         (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(
          tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0));
}

__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

// 32 consecutive TMEM columns of this thread's lane.  These instructions are .aligned:
// all lanes execute them together.  Where the code before one may have diverged (rows
// without a token, keys that only some rows see), nothing but a warp barrier or another
// warp-wide .sync instruction promises that its lanes have met again.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]));
}

__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Keeps uses of loaded registers behind the wait: to the compiler the load's outputs are
// there at once.
__device__ __forceinline__ void tmem_settle(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 3-D tiled load (query tile): coordinates (dim, head, token).
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// One lane of a converged warp (the same one each time).
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t mine;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(mine));
  return mine;
}

// The products below are executed by the lanes with `mine` set, but called by the
// whole warp: their operands are then warp-uniform values in uniform registers, where
// the instruction takes them.  Inside an `if (lane == 0)` each operand has to be moved
// there first, which made an issue take about 65 cycles.  Descriptors come as their
// low word (start address and leading offset), to which the slice's offset is added
// here (so that no loop keeps them all in registers), and the high word they share.
template <uint32_t kOffA, uint32_t kOffB>
__device__ __forceinline__ void umma_f16_elect(uint32_t mine, uint32_t tmem_d, uint32_t a_lo,
                                               uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b32 x, y;\n .reg .b64 a, b;\n"
      " setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n"
      " add.u32 x, %1, %7;\n add.u32 y, %2, %8;\n mov.b64 a, {x, %3};\n mov.b64 b, {y, %3};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(tmem_d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(mine), "n"(kOffA),
      "n"(kOffB));
}

// A from TMEM (packed pairs along K, lane = row), B from shared memory.
template <uint32_t kOffA, uint32_t kOffB>
__device__ __forceinline__ void umma_f16_ts_elect(uint32_t mine, uint32_t tmem_d, uint32_t tmem_a,
                                                  uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                                  uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b32 x, y;\n .reg .b64 b;\n"
      " setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n"
      " add.u32 x, %1, %7;\n add.u32 y, %2, %8;\n mov.b64 b, {y, %3};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(mine), "n"(kOffA),
      "n"(kOffB));
}

// Calls fn(std::integral_constant) for 0 .. N - 1.
template <int N, typename Fn, int I = 0>
__device__ __forceinline__ void unroll(Fn&& fn) {
  if constexpr (I < N) {
    fn(std::integral_constant<int, I>());
    unroll<N, Fn, I + 1>(static_cast<Fn&&>(fn));
  }
}

__device__ __forceinline__ void umma_commit_elect(uint32_t mine, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
          smem_u32(bar)),
      "r"(mine)
      : "memory");
}

}  // namespace bsb
