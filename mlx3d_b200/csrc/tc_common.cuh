// tcgen05 (5th-generation tensor core) helpers: shared-memory and instruction
// descriptors, TMEM allocation, matrix issue, TMEM loads and stores.
//
// Operand layout used throughout: 128-byte-swizzled panels.  A panel is R rows
// of 64 16-bit elements (128 bytes a row); the 16-byte unit u of row r lies at
// r * 128 + ((u ^ (r & 7)) << 4), panels start on 1024-byte boundaries.  The
// same panel is a K-major operand (rows = M or N index, the 64 elements = K)
// or an MN-major one (rows = K index, the 64 elements = M or N index),
// depending on the descriptor; no transposed copies are needed.
#pragma once

#include "gs_common.cuh"

namespace gs {
namespace tc {

constexpr int kPanelRow = 128;  // bytes of a panel row

__device__ __forceinline__ uint32_t panel_offset(int row, int unit) {
  return (uint32_t)(row * kPanelRow + ((unit ^ (row & 7)) << 4));
}

// Shared-memory matrix descriptor, 128-byte swizzle: bits 0-13 address / 16,
// 16-29 leading byte offset / 16, 32-45 stride byte offset / 16, bits 46-48 =
// 1, bits 61-63 = 2 (128-byte swizzle).  8-row groups are 1024 bytes apart in
// every layout used here, so the upper word is a constant and a descriptor is
// handled as its lower word; an offset of n bytes adds n / 16 to it.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// K-major panel: 16 K elements = 32 bytes.
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr & 0x3ffff) >> 4) | (1u << 16); }
// MN-major panels, `panel_bytes` apart; 16 K rows = 2048 bytes.
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr, uint32_t panel_bytes) {
  return ((addr & 0x3ffff) >> 4) | ((panel_bytes >> 4) << 16);
}
// The value of lane 0, known to be the same in every lane: it can be kept in a
// uniform register, which the matrix instructions take their operands from.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(~0u, v, 0); }

// Instruction descriptor of kind::f16, float32 accumulators, M = 128:
// bits 4-5 accumulator type (1 = f32), 7-9 / 10-12 A / B type (0 = f16, 1 =
// bf16), 15 / 16 A / B MN-major, 17-22 N / 8, 24-28 M / 16.
__host__ __device__ constexpr uint32_t instr_desc(bool bf16, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// True in one lane of a converged warp.  Matrix instructions are issued under
// this by warps whose control flow is uniform, so that their descriptors stay in
// uniform registers; under `lane == 0` each costs about 110 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

// D[128 x N] (TMEM) (+)= A (smem) B (smem), K = 16.  One thread issues.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n"
      " mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((int)accumulate), "n"(kDescHigh)
      : "memory");
}
// As mma_ss with A in TMEM (two 16-bit elements a column, lane = row).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((int)accumulate), "n"(kDescHigh)
      : "memory");
}
// The barrier completes a phase when every matrix instruction this thread
// issued before has finished.
__device__ __forceinline__ void commit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// One full warp allocates / frees; `cols` is a power of two >= 32.
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}

// 8, 16 or 32 consecutive columns of this thread's lane (lane quarter = warp % 4, given
// in the address's bits 16-31); tmem_wait_ld before the values are used.
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
      " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15},"
      " [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Ties values loaded before a tmem_wait_ld to the code after it: the compiler
// sees the loads' registers as ready at once and could use them too early.
template <int N>
__device__ __forceinline__ void after_wait(uint32_t (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}

__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

}  // namespace tc
}  // namespace gs
