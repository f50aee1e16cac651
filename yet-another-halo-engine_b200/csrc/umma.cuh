// tcgen05 pieces of the attention kernels that run as CTA pairs (prefill_attn.cu, shared_attn.cu): operand and instruction
// descriptors, the pair MMA, commits, tensor-memory loads and stores, and the bounded, abortable barrier wait.
#pragma once

#include "ptx.cuh"

namespace yahkv {

// Shared-memory matrix descriptors, 128-byte swizzle (layout type 2), descriptor version 1: bits 0-13 start address
// >> 4, 16-29 leading byte offset >> 4, 32-45 stride byte offset >> 4, bit 46 version, 61-63 layout.
//   K-major operand  [rows][64 fp16]: rows 128 B apart, groups of 8 rows 1024 B apart (stride byte offset).
//   MN-major operand [keys][64 fp16] x blocks: 8-key groups 1024 B apart (stride), 64-element blocks `lbo` apart.
// The high word is the same for every operand.
constexpr std::uint32_t kDescHi = (1024U >> 4) | (1U << 14) | (2U << 29);
__device__ __forceinline__ std::uint32_t DescLo(std::uint32_t addr, std::uint32_t lbo_bytes) {
  return ((addr >> 4) & 0x3FFFU) | (((lbo_bytes >> 4) & 0x3FFFU) << 16);
}
// Instruction descriptor of kind::f16: fp16 A and B, fp32 accumulate, A K-major.
__host__ __device__ constexpr std::uint32_t InstrDesc(int m, int n, bool b_mn_major) {
  return (1U << 4) | (0U << 7) | (0U << 10) | (0U << 15) | ((b_mn_major ? 1U : 0U) << 16) |
         (static_cast<std::uint32_t>(n >> 3) << 17) | (static_cast<std::uint32_t>(m >> 4) << 24);
}

// D(tmem) (+)= A * B over the CTA pair: M = 256 (128 rows in each CTA's tensor memory, the same columns in both), the
// B half of each CTA from its shared memory at the same offset. Issued by one thread of the leader CTA.
//   Ts: A from each CTA's own tensor memory (two fp16 per 32-bit column). Q is held there for the whole CTA: with it
//       in shared memory the kernel was bound by shared-memory bandwidth (the 64 KB tile re-read for every key tile).
//   Ss: A from each CTA's own shared memory (descriptor), used for P.
__device__ __forceinline__ void UmmaF16Ts2(std::uint32_t d_tmem, std::uint32_t a_tmem, std::uint32_t b_desc_lo,
                                           std::uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 bd;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "mov.b64 bd, {%2, %3};\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], bd, %4, p;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_desc_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate ? 1U : 0U)
      : "memory");
}
__device__ __forceinline__ void UmmaF16Ss2(std::uint32_t d_tmem, std::uint32_t a_desc_lo, std::uint32_t b_desc_lo,
                                           std::uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 ad, bd;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "mov.b64 ad, {%1, %3};\n"
      "mov.b64 bd, {%2, %3};\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %4, p;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_desc_lo), "r"(b_desc_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate ? 1U : 0U)
      : "memory");
}
// Arrives, once every tcgen05 operation this thread issued before has completed, on the barrier at this shared-memory
// offset in both CTAs of the pair (one commit per CTA).
__device__ __forceinline__ void UmmaCommitPair(std::uint64_t* bar) {
  const std::uint32_t a = SmemAddr(bar);
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(MapToCta(a, 0))
               : "memory");
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(MapToCta(a, 1))
               : "memory");
}
__device__ __forceinline__ void TcFenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void TcFenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void TmemLd32(std::uint32_t addr, std::uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void TmemSt32(std::uint32_t addr, const std::uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void TmemLd16(std::uint32_t addr, std::uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void TmemSt16(std::uint32_t addr, const std::uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void TmemWaitLd() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void TmemWaitSt() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded, abortable wait: gives up after ~2 s or as soon as another role of this CTA has raised the abort flag.
// kCluster: the barrier is arrived on from the other CTA of the pair (acquire at cluster scope).
template <bool kCluster = false>
__device__ __forceinline__ bool WaitOrAbort(std::uint64_t* bar, std::uint32_t parity, volatile int* abort_flag) {
  auto poll = [&]() { return kCluster ? MbarTryWaitCluster(bar, parity) : MbarTryWait(bar, parity); };
  if (poll()) return true;
  const std::uint64_t t0 = GlobalTimerNs();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (poll()) return true;
    if (*abort_flag != 0) return false;
    if (GlobalTimerNs() - t0 > 2000000000ULL) {
      *abort_flag = 1;
      return false;
    }
  }
}

}  // namespace yahkv
