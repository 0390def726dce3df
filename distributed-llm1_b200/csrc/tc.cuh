// tc.cuh — device helpers of the tcgen05 kernels: mbarriers, TMA tile loads, shared-
// memory matrix descriptors, MMA issue and tensor-memory access (hand-written PTX for
// sm_100a), and the host's tensor-map encoder.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace dllm {

constexpr long long kTcWaitCycles = 1ll << 32;  // ~2 s of SM cycles

DLLM_DEV uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

DLLM_DEV void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
DLLM_DEV void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// Bounded wait for completion of the phase with parity `parity`.
DLLM_DEV bool mbar_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t a = smem_u32(bar);
  const long long t0 = clock64();
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
    if (clock64() - t0 > kTcWaitCycles) return false;
  }
}

// 2-D tiled TMA load of box (x = K offset, y = row offset) into shared memory,
// completing on `bar` (no multicast: the tensor always lies in this GPU's memory).
DLLM_DEV void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// Shared-memory matrix descriptor of a K-major tile written by TMA with the
// 128-byte swizzle: rows of 128 bytes, 8-row groups 1024 bytes apart (stride
// byte offset 1024 >> 4), leading byte offset unused (1), descriptor version 1,
// layout type 2 (SWIZZLE_128B). The tile base must be 1024-byte aligned.
DLLM_DEV uint64_t umma_desc_sw128(const void* tile) {
  const uint64_t a = smem_u32(tile);
  return ((a & 0x3FFFFull) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// D[tmem] (+)= A[128 x 16] * B[N x 16]^T, bf16 inputs, fp32 accumulate.
DLLM_DEV void umma_bf16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Arrive on `bar` once every tcgen05.mma this thread issued so far has completed.
DLLM_DEV void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
DLLM_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
DLLM_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 8 consecutive fp32 accumulator columns of this thread's TMEM lane.
DLLM_DEV void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
DLLM_DEV void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

DLLM_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Waits for a phase, at most about 2 s (200000 tries of up to 10 us each), and less once
// another wait of the CTA has given up: then it returns false at once, and the CTA runs on
// through its loops without waiting, computes nothing of use, reports the error and ends.
// One asm block, so that the compiler sees no branch: a warp that issues MMAs has to stay
// one piece (a loop with votes cost 200 cycles even where the phase had completed).
DLLM_DEV bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n, gone;\n\t"
      "mov.u32 n, 0;\n\t"
      "mov.u32 %0, 1;\n\t"
      "TRY:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 10000;\n\t"
      "@p bra DONE;\n\t"
      "ld.volatile.shared.u32 gone, [%3];\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.ne.u32 q, gone, 0;\n\t"
      "setp.gt.or.u32 q, n, 200000, q;\n\t"
      "@!q bra TRY;\n\t"
      "mov.u32 %0, 0;\n\t"
      "st.volatile.shared.u32 [%3], 1;\n\t"
      "DONE:\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(smem_u32(const_cast<const int*>(abort)))
      : "memory");
  return ok;
}
DLLM_DEV uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}

// D[tmem] (+)= A[tmem, 128 x 16] * B[16 x N]: the A operand as packed bf16 pairs, 8 columns.
DLLM_DEV void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Shared-memory descriptor of a 16 x N operand whose contiguous direction is the MMA's N
// (dims): rows of 64 dims (128 bytes, swizzled), one per K index (slot), 8-slot groups 1024
// bytes apart (stride offset), 64-dim boxes `box` bytes apart (leading offset).
DLLM_DEV uint64_t umma_desc_mn_sw128(const void* tile, uint32_t box) {
  const uint64_t a = smem_u32(tile);
  return ((a & 0x3FFFFull) >> 4) | ((uint64_t)(box >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

#define R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 consecutive columns of this thread's lane.
DLLM_DEV void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24)
      : "r"(addr));
}
DLLM_DEV void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::W8(r, 0), "r"(addr)
               : "memory");
}
#undef R8
#undef W8
DLLM_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Row-major bf16 [outer][inner] as a 2-D tensor map with a (64 x box_rows) box and the
// 128-byte swizzle (gemm_tc.cu).
bool tc_encode_rows(CUtensorMap* m, const void* base, int inner, int outer, int box_rows);
// Row-major fp32 [outer][inner] as a 2-D tensor map with an (inner x box_rows) box, as it lies.
bool tc_encode_rows_f32(CUtensorMap* m, const void* base, int inner, int outer, int box_rows);

}  // namespace dllm
