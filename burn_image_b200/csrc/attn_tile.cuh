// attn_tile.cuh -- what the attention kernels with scores in TMEM share: waits
// that end every role when one gives up, TMEM reads of 64 columns, and the
// packed and three-input f32 instructions of their softmax.
#pragma once
#include "bq4_internal.h"
#include "sm100_ptx.cuh"

namespace bq4 {

__device__ __forceinline__ bool attn_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  if (ptx::mbar_wait(bar, parity, abort_flag)) return true;
  if (!*abort_flag) {
    *abort_flag = 1;
    if (err) atomicCAS(err, 0, (int)BQ4_ETIMEOUT);
  }
  return false;
}

// As attn_wait, polling with test_wait instead of parking the thread: for the
// MMA issuer, whose wake-up latency after a suspended try_wait (about 170
// cycles, measured) would leave the tensor core idle at every hand-off.
__device__ __forceinline__ bool attn_wait_poll(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  if (ptx::mbar_wait_spin(bar, parity, abort_flag)) return true;
  if (!*abort_flag) {
    *abort_flag = 1;
    if (err) atomicCAS(err, 0, (int)BQ4_ETIMEOUT);
  }
  return false;
}

// 2^x by the PTX instruction ex2.approx.ftz.f32 (one MUFU op; relative error
// near 2^-22, results below 2^-126 flush to 0 -- far under the smallest f16
// probability the P operand can hold).
__device__ __forceinline__ float attn_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Blackwell's three-input max and packed two-lane f32 arithmetic (PTX
// max.f32 with three sources; fma / add .f32x2 on a b64 pair, low lane first).
__device__ __forceinline__ float attn_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t attn_pack2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void attn_unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t attn_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t attn_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Bounded wait that ignores the abort flag: for draining this CTA's own
// copies and MMAs before its shared memory and TMEM are released.
__device__ __forceinline__ void attn_drain(uint64_t* bar, uint32_t parity) {
  volatile int never = 0;
  (void)ptx::mbar_wait(bar, parity, &never);
}

__device__ __forceinline__ void attn_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  ptx::tmem_ld_32x32b_x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(r));
  ptx::tmem_ld_32x32b_x32(taddr + 32, *reinterpret_cast<uint32_t(*)[32]>(r + 32));
  ptx::tmem_ld_wait();
}

}  // namespace bq4
