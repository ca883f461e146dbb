// serve.cuh -- helpers shared by the serving operators (packed-prompt and
// single-token attention, few-token MoE, few-token packed products).
//
// Times in the comments of these kernels compare two forms of one kernel, most
// of them as the best of five replays of a graph; a stream of calls over changing
// inputs runs 5 to 15 % longer.
#pragma once

#include <mutex>

#include "apart.cuh"
#include "common.cuh"

namespace ennx {

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr int kMaxServingDevices = 64;
// The current device and the status word that kernels of the serving operators
// write where a bounded wait gave up (static device memory, registered for
// ennx_b200_device_status; nothing is allocated).
int32_t serving_device(int* device, int** status);
// Dynamic shared memory of `kernel`, once per device (a flag and a result each).
int32_t allow_shared_memory(std::once_flag& once, int32_t& result, const void* kernel, int bytes);
struct SharedMemorySetup {
  std::once_flag once[kMaxServingDevices];
  int32_t result[kMaxServingDevices] = {};
};
template <typename K>
int32_t allow_shared_memory(SharedMemorySetup& s, int device, K kernel, int bytes) {
  return allow_shared_memory(s.once[device], s.result[device], (const void*)kernel, bytes);
}

// ---------------------------------------------------------------------------
// device
// ---------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Programmatic launch chain: a kernel lets the next one start (its prologue
// runs early) and waits for the previous one's results.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// contiguous copy, completing on `bar`: 16-byte aligned addresses, a size of a multiple of 16
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// c += a b, 16 x 8 x 16, bf16 with fp32 sums
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Rotary table in turns: angle of pair i at position p is 2*pi * p * inv[i].
// Positions reach 10^5 and more, where a 32-bit product has lost the angle, so
// p * inv[i] is formed and reduced to [-1/2, 1/2] in 64 bits; only the reduced
// turn is rounded to 32 (error 2^-25 turns, 2e-7 radians).
struct RopeTable {
  double inv[64];
};
__device__ __forceinline__ void rope_sincos(double inv, int pos, float* s, float* c) {
  const double turns = (double)pos * inv;
  sincospif((float)(2.0 * (turns - rint(turns))), s, c);
}
// inv[i] for an i of the lane's own.  An indexed read of a parameter goes to the
// constant cache, one lane after another; the generic address does not.
__device__ __forceinline__ double rope_inv(const RopeTable& table, int i) {
  double v;
  asm("ld.f64 %0, [%1];" : "=d"(v) : "l"(table.inv + i));
  return v;
}
// A pair turned.  The operations are spelled out, so that a prompt's pass and a
// token step leave the same bits in a cache.
__device__ __forceinline__ void rope_turn(float& x1, float& x2, float s, float c) {
  const float y1 = fmaf(x1, c, -__fmul_rn(x2, s));
  x2 = fmaf(x2, c, __fmul_rn(x1, s));
  x1 = y1;
}
// host: inv[i] = theta^(-2i/128) / (2*pi)
const RopeTable& rope_table(float theta);

}  // namespace ennx
