// Warp-level bf16 matrix products (m16n8k16, fp32 accumulators) for kernels whose operands change
// between products in registers, where the accumulator-in-tensor-memory form does not fit.
#pragma once
#include "elem.cuh"

namespace cdeep {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// four 8 x 8 bf16 matrices; lane l gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d += a b: a 16 x 16 (row-major fragments), b 16 x 8
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// v0, v1 as two bf16 pairs hi + lo (16 significant bits each)
__device__ __forceinline__ void split_pair(float v0, float v1, uint32_t& hi, uint32_t& lo) {
  hi = bf_pack(v0, v1);
  lo = bf_pack(v0 - bf_lo(hi), v1 - bf_hi(hi));
}
// v0, v1 as three bf16 pairs hi + lo + rest: all of their 24 significant bits, down to the smallest bf16
__device__ __forceinline__ void split_all(float v0, float v1, uint32_t& hi, uint32_t& lo, uint32_t& rest) {
  hi = bf_pack(v0, v1);
  const float r0 = v0 - bf_lo(hi), r1 = v1 - bf_hi(hi);
  lo = bf_pack(r0, r1);
  rest = bf_pack(r0 - bf_lo(lo), r1 - bf_hi(lo));
}

}  // namespace cdeep
