// Accesses shared by the kernels that walk the rows of partial states (merge_states.cu, merge_rows.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dtb {

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void st_stream(void* p, uint4 v) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Offset of row = (b*S + s)*H + h in an lse tensor.  Rows fit 32 bits (checked by the launchers), so
// the two divisions are 32-bit.
__device__ __forceinline__ uint32_t lse_offset(int layout, uint32_t row, uint32_t H, uint32_t S) {
  if (layout == 1) return row;                    // [B,S,H]
  const uint32_t tok = row / H;
  const uint32_t h = row - tok * H;
  const uint32_t b = tok / S;
  const uint32_t s = tok - b * S;
  return (b * H + h) * S + s;                     // [B,H,S]
}

}  // namespace dtb
