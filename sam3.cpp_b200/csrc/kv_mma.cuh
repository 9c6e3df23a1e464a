// Fragments of the warp-wide products over the quantised key / value cache.
#pragma once
#include "kv_attention.cuh"

namespace s3b {

// ---------------------------------------------------------------- fragments
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same onto zeros
__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// transpose of the 8 x 8 matrix of 16-bit values that a warp holds as one m8n8 fragment
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <int BYTES>
__device__ __forceinline__ void lds(const uint8_t* at, uint32_t (&r)[BYTES / 4]) {
  if (BYTES == 4) {
    r[0] = *reinterpret_cast<const uint32_t*>(at);
  } else if (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    r[0] = v.x;
    r[BYTES >= 8 ? 1 : 0] = v.y;
    r[BYTES >= 8 ? BYTES / 4 - 2 : 0] = v.z;
    r[BYTES / 4 - 1] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    r[0] = v.x;
    r[BYTES >= 8 ? 1 : 0] = v.y;
  }
}

}  // namespace s3b
