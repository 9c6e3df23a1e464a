// Shared by the two attention kernels over the quantised cache: which tokens a query sees, codes to f16, output stores.
#pragma once
#include "kv_cache.cuh"

namespace s3b {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoScore = -1e30f;  // reference maximum before the first visible token: finite, so that no inf - inf arises

// Tokens of sequence b, held to what its page table can name.
__device__ __forceinline__ int sequence_length(const KvAttnParams& p, int b, int* err) {
  const int n = p.lengths[b];
  const int most = p.max_pages * p.c.page_size;
  if (n < 0 || n > most) {
    atomicCAS(err, 0, kDevErrIndex);
    return n < 0 ? 0 : most;
  }
  return n;
}

// Tokens [lo, hi) that query i of a sequence of len tokens sees.
__device__ __forceinline__ void row_span(const KvAttnParams& p, int len, int i, int* lo, int* hi) {
  *lo = 0;
  *hi = len;
  if (p.causal) {
    *hi = max(0, len - p.nq + i + 1);
    if (p.window) *lo = max(0, *hi - p.window);
  }
}

// Groups of 16 tokens [g0, g1) that queries [i0, i1] of a sequence of len tokens see between them.
__device__ __forceinline__ void group_span(const KvAttnParams& p, int len, int i0, int i1, int* g0, int* g1) {
  int lo, hi, none;
  row_span(p, len, i0, &lo, &none);
  row_span(p, len, i1, &none, &hi);
  *g0 = lo >> 4;
  *g1 = max(*g0, (hi + 15) >> 4);
}

__device__ __forceinline__ void store_out(const KvAttnParams& p, long long at, float4 v) {
  if (p.out_f32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = v;
  } else {
    __half2 h[2] = {__floats2half2_rn(v.x, v.y), __floats2half2_rn(v.z, v.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + at) = *reinterpret_cast<uint2*>(h);
  }
}

// Asynchronous copy of `bytes` (a multiple of 16) from 16-byte aligned global memory, counted on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ---------------------------------------------------------------- codes
__device__ __forceinline__ uint32_t h2_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u32_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// (w & MASK) | 0x64006400 in one instruction
template <uint32_t MASK>
__device__ __forceinline__ uint32_t under_1024(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(0x64006400u));
  return r;
}

// Exact f16 pairs of the codes (less 8 for q4_0) whose nibbles lie at bits 0, 4, 8, 12 of each half of w: a nibble under
// the exponent of 1024 reads 1024 + c at bit 0 and 1024 + 16 c at bit 4; one subtraction (or multiply-add by 1/16)
// leaves the integer.
template <int QT>
__device__ __forceinline__ void nibble_pairs(uint32_t w, uint32_t (&out)[4]) {
  const __half2 off0 = u32_h2(QT == QT_Q4_0 ? 0xE408E408u : 0xE400E400u);  // -1032, -1024
  const __half2 off1 = u32_h2(QT == QT_Q4_0 ? 0xD480D480u : 0xD400D400u);  // -72, -64
  const __half2 sixteenth = u32_h2(0x2C002C00u);
  const uint32_t x = w >> 8;
  out[0] = h2_u32(__hadd2(u32_h2(under_1024<0x000F000Fu>(w)), off0));
  out[1] = h2_u32(__hfma2(u32_h2(under_1024<0x00F000F0u>(w)), sixteenth, off1));
  out[2] = h2_u32(__hadd2(u32_h2(under_1024<0x000F000Fu>(x)), off0));
  out[3] = h2_u32(__hfma2(u32_h2(under_1024<0x00F000F0u>(x)), sixteenth, off1));
}
// The same for the bytes 0, 1 and 2, 3 of w (8-bit codes with 128 added).
__device__ __forceinline__ void byte_pairs(uint32_t w, uint32_t& a, uint32_t& b) {
  const __half2 off = u32_h2(0xE480E480u);  // -1152
  a = h2_u32(__hadd2(u32_h2(__byte_perm(w, 0x64646464u, 0x4140)), off));
  b = h2_u32(__hadd2(u32_h2(__byte_perm(w, 0x64646464u, 0x4342)), off));
}

}  // namespace s3b
