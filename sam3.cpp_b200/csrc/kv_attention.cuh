// Shared by the two attention kernels over the quantised cache: which tokens a query sees, codes to f16, output stores.
#pragma once
#include "kv_cache.cuh"

namespace s3b {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoScore = -1e30f;  // reference maximum before the first visible token: finite, so that no inf - inf arises, and
                                    // below every score (f16 sums, a scale of 2^56 at most)

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

}  // namespace s3b
