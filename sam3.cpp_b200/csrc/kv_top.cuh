// The k largest of n values, the first among equals, in order of their places: for choosing pages by score and tokens by weight.
#pragma once
#include "kv_cache.cuh"

namespace s3b {

// Unsigned keys that order as the values: NaN below all, -0 as 0. Those of values end at that of +inf, 0xFF800000.
constexpr uint32_t kTopForced = 0xFFFFFFFFu;  // taken before any value
__device__ __forceinline__ uint32_t top_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// a word of the shared memory of CTA `rank` of the cluster, at the place of `p` here
__device__ __forceinline__ uint32_t cluster_load(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(smem_u32(p), rank)) : "memory");
  return v;
}

template <int T>
struct TopShared {
  uint32_t hist[256 * 32];  // a digit's count, apart for each lane: no two lanes of a warp meet in a bank
  uint32_t total[2][256];   // of this CTA, by digit; two of them, so that one round's may still be read during the next
  uint32_t above[T / 32], equal[T / 32], cta[2];
  uint32_t digit, left, count;
};

// Radix selection from the top, 8 bits a round: the digit in which the k-th largest lies, then the same among the keys that
// share it. Each of a cluster's CTAs (CL: 1, or the cluster's size) has the places [first, first + n) of a line; within it each
// warp has a run of rows of 32. key(i) is asked for place i (of the whole line) once where a thread's share fits KPT registers,
// in every round otherwise. emit(position, place, key) is called for the taken ones, k of them in all (k <= the line's length,
// and at least the number of forced keys).
template <int T, int KPT, int CL, typename Key, typename Emit>
__device__ void top_select(TopShared<T>& s, int first, int n, uint32_t k, Key key, Emit emit) {
  constexpr int W = T / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows_all = (n + 31) / 32, rows_warp = (rows_all + W - 1) / W;
  const int base = warp * rows_warp * 32;                       // of this warp's run, from `first`
  const int rows = max(0, min(rows_warp, rows_all - warp * rows_warp));
  const bool kept = rows_warp <= KPT;
  uint32_t keys[KPT];
  if (kept) {
#pragma unroll
    for (int r = 0; r < KPT; ++r) keys[r] = r < rows && base + r * 32 + lane < n ? key(first + base + r * 32 + lane) : 0u;
  }
  // f(row, whether there is a key, key): a whole warp each
  auto each = [&](auto&& f) {
    if (kept) {
#pragma unroll
      for (int r = 0; r < KPT; ++r)
        if (r < rows) f(r, base + r * 32 + lane < n, keys[r]);
    } else {
      for (int r = 0; r < rows; ++r) {
        const bool there = base + r * 32 + lane < n;
        f(r, there, there ? key(first + base + r * 32 + lane) : 0u);
      }
    }
  };
  for (int e = threadIdx.x; e < 256 * 32; e += T) s.hist[e] = 0;
  uint32_t prefix = 0, left = k;
  uint32_t from_above = 1, from_equal = 0;  // keys >= from_above are taken, then the first of those >= from_equal
#pragma unroll 1
  for (int round = 0; round < 4; ++round) {
    const int shift = 24 - 8 * round;
    __syncthreads();
    each([&](int, bool there, uint32_t x) {
      if (there && (round == 0 || (x ^ prefix) >> (shift + 8) == 0)) atomicAdd(&s.hist[(x >> shift & 255) * 32 + lane], 1u);
    });
    __syncthreads();
    for (int bin = warp; bin < 256; bin += W) {
      const uint32_t c = __reduce_add_sync(~0u, s.hist[bin * 32 + lane]);
      s.hist[bin * 32 + lane] = 0;
      if (lane == 0) s.total[round & 1][bin] = c;
    }
    if (CL > 1) cluster_sync_all();
    else __syncthreads();
    if (warp == 0) {  // lane i: the 8 digits from 255 - 8 i down
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) {
          const uint32_t* at = &s.total[round & 1][255 - 8 * lane - e];
          c[e] += CL > 1 ? cluster_load(at, r) : *at;
        }
        sum += c[e];
      }
      uint32_t end = sum;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const uint32_t up = __shfl_up_sync(~0u, end, x);
        if (lane >= x) end += up;
      }
      uint32_t before = end - sum;
      if (before < left && left <= end) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (before < left && left <= before + c[e]) {
            s.digit = 255 - 8 * lane - e;
            s.left = left - before;
            s.count = c[e];
          }
          before += c[e];
        }
      }
    }
    __syncthreads();
    prefix |= s.digit << shift;
    left = s.left;
    if (left == s.count) {  // all that share the digits so far
      from_above = from_equal = prefix;
      left = 0;
      break;
    }
    from_equal = prefix;
    from_above = prefix + 1;  // no overflow: the forced keys, all taken, end in the branch above
  }
  // places of what each warp takes
  uint32_t above = 0, equal = 0;
  each([&](int, bool there, uint32_t x) {
    above += __popc(__ballot_sync(~0u, there && x >= from_above));
    equal += __popc(__ballot_sync(~0u, there && x >= from_equal && x < from_above));
  });
  if (lane == 0) s.above[warp] = above, s.equal[warp] = equal;
  __syncthreads();
  uint32_t a = 0, q = 0;
  for (int w = 0; w < warp; ++w) a += s.above[w], q += s.equal[w];
  if (CL > 1) {
    if (threadIdx.x == T - 32) s.cta[0] = a + above, s.cta[1] = q + equal;  // the last warp's
    cluster_sync_all();
    const uint32_t rank = cluster_rank();
    for (uint32_t r = 0; r < rank; ++r) a += cluster_load(&s.cta[0], r), q += cluster_load(&s.cta[1], r);
  }
  each([&](int r, bool there, uint32_t x) {
    const bool is_above = there && x >= from_above, is_equal = there && x >= from_equal && x < from_above;
    const uint32_t ma = __ballot_sync(~0u, is_above), mq = __ballot_sync(~0u, is_equal), below = (1u << lane) - 1;
    const uint32_t pa = a + __popc(ma & below), pq = q + __popc(mq & below);
    if (is_above || (is_equal && pq < left)) emit(pa + min(pq, left), first + base + r * 32 + lane, x);
    a += __popc(ma);
    q += __popc(mq);
  });
  if (CL > 1) cluster_sync_all();  // no CTA leaves while another reads its counts
}

}  // namespace s3b
