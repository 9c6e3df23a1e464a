// The k largest of n values, the first among equals, in order of their places: for choosing pages by score and tokens by weight.
#pragma once
#include <type_traits>

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
  static constexpr int kCopies = T >= 1024 ? 16 : 8;
  static constexpr int kDigits = T >= 256 ? 256 : 1;  // small blocks take few keys, by votes alone
  uint32_t hist[kDigits * kCopies];  // a digit's counts, apart for lanes that differ modulo kCopies: keys of one size share their digits
  uint32_t total[2][kDigits];        // of this CTA, by digit; two of them, so that one round's may still be read during the next
  uint32_t warp_sum[8];
  uint32_t above[T / 32], equal[T / 32], cta[2];
  uint32_t digit, left, count;
};

// Radix selection from the top, 8 bits a round: the digit in which the k-th largest lies, then the same among the keys that
// share it; it ends with the round in which all of those are taken. Each of a cluster's CL CTAs has n places of a line, one CTA's
// behind another's; within a CTA each warp has a run of rows of 32. In the first round make(i, fetch(i)) gives the key of its place
// i (all of a step's fetches come before its makes, which may write: 18000 cycles otherwise, 128 KB at one load's latency after
// the other's), key(i) after that: from shared memory where they fit. emit(position, place) is called for the taken ones, k of
// them in all (0 < k <= the line's length, and at least the number of forced keys).
// Measured (cycles of the SM), 16 CTAs of 1024 threads and 32768 keys each: a round 5000 to 7000 to count (instructions, and the
// atomics on shared memory), 500 to add up, 3700 for the cluster to meet and find the digit; 6000 to count what is taken, 9000 to
// write it. 256 keys, 256 threads: see the branch for few keys.
template <int T, int CL, typename Fetch, typename Make, typename Key, typename Emit>
__device__ void top_select(TopShared<T>& s, int n, uint32_t k, Fetch fetch, Make make, Key key, Emit emit) {
  constexpr int W = T / 32, C = TopShared<T>::kCopies, P = T >= 256 ? T / 256 : 1;  // P threads a digit
  static_assert(T >= 256 ? T % 256 == 0 && C % P == 0 : T % 32 == 0 && CL == 1, "threads of top_select");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows_all = (n + 31) / 32, rows_warp = (rows_all + W - 1) / W;
  const int from = min(warp * rows_warp, rows_all) * 32, to = min(n, from + rows_warp * 32);  // of this warp's run
  // f(whether there is a key, place, key): a whole warp each. Full steps know that there is.
  auto each_of = [&](auto&& of, auto unroll, auto&& f) {
    constexpr int U = decltype(unroll)::value;
    decltype(of(0)) x[U];
    int i0 = from + lane;
    for (; i0 - lane + 32 * U <= to; i0 += 32 * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = of(i0 + 32 * u);
#pragma unroll
      for (int u = 0; u < U; ++u) f(std::true_type(), i0 + 32 * u, x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = i0 + 32 * u < to ? of(i0 + 32 * u) : decltype(of(0))(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 - lane + 32 * u < to) f(i0 + 32 * u < to, i0 + 32 * u, x[u]);
  };
  auto each = [&](auto&& f) { each_of(key, std::integral_constant<int, 4>(), f); };
  uint32_t left = k;
  uint32_t from_above = 1, from_equal = 0;  // keys >= from_above are taken, then the first of those >= from_equal
  if (T < 256 || (CL == 1 && n <= 2 * T)) {
    // Few keys, one or two a thread: the threshold bit by bit, by the block's votes (some 50 cycles each, and most searches end well
    // before the last bit: 256 keys in 1000 cycles where two rounds below take 2500).
    const bool two = n > T;  // a run is one row, or two
    const int i = from + lane, i2 = i + 32;
    const bool there = i < to, there2 = i2 < to;
    const uint32_t x = there ? make(i, fetch(i)) : 0u, x2 = there2 ? make(i2, fetch(i2)) : 0u;
    auto votes = [&](uint32_t at) {
      uint32_t c = __syncthreads_count(there && x >= at);
      if (two) c += __syncthreads_count(there2 && x2 >= at);
      return c;
    };
    uint32_t count = 0;
    for (int bit = 31; bit >= 0 && count != k; --bit) {
      const uint32_t at = from_equal | 1u << bit, c = votes(at);
      if (c >= k) from_equal = at, count = c;
    }
    from_above = from_equal;
    left = 0;
    if (count != k) {  // equal ones are left out (no forced key is: they are at most k)
      from_above = from_equal + 1;
      left = k - votes(from_above);
    }
  } else if constexpr (T >= 256) {
#pragma unroll
    for (int e = 0; e < 256 * C / T; ++e) s.hist[e * T + threadIdx.x] = 0;
    uint32_t prefix = 0;
#pragma unroll 1
    for (int round = 0; round < 4; ++round) {
      const int shift = 24 - 8 * round;
      __syncthreads();
      if (round == 0) {
        each_of(fetch, std::integral_constant<int, 8>(), [&](auto there, int i, decltype(fetch(0)) v) {
          if (there) atomicAdd(&s.hist[(make(i, v) >> 24) * C + lane % C], 1u);
        });
      } else {
        each([&](auto there, int, uint32_t x) {
          if (there && (x ^ prefix) >> (shift + 8) == 0) atomicAdd(&s.hist[(x >> shift & 255) * C + lane % C], 1u);
        });
      }
      __syncthreads();
      {  // the digit's copies, P threads share them; rotated, so that a warp's lanes meet in no bank
        uint32_t* h = s.hist + threadIdx.x / P * C;
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < C / P; ++e) {
          const int at = (threadIdx.x % P) * (C / P) + (e + threadIdx.x / (P * (32 / C))) % (C / P);
          c += h[at];
          h[at] = 0;
        }
#pragma unroll
        for (int x = 1; x < P; x <<= 1) c += __shfl_xor_sync(~0u, c, x);
        if (threadIdx.x % P == 0) s.total[round & 1][threadIdx.x / P] = c;
      }
      if (CL > 1) cluster_sync_all();
      else __syncthreads();
      uint32_t c = 0, end = 0;
      if (warp < 8) {  // thread i: digit 255 - i, and how many have it or a higher one
        const uint32_t* at = &s.total[round & 1][255 - threadIdx.x];
        if (CL > 1) {
#pragma unroll
          for (int r = 0; r < CL; ++r) c += cluster_load(at, r);
        } else {
          c = *at;
        }
        end = c;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const uint32_t up = __shfl_up_sync(~0u, end, x);
          if (lane >= x) end += up;
        }
        if (lane == 31) s.warp_sum[warp] = end;
      }
      __syncthreads();
      if (warp < 8) {
#pragma unroll
        for (int w = 0; w < 7; ++w)
          if (w < warp) end += s.warp_sum[w];
        if (end - c < left && left <= end) {
          s.digit = 255 - threadIdx.x;
          s.left = left - (end - c);
          s.count = c;
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
  }
  // places of what each warp takes (counted by lanes: POPC runs at an eighth of the rate of an addition)
  uint32_t above = 0, equal = 0;
  each([&](auto there, int, uint32_t x) {
    above += there && x >= from_above;
    equal += there && x >= from_equal && x < from_above;
  });
  above = __reduce_add_sync(~0u, above);
  equal = __reduce_add_sync(~0u, equal);
  if (lane == 0) s.above[warp] = above, s.equal[warp] = equal;
  __syncthreads();
  uint32_t a = lane < warp ? s.above[lane] : 0, q = lane < warp ? s.equal[lane] : 0;
  a = __reduce_add_sync(~0u, a);
  q = __reduce_add_sync(~0u, q);
  if (CL > 1) {
    if (threadIdx.x == T - 32) s.cta[0] = a + above, s.cta[1] = q + equal;  // the last warp's
    cluster_sync_all();
    const uint32_t rank = cluster_rank();
    uint32_t ca = lane < (int)rank ? cluster_load(&s.cta[0], lane) : 0, cq = lane < (int)rank ? cluster_load(&s.cta[1], lane) : 0;
    a += __reduce_add_sync(~0u, ca);
    q += __reduce_add_sync(~0u, cq);
    // no CTA leaves while another reads its counts: this one has read those of others
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
  each([&](auto there, int i, uint32_t x) {
    const bool is_above = there && x >= from_above, is_equal = there && x >= from_equal && x < from_above;
    const uint32_t ma = __ballot_sync(~0u, is_above), mq = left ? __ballot_sync(~0u, is_equal) : 0u, below = (1u << lane) - 1;
    if (!(ma | mq)) return;
    uint32_t at = a + __popc(ma & below);
    a += __popc(ma);
    bool taken = is_above;
    if (mq) {
      const uint32_t before = q + __popc(mq & below);
      taken |= is_equal && before < left;
      at += min(before, left);
      q += __popc(mq);
    } else {
      at += min(q, left);
    }
    if (taken && at < k) emit(at, i);  // more only where the caller changes the values meanwhile
  });
  if (CL > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// kernel_setup for a kernel whose blocks form clusters of `cluster`. 16 are more than every GPU takes: they have to be allowed, and
// where none finds its place the set-up fails (and a smaller cluster is taken).
inline int wide_clusters(const void* kernel, size_t smem, int threads) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 16;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(16);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0)
    return n;
  cudaGetLastError();
  return -13;
}
template <typename K>
int cluster_setup(K* kernel, size_t smem, int threads, int cluster) {
  return kernel_setup(reinterpret_cast<const void*>(kernel), smem, cluster > 8 ? wide_clusters : nullptr, threads);
}

// Launch of such a kernel, which may take its place while its predecessor runs.
template <typename K, typename... A>
int launch_clusters(K* kernel, unsigned grid, int threads, size_t smem, unsigned cluster, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? 0 : -12;
}

}  // namespace s3b
