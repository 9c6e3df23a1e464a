// Attention over the quantised key / value cache (layout: kv_cache.cuh).
//   s_j = scale * q . k_j,  p_j = exp(s_j - max s),  out = sum_j p_j v_j / sum_j p_j
// over the tokens j that the query sees.
//
// Few query rows (rows of one key / value head = queries x heads of its group; up to 32, 16 at d = 256): rows_kernel. The
// cache is read once, so HBM is the floor; the products run on m16n8k16 fragments whose A operand is the cache (16 tokens,
// or 16 values of a row) and whose 8 columns are the query rows, so that a single row wastes no more than the padding of
// its column. Codes enter the products as exact small integers; a block's scale multiplies the 32-value partial score in
// f32 (keys), or the weight before it is rounded to f16 (values), so no dequantised value is ever formed. What is rounded
// to f16 is the weight (as every f16 product of this kind does; sums of weights are f32 of the unrounded ones) and weight
// times scale: the output is off by 3.5e-4 of its norm, where rounding it to f16 alone costs 2.1e-4, for values of any size
// (ScaleRange keeps both in f16's normal range).
//
// Measured: 32 sequences of 1384 to 16384 tokens, 32 heads on 8, d = 128, q4_0: 319 MB in 82 us, 3.9 TB/s of the 6.5 that a
// copy reaches; one sequence of 524288 tokens, 16 heads on 2, q4_1: 168 MB in 53 us. Instruction issue bounds it (62% of
// the cycles issue, the integer pipe is half busy): some 350 instructions for 16 tokens of a head, most of them unpacking
// codes and scaling partial scores and weights. Looking at the scales of each step (ScaleRange) is 3% of the time. The output's
// and the query's registers leave 33 of the 48 variants 4 to 84 bytes of spills a thread (one query tile of d = 128 in q4_0: 24
// and 32, in q4_1 16 and 32).
#include <algorithm>

#include "kv_attention.cuh"

namespace s3b {

namespace {

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

// ---------------------------------------------------------------- range of the values' scales
// A weight w and its product w * scale are f16, and scales reach from 2^-24 to 2^13. So that neither of the two passes f16's
// largest, and both keep their digits for tokens far below the maximum whatever the size of the values:
//   weights are 2^kBias at the reference (and up to 2^(kBias + 2.9));
//   for each of the D / 32 blocks of a row a warp holds a bound 2^A on the scales that it has met (A only grows). Where A
//   lies outside kLow .. kHigh, the block's scales and minima are multiplied by 2^lift, lift = kHigh - A, in shared memory before
//   their use, and its outputs by 2^-lift at the end.
// A product then goes below f16's normal range (2^-14) for tokens whose weight is 2^-17 of the largest or less, and to zero
// below 2^-28. The zone without a lift holds values (largest of a block) from 1/16 to 64 in q4_0, 1/8 to 120 in q8_0.
// Lane i holds the state of block i % (2 NB) / 2, whose scales it reads.
template <int QT, int NB>
struct ScaleRange {
  static constexpr int kBias = QT == QT_Q8_0 ? 13 : 10;
  static constexpr int kHigh = 13 - kBias, kLow = kHigh - 8;
  uint32_t limit = 0, limit_min = 0;  // 2^A as f16 twice, the same for the minima; 0: everything passes it
  bool lifted = false;                // any block of the warp
  __device__ __forceinline__ bool passed(uint32_t x, bool minima) const {
    return !__hblt2(__habs2(u32_h2(x)), u32_h2(minima ? limit_min : limit));
  }
  __device__ __forceinline__ int lift() const {
    const int a = (int)(limit >> 26) - 15;
    return a < kLow || a > kHigh ? min(kHigh - a, 15) : 0;
  }
  __device__ __forceinline__ uint32_t factor() const { return (uint32_t)(15 + lift()) * 0x04000400u; }
  __device__ __forceinline__ float lowered() const { return __int_as_float((127 - lift()) << 23); }
  // Takes in the largest scale and minimum (f16 bits) that this lane has seen of a step; returns the factor on its block's
  // outputs so far that comes of it. The whole warp.
  __device__ __forceinline__ float raise(uint32_t most, uint32_t most_min) {
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      if (x > 1 && x < 2 * NB) continue;
      most = max(most, __shfl_xor_sync(~0u, most, x));
      if (QT == QT_Q4_1) most_min = max(most_min, __shfl_xor_sync(~0u, most_min, x));
    }
    const int before = lift();
    if (most >= (limit & 0xFFFF) || (QT == QT_Q4_1 && most_min >= (limit_min & 0xFFFF))) {
      // twice to four times the largest; where there is a lift, the minima have to be below 2^(A + 4)
      int a = max(max((int)(limit >> 26) - 15, (int)(most >> 10) - 13), -14);
      if (QT == QT_Q4_1 && a < kLow) a = max(a, min((int)(most_min >> 10) - 17, kLow));
      a = min(a, 14);
      limit = (uint32_t)(15 + a) * 0x04000400u;
      limit_min = a < kLow ? (uint32_t)(19 + a) * 0x04000400u : 0x7C007C00u;
    }
    lifted = __any_sync(~0u, lift() != 0);
    return __int_as_float((127 + lift() - before) << 23);
  }
};

// ---------------------------------------------------------------- few query rows
// The work is one line of chunks of W groups of 16 tokens, unit after unit (a unit is one sequence and key / value
// head), cut into equal shares for the CTAs, so sequences of uneven length leave no SM idle and one long sequence
// spreads over all of them. In a share each warp takes every W-th group: its own ring of bulk copies, its own running
// maximum, sum and output (no barrier in the loop); the W states are joined in shared memory at the end of a unit's
// part. A unit that several CTAs share leaves its parts in the workspace and the last CTA to arrive joins them in the
// order of the shares, so the result does not depend on who that is. (A kernel of its own for the joins took 16 us instead of
// 24 for 8 sequences of 4096 tokens, 16 rows of 256, but 73 instead of 67 for 256 sequences of 100 to 1000 tokens, 32 heads on
// 8, whose few parts are joined beside other blocks' work here.)
template <int QT, int D, int NT, int W>
struct Rows {
  typedef KvL<QT, D> L;
  static constexpr int kRows = 8 * NT;
  static constexpr bool kQSmem = NT * D > 128;  // the query fragments of more would not fit beside the output's registers
  // Warps of an SM, each with its ring: the output takes NT * D / 4 registers, so 128, 168 or 255 registers a thread (12
  // instead of 16 warps at 64 output registers: 16 rows of d = 128 133 -> 123 us, d = 256 61 -> 60 us; at 32 it cost 5%).
  static constexpr int kWarps = NT * D >= 512 || (QT == QT_Q8_0 && D == 256) ? 8 : NT * D >= 256 ? 12 : 16;
  static constexpr int kCtas = kWarps / W;
  static constexpr int kQBytes = kQSmem ? NT * L::kNB * 512 : 0;
  static constexpr int kOStride = D + 4;        // floats; the padding spreads the rows of a store over the banks
  static constexpr int kJoin = W * kRows * kOStride * 4;
  static constexpr int kFixed = kQBytes + 3 * W * kRows * 4 + 1024;
  static constexpr int kBudget = (225 * 1024) / kCtas - kFixed - 1024;
  // groups of 16 tokens of a step: two share the waits, the votes and the copies where two stages of them fit
  static constexpr int kG = NT == 1 && D <= (QT == QT_Q8_0 ? 64 : 128) ? 2 : 1;
  static constexpr int kStageBytes = kG * 2 * L::kHalf;
  static constexpr int kFit = kBudget / (W * kStageBytes);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kRing = W * kStages * kStageBytes;
  static constexpr int kMain = kRing > kJoin ? kRing : kJoin;
  static constexpr int kSmem = kMain + kFixed;
  static_assert(kStages >= 2 && kMain + kFixed + 1024 <= (227 * 1024) / kCtas, "shared memory of rows_kernel");
};

struct RowsArgs {
  KvAttnParams p;
  float* part;  // [2 * grid] x (kRows * D outputs, kRows maxima, kRows sums)
  int* count;   // [units], zero between launches
};

template <int QT, int D, int NT, int W>
__global__ void __launch_bounds__(32 * W, Rows<QT, D, NT, W>::kCtas)
    rows_kernel(const __grid_constant__ RowsArgs a, int* err) {
  typedef KvL<QT, D> L;
  typedef Rows<QT, D, NT, W> C;
  constexpr int NB = L::kNB, NS = C::kStages, G = C::kG;
  typedef ScaleRange<QT, NB> Range;
  constexpr float kBias = Range::kBias;
  constexpr float kLazy = 2.9f;  // log2 by which a score may pass the reference: 2^(kBias + 2.9) < 65504
  // Units of at most so many chunks stay whole where there is a block for each: two or three more chunks for a block cost less
  // than joining parts (8 heads of 128, 2 chunks each: 10.3 us cut, 9.5 whole; 8 of 256, 3 chunks: 16.4, 14.3; 4 of 64, 3 chunks:
  // 9.3, 8.7; but 8 of 128, 3 chunks: 10.7, 11.6, and 4 chunks 10.9, 13.7).
  constexpr int kWhole = 3;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* s_q = smem + C::kMain;
  float* s_m = reinterpret_cast<float*>(s_q + C::kQBytes);  // [W][rows]
  float* s_l = s_m + W * C::kRows;
  float* s_f = s_l + W * C::kRows;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_f + W * C::kRows);
  __shared__ long long s_total, s_ctas, s_base, s_p0, s_p1;
  __shared__ int s_b, s_abort_word, s_last;
  volatile int* s_abort = &s_abort_word;
  static_assert(W * NS * 8 <= 1024, "barriers of rows_kernel");

  const KvAttnParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group_heads = p.heads / p.c.heads;
  const int n_rows = p.nq * group_heads;
  const int per_page = p.c.page_size >> 4;

  auto chunks_of = [&](int b, int* g0, int* g1) -> int {
    group_span(p, sequence_length(p, b, err), 0, p.nq - 1, g0, g1);
    return (*g1 - *g0 + W * G - 1) / (W * G);
  };

  if (threadIdx.x < W * NS) mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) {
    s_abort_word = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  let_next();
  wait_before();
  // total chunks, this CTA's share of them and the sequence in which it begins
  if (warp == 0) {
    long long total = 0;
    int most = 0, g0, g1;
    for (int b = lane; b < p.batch; b += 32) {
      const int n = chunks_of(b, &g0, &g1);
      total += n;
      most = max(most, n);
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) total += __shfl_xor_sync(~0u, total, x);
    most = __reduce_max_sync(~0u, most);
    total *= p.c.heads;
    long long ctas = min((long long)gridDim.x, total), base = 0, p0 = 0, p1 = 0;
    int found = -1;
    if (most <= kWhole && (long long)p.batch * p.c.heads <= gridDim.x) {
      const int b = blockIdx.x / p.c.heads;
      if (b < p.batch) {
        const int n = chunks_of(b, &g0, &g1);
        found = b;
        p0 = (blockIdx.x - b * p.c.heads) * n;
        p1 = p0 + n;
      }
    } else if ((int)blockIdx.x < ctas) {
      p0 = total * blockIdx.x / ctas;
      p1 = total * (blockIdx.x + 1) / ctas;
      for (int b0 = 0; b0 < p.batch && found < 0; b0 += 32) {
        const long long n = b0 + lane < p.batch ? (long long)chunks_of(b0 + lane, &g0, &g1) * p.c.heads : 0;
        long long end = n;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const long long up = __shfl_up_sync(~0u, end, x);
          if (lane >= x) end += up;
        }
        const uint32_t past = __ballot_sync(~0u, base + end > p0);
        if (past) {
          const int who = __ffs(past) - 1;
          found = b0 + who;
          base += __shfl_sync(~0u, end - n, who);
        } else {
          base += __shfl_sync(~0u, end, 31);
        }
      }
    }
    if (lane == 0) {
      s_total = total;
      s_ctas = ctas;
      s_base = base;
      s_p0 = p0;
      s_p1 = p1;
      s_b = found;
    }
  }
  __syncthreads();

  // sequences of which no query sees a token
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    int g0, g1;
    if (chunks_of(b, &g0, &g1)) continue;
    for (int e = threadIdx.x; e < p.nq * p.heads * (D / 4); e += 32 * W) {
      const int h = e / (D / 4) % p.heads, i = e / (D / 4) / p.heads;
      store_out(p, b * p.o_b + i * p.o_n + h * p.o_h + e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
      if (p.lse && e % (D / 4) == 0) p.lse[((long long)b * p.nq + i) * p.heads + h] = -INFINITY;
    }
  }
  const long long p0 = s_p0, p1 = s_p1, total = s_total, ctas = s_ctas;
  if (p0 >= p1) return;

  const float sl2 = p.scale * kLog2e;
  const long long v_offset = (long long)per_page * L::kHalf;  // of a page's values from its keys
  uint8_t* ring = smem + warp * NS * C::kStageBytes;
  uint64_t* full = bars + warp * NS;
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;

  long long pos = p0, base = s_base;
  for (int b = s_b; pos < p1; ++b) {
    int g0, g1;
    const int n_chunks = chunks_of(b, &g0, &g1);
    const int len = sequence_length(p, b, err);
    int min_lo, max_lo, min_hi, max_hi;  // of the spans of the unit's rows
    row_span(p, len, 0, &min_lo, &min_hi);
    row_span(p, len, p.nq - 1, &max_lo, &max_hi);
    const int* table = p.pages + b * p.pages_stride;
    for (; pos < p1 && pos < base + (long long)n_chunks * p.c.heads;) {
      const int head = (int)((pos - base) / n_chunks);
      const long long unit_start = base + (long long)head * n_chunks;
      const int ca = (int)(pos - unit_start);
      const int cb = (int)min((long long)n_chunks, p1 - unit_start);
      pos += cb - ca;

      // ---- this warp's groups: G from g0 + (chunk * W + warp) * G
      const int first = g0 + (ca * W + warp) * G;
      const int n_it = first < g1 ? min(cb - ca, (g1 - first + W * G - 1) / (W * G)) : 0;
      long long src = 0;  // lane i: address of group i % G of step (of a batch of 32 / G) + i / G
      auto locate = [&](int it0) {
        const int gi = first + (it0 + lane / G) * (W * G) + lane % G;
        if (it0 + lane / G < n_it && gi < g1) {
          long long page = table[gi / per_page];
          if (page < 0 || page >= p.c.n_pages) {
            atomicCAS(err, 0, kDevErrIndex);
            page = 0;
          }
          src = kv_group_offset<QT, D>(p.c, page, head, 0, gi % per_page);
        }
      };
      int st_issue = stage;
      auto issue = [&](int it) {
        const long long from = __shfl_sync(~0u, src, it * G & 31);
        const long long from1 = G == 2 ? __shfl_sync(~0u, src, it * G + 1 & 31) : 0;
        if (lane == 0) {
          const bool both = G == 2 && first + it * (W * G) + 1 < g1;
          uint8_t* to = ring + st_issue * C::kStageBytes;
          const uint8_t* k = p.c.data + from;
          mbar_arrive_expect_tx(&full[st_issue], (both ? 4 : 2) * L::kHalf);
          const bool joined = both && from1 == from + L::kHalf;  // neighbours in a page
          const uint32_t bytes = joined ? 2 * L::kHalf : L::kHalf;
          bulk_load(to, k, bytes, &full[st_issue]);
          bulk_load(to + G * L::kHalf, k + v_offset, bytes, &full[st_issue]);
          if (both && !joined) {
            k = p.c.data + from1;
            bulk_load(to + L::kHalf, k, L::kHalf, &full[st_issue]);
            bulk_load(to + (G + 1) * L::kHalf, k + v_offset, L::kHalf, &full[st_issue]);
          }
        }
        st_issue = st_issue + 1 == NS ? 0 : st_issue + 1;
      };
      locate(0);
      int issued = 0;
      for (; issued < min(NS, n_it); ++issued) issue(issued);

      // ---- query fragments: column g of tile nt is row 8 nt + g; block n's values 8 t .. 8 t + 7
      uint32_t qf[C::kQSmem ? 1 : NT * NB][4];
      uint32_t qmin[NT][2];  // q4_1: sums of the query over blocks 2t, 2t + 1, as f16 and f16 remainder
      float q_sum[NT][2], q_most = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = 8 * nt + g;
        const int i = r / group_heads, h = head * group_heads + r % group_heads;
        const __half* q = p.q + b * p.q_b + i * p.q_n + h * p.q_h + 8 * t;
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (r < n_rows) v = *reinterpret_cast<const uint4*>(q + 32 * n);
          if (C::kQSmem) {
            if (warp == 0) *reinterpret_cast<uint4*>(s_q + ((nt * NB + n) * 32 + lane) * 16) = v;
          } else {
            qf[C::kQSmem ? 0 : nt * NB + n][0] = v.x;
            qf[C::kQSmem ? 0 : nt * NB + n][1] = v.y;
            qf[C::kQSmem ? 0 : nt * NB + n][2] = v.z;
            qf[C::kQSmem ? 0 : nt * NB + n][3] = v.w;
          }
          if (QT == QT_Q4_1) {
            const float2 x0 = __half22float2(u32_h2(v.x)), x1 = __half22float2(u32_h2(v.y));
            const float2 x2 = __half22float2(u32_h2(v.z)), x3 = __half22float2(u32_h2(v.w));
            float sum = ((x0.x + x0.y) + (x1.x + x1.y)) + ((x2.x + x2.y) + (x3.x + x3.y));
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            if (n == 2 * t) lo = sum;
            if (n == 2 * t + 1) hi = sum;
          }
        }
        q_sum[nt][0] = lo;
        q_sum[nt][1] = hi;
        q_most = fmaxf(q_most, fmaxf(fabsf(lo), fabsf(hi)));
      }
      // 32 queries of one sign may sum to more than an f16 holds: a unit that has such a sum takes them all less 2^6
      const bool q_large = QT == QT_Q4_1 && __any_sync(~0u, q_most >= 32768.f);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (QT == QT_Q4_1) {
          const float f = q_large ? 0.015625f : 1.f, lo = q_sum[nt][0] * f, hi = q_sum[nt][1] * f;
          const __half2 s = __floats2half2_rn(lo, hi);
          const float2 x = __half22float2(s);
          qmin[nt][0] = h2_u32(s);
          qmin[nt][1] = h2_u32(__floats2half2_rn(lo - x.x, hi - x.y));
        }
      }
      if (C::kQSmem) __syncthreads();

      // ---- state: columns 2t, 2t + 1 of each tile
      float o[NT][D / 16][4], omin[NT][4], m[NT][2], l[NT][2];
      Range range;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][x][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) omin[nt][e] = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          m[nt][c] = kNoScore;
          l[nt][c] = 0.f;
        }
      }

      for (int it = 0; it < n_it; ++it) {
        if (!mbar_wait(&full[stage], phase, s_abort, err, kErrWaitFull)) ok = false;
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        const int tok0 = (first + it * (W * G)) * 16;
        const bool whole = tok0 >= max_lo && tok0 + 16 * G <= min_hi;

        // -- scales (and minima) of the values, a word (two tokens) a lane; those of tokens outside the sequence's span, which
        // may hold anything, become zero
        uint8_t* v_scales = ring + stage * C::kStageBytes + G * L::kHalf + L::kVal;
        auto each_scale = [&](auto&& f) {  // f(word, whether of the minima, tokens of the word after tok0)
#pragma unroll
          for (int gg = 0; gg < G; ++gg)
#pragma unroll
            for (int e0 = 0; e0 < 8 * NB * L::kPlanes; e0 += 32) {
              const int e = e0 + lane, of = e % (8 * NB);
              if (8 * NB * L::kPlanes % 32 == 0 || e < 8 * NB * L::kPlanes)
                f(reinterpret_cast<uint32_t*>(v_scales + gg * L::kHalf) + e, e >= 8 * NB,
                  16 * gg + of / (2 * NB) * 2 + 8 * (of & 1));
            }
        };
        bool grow = false;
        if (!whole) {
          each_scale([&](uint32_t* at, bool, int after) {
            const int tok = tok0 + after;
            const uint32_t keep = (tok >= min_lo && tok < max_hi ? 0xFFFFu : 0u) | (tok + 1 >= min_lo && tok + 1 < max_hi ? 0xFFFF0000u : 0u);
            *at &= keep;
          });
        }
        each_scale([&](uint32_t* at, bool minima, int) { grow |= range.passed(*at, minima); });

        // -- scores
        float s_all[G][NT][4];
#pragma unroll
        for (int gg = 0; gg < G; ++gg) {
          const uint8_t* gp = ring + stage * C::kStageBytes + gg * L::kHalf;
          float (&s)[NT][4] = s_all[gg];
          uint32_t sc0[NB / 2], sc1[NB / 2];  // scales of tokens g and g + 8
          lds<NB * 2>(gp + L::k_scale(g, 0), sc0);
          lds<NB * 2>(gp + L::k_scale(g + 8, 0), sc1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
          if (QT == QT_Q4_1) {  // sum over blocks of minimum * (sum of the query over the block)
            uint32_t am[4] = {0, 0, 0, 0};
            if (2 * t < NB) {
              am[0] = am[2] = *reinterpret_cast<const uint32_t*>(gp + L::kSc + L::k_scale(g, 2 * t));
              am[1] = am[3] = *reinterpret_cast<const uint32_t*>(gp + L::kSc + L::k_scale(g + 8, 2 * t));
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(s[nt], am, qmin[nt][0], qmin[nt][1]);
            if (q_large) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] *= 64.f;
            }
          }
#pragma unroll
          for (int sb = 0; sb < D / L::kSB; ++sb) {
            constexpr int PB = L::kNBS * L::kBits;  // bytes of a lane's piece of one token
            uint32_t k0[PB / 4], k1[PB / 4];
            lds<PB>(gp + L::k_val(g, sb * L::kNBS, t), k0);
            lds<PB>(gp + L::k_val(g + 8, sb * L::kNBS, t), k1);
#pragma unroll
            for (int nn = 0; nn < L::kNBS; ++nn) {
              const int n = sb * L::kNBS + nn;
              uint32_t x0[4], x1[4];
              if (QT == QT_Q8_0) {
                byte_pairs(k0[2 * nn], x0[0], x0[1]);
                byte_pairs(k0[2 * nn + 1], x0[2], x0[3]);
                byte_pairs(k1[2 * nn], x1[0], x1[1]);
                byte_pairs(k1[2 * nn + 1], x1[2], x1[3]);
              } else {
                nibble_pairs<QT>(k0[nn], x0);
                nibble_pairs<QT>(k1[nn], x1);
              }
              const uint32_t a0[4] = {x0[0], x1[0], x0[1], x1[1]}, a1[4] = {x0[2], x1[2], x0[3], x1[3]};
              const __half2 h0 = u32_h2(sc0[n / 2]), h1 = u32_h2(sc1[n / 2]);
              const float f0 = n & 1 ? __high2float(h0) : __low2float(h0), f1 = n & 1 ? __high2float(h1) : __low2float(h1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const int at = C::kQSmem ? 0 : nt * NB + n;
                const uint4 qv = C::kQSmem ? *reinterpret_cast<const uint4*>(s_q + ((nt * NB + n) * 32 + lane) * 16)
                                           : make_uint4(qf[at][0], qf[at][1], qf[at][2], qf[at][3]);
                float c[4];
                mma16816_first(c, a0, qv.x, qv.y);
                mma16816(c, a1, qv.z, qv.w);
                s[nt][0] = fmaf(f0, c[0], s[nt][0]);
                s[nt][1] = fmaf(f0, c[1], s[nt][1]);
                s[nt][2] = fmaf(f1, c[2], s[nt][2]);
                s[nt][3] = fmaf(f1, c[3], s[nt][3]);
              }
            }
          }
        }

        // -- weights: the reference maximum of a column moves only when a score passes it by kLazy
        bool move = grow;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int gg = 0; gg < G; ++gg) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s_all[gg][nt][e] *= sl2;
            if (!whole) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                int lo, hi;
                row_span(p, len, min((8 * nt + 2 * t + c) / group_heads, p.nq - 1), &lo, &hi);
                const int tok = tok0 + 16 * gg + g;
                if (tok < lo || tok >= hi) s_all[gg][nt][c] = -INFINITY;
                if (tok + 8 < lo || tok + 8 >= hi) s_all[gg][nt][c + 2] = -INFINITY;
              }
            }
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            top[nt][c] = fmaxf(s_all[0][nt][c], s_all[0][nt][c + 2]);
#pragma unroll
            for (int gg = 1; gg < G; ++gg) top[nt][c] = fmaxf(top[nt][c], fmaxf(s_all[gg][nt][c], s_all[gg][nt][c + 2]));
            move |= top[nt][c] > m[nt][c] + kBias + kLazy;
          }
        }
        if (__any_sync(~0u, move)) {
          if (__any_sync(~0u, grow)) {
            uint32_t most[2] = {0, 0};
            each_scale([&](uint32_t* at, bool minima, int) {
              const uint32_t x = *at & 0x7FFF7FFFu;
              most[minima] = max(most[minima], max(x & 0xFFFF, x >> 16));
            });
            const float by = range.raise(most[0], most[1]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const float f = __shfl_sync(~0u, by, 2 * n);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  o[nt][2 * n][e] *= f;
                  o[nt][2 * n + 1][e] *= f;
                }
            }
            if (QT == QT_Q4_1) {
              const float f = __shfl_sync(~0u, by, 2 * (g % NB));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) omin[nt][c] *= f;
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) top[nt][c] = fmaxf(top[nt][c], __shfl_xor_sync(~0u, top[nt][c], x));
              const float m2 = fmaxf(m[nt][c], top[nt][c] - kBias);
              f[c] = ex2_approx(m[nt][c] - m2);
              m[nt][c] = m2;
              l[nt][c] *= f[c];
            }
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][x][e] *= f[e & 1];
#pragma unroll
            for (int e = 0; e < 4; ++e) omin[nt][e] *= f[e & 1];
          }
        }
        // weights of column g for tokens 2t, 2t + 1 and 2t + 8, 2t + 9 of each group
        uint32_t w0_all[G][NT], w1_all[G][NT];
#pragma unroll
        for (int gg = 0; gg < G; ++gg)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float e4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) e4[e] = ex2_approx(s_all[gg][nt][e] - m[nt][e & 1]);
            l[nt][0] += e4[0] + e4[2];
            l[nt][1] += e4[1] + e4[3];
            w0_all[gg][nt] = movmatrix(h2_u32(__floats2half2_rn(e4[0], e4[1])));
            w1_all[gg][nt] = movmatrix(h2_u32(__floats2half2_rn(e4[2], e4[3])));
          }

        // -- outputs
        if (range.lifted) {
          const __half2 by = u32_h2(range.factor());
          each_scale([&](uint32_t* at, bool, int) { *at = h2_u32(__hmul2(u32_h2(*at), by)); });
        }
        if (!whole || range.lifted) {
          fence_proxy_async_smem();  // the next copy into this stage comes after these writes
          __syncwarp();
        }
#pragma unroll
        for (int gg = 0; gg < G; ++gg) {
          const uint8_t* vp = ring + stage * C::kStageBytes + (G + gg) * L::kHalf;
          const uint32_t (&w0)[NT] = w0_all[gg], (&w1)[NT] = w1_all[gg];
          if (QT == QT_Q4_1) {
            // v = scale * (code - 8) + (minimum + 8 scale): the second term summed over tokens with the weights, a row for
            // each block. It is small where values surround 0; codes from 0 with the minimum would leave two large sums of
            // opposite sign, and the output over 524288 tokens off by 1.6e-3 (accumulation in the tensor core), not 3.5e-4.
            uint32_t am[4] = {0, 0, 0, 0}, as[4] = {0, 0, 0, 0};
            if (g < NB) {
              const uint2 v = *reinterpret_cast<const uint2*>(vp + L::kSc + L::v_scale(2 * t, g));
              const uint2 s = *reinterpret_cast<const uint2*>(vp + L::v_scale(2 * t, g));
              am[0] = v.x;
              am[2] = v.y;
              as[0] = s.x;
              as[2] = s.y;
            }
            const __half2 eight = u32_h2(0x48004800u);
            as[0] = h2_u32(__hmul2(u32_h2(as[0]), eight));  // exact, and below f16's largest: ScaleRange
            as[2] = h2_u32(__hmul2(u32_h2(as[2]), eight));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816(omin[nt], am, w0[nt], w1[nt]);
              mma16816(omin[nt], as, w0[nt], w1[nt]);
            }
          }
#pragma unroll
          for (int sb = 0; sb < D / L::kSB; ++sb) {
            constexpr int PB = L::kNBS * L::kBits;  // bytes of a lane's piece of two tokens
            constexpr int PW = PB / 8;              // words of a token's
            uint32_t va[PB / 4], vb[PB / 4];
            lds<PB>(vp + L::v_val(2 * t, sb * L::kNBS, g), va);
            lds<PB>(vp + L::v_val(2 * t + 8, sb * L::kNBS, g), vb);
#pragma unroll
            for (int nn = 0; nn < L::kNBS; ++nn) {
              const int n = sb * L::kNBS + nn;
              uint32_t x0[4], x1[4];  // values 4g .. 4g + 3 of tokens (2t, 2t + 1) and (2t + 8, 2t + 9)
              if (QT == QT_Q8_0) {
                byte_pairs(__byte_perm(va[nn], va[PW + nn], 0x5140), x0[0], x0[1]);
                byte_pairs(__byte_perm(va[nn], va[PW + nn], 0x7362), x0[2], x0[3]);
                byte_pairs(__byte_perm(vb[nn], vb[PW + nn], 0x5140), x1[0], x1[1]);
                byte_pairs(__byte_perm(vb[nn], vb[PW + nn], 0x7362), x1[2], x1[3]);
              } else {
                nibble_pairs<QT_Q4_0>(__byte_perm(va[nn / 2], va[PW + nn / 2], nn & 1 ? 0x7632 : 0x5410), x0);
                nibble_pairs<QT_Q4_0>(__byte_perm(vb[nn / 2], vb[PW + nn / 2], nn & 1 ? 0x7632 : 0x5410), x1);
              }
              const uint32_t a0[4] = {x0[0], x0[1], x1[0], x1[1]}, a1[4] = {x0[2], x0[3], x1[2], x1[3]};
              const uint2 sc = *reinterpret_cast<const uint2*>(vp + L::v_scale(2 * t, n));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t b0 = h2_u32(__hmul2(u32_h2(w0[nt]), u32_h2(sc.x)));
                const uint32_t b1 = h2_u32(__hmul2(u32_h2(w1[nt]), u32_h2(sc.y)));
                mma16816(o[nt][2 * n], a0, b0, b1);
                mma16816(o[nt][2 * n + 1], a1, b0, b1);
              }
            }
          }
        }
        stage = stage + 1 == NS ? 0 : stage + 1;
        if (stage == 0) phase ^= 1;
        __syncwarp();
        if (issued < n_it) {
          if (issued * G % 32 == 0) locate(issued);
          issue(issued);
          ++issued;
        }
      }

      // ---- join the warps: maxima and sums, then the scaled outputs
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(~0u, l[nt][c], x);
          if (g == 0) {
            s_m[warp * C::kRows + 8 * nt + 2 * t + c] = m[nt][c];
            s_l[warp * C::kRows + 8 * nt + 2 * t + c] = l[nt][c];
          }
        }
      if (!ok) *s_abort = 1;
      __syncthreads();
      if (*s_abort) {  // a wait ran out: no copy may still be landing when the CTA exits
        ok = false;
        break;
      }
      float* s_o = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = kNoScore;
#pragma unroll
          for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w * C::kRows + 8 * nt + 2 * t + c]);
          f[c] = ex2_approx(m[nt][c] - top);
          if (g == 0) s_f[warp * C::kRows + 8 * nt + 2 * t + c] = f[c];
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float mn[2] = {0.f, 0.f};
          if (QT == QT_Q4_1) {
            mn[0] = __shfl_sync(~0u, omin[nt][0], 4 * n + t);
            mn[1] = __shfl_sync(~0u, omin[nt][1], 4 * n + t);
          }
          const float lowered = __shfl_sync(~0u, range.lowered(), 2 * n), fo[2] = {f[0] * lowered, f[1] * lowered};
#pragma unroll
          for (int c = 0; c < 2; ++c)
            *reinterpret_cast<float4*>(s_o + (warp * C::kRows + 8 * nt + 2 * t + c) * C::kOStride + 32 * n + 4 * g) =
                make_float4((o[nt][2 * n][c] + mn[c]) * fo[c], (o[nt][2 * n][c + 2] + mn[c]) * fo[c],
                            (o[nt][2 * n + 1][c] + mn[c]) * fo[c], (o[nt][2 * n + 1][c + 2] + mn[c]) * fo[c]);
        }
      }
      __syncthreads();
      const bool split = ca > 0 || cb < n_chunks;
      const long long unit = (long long)b * p.c.heads + head;
      constexpr int kPart = C::kRows * (D + 2);
      float* part = a.part + (2 * (long long)blockIdx.x + (unit_start > p0 ? 1 : 0)) * kPart;
      auto finish = [&](int r, int d4, float4 v, float top, float sum) {
        const int i = r / group_heads, h = head * group_heads + r % group_heads;
        const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
        store_out(p, b * p.o_b + i * p.o_n + h * p.o_h + d4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        if (p.lse && d4 == 0)
          p.lse[((long long)b * p.nq + i) * p.heads + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
      };
      for (int e = threadIdx.x; e < n_rows * (D / 4); e += 32 * W) {
        const int r = e / (D / 4), d4 = e % (D / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f, top = kNoScore;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(s_o + (w * C::kRows + r) * C::kOStride + d4);
          v.x += x.x;
          v.y += x.y;
          v.z += x.z;
          v.w += x.w;
          sum = fmaf(s_l[w * C::kRows + r], s_f[w * C::kRows + r], sum);
          top = fmaxf(top, s_m[w * C::kRows + r]);
        }
        if (split) {
          __stcg(reinterpret_cast<float4*>(part + r * D + d4), v);
          if (d4 == 0) {
            __stcg(part + C::kRows * D + r, top);
            __stcg(part + C::kRows * (D + 1) + r, sum);
          }
        } else {
          finish(r, d4, v, top, sum);
        }
      }
      if (split) {
        // CTAs whose shares touch the unit: those of its first and last chunk, and all between
        const long long c0 = ((unit_start + 1) * ctas - 1) / total, c1 = ((unit_start + n_chunks) * ctas - 1) / total;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) s_last = atomicAdd(a.count + unit, 1) == (int)(c1 - c0);
        __syncthreads();
        if (s_last) {
          __threadfence();
          // the unit begins inside the first CTA's share or with it, and inside no other's
          const int n = (int)(c1 - c0) + 1, second = unit_start > total * c0 / ctas;
          auto part_of = [&](int k) { return a.part + (2 * (c0 + k) + (k == 0 ? second : 0)) * kPart; };
          // maxima of the rows over the parts: a warp a row
          for (int r = warp; r < n_rows; r += W) {
            float top = kNoScore;
            for (int k = lane; k < n; k += 32) top = fmaxf(top, __ldcg(part_of(k) + C::kRows * D + r));
#pragma unroll
            for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
            if (lane == 0) s_m[r] = top;
          }
          __syncthreads();
          // the threads share the parts between them where there are fewer outputs than threads
          constexpr int kItems = C::kRows * (D / 4), kShare = 32 * W > kItems ? 32 * W / kItems : 1;
          float4* s_v = reinterpret_cast<float4*>(smem);  // [kShare][kItems], and behind it the sums
          float* s_sum = reinterpret_cast<float*>(s_v + kShare * kItems);
          for (int e0 = threadIdx.x; e0 < kShare * kItems; e0 += 32 * W) {
            const int e = e0 % kItems, r = e / (D / 4), d4 = e % (D / 4) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
            if (r < n_rows) {
              const float top = s_m[r];
#pragma unroll 8
              for (int k = e0 / kItems; k < n; k += kShare) {
                const float* from = part_of(k);
                const float f = ex2_approx(__ldcg(from + C::kRows * D + r) - top);
                const float4 x = __ldcg(reinterpret_cast<const float4*>(from + r * D + d4));
                sum = fmaf(__ldcg(from + C::kRows * (D + 1) + r), f, sum);
                v.x = fmaf(x.x, f, v.x);
                v.y = fmaf(x.y, f, v.y);
                v.z = fmaf(x.z, f, v.z);
                v.w = fmaf(x.w, f, v.w);
              }
            }
            s_v[e0] = v;
            if (d4 == 0) s_sum[e0 / kItems * C::kRows + r] = sum;
          }
          __syncthreads();
          for (int e = threadIdx.x; e < n_rows * (D / 4); e += 32 * W) {
            const int r = e / (D / 4), d4 = e % (D / 4) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < kShare; ++k) {
              const float4 x = s_v[k * kItems + e];
              v.x += x.x;
              v.y += x.y;
              v.z += x.z;
              v.w += x.w;
              sum += s_sum[k * C::kRows + r];
            }
            finish(r, d4, v, s_m[r], sum);
          }
          if (threadIdx.x == 0) a.count[unit] = 0;
        }
      }
      fence_proxy_async_smem();  // the ring is written by copies again
      __syncthreads();
    }
    if (!ok) break;
    base += (long long)n_chunks * p.c.heads;
  }
  if (!ok) {
    // bounded: copies of this warp that were issued and not waited for
    for (int s = 0; s < NS; ++s) {
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(&full[s], s >= stage ? phase : phase ^ 1) && globaltimer_ns() - t0 < 10000000ull) {
      }
    }
  }
}

template <int QT, int D, int NT, int W>
int launch_rows(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  typedef Rows<QT, D, NT, W> C;
  auto* k = rows_kernel<QT, D, NT, W>;
  if (kernel_setup(k, C::kSmem) <= 0) return -13;
  RowsArgs a;
  a.p = p;
  a.part = w.part;
  a.count = w.count;
  return launch_dependent(k, dim3(C::kCtas * w.sms), 32 * W, C::kSmem, st, a, err);
}

// ---------------------------------------------------------------- dispatch
// Rows of one key / value head that rows_kernel takes (its output registers end at 128 a thread). tiles_kernel fills 128 or
// 256 rows whatever the count, so this one is ahead as far as it goes: 32 rows over 32 x 8192 tokens and 8 heads of 128
// take 207 us against 256, 16 rows over 8 x 28736 tokens and one head of 256 take 55 against 84.
int most_rows(int d) { return d == 256 ? 16 : 32; }

template <int QT, int D, int NT>
int launch_rows_nt(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  // Blocks of four warps, several on an SM, where there is a unit for each SM: a unit's beginning and end then run beside
  // other blocks' loops (32 sequences, 8 heads: 123 -> 96 us). One block an SM where few units are cut into many parts,
  // which have to be joined (one sequence, 2 heads, 524288 tokens: 477 -> 119 us).
  constexpr int kMost = Rows<QT, D, NT, 4>::kWarps;
  if ((long long)p.batch * p.c.heads >= w.sms) return launch_rows<QT, D, NT, 4>(p, w, err, st);
  return launch_rows<QT, D, NT, kMost>(p, w, err, st);
}

template <int QT, int D>
int attend(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  const int rows = p.nq * (p.heads / p.c.heads);
  if (rows <= 8) return launch_rows_nt<QT, D, 1>(p, w, err, st);
  if (D == 256 || rows <= 16) return launch_rows_nt<QT, D, 2>(p, w, err, st);
  return launch_rows_nt<QT, D, D == 256 ? 2 : 4>(p, w, err, st);
}

template <int QT>
int attend_d(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  return p.c.d == 64 ? attend<QT, 64>(p, w, err, st)
                     : p.c.d == 128 ? attend<QT, 128>(p, w, err, st) : attend<QT, 256>(p, w, err, st);
}

}  // namespace

KvAttnBytes kv_attention_work(const KvAttnParams& p, int sms) {
  // two parts for each of rows_kernel's CTAs: at most 4 an SM with 8 rows, 3 with 16 and 2 with 32 of d = 128, or with 16 of 256
  constexpr int kMost = 2 * Rows<QT_Q4_0, 128, 4, 4>::kCtas * 32 * (128 + 2);
  static_assert(2 * Rows<QT_Q4_0, 128, 1, 4>::kCtas * 8 * 130 <= kMost && 2 * Rows<QT_Q4_0, 128, 2, 4>::kCtas * 16 * 130 <= kMost &&
                    2 * Rows<QT_Q4_0, 64, 4, 4>::kCtas * 32 * 66 <= kMost && 2 * Rows<QT_Q4_0, 64, 2, 4>::kCtas * 16 * 66 <= kMost &&
                    2 * Rows<QT_Q4_0, 256, 1, 4>::kCtas * 8 * 258 <= kMost && 2 * Rows<QT_Q4_0, 256, 2, 4>::kCtas * 16 * 258 <= kMost,
                "parts of rows_kernel");
  KvAttnBytes b;
  b.part = std::max((size_t)sms * kMost * 4, kv_attention_tc_parts(sms));
  b.count = (size_t)p.batch * p.c.heads * 4;
  b.image = p.nq * (long long)(p.heads / p.c.heads) > most_rows(p.c.d) ? kv_attention_tc_image(p) : 0;
  return b;
}

int kv_attention_launches(const KvAttnParams& p) {
  return p.nq * (long long)(p.heads / p.c.heads) > most_rows(p.c.d) ? kv_attention_tc_launches(p) : 1;
}

int kv_attention(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  if (p.nq * (long long)(p.heads / p.c.heads) > most_rows(p.c.d)) return kv_attention_tc(p, w, err, st);
  return p.c.type == QT_Q4_0 ? attend_d<QT_Q4_0>(p, w, err, st)
                             : p.c.type == QT_Q4_1 ? attend_d<QT_Q4_1>(p, w, err, st) : attend_d<QT_Q8_0>(p, w, err, st);
}

}  // namespace s3b
