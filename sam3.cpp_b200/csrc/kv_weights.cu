// Attention weight that each token of the quantised cache gathers: w[token] = decay w[token] + sum over rows exp(scale q k - lse).
// Scores as in rows_kernel: codes as exact integers, block scales on the f32 partial scores, so that weights are off by 1e-6 and
// less. Up to 32 rows of a head (16 at d = 256): stream_kernel; up to 128: sweep_kernel; more: the tiles of kv_weights_tc.cu.
#include <algorithm>

#include "kv_mma.cuh"

namespace s3b {

namespace {

constexpr int kWarps = 8, kTile = 8;

// q4_1: a score's part from the minima is sum over blocks of minimum * (sum of the query over the block), a product of its own. The
// sums enter it as f16 and f16 remainder, less by 2^6: 32 queries of one sign may sum to more than an f16 holds.
constexpr float kSumsLess = 64.f;
__device__ __forceinline__ float block_sum(const uint4& v) {  // of 8 values a lane and 4 lanes
  const float2 x0 = __half22float2(u32_h2(v.x)), x1 = __half22float2(u32_h2(v.y));
  const float2 x2 = __half22float2(u32_h2(v.z)), x3 = __half22float2(u32_h2(v.w));
  float s = ((x0.x + x0.y) + (x1.x + x1.y)) + ((x2.x + x2.y) + (x3.x + x3.y));
  s += __shfl_xor_sync(~0u, s, 1);
  return s + __shfl_xor_sync(~0u, s, 2);
}
__device__ __forceinline__ uint2 split_sums(float a, float b) {
  a *= 1.f / kSumsLess;
  b *= 1.f / kSumsLess;
  const __half2 m = __floats2half2_rn(a, b);
  const float2 x = __half22float2(m);
  return make_uint2(h2_u32(m), h2_u32(__floats2half2_rn(a - x.x, b - x.y)));
}
// the pairs of block nn of a lane's piece of one token
template <int QT, int NBS>
__device__ __forceinline__ void key_pairs(const uint32_t* piece, int nn, uint32_t (&x)[4]) {
  if (QT == QT_Q8_0) {
    byte_pairs(piece[2 * nn], x[0], x[1]);
    byte_pairs(piece[2 * nn + 1], x[2], x[3]);
  } else {
    nibble_pairs<QT>(piece[nn], x);
  }
}

// ---------------------------------------------------------------- many rows
template <int QT, int D, int NG>
struct Sweep {
  typedef KvL<QT, D> L;
  static constexpr int kRows = 128;                                 // query rows staged at a time
  static constexpr int kQ = kRows * D * 2;                          // their fragments
  static constexpr int kMin = QT == QT_Q4_1 ? kRows * 4 * 8 : 0;    // q4_1: sums of the query over the blocks
  static constexpr int kSmem = kQ + kMin + kRows * 12;
  static constexpr int kTokens = kWarps * NG * 16;                  // of a CTA's step
  static constexpr int kBlocks = D == 256 ? 2 : D == 128 ? 3 : 4;   // that an SM's registers take
};

struct WeightArgs {
  KvAttnParams p;
  KvWeights w;
};

// decay * old + sum; with a decay of 0 what was there does not count, whatever it is
__device__ __forceinline__ float weigh(float decay, float old, float sum) { return decay != 0.f ? fmaf(decay, old, sum) : sum; }

// The sequence of the line's place `pos` where sequence b has span(b) places, and the place of its first; `batch` where the lengths
// have become shorter since they were added up. The whole warp.
template <typename Span>
__device__ __forceinline__ int sequence_at(int batch, long long pos, long long* base, Span span) {
  const int lane = threadIdx.x & 31;
  *base = 0;
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const long long n = b0 + lane < batch ? span(b0 + lane) : 0;
    long long last = n;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const long long up = __shfl_up_sync(~0u, last, x);
      if (lane >= x) last += up;
    }
    const uint32_t past = __ballot_sync(~0u, *base + last > pos);
    if (past) {
      const int who = __ffs(past) - 1;
      *base += __shfl_sync(~0u, last - n, who);
      return b0 + who;
    }
    *base += __shfl_sync(~0u, last, 31);
  }
  return batch;
}
template <typename Span>
__device__ __forceinline__ long long line_length(int batch, Span span) {
  long long total = 0;
  for (int b = threadIdx.x & 31; b < batch; b += 32) total += span(b);
#pragma unroll
  for (int x = 16; x; x >>= 1) total += __shfl_xor_sync(~0u, total, x);
  return total;
}

// A unit is a sequence and a key / value head. Each warp holds NG groups of 16 tokens, their codes as the exact f16 integers of
// the A operand, and sweeps over all rows of the unit, 8 at a time, with the rows' fragments in shared memory: for every block of
// 32 channels two m16n8k16 products and the block's scale on the f32 result, then the weight exp2(s - lse) of each (row, token),
// summed per token in f32 registers in the order of the rows. No atomics: a token belongs to one warp. The blocks of 128 tokens of all
// units are one line, cut into equal shares for the CTAs; up to 128 rows stay in shared memory from one to the next.
// Measured: 64 rows, 4 x 8000 tokens, 8 heads of 128, q4_0: 33 us, 128 rows 51 us, 164 TFLOP/s of the 550 that these fragments reach
// (a block's scale on the f32 result takes as many instructions again); a grid of one CTA for 128 tokens 33 and 56.
template <int QT, int D, int NG>
__global__ void __launch_bounds__(32 * kWarps, Sweep<QT, D, NG>::kBlocks) sweep_kernel(const __grid_constant__ WeightArgs a, int* err) {
  typedef KvL<QT, D> L;
  typedef Sweep<QT, D, NG> C;
  constexpr int NB = L::kNB;
  extern __shared__ __align__(128) uint8_t smem[];
  uint4* s_q = reinterpret_cast<uint4*>(smem);                       // [row tile][block][lane]
  uint2* s_min = reinterpret_cast<uint2*>(smem + C::kQ);             // [row tile][lane]
  float* s_lse = reinterpret_cast<float*>(smem + C::kQ + C::kMin);   // in units of log2; +inf: no row
  int* s_lo = reinterpret_cast<int*>(s_lse + C::kRows);
  int* s_hi = s_lo + C::kRows;
  const KvAttnParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group_heads = p.heads / p.c.heads, n_rows = p.nq * group_heads;
  const int per_page = p.c.page_size >> 4;
  const float sl2 = p.scale * kLog2e;
  let_next();
  wait_before();
  // this CTA's share of the line and its present sequence, read by one warp or thread for all of them: a length that a caller changes
  // meanwhile may cost it tokens, but no barrier a thread, and the walk ends with the batch
  __shared__ long long s_total, s_base;
  __shared__ int s_b, s_len;
  auto blocks_of = [&](int len) { return (len + C::kTokens - 1) / C::kTokens; };
  if (warp == 0) {
    auto span = [&](int b) { return (long long)blocks_of(sequence_length(p, b, err)) * p.c.heads; };
    const long long total = line_length(p.batch, span), first = total * blockIdx.x / gridDim.x;
    long long base;
    const int b = sequence_at(p.batch, first, &base, span);
    if (lane == 0) {
      s_total = total;
      s_base = base;
      s_b = b;
      s_len = b < p.batch ? sequence_length(p, b, err) : 0;
    }
  }
  __syncthreads();
  long long pos = s_total * blockIdx.x / gridDim.x, base = s_base;
  const long long end = s_total * (blockIdx.x + 1) / gridDim.x;
  int b = s_b, len = s_len, blocks = blocks_of(len);
  long long staged = -1;  // the unit whose rows are in shared memory, all of them
  for (; pos < end; ++pos) {
    if (pos >= base + (long long)blocks * p.c.heads) {
      __syncthreads();  // the sequence before is known to all
      if (threadIdx.x == 0) {
        while (b < p.batch && pos >= base + (long long)blocks * p.c.heads) {
          base += (long long)blocks * p.c.heads;
          len = ++b < p.batch ? sequence_length(p, b, err) : 0;
          blocks = blocks_of(len);
        }
        s_base = base;
        s_b = b;
        s_len = len;
      }
      __syncthreads();
      base = s_base, b = s_b, len = s_len, blocks = blocks_of(len);
    }
    if (b >= p.batch) return;
    const int head = (int)((pos - base) / blocks);
    const int tok_cta = (int)(pos - base - (long long)head * blocks) * C::kTokens;
    const long long unit = (long long)b * p.c.heads + head;
    const int* table = p.pages + b * p.pages_stride;
    float* w = a.w.w + b * a.w.w_b + head * a.w.w_h;
    int first, last, none;
    row_span(p, len, 0, &first, &none);
    row_span(p, len, p.nq - 1, &none, &last);
    if (tok_cta >= last || tok_cta + C::kTokens <= first) {  // no row sees any of them
      const int tok = tok_cta + threadIdx.x;
      if (a.w.decay != 1.f && threadIdx.x < C::kTokens && tok < len) w[tok] = weigh(a.w.decay, w[tok], 0.f);
      continue;
    }

    // ---- this warp's tokens: group gg, tokens g and g + 8
    int tok0[NG];
    uint32_t ka[NG][NB][8];   // A fragments of the two products of a block
    uint32_t sc[NG][NB];      // scales of tokens g, g + 8
    uint32_t am[NG][4];       // minima
#pragma unroll
    for (int gg = 0; gg < NG; ++gg) {
      tok0[gg] = tok_cta + (warp * NG + gg) * 16;
      if (tok0[gg] >= len) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          sc[gg][n] = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) ka[gg][n][e] = 0;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) am[gg][e] = 0;
        continue;
      }
      const int gi = tok0[gg] >> 4;
      long long page = table[gi / per_page];
      if (page < 0 || page >= p.c.n_pages) {
        atomicCAS(err, 0, kDevErrIndex);
        page = 0;
      }
      const uint8_t* gp = p.c.data + kv_group_offset<QT, D>(p.c, page, head, 0, gi % per_page);
      uint32_t s0[NB / 2], s1[NB / 2];
      lds<NB * 2>(gp + L::k_scale(g, 0), s0);
      lds<NB * 2>(gp + L::k_scale(g + 8, 0), s1);
#pragma unroll
      for (int n = 0; n < NB; ++n) sc[gg][n] = __byte_perm(s0[n / 2], s1[n / 2], n & 1 ? 0x7632 : 0x5410);
#pragma unroll
      for (int e = 0; e < 4; ++e) am[gg][e] = 0;
      if (QT == QT_Q4_1 && 2 * t < NB) {
        am[gg][0] = am[gg][2] = *reinterpret_cast<const uint32_t*>(gp + L::kSc + L::k_scale(g, 2 * t));
        am[gg][1] = am[gg][3] = *reinterpret_cast<const uint32_t*>(gp + L::kSc + L::k_scale(g + 8, 2 * t));
      }
#pragma unroll
      for (int sb = 0; sb < D / L::kSB; ++sb) {
        constexpr int PB = L::kNBS * L::kBits;
        uint32_t k0[PB / 4], k1[PB / 4];
        lds<PB>(gp + L::k_val(g, sb * L::kNBS, t), k0);
        lds<PB>(gp + L::k_val(g + 8, sb * L::kNBS, t), k1);
#pragma unroll
        for (int nn = 0; nn < L::kNBS; ++nn) {
          const int n = sb * L::kNBS + nn;
          uint32_t x0[4], x1[4];
          key_pairs<QT, L::kNBS>(k0, nn, x0);
          key_pairs<QT, L::kNBS>(k1, nn, x1);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ka[gg][n][2 * e] = x0[e];
            ka[gg][n][2 * e + 1] = x1[e];
          }
        }
      }
    }

    float sum[NG][2];
#pragma unroll
    for (int gg = 0; gg < NG; ++gg) sum[gg][0] = sum[gg][1] = 0.f;
    for (int row0 = 0; row0 < n_rows; row0 += C::kRows) {
      const int rows = min(C::kRows, n_rows - row0), tiles = (rows + kTile - 1) / kTile;
      if (staged != unit) {
        __syncthreads();
        for (int e = threadIdx.x; e < tiles * NB * 32; e += 32 * kWarps) {
          const int l = e & 31, n = e / 32 % NB, r = e / (32 * NB) * 8 + (l >> 2);
          uint4 v = make_uint4(0, 0, 0, 0);
          if (r < rows) {
            const int i = (row0 + r) / group_heads, h = head * group_heads + (row0 + r) % group_heads;
            v = *reinterpret_cast<const uint4*>(p.q + b * p.q_b + i * p.q_n + h * p.q_h + 32 * n + 8 * (l & 3));
          }
          s_q[e] = v;
        }
        for (int r = threadIdx.x; r < tiles * kTile; r += 32 * kWarps) {
          float lse = INFINITY;
          int lo = 0, hi = 0;
          if (r < rows) {
            const int i = (row0 + r) / group_heads, h = head * group_heads + (row0 + r) % group_heads;
            lse = p.lse[((long long)b * p.nq + i) * p.heads + h] * kLog2e;
            if (lse != -INFINITY) row_span(p, len, i, &lo, &hi);  // else a row that has seen nothing, and sees nothing here
          }
          s_lse[r] = lse;
          s_lo[r] = lo;
          s_hi[r] = hi;
        }
        __syncthreads();
        if (QT == QT_Q4_1) {  // sums of the query over blocks 2t, 2t + 1 as f16 and f16 remainder: a warp a row tile
          for (int nt = warp; nt < tiles; nt += kWarps) {
            float lo = 0.f, hi = 0.f;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const uint4 v = s_q[(nt * NB + n) * 32 + lane];
              const float s = block_sum(v);
              if (n == 2 * t) lo = s;
              if (n == 2 * t + 1) hi = s;
            }
            s_min[nt * 32 + lane] = split_sums(lo, hi);
          }
          __syncthreads();
        }
        if (n_rows <= C::kRows) staged = unit;
      }
      for (int nt = 0; nt < tiles; ++nt) {
        float s[NG][4];
#pragma unroll
        for (int gg = 0; gg < NG; ++gg)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[gg][e] = 0.f;
        if (QT == QT_Q4_1) {
          const uint2 m = s_min[nt * 32 + lane];
#pragma unroll
          for (int gg = 0; gg < NG; ++gg) {
            mma16816(s[gg], am[gg], m.x, m.y);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[gg][e] *= kSumsLess;
          }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const uint4 q = s_q[(nt * NB + n) * 32 + lane];
#pragma unroll
          for (int gg = 0; gg < NG; ++gg) {
            const uint32_t(&k)[8] = ka[gg][n];
            const uint32_t a0[4] = {k[0], k[1], k[2], k[3]}, a1[4] = {k[4], k[5], k[6], k[7]};
            float c[4];
            mma16816_first(c, a0, q.x, q.y);
            mma16816(c, a1, q.z, q.w);
            const float2 f = __half22float2(u32_h2(sc[gg][n]));
            s[gg][0] = fmaf(f.x, c[0], s[gg][0]);
            s[gg][1] = fmaf(f.x, c[1], s[gg][1]);
            s[gg][2] = fmaf(f.y, c[2], s[gg][2]);
            s[gg][3] = fmaf(f.y, c[3], s[gg][3]);
          }
        }
        const int r = nt * kTile + 2 * t;
        const float2 lse = *reinterpret_cast<const float2*>(s_lse + r);
        const int2 lo = *reinterpret_cast<const int2*>(s_lo + r), hi = *reinterpret_cast<const int2*>(s_hi + r);
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int tok = tok0[gg] + g + 8 * u;
            const float e0 = ex2_approx(fmaf(s[gg][2 * u], sl2, -lse.x)), e1 = ex2_approx(fmaf(s[gg][2 * u + 1], sl2, -lse.y));
            sum[gg][u] += tok >= lo.x && tok < hi.x ? e0 : 0.f;
            sum[gg][u] += tok >= lo.y && tok < hi.y ? e1 : 0.f;
          }
        }
      }
    }
#pragma unroll
    for (int gg = 0; gg < NG; ++gg)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float v = sum[gg][u];
        v += __shfl_xor_sync(~0u, v, 1);
        v += __shfl_xor_sync(~0u, v, 2);
        const int tok = tok0[gg] + g + 8 * u;
        if (t == 0 && tok < len) w[tok] = weigh(a.w.decay, w[tok], v);
      }
  }
}

// ---------------------------------------------------------------- few rows
// Rows of a unit that stay in a warp's registers as fragments: 32, 16 at d = 256.
template <int QT, int D, int NT>
struct Stream {
  typedef KvL<QT, D> L;
  static constexpr int kBlocks = NT == 4 || NT * D >= 512 ? 3 : 4;  // of 4 warps, on an SM: 168 or 128 registers
  static constexpr int kG = NT == 1 && D <= 128 ? 2 : 1;                        // groups of a step
  static constexpr int kFit = (224 * 1024) / (4 * kBlocks * kG * L::kHalf);
  static constexpr int kStages = kFit > 8 / kG ? 8 / kG : kFit;                // steps of a warp in shared memory
  static constexpr int kSmem = 4 * kStages * kG * L::kHalf;
  static_assert(kStages >= 2, "stages of stream_kernel");
};

// All groups of 16 tokens of all units are one line, cut into equal shares for the warps; a token belongs to one warp, so nothing is
// joined and no two warps wait for each other. A warp has its own ring of groups in shared memory, copied while those before them are
// worked on, keeps the unit's query rows as fragments and adds each token's weights over the rows in two shuffles.
// Measured: 32 sequences of 1384 to 16384 tokens, 32 heads on 8, d = 128, q4_0: 177 MB in 48 us, 3.7 TB/s of the 6.5 that a copy
// reaches. Instruction issue bounds it (63% of the cycles): 220 for 16 tokens of a head, a third of them unpacking. Loads
// straight into registers, one or two groups ahead, took 72 us, rings of one group a step 59, five blocks an SM instead of four 61.
// 9 of the 24 variants spill 20 to 116 bytes a thread (four query tiles of d = 128: 56 to 116).
template <int QT, int D, int NT>
__global__ void __launch_bounds__(128, Stream<QT, D, NT>::kBlocks) stream_kernel(const __grid_constant__ WeightArgs a, int* err) {
  typedef KvL<QT, D> L;
  typedef Stream<QT, D, NT> C;
  constexpr int NB = L::kNB, NSB = D / L::kSB, PW = L::kNBS * L::kBits / 4, NS = C::kStages, G = C::kG;  // PW: words of a lane's piece of a token
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem + (threadIdx.x >> 5) * NS * G * L::kHalf;
  const KvAttnParams& p = a.p;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group_heads = p.heads / p.c.heads, n_rows = p.nq * group_heads;
  const int per_page = p.c.page_size >> 4;
  const long long warp = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), warps = (long long)gridDim.x * 4;
  let_next();
  wait_before();
  // this warp's share of the line, and the sequence in which it begins
  auto span = [&](int b) { return (long long)((sequence_length(p, b, err) + 15) >> 4) * p.c.heads; };
  const long long total = line_length(p.batch, span);
  long long pos = total * warp / warps, base;
  const long long end = total * (warp + 1) / warps;
  if (pos >= end) return;
  int b = sequence_at(p.batch, pos, &base, span);

  const float sl2 = p.scale * kLog2e;
  for (; pos < end && b < p.batch; ++b) {
    const int len = sequence_length(p, b, err), groups = (len + 15) >> 4;
    const int* table = p.pages + b * p.pages_stride;
    for (; pos < end && pos < base + (long long)groups * p.c.heads;) {
      const int head = (int)((pos - base) / groups);
      const int first = (int)(pos - base - (long long)head * groups);
      const int n_it = (int)min((long long)groups - first, end - pos);
      pos += n_it;
      float* w = a.w.w + b * a.w.w_b + head * a.w.w_h;

      // ---- query fragments: column g of tile nt is row 8 nt + g; the spans and ln sums of columns 2t, 2t + 1
      uint32_t qf[NT][NB][4], qmin[NT][2];
      float lse[NT][2];
      int row_lo[NT][2], row_hi[NT][2], min_lo = 0x7FFFFFFF, max_lo = 0, min_hi = 0x7FFFFFFF, max_hi = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = 8 * nt + g;
        int lo = 0, hi = 0;
        float mine = INFINITY;
        const __half* q = nullptr;
        if (r < n_rows) {
          const int i = r / group_heads, h = head * group_heads + r % group_heads;
          mine = p.lse[((long long)b * p.nq + i) * p.heads + h] * kLog2e;
          if (mine != -INFINITY) {  // else a row that has seen nothing, and sees nothing here
            row_span(p, len, i, &lo, &hi);
            q = p.q + b * p.q_b + i * p.q_n + h * p.q_h + 8 * t;
            min_lo = min(min_lo, lo), max_lo = max(max_lo, lo), min_hi = min(min_hi, hi), max_hi = max(max_hi, hi);
          } else {
            mine = INFINITY;
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          lse[nt][c] = __shfl_sync(~0u, mine, 8 * t + 4 * c);
          row_lo[nt][c] = __shfl_sync(~0u, lo, 8 * t + 4 * c);
          row_hi[nt][c] = __shfl_sync(~0u, hi, 8 * t + 4 * c);
        }
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const uint4 v = q ? *reinterpret_cast<const uint4*>(q + 32 * n) : make_uint4(0, 0, 0, 0);
          qf[nt][n][0] = v.x, qf[nt][n][1] = v.y, qf[nt][n][2] = v.z, qf[nt][n][3] = v.w;
          if (QT == QT_Q4_1) {
            const float s = block_sum(v);
            if (n == 2 * t) s0 = s;
            if (n == 2 * t + 1) s1 = s;
          }
        }
        if (QT == QT_Q4_1) {
          const uint2 m = split_sums(s0, s1);
          qmin[nt][0] = m.x, qmin[nt][1] = m.y;
        }
      }
      min_lo = __reduce_min_sync(~0u, min_lo), max_lo = __reduce_max_sync(~0u, max_lo);
      min_hi = __reduce_min_sync(~0u, min_hi), max_hi = __reduce_max_sync(~0u, max_hi);

      // ---- steps of G groups, on their way while others are worked on
      const int steps = (n_it + G - 1) / G;
      const bool all = a.w.decay != 1.f;                                      // tokens that no row sees change too
      const int seen_from = min_lo >> 4, seen_to = (max_hi + 15) >> 4;        // groups that some row sees
      auto seen = [&](int it) { return first + it * G < seen_to && first + it * G + G > seen_from; };
      long long src = 0;  // lane i: address of the keys of group (of a batch of 32) + i
      int to = 0;         // stage of the next step
      auto issue = [&](int it) {
        if (it < steps) {
          if ((it * G & 31) == 0 && it * G + lane < n_it) {
            const int gi = first + it * G + lane;
            long long page = table[gi / per_page];
            if (page < 0 || page >= p.c.n_pages) {
              atomicCAS(err, 0, kDevErrIndex);
              page = 0;
            }
            src = kv_group_offset<QT, D>(p.c, page, head, 0, gi % per_page);
          }
          if (seen(it)) {
#pragma unroll
            for (int gg = 0; gg < G; ++gg) {
              const uint8_t* from = p.c.data + __shfl_sync(~0u, src, (it * G & 31) + gg) + lane * 16;
              const uint32_t at = smem_u32(ring + (to * G + gg) * L::kHalf) + lane * 16;
              if (gg == 0 || it * G + gg < n_it) {
#pragma unroll
                for (int x = 0; x < L::kHalf; x += 512)
                  if (x + 512 <= L::kHalf || x + lane * 16 < L::kHalf)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + x), "l"(from + x) : "memory");
              }
            }
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        to = to + 1 == NS ? 0 : to + 1;
      };
      // the token whose weight this lane holds: lane t of a quad has token g + 8 (t % 2) of group t / 2
      const int mine_tok = first * 16 + (G == 2 ? 16 * (t >> 1) : 0) + g + 8 * (t & 1);
      const int tok_end = min(len, (first + n_it) * 16);
      auto mine = [&](int it) { return (G == 2 || t < 2) && mine_tok + it * (16 * G) < tok_end && (all || seen(it)); };
      for (int it = 0; it < NS - 1; ++it) issue(it);
      float next = mine(0) ? w[mine_tok] : 0.f;
      int stage = 0;
      for (int it = 0; it < steps; ++it) {
        const int tok0 = (first + it * G) * 16;
        asm volatile("cp.async.wait_group %0;" ::"n"(NS - 2) : "memory");
        __syncwarp();  // the copies of all lanes are there, and all are done with the stage that is filled next
        issue(it + NS - 1);
        const uint8_t* gp = ring + stage * (G * L::kHalf);
        stage = stage + 1 == NS ? 0 : stage + 1;
        const float old = next;
        if (mine(it + 1)) next = w[mine_tok + (it + 1) * (16 * G)];
        float sum[G][2];
#pragma unroll
        for (int gg = 0; gg < G; ++gg) sum[gg][0] = sum[gg][1] = 0.f;
        if (seen(it)) {
          const bool whole = tok0 >= max_lo && tok0 + 16 * G <= min_hi;
#pragma unroll
          for (int gg = 0; gg < G; ++gg, gp += L::kHalf) {
            uint32_t k0[NSB][PW], k1[NSB][PW], s0[NB / 2], s1[NB / 2];
#pragma unroll
            for (int sb = 0; sb < NSB; ++sb) {
              lds<PW * 4>(gp + L::k_val(g, sb * L::kNBS, t), k0[sb]);
              lds<PW * 4>(gp + L::k_val(g + 8, sb * L::kNBS, t), k1[sb]);
            }
            lds<NB * 2>(gp + L::k_scale(g, 0), s0);
            lds<NB * 2>(gp + L::k_scale(g + 8, 0), s1);
            float s[NT][4];
            uint32_t am[4] = {0, 0, 0, 0};
            if (QT == QT_Q4_1 && 2 * t < NB) {
              am[0] = am[2] = *reinterpret_cast<const uint32_t*>(gp + L::kSc + L::k_scale(g, 2 * t));
              am[1] = am[3] = *reinterpret_cast<const uint32_t*>(gp + L::kSc + L::k_scale(g + 8, 2 * t));
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
              if (QT == QT_Q4_1) {
                mma16816(s[nt], am, qmin[nt][0], qmin[nt][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] *= kSumsLess;
              }
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              uint32_t x0[4], x1[4];
              key_pairs<QT, L::kNBS>(k0[n / L::kNBS], n % L::kNBS, x0);
              key_pairs<QT, L::kNBS>(k1[n / L::kNBS], n % L::kNBS, x1);
              const uint32_t a0[4] = {x0[0], x1[0], x0[1], x1[1]}, a1[4] = {x0[2], x1[2], x0[3], x1[3]};
              const __half2 h0 = u32_h2(s0[n / 2]), h1 = u32_h2(s1[n / 2]);
              const float f0 = n & 1 ? __high2float(h0) : __low2float(h0), f1 = n & 1 ? __high2float(h1) : __low2float(h1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float c[4];
                mma16816_first(c, a0, qf[nt][n][0], qf[nt][n][1]);
                mma16816(c, a1, qf[nt][n][2], qf[nt][n][3]);
                s[nt][0] = fmaf(f0, c[0], s[nt][0]);
                s[nt][1] = fmaf(f0, c[1], s[nt][1]);
                s[nt][2] = fmaf(f1, c[2], s[nt][2]);
                s[nt][3] = fmaf(f1, c[3], s[nt][3]);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float v = ex2_approx(fmaf(s[nt][e], sl2, -lse[nt][e & 1]));
                if (!whole) {
                  const int tok = tok0 + 16 * gg + g + 8 * (e >> 1);
                  if (tok < row_lo[nt][e & 1] || tok >= row_hi[nt][e & 1]) v = 0.f;
                }
                sum[gg][e >> 1] += v;
              }
          }
#pragma unroll
          for (int gg = 0; gg < G; ++gg)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              sum[gg][u] += __shfl_xor_sync(~0u, sum[gg][u], 1);
              sum[gg][u] += __shfl_xor_sync(~0u, sum[gg][u], 2);
            }
        }
        if (mine(it)) {
          const float s0 = t & 1 ? sum[0][1] : sum[0][0], s1 = t & 1 ? sum[G - 1][1] : sum[G - 1][0];
          w[mine_tok + it * (16 * G)] = weigh(a.w.decay, old, G == 2 && (t & 2) ? s1 : s0);
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();  // the ring begins again
    }
    base += (long long)groups * p.c.heads;
  }
}

template <int QT, int D, int NG>
int launch_sweep(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  typedef Sweep<QT, D, NG> C;
  auto* k = sweep_kernel<QT, D, NG>;
  if (kernel_setup(k, C::kSmem) <= 0) return -13;
  const WeightArgs a{p, w};
  return launch_dependent(k, dim3(sms * C::kBlocks), 32 * kWarps, C::kSmem, st, a, err);
}

template <int QT, int D, int NT>
int launch_stream(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  typedef Stream<QT, D, NT> C;
  auto* k = stream_kernel<QT, D, NT>;
  if (kernel_setup(k, C::kSmem) <= 0) return -13;
  const WeightArgs a{p, w};
  return launch_dependent(k, dim3(sms * C::kBlocks), 128, C::kSmem, st, a, err);
}

// Whether the tiles of 128 rows take the call: they are ahead from where a second one is used, at d = 64 from where it is half full (4
// sequences of 8000 tokens, 8 heads, us at d = 64 / 128 / 256: 128 rows 77 / 88 / 112 against 38 / 51 / 82 here, 192 rows 65 / 83 /
// 111 against 63 / 92 / 155, 256 rows 66 / 83 / 111 against 78 / 103 / 203).
bool many_rows(const KvAttnParams& p) { return p.nq * (long long)(p.heads / p.c.heads) > (p.c.d == 64 ? 192 : 128); }

template <int QT, int D>
int weights_for(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  const long long rows = p.nq * (long long)(p.heads / p.c.heads);
  if (rows <= 8) return launch_stream<QT, D, 1>(p, w, sms, err, st);
  if (rows <= 16) return launch_stream<QT, D, 2>(p, w, sms, err, st);
  if (D < 256 && rows <= 32) return launch_stream<QT, D, D < 256 ? 4 : 2>(p, w, sms, err, st);
  if (many_rows(p)) return kv_weights_tc(p, w, sms, err, st);
  return launch_sweep<QT, D, 1>(p, w, sms, err, st);
}

template <int QT>
int weights_d(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  return p.c.d == 64 ? weights_for<QT, 64>(p, w, sms, err, st)
                     : p.c.d == 128 ? weights_for<QT, 128>(p, w, sms, err, st) : weights_for<QT, 256>(p, w, sms, err, st);
}

}  // namespace

size_t kv_weights_part(const KvAttnParams& p, int sms) { return many_rows(p) ? kv_weights_tc_part(sms) : 0; }

int kv_weights(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  return p.c.type == QT_Q4_0 ? weights_d<QT_Q4_0>(p, w, sms, err, st)
                             : p.c.type == QT_Q4_1 ? weights_d<QT_Q4_1>(p, w, sms, err, st) : weights_d<QT_Q8_0>(p, w, sms, err, st);
}

}  // namespace s3b
