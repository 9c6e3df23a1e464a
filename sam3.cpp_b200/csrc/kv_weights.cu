// Attention weight that each token of the quantised cache gathers: w[token] = decay w[token] + sum over rows exp(scale q k - lse).
#include <algorithm>

#include "kv_mma.cuh"

namespace s3b {

namespace {

constexpr int kWarps = 8, kTile = 8;

template <int QT, int D, int NG>
struct Sweep {
  typedef KvL<QT, D> L;
  static constexpr int kRows = 64;                                  // query rows staged at a time
  static constexpr int kQ = kRows * D * 2;                          // their fragments
  static constexpr int kMin = QT == QT_Q4_1 ? kRows * 4 * 8 : 0;    // q4_1: sums of the query over the blocks
  static constexpr int kSmem = kQ + kMin + kRows * 12;
  static constexpr int kTokens = kWarps * NG * 16;                  // of a CTA's pass
};

struct WeightArgs {
  KvAttnParams p;
  KvWeights w;
  int token_blocks;  // of a sequence: max tokens / kTokens
};

// A unit is a sequence and a key / value head. Each warp holds NG groups of 16 tokens, their codes as the exact f16 integers of
// the A operand, and sweeps over all rows of the unit, 8 at a time, with the rows' fragments in shared memory: for every block of
// 32 channels two m16n8k16 products and the block's scale on the f32 result, then the weight exp2(s - lse) of each (row, token),
// summed per token in f32 registers in the order of the rows. No atomics: a token belongs to one warp.
template <int QT, int D, int NG>
__global__ void __launch_bounds__(32 * kWarps) sweep_kernel(const __grid_constant__ WeightArgs a, int* err) {
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
  const long long unit = blockIdx.x / a.token_blocks;
  const int head = (int)(unit % p.c.heads), b = (int)(unit / p.c.heads);
  let_next();
  wait_before();
  const int len = sequence_length(p, b, err);
  const int tok_cta = blockIdx.x % a.token_blocks * C::kTokens;
  if (tok_cta >= len) return;
  const float sl2 = p.scale * kLog2e;
  const int* table = p.pages + b * p.pages_stride;
  float* w = a.w.w + b * a.w.w_b + head * a.w.w_h;

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
        if (QT == QT_Q8_0) {
          byte_pairs(k0[2 * nn], x0[0], x0[1]);
          byte_pairs(k0[2 * nn + 1], x0[2], x0[3]);
          byte_pairs(k1[2 * nn], x1[0], x1[1]);
          byte_pairs(k1[2 * nn + 1], x1[2], x1[3]);
        } else {
          nibble_pairs<QT>(k0[nn], x0);
          nibble_pairs<QT>(k1[nn], x1);
        }
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
          const float2 x0 = __half22float2(u32_h2(v.x)), x1 = __half22float2(u32_h2(v.y));
          const float2 x2 = __half22float2(u32_h2(v.z)), x3 = __half22float2(u32_h2(v.w));
          float s = ((x0.x + x0.y) + (x1.x + x1.y)) + ((x2.x + x2.y) + (x3.x + x3.y));
          s += __shfl_xor_sync(~0u, s, 1);
          s += __shfl_xor_sync(~0u, s, 2);
          if (n == 2 * t) lo = s;
          if (n == 2 * t + 1) hi = s;
        }
        lo *= 0.015625f;  // 32 queries of one sign may sum to more than an f16 holds: all less 2^6
        hi *= 0.015625f;
        const __half2 m = __floats2half2_rn(lo, hi);
        const float2 x = __half22float2(m);
        s_min[nt * 32 + lane] = make_uint2(h2_u32(m), h2_u32(__floats2half2_rn(lo - x.x, hi - x.y)));
      }
      __syncthreads();
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
          for (int e = 0; e < 4; ++e) s[gg][e] *= 64.f;
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
      if (t == 0 && tok < len) w[tok] = fmaf(a.w.decay, w[tok], v);
    }
}

template <int QT, int D, int NG>
int launch_sweep(const KvAttnParams& p, const KvWeights& w, int* err, cudaStream_t st) {
  typedef Sweep<QT, D, NG> C;
  auto* k = sweep_kernel<QT, D, NG>;
  if (kernel_setup(k, C::kSmem) <= 0) return -13;
  const long long tokens = (long long)p.max_pages * p.c.page_size;
  WeightArgs a{p, w, (int)((tokens + C::kTokens - 1) / C::kTokens)};
  const long long grid = (long long)p.batch * p.c.heads * a.token_blocks;
  if (grid == 0) return 0;
  if (grid > 0x7fffffffLL) return -2;
  return launch_dependent(k, dim3((unsigned)grid), 32 * kWarps, C::kSmem, st, a, err);
}

template <int QT>
int weights_d(const KvAttnParams& p, const KvWeights& w, int* err, cudaStream_t st) {
  return p.c.d == 64 ? launch_sweep<QT, 64, 1>(p, w, err, st)
                     : p.c.d == 128 ? launch_sweep<QT, 128, 1>(p, w, err, st) : launch_sweep<QT, 256, 1>(p, w, err, st);
}

}  // namespace

size_t kv_weights_work(const KvAttnParams&, int) { return 0; }

int kv_weights_launches(const KvAttnParams&, int) { return 1; }

int kv_weights(const KvAttnParams& p, const KvWeights& w, int, int* err, cudaStream_t st) {
  return p.c.type == QT_Q4_0 ? weights_d<QT_Q4_0>(p, w, err, st)
                             : p.c.type == QT_Q4_1 ? weights_d<QT_Q4_1>(p, w, err, st) : weights_d<QT_Q8_0>(p, w, err, st);
}

}  // namespace s3b
