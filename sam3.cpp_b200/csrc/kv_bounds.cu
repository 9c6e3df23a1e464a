// Bounds of the keys of each page of the quantised cache, for choosing pages by them (layout of the cache: kv_cache.cuh).
#include <algorithm>

#include "kv_mma.cuh"

namespace s3b {

namespace {

struct BoundsArgs {
  KvAttnParams p;   // cache, pages, lengths
  KvBounds out;
  long long recent;  // tokens from the end whose pages are looked at
  int many;          // pages of a sequence that can hold them
};

// Of 2 H pairs the lower half goes on in lanes without bit X, the upper in those with it, each joined with the partner's.
template <int H, int X, int R>
__device__ __forceinline__ void fold(__half2 (&lo)[R], __half2 (&hi)[R], int lane) {
  const bool upper = lane & X;
#pragma unroll
  for (int r = 0; r < H; ++r) {
    // by value: a choice between array elements would keep the arrays in memory
    const uint32_t l0 = h2_u32(lo[r]), l1 = h2_u32(lo[r + H]), h0 = h2_u32(hi[r]), h1 = h2_u32(hi[r + H]);
    const uint32_t get_lo = __shfl_xor_sync(~0u, upper ? l0 : l1, X), get_hi = __shfl_xor_sync(~0u, upper ? h0 : h1, X);
    lo[r] = __hmin2(u32_h2(upper ? l1 : l0), u32_h2(get_lo));
    hi[r] = __hmax2(u32_h2(upper ? h1 : h0), u32_h2(get_hi));
  }
}

// A warp a page and head: lane (g, t) takes the tokens 8 i + g and of every block of 32 channels the 8 that its pieces of the
// keys' layout hold, as f16 pairs: the row as cache_read gives it in f16 (one rounding, which keeps the order of values, so that
// least and largest of the rounded are the rounded least and largest), two values an instruction. Then the 8 lanes of a t share
// the channels out among themselves, the larger half of the exchange first, and the row's largest magnitude sets the step.
// Measured: 2 x 65536 tokens, 4 heads of 128 in pages of 64: q4_0 37.7 MB of keys in 18.7 us, 2.0 TB/s; q4_1 18.7, q8_0 26.5.
// Half of the cycles issue (55% of the ALU's: minima, maxima, unpacking), the rest waits for a page's first words behind length
// and page table. Four tokens ahead instead of two (23.2 us), blocks that stay and read the next page's place ahead (19.4) and more
// blocks by fewer registers (18.9) were no faster.
template <int QT, int D>
__global__ void __launch_bounds__(128) bounds_kernel(const __grid_constant__ BoundsArgs a, int* err) {
  typedef KvL<QT, D> L;
  constexpr int R = D / 8;  // pairs of a lane
  const KvAttnParams& p = a.p;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long units = (long long)p.batch * a.many * p.c.heads;
  let_next();
  wait_before();
  for (long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); u < units; u += (long long)gridDim.x * 4) {
    const int head = (int)(u % p.c.heads), b = (int)(u / p.c.heads / a.many);
    const int len = sequence_length(p, b, err);
    const long long first = max(0LL, len - a.recent) / p.c.page_size;
    const long long j = first + u / p.c.heads % a.many;
    const long long left = len - j * p.c.page_size;
    if (left <= 0) continue;
    long long page = p.pages[b * p.pages_stride + j];
    if (page < 0 || page >= p.c.n_pages) {
      if (lane == 0) atomicCAS(err, 0, kDevErrIndex);
      continue;
    }
    const int n = (int)min((long long)p.c.page_size, left);
    const uint8_t* keys = p.c.data + kv_group_offset<QT, D>(p.c, page, head, 0, 0);
    __half2 lo[R], hi[R];
#pragma unroll
    for (int r = 0; r < R; ++r) lo[r] = u32_h2(0x7C007C00u), hi[r] = u32_h2(0xFC00FC00u);
#pragma unroll 2
    for (int tok = g; tok < n; tok += 8) {
      const uint8_t* gp = keys + (long long)(tok >> 4) * L::kHalf;
      const int in = tok & 15;
      uint32_t scales[L::kNB / 2], minima[L::kNB / 2];
      lds<L::kNB * 2>(gp + L::k_scale(in, 0), scales);
      if (QT == QT_Q4_1) lds<L::kNB * 2>(gp + L::kSc + L::k_scale(in, 0), minima);
#pragma unroll
      for (int sb = 0; sb < D / L::kSB; ++sb) {
        constexpr int PB = L::kNBS * L::kBits;
        uint32_t w[PB / 4];
        lds<PB>(gp + L::k_val(in, sb * L::kNBS, t), w);
#pragma unroll
        for (int nn = 0; nn < L::kNBS; ++nn) {
          const int blk = sb * L::kNBS + nn;
          const __half2 pair = u32_h2(scales[blk / 2]), sc = blk & 1 ? __high2half2(pair) : __low2half2(pair);
          uint32_t x[4];
          if (QT == QT_Q8_0) {
            byte_pairs(w[2 * nn], x[0], x[1]);
            byte_pairs(w[2 * nn + 1], x[2], x[3]);
          } else {
            nibble_pairs<QT>(w[nn], x);
          }
          __half2 low = u32_h2(0);
          if (QT == QT_Q4_1) low = blk & 1 ? __high2half2(u32_h2(minima[blk / 2])) : __low2half2(u32_h2(minima[blk / 2]));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 v = QT == QT_Q4_1 ? __hfma2(u32_h2(x[e]), sc, low) : __hmul2(u32_h2(x[e]), sc);
            lo[4 * blk + e] = __hmin2(lo[4 * blk + e], v);
            hi[4 * blk + e] = __hmax2(hi[4 * blk + e], v);
          }
        }
      }
    }
    // lanes g and g ^ 4 exchange halves of their pairs, then g ^ 2, then g ^ 1: R / 8 pairs are left to each
    fold<R / 2, 16>(lo, hi, lane);
    fold<R / 4, 8>(lo, hi, lane);
    fold<R / 8, 4>(lo, hi, lane);
    constexpr int O = R / 8;  // pairs of a lane now
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < O; ++r) {
      const __half2 m = __hmax2(__habs2(lo[r]), __habs2(hi[r]));
      top = max(top, max(h2_u32(m) & 0xFFFF, h2_u32(m) >> 16));
    }
    top = __reduce_max_sync(~0u, top);  // f16 magnitudes order as their bits
    const float peak = fminf(__half2float(__ushort_as_half((unsigned short)top)), 65504.f);
    const float inv = peak != 0.f ? __fdiv_rn(127.f, peak) : 0.f;
    const int r0 = (g >> 2 & 1) * (R / 2) + (g >> 1 & 1) * (R / 4) + (g & 1) * (R / 8);  // the first of its pairs
    const long long row = page * p.c.heads + head;
    int8_t* to = a.out.codes + row * 2 * D + 32 * (r0 / 4) + 8 * t + 2 * (r0 % 4);
#pragma unroll
    for (int r = 0; r < O; ++r) {
      const float2 l = __half22float2(lo[r]), h = __half22float2(hi[r]);
      auto code = [](float x) { return (signed char)fminf(fmaxf(x, -127.f), 127.f); };  // |x| * inv passes 127 by a rounding at most
      const char2 cl = make_char2(code(floorf(__fmul_rn(l.x, inv))), code(floorf(__fmul_rn(l.y, inv))));
      const char2 ch = make_char2(code(ceilf(__fmul_rn(h.x, inv))), code(ceilf(__fmul_rn(h.y, inv))));
      *reinterpret_cast<char2*>(to + 2 * r) = cl;
      *reinterpret_cast<char2*>(to + D + 2 * r) = ch;
    }
    if (lane == 0) a.out.steps[row] = __fdiv_rn(peak, 127.f);
  }
}

// What the codes of n pages stand for: f32 [n][heads][2][d], 4 values a thread.
__global__ void __launch_bounds__(256) values_kernel(const int8_t* codes, const float* steps, const long long* pages, long long n, long long n_pages,
                                                     int heads, int d, float* out) {
  const int quads = d / 2;  // of a page and head
  let_next();
  wait_before();
  const long long all = n * heads * quads;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long long)gridDim.x * 256) {
    const long long row = e / quads, i = row / heads, page = pages[i];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (page >= 0 && page < n_pages) {
      const long long at = page * heads + (row - i * heads);
      const char4 c = *reinterpret_cast<const char4*>(codes + at * 2 * d + (e - row * quads) * 4);
      const float step = steps[at];
      v = make_float4(c.x * step, c.y * step, c.z * step, c.w * step);
    }
    reinterpret_cast<float4*>(out)[e] = v;
  }
}

typedef void (*BoundsKernel)(BoundsArgs, int*);

template <int QT>
BoundsKernel bounds_for(int d) {
  return d == 64 ? bounds_kernel<QT, 64> : d == 128 ? bounds_kernel<QT, 128> : bounds_kernel<QT, 256>;
}

}  // namespace

int kv_bounds_values(const KvCache& shape, const KvBounds& bounds, const long long* pages, long long n, float* out, cudaStream_t st) {
  const long long blocks = (n * shape.heads * (shape.d / 2) + 255) / 256;
  return launch_dependent(values_kernel, dim3((unsigned)std::min(blocks, 1LL << 20)), 256, 0, st, (const int8_t*)bounds.codes, (const float*)bounds.steps, pages, n,
                          shape.n_pages, shape.heads, shape.d, out);
}

int kv_bounds(const KvAttnParams& p, const KvBounds& out, long long recent, int* err, cudaStream_t st) {
  BoundsArgs a{p, out, recent, p.max_pages};
  const long long spanned = (recent + p.c.page_size - 2) / p.c.page_size + 1;  // pages that so many tokens can touch
  if (spanned < a.many) a.many = (int)spanned;
  const long long blocks = std::min(((long long)p.batch * a.many * p.c.heads + 3) / 4, 1LL << 17);  // they walk over wider tables
  const BoundsKernel k = p.c.type == QT_Q4_0 ? bounds_for<QT_Q4_0>(p.c.d)
                                             : p.c.type == QT_Q4_1 ? bounds_for<QT_Q4_1>(p.c.d) : bounds_for<QT_Q8_0>(p.c.d);
  return launch_dependent(k, dim3((unsigned)blocks), 128, 0, st, a, err);
}

}  // namespace s3b
