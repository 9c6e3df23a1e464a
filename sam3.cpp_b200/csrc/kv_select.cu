// Choosing pages of a key / value cache for each block of queries by a bound on their scores (bounds: kv_bounds.cu).
#include <algorithm>

#include "kv_mma.cuh"
#include "kv_top.cuh"

namespace s3b {

namespace {

constexpr int kThreads = 256;
constexpr int kSpan = 512;  // pages of a CTA: 16 at a time for each of 8 warps, four times

struct SelectArgs {
  KvAttnParams p;  // c: heads, d, page_size, n_pages; q; pages, lengths; share, keep; causal, window
  KvBounds bounds;
  int sink, recent;
  float* scores;   // [units][max_pages]
  bool all;        // the scores of all pages are wanted
  int* count;      // [units], zero between launches
  int* selected;   // [units][keep]
  int splits;      // CTAs of a unit
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A unit is a block of queries and a key / value head; its CTAs take 512 pages each, and the last of them to end chooses.
// Whole numbers carry the score: sum over channels of max(c low, c high) = c+ high + c- low with c+ = max(c, 0), c- = min(c, 0), two
// products of 8-bit codes (16 pages x 32 channels x 8 rows an instruction), exact in 32 bits; then two f32 products, each
// rounded, so that the choice is the same whatever the order. Lane (g, t) holds 16 channels of 64 as the contraction's share of
// its rows (pages g, g + 8; query row g): whole 16-byte words of both.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ SelectArgs a, int* err) {
  constexpr int NC = D / 64;
  __shared__ TopShared<kThreads> s_top;
  __shared__ int s_last;
  const KvAttnParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long unit = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  const int blocks = (p.nq - 1) / p.share + 1;
  const int head = (int)(unit % p.c.heads), b = (int)(unit / p.c.heads / blocks);
  const int i0 = (int)(unit / p.c.heads % blocks) * p.share, i1 = min(i0 + p.share, p.nq);
  const int group_heads = p.heads / p.c.heads, n_rows = (i1 - i0) * group_heads;
  let_next();
  wait_before();
  const int len = sequence_length(p, b, err);
  int lo, hi, none;
  row_span(p, len, i0, &lo, &none);
  row_span(p, len, i1 - 1, &none, &hi);
  const int pa = lo / p.c.page_size, pe = max(pa, (int)((hi + (long long)p.c.page_size - 1) / p.c.page_size));
  const int n = pe - pa;
  int* selected = a.selected + unit * p.keep;
  float* scores = a.scores + unit * p.max_pages;
  const int begin = split * kSpan, end = min(begin + kSpan, p.max_pages);
  const bool trivial = n <= p.keep;
  if (trivial && split == 0)
    for (int e = threadIdx.x; e < p.keep; e += kThreads) selected[e] = e < n ? pa + e : -1;
  if (trivial && !a.all) return;
  if (a.all)
    for (int j = begin + threadIdx.x; j < end; j += kThreads)
      if (j < pa || j >= pe) scores[j] = -INFINITY;
  if (begin >= pe || end <= pa) return;

  // ---- the query rows' codes, of either sign apart: column g of tile nt is row 8 nt + g
  uint32_t pos[NT][NC][4], neg[NT][NC][4];
  float step[NT][2];  // of columns 2t, 2t + 1; < 0: no such row
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 8 * nt + g;
    const int i = i0 + r / group_heads, h = head * group_heads + r % group_heads;
    const __half* q = p.q + b * p.q_b + i * p.q_n + h * p.q_h + 16 * t;
    uint32_t raw[NC][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (r < n_rows) {
        v[0] = *reinterpret_cast<const uint4*>(q + 64 * c);
        v[1] = *reinterpret_cast<const uint4*>(q + 64 * c + 8);
      }
      const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // a NaN counts as 0, infinities as f16's largest
        __half2 x = u32_h2(w[e]);
        x = __hmin2(__hmax2(x, u32_h2(0xFBFFFBFFu)), u32_h2(0x7BFF7BFFu));
        uint32_t y = h2_u32(x);
        if ((w[e] & 0x7FFFu) > 0x7C00u) y &= 0xFFFF0000u;
        if ((w[e] & 0x7FFF0000u) > 0x7C000000u) y &= 0x0000FFFFu;
        raw[c][e] = y;
        top = max(top, max(y & 0x7FFFu, y >> 16 & 0x7FFFu));
      }
    }
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    top = max(top, __shfl_xor_sync(~0u, top, 2));
    const float peak = __half2float(__ushort_as_half((unsigned short)top));
    const float inv = peak != 0.f ? __fdiv_rn(127.f, peak) : 0.f;
    const float mine = r < n_rows ? __fdiv_rn(peak, 127.f) : -1.f;
    step[nt][0] = __shfl_sync(~0u, mine, 8 * t);
    step[nt][1] = __shfl_sync(~0u, mine, 8 * t + 4);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x0 = __half22float2(u32_h2(raw[c][2 * e])), x1 = __half22float2(u32_h2(raw[c][2 * e + 1]));
        const float x[4] = {x0.x, x0.y, x1.x, x1.y};
        uint32_t wp = 0, wn = 0;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int code = max(-127, min(127, __float2int_rn(__fmul_rn(x[f], inv))));
          wp |= (uint32_t)max(code, 0) << (8 * f);
          wn |= (uint32_t)(min(code, 0) & 255) << (8 * f);
        }
        pos[nt][c][e] = wp;
        neg[nt][c][e] = wn;
      }
  }

  // ---- scores of 16 pages at a time
  const int* table = p.pages + b * p.pages_stride;
  for (int j0 = begin + 16 * warp; j0 < end; j0 += 16 * (kThreads / 32)) {
    if (j0 >= pe || j0 + 16 <= pa) continue;
    uint4 low[2][NC], high[2][NC];
    float page_step[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = j0 + g + 8 * u;
      page_step[u] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) low[u][c] = high[u][c] = make_uint4(0, 0, 0, 0);
      if (j >= pa && j < pe) {
        long long page = table[j];
        if (page < 0 || page >= p.c.n_pages) {
          atomicCAS(err, 0, kDevErrIndex);
          page = 0;
        }
        const long long row = page * p.c.heads + head;
        const int8_t* at = a.bounds.codes + row * 2 * D + 16 * t;
        page_step[u] = a.bounds.steps[row];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          low[u][c] = *reinterpret_cast<const uint4*>(at + 64 * c);
          high[u][c] = *reinterpret_cast<const uint4*>(at + D + 64 * c);
        }
      }
    }
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int acc[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        mma_s8(acc, high[0][c].x, high[1][c].x, high[0][c].y, high[1][c].y, pos[nt][c][0], pos[nt][c][1]);
        mma_s8(acc, high[0][c].z, high[1][c].z, high[0][c].w, high[1][c].w, pos[nt][c][2], pos[nt][c][3]);
        mma_s8(acc, low[0][c].x, low[1][c].x, low[0][c].y, low[1][c].y, neg[nt][c][0], neg[nt][c][1]);
        mma_s8(acc, low[0][c].z, low[1][c].z, low[0][c].w, low[1][c].w, neg[nt][c][2], neg[nt][c][3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float s = __fmul_rn(__fmul_rn((float)acc[e], page_step[e >> 1]), step[nt][e & 1]);
        if (step[nt][e & 1] >= 0.f) best[e >> 1] = fmaxf(best[e >> 1], s);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      best[u] = fmaxf(best[u], __shfl_xor_sync(~0u, best[u], 1));
      best[u] = fmaxf(best[u], __shfl_xor_sync(~0u, best[u], 2));
      const int j = j0 + g + 8 * u;
      if (t == 0 && j >= pa && j < pe) __stcg(scores + j, best[u]);
    }
  }
  if (trivial) return;

  // ---- the choice, by the CTA of the unit that ends last
  const int needed = (pe - 1) / kSpan - pa / kSpan + 1;
  __threadfence();
  __syncthreads();
  if (needed > 1) {
    if (threadIdx.x == 0) s_last = atomicAdd(a.count + unit, 1) == needed - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    if (threadIdx.x == 0) a.count[unit] = 0;
  }
  const int sink = a.sink, recent = a.recent;
  top_select<kThreads, 16, 1>(
      s_top, 0, n, (uint32_t)p.keep,
      [&](int i) { return i < sink || i >= n - recent ? kTopForced : top_key(__ldcg(scores + pa + i)); },
      [&](uint32_t at, int i, uint32_t) { selected[at] = pa + i; });
}

typedef void (*SelectKernel)(SelectArgs, int*);

template <int D>
SelectKernel select_for(int rows) {
  return rows <= 8 ? select_kernel<D, 1> : D == 256 || rows <= 16 ? select_kernel<D, 2> : select_kernel<D, D == 256 ? 2 : 4>;
}

}  // namespace

int kv_select(const KvAttnParams& p, const KvBounds& bounds, int sink, int recent, float* scores, bool all, int* count,
              int* selected, int* err, cudaStream_t st) {
  SelectArgs a{p, bounds, sink, recent, scores, all, count, selected, std::max(1, (p.max_pages + kSpan - 1) / kSpan)};
  const long long grid = kv_attention_units(p) * a.splits;
  if (grid > 0x7fffffffLL) return -2;
  const int rows = p.share * (p.heads / p.c.heads);
  const SelectKernel k = p.c.d == 64 ? select_for<64>(rows) : p.c.d == 128 ? select_for<128>(rows) : select_for<256>(rows);
  return launch_dependent(k, dim3((unsigned)grid), kThreads, 0, st, a, err);
}

}  // namespace s3b
