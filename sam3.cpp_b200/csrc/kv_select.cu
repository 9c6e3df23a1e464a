// Choosing pages of a key / value cache for each block of queries by a bound on their scores (bounds: kv_bounds.cu).
#include <algorithm>

#include "kv_mma.cuh"
#include "kv_top.cuh"

namespace s3b {

namespace {

constexpr int kMostKeys = 24576;  // pages of a CTA whose scores' keys stay in its shared memory

struct SelectArgs {
  KvAttnParams p;  // c: heads, d, page_size, n_pages; q; pages, lengths; share, keep; causal, window
  KvBounds bounds;
  int sink, recent;
  int first;       // the launch's first unit
  float* scores;   // [units][max_pages] with `all`, else from the launch's first on, or none
  bool all;        // they are wanted, of all pages
  int* selected;   // [units][keep]
  int keys;        // room for so many in a CTA's shared memory; those of more pages are made from the scores again
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A unit is a block of queries and a key / value head, of one CTA or a cluster of them (CL) that share its pages and then choose
// together (kv_top.cuh). Whole numbers carry the score: sum over channels of max(c low, c high) = c+ high + c- low with
// c+ = max(c, 0), c- = min(c, 0), two products of 8-bit codes (16 pages x 32 channels x 8 rows an instruction), exact in 32 bits;
// then two f32 products, each rounded, so that the choice is the same whatever the order. Lane (g, t) holds 16 channels of 64 as
// the contraction's share of its rows (pages g, g + 8; query row g): whole 16-byte words of both. 16 warps where there is a CTA or
// less for each SM, else 8, so that several share one (32 x 8 lists of 256 pages: 14.8 us with 16, 11.5 with 8), and
// fewer for many lists of few pages (select_plan).
// Measured: 8 lists of 301 pages, d = 64: 7.2 us; 32 x 8 lists of up to 256 pages, d = 128: 8.8 us (the call's host time) for 9.6 MB;
// 2 lists of 16384 pages, d = 64: 13.6 us. A chain of latencies bounds it: length, table, codes, the votes or rounds of the
// choice. Products are 2% of it.
template <int D, int NT, int CL, int kThreads>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) select_kernel(const __grid_constant__ SelectArgs a, int* err) {
  constexpr int NC = D / 64;
  extern __shared__ uint32_t s_keys[];
  __shared__ TopShared<kThreads> s_top;
  __shared__ uint4 s_codes[NT * NC * 2 * 32];  // [tile][64 channels][positive, negative][lane]
  __shared__ float s_step[NT * 8];
  const KvAttnParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int in_launch = blockIdx.x / CL, unit = a.first + in_launch;
  const int blocks = (p.nq - 1) / p.share + 1;
  const int head = unit % p.c.heads, b = unit / p.c.heads / blocks;
  const int i0 = unit / p.c.heads % blocks * p.share, i1 = min(i0 + p.share, p.nq);
  const int group_heads = p.heads / p.c.heads, n_rows = (i1 - i0) * group_heads;
  let_next();
  wait_before();
  const int len = sequence_length(p, b, err);
  int lo, hi, none;
  row_span(p, len, i0, &lo, &none);
  row_span(p, len, i1 - 1, &none, &hi);
  const int pa = lo / p.c.page_size, pe = max(pa, hi > 0 ? (hi - 1) / p.c.page_size + 1 : 0);
  const int n = pe - pa;
  // this CTA's pages
  const int rank = CL > 1 ? blockIdx.x % CL : 0;
  const int share = CL > 1 ? ((n + CL - 1) / CL + 31) / 32 * 32 : n;
  const int begin = pa + (int)min((long long)n, (long long)rank * share), end = min(pe, begin + share);
  int* selected = a.selected + (long long)unit * p.keep;
  float* scores = a.scores + (long long)(a.all ? unit : in_launch) * p.max_pages;
  const bool trivial = n <= p.keep, in_smem = share <= a.keys;
  if (trivial && rank == 0)
    for (int e = threadIdx.x; e < p.keep; e += kThreads) selected[e] = e < n ? pa + e : -1;
  if (trivial && !a.all) return;
  if (a.all)
    for (int j = rank * kThreads + threadIdx.x; j < p.max_pages; j += CL * kThreads)
      if (j < pa || j >= pe) scores[j] = -INFINITY;

  // ---- bounds of 16 pages a warp; those of the first step are on their way while the queries are made into codes
  constexpr int kPass = 16 * (kThreads / 32);
  const int* table = p.pages + b * p.pages_stride;
  auto page_of = [&](int j) -> long long {
    if (j >= end) return 0;
    const long long page = table[j];
    if (page >= 0 && page < p.c.n_pages) return page;
    atomicCAS(err, 0, kDevErrIndex);
    return 0;
  };
  const int sink = pa + a.sink, recent = pe - a.recent;
  uint4 low[2][NC], high[2][NC];
  float page_step[2];
  long long next[2];  // pages of the step after
  auto load = [&](int j0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = j0 + g + 8 * u;
      page_step[u] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) low[u][c] = high[u][c] = make_uint4(0, 0, 0, 0);
      if (j < end) {
        const long long row = next[u] * p.c.heads + head;
        const int8_t* at = a.bounds.codes + row * 2 * D + 16 * t;
        page_step[u] = a.bounds.steps[row];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          low[u][c] = *reinterpret_cast<const uint4*>(at + 64 * c);
          high[u][c] = *reinterpret_cast<const uint4*>(at + D + 64 * c);
        }
      }
      next[u] = page_of(j + kPass);
    }
  };
#pragma unroll
  for (int u = 0; u < 2; ++u) next[u] = page_of(begin + 16 * warp + g + 8 * u);
  load(begin + 16 * warp);

  // ---- the query rows' codes, of either sign apart, a warp a row: D / 32 neighbouring channels a lane
  constexpr int V = D / 32, kWarps = kThreads / 32;
  for (int r = warp; r < 8 * NT; r += kWarps) {
    uint32_t w[V / 2], top = 0;
#pragma unroll
    for (int e = 0; e < V / 2; ++e) w[e] = 0;
    if (r < n_rows) {
      const int i = i0 + r / group_heads, h = head * group_heads + r % group_heads;
      lds<V * 2>(reinterpret_cast<const uint8_t*>(p.q + b * p.q_b + i * p.q_n + h * p.q_h + V * lane), w);
    }
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      // a NaN counts as 0, infinities as f16's largest
      uint32_t y = h2_u32(__hmin2(__hmax2(u32_h2(w[e]), u32_h2(0xFBFFFBFFu)), u32_h2(0x7BFF7BFFu)));
      if ((w[e] & 0x7FFFu) > 0x7C00u) y &= 0xFFFF0000u;
      if ((w[e] & 0x7FFF0000u) > 0x7C000000u) y &= 0x0000FFFFu;
      w[e] = y;
      top = max(top, max(y & 0x7FFFu, y >> 16 & 0x7FFFu));
    }
    const float peak = __half2float(__ushort_as_half((unsigned short)__reduce_max_sync(~0u, top)));
    const float inv = peak != 0.f ? __fdiv_rn(127.f, peak) : 0.f;
    if (lane == 0) s_step[r] = r < n_rows ? __fdiv_rn(peak, 127.f) : -1.f;  // < 0: no such row
    unsigned long long wp = 0, wn = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 x = __half22float2(u32_h2(w[e / 2]));
      const int code = max(-127, min(127, __float2int_rn(__fmul_rn(e & 1 ? x.y : x.x, inv))));
      wp |= (unsigned long long)max(code, 0) << (8 * e);
      wn |= (unsigned long long)(min(code, 0) & 255) << (8 * e);
    }
    // lane (r % 8, t) of tile r / 8 takes the channels 16 t .. 16 t + 15 of each 64
    const int ch = V * lane;
    uint8_t* at = reinterpret_cast<uint8_t*>(s_codes) + (((r >> 3) * NC + ch / 64) * 64 + (r & 7) * 4 + ch % 64 / 16) * 16 + ch % 16;
    if (V == 2) {
      *reinterpret_cast<uint16_t*>(at) = (uint16_t)wp;
      *reinterpret_cast<uint16_t*>(at + 512) = (uint16_t)wn;
    } else if (V == 4) {
      *reinterpret_cast<uint32_t*>(at) = (uint32_t)wp;
      *reinterpret_cast<uint32_t*>(at + 512) = (uint32_t)wn;
    } else {
      *reinterpret_cast<unsigned long long*>(at) = wp;
      *reinterpret_cast<unsigned long long*>(at + 512) = wn;
    }
  }
  __syncthreads();
  float step[NT][2];  // of rows 2t, 2t + 1 of a tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    step[nt][0] = s_step[8 * nt + 2 * t];
    step[nt][1] = s_step[8 * nt + 2 * t + 1];
  }

  // ---- scores of 16 pages at a time
  for (int j0 = begin + 16 * warp; j0 < end; j0 += kPass) {
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int acc[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint4 qp = s_codes[((nt * NC + c) * 2 + 0) * 32 + lane], qn = s_codes[((nt * NC + c) * 2 + 1) * 32 + lane];
        mma_s8(acc, high[0][c].x, high[1][c].x, high[0][c].y, high[1][c].y, qp.x, qp.y);
        mma_s8(acc, high[0][c].z, high[1][c].z, high[0][c].w, high[1][c].w, qp.z, qp.w);
        mma_s8(acc, low[0][c].x, low[1][c].x, low[0][c].y, low[1][c].y, qn.x, qn.y);
        mma_s8(acc, low[0][c].z, low[1][c].z, low[0][c].w, low[1][c].w, qn.z, qn.w);
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
      if (t == 0 && j < end) {
        if (in_smem) s_keys[j - begin] = j < sink || j >= recent ? kTopForced : top_key(best[u]);
        if (a.all || !in_smem) scores[j] = best[u];
      }
    }
    load(j0 + kPass);
  }
  if (trivial) return;
  __syncthreads();
  auto emit = [&](uint32_t at, int i) { selected[at] = begin + i; };
  if (in_smem) {
    auto key = [&](int i) { return s_keys[i]; };
    top_select<kThreads, CL>(s_top, end - begin, (uint32_t)p.keep, key, [](int, uint32_t x) { return x; }, key, emit);
  } else {
    auto fetch = [&](int i) { return scores[begin + i]; };
    auto make = [&](int i, float x) { return begin + i < sink || begin + i >= recent ? kTopForced : top_key(x); };
    top_select<kThreads, CL>(s_top, end - begin, (uint32_t)p.keep, fetch, make, [&](int i) { return make(i, scores[begin + i]); }, emit);
  }
}

struct SelectKernel {
  void (*kernel)(SelectArgs, int*);
  int threads;
};
template <int D, int CL, int T>
SelectKernel select_rows(int rows) {
  return {rows <= 8 ? select_kernel<D, 1, CL, T> : D == 256 || rows <= 16 ? select_kernel<D, 2, CL, T> : select_kernel<D, D == 256 ? 2 : 4, CL, T>, T};
}
template <int CL, int T>
SelectKernel select_for(int d, int rows) {
  return d == 64 ? select_rows<64, CL, T>(rows) : d == 128 ? select_rows<128, CL, T>(rows) : select_rows<256, CL, T>(rows);
}

struct SelectPlan {
  SelectKernel k;
  int cl;           // CTAs of a unit
  long long share;  // pages of the largest share of a CTA
};
// CTAs of a unit: about 512 pages each (two steps of 16 for each warp), on half of the SMs: large clusters find no place on all of
// them (8 lists of 8192 pages: 24.2 us in clusters of 16, 14.4 of 8; 16 lists of 16384: 32.5 of 8, 25.8 of 4).
// Many lists of few pages: small CTAs, as many warps as two keys a lane and a list's latencies ask for, more of them on an SM (with 8
// warps and so: 68880 lists of one page 296 -> 105 us, 4096 of 64 pages 51 -> 27 in one warp; 16000 of 100 pages 184 -> 93 in two;
// 8192 of 250 pages 127 -> 103 in four; but 256 of 100 pages 7.2 -> 9.0).
bool select_plan(const KvAttnParams& p, int sms, SelectPlan* plan) {
  const int rows = p.share * (p.heads / p.c.heads), d = p.c.d;
  int cl = 1;
  while (cl < 16 && cl * 512LL < p.max_pages && kv_attention_units(p) * cl * 4 <= sms) cl *= 2;
  auto of = [&](int n) {
    if (n == 1 && kv_attention_units(p) > 4LL * sms) {
      if (p.max_pages <= 64) return select_for<1, 32>(d, rows);
      if (p.max_pages <= 128) return select_for<1, 64>(d, rows);
      if (p.max_pages <= 256) return select_for<1, 128>(d, rows);
    }
    return n == 1 ? (kv_attention_units(p) <= sms ? select_for<1, 512>(d, rows) : select_for<1, 256>(d, rows))
           : n == 2 ? select_for<2, 512>(d, rows) : n == 4 ? select_for<4, 512>(d, rows)
           : n == 8 ? select_for<8, 512>(d, rows) : select_for<16, 512>(d, rows);
  };
  plan->k = of(cl);
  if (cl == 16 && cluster_setup(plan->k.kernel, kMostKeys * 4, plan->k.threads, cl) <= 0) plan->k = of(cl = 8);
  plan->cl = cl;
  plan->share = cl > 1 ? ((p.max_pages + cl - 1LL) / cl + 31) / 32 * 32 : p.max_pages;
  return cluster_setup(plan->k.kernel, kMostKeys * 4, plan->k.threads, cl) > 0;
}

}  // namespace

bool kv_select_needs_scores(const KvAttnParams& p, int sms) {
  if (p.max_pages <= kMostKeys) return false;
  SelectPlan plan;
  return !select_plan(p, sms, &plan) || plan.share > kMostKeys;
}

int kv_select(const KvAttnParams& p, const KvBounds& bounds, int sink, int recent, float* scores, bool all, int* selected, long long first,
              long long n, int sms, int* err, cudaStream_t st) {
  SelectPlan plan;
  if (!select_plan(p, sms, &plan)) return -13;
  const long long grid = n * plan.cl;
  if (grid > 0x7fffffffLL) return -2;
  const SelectArgs a{p, bounds, sink, recent, (int)first, scores, all, selected, (int)std::min<long long>(plan.share, kMostKeys)};
  return launch_clusters(plan.k.kernel, (unsigned)grid, plan.k.threads, (size_t)a.keys * 4, plan.cl, st, a, err);
}

}  // namespace s3b
