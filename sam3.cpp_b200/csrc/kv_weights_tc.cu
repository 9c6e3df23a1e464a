// Gathered attention weights for many query rows: tcgen05 tiles of 128 tokens by 128 query rows.
//
// w[token] sums over query rows, so the tokens stand in the rows of the product: S = K Q^T, and a thread that owns a token (a
// lane of TMEM) adds up exp2(s - lse) along its row of S with no exchange between threads. K of 128 tokens is the A operand and
// stays in TMEM while all query rows of the head pass by as B: from shared memory only B is read, which an operand A there would
// double. The scores are exact to f32's sums: a key is the sum of two f16 numbers, its f16 rounding and what that left (code x scale
// has 15 or 19 bits), and both are multiplied; rounding K to f16 alone would put the weights off by 1e-4 and more, beside an
// lse that was not made with the same rounding. That doubles the products: 2 x 128 x 128 x d for 16384 exponentials, so
// the tensor pipe bounds d = 256 and the exponentials d = 64.
//
// The line of (tile of 128 tokens, 128 query rows) of all sequences and heads is cut into equal shares for the CTAs. A tile that
// several CTAs share leaves its sums in the workspace; the last CTA to arrive adds them in the order of the shares.
//
// Measured: 4096 rows over 28736 tokens, one head of 256, q4_0: 102 us, 590 TFLOP/s of the product itself and twice that in the tensor
// cores (65% of the kernel's cycles; what is left is K's way into TMEM at each tile's beginning, when no product runs, and the
// chain product - exponentials of the two S regions); a chunk of 128 rows takes 1.4 us at d = 256, 0.8 at 64. The same on mma.sync
// fragments took 434 us.
//
// Roles: warps 0-3 and 4-7 take turns at S of every other 128 rows, and dequantise half of K's channels each; warps 8-11
// copy the query rows (asynchronously, in the 128-byte swizzle); warp 12 issues the products; warp 13 reads the rows' ln sums.
#include <algorithm>
#include <type_traits>

#include "kv_mma.cuh"
#include "kv_tmem.cuh"

namespace s3b {

namespace {

constexpr int kTile = 128, kSlot = 16384;  // tokens and rows of a tile; bytes of 128 rows of 64 f16

template <int QT, int D>
struct Wt {
  typedef KvL<QT, D> L;
  static constexpr int kParts = D / 64;
  static constexpr int kStageBytes = kParts * kSlot;
  static constexpr int kStages = D == 256 ? 3 : 6;   // of query rows
  static constexpr int kInfos = 4;                   // of their ln sums and spans
  static constexpr int kThreads = 14 * 32;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kInfos * (kTile * 12 + 16) + 2 * kTile * 4 + 512;
  static constexpr int kS = 256;                     // TMEM: K and its remainder, then two S regions
};

struct WtArgs {
  KvAttnParams p;
  KvWeights w;
  float* part;  // [2 * grid][128]
  int* count;   // [grid], zero between launches
  int chunks;   // of 128 query rows of a head
};

// One CTA's walk over its share [pos, end) of the line, tile by tile. Every role takes the same steps, by lengths that are read once
// (those of its first kLens sequences: as many as 128 tokens each and more than 1024 sequences for each SM would need).
constexpr int kLens = 1024;
struct WtWalk {
  long long pos, end, base;
  int b;
  const int* lens;  // of the sequences from b_first on, in shared memory
  int b_first;
};
struct WtSeg {
  int b, head, len, tok0;
  int ca, cb;       // chunks of the share that see a token of the tile
  bool whole;       // the share has all chunks of the tile
  long long start;  // the tile's place in the line
};

__device__ __forceinline__ bool wt_next(const WtArgs& a, int* err, WtWalk& w, WtSeg& s) {
  const KvAttnParams& p = a.p;
  while (w.pos < w.end && w.b < p.batch) {
    s.len = w.b - w.b_first < kLens ? w.lens[w.b - w.b_first] : sequence_length(p, w.b, err);
    const int tiles = (s.len + kTile - 1) / kTile;
    const long long span = (long long)tiles * p.c.heads * a.chunks;
    if (w.pos >= w.base + span) {
      w.base += span;
      ++w.b;
      continue;
    }
    const long long unit = (w.pos - w.base) / a.chunks;
    const int ca = (int)((w.pos - w.base) - unit * a.chunks), cb = (int)min((long long)a.chunks, ca + w.end - w.pos);
    s.b = w.b;
    s.head = (int)(unit / tiles);
    s.tok0 = (int)(unit - (long long)s.head * tiles) * kTile;
    s.start = w.pos - ca;
    s.whole = ca == 0 && cb == a.chunks;
    w.pos += cb - ca;
    int va = 0, vb = a.chunks;
    if (p.causal) {  // queries i with a span (i + 1 + len - nq less the window ..) that meets the tile
      const int group = p.heads / p.c.heads, before = s.len - p.nq;
      const int i0 = min(max(0, s.tok0 - before), p.nq);
      va = (int)((long long)i0 * group / kTile);
      if (p.window) {
        const long long i1 = min((long long)p.nq, max(0LL, (long long)min(s.tok0 + kTile, s.len) + p.window - before - 1));
        vb = (int)((i1 * group + kTile - 1) / kTile);
      }
      if (i0 == p.nq) vb = va;
    }
    s.ca = max(ca, va);
    s.cb = max(s.ca, min(cb, vb));
    return true;
  }
  return false;
}

template <int QT, int D>
__global__ void __launch_bounds__(Wt<QT, D>::kThreads, 1) weights_tiles_kernel(const __grid_constant__ WtArgs a, int* err) {
  typedef KvL<QT, D> L;
  typedef Wt<QT, D> C;
  constexpr int S = C::kStages, I = C::kInfos, NB = L::kNB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;                                                    // [S][D / 64][128 rows][64]
  float* s_lse = reinterpret_cast<float*>(s_q + S * C::kStageBytes);      // [I][128], in units of -log2
  int* s_lo = reinterpret_cast<int*>(s_lse + I * kTile);                  // [I][128]
  int* s_hi = s_lo + I * kTile;
  int* s_span = s_hi + I * kTile;                                         // [I][4]: largest lo, least hi of the rows
  float* s_red = reinterpret_cast<float*>(s_span + I * 4);                // [2][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_red + 2 * kTile);
  uint64_t* q_full = bars;              // [S]
  uint64_t* q_empty = q_full + S;       // [S]
  uint64_t* i_full = q_empty + S;       // [I]
  uint64_t* i_empty = i_full + I;       // [I]
  uint64_t* s_full = i_empty + I;       // [2]
  uint64_t* s_empty = s_full + 2;       // [2]
  uint64_t* k_full = s_empty + 2;
  uint64_t* k_empty = k_full + 1;
  uint64_t* mma_done = k_empty + 1;
  static_assert((2 * S + 2 * I + 7) * 8 <= 512, "barriers of weights_tiles_kernel");
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort_word, s_stop[2], s_last, s_b;
  __shared__ long long s_total, s_base;
  __shared__ int s_lens[kLens];
  volatile int* s_abort = &s_abort_word;

  const KvAttnParams& p = a.p;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int group = p.heads / p.c.heads, n_rows = p.nq * group;

  if (threadIdx.x == 0) {
    for (int x = 0; x < S; ++x) {
      mbar_init(&q_full[x], 128);
      mbar_init(&q_empty[x], 1);
    }
    for (int x = 0; x < I; ++x) {
      mbar_init(&i_full[x], 1);
      mbar_init(&i_empty[x], 4);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&s_empty[x], 4);
    }
    mbar_init(k_full, 8);
    mbar_init(k_empty, 1);
    mbar_init(mma_done, 1);
    s_abort_word = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 12) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  let_next();
  wait_before();
  // ---- the line's length, and the sequence in which this CTA's share begins
  auto span_of = [&](int b) { return (long long)((sequence_length(p, b, err) + kTile - 1) / kTile) * p.c.heads * a.chunks; };
  if (warp == 0) {
    long long total = 0;
    for (int b = lane; b < p.batch; b += 32) total += span_of(b);
#pragma unroll
    for (int x = 16; x; x >>= 1) total += __shfl_xor_sync(~0u, total, x);
    const long long ctas = min((long long)gridDim.x, total), p0 = blockIdx.x < ctas ? total * blockIdx.x / ctas : total;
    long long base = 0;
    int found = p.batch;
    for (int b0 = 0; b0 < p.batch && found == p.batch; b0 += 32) {
      const long long n = b0 + lane < p.batch ? span_of(b0 + lane) : 0;
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
    // lengths from there on, as far as the share goes
    long long past = base;
    const long long p1 = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : 0;
    for (int b0 = found; b0 < p.batch && b0 - found < kLens && past < p1; b0 += 32) {
      const int len = b0 + lane < p.batch ? sequence_length(p, b0 + lane, err) : 0;
      s_lens[b0 - found + lane] = len;
      long long n = (long long)((len + kTile - 1) / kTile) * p.c.heads * a.chunks;
#pragma unroll
      for (int x = 16; x; x >>= 1) n += __shfl_xor_sync(~0u, n, x);
      past += n;
    }
    if (lane == 0) {
      s_total = total;
      s_base = base;
      s_b = found;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const long long total = s_total, ctas = min((long long)gridDim.x, total);
  const bool works = blockIdx.x < ctas;
  const long long p0 = works ? total * blockIdx.x / ctas : 0;
  WtWalk w{p0, works ? total * (blockIdx.x + 1) / ctas : 0, s_base, s_b, s_lens, s_b};
  WtSeg s;
  const float sl2 = p.scale * kLog2e;
  uint32_t n = 0;     // chunks so far
  uint32_t segs = 0;  // tiles with a chunk so far
  bool ok = true;

  if (warp < 8) {
    // ---- K into TMEM, then the weights of every other chunk: a thread a token
    const int e = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t tiles = 0;
    while (wt_next(a, err, w, s)) {
      const int tok = s.tok0 + row;
      float sum = 0.f;
      if (s.ca < s.cb) {
        if (ok && segs) ok = mbar_wait(k_empty, (segs - 1) & 1, s_abort, err, kErrWaitEmpty);
        ok = __all_sync(~0u, ok);
        if (ok) {
          tc_fence_after();
          const uint8_t* gp = nullptr;
          if (tok < s.len) {
            const int gi = tok >> 4, per_page = p.c.page_size >> 4;
            long long page = p.pages[s.b * p.pages_stride + gi / per_page];
            if (page < 0 || page >= p.c.n_pages) {
              atomicCAS(err, 0, kDevErrIndex);
              page = 0;
            }
            gp = p.c.data + kv_group_offset<QT, D>(p.c, page, s.head, 0, gi % per_page);
          }
          constexpr int BW = L::kBits / 4;  // words of a lane's piece in one block
          uint32_t code[NB / 2][4][BW];
          __half sc[NB / 2], mn[NB / 2];
#pragma unroll
          for (int x = 0; x < NB / 2; ++x) {
            const int blk = e * (NB / 2) + x;
            sc[x] = mn[x] = __ushort_as_half(0);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int y = 0; y < BW; ++y) code[x][t][y] = QT == QT_Q8_0 ? 0x80808080u : 0u;
            if (gp) {
              sc[x] = *reinterpret_cast<const __half*>(gp + L::k_scale(tok & 15, blk));
              if (QT == QT_Q4_1) mn[x] = *reinterpret_cast<const __half*>(gp + L::kSc + L::k_scale(tok & 15, blk));
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                const uint32_t* at = reinterpret_cast<const uint32_t*>(gp + L::k_val(tok & 15, blk, t));
#pragma unroll
                for (int y = 0; y < BW; ++y) code[x][t][y] = at[y];
              }
            }
          }
#pragma unroll
          for (int x = 0; x < NB / 2; ++x) {
            const int blk = e * (NB / 2) + x;
            const __half2 s2 = __half2half2(sc[x]);
            const float s1 = __half2float(sc[x]), m1 = __half2float(mn[x]);
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              uint32_t v[4];
              if (QT == QT_Q8_0) {
                byte_pairs(code[x][t][0], v[0], v[1]);
                byte_pairs(code[x][t][BW - 1], v[2], v[3]);
              } else {
                nibble_pairs<QT>(code[x][t][0], v);
              }
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                __half2 h, r;
                if (QT == QT_Q4_1) {
                  const float2 f = __half22float2(u32_h2(v[y]));
                  const float f0 = fmaf(f.x, s1, m1), f1 = fmaf(f.y, s1, m1);
                  h = __floats2half2_rn(f0, f1);
                  const float2 back = __half22float2(h);
                  r = __floats2half2_rn(f0 - back.x, f1 - back.y);
                } else {
                  h = __hmul2(u32_h2(v[y]), s2);
                  r = __hfma2(u32_h2(v[y]), s2, __hneg2(h));
                }
                hi[4 * t + y] = h2_u32(h);
                lo[4 * t + y] = h2_u32(r);
              }
            }
            KV_TMEM_ST16(tmem + lane_off + blk * 16, hi);
            KV_TMEM_ST16(tmem + lane_off + D / 2 + blk * 16, lo);
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(k_full);
        }
        ++segs;
      }
      for (int c = s.ca; c < s.cb; ++c, ++n) {
        if ((int)(n & 1) != e) continue;
        ok = ok && mbar_wait(&i_full[n % I], (n / I) & 1, s_abort, err, kErrWaitFull);
        ok = ok && mbar_wait(&s_full[e], (n >> 1) & 1, s_abort, err, kErrWaitTmemFull);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        tc_fence_after();
        const int info = n % I * kTile;
        const float* lse = s_lse + info;
        const uint32_t at = tmem + lane_off + C::kS + e * kTile;
        const bool whole = s_span[n % I * 4] <= s.tok0 && s_span[n % I * 4 + 1] >= min(s.tok0 + kTile, s.len);
        const unsigned long long scale2 = f2_pack(sl2, sl2);
        unsigned long long acc[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        auto add = [&](const uint32_t (&r)[32], int c0, auto masked) {
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            const float4 l = *reinterpret_cast<const float4*>(lse + c0 + x);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float e0, e1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(r[x + 2 * y]), __uint_as_float(r[x + 2 * y + 1])), scale2,
                               y ? f2_pack(l.z, l.w) : f2_pack(l.x, l.y)),
                        e0, e1);
              e0 = ex2_approx(e0), e1 = ex2_approx(e1);
              if (decltype(masked)::value) {
                const int2 a0 = *reinterpret_cast<const int2*>(s_lo + info + c0 + x + 2 * y);
                const int2 a1 = *reinterpret_cast<const int2*>(s_hi + info + c0 + x + 2 * y);
                if (tok < a0.x || tok >= a1.x) e0 = 0.f;
                if (tok < a0.y || tok >= a1.y) e1 = 0.f;
              }
              acc[y] = f2_add(acc[y], f2_pack(e0, e1));
            }
          }
        };
        auto sweep = [&](auto masked) {
          uint32_t ra[32], rb[32];
          KV_TMEM_LD32(at, ra);
          tc_wait_ld();
#pragma unroll 1
          for (int c0 = 0; c0 < kTile; c0 += 64) {
            KV_TMEM_LD32(at + c0 + 32, rb);
            add(ra, c0, masked);
            tc_wait_ld();
            KV_TMEM_LD32(at + ((c0 + 64) & (kTile - 1)), ra);  // unused at the end
            add(rb, c0 + 32, masked);
            tc_wait_ld();
          }
        };
        if (whole) sweep(std::false_type());
        else sweep(std::true_type());
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_empty[e]);
          mbar_arrive(&i_empty[n % I]);
        }
        float s0, s1, s2, s3;
        f2_unpack(acc[0], s0, s1);
        f2_unpack(acc[1], s2, s3);
        sum += (s0 + s1) + (s2 + s3);
      }
      // ---- both halves of the rows, then the token's weight or this CTA's part of it. The barriers are taken also after a wait ran
      // out, until both warpgroups have seen that: one thread says so for all.
      const uint32_t turn = tiles++ & 1;
      if (e == 1) {
        s_red[turn * kTile + row] = sum;
        if (row == 0) s_stop[turn] = *s_abort;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (s_stop[turn]) break;
      if (e == 1) continue;
      sum += s_red[turn * kTile + row];
      float* to = a.w.w + s.b * a.w.w_b + s.head * a.w.w_h;
      if (s.whole) {
        if (tok < s.len) to[tok] = a.w.decay != 0.f ? fmaf(a.w.decay, to[tok], sum) : sum;
        continue;
      }
      const long long c0 = ((s.start + 1) * ctas - 1) / total, c1 = min(ctas - 1, ((s.start + a.chunks) * ctas - 1) / total);
      __stcg(a.part + (2 * (long long)blockIdx.x + (s.start > p0 ? 1 : 0)) * kTile + row, sum);
      __threadfence();
      asm volatile("bar.sync 2, 128;" ::: "memory");
      if (row == 0) s_last = atomicAdd(a.count + c0, 1) == (int)(c1 - c0);
      asm volatile("bar.sync 2, 128;" ::: "memory");
      if (s_last) {
        __threadfence();
        sum = 0.f;
        const int second = s.start > total * c0 / ctas;
        for (long long k = c0; k <= c1; ++k) sum += __ldcg(a.part + (2 * k + (k == c0 ? second : 0)) * kTile + row);
        if (tok < s.len) to[tok] = a.w.decay != 0.f ? fmaf(a.w.decay, to[tok], sum) : sum;
        if (row == 0) a.count[c0] = 0;
      }
    }
  } else if (warp < 12) {
    // ---- query rows into the swizzled slots
    constexpr int PR = D / 8, kStep = 128 / PR;  // 16-byte pieces of a row, rows of a pass
    const int t = threadIdx.x - 256, piece = t % PR, row0 = t / PR;
    const int step_h = kStep % group;
    const long long step = kStep / group * p.q_n + step_h * p.q_h, turn = p.q_n - group * p.q_h;  // to the row kStep on; where its head wraps
    while (ok && wt_next(a, err, w, s)) {
      for (int c = s.ca; c < s.cb; ++c, ++n) {
        ok = __all_sync(~0u, mbar_wait(&q_empty[n % S], ((n / S) & 1) ^ 1, s_abort, err, kErrWaitEmpty));
        if (!ok) break;
        const int r0 = c * kTile + row0, i0 = r0 / group;
        int hh = r0 - i0 * group;
        const __half* from = p.q + s.b * p.q_b + i0 * p.q_n + (s.head * group + hh) * p.q_h + 8 * piece;
        const uint32_t to = smem_u32(s_q) + n % S * C::kStageBytes + piece / 8 * kSlot;
#pragma unroll 8
        for (int x = 0; x < PR; ++x) {
          const int row = row0 + x * kStep;
          const bool there = r0 + x * kStep < n_rows;  // the other rows are zeros
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + row * 128 + (((piece & 7) ^ (row & 7)) * 16)),
                       "l"(there ? from : p.q), "r"(there ? 16 : 0)
                       : "memory");
          from += step;
          hh += step_h;
          if (hh >= group) hh -= group, from += turn;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        mbar_arrive(&q_full[n % S]);
      }
    }
  } else if (warp == 13) {
    // ---- ln sums and spans of the rows, 4 a lane
    while (ok && wt_next(a, err, w, s)) {
      for (int c = s.ca; c < s.cb; ++c, ++n) {
        float4 l;
        int4 lo4, hi4;
        float* lv = reinterpret_cast<float*>(&l);
        int *lov = reinterpret_cast<int*>(&lo4), *hiv = reinterpret_cast<int*>(&hi4);
        int max_lo = 0, min_hi = 0x7FFFFFFF;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int rr = c * kTile + 4 * lane + x;
          lv[x] = -INFINITY;  // no row: no weight, and its zeros in the product are finite
          lov[x] = hiv[x] = 0;
          if (rr < n_rows) {
            const int ii = rr / group;
            const float ls = p.lse[((long long)s.b * p.nq + ii) * p.heads + s.head * group + rr - ii * group];
            if (ls != -INFINITY) {  // else a row that has seen nothing, and sees nothing here
              lv[x] = -ls * kLog2e;
              row_span(p, s.len, ii, &lov[x], &hiv[x]);
            }
            max_lo = max(max_lo, lov[x]);
            min_hi = min(min_hi, hiv[x]);
          }
        }
        max_lo = __reduce_max_sync(~0u, max_lo);
        min_hi = __reduce_min_sync(~0u, min_hi);
        ok = __all_sync(~0u, mbar_wait(&i_empty[n % I], ((n / I) & 1) ^ 1, s_abort, err, kErrWaitEmpty));
        if (!ok) break;
        const int at = n % I * kTile + 4 * lane;
        *reinterpret_cast<float4*>(s_lse + at) = l;
        *reinterpret_cast<int4*>(s_lo + at) = lo4;
        *reinterpret_cast<int4*>(s_hi + at) = hi4;
        if (lane == 0) {
          s_span[n % I * 4] = max_lo;
          s_span[n % I * 4 + 1] = min_hi;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&i_full[n % I]);
      }
    }
  } else {
    // ---- the products
    constexpr uint32_t idesc = idesc_f16(kTile, kTile, 0);
    bool issued = false;
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
      if (!__all_sync(~0u, mbar_wait(bar, parity, s_abort, err, code))) return false;
      tc_fence_after();
      return true;
    };
    while (ok && wt_next(a, err, w, s)) {
      if (s.ca >= s.cb) continue;
      ok = wait(k_full, segs & 1, kErrWaitFull);
      ++segs;
      for (int c = s.ca; c < s.cb && ok; ++c, ++n) {
        ok = wait(&q_full[n % S], (n / S) & 1, kErrWaitFull) && wait(&s_empty[n & 1], ((n >> 1) & 1) ^ 1, kErrWaitTmemEmpty);
        if (!ok) break;
        const uint32_t d = tmem + C::kS + (n & 1) * kTile;
        const uint32_t q = smem_u32(s_q) + n % S * C::kStageBytes;
        if (elect_one()) {
#pragma unroll
          for (int part = 0; part < C::kParts; ++part) {
            const uint64_t dq = sdesc_k_sw128(q + part * kSlot);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              tc_mma_f16_ts(d, tmem + part * 32 + kk * 8, dq + kk * 2, idesc, part != 0 || kk != 0);
              tc_mma_f16_ts(d, tmem + D / 2 + part * 32 + kk * 8, dq + kk * 2, idesc, 1);
            }
          }
          tc_commit(&q_empty[n % S]);
          tc_commit(&s_full[n & 1]);
          if (c == s.cb - 1) tc_commit(k_empty);
        }
        issued = true;
        __syncwarp();
      }
    }
    if (issued && elect_one()) {
      tc_commit(mma_done);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(mma_done, 0)) {
        if (globaltimer_ns() - t0 > kWaitNs) {
          atomicCAS(err, 0, kErrWaitDrain);
          break;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int QT, int D>
int launch_tiles(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  typedef Wt<QT, D> C;
  auto* k = weights_tiles_kernel<QT, D>;
  if (kernel_setup(k, C::kSmem) <= 0) return -13;
  const WtArgs a{p, w, w.part, w.count, (int)((p.nq * (long long)(p.heads / p.c.heads) + kTile - 1) / kTile)};
  return launch_dependent(k, dim3(sms), C::kThreads, C::kSmem, st, a, err);
}

template <int QT>
int tiles_d(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  return p.c.d == 64 ? launch_tiles<QT, 64>(p, w, sms, err, st)
                     : p.c.d == 128 ? launch_tiles<QT, 128>(p, w, sms, err, st) : launch_tiles<QT, 256>(p, w, sms, err, st);
}

}  // namespace

size_t kv_weights_tc_part(int sms) { return (size_t)2 * sms * kTile * 4; }

int kv_weights_tc(const KvAttnParams& p, const KvWeights& w, int sms, int* err, cudaStream_t st) {
  return p.c.type == QT_Q4_0 ? tiles_d<QT_Q4_0>(p, w, sms, err, st)
                             : p.c.type == QT_Q4_1 ? tiles_d<QT_Q4_1>(p, w, sms, err, st) : tiles_d<QT_Q8_0>(p, w, sms, err, st);
}

}  // namespace s3b
