// Writing and reading the quantised key / value cache (layout: kv_cache.cuh).
#include <algorithm>

#include "kv_cache.cuh"

namespace s3b {

namespace {

constexpr float kLimit = 65024.0f;  // f16's largest value less what rounding scale and minimum of a q4_1 block can add

struct Job {
  KvCache c;
  KvRows r;
  const long long* slots;
  long long n;
  int* err;
  int tokens;         // that a block takes
  unsigned div_mul;   // slot / page_size = (slot * div_mul) >> (32 + div_shift) for slots below 2^31; 0: 64-bit division
  int div_shift;
  long long page_bytes, v_bytes;  // of a page; from a page's keys of a head to its values
};

// Byte offset of the keys of a slot's group for head 0, and the token's place in the group; false for a slot that is
// skipped.
template <int HALF>
__device__ __forceinline__ bool slot_place(const Job& j, long long slot, long long* at, int* tok) {
  if (slot < 0) return false;
  if (slot >= j.c.n_pages * j.c.page_size) {
    atomicCAS(j.err, 0, kDevErrIndex);
    return false;
  }
  int pos;
  if (j.div_mul) {
    const unsigned s = (unsigned)slot, q = __umulhi(s, j.div_mul) >> j.div_shift;
    *at = q * j.page_bytes;
    pos = (int)(s - q * j.c.page_size);
  } else {
    const long long q = slot / j.c.page_size;
    *at = q * j.page_bytes;
    pos = (int)(slot - q * j.c.page_size);
  }
  *at += (pos >> 4) * HALF;
  *tok = pos & 15;
  return true;
}

// 8 values of a row as they are in memory, and as f32.
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void load8(const T* at, Eight<T>& r) {
#pragma unroll
  for (int e = 0; e < (int)sizeof(T) / 2; ++e) r.w[e] = reinterpret_cast<const uint4*>(at)[e];
}
__device__ __forceinline__ void floats8(const Eight<float>& r, float (&x)[8]) {
  const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
}
__device__ __forceinline__ void floats8(const Eight<__half>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(u32_h2(w[e]));
    x[2 * e] = f.x, x[2 * e + 1] = f.y;
  }
}
__device__ __forceinline__ float max3n(float a, float b, float c) {  // a NaN among them stays
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3n(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// largest and smallest value of the block that four neighbouring lanes hold
__device__ __forceinline__ void block_range(const float (&x)[8], float* hi, float* lo) {
  *hi = max3n(max3n(x[0], x[1], x[2]), max3n(x[3], x[4], x[5]), max3n(x[6], x[7], x[7]));
  *lo = min3n(min3n(x[0], x[1], x[2]), min3n(x[3], x[4], x[5]), min3n(x[6], x[7], x[7]));
#pragma unroll
  for (int s = 1; s < 4; s <<= 1) {
    const float h = __shfl_xor_sync(~0u, *hi, s), l = __shfl_xor_sync(~0u, *lo, s);
    *hi = max3n(*hi, h, h);
    *lo = min3n(*lo, l, l);
  }
}

constexpr uint32_t kWhole = 0x4B000000u;  // 2^23 as f32

// x / N rounded to nearest: 1 / N as the sum of two floats, a product with each (Brisebarre, Muller and Raina, Accelerating
// correctly rounded floating-point division when the divisor is known in advance). Holds for every significand with N = 15
// and 127 (all 2^23 compared) where nothing is subnormal: far below, the scale is 0 in f16 and the codes mean nothing.
template <int N>
__device__ __forceinline__ float over(float x) {
  constexpr float hi = 1.0f / N, lo = (float)(1.0 / N - (double)hi);
  return __fmaf_rn(x, hi, __fmul_rn(x, lo));
}

// Quantises the block of 32 values that four neighbouring lanes hold, 8 each (t: which 8), in the steps of
// quantize_row_host, each rounded to f32 as there. The codes come out as kWhole + code (q8_0: code + 128): truncation of
// a value >= 0 is the addition of 2^23 rounded to zero. A 4-bit code may still be 16 here: pack_nibbles takes it to 15.
template <int QT>
__device__ __forceinline__ void quantise8(float (&x)[8], int t, uint32_t (&code)[8], __half& scale, __half& low) {
  float hi, lo;
  block_range(x, &hi, &lo);
  if (__any_sync(~0u, !(hi <= kLimit && lo >= -kLimit))) {  // what is not finite or beyond the limit, rare
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -kLimit), kLimit) : 0.f;
    block_range(x, &hi, &lo);
  }
  low = __ushort_as_half(0);
  float d;
  if (QT == QT_Q4_1) {
    d = over<15>(__fsub_rn(hi, lo));
    low = __float2half_rn(lo);
  } else if (QT == QT_Q8_0) {
    d = over<127>(fmaxf(hi, -lo));
  } else {
    float v = hi > -lo ? hi : lo;
    if (__any_sync(~0u, hi == -lo && hi != 0.f)) {  // the first of the two
      int first = 32;
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (fabsf(x[e]) == hi) first = 8 * t + e;
      float mine = lo;
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (fabsf(x[e]) == hi) mine = x[e];
#pragma unroll
      for (int s = 1; s < 4; s <<= 1) {
        const int f = __shfl_xor_sync(~0u, first, s);
        const float m = __shfl_xor_sync(~0u, mine, s);
        if (f < first) first = f, mine = m;
      }
      if (hi == -lo) v = mine;
    }
    d = v * -0.125f;
  }
  const float id = d != 0.f ? __frcp_rn(d) : 0.f;
  scale = __float2half_rn(d);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (QT == QT_Q8_0) {
      const float y = __fmul_rn(x[e], id);
      const uint32_t q = min(__float_as_uint(__fadd_rz(__fadd_rz(fabsf(y), 0.5f), 8388608.f)), kWhole + 127u);
      code[e] = y < 0.f ? 2u * kWhole + 128u - q : q + 128u;  // halves away from zero
    } else {
      const float y = QT == QT_Q4_0 ? __fadd_rn(__fmul_rn(x[e], id), 8.5f)
                                    : __fadd_rn(__fmul_rn(__fsub_rn(x[e], lo), id), 0.5f);
      code[e] = __float_as_uint(__fadd_rz(y, 8388608.f));
    }
  }
}

// four 8-bit codes as bytes
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t* c) {
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
// eight 4-bit codes, no more than 15 each: those of pair e at bits 4 e and 16 + 4 e. A pair is values 2 e, 2 e + 1 (keys) or
// e, e + 4 (values).
template <bool APART>
__device__ __forceinline__ uint32_t pack_nibbles(const uint32_t (&c)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t pair = __byte_perm(APART ? c[e] : c[2 * e], APART ? c[e + 4] : c[2 * e + 1], 0x5410);
    asm("min.u16x2 %0, %1, %2;" : "=r"(pair) : "r"(pair), "r"(0x000F000Fu));
    w += pair << (4 * e);
  }
  return w;
}

// Four lanes a block of 32 values, 8 each: rows are read in 16-byte pieces, and the 8 values of a lane are a whole word of
// the keys' layout (4-bit codes; two words of 8-bit ones) and two pieces of the values'. The blocks walk over the tokens of
// their head, and the K and V rows of the next two tokens are on their way while these are quantised (loading, then quantising,
// then storing left the memory idle half of the time: 72 -> 59 us for the case below).
// Measured: 65536 tokens, 4 heads of 128, q4_1 from f16: 176 MB in 53 us cold, 3.3 TB/s (a copy of as many bytes takes 35 us).
// Instruction issue bounds it (77% of the cycles): a block's range, its two divisions and five steps a value, all in f32 to
// give the codes of the host's quantiser, one value an instruction.
template <int QT, int D, typename T>
__global__ void __launch_bounds__(256) write_kernel(const __grid_constant__ Job j) {
  typedef KvL<QT, D> L;
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;  // lanes of a row, rows of a pass
  const int head = blockIdx.x % j.c.heads;
  const long long step = (long long)(gridDim.x / j.c.heads) * j.tokens;
  const int c8 = threadIdx.x % kLanes, t = c8 & 3, b = c8 >> 2;
  uint8_t* base = j.c.data + head * 2 * j.v_bytes;
  const T* k = reinterpret_cast<const T*>(j.r.k) + head * j.r.k_h + c8 * 8;
  const T* v = reinterpret_cast<const T*>(j.r.v) + head * j.r.v_h + c8 * 8;
  Eight<T> raw[2][2] = {};
  long long slot[2];
  auto load = [&](long long i0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long long i = i0 + u * kRows;
      slot[u] = -1;
      if (i < j.n) {
        slot[u] = j.slots[i];
        load8(k + i * j.r.k_n, raw[u][0]);
        load8(v + i * j.r.v_n, raw[u][1]);
      }
    }
  };
  let_next();
  wait_before();
  long long i0 = (long long)(blockIdx.x / j.c.heads) * j.tokens;
  load(i0 + threadIdx.x / kLanes);
  for (; i0 < j.n; i0 += step) {
    Eight<T> now[2][2];
    long long at[2];
    int tok[2];
    bool use[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      now[u][0] = raw[u][0];
      now[u][1] = raw[u][1];
      use[u] = slot_place<L::kHalf>(j, slot[u], &at[u], &tok[u]);
    }
    load(i0 + step + threadIdx.x / kLanes);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        // the lanes of a skipped token go along: the lanes of a block exchange values
        float x[8];
        uint32_t c[8];
        __half scale, low;
        floats8(now[u][kv], x);
        quantise8<QT>(x, t, c, scale, low);
        if (!use[u]) continue;
        uint8_t* gp = base + at[u] + kv * j.v_bytes;
        if (L::kBits == 8) {
          const uint32_t w0 = pack_bytes(c), w1 = pack_bytes(c + 4);
          if (kv == 0) {
            *reinterpret_cast<uint2*>(gp + L::k_val(tok[u], b, t)) = make_uint2(w0, w1);
          } else {
            *reinterpret_cast<uint32_t*>(gp + L::v_val(tok[u], b, 2 * t)) = w0;
            *reinterpret_cast<uint32_t*>(gp + L::v_val(tok[u], b, 2 * t + 1)) = w1;
          }
        } else if (kv == 0) {
          *reinterpret_cast<uint32_t*>(gp + L::k_val(tok[u], b, t)) = pack_nibbles<false>(c);
        } else {
          const uint32_t w = pack_nibbles<true>(c);
          *reinterpret_cast<uint16_t*>(gp + L::v_val(tok[u], b, 2 * t)) = (uint16_t)w;
          *reinterpret_cast<uint16_t*>(gp + L::v_val(tok[u], b, 2 * t + 1)) = (uint16_t)(w >> 16);
        }
        if (t == 0) {
          __half* sp = reinterpret_cast<__half*>(gp + (kv ? L::v_scale(tok[u], b) : L::k_scale(tok[u], b)));
          sp[0] = scale;
          if (QT == QT_Q4_1) sp[L::kSc / 2] = low;
        }
      }
    }
  }
}

// The reverse, in the same shape: 8 values of a row a lane, K and V of two tokens read before any is unpacked. Bound by
// memory: 65536 tokens, 4 heads of 128, q4_1 to f16: 176 MB in 43 us cold, 4.1 TB/s, where a copy of as many bytes takes 35 us.
// Blocks that stay and read ahead and streaming stores were no faster (47 us each, against 45 of that time).
template <int QT, int D, typename T>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ Job j) {
  typedef KvL<QT, D> L;
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;
  const int head = blockIdx.x % j.c.heads;
  const long long first = (long long)(blockIdx.x / j.c.heads) * j.tokens + threadIdx.x / kLanes;
  const int c8 = threadIdx.x % kLanes, t = c8 & 3, b = c8 >> 2;
  const uint8_t* base = j.c.data + head * 2 * j.v_bytes;
  uint32_t w[2][2][2];
  __half sc[2][2], low[2][2];
  let_next();
  wait_before();
  long long slot[2], at[2];
  int tok[2];
  bool use[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) slot[u] = first + u * kRows < j.n ? j.slots[first + u * kRows] : -1;
#pragma unroll
  for (int u = 0; u < 2; ++u) use[u] = slot_place<L::kHalf>(j, slot[u], &at[u], &tok[u]);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {  // of a skipped slot: zeros
      w[u][kv][0] = w[u][kv][1] = L::kBits == 8 ? 0x80808080u : 0x88888888u;
      sc[u][kv] = low[u][kv] = __ushort_as_half(0);
    }
    if (use[u]) {
      const uint8_t *kp = base + at[u], *vp = kp + j.v_bytes;
      if (L::kBits == 8) {
        const uint2 k = *reinterpret_cast<const uint2*>(kp + L::k_val(tok[u], b, t));
        w[u][0][0] = k.x, w[u][0][1] = k.y;
        w[u][1][0] = *reinterpret_cast<const uint32_t*>(vp + L::v_val(tok[u], b, 2 * t));
        w[u][1][1] = *reinterpret_cast<const uint32_t*>(vp + L::v_val(tok[u], b, 2 * t + 1));
      } else {
        w[u][0][0] = *reinterpret_cast<const uint32_t*>(kp + L::k_val(tok[u], b, t));
        w[u][1][0] = __byte_perm(*reinterpret_cast<const uint16_t*>(vp + L::v_val(tok[u], b, 2 * t)),
                                 *reinterpret_cast<const uint16_t*>(vp + L::v_val(tok[u], b, 2 * t + 1)), 0x5410);
      }
      const __half* ks = reinterpret_cast<const __half*>(kp + L::k_scale(tok[u], b));
      const __half* vs = reinterpret_cast<const __half*>(vp + L::v_scale(tok[u], b));
      sc[u][0] = *ks, sc[u][1] = *vs;
      if (QT == QT_Q4_1) low[u][0] = ks[L::kSc / 2], low[u][1] = vs[L::kSc / 2];
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const long long i = first + u * kRows;
    if (i >= j.n) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      T* out = reinterpret_cast<T*>(kv ? j.r.v : j.r.k);
      if (!out) continue;
      // codes as exact f16 pairs, then one multiply-add in the output's type, rounded once: scales and minima are f16
      uint32_t p[4];
      if (L::kBits == 8) {
        byte_pairs(w[u][kv][0], p[0], p[1]);
        byte_pairs(w[u][kv][1], p[2], p[3]);
      } else {
        nibble_pairs<QT>(w[u][kv][0], p);
      }
      T* to = out + i * (kv ? j.r.v_n : j.r.k_n) + head * (kv ? j.r.v_h : j.r.k_h) + c8 * 8;
      constexpr bool kWide = sizeof(T) == 4;
      const bool apart = L::kBits == 4 && kv;  // a value word pairs values e and e + 4
      if (kWide) {
        const float s = __half2float(sc[u][kv]), m = __half2float(low[u][kv]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __half22float2(u32_h2(p[e]));
          x[apart ? e : 2 * e] = fmaf(f.x, s, m);
          x[apart ? e + 4 : 2 * e + 1] = fmaf(f.y, s, m);
        }
        reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        const __half2 s = __half2half2(sc[u][kv]), m = __half2half2(low[u][kv]);
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = h2_u32(__hfma2(u32_h2(p[e]), s, m));
        *reinterpret_cast<uint4*>(to) =
            apart ? make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410),
                               __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632))
                  : make_uint4(p[0], p[1], p[2], p[3]);
      }
    }
  }
}

typedef void (*JobKernel)(Job);

template <int QT, int D>
JobKernel job_kernel(bool write, bool f32) {
  return write ? (f32 ? write_kernel<QT, D, float> : write_kernel<QT, D, __half>)
               : (f32 ? read_kernel<QT, D, float> : read_kernel<QT, D, __half>);
}
template <int QT>
JobKernel job_kernel_d(int d, bool write, bool f32) {
  return d == 64 ? job_kernel<QT, 64>(write, f32)
                 : d == 128 ? job_kernel<QT, 128>(write, f32) : job_kernel<QT, 256>(write, f32);
}

int launch(bool write, const KvCache& c, const KvRows& r, const long long* slots, long long n, int* err,
           cudaStream_t st) {
  const long long region = kv_cache_bytes(c) / c.n_pages / c.heads;  // of one page and head
  Job j{c, r, slots, n, err, 2 * 256 / (c.d / 8), 0, 0, region * c.heads, region / 2};
  if (c.n_pages * c.page_size < (1LL << 31) && c.page_size > 1) {
    // shift = ceil(log2(page_size)) - 1, mul = ceil(2^(32 + shift) / page_size) < 2^32: exact for slots below 2^31
    while ((2LL << j.div_shift) < c.page_size) ++j.div_shift;
    j.div_mul = (unsigned)(((1ULL << (32 + j.div_shift)) + c.page_size - 1) / c.page_size);
  }
  long long blocks = (n + j.tokens - 1) / j.tokens * c.heads;
  if (write) {  // blocks that walk: 6 an SM (71 to 95 registers: 2 or 3 of them at a time), a multiple of the heads
    const long long walking = 6LL * num_sms() / c.heads * c.heads;
    blocks = std::min(blocks, std::max(walking, (long long)c.heads));
  }
  if (blocks > 0x7fffffffLL) return -2;
  const JobKernel k = c.type == QT_Q4_0 ? job_kernel_d<QT_Q4_0>(c.d, write, r.f32)
                      : c.type == QT_Q4_1 ? job_kernel_d<QT_Q4_1>(c.d, write, r.f32)
                                          : job_kernel_d<QT_Q8_0>(c.d, write, r.f32);
  return launch_dependent(k, dim3((unsigned)blocks), 256, 0, st, j);
}

}  // namespace

long long kv_cache_bytes(const KvCache& c) {
  if ((c.type != QT_Q4_0 && c.type != QT_Q4_1 && c.type != QT_Q8_0) || (c.d != 64 && c.d != 128 && c.d != 256) ||
      c.heads <= 0 || c.page_size <= 0 || c.page_size % 16 || c.n_pages <= 0)
    return -1;
  const long long row = c.type == QT_Q8_0 ? c.d + c.d / 16 : c.type == QT_Q4_1 ? c.d / 2 + c.d / 8 : c.d / 2 + c.d / 16;
  const long long per_page = 2 * row * c.page_size;  // < 2^42
  const long long most = 1LL << 48;
  if (per_page > most / c.heads || c.n_pages > most / (per_page * c.heads)) return -1;
  return per_page * c.heads * c.n_pages;
}

int kv_cache_write(const KvCache& c, const KvRows& r, const long long* slots, long long n, int* err, cudaStream_t st) {
  return launch(true, c, r, slots, n, err, st);
}

int kv_cache_read(const KvCache& c, const KvRows& r, const long long* slots, long long n, int* err, cudaStream_t st) {
  return launch(false, c, r, slots, n, err, st);
}

}  // namespace s3b
