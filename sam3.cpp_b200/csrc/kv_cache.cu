// Writing and reading the quantised key / value cache (layout: kv_cache.cuh).
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
  int vec;            // tokens that a block takes
  unsigned div_mul;   // slot / page_size = (slot * div_mul) >> (32 + div_shift) for slots below 2^31; 0: 64-bit division
  int div_shift;
};

// Page and position of a slot; false for a slot that is skipped.
__device__ __forceinline__ bool slot_place(const Job& j, long long slot, long long* page, int* pos) {
  if (slot < 0) return false;
  if (slot >= j.c.n_pages * j.c.page_size) {
    atomicCAS(j.err, 0, kDevErrIndex);
    return false;
  }
  if (j.div_mul) {
    const unsigned s = (unsigned)slot, q = __umulhi(s, j.div_mul) >> j.div_shift;
    *page = q;
    *pos = (int)(s - q * j.c.page_size);
  } else {
    *page = slot / j.c.page_size;
    *pos = (int)(slot - *page * j.c.page_size);
  }
  return true;
}

// 8 values of a row as f32.
__device__ __forceinline__ void load8(const float* at, float (&x)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(at)), b = __ldg(reinterpret_cast<const float4*>(at) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* at, float (&x)[8]) {
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(at));
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
    x[2 * e] = f.x, x[2 * e + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(float* at, const float (&x)[8]) {
  reinterpret_cast<float4*>(at)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(at)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__half* at, const float (&x)[8]) {
  __half2 h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
  *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(h);
}

// Quantises the block of 32 values that four neighbouring lanes hold, 8 each (t: which 8), in the steps of
// quantize_row_host, each rounded to f32 as there. Truncation of a value >= 0 is an addition of 2^23 rounded to zero.
template <int QT>
__device__ __forceinline__ void quantise8(float (&x)[8], int t, uint32_t (&code)[8], __half& scale, __half& low) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -kLimit), kLimit) : 0.f;
  low = __ushort_as_half(0);
  auto whole = [](float f) -> uint32_t { return __float_as_uint(__fadd_rz(f, 8388608.f)) & 0x7FFFFFu; };
  if (QT == QT_Q4_1) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(~0u, lo, s));
      hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, s));
    }
    const float d = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      code[e] = min(15u, whole(fmaxf(__fadd_rn(__fmul_rn(__fsub_rn(x[e], lo), id), 0.5f), 0.f)));
    scale = __float2half_rn(d);
    low = __float2half_rn(lo);
  } else {
    // the first value of largest magnitude
    float amax = fabsf(x[0]), vmax = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e)
      if (fabsf(x[e]) > amax) amax = fabsf(x[e]), vmax = x[e];
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
      const float v = __shfl_xor_sync(~0u, vmax, s);
      if (fabsf(v) > amax || (fabsf(v) == amax && (t & s))) amax = fabsf(v), vmax = v;
    }
    const float d = QT == QT_Q4_0 ? vmax * -0.125f : __fdiv_rn(amax, 127.0f);
    const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = __fmul_rn(x[e], id);
      if (QT == QT_Q4_0) {
        code[e] = min(15u, whole(fmaxf(__fadd_rn(y, 8.5f), 0.f)));
      } else {
        const int q = (int)min(127u, whole(__fadd_rz(fabsf(y), 0.5f)));  // halves away from zero
        code[e] = (uint32_t)((y < 0.f ? -q : q) + 128);
      }
    }
    scale = __float2half_rn(d);
  }
}

// Four lanes a block of 32 values, 8 each: rows are read in 16-byte pieces, and the 8 values of a lane are a whole word of
// the keys' layout (4-bit codes; two words of 8-bit ones) and two pieces of the values'. Bound by HBM: a block of threads
// reads its K and V rows of a few tokens before it quantises any of them, so that enough loads are in flight.
template <int QT, int D, typename T>
__global__ void __launch_bounds__(256) write_kernel(const __grid_constant__ Job j) {
  typedef KvL<QT, D> L;
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;  // lanes of a row, rows of a pass
  const int head = blockIdx.x % j.c.heads;
  const long long first = (long long)(blockIdx.x / j.c.heads) * j.vec;
  const int c8 = threadIdx.x % kLanes, t = c8 & 3, b = c8 >> 2;
  for (int r0 = 0; r0 < j.vec; r0 += 2 * kRows) {
    float x[2][2][8];
    long long page[2];
    int pos[2];
    bool use[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long long i = first + r0 + u * kRows + threadIdx.x / kLanes;
      use[u] = r0 + u * kRows + threadIdx.x / kLanes < j.vec && i < j.n && slot_place(j, __ldg(j.slots + i), &page[u], &pos[u]);
      if (use[u]) {
        load8(reinterpret_cast<const T*>(j.r.k) + i * j.r.k_n + head * j.r.k_h + c8 * 8, x[u][0]);
        load8(reinterpret_cast<const T*>(j.r.v) + i * j.r.v_n + head * j.r.v_h + c8 * 8, x[u][1]);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t kc[8], vc[8];
      __half ks, kl, vs, vl;
      if (!use[u]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[u][0][e] = x[u][1][e] = 0.f;
      }
      quantise8<QT>(x[u][0], t, kc, ks, kl);
      quantise8<QT>(x[u][1], t, vc, vs, vl);
      if (!use[u]) continue;
      const int tok = pos[u] & 15;
      uint8_t* kp = j.c.data + kv_group_offset<QT, D>(j.c, page[u], head, 0, pos[u] >> 4);
      uint8_t* vp = j.c.data + kv_group_offset<QT, D>(j.c, page[u], head, 1, pos[u] >> 4);
      if (L::kBits == 8) {
        *reinterpret_cast<uint2*>(kp + L::k_val(tok, b, t)) =
            make_uint2(kc[0] | kc[1] << 8 | kc[2] << 16 | kc[3] << 24, kc[4] | kc[5] << 8 | kc[6] << 16 | kc[7] << 24);
        *reinterpret_cast<uint32_t*>(vp + L::v_val(tok, b, 2 * t)) = vc[0] | vc[1] << 8 | vc[2] << 16 | vc[3] << 24;
        *reinterpret_cast<uint32_t*>(vp + L::v_val(tok, b, 2 * t + 1)) = vc[4] | vc[5] << 8 | vc[6] << 16 | vc[7] << 24;
      } else {
        *reinterpret_cast<uint32_t*>(kp + L::k_val(tok, b, t)) = kc[0] | kc[2] << 4 | kc[4] << 8 | kc[6] << 12 |
                                                                 kc[1] << 16 | kc[3] << 20 | kc[5] << 24 | kc[7] << 28;
        *reinterpret_cast<uint16_t*>(vp + L::v_val(tok, b, 2 * t)) =
            (uint16_t)(vc[0] | vc[1] << 4 | vc[2] << 8 | vc[3] << 12);
        *reinterpret_cast<uint16_t*>(vp + L::v_val(tok, b, 2 * t + 1)) =
            (uint16_t)(vc[4] | vc[5] << 4 | vc[6] << 8 | vc[7] << 12);
      }
      if (t == 0) {
        __half* sp = reinterpret_cast<__half*>(kp + L::k_scale(tok, b));
        sp[0] = ks;
        if (QT == QT_Q4_1) sp[L::kSc / 2] = kl;
      } else if (t == 1) {
        __half* sp = reinterpret_cast<__half*>(vp + L::v_scale(tok, b));
        sp[0] = vs;
        if (QT == QT_Q4_1) sp[L::kSc / 2] = vl;
      }
    }
  }
}

// The reverse, in the same shape: 8 values of a row a lane.
template <int QT, int D, typename T>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ Job j) {
  typedef KvL<QT, D> L;
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;
  const int head = blockIdx.x % j.c.heads;
  const long long first = (long long)(blockIdx.x / j.c.heads) * j.vec;
  const int c8 = threadIdx.x % kLanes, t = c8 & 3, b = c8 >> 2;
  for (int r0 = 0; r0 < j.vec; r0 += 2 * kRows) {
    uint32_t w[2][2][2];
    __half sc[2][2], low[2][2];
    long long i[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      i[u] = first + r0 + u * kRows + threadIdx.x / kLanes;
      if (r0 + u * kRows + threadIdx.x / kLanes >= j.vec) i[u] = j.n;
      long long page;
      int pos;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        w[u][kv][0] = w[u][kv][1] = L::kBits == 8 ? 0x80808080u : QT == QT_Q4_0 ? 0x88888888u : 0u;
        sc[u][kv] = low[u][kv] = __ushort_as_half(0);
      }
      if (i[u] < j.n && slot_place(j, __ldg(j.slots + i[u]), &page, &pos)) {
        const int tok = pos & 15;
        const uint8_t* kp = j.c.data + kv_group_offset<QT, D>(j.c, page, head, 0, pos >> 4);
        const uint8_t* vp = j.c.data + kv_group_offset<QT, D>(j.c, page, head, 1, pos >> 4);
        if (L::kBits == 8) {
          const uint2 k = __ldg(reinterpret_cast<const uint2*>(kp + L::k_val(tok, b, t)));
          w[u][0][0] = k.x, w[u][0][1] = k.y;
          w[u][1][0] = __ldg(reinterpret_cast<const uint32_t*>(vp + L::v_val(tok, b, 2 * t)));
          w[u][1][1] = __ldg(reinterpret_cast<const uint32_t*>(vp + L::v_val(tok, b, 2 * t + 1)));
        } else {
          w[u][0][0] = __ldg(reinterpret_cast<const uint32_t*>(kp + L::k_val(tok, b, t)));
          w[u][1][0] = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(vp + L::v_val(tok, b, 2 * t))) |
                       (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(vp + L::v_val(tok, b, 2 * t + 1))) << 16;
        }
        const __half* ks = reinterpret_cast<const __half*>(kp + L::k_scale(tok, b));
        const __half* vs = reinterpret_cast<const __half*>(vp + L::v_scale(tok, b));
        sc[u][0] = __ldg(ks), sc[u][1] = __ldg(vs);
        if (QT == QT_Q4_1) low[u][0] = __ldg(ks + L::kSc / 2), low[u][1] = __ldg(vs + L::kSc / 2);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (i[u] >= j.n) continue;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        T* out = reinterpret_cast<T*>(kv ? j.r.v : j.r.k);
        if (!out) continue;
        const float s = __half2float(sc[u][kv]), m = __half2float(low[u][kv]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          int code;
          if (L::kBits == 8)
            code = (int)(w[u][kv][e >> 2] >> (8 * (e & 3)) & 255u) - 128;
          else
            code = (int)(w[u][kv][0] >> (kv ? 4 * e : 4 * (e >> 1) + 16 * (e & 1)) & 15u) - (QT == QT_Q4_0 ? 8 : 0);
          x[e] = __fadd_rn(__fmul_rn((float)code, s), m);
        }
        store8(out + i[u] * (kv ? j.r.v_n : j.r.k_n) + head * (kv ? j.r.v_h : j.r.k_h) + c8 * 8, x);
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
  Job j{c, r, slots, n, err, 2 * 256 / (c.d / 8), 0, 0};  // two passes of rows a block
  if (c.n_pages * c.page_size < (1LL << 31) && c.page_size > 1) {
    // shift = ceil(log2(page_size)) - 1, mul = ceil(2^(32 + shift) / page_size) < 2^32: exact for slots below 2^31
    while ((2LL << j.div_shift) < c.page_size) ++j.div_shift;
    j.div_mul = (unsigned)(((1ULL << (32 + j.div_shift)) + c.page_size - 1) / c.page_size);
  }
  const long long blocks = (n + j.vec - 1) / j.vec * c.heads;
  if (blocks > 0x7fffffffLL) return -2;
  const JobKernel k = c.type == QT_Q4_0 ? job_kernel_d<QT_Q4_0>(c.d, write, r.f32)
                      : c.type == QT_Q4_1 ? job_kernel_d<QT_Q4_1>(c.d, write, r.f32)
                                          : job_kernel_d<QT_Q8_0>(c.d, write, r.f32);
  k<<<(unsigned)blocks, 256, 0, st>>>(j);
  return cudaGetLastError() == cudaSuccess ? 0 : -12;
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
