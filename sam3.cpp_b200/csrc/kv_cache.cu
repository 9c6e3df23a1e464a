// Writing and reading the quantised key / value cache (layout: kv_cache.cuh).
#include "kv_cache.cuh"

namespace s3b {

namespace {

constexpr float kLimit = 65024.0f;  // f16's largest value less what rounding scale and minimum of a q4_1 block can add

// One block of 32 values quantised in the steps of quantize_row_host, each rounded to f32 as there.
template <int QT>
__device__ __forceinline__ void quantise_block(const float (&x)[32], uint32_t (&code)[32], __half& scale, __half& low) {
  low = __float2half_rn(0.f);
  if (QT == QT_Q4_1) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
    const float d = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      code[i] = (uint32_t)min(15, (int)__fadd_rn(__fmul_rn(__fsub_rn(x[i], lo), id), 0.5f));
    scale = __float2half_rn(d);
    low = __float2half_rn(lo);
  } else {
    float amax = 0.f, vmax = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (fabsf(x[i]) > amax) {
        amax = fabsf(x[i]);
        vmax = x[i];
      }
    const float d = QT == QT_Q4_0 ? vmax * -0.125f : __fdiv_rn(amax, 127.0f);
    const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float y = __fmul_rn(x[i], id);
      code[i] = QT == QT_Q4_0 ? (uint32_t)max(0, min(15, (int)__fadd_rn(y, 8.5f)))
                              : (uint32_t)(max(-127, min(127, (int)roundf(y))) + 128);
    }
    scale = __float2half_rn(d);
  }
}

struct Job {
  KvCache c;
  KvRows r;
  const long long* slots;
  long long n;
  int* err;
};

// Group address and token of a slot; false for a slot that is skipped.
template <int QT, int D>
__device__ __forceinline__ bool slot_group(const Job& j, long long slot, int head, int kv, uint8_t** group, int* tok) {
  if (slot < 0) return false;
  const long long page = slot / j.c.page_size;
  if (page >= j.c.n_pages) {
    atomicCAS(j.err, 0, kDevErrIndex);
    return false;
  }
  const int pos = (int)(slot - page * j.c.page_size);
  *group = j.c.data + kv_group_offset<QT, D>(j.c, page, head, kv, pos >> 4);
  *tok = pos & 15;
  return true;
}

// One thread per block of 32 values.
template <int QT, int D, typename T>
__global__ void __launch_bounds__(128) write_kernel(Job j) {
  typedef KvL<QT, D> L;
  const long long u = (long long)blockIdx.x * 128 + threadIdx.x;
  const int b = (int)(u % L::kNB);
  const int kv = (int)(u / L::kNB % 2);
  const int head = (int)(u / (2 * L::kNB) % j.c.heads);
  const long long i = u / (2 * L::kNB) / j.c.heads;
  if (i >= j.n) return;
  uint8_t* gp;
  int tok;
  if (!slot_group<QT, D>(j, j.slots[i], head, kv, &gp, &tok)) return;
  const T* src = reinterpret_cast<const T*>(kv ? j.r.v : j.r.k) + i * (kv ? j.r.v_n : j.r.k_n) +
                 head * (kv ? j.r.v_h : j.r.k_h) + b * 32;
  float x[32];
  uint32_t code[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    const float f = (float)src[e];
    x[e] = f == f ? fminf(fmaxf(f, -kLimit), kLimit) : 0.f;
  }
  __half scale, low;
  quantise_block<QT>(x, code, scale, low);
  __half* sp = reinterpret_cast<__half*>(gp + (kv ? L::v_scale(tok, b) : L::k_scale(tok, b)));
  sp[0] = scale;
  if (QT == QT_Q4_1) sp[L::kSc / 2] = low;
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    if (L::kBits == 8) {
      gp[kv ? L::v_val(tok, b, e / 4) + e % 4 : L::k_val(tok, b, e / 8) + e % 8] = (uint8_t)code[e];
    }
  }
  if (L::kBits == 4) {
    if (kv) {
#pragma unroll
      for (int g = 0; g < 8; ++g)
        *reinterpret_cast<uint16_t*>(gp + L::v_val(tok, b, g)) =
            (uint16_t)(code[4 * g] | code[4 * g + 1] << 4 | code[4 * g + 2] << 8 | code[4 * g + 3] << 12);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t w = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) w |= code[8 * t + 2 * p] << (4 * p) | code[8 * t + 2 * p + 1] << (4 * p + 16);
        *reinterpret_cast<uint32_t*>(gp + L::k_val(tok, b, t)) = w;
      }
    }
  }
}

// One thread per block of 32 values.
template <int QT, int D, typename T>
__global__ void __launch_bounds__(128) read_kernel(Job j) {
  typedef KvL<QT, D> L;
  const long long u = (long long)blockIdx.x * 128 + threadIdx.x;
  const int b = (int)(u % L::kNB);
  const int kv = (int)(u / L::kNB % 2);
  const int head = (int)(u / (2 * L::kNB) % j.c.heads);
  const long long i = u / (2 * L::kNB) / j.c.heads;
  if (i >= j.n || !(kv ? j.r.v : j.r.k)) return;
  T* dst = reinterpret_cast<T*>(kv ? j.r.v : j.r.k) + i * (kv ? j.r.v_n : j.r.k_n) + head * (kv ? j.r.v_h : j.r.k_h) +
           b * 32;
  uint8_t* gp;
  int tok;
  if (!slot_group<QT, D>(j, j.slots[i], head, kv, &gp, &tok)) {
    for (int e = 0; e < 32; ++e) dst[e] = (T)0.f;
    return;
  }
  const __half* sp = reinterpret_cast<const __half*>(gp + (kv ? L::v_scale(tok, b) : L::k_scale(tok, b)));
  const float scale = __half2float(sp[0]);
  const float low = QT == QT_Q4_1 ? __half2float(sp[L::kSc / 2]) : 0.f;
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    int code;
    if (L::kBits == 8) {
      code = (int)gp[kv ? L::v_val(tok, b, e / 4) + e % 4 : L::k_val(tok, b, e / 8) + e % 8] - 128;
    } else if (kv) {
      code = *reinterpret_cast<const uint16_t*>(gp + L::v_val(tok, b, e / 4)) >> (4 * (e % 4)) & 15;
    } else {
      code = *reinterpret_cast<const uint32_t*>(gp + L::k_val(tok, b, e / 8)) >> (4 * (e % 8 / 2) + 16 * (e % 2)) & 15;
    }
    if (QT == QT_Q4_0) code -= 8;
    dst[e] = (T)__fadd_rn(__fmul_rn((float)code, scale), low);
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
  const long long blocks = (n * c.heads * 2 * (c.d / 32) + 127) / 128;
  if (blocks > 0x7fffffffLL) return -2;
  const JobKernel k = c.type == QT_Q4_0 ? job_kernel_d<QT_Q4_0>(c.d, write, r.f32)
                      : c.type == QT_Q4_1 ? job_kernel_d<QT_Q4_1>(c.d, write, r.f32)
                                          : job_kernel_d<QT_Q8_0>(c.d, write, r.f32);
  k<<<(unsigned)blocks, 128, 0, st>>>(Job{c, r, slots, n, err});
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
