// Attention over the quantised key / value cache (layout: kv_cache.cuh).
//   s_j = scale * q . k_j,  p_j = exp(s_j - max s),  out = sum_j p_j v_j / sum_j p_j
// over the tokens j that the query sees.
#include "kv_cache.cuh"

namespace s3b {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Tokens of sequence b, held to what its page table can name.
__device__ __forceinline__ int sequence_length(const KvAttnParams& p, int b, int* err) {
  const int n = p.lengths[b];
  const int most = p.max_pages * p.c.page_size;
  if (n < 0 || n > most) {
    atomicCAS(err, 0, kDevErrIndex);
    return n < 0 ? 0 : most;
  }
  return n;
}

// Values 32 b + lane of a key (KV = 0) or value row.
template <int QT, int D, int KV>
__device__ __forceinline__ float cached(const uint8_t* gp, int tok, int b, int lane) {
  typedef KvL<QT, D> L;
  const __half* sp = reinterpret_cast<const __half*>(gp + (KV ? L::v_scale(tok, b) : L::k_scale(tok, b)));
  int code;
  if (L::kBits == 8) {
    code = (int)gp[KV ? L::v_val(tok, b, lane / 4) + lane % 4 : L::k_val(tok, b, lane / 8) + lane % 8] - 128;
  } else if (KV) {
    code = *reinterpret_cast<const uint16_t*>(gp + L::v_val(tok, b, lane / 4)) >> (4 * (lane % 4)) & 15;
  } else {
    code = *reinterpret_cast<const uint32_t*>(gp + L::k_val(tok, b, lane / 8)) >>
               (4 * (lane % 8 / 2) + 16 * (lane % 2)) & 15;
  }
  if (QT == QT_Q4_0) code -= 8;
  return (float)code * __half2float(sp[0]) + (QT == QT_Q4_1 ? __half2float(sp[L::kSc / 2]) : 0.f);
}

// One warp per query row, one token after the other.
template <int QT, int D>
__global__ void __launch_bounds__(128) row_kernel(KvAttnParams p, int* err) {
  typedef KvL<QT, D> L;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (long long)p.batch * p.nq * p.heads) return;
  const int h = (int)(row % p.heads), i = (int)(row / p.heads % p.nq), b = (int)(row / p.heads / p.nq);
  const int kvh = h / (p.heads / p.c.heads);
  const int len = sequence_length(p, b, err);
  int lo = 0, hi = len;
  if (p.causal) {
    hi = len - p.nq + i + 1;
    if (p.window) lo = max(0, hi - p.window);
  }
  const __half* q = p.q + b * p.q_b + i * p.q_n + h * p.q_h;
  float qv[L::kNB], o[L::kNB];
#pragma unroll
  for (int n = 0; n < L::kNB; ++n) {
    qv[n] = __half2float(q[32 * n + lane]) * p.scale * kLog2e;
    o[n] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = lo; j < hi; ++j) {
    long long page = p.pages[b * p.pages_stride + j / p.c.page_size];
    if (page < 0 || page >= p.c.n_pages) {
      atomicCAS(err, 0, kDevErrIndex);
      page = 0;
    }
    const int pos = j % p.c.page_size;
    const uint8_t* gp = p.c.data + kv_group_offset<QT, D>(p.c, page, kvh, pos >> 4);
    float s = 0.f;
#pragma unroll
    for (int n = 0; n < L::kNB; ++n) s += qv[n] * cached<QT, D, 0>(gp, pos & 15, n, lane);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    const float m2 = fmaxf(m, s);
    const float a = exp2f(m - m2), w = exp2f(s - m2);
    m = m2;
    l = l * a + w;
#pragma unroll
    for (int n = 0; n < L::kNB; ++n) o[n] = o[n] * a + w * cached<QT, D, 1>(gp, pos & 15, n, lane);
  }
  const float inv = hi > lo ? 1.f / l : 0.f;
#pragma unroll
  for (int n = 0; n < L::kNB; ++n) {
    const long long at = b * p.o_b + i * p.o_n + h * p.o_h + 32 * n + lane;
    if (p.out_f32)
      reinterpret_cast<float*>(p.out)[at] = o[n] * inv;
    else
      reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(o[n] * inv);
  }
  if (p.lse && lane == 0) p.lse[row] = hi > lo ? (m + log2f(l)) / kLog2e : -INFINITY;
}

typedef void (*AttnKernel)(KvAttnParams, int*);

template <int QT>
AttnKernel attn_kernel(int d) {
  return d == 64 ? row_kernel<QT, 64> : d == 128 ? row_kernel<QT, 128> : row_kernel<QT, 256>;
}

}  // namespace

int kv_attention(const KvAttnParams& p, int* err, cudaStream_t st) {
  const long long rows = (long long)p.batch * p.nq * p.heads;
  if ((rows + 3) / 4 > 0x7fffffffLL) return -2;
  const AttnKernel k = p.c.type == QT_Q4_0 ? attn_kernel<QT_Q4_0>(p.c.d)
                       : p.c.type == QT_Q4_1 ? attn_kernel<QT_Q4_1>(p.c.d) : attn_kernel<QT_Q8_0>(p.c.d);
  k<<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(p, err);
  return cudaGetLastError() == cudaSuccess ? 0 : -12;
}

}  // namespace s3b
