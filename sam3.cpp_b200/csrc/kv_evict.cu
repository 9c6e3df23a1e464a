// Eviction from the quantised key / value cache: each head's tokens of highest weight, moved in order to other pages.
#include <algorithm>

#include "kv_attention.cuh"
#include "kv_top.cuh"

namespace s3b {

namespace {

constexpr int kThreads = 1024;
constexpr int kMostKeys = 49152;  // weights of a CTA whose keys stay in its shared memory

struct EvictArgs {
  KvAttnParams p;  // source cache, pages, lengths
  KvEvict e;
  int keys;  // room for so many in a CTA's shared memory; those of more tokens are made from the weights again
};

// A unit is a sequence and a key / value head: one CTA, or a cluster of them (CL) that share the tokens. Measured: 2 heads of 524288
// tokens 30 us, 64 units of up to 16384 tokens 13 us (see kv_top.cuh for where the time goes).
template <int CL>
__global__ void __launch_bounds__(kThreads) choose_kernel(const __grid_constant__ EvictArgs a, int* err) {
  extern __shared__ uint32_t s_keys[];
  __shared__ TopShared<kThreads> s_top;
  const KvAttnParams& p = a.p;
  const int unit = blockIdx.x / CL, rank = blockIdx.x % CL;
  const int head = unit % p.c.heads, b = unit / p.c.heads;
  let_next();
  wait_before();
  const int len = sequence_length(p, b, err);
  const int keep = a.e.keep, m = min(len, keep);
  const float* weights = a.e.weights + b * a.e.w_b + head * a.e.w_h;
  int* kept = a.e.kept + (long long)unit * keep;
  if (head == 0 && rank == 0 && threadIdx.x == 0) a.e.lengths_out[b] = m;
  if (keep == 0) return;
  if (len <= keep) {
    for (long long i = rank * kThreads + threadIdx.x; i < keep; i += CL * kThreads) kept[i] = i < len ? (int)i : -1;
    return;
  }
  const int share = CL > 1 ? (int)(((long long)len + 32 * CL - 1) / (32 * CL)) * 32 : len;
  const int first = (int)min((long long)rank * share, (long long)len), n = min(share, len - first);
  const int sink = a.e.sink, from = len - a.e.recent;
  weights += first;
  auto fetch = [&](int i) { return weights[i]; };
  auto make = [&](int i, float w) { return first + i < sink || first + i >= from ? kTopForced : top_key(w); };
  auto emit = [&](uint32_t at, int i) { kept[at] = first + i; };
  if (share <= a.keys) {
    top_select<kThreads, CL>(
        s_top, n, (uint32_t)keep, fetch, [&](int i, float w) { return s_keys[i] = make(i, w); }, [&](int i) { return s_keys[i]; }, emit);
  } else {
    top_select<kThreads, CL>(s_top, n, (uint32_t)keep, fetch, make, [&](int i) { return make(i, weights[i]); }, emit);
  }
}

template <typename V>
__device__ __forceinline__ V load_as(const uint8_t* at) {
  return *reinterpret_cast<const V*>(at);
}
template <int BYTES>
struct Word;
template <>
struct Word<4> { typedef uint32_t type; };
template <>
struct Word<8> { typedef uint2 type; };
template <>
struct Word<16> { typedef uint4 type; };

// A warp a group of 16 places of the new pages: codes, scales and minima of its tokens are gathered as they are, in the widest
// words that one token has in the layout (keys 16 bytes, values 8 or 4), and stored as the group's consecutive words. Measured: 8
// sequences, 4096 tokens each kept of up to 16384, 8 heads of 128, q4_0: 38 MB read and as many written in 17 us; a token's values lie
// in 8-byte pieces of a group's, so two thirds of the sectors of all values are read for a quarter of the tokens.
template <int QT, int D>
__global__ void __launch_bounds__(128) move_kernel(const __grid_constant__ EvictArgs a, int* err) {
  typedef KvL<QT, D> L;
  constexpr int KW = L::kSB * L::kBits / 128;         // words of a token and super-block: keys
  constexpr int VB = L::kNBS * L::kBits / 2;          // bytes of a token's piece: values
  constexpr int NK = L::kVal / 16 / 32, NV = L::kVal / VB / 32, NS = 16 * L::kNB * L::kPlanes / 32;  // of a lane
  typedef typename Word<VB>::type VWord;
  typedef typename Word<L::kNB * 2>::type SWord;
  const KvAttnParams& p = a.p;
  const int lane = threadIdx.x & 31;
  const int groups = (a.e.keep + 15) / 16;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  let_next();
  wait_before();
  const long long unit = item / groups;
  if (unit >= (long long)p.batch * p.c.heads) return;
  const int i0 = (int)(item % groups) * 16;
  const int head = (int)(unit % p.c.heads), b = (int)(unit / p.c.heads);
  const int m = min(sequence_length(p, b, err), a.e.keep);
  float* w_out = a.e.weights_out ? a.e.weights_out + unit * a.e.keep + i0 + lane : nullptr;
  if (w_out && lane < 16 && i0 + lane >= m && i0 + lane < a.e.keep) *w_out = 0.f;
  if (i0 >= m) return;
  const int n = min(16, m - i0);
  const int mine = a.e.kept[unit * a.e.keep + i0 + min(lane & 15, n - 1)];
  if (w_out && lane < n) *w_out = a.e.weights[b * a.e.w_b + head * a.e.w_h + mine];
  const KvCache& to = a.e.to;
  long long new_page = a.e.pages_out[b * a.e.out_stride + i0 / to.page_size];
  if (new_page < 0 || new_page >= to.n_pages) {  // nowhere to go
    if (lane == 0) atomicCAS(err, 0, kDevErrIndex);
    return;
  }
  uint8_t* dk = to.data + kv_group_offset<QT, D>(to, new_page, head, 0, i0 % to.page_size >> 4);
  uint8_t* dv = dk + (long long)(to.page_size >> 4) * L::kHalf;
  // lane i: the keys of the group that holds token i % 16, and the token's place there
  long long page = p.pages[b * p.pages_stride + mine / p.c.page_size];
  if (page < 0 || page >= p.c.n_pages) {
    atomicCAS(err, 0, kDevErrIndex);
    page = 0;
  }
  const long long src = kv_group_offset<QT, D>(p.c, page, head, 0, mine % p.c.page_size >> 4);
  const int in = mine & 15;
  const long long v_offset = (long long)(p.c.page_size >> 4) * L::kHalf;
  uint4 k[NK];
  VWord v[NV];
  unsigned short vs[NS];
  SWord ks[L::kPlanes];
#pragma unroll
  for (int x = 0; x < NK; ++x) {
    const int w = x * 32 + lane, sb = w / (L::kSuper / 16), tok = w % (L::kSuper / 16) / KW;
    const uint8_t* at = p.c.data + __shfl_sync(~0u, src, tok) + sb * L::kSuper + __shfl_sync(~0u, in, tok) * KW * 16 + w % KW * 16;
    k[x] = load_as<uint4>(at);
  }
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int w = x * 32 + lane, sb = w / (L::kSuper / VB), r = w % (L::kSuper / VB);
    const int tok = (r >> 6) * 8 + (r >> 1 & 3) * 2 + (r & 1), g = r >> 3 & 7;
    const int from = __shfl_sync(~0u, in, tok);
    v[x] = load_as<VWord>(p.c.data + __shfl_sync(~0u, src, tok) + v_offset + sb * L::kSuper +
                          (((from >> 3) * 32 + g * 4 + ((from & 7) >> 1)) * 2 + (from & 1)) * VB);
  }
#pragma unroll
  for (int x = 0; x < L::kPlanes; ++x) ks[x] = load_as<SWord>(p.c.data + src + x * L::kSc + L::k_scale(in, 0));
#pragma unroll
  for (int x = 0; x < NS; ++x) {
    const int w = (x * 32 + lane) % (16 * L::kNB), plane = x * 32 / (16 * L::kNB);
    const int tok = (w >> 1 & 1) * 8 + (w >> 2) / L::kNB * 2 + (w & 1), blk = (w >> 2) % L::kNB;
    vs[x] = load_as<unsigned short>(p.c.data + __shfl_sync(~0u, src, tok) + v_offset + plane * L::kSc +
                                    L::v_scale(__shfl_sync(~0u, in, tok), blk));
  }
#pragma unroll
  for (int x = 0; x < NK; ++x) {
    const int w = x * 32 + lane;
    if (w % (L::kSuper / 16) / KW < n) reinterpret_cast<uint4*>(dk)[w] = k[x];
  }
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int w = x * 32 + lane, r = w % (L::kSuper / VB);
    if ((r >> 6) * 8 + (r >> 1 & 3) * 2 + (r & 1) < n) reinterpret_cast<VWord*>(dv)[w] = v[x];
  }
  if (lane < n) {
#pragma unroll
    for (int x = 0; x < L::kPlanes; ++x) *reinterpret_cast<SWord*>(dk + x * L::kSc + L::k_scale(lane, 0)) = ks[x];
  }
#pragma unroll
  for (int x = 0; x < NS; ++x) {
    const int w = (x * 32 + lane) % (16 * L::kNB), plane = x * 32 / (16 * L::kNB);
    if ((w >> 1 & 1) * 8 + (w >> 2) / L::kNB * 2 + (w & 1) < n)
      reinterpret_cast<unsigned short*>(dv + L::kVal + plane * L::kSc)[w] = vs[x];
  }
}

typedef void (*EvictKernel)(EvictArgs, int*);

template <int QT>
EvictKernel move_for(int d) {
  return d == 64 ? move_kernel<QT, 64> : d == 128 ? move_kernel<QT, 128> : move_kernel<QT, 256>;
}

EvictKernel choose_for(int cl) {
  return cl == 1 ? choose_kernel<1> : cl == 2 ? choose_kernel<2> : cl == 4 ? choose_kernel<4> : cl == 8 ? choose_kernel<8> : choose_kernel<16>;
}

}  // namespace

int kv_evict(const KvAttnParams& p, const KvEvict& e, int* err, cudaStream_t st) {
  const long long units = (long long)p.batch * p.c.heads, moves = (units * ((e.keep + 15) / 16) + 3) / 4;
  if (units > 0x7fffffffLL / 8 || moves > 0x7fffffffLL) return -2;
  // CTAs of a unit: 4096 tokens each or more, as far as there are SMs for them. Of clusters of 16, each in a GPC of its own, few run at
  // a time: they are taken for half of the SMs (8 heads of 65536 tokens: 18.2 us in clusters of 16, 12.7 of 8; 4 heads 14.6, 18.2).
  const long long tokens = (long long)p.max_pages * p.c.page_size;
  const int sms = num_sms();
  int cl = 1;
  while (cl < 16 && cl * 4096LL < tokens && units * cl * 2 <= (cl == 8 ? sms / 2 : sms)) cl *= 2;
  EvictKernel choose = choose_for(cl);
  if (cl == 16 && cluster_setup(choose, kMostKeys * 4, kThreads, cl) <= 0) choose = choose_for(cl = 8);
  if (cluster_setup(choose, kMostKeys * 4, kThreads, cl) <= 0) return -13;
  const long long share = cl > 1 ? (tokens + 32 * cl - 1) / (32 * cl) * 32 : tokens;
  const EvictArgs a{p, e, (int)std::min<long long>(share, kMostKeys)};
  int rc = launch_clusters(choose, (unsigned)units * cl, kThreads, (size_t)a.keys * 4, cl, st, a, err);
  if (rc || e.keep == 0) return rc;
  const EvictKernel k = p.c.type == QT_Q4_0 ? move_for<QT_Q4_0>(p.c.d)
                                            : p.c.type == QT_Q4_1 ? move_for<QT_Q4_1>(p.c.d) : move_for<QT_Q8_0>(p.c.d);
  return launch_dependent(k, dim3((unsigned)moves), 128, 0, st, a, err);
}

}  // namespace s3b
