// Layout of the quantised key / value cache, shared by the kernels that write, read and attend over it.
//
// The cache is a sequence of (page, head) regions; a region holds the keys of its tokens and then their values, both as a
// sequence of groups of 16 tokens, so that the keys (or values) of neighbouring tokens of a page are one piece of memory.
// A group of KvL<QT, D>::kHalf bytes holds its quantised values, then their scales, then for q4_1 their minima. The order
// of the values inside a group is that of the m16n8k16 fragments of the few-query attention kernel, so that lane (g, t) =
// (lane / 4, lane % 4) of a warp finds its share of the group as whole 8- or 16-byte words, contiguous over the lanes:
//   keys    A operand of S^T = K Q^T, rows = tokens: lane (g, t) takes tokens g and g + 8, and of every block of 32 the
//           8 consecutive values 8 t .. 8 t + 7 (the contraction may run in any order that Q shares).
//   values  A operand of O^T = V^T P^T, columns = tokens: lane (g, t) takes tokens 2t, 2t + 1, 2t + 8, 2t + 9, and of
//           every block of 32 the 4 values 4 g .. 4 g + 3 (the rows of O^T may stand in any order).
// Values come in super-blocks of 128 (4 bits) or 64 (8 bits, or D = 64), the widest that one 16-byte load per lane takes.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace s3b {

template <int QT, int D>
struct KvL {
  static constexpr int kBits = QT == QT_Q8_0 ? 8 : 4;
  static constexpr int kNB = D / 32;                                         // blocks of a row
  static constexpr int kSB = (kBits == 4 && D >= 128) ? 128 : 64;            // values of a super-block
  static constexpr int kNBS = kSB / 32;                                      // blocks of a super-block
  static constexpr int kSuper = 16 * kSB * kBits / 8;                        // bytes of a super-block of 16 tokens
  static constexpr int kVal = 16 * D * kBits / 8;                            // bytes of the keys (or values) of a group
  static constexpr int kPlanes = QT == QT_Q4_1 ? 2 : 1;                      // scale, minimum
  static constexpr int kSc = 16 * kNB * 2;                                   // bytes of one plane
  static constexpr int kHalf = kVal + kPlanes * kSc;                         // bytes of a group

  // byte offsets in a group of keys (k_) or of values (v_)
  // keys: values 8 t .. 8 t + 7 of block b of token tok (4 or 8 bytes)
  static __host__ __device__ constexpr int k_val(int tok, int b, int t) {
    return (b / kNBS) * kSuper + tok * (kSB * kBits / 8) + (t * kNBS + b % kNBS) * kBits;
  }
  // values: values 4 g .. 4 g + 3 of block b of token tok (2 or 4 bytes)
  static __host__ __device__ constexpr int v_val(int tok, int b, int g) {
    return (b / kNBS) * kSuper +
           ((((tok >> 3) * 32 + g * 4 + ((tok & 7) >> 1)) * 2 + (tok & 1)) * kNBS + b % kNBS) * (kBits / 2);
  }
  static __host__ __device__ constexpr int k_scale(int tok, int b) { return kVal + (tok * kNB + b) * 2; }
  // the four tokens of lane t (2t, 2t + 1, 2t + 8, 2t + 9) side by side
  static __host__ __device__ constexpr int v_scale(int tok, int b) {
    return kVal + ((((tok & 7) >> 1) * kNB + b) * 4 + (tok & 1) + 2 * (tok >> 3)) * 2;
  }
};

// Byte offset of the keys (kv = 0) or values (1) of the group of 16 tokens `group` of (page, head).
template <int QT, int D>
__device__ __forceinline__ long long kv_group_offset(const KvCache& c, long long page, int head, int kv, int group) {
  return (((page * c.heads + head) * 2 + kv) * (c.page_size >> 4) + group) * (long long)KvL<QT, D>::kHalf;
}

// The 8 nibbles of a key word: value 2p in nibble p, value 2p + 1 in nibble p + 4. The 4 nibbles of a value half-word
// stand in order. 8-bit codes are stored with 128 added, in order.

// ---------------------------------------------------------------- codes
__device__ __forceinline__ uint32_t h2_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u32_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// (w & MASK) | 0x64006400 in one instruction
template <uint32_t MASK>
__device__ __forceinline__ uint32_t under_1024(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(0x64006400u));
  return r;
}

// Exact f16 pairs of the codes (less 8 for q4_0) whose nibbles lie at bits 0, 4, 8, 12 of each half of w: a nibble under
// the exponent of 1024 reads 1024 + c at bit 0 and 1024 + 16 c at bit 4; one subtraction (or multiply-add by 1/16)
// leaves the integer.
template <int QT>
__device__ __forceinline__ void nibble_pairs(uint32_t w, uint32_t (&out)[4]) {
  const __half2 off0 = u32_h2(QT == QT_Q4_0 ? 0xE408E408u : 0xE400E400u);  // -1032, -1024
  const __half2 off1 = u32_h2(QT == QT_Q4_0 ? 0xD480D480u : 0xD400D400u);  // -72, -64
  const __half2 sixteenth = u32_h2(0x2C002C00u);
  const uint32_t x = w >> 8;
  out[0] = h2_u32(__hadd2(u32_h2(under_1024<0x000F000Fu>(w)), off0));
  out[1] = h2_u32(__hfma2(u32_h2(under_1024<0x00F000F0u>(w)), sixteenth, off1));
  out[2] = h2_u32(__hadd2(u32_h2(under_1024<0x000F000Fu>(x)), off0));
  out[3] = h2_u32(__hfma2(u32_h2(under_1024<0x00F000F0u>(x)), sixteenth, off1));
}
// The same for the bytes 0, 1 and 2, 3 of w (8-bit codes with 128 added).
__device__ __forceinline__ void byte_pairs(uint32_t w, uint32_t& a, uint32_t& b) {
  const __half2 off = u32_h2(0xE480E480u);  // -1152
  a = h2_u32(__hadd2(u32_h2(__byte_perm(w, 0x64646464u, 0x4140)), off));
  b = h2_u32(__hadd2(u32_h2(__byte_perm(w, 0x64646464u, 0x4342)), off));
}


// ---------------------------------------------------------------- launches
// A kernel that may take its place on the GPU while its predecessor in the stream still runs. Every thread that touches what
// the predecessor reads or writes calls wait_before first, and some thread of every block does, so that a kernel's end means
// that its predecessors have ended. What a predecessor may have written (cache, rows, slots, pages, lengths, queries) is read by
// ordinary loads: read-only ones (__ldg) promise memory that stays as it is from the kernel's beginning, which here lies
// before its predecessors' end, and the wait need not order them. In turn, against plain launches: a read of 28736 tokens of 256 7.2 us against 10.2,
// attention of one query over 577 tokens 8.7 against 11.3, of 4096 over 28736 (three kernels) 137 against 142.
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The successor may take its place now.
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename K, typename... A>
int launch_dependent(K* kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? 0 : -12;
}

}  // namespace s3b
