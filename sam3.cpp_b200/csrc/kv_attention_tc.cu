// Attention over the quantised key / value cache for many query rows: tcgen05 tiles of 128 query rows by 128 tokens.
//
// A unit is one key / value head, one sequence and one block of TQ x 128 query rows (queries x heads of the group side by
// side, so all of them share one pass over the cache). The line of 128-token tiles of all units is cut into equal shares,
// one for each CTA (one per SM): uneven lengths, causal diagonals and few long units all fill the GPU. A unit that
// several CTAs share leaves unnormalised parts in the workspace, which join_kernel adds up in the order of the shares.
//
// Roles. The f16 operands come from the cache in one of two ways (tc_plan): staged by stage_kernel as images of the 16 KB
// slots before this kernel runs, or made by warps of this kernel.
//   warps 0, 1     issue the MMAs of query tile 0 / 1 (the warp waits together, one elected lane issues): S = Q K^T into
//                  TMEM, then O += P V with P read from TMEM
//   warp 2         staged: copies slot images and Q into the ring, slot by slot. Else: copies the cache in block form (64
//                  tokens of keys or values an entry, as few copies as the pages allow) into a second ring
//   warp 3         allocates TMEM
//   softmax        one warpgroup per query tile, a thread per query row: running reference maximum (moved only when a row's
//                  maximum passes it by 2^8), p = 2^(s - m) written as f16 over the scores, sum in f32; at a unit's end
//                  O / sum to the output
//   dequantising   not staged: 8 warps (16 at D = 256) turn the block form into slots in the 128-byte swizzle, item by item
//                  (K or V of 128 tokens); they also load Q
// Every query tile has two S regions, so S of the next tokens runs beside the softmax of these: 64 tokens a region for D =
// 64 and 128 (two query tiles and their O fill TMEM), 128 for D = 256 (one tile: O takes half of TMEM).
//
// Rounded to f16: the operands of the two products (a value of the cache once, the weight once). Sums, maxima and O are f32.
//
// Measured, staged, one call at a time: 4096 rows over 28736 tokens, one head of 256: 120 us in all, of which this kernel 100
// (tensor pipe 69% of the cycles active; what is left is the chain S, softmax, P V of the only tile that fits). 4 x 2048
// causal queries over 3 to 8 thousand tokens, 16 heads on 4, d = 128: 344 us, 910 TFLOP/s (tensor pipe 53%, exponentials 53%
// of the MUFU's rate: the two take turns on shared memory and TMEM ports). d = 64: 618 TFLOP/s, where the exponentials are
// twice as many a FLOP. (Back to back, under the power cap, the first two take 125 and 379 us.)
//
// The f16 operand is code * scale (+ minimum) rounded once. The 16 tokens of a group stand in the order
// 0 1 8 9 2 3 10 11 4 5 12 13 6 7 14 15 (both in K's rows and V's columns; a softmax does not mind), which is the order
// in which a lane holds them, so V goes to shared memory transposed, [D values][64 tokens], in 8-byte pieces and is a
// K-major operand like K.
#include <algorithm>

#include "kv_tmem.cuh"

namespace s3b {

namespace {

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

constexpr int kTile = 128;          // query rows of a tile and tokens of a tile
constexpr int kSlotBytes = 16384;   // 128 x 64 f16
constexpr int kUnit = 64;           // tokens of an entry of the block-form ring
constexpr float kLazy = 8.f;        // log2 of the largest weight before the reference maximum moves

// STAGED: the operands come as f16 slot images (stage_kernel) instead of being dequantised by warps of the kernel.
template <int QT, int D, bool STAGED>
struct Tc {
  typedef KvL<QT, D> L;
  static constexpr int kTQ = D == 256 ? 1 : 2;
  static constexpr int kSub = D == 256 ? 128 : 64;          // tokens of an S region
  static constexpr int kSubs = kTile / kSub;
  // dequantising warps: teams of 8; with two teams, team p makes part p of every item (K: 128 of the 256 values of a row,
  // V: 64 of the 128 tokens), so a part is published on its own
  static constexpr int kTeams = D == 256 ? 2 : 1;
  static constexpr int kDeqWarp0 = 4 + 4 * kTQ;
  static constexpr int kDeqWarps = STAGED ? 0 : 8 * kTeams;
  static constexpr int kThreads = 32 * (kDeqWarp0 + kDeqWarps);
  static constexpr int kParts = D / 64;                     // slots of an item (K: 64-value chunks; V: D x 64 tokens)
  static constexpr int kTeamSlots = kParts / kTeams;        // slots that a warp's item publishes
  static constexpr int kNSB = D / L::kSB;                   // super-blocks of a row
  static constexpr int kTasks = kNSB / kTeams;              // super-blocks of 16 tokens that a warp makes of an item
  static constexpr int kQBytes = kTQ * kTile * D * 2;
  static constexpr int kSlots = STAGED ? (D == 64 ? 11 : D == 128 ? 9 : 8) : D == 256 ? 6 : 8;
  static constexpr int kUnitBytes = kUnit / 16 * L::kHalf;
  static constexpr int kRawFit = (224 * 1024 - 1024 - kQBytes - kSlots * kSlotBytes - 512) / kUnitBytes;
  static constexpr int kRaw = STAGED ? 0 : kRawFit > 8 ? 8 : kRawFit;  // entries of the block-form ring
  // An item takes two entries, tokens 0 .. 63 and 64 .. 127, and a warp reads one of them. In an odd ring it would meet a barrier
  // in every other phase only, and its wait, which knows the phases' parity alone, could pass while the load before the one it
  // waits for is still on its way. There each warp waits for both entries and gives both back. In an even ring the halves keep
  // their entries: a warp that always reads the same half meets every phase, and with two teams (K by tokens, V by team) the
  // slots of an item come free only when the item two before it has been read whole, which lies behind the entries' last use.
  static constexpr bool kBoth = kRaw & 1;
  static constexpr int kSmem = 1024 + kQBytes + kSlots * kSlotBytes + kRaw * kUnitBytes + 512;
  static_assert(STAGED || kRaw >= 3, "K of a tile takes two entries of tiles_kernel's ring, and one has to be on its way");
  static constexpr int kOCol = 256;                         // TMEM: two S regions of kSub columns a tile, then O
  // Registers a thread at launch (65536 / threads, whole eights) and after the warpgroups trade: the issuing one, softmax
  // (kTQ warpgroups), dequantising (2 kTeams). The sum over warpgroups stays within the launch's.
  static constexpr int kRegsLaunch = 65536 / kThreads / 8 * 8;
  static constexpr int kRegsIssue = 72;
  static constexpr int kRegsSoft = 120;
  static constexpr int kRegsDeq = D == 256 ? 72 : 80;
  static_assert(STAGED || kRegsIssue + kTQ * kRegsSoft + 2 * kTeams * kRegsDeq <= kThreads / 128 * kRegsLaunch,
                "register shares");
  static constexpr int kPart = kTQ * kTile * (D + 2);       // floats of a unit's part
};

// A unit that several CTAs share, written by the CTA in whose share it begins (its entry's index).
struct Shared {
  int valid, b, head, row0;
  int c1, second;  // last of its CTAs; whether its first CTA's part is that CTA's second
};

struct TcArgs {
  KvAttnParams p;
  float* part;     // [2 * grid][TQ][128 * D outputs, as [D / 4][128] float4; 128 maxima; 128 sums]
  Shared* shared;  // [grid]
  int blocks;      // row blocks of a sequence
  // staged operands: [sequence][head][tiles] of a K and a V item (D * 256 bytes each), and [sequence][head][blocks] of Q
  uint8_t* image;
  uint8_t* q_image;
  int tiles;       // token tiles that a page table can name
};

// Rows of a unit: packed row r = query * group + head of the group.
struct Unit {
  int b, head, row0;  // sequence, key / value head, first packed row
  int len, t0, tiles; // tokens, first 128-token tile, tiles
  int lo, hi;         // tokens that any row sees
};

template <int ROWS>
__device__ __forceinline__ int unit_tiles(const KvAttnParams& p, int group, int len, int block, int* lo, int* hi) {
  int none;
  row_span(p, len, block * ROWS / group, lo, &none);
  row_span(p, len, min(p.nq - 1, (block * ROWS + ROWS - 1) / group), &none, hi);
  return *hi > *lo ? (*hi + kTile - 1) / kTile - *lo / kTile : 0;
}

// The segments (unit, tiles [ca, cb) of it) of the share [pos, end) of the line, in order. Kept in shared memory, one for
// each warp, so that the roles' loops hold only what they use.
struct Walk {
  long long pos, end, start;  // start: position of the unit's first tile
  int head, pair;
  Unit u;
  int ca, cb, more;
};

// The next segment; false at the share's end. One thread.
template <int ROWS>
__device__ __forceinline__ bool walk_next(const KvAttnParams& p, int blocks, int* err, Walk* w) {
  const int group = p.heads / p.c.heads;
  w->more = 0;
  while (w->pos < w->end) {
    Unit u;
    u.b = w->pair / blocks;
    u.head = w->head;
    const int block = w->pair - u.b * blocks;
    u.row0 = block * ROWS;
    u.len = sequence_length(p, u.b, err);
    u.tiles = unit_tiles<ROWS>(p, group, u.len, block, &u.lo, &u.hi);
    u.t0 = u.lo / kTile;
    if (w->pos < w->start + u.tiles) {
      w->u = u;
      w->ca = (int)(w->pos - w->start);
      w->cb = (int)min((long long)u.tiles, w->end - w->start);
      w->pos += w->cb - w->ca;
      w->more = 1;
      break;
    }
    w->start += u.tiles;
    if (++w->pair == p.batch * blocks) {
      w->pair = 0;
      ++w->head;
    }
  }
  return w->more;
}
// The same for a whole warp.
template <int ROWS>
__device__ __forceinline__ bool walk_next_warp(const KvAttnParams& p, int blocks, int* err, Walk* w, int lane) {
  __syncwarp();
  if (lane == 0) walk_next<ROWS>(p, blocks, err, w);
  __syncwarp();
  return *const_cast<volatile int*>(&w->more) != 0;
}

// token of a group that stands at position p
__host__ __device__ constexpr int token_at(int p) { return 2 * (p >> 2) + (p & 1) + 8 * ((p >> 1) & 1); }

template <int WORDS>
__device__ __forceinline__ void lds(const uint8_t* at, uint32_t* r) {
  if (WORDS == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    r[0] = v.x;
    r[1] = v.y;
    r[2] = v.z;
    r[3] = v.w;
  } else if (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    r[0] = v.x;
    r[1] = v.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(at);
  }
}

template <int QT>
__device__ __forceinline__ uint32_t scaled(uint32_t code, uint32_t s, uint32_t m) {
  return QT == QT_Q4_1 ? h2_u32(__hfma2(u32_h2(code), u32_h2(s), u32_h2(m))) : h2_u32(__hmul2(u32_h2(code), u32_h2(s)));
}

// Keys of 16 tokens (at `half`, block form), super-block sb, into its slots at `item`: chunk n / 2, row =
// position in the tile, 16-byte column in the swizzle. Lane (g, t) takes tokens g and g + 8, quarter t of each block:
// reads and writes then meet no bank twice once the lanes of odd rows take the blocks of a pair in the other order. Rows
// of tokens outside the sequence may hold anything: their scores are masked.
template <int QT, int D>
__device__ __forceinline__ void emit_k(const uint8_t* half, uint8_t* item, int grp, int sb, int lane) {
  typedef KvL<QT, D> L;
  constexpr int PW = L::kNBS * L::kBits / 4, PB = PW / L::kNBS;  // words of a piece, of a block in it
  const int g = lane >> 2, t = lane & 3, odd = g & 1;
  const uint32_t sel[2] = {odd ? 0x3232u : 0x1010u, odd ? 0x1010u : 0x3232u};
  uint32_t w[2][PW], s[2][L::kNBS / 2], m[2][L::kNBS / 2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    lds<PW>(half + L::k_val(g + 8 * x, sb * L::kNBS, t), w[x]);
    lds<L::kNBS / 2>(half + L::k_scale(g + 8 * x, sb * L::kNBS), s[x]);
    if (QT == QT_Q4_1) lds<L::kNBS / 2>(half + L::kSc + L::k_scale(g + 8 * x, sb * L::kNBS), m[x]);
  }
  // position of token g: 4 (g / 2) + g % 2, of token g + 8: two further
  uint8_t* row = item + (grp * 16 + 4 * (g >> 1) + odd) * 128;
  const int col = (odd * 4 + t) ^ (4 * ((g >> 1) & 1) + odd);  // of the first block taken, for token g
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int n = 0; n < L::kNBS; ++n) {
      uint32_t v[4], u[PB];
#pragma unroll
      for (int e = 0; e < PB; ++e) u[e] = odd ? w[x][(n ^ 1) * PB + e] : w[x][n * PB + e];
      if (QT == QT_Q8_0) {
        byte_pairs(u[0], v[0], v[1]);
        byte_pairs(u[PB - 1], v[2], v[3]);
      } else {
        nibble_pairs<QT>(u[0], v);
      }
      const uint32_t sc = __byte_perm(s[x][n >> 1], 0, sel[n & 1]);
      const uint32_t mn = QT == QT_Q4_1 ? __byte_perm(m[x][n >> 1], 0, sel[n & 1]) : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = scaled<QT>(v[e], sc, mn);
      *reinterpret_cast<uint4*>(row + x * 256 + n / 2 * kSlotBytes + ((col ^ (4 * (n & 1)) ^ (2 * x)) * 16)) =
          make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

// Values of 16 tokens (at `half`), super-block sb, into the slots of their 64 tokens at `item`, row = value.
// Lane (g, t) holds tokens 2t, 2t + 1, 2t + 8, 2t + 9 (positions 4t .. 4t + 3), values 4g .. 4g + 3 of each block; lanes
// whose rows would meet another lane's banks (bit 1 of g) take the values in the order 2, 3, 0, 1. keep: masks of the
// token pairs that the sequence holds; the scales of others count as zero.
template <int QT, int D>
__device__ __forceinline__ void emit_v(const uint8_t* half, uint32_t keep0, uint32_t keep1, uint8_t* item, int grp, int sb,
                                       int lane) {
  typedef KvL<QT, D> L;
  constexpr int PW = L::kNBS * L::kBits / 4, TW = PW / 2;  // words of a piece (two tokens), of a token
  const int g = lane >> 2, t = lane & 3, f = (g >> 1) & 1;
  uint32_t w0[PW], w1[PW], s[2 * L::kNBS], m[2 * L::kNBS];
  lds<PW>(half + L::v_val(2 * t, sb * L::kNBS, g), w0);
  lds<PW>(half + L::v_val(2 * t + 8, sb * L::kNBS, g), w1);
#pragma unroll
  for (int n = 0; n < L::kNBS; n += 2) {
    lds<4>(half + L::v_scale(2 * t, sb * L::kNBS + n), s + 2 * n);
    if (QT == QT_Q4_1) lds<4>(half + L::kSc + L::v_scale(2 * t, sb * L::kNBS + n), m + 2 * n);
  }
  uint8_t* base = item + (sb * L::kSB + 4 * g) * 128 + (t & 1) * 8;
  const int at0 = (f << 8) | ((((t >> 1) ^ ((g & 1) * 4) ^ (2 * f)) * 16) ^ ((grp & 3) * 32));
#pragma unroll
  for (int n = 0; n < L::kNBS; ++n) {
    uint32_t v0[4], v1[4];
    if (QT == QT_Q8_0) {
      const int lo = f ? 0x7362 : 0x5140, hi = f ? 0x5140 : 0x7362;
      byte_pairs(__byte_perm(w0[n], w0[TW + n], lo), v0[0], v0[1]);
      byte_pairs(__byte_perm(w0[n], w0[TW + n], hi), v0[2], v0[3]);
      byte_pairs(__byte_perm(w1[n], w1[TW + n], lo), v1[0], v1[1]);
      byte_pairs(__byte_perm(w1[n], w1[TW + n], hi), v1[2], v1[3]);
    } else {
      const int sel = n & 1 ? (f ? 0x6723 : 0x7632) : (f ? 0x4501 : 0x5410);
      nibble_pairs<QT>(__byte_perm(w0[n / 2], w0[TW + n / 2], sel), v0);
      nibble_pairs<QT>(__byte_perm(w1[n / 2], w1[TW + n / 2], sel), v1);
    }
    const uint32_t s0 = s[2 * n] & keep0, s1 = s[2 * n + 1] & keep1;
    const uint32_t m0 = QT == QT_Q4_1 ? m[2 * n] & keep0 : 0u, m1 = QT == QT_Q4_1 ? m[2 * n + 1] & keep1 : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<uint2*>(base + n * (32 * 128) + (at0 ^ (e * 144))) =
          make_uint2(scaled<QT>(v0[e], s0, m0), scaled<QT>(v1[e], s1, m1));
  }
}

template <bool MASKED>
__device__ __forceinline__ void mask_scores(uint32_t (&r)[32], int c0, int lo, int hi) {
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const int tok = c0 + (c & 16) + token_at(c & 15);
    if (MASKED && (tok < lo || tok >= hi)) r[c] = __float_as_uint(-INFINITY);
  }
}
__device__ __forceinline__ void max_scores(const uint32_t (&r)[32], float (&mx)[4]) {
#pragma unroll
  for (int c = 0; c < 32; c += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(r[c + 2 * k]), __uint_as_float(r[c + 2 * k + 1]));
}
// weights of 32 scores to the 16 columns at `at`; acc: the sums of even and odd pairs
__device__ __forceinline__ void weigh_scores(const uint32_t (&r)[32], uint32_t at, unsigned long long sl2x2,
                                             unsigned long long negm2, unsigned long long& acc0, unsigned long long& acc1) {
  uint32_t pk[16];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    float pv[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int c = 8 * u + e;
      float x0, x1;
      f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), sl2x2, negm2), x0, x1);
      // a hidden token's -inf gives 0 exactly, so a row that sees nothing keeps the sum 0; a share of the exponentials on
      // the FMA pipe gained nothing (d = 64) or cost 5% (d = 128, 2 of 8)
      pv[e] = ex2_approx(x0);
      pv[e + 1] = ex2_approx(x1);
    }
    acc0 = f2_add(acc0, f2_add(f2_pack(pv[0], pv[1]), f2_pack(pv[4], pv[5])));
    acc1 = f2_add(acc1, f2_add(f2_pack(pv[2], pv[3]), f2_pack(pv[6], pv[7])));
#pragma unroll
    for (int e = 0; e < 4; ++e) pk[4 * u + e] = h2_u32(__floats2half2_rn(pv[2 * e], pv[2 * e + 1]));
  }
  KV_TMEM_ST8(at, pk);
  KV_TMEM_ST8(at + 8, pk + 8);
}

// One S region (N tokens) of one query row: the row's scores from TMEM at `at`, the lazy reference maximum, the weights as
// f16 pairs over the first half of the region, the sum into l. MASKED: only tokens [lo, hi) of the region count. Returns
// true when a maximum of the warp moved and the rows of O have to be scaled by alpha. any_large: whether the warp has a row
// with a large reference. 64 scores stay in registers; 128 are read twice,
// 32 at a time with 32 more on their way, in loops that stay rolled (unrolled, the loop's code was fetched again and again).
__device__ __forceinline__ bool is_large(float m_ref) { return fabsf(m_ref) > 0x1p20f && m_ref > kNoScore; }
template <int N, bool MASKED>
__device__ __forceinline__ bool softmax_tile(uint32_t at, int lo, int hi, float sl2, float& m_ref, float& l, float& alpha,
                                             bool& any_large) {
  uint32_t ra[32], rb[32];
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  KV_TMEM_LD32(at, ra);
  if (N == 64) {
    KV_TMEM_LD32(at + 32, rb);
    tc_wait_ld();
    mask_scores<MASKED>(ra, 0, lo, hi);
    mask_scores<MASKED>(rb, 32, lo, hi);
    max_scores(ra, mx);
    max_scores(rb, mx);
  } else {
    tc_wait_ld();
#pragma unroll 1
    for (int c0 = 0; c0 < N; c0 += 64) {
      KV_TMEM_LD32(at + c0 + 32, rb);
      mask_scores<MASKED>(ra, c0, lo, hi);
      max_scores(ra, mx);
      tc_wait_ld();
      KV_TMEM_LD32(at + ((c0 + 64) & (N - 1)), ra);  // at the end the first ones again
      mask_scores<MASKED>(rb, c0 + 32, lo, hi);
      max_scores(rb, mx);
      tc_wait_ld();
    }
  }
  const float top = max3(mx[0], mx[1], fmaxf(mx[2], mx[3])) * sl2;
  alpha = 1.f;
  const bool moved = __any_sync(~0u, top > m_ref + kLazy);
  if (moved) {
    if (top > m_ref + kLazy) {
      alpha = ex2_approx(m_ref - top);
      m_ref = top;
      l *= alpha;
    }
    any_large = __any_sync(~0u, is_large(m_ref));
  }
  const unsigned long long sl2x2 = f2_pack(sl2, sl2), negm2 = f2_pack(-m_ref, -m_ref);
  unsigned long long acc0 = f2_pack(0.f, 0.f), acc1 = acc0;
  // A weight's exponent is score * sl2 - m_ref in one rounding, m_ref the rounded product of another score. The difference that
  // m_ref's rounding makes is common to a row and cancels, but for scores past 2^31 it leaves the exponent's range: rows of
  // large scores take the rounded product of each score first.
  if (any_large) {
    const float first = is_large(m_ref) ? sl2 : 1.f, then = is_large(m_ref) ? 1.f : sl2;
#pragma unroll 1
    for (int c0 = 0; c0 < N; c0 += 32) {
      KV_TMEM_LD32(at + c0, ra);
      tc_wait_ld();
      mask_scores<MASKED>(ra, c0, lo, hi);
#pragma unroll
      for (int c = 0; c < 32; ++c) ra[c] = __float_as_uint(__fmul_rn(__uint_as_float(ra[c]), first));
      weigh_scores(ra, at + c0 / 2, f2_pack(then, then), negm2, acc0, acc1);
    }
  } else if (N == 64) {
    weigh_scores(ra, at, sl2x2, negm2, acc0, acc1);
    weigh_scores(rb, at + 16, sl2x2, negm2, acc0, acc1);
  } else {
#pragma unroll 1
    for (int c0 = 0; c0 < N; c0 += 64) {
      // the weights of 32 scores go over columns whose scores have been read
      KV_TMEM_LD32(at + c0 + 32, rb);
      mask_scores<MASKED>(ra, c0, lo, hi);
      weigh_scores(ra, at + c0 / 2, sl2x2, negm2, acc0, acc1);
      tc_wait_ld();
      KV_TMEM_LD32(at + ((c0 + 64) & (N - 1)), ra);  // unused at the end
      mask_scores<MASKED>(rb, c0 + 32, lo, hi);
      weigh_scores(rb, at + c0 / 2 + 16, sl2x2, negm2, acc0, acc1);
      tc_wait_ld();
    }
  }
  float a0, a1, b0, b1;
  f2_unpack(acc0, a0, a1);
  f2_unpack(acc1, b0, b1);
  l += (a0 + a1) + (b0 + b1);
  return moved;
}

template <int QT, int D, bool STAGED>
__global__ void __launch_bounds__(Tc<QT, D, STAGED>::kThreads, 1) tiles_kernel(const __grid_constant__ TcArgs a, int* err) {
  typedef KvL<QT, D> L;
  typedef Tc<QT, D, STAGED> C;
  constexpr int TQ = C::kTQ, ROWS = TQ * kTile, kSlots = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;                       // [TQ][D / 64 chunks][128 rows][64]
  uint8_t* s_ring = s_q + C::kQBytes;        // [kSlots] x 16 KB
  uint8_t* s_raw = s_ring + kSlots * kSlotBytes;  // [kRaw] keys or values of 64 tokens in block form
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_raw + C::kRaw * C::kUnitBytes);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* full = bars + 2;                 // [kSlots]
  uint64_t* empty = full + kSlots;           // [kSlots]
  uint64_t* s_full = empty + kSlots;         // [2 tiles][2 regions]
  uint64_t* p_full = s_full + 4;             // [2 tiles][2 regions]: the softmax of the next region may be done before the
                                             // issuer looks at this one
  uint64_t* pv_done = p_full + 4;            // [2 tiles]
  uint64_t* o_full = pv_done + 2;            // [2 tiles]
  uint64_t* mma_done = o_full + 2;           // [2 tiles]
  uint64_t* raw_full = mma_done + 2;         // [kRaw]
  uint64_t* raw_empty = raw_full + C::kRaw;  // [kRaw]
  static_assert((2 + 2 * kSlots + 14 + 2 * C::kRaw) * 8 <= 512, "barriers of tiles_kernel");
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort_word, s_pair;
  __shared__ long long s_sum[24], s_start;
  __shared__ Walk s_walk[24];
  volatile int* s_abort = &s_abort_word;

  const KvAttnParams& p = a.p;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // uniform for the compiler
  const int group = p.heads / p.c.heads;
  const int n_rows = p.nq * group;
  const int pairs = p.batch * a.blocks;

  if (threadIdx.x == 0) {
    mbar_init(q_full, STAGED ? 1 : C::kDeqWarps);
    mbar_init(q_empty, TQ);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full[s], STAGED ? 1 : 8);  // the copy, or the warps of a team
      mbar_init(&empty[s], TQ);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[2 * x], 1);
      mbar_init(&s_full[2 * x + 1], 1);
      mbar_init(&p_full[2 * x], 4);
      mbar_init(&p_full[2 * x + 1], 4);
      mbar_init(&pv_done[x], 1);
      mbar_init(&o_full[x], 1);
      mbar_init(&mma_done[x], 1);
    }
    for (int x = 0; x < C::kRaw; ++x) {
      mbar_init(&raw_full[x], 1);
      mbar_init(&raw_empty[x], C::kBoth ? C::kDeqWarps : C::kDeqWarps / 2);
    }
    s_abort_word = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 3) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }

  // staged: the predecessor is stage_kernel, which lets this kernel in after its own wait; only the copies wait for its end
  if (!STAGED) wait_before();

  // ---- tiles of one head, by the warps' shares of the (sequence, row block) pairs; then the pair in which the share begins
  constexpr int kWarps = C::kThreads / 32;
  const int per_warp = (pairs + kWarps - 1) / kWarps;
  auto pair_tiles = [&](int k) -> int {
    if (k >= pairs) return 0;
    const int b = k / a.blocks;
    int lo, hi;
    return unit_tiles<ROWS>(p, group, sequence_length(p, b, err), k - b * a.blocks, &lo, &hi);
  };
  {
    long long sum = 0;
    for (int k = warp * per_warp + lane; k < min(pairs, (warp + 1) * per_warp); k += 32) sum += pair_tiles(k);
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
    if (lane == 0) s_sum[warp] = sum;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  long long per_head = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) per_head += s_sum[w];
  const long long total = per_head * p.c.heads;
  const long long ctas = min((long long)gridDim.x, total);
  const bool works = (int)blockIdx.x < ctas;
  const long long p0 = works ? total * blockIdx.x / ctas : 0, p1 = works ? total * (blockIdx.x + 1) / ctas : 0;
  if (works) {
    const int head = (int)(p0 / per_head);
    const long long rem = p0 - head * per_head;
    long long before = 0;
    int w = 0;
    while (w < kWarps - 1 && before + s_sum[w] <= rem) before += s_sum[w++];
    if (warp == w) {
      for (int k0 = w * per_warp;; k0 += 32) {
        const long long n = k0 + lane < min(pairs, (w + 1) * per_warp) ? pair_tiles(k0 + lane) : 0;
        long long end = n;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const long long up = __shfl_up_sync(~0u, end, x);
          if (lane >= x) end += up;
        }
        const uint32_t past = __ballot_sync(~0u, before + end > rem);
        if (past || k0 + 32 >= (w + 1) * per_warp) {
          const int who = past ? __ffs(past) - 1 : 0;
          const long long skipped = __shfl_sync(~0u, end - n, who);
          if (lane == 0) {
            s_pair = k0 + who;
            s_start = head * per_head + before + skipped;
          }
          break;
        }
        before += __shfl_sync(~0u, end, 31);
      }
    }
  }
  __syncthreads();
  // row blocks that see no token
  for (int k = blockIdx.x; k < pairs; k += gridDim.x) {
    if (pair_tiles(k)) continue;
    const int b = k / a.blocks, row0 = (k - b * a.blocks) * ROWS;
    for (int h = 0; h < p.c.heads; ++h)
      for (int e = threadIdx.x; e < min(ROWS, n_rows - row0) * (D / 4); e += C::kThreads) {
        const int r = row0 + e / (D / 4), i = r / group, hq = h * group + r % group;
        store_out(p, b * p.o_b + i * p.o_n + hq * p.o_h + e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
        if (p.lse && e % (D / 4) == 0) p.lse[((long long)b * p.nq + i) * p.heads + hq] = -INFINITY;
      }
  }
  Walk& w = s_walk[warp];
  if (lane == 0) {
    w.pos = p0;
    w.end = p1;
    w.start = s_start;
    w.head = works ? (int)(p0 / per_head) : 0;
    w.pair = s_pair;
  }
  __syncwarp();
  const float sl2 = p.scale * kLog2e;
  // Item x of a segment of n tiles: K or V of tile *j, in the order in which the MMAs first take them. Tiles of two S
  // regions: K_0 V_0 K_1 V_1 ...; of one: K_0 K_1 V_0 K_2 V_1 ... V_last.
  auto order = [](int x, int n, int* j) -> bool {
    if (C::kSubs == 2 || x == 0) {
      *j = x >> 1;
      return !(x & 1);
    }
    const bool k = (x & 1) && x != 2 * n - 1;
    *j = x == 2 * n - 1 ? n - 1 : k ? (x + 1) >> 1 : (x >> 1) - 1;
    return k;
  };
  // and the place of K_j and V_j in it
  auto k_item = [](int j) -> int { return C::kSubs == 2 ? 2 * j : j ? 2 * j - 1 : 0; };
  auto v_item = [](int j, int n) -> int { return C::kSubs == 2 ? 2 * j + 1 : j == n - 1 ? 2 * n - 1 : 2 * j + 2; };

  if (warp < 4) {
    if (!STAGED) regs_dec<C::kRegsIssue>();
    if (warp == 2 && STAGED) {
      // ---- copies of the staged operands, slot by slot
      if (lane == 0) {
        // stage_kernel has written them. Every CTA waits, also one without work: no call may end before its stage_kernel.
        wait_before();
        uint32_t slot = 0, q_n = 0;
        bool ok = true;
        while (ok && walk_next<ROWS>(p, a.blocks, err, &w)) {
          const long long unit = (long long)w.u.b * p.c.heads + w.u.head;
          const int q_tiles = w.u.row0 + kTile < n_rows ? TQ : 1;
          if (!mbar_wait(q_empty, (q_n & 1) ^ 1, s_abort, err, kErrWaitEmpty)) break;
          mbar_arrive_expect_tx(q_full, q_tiles * kTile * D * 2);
          bulk_load(s_q, a.q_image + (unit * a.blocks + w.u.row0 / ROWS) * (ROWS * D * 2), q_tiles * kTile * D * 2, q_full);
          ++q_n;
          const uint8_t* tiles = a.image + (unit * a.tiles + w.u.t0 + w.ca) * (D * 512);
          const int n = w.cb - w.ca;
          for (int x = 0; x < 2 * n && ok; ++x) {
            int j;
            const bool is_k = order(x, n, &j);
            const uint8_t* from = tiles + (long long)j * (D * 512) + (is_k ? 0 : D * 256);
            for (int c = 0; c < C::kParts; ++c, ++slot) {
              const uint32_t s = slot % kSlots;
              if (!mbar_wait(&empty[s], ((slot / kSlots) & 1) ^ 1, s_abort, err, kErrWaitEmpty)) { ok = false; break; }
              mbar_arrive_expect_tx(&full[s], kSlotBytes);
              bulk_load(s_ring + s * kSlotBytes, from + c * kSlotBytes, kSlotBytes, &full[s]);
            }
          }
        }
        // no copy may still be landing when the CTA exits
        auto drain = [&](uint64_t* bar, uint32_t parity) {
          const unsigned long long t0 = globaltimer_ns();
          while (!mbar_try_wait(bar, parity)) {
            if (globaltimer_ns() - t0 > kWaitNs) {
              atomicCAS(err, 0, kErrWaitDrain);
              break;
            }
          }
        };
        if (q_n) drain(q_full, (q_n - 1) & 1);
        for (uint32_t x = slot > kSlots ? slot - kSlots : 0; x < slot; ++x) drain(&full[x % kSlots], (x / kSlots) & 1);
      }
    } else if (warp == 2) {
      // ---- copies of the cache in block form: two ring entries per item, as few copies as the pages allow
      const int per_page = p.c.page_size >> 4;
      constexpr int kRaw = C::kRaw > 0 ? C::kRaw : 1;
      int entry = 0;
      uint32_t phase = 0, armed = 0, armed_phase = 0;
      bool ok = true;
      while (ok && walk_next_warp<ROWS>(p, a.blocks, err, &w, lane)) {
        const int* table = p.pages + w.u.b * p.pages_stride;
        const int t0 = w.u.t0, ca = w.ca, cb = w.cb, head = w.u.head, g_lo = w.u.lo >> 4, g_hi = (w.u.hi + 15) >> 4;
        // lane k < 8: where the keys of group k of tile j are, -1 outside the groups that the unit sees. A copy begins at a
        // group that does not follow its predecessor in memory, and takes those that follow it.
        auto locate = [&](int j) -> long long {
          const int gi = (t0 + j) * 8 + (lane & 7);
          if (j >= cb || gi < g_lo || gi >= g_hi) return -1;
          long long page = table[gi / per_page];
          if (page < 0 || page >= p.c.n_pages) {
            atomicCAS(err, 0, kDevErrIndex);
            page = 0;
          }
          return kv_group_offset<QT, D>(p.c, page, head, 0, gi % per_page);
        };
        const long long v_offset = (long long)per_page * L::kHalf;
        long long at0 = locate(ca), at1 = locate(ca + 1);  // of tiles j, j + 1
        const int n = cb - ca;
        int first = 0;
        for (int x = 0; x < 2 * n && ok; ++x) {
          int j;
          const bool is_k = order(x, n, &j);
          const long long mine = j == first ? at0 : at1;
          const long long before = __shfl_up_sync(~0u, mine, 1);
          const int grp = lane & 7;
          // runs end at an entry's end too
          const bool starts = lane < 8 && mine >= 0 && ((grp & 3) == 0 || before != mine - L::kHalf);
          const uint32_t heads = __ballot_sync(~0u, starts), live = __ballot_sync(~0u, lane < 8 && mine >= 0);
          for (int half = 0; half < 2; ++half) {
            if (lane == 0) {
              ok = mbar_wait(&raw_empty[entry], phase ^ 1, s_abort, err, kErrWaitEmpty);
              const int groups = __popc(live >> (4 * half) & 15);
              if (ok && groups) {
                mbar_arrive_expect_tx(&raw_full[entry], groups * L::kHalf);
                armed |= 1u << entry;
                armed_phase = (armed_phase & ~(1u << entry)) | (phase << entry);
              } else if (ok) {
                mbar_arrive(&raw_full[entry]);
                armed &= ~(1u << entry);
              }
            }
            ok = __shfl_sync(~0u, (int)ok, 0);
            if (!ok) break;
            if (starts && grp >> 2 == half) {
              // groups up to the next start, the next hole or the entry's end
              const uint32_t stop = (heads | ~live | 0xFFFFFFF0u << (4 * half)) >> (grp + 1);
              bulk_load(s_raw + entry * C::kUnitBytes + (grp & 3) * L::kHalf, p.c.data + mine + (is_k ? 0 : v_offset),
                        __ffs(stop) * L::kHalf, &raw_full[entry]);
            }
            __syncwarp();
            if (++entry == kRaw) {
              entry = 0;
              phase ^= 1;
            }
          }
          if (!is_k) {  // the last use of tile j's addresses
            ++first;
            at0 = at1;
            at1 = locate(ca + first + 1);
          }
        }
      }
      // no copy may still be landing when the CTA exits
      if (lane == 0)
        for (int x = 0; x < C::kRaw; ++x)
          if (armed >> x & 1) {
            const unsigned long long t0 = globaltimer_ns();
            while (!mbar_try_wait(&raw_full[x], armed_phase >> x & 1)) {
              if (globaltimer_ns() - t0 > kWaitNs) {
                atomicCAS(err, 0, kErrWaitDrain);
                break;
              }
            }
          }
    } else if (warp < TQ) {
      // ---- MMA issue for query tile `warp`: the warp waits together, one lane issues
      const int t = warp;
      constexpr uint32_t idesc_s = idesc_f16(kTile, C::kSub, 0), idesc_o = idesc_f16(kTile, D, 0);
      const uint32_t q_base = smem_u32(s_q) + t * (kTile * D * 2), ring = smem_u32(s_ring);
      const uint32_t o_tmem = tmem + C::kOCol + t * D;
      uint32_t slot0 = 0, q_n = 0, ns = 0, npv = 0;  // slots before the segment; Q loads, S and P V products so far
      bool ok = true, issued = false;
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
        if (!__all_sync(~0u, mbar_wait(bar, parity, s_abort, err, code))) return false;
        tc_fence_after();
        return true;
      };
      auto wait_slot = [&](uint32_t s) -> bool { return wait(&full[s % kSlots], (s / kSlots) & 1, kErrWaitFull); };
      auto s_region = [&](uint32_t n) -> uint32_t { return tmem + (2 * t + (n & 1)) * C::kSub; };
      // S of sub-tile u of the segment: kSub tokens of tile u / kSubs
      auto issue_s = [&](int u, bool last) -> bool {
        const int j = u / C::kSubs, sub = u % C::kSubs;
        const uint32_t s0 = slot0 + k_item(j) * C::kParts;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          if (sub == 0 && !wait_slot(s0 + c)) return false;
          const uint64_t dq = sdesc_k_sw128(q_base + c * kSlotBytes);
          const uint64_t dk = sdesc_k_sw128(ring + (s0 + c) % kSlots * kSlotBytes + sub * (kSlotBytes / 2));
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) tc_mma_f16(s_region(ns), dq + kk * 2, dk + kk * 2, idesc_s, c != 0 || kk != 0);
            if (sub == C::kSubs - 1) tc_commit(&empty[(s0 + c) % kSlots]);
            if (c == D / 64 - 1) {
              tc_commit(&s_full[2 * t + (ns & 1)]);
              if (last) tc_commit(q_empty);
            }
          }
        }
        ++ns;
        issued = true;
        return true;
      };
      // O += P V of sub-tile u, by 64 tokens of V
      auto issue_pv = [&](int u, int n) -> bool {
        const int j = u / C::kSubs, sub = u % C::kSubs;
        if (!wait(&p_full[2 * t + (npv & 1)], (npv >> 1) & 1, kErrWaitMisc)) return false;
#pragma unroll
        for (int x = 0; x < C::kSub / 64; ++x) {
          const int half = C::kSubs == 2 ? sub : x;
          const uint32_t s0 = slot0 + v_item(j, n) * C::kParts + (D == 64 ? 0 : half * (D / 128));
          // every slot of the product: staged ones land one by one
          if (D > 64 || half == 0) {
#pragma unroll
            for (int y = 0; y < (D > 64 ? D / 128 : 1); ++y)
              if (!wait_slot(s0 + y)) return false;
          }
          const uint64_t dv = sdesc_k_sw128(ring + s0 % kSlots * kSlotBytes + (D == 64 ? half * (D * 128) : 0));
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_f16_ts(o_tmem, s_region(npv) + x * 32 + kk * 8, dv + kk * 2, idesc_o, u != 0 || x != 0 || kk != 0);
            if (D > 64 || half == 1) {
#pragma unroll
              for (int y = 0; y < (D > 64 ? D / 128 : 1); ++y) tc_commit(&empty[(s0 + y) % kSlots]);
            }
            if (x == C::kSub / 64 - 1) {
              tc_commit(&pv_done[t]);
              if (u == n * C::kSubs - 1) tc_commit(&o_full[t]);
            }
          }
        }
        ++npv;
        return true;
      };
      while (ok && walk_next_warp<ROWS>(p, a.blocks, err, &w, lane)) {
        const int n = w.cb - w.ca, subs = n * C::kSubs;
        if (!wait(q_full, q_n & 1, kErrWaitFull)) break;
        ++q_n;
        if (w.u.row0 + t * kTile >= n_rows) {
          // no second tile: release the slots as they fill, so that the counts of both issuers stay in step
          if (lane == 0) mbar_arrive(q_empty);
          for (int x = 0; x < n * 2 * C::kParts && ok; ++x) {
            ok = wait_slot(slot0 + x);
            if (ok && lane == 0) mbar_arrive(&empty[(slot0 + x) % kSlots]);
          }
        } else {
          // S of the next sub-tile runs beside the softmax of this one
          ok = issue_s(0, subs == 1);
          for (int u = 0; u < subs && ok; ++u) {
            if (u + 1 < subs) ok = issue_s(u + 1, u + 2 == subs);
            ok = ok && issue_pv(u, n);
          }
        }
        slot0 += n * 2 * C::kParts;
      }
      if (issued && elect_one()) {
        tc_commit(&mma_done[t]);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(&mma_done[t], 0)) {
          if (globaltimer_ns() - t0 > kWaitNs) {
            atomicCAS(err, 0, kErrWaitDrain);
            break;
          }
        }
      }
    }
  } else if (warp < 4 + 4 * TQ) {
    // ---- softmax and output of query tile t, one row per thread
    if (!STAGED) regs_inc<C::kRegsSoft>();
    const int t = (warp - 4) >> 2, w4 = warp & 3, row = w4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(w4 * 32) << 16;
    const uint32_t o_at = tmem + lane_off + C::kOCol + t * D;
    uint32_t n = 0, segs = 0;  // S regions and segments of this query tile so far
    bool ok = true;
    if (t == 0 && row == 0) a.shared[blockIdx.x].valid = 0;
    while (ok && walk_next_warp<ROWS>(p, a.blocks, err, &w, lane)) {
      const int r0 = w.u.row0 + t * kTile;
      if (r0 >= n_rows) continue;
      int lo, hi, all_lo, all_hi, none;
      row_span(p, w.u.len, min(r0 + row, n_rows - 1) / group, &lo, &hi);
      row_span(p, w.u.len, r0 / group, &none, &all_hi);
      row_span(p, w.u.len, min(n_rows - 1, r0 + kTile - 1) / group, &all_lo, &none);
      const int tok_first = (w.u.t0 + w.ca) * kTile, tok_end = (w.u.t0 + w.cb) * kTile;
      float m_ref = kNoScore, l = 0.f;
      bool any_large = false;
      for (int tok0 = tok_first; tok0 < tok_end; tok0 += C::kSub, ++n) {
        if (!mbar_wait(&s_full[2 * t + (n & 1)], (n >> 1) & 1, s_abort, err, kErrWaitTmemFull)) ok = false;
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_at = tmem + lane_off + (2 * t + (n & 1)) * C::kSub;
        float alpha;
        const bool moved =
            tok0 >= all_lo && tok0 + C::kSub <= all_hi
                ? softmax_tile<C::kSub, false>(s_at, 0, 0, sl2, m_ref, l, alpha, any_large)
                : softmax_tile<C::kSub, true>(s_at, lo - tok0, hi - tok0, sl2, m_ref, l, alpha, any_large);
        if (tok0 > tok_first && moved) {
          // O is current once the previous P V product of this tile has completed. The one before it has: S of this
          // region was issued after it, so the barrier cannot be a phase behind.
          if (!mbar_wait(&pv_done[t], (n - 1) & 1, s_abort, err, kErrWaitMisc)) ok = false;
          ok = __all_sync(~0u, ok);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            KV_TMEM_LD32(o_at + c, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            KV_TMEM_ST32(o_at + c, o);
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + (n & 1)]);
      }
      if (!ok) break;
      if (!mbar_wait(&o_full[t], segs & 1, s_abort, err, kErrWaitMisc)) ok = false;
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      ++segs;
      tc_fence_after();
      const int r = r0 + row, i = min(r, n_rows - 1) / group, h = w.u.head * group + r % group;
      const bool real = r < n_rows;
      const long long o_row = w.u.b * p.o_b + i * p.o_n + h * p.o_h;
      auto finish = [&](int c, const float* v, float inv) {  // 16 values of the row from column c
        if (!real) return;
        if (p.out_f32) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + o_row + c + e) =
                make_float4(v[e] * inv, v[e + 1] * inv, v[e + 2] * inv, v[e + 3] * inv);
        } else {
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            uint4 x;
            x.x = h2_u32(__floats2half2_rn(v[e] * inv, v[e + 1] * inv));
            x.y = h2_u32(__floats2half2_rn(v[e + 2] * inv, v[e + 3] * inv));
            x.z = h2_u32(__floats2half2_rn(v[e + 4] * inv, v[e + 5] * inv));
            x.w = h2_u32(__floats2half2_rn(v[e + 6] * inv, v[e + 7] * inv));
            *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(p.out) + o_row + c + e) = x;
          }
        }
      };
      auto finish_lse = [&](float top, float sum) {
        if (real && p.lse)
          p.lse[((long long)w.u.b * p.nq + i) * p.heads + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
      };
      if (w.ca == 0 && w.cb == w.u.tiles) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          KV_TMEM_LD32(o_at + c, o);
          tc_wait_ld();
          finish(c, reinterpret_cast<float*>(o), inv);
          finish(c + 16, reinterpret_cast<float*>(o) + 16, inv);
          __syncwarp();  // lanes of rows past the end come along
        }
        finish_lse(m_ref, l);
        continue;
      }
      // part of a unit that CTAs c0 .. c1 share: outputs as [D / 4][128 rows] float4, maxima, sums
      float* mine = a.part + (2 * (long long)blockIdx.x + (w.start > p0 ? 1 : 0)) * C::kPart + t * (kTile * (D + 2));
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        KV_TMEM_LD32(o_at + c, o);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          __stcg(reinterpret_cast<float4*>(mine) + (c + e) / 4 * kTile + row,
                 make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                             __uint_as_float(o[e + 3])));
      }
      __stcg(mine + kTile * D + row, m_ref);
      __stcg(mine + kTile * (D + 1) + row, l);
      if (w.ca == 0 && t == 0 && row == 0) {
        Shared* e = a.shared + blockIdx.x;
        e->valid = 1;
        e->b = w.u.b;
        e->head = w.u.head;
        e->row0 = w.u.row0;
        e->c1 = (int)(((w.start + w.u.tiles) * ctas - 1) / total);
        e->second = w.start > p0;
      }
    }
  } else if (!STAGED) {
    // ---- dequantising warps
    regs_dec<C::kRegsDeq>();
    const int dw = warp - C::kDeqWarp0, team = dw >> 3, tw = dw & 7;
    uint32_t slot = team * C::kTeamSlots, q_n = 0;
    int raw0 = 0;            // block-form ring entry of the item's tokens 0 .. 63; 64 .. 127 follow
    uint32_t raw_phase = 0;  // its phase
    bool ok = true;
    while (ok && walk_next_warp<ROWS>(p, a.blocks, err, &w, lane)) {
      // Q rows into the swizzled chunks
      ok = __all_sync(~0u, mbar_wait(q_empty, (q_n & 1) ^ 1, s_abort, err, kErrWaitEmpty));
      if (!ok) break;
      ++q_n;
      for (int e = dw * 32 + lane; e < ROWS * (D / 8); e += 32 * (C::kDeqWarps + STAGED)) {
        const int rr = e / (D / 8), c16 = e % (D / 8), r = w.u.row0 + rr;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < n_rows) {
          const int i = r / group, h = w.u.head * group + r % group;
          v = *reinterpret_cast<const uint4*>(p.q + w.u.b * p.q_b + i * p.q_n + h * p.q_h + c16 * 8);
        }
        *reinterpret_cast<uint4*>(s_q + rr / kTile * (kTile * D * 2) + c16 / 8 * kSlotBytes + rr % kTile * 128 +
                                  ((c16 & 7) ^ (rr & 7)) * 16) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      const int n = w.cb - w.ca, tok_first = (w.u.t0 + w.ca) * kTile, lo = w.u.lo, hi = w.u.hi;
#pragma unroll 1
      for (int x = 0; x < 2 * n; ++x) {
        int j;
        const bool is_k = order(x, n, &j);
        // this warp's 16 tokens of the tile and its super-blocks of them
        const int grp = C::kTeams == 1 || is_k ? tw : 4 * team + (tw & 3);
        const int sb0 = C::kTeams == 1 ? 0 : (is_k ? team : tw >> 2) * C::kTasks;
        int e = raw0 + (grp >> 2), other = raw0 + 1 - (grp >> 2);
        uint32_t ph = raw_phase, other_ph = raw_phase;
        if (e >= C::kRaw) {
          e -= C::kRaw;
          ph ^= 1;
        }
        if (other >= C::kRaw) {
          other -= C::kRaw;
          other_ph ^= 1;
        }
        const uint32_t slot_i = slot % kSlots, slot_ph = ((slot / kSlots) & 1) ^ 1;
        bool got = mbar_wait(&raw_full[e], ph, s_abort, err, kErrWaitFull);
        if (C::kBoth) {
          got = got && mbar_wait(&raw_full[other], other_ph, s_abort, err, kErrWaitFull);
          __syncwarp();
          if (got && lane == 0) mbar_arrive(&raw_empty[other]);
        }
#pragma unroll
        for (int y = 0; y < C::kTeamSlots; ++y)  // side by side: the slots of an item never wrap
          got = got && mbar_wait(&empty[slot_i + y], slot_ph, s_abort, err, kErrWaitEmpty);
        ok = __all_sync(~0u, got);
        if (!ok) break;
        uint8_t* dst = s_ring + slot_i * kSlotBytes;
        const uint8_t* from = s_raw + e * C::kUnitBytes + (grp & 3) * L::kHalf;
        if (is_k) {
#pragma unroll 1
          for (int k = 0; k < C::kTasks; ++k)
            emit_k<QT, D>(from, dst + k * (L::kSB / 64) * kSlotBytes, grp, sb0 + k, lane);
        } else {
          const int tok0 = tok_first + j * kTile;
          uint32_t keep0 = ~0u, keep1 = ~0u;
          if (tok0 < lo || tok0 + kTile > hi) {
            const int first = tok0 + grp * 16 + 2 * (lane & 3);
            auto in = [&](int tok) -> bool { return tok >= lo && tok < hi; };
            keep0 = (in(first) ? 0xFFFFu : 0u) | (in(first + 1) ? 0xFFFF0000u : 0u);
            keep1 = (in(first + 8) ? 0xFFFFu : 0u) | (in(first + 9) ? 0xFFFF0000u : 0u);
          }
          if (C::kTeams == 1) dst += (grp >> 2) * (D * 128);
#pragma unroll 1
          for (int k = 0; k < C::kTasks; ++k) emit_v<QT, D>(from, keep0, keep1, dst, grp, sb0 + k, lane);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane < C::kTeamSlots) mbar_arrive(&full[slot_i + lane]);
        if (lane == C::kTeamSlots) mbar_arrive(&raw_empty[e]);
        slot += C::kParts;
        raw0 += 2;
        if (raw0 >= C::kRaw) {
          raw0 -= C::kRaw;
          raw_phase ^= 1;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the units that several CTAs of tiles_kernel share: block (c, y, z) the columns 64 z .. 64 z + 63 of rows
// 32 y .. 32 y + 31 of the unit that begins in CTA c's share, if one does. A lane is a row, as in the parts (512 bytes of
// 32 rows side by side), a warp 8 columns; the outputs turn in shared memory. L2 and latency bound it: each part is read
// once, by enough blocks to cover the waits (25 us with 64-byte pieces and a block for all columns, 10 now, both with the
// parts out of L2: 148 shares, 20 MB).
template <int D, int TQ>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TcArgs a) {
  constexpr int kPart = TQ * kTile * (D + 2), kMost = 160;
  __shared__ float s_f[kMost][32], s_top[8][32], s_sum[8][32], s_inv[32];
  __shared__ float4 s_v[32][17];
  wait_before();
  const int c0 = blockIdx.x;
  const Shared u = a.shared[c0];
  if (!u.valid) return;
  const KvAttnParams& p = a.p;
  const int group = p.heads / p.c.heads, n_rows = p.nq * group;
  const int tile = blockIdx.y >> 2, row0 = (blockIdx.y & 3) * 32;
  if (u.row0 + tile * kTile + row0 >= n_rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = u.c1 - c0 + 1, at = row0 + lane;
  auto part_of = [&](int k) -> const float* {
    return a.part + (2 * (long long)(c0 + k) + (k == 0 ? u.second : 0)) * kPart + tile * (kTile * (D + 2)) + at;
  };
  // factors of the parts
  float top = kNoScore;
  for (int k = warp; k < n; k += 8) top = fmaxf(top, s_f[k][lane] = __ldcg(part_of(k) + kTile * D));
  s_top[warp][lane] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) top = fmaxf(top, s_top[k][lane]);
  float sum = 0.f;
  for (int k = warp; k < n; k += 8) {
    const float f = ex2_approx(s_f[k][lane] - top);
    s_f[k][lane] = f;
    sum = fmaf(__ldcg(part_of(k) + kTile * (D + 1)), f, sum);
  }
  s_sum[warp][lane] = sum;
  __syncthreads();
  const int first = u.row0 + tile * kTile + row0;  // row of lane 0
  if (warp == 0) {
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += s_sum[k][lane];
    s_inv[lane] = sum == 0.f ? 0.f : 1.f / sum;
    const int r = first + lane;
    if (p.lse && blockIdx.z == 0 && r < n_rows)
      p.lse[((long long)u.b * p.nq + r / group) * p.heads + u.head * group + r % group] =
          sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  }
  float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    // float4 x of the parts' row: [D / 4][128 rows]
    const float4* from = reinterpret_cast<const float4*>(part_of(k) - at) + (blockIdx.z * 16 + 2 * warp) * kTile + at;
    const float f = s_f[k][lane];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float4 x = __ldcg(from + e * kTile);
      v[e].x = fmaf(x.x, f, v[e].x);
      v[e].y = fmaf(x.y, f, v[e].y);
      v[e].z = fmaf(x.z, f, v[e].z);
      v[e].w = fmaf(x.w, f, v[e].w);
    }
  }
  s_v[lane][2 * warp] = v[0];
  s_v[lane][2 * warp + 1] = v[1];
  __syncthreads();
#pragma unroll
  for (int e = threadIdx.x; e < 32 * 16; e += 256) {
    const int rr = e >> 4, r = first + rr;
    if (r >= n_rows) break;
    const float4 x = s_v[rr][e & 15];
    const float inv = s_inv[rr];
    store_out(p, u.b * p.o_b + r / group * p.o_n + (u.head * group + r % group) * p.o_h + blockIdx.z * 64 + (e & 15) * 4,
              make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
  }
}

// The f16 operands of tiles_kernel, once for all its CTAs: block (x < kv_blocks) the K or the V item of one token tile of
// one sequence and head, a warp for each 16 tokens; the blocks after them the Q rows of one tile. Bound by HBM and L2: the
// cache read once, 4 bytes written per value pair. Rows and tokens outside every span are left as they are.
template <int QT, int D>
__global__ void __launch_bounds__(256) stage_kernel(const __grid_constant__ TcArgs a, int kv_blocks, int* err) {
  typedef KvL<QT, D> L;
  constexpr int TQ = D == 256 ? 1 : 2;
  wait_before();
  let_next();
  const KvAttnParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads / p.c.heads;
  if ((int)blockIdx.x >= kv_blocks) {
    const int x = blockIdx.x - kv_blocks, tile = x % (a.blocks * TQ), unit = x / (a.blocks * TQ);
    const int head = unit % p.c.heads, b = unit / p.c.heads;
    int lo, hi;
    if (!unit_tiles<kTile>(p, group, sequence_length(p, b, err), tile, &lo, &hi)) return;  // rows that see no token
    uint8_t* to = a.q_image + (long long)x * (kTile * D * 2);
    for (int e = threadIdx.x; e < kTile * (D / 8); e += 256) {
      const int rr = e / (D / 8), c16 = e % (D / 8), r = tile * kTile + rr;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < p.nq * group)
        v = *reinterpret_cast<const uint4*>(p.q + b * p.q_b + r / group * p.q_n + (head * group + r % group) * p.q_h + c16 * 8);
      *reinterpret_cast<uint4*>(to + c16 / 8 * kSlotBytes + rr * 128 + ((c16 & 7) ^ (rr & 7)) * 16) = v;
    }
    return;
  }
  const int kv = blockIdx.x & 1, x = blockIdx.x >> 1, j = x % a.tiles, unit = x / a.tiles;
  const int head = unit % p.c.heads, b = unit / p.c.heads;
  const int len = sequence_length(p, b, err);
  int lo, hi, none;
  row_span(p, len, 0, &lo, &none);
  row_span(p, len, p.nq - 1, &none, &hi);
  const int tok0 = j * kTile, first = tok0 + warp * 16;
  if (tok0 >= hi || tok0 + kTile <= lo) return;
  const int per_page = p.c.page_size >> 4;
  // tokens outside the span: their keys may hold anything, their values become zero
  const bool live = first < hi && first + 16 > lo;
  const int gi = live ? first >> 4 : max(lo, tok0) >> 4;
  long long page = p.pages[b * p.pages_stride + gi / per_page];
  if (page < 0 || page >= p.c.n_pages) {
    atomicCAS(err, 0, kDevErrIndex);
    page = 0;
  }
  const uint8_t* from = p.c.data + kv_group_offset<QT, D>(p.c, page, head, kv, gi % per_page);
  uint8_t* item = a.image + (long long)blockIdx.x * (D * 256);
  if (kv == 0) {
#pragma unroll
    for (int sb = 0; sb < D / L::kSB; ++sb)
      emit_k<QT, D>(from, item + sb * (L::kSB / 64) * kSlotBytes, warp, sb, lane);
  } else {
    const int mine = first + 2 * (lane & 3);
    auto in = [&](int tok) -> bool { return tok >= lo && tok < hi; };
    const uint32_t keep0 = (in(mine) ? 0xFFFFu : 0u) | (in(mine + 1) ? 0xFFFF0000u : 0u);
    const uint32_t keep1 = (in(mine + 8) ? 0xFFFFu : 0u) | (in(mine + 9) ? 0xFFFF0000u : 0u);
#pragma unroll
    for (int sb = 0; sb < D / L::kSB; ++sb)
      emit_v<QT, D>(from, keep0, keep1, item + (warp >> 2) * (D * 128), warp, sb, lane);
  }
}

// Whether the operands are staged as f16 first. Each row block of a unit would dequantise the whole cache again; staged, it
// is done once, at the cost of 4 bytes written and read for each value pair. Measured for 8 sequences, fused / staged:
//   d = 64,  8192 tokens, 16 heads on 4, 1, 2, 3 blocks of 256 rows: 71 / 73, 99 / 93, 128 / 115 us
//   d = 128, the same:                                               91 / 101, 122 / 126, 158 / 154 us
//   d = 256, 16384 tokens, 1 head, 3, 4, 5 blocks of 128 rows:       111 / 119, 127 / 138, 142 / 144 us
// and with many blocks 198 / 151 us (4096 rows over 28736 tokens, d = 256) and 417 / 362 (4 x 2048 causal queries, d = 128)
// when staging came in. The images have to fit a bounded workspace.
constexpr long long kStageMost = 1LL << 30;
struct TcPlan {
  int tq;
  long long blocks, tiles, kv_bytes, q_bytes;
  bool staged;
};
TcPlan tc_plan(const KvAttnParams& p) {
  TcPlan t;
  t.tq = p.c.d == 256 ? 1 : 2;
  t.blocks = (p.nq * (long long)(p.heads / p.c.heads) + t.tq * kTile - 1) / (t.tq * kTile);
  t.tiles = ((long long)p.max_pages * p.c.page_size + kTile - 1) / kTile;
  const long long units = (long long)p.batch * p.c.heads;
  t.kv_bytes = units * t.tiles * p.c.d * 512;
  t.q_bytes = units * t.blocks * t.tq * kTile * p.c.d * 2;
  t.staged = t.blocks >= (p.c.d == 256 ? 6 : p.c.d == 128 ? 3 : 2) && t.tiles > 0 && units < (1 << 24) && t.tiles < (1 << 24) &&
             t.kv_bytes + t.q_bytes <= kStageMost;
  return t;
}
size_t part_floats(int sms, int tq, int d) { return (size_t)2 * sms * tq * kTile * (d + 2); }

template <int QT, int D>
int launch_tiles(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  constexpr int TQ = D == 256 ? 1 : 2;
  if (w.sms > 160) return -2;  // join_kernel's table of factors
  const TcPlan t = tc_plan(p);
  TcArgs a;
  a.p = p;
  a.part = w.part;
  a.shared = reinterpret_cast<Shared*>(w.part + part_floats(w.sms, TQ, D));
  a.blocks = (int)t.blocks;
  a.tiles = (int)t.tiles;
  a.image = w.image;
  a.q_image = a.image + t.kv_bytes;
  int rc;
  if (t.staged) {
    typedef Tc<QT_Q4_0, D, true> C;  // the staged kernel does not depend on the cache's type
    auto* k = tiles_kernel<QT_Q4_0, D, true>;
    if (kernel_setup(k, C::kSmem) <= 0) return -13;
    const long long kv_blocks = 2LL * p.batch * p.c.heads * t.tiles;
    const long long q_blocks = (long long)p.batch * p.c.heads * t.blocks * TQ;
    rc = launch_dependent(stage_kernel<QT, D>, dim3((unsigned)(kv_blocks + q_blocks)), 256, 0, st, a, (int)kv_blocks, err);
    if (rc) return rc;
    rc = launch_dependent(k, dim3(w.sms), C::kThreads, C::kSmem, st, a, err);
  } else {
    typedef Tc<QT, D, false> C;
    auto* k = tiles_kernel<QT, D, false>;
    if (kernel_setup(k, C::kSmem) <= 0) return -13;
    rc = launch_dependent(k, dim3(w.sms), C::kThreads, C::kSmem, st, a, err);
  }
  if (rc) return rc;
  return launch_dependent(join_kernel<D, TQ>, dim3(w.sms, TQ * 4, D / 64), 256, 0, st, a);
}

template <int QT>
int launch_tiles_d(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  return p.c.d == 64 ? launch_tiles<QT, 64>(p, w, err, st)
                     : p.c.d == 128 ? launch_tiles<QT, 128>(p, w, err, st) : launch_tiles<QT, 256>(p, w, err, st);
}

}  // namespace

size_t kv_attention_tc_parts(int sms) {
  return std::max(part_floats(sms, 2, 128), part_floats(sms, 1, 256)) * 4 + sms * sizeof(Shared);
}

size_t kv_attention_tc_image(const KvAttnParams& p) {
  const TcPlan t = tc_plan(p);
  return t.staged ? (size_t)(t.kv_bytes + t.q_bytes) : 0;
}

int kv_attention_tc_launches(const KvAttnParams& p) { return tc_plan(p).staged ? 3 : 2; }

int kv_attention_tc(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  return p.c.type == QT_Q4_0 ? launch_tiles_d<QT_Q4_0>(p, w, err, st)
                             : p.c.type == QT_Q4_1 ? launch_tiles_d<QT_Q4_1>(p, w, err, st)
                                                   : launch_tiles_d<QT_Q8_0>(p, w, err, st);
}

}  // namespace s3b
