// Attention over the quantised key / value cache: which kernel takes a call (kv_rows.cuh, kv_attention_tc.cu).
#include "kv_rows.cuh"

namespace s3b {

// Rows of one key / value head that rows_kernel takes (its output registers end at 128 a thread). tiles_kernel fills 128 or
// 256 rows whatever the count, so this one is ahead as far as it goes: 32 rows over 32 x 8192 tokens and 8 heads of 128
// take 207 us against 256, 16 rows over 8 x 28736 tokens and one head of 256 take 55 against 84.
int kv_attention_most_rows(int d) { return d == 256 ? 16 : 32; }

KvAttnBytes kv_attention_work(const KvAttnParams& p, int sms) {
  // two parts for each of rows_kernel's CTAs: at most 4 an SM with 8 rows, 3 with 16 and 2 with 32 of d = 128, or with 16 of 256
  constexpr int kMost = 2 * Rows<QT_Q4_0, 128, 4, 4>::kCtas * 32 * (128 + 2);
  static_assert(2 * Rows<QT_Q4_0, 128, 1, 4>::kCtas * 8 * 130 <= kMost && 2 * Rows<QT_Q4_0, 128, 2, 4>::kCtas * 16 * 130 <= kMost &&
                    2 * Rows<QT_Q4_0, 64, 4, 4>::kCtas * 32 * 66 <= kMost && 2 * Rows<QT_Q4_0, 64, 2, 4>::kCtas * 16 * 66 <= kMost &&
                    2 * Rows<QT_Q4_0, 256, 1, 4>::kCtas * 8 * 258 <= kMost && 2 * Rows<QT_Q4_0, 256, 2, 4>::kCtas * 16 * 258 <= kMost,
                "parts of rows_kernel");
  KvAttnBytes b;
  b.part = std::max((size_t)sms * kMost * 4, kv_attention_tc_parts(sms));
  b.count = (size_t)kv_attention_units(p) * 4;
  b.image = !p.share && p.nq * (long long)(p.heads / p.c.heads) > kv_attention_most_rows(p.c.d) ? kv_attention_tc_image(p) : 0;
  return b;
}

int kv_attention_launches(const KvAttnParams& p) {
  return p.nq * (long long)(p.heads / p.c.heads) > kv_attention_most_rows(p.c.d) ? kv_attention_tc_launches(p) : 1;
}

int kv_attention(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  if (p.nq * (long long)(p.heads / p.c.heads) > kv_attention_most_rows(p.c.d)) return kv_attention_tc(p, w, err, st);
  return p.c.type == QT_Q4_0 ? attend_d<QT_Q4_0, kAllPages>(p, w, err, st)
                             : p.c.type == QT_Q4_1 ? attend_d<QT_Q4_1, kAllPages>(p, w, err, st) : attend_d<QT_Q8_0, kAllPages>(p, w, err, st);
}

}  // namespace s3b
