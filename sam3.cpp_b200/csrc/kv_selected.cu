// Attention over selected pages of the quantised key / value cache: rows_kernel (kv_rows.cuh) by lists.
#include "kv_rows.cuh"

namespace s3b {

int kv_attention_selected(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  if (p.out_f32) return kv_attention_selected_f32(p, w, err, st);
  return p.c.type == QT_Q4_0 ? attend_d<QT_Q4_0, kLists>(p, w, err, st)
                             : p.c.type == QT_Q4_1 ? attend_d<QT_Q4_1, kLists>(p, w, err, st) : attend_d<QT_Q8_0, kLists>(p, w, err, st);
}

}  // namespace s3b
