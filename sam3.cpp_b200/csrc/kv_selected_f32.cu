// Attention over selected pages with f32 outputs.
#include "kv_rows.cuh"

namespace s3b {

int kv_attention_selected_f32(const KvAttnParams& p, const KvAttnWork& w, int* err, cudaStream_t st) {
  return p.c.type == QT_Q4_0 ? attend_d<QT_Q4_0, kListsF32>(p, w, err, st)
                             : p.c.type == QT_Q4_1 ? attend_d<QT_Q4_1, kListsF32>(p, w, err, st) : attend_d<QT_Q8_0, kListsF32>(p, w, err, st);
}

}  // namespace s3b
