// Attention of new tokens over the 4-bit cache, a sequence's last ones (kv_attend_kernels.h).
#include "kv_attend_kernels.h"

extern "C" {

int64_t gptq2d_kv_attend_workspace(int64_t tokens, int64_t seqs, int32_t heads, int32_t group, int32_t dim, int64_t most,
                                   int64_t window) {
  if (!attend_ok(tokens, seqs, heads, group, dim, most, window)) return -1;
  return 4 * make_plan(tokens, seqs, heads, group, dim, most, window).part;
}

int gptq2d_kv_attend(const void* pages, int64_t page_count, int32_t heads, int32_t dim, int32_t page, const void* q,
                     int64_t q_token, int64_t q_head, int32_t group, int32_t type, const int32_t* table, int64_t seqs,
                     int64_t width, int64_t table_stride, const int32_t* lengths, const int32_t* offsets, int64_t tokens,
                     double scale, int64_t window, void* out, int64_t out_token, int64_t out_head, float* lse, void* work,
                     int64_t work_bytes, void* stream) {
  KvCache c;
  if (!make_cache(c, pages, page_count, heads, dim, page, table, seqs, width, table_stride, lengths, offsets, tokens))
    return GPTQ2D_EINVAL;
  return attend<false>(c, Attend{}, q, q_token, q_head, group, type, scale, window, out, out_token, out_head, lse, work,
                       work_bytes, stream);
}

}  // extern "C"
