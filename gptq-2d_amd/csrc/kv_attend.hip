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
  const int64_t most = width * page;
  if (!attend_ok(tokens, seqs, heads, group, dim, most, window)) return GPTQ2D_EINVAL;
  if (tokens == 0) return 0;
  Attend a = {};
  const Plan p = make_plan(tokens, seqs, heads, group, dim, most, window);
  const int rc = set_call(a, p, !p.prompt, q, q_token, q_head, group, scale, window, out, out_token, out_head, lse, work, work_bytes);
  if (rc) return rc;
  switch (type) {
    case TYPE_F32:
      return launch_type<false, TYPE_F32>(c, a, p, (hipStream_t)stream);
    case TYPE_BF16:
      return launch_type<false, TYPE_BF16>(c, a, p, (hipStream_t)stream);
    case TYPE_F16:
      return launch_type<false, TYPE_F16>(c, a, p, (hipStream_t)stream);
  }
  return GPTQ2D_EINVAL;
}

}  // extern "C"
