// Attention of trees of drafted tokens over the 4-bit cache (kv_attend_kernels.h).
#include "kv_attend_kernels.h"

namespace {

bool tree_ok(int64_t nodes, int64_t window) {
  return nodes >= 1 && nodes <= 512 && (window == 0 || window >= nodes);
}

}  // namespace

extern "C" {

int64_t gptq2d_kv_attend_tree_workspace(int64_t tokens, int64_t seqs, int32_t heads, int32_t group, int32_t dim, int64_t most,
                                        int64_t window, int64_t nodes) {
  if (!attend_ok(tokens, seqs, heads, group, dim, most, window) || !tree_ok(nodes, window)) return -1;
  return 4 * make_plan(tokens, seqs, heads, group, dim, most, window, (nodes + 31) / 32 * 32).part;
}

int gptq2d_kv_attend_tree(const void* pages, int64_t page_count, int32_t heads, int32_t dim, int32_t page, const void* q,
                          int64_t q_token, int64_t q_head, int32_t group, int32_t type, const int32_t* table, int64_t seqs,
                          int64_t width, int64_t table_stride, const int32_t* lengths, const int32_t* offsets, int64_t tokens,
                          const uint32_t* ancestors, const int32_t* positions, int64_t nodes, double scale, int64_t window,
                          void* out, int64_t out_token, int64_t out_head, float* lse, void* work, int64_t work_bytes,
                          void* stream) {
  KvCache c;
  if (!make_cache(c, pages, page_count, heads, dim, page, table, seqs, width, table_stride, lengths, offsets, tokens) ||
      !offsets || !tree_ok(nodes, window))
    return GPTQ2D_EINVAL;
  Attend a = {};
  a.seen = ancestors, a.at = positions, a.words = (int)((nodes + 31) / 32);
  return attend<true>(c, a, q, q_token, q_head, group, type, scale, window, out, out_token, out_head, lse, work, work_bytes,
                      stream);
}

}  // extern "C"
