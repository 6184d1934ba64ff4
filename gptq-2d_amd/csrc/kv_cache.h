// The paged cache of keys and values in 4 bits: its layout, and what its kernels (append, read, attention) share.
//
// Values.  A token's key (or value) vector x of one head is held as codes c in 0..15 with a scale s and a zero z of 16
// bits each: s = bf16((max x - min x) / 15), 1 where that is 0; z = bf16(min x); c = clamp(rint((x - z) / s), 0, 15), every
// step in fp32.  It stands for c s + z, which the kernels take as (c - 8) s + (z + 8 s): c - 8 is exact in fp16 and
// centred, so products with it keep no offset that a later subtraction would have to cancel.  Where s is 1 in the place of 0
// and all c are 0, s is held as -0: the same value, without an offset of 8.  No other scale has a sign, not a NaN's either.
//
// Layout.  The head size is padded to DP = 64 ND with codes that no query meets (its elements there are 0) and no
// output shows.  A page holds `page` tokens (a multiple of 32) of every head, head by head; one head's part is
//   K codes, V codes: page / 32 blocks of 32 tokens, each ND chunks of 64 lanes x 4 words;
//   K scales, V scales: one word per token, s in the low half and z in the high one.
// The words of a block are what the lanes of one wave feed to v_mfma_f32_16x16x32_f16 as its A operand (lane l: row
// l % 16, elements 8 (l / 16) .. + 7), so that every load of codes is 16 bytes a lane, 1 KB a wave, in lane order:
//   K: word W of lane l is key 16 (W / (2 ND)) + l % 16, elements d = 32 (W % (2 ND)) + 8 (l / 16) .. + 7 (Q K^T with the
//      keys as rows);
//   V: word W of lane l is element d = 16 W + l % 16 of the eight tokens 4 (l / 16) + {0..3}, 16 + 4 (l / 16) + {0..3}
//      (V^T P^T with the elements as rows).  The result of K Q^T (lane l: keys 4 (l / 16) .. + 3 of a tile of 16, query
//      l % 16) is then already the B operand of V^T P^T: P never leaves its lane.
// Word W lies in chunk W / 4 at 4 l + W % 4.  Element 2 j of a word's eight is its nibble j, element 2 j + 1 nibble j + 4:
// masking gives both halves of a pair of fp16 at once.
#pragma once

#include "elements.h"

namespace {

// The eight codes of a word, less 8, in fp16.  1024 + c and 1024 + 16 c are fp16 numbers with the code in their low
// bits; one subtraction (or multiplication by 1/16 and subtraction) leaves c - 8, exactly: nine instructions a word.
__device__ __forceinline__ half8 centred_codes(unsigned w) {
  union {
    half2v h[4];
    half8 v;
  } r;
  const unsigned x = w >> 8;
  r.h[0] = codes_at(w, 0x000f000fu) + both(-1032.f);
  r.h[1] = __builtin_elementwise_fma(codes_at(w, 0x00f000f0u), both(0.0625f), both(-72.f));
  r.h[2] = codes_at(x, 0x000f000fu) + both(-1032.f);
  r.h[3] = __builtin_elementwise_fma(codes_at(x, 0x00f000f0u), both(0.0625f), both(-72.f));
  return r.v;
}

constexpr unsigned FLAT = 0x8000u;  // scale -0, zero 0

struct KvCache {
  unsigned* pages;
  int64_t page_count;
  int64_t page_words;  // of one page, all heads
  int heads, dim, page, blocks;  // blocks: 32-token blocks of a page
  unsigned mag;                  // ceil(2^32 / blocks): kb / blocks = umulhi(kb, mag) for kb blocks < 2^32
  const int32_t* table;          // [seqs, width], rows table_stride apart
  int64_t table_stride;
  int width;
  int64_t seqs;
  const int32_t* lengths;  // [seqs]
  const int32_t* offsets;  // [seqs + 1], or none: one token a sequence
  int64_t tokens;
};

__host__ __device__ __forceinline__ int64_t kv_head_words(int nd, int page) { return (int64_t)page * (16 * nd + 2); }

// First token of sequence b among the packed ones, kept within them whatever the array holds.
__device__ __forceinline__ int64_t kv_offset(const KvCache& c, int64_t b) {
  if (!c.offsets) return b < c.tokens ? b : c.tokens;
  const int64_t o = c.offsets[b < c.seqs ? b : c.seqs];
  return o < 0 ? 0 : o > c.tokens ? c.tokens : o;
}

// Sequence b's tokens (times `mul`) are dealt to groups of `per` in slots first(b) .. first(b + 1) - 1 with
// first(b) = mul offset(b) / per + extra b: with extra = 1 a sequence has slots for all of its groups, with extra = 2 also
// where its first group begins inside another.  No sequence's slots depend on more than its offset, so a workgroup finds
// its own with one wave-wide search of 64 candidates a step.  Slots before the first sequence's are found as its: they, and
// the last sequence's past its groups, are where the rows that no sequence has are dealt with.  (No sequences: slots of one
// without tokens.)
__device__ __forceinline__ int64_t kv_first_slot(const KvCache& c, int64_t b, int mul, int per, int extra) {
  return (int64_t)((uint64_t)(kv_offset(c, b) * mul) / (unsigned)per) + extra * b;
}

__device__ __forceinline__ int64_t kv_find(const KvCache& c, int64_t slot, int mul, int per, int extra) {
  int64_t lo = 0, n = c.seqs;
  const int lane = threadIdx.x & 63;
  while (n > 1) {
    const int64_t step = (n + 63) / 64;
    const bool ok = lane * step < n && kv_first_slot(c, lo + lane * step, mul, per, extra) <= slot;
    const int cnt = __popcll(__builtin_amdgcn_ballot_w64(ok));
    const int64_t skip = (cnt > 0 ? cnt - 1 : 0) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  return lo;
}

// Block kb (of 32 tokens) of sequence b, head h: its first K code, or none where the table's entry is no page.
// `at`: the block's number in its page.
__device__ __forceinline__ unsigned* kv_head(const KvCache& c, int64_t b, int kb, int h, int head_words, int& at) {
  const int p = (int)__umulhi((unsigned)kb, c.mag);
  at = kb - p * c.blocks;
  if (c.blocks == 1) at = 0;
  // a uniform index: through the scalar data cache (no kernel writes the table), whose loads wait for no others
  typedef const __attribute__((address_space(4))) int32_t* scalar;
  const int64_t id = ((scalar)(c.table + b * c.table_stride))[__builtin_amdgcn_readfirstlane(c.blocks == 1 ? kb : p)];
  if (id < 0 || id >= c.page_count) return nullptr;
  return c.pages + id * c.page_words + (int64_t)h * head_words;
}

// The cache's description from the C entries' arguments; false where they cannot be one.
inline bool make_cache(KvCache& c, const void* pages, int64_t page_count, int32_t heads, int32_t dim, int32_t page,
                       const int32_t* table, int64_t seqs, int64_t width, int64_t table_stride, const int32_t* lengths,
                       const int32_t* offsets, int64_t tokens) {
  if (heads < 1 || heads > 65535 || dim < 1 || dim > 256 || page < 32 || page > 4096 || page % 32 || page_count < 0 ||
      seqs < 0 || width < 0 || width * page >= ((int64_t)1 << 29) || table_stride < 0 || tokens < 0 ||
      seqs > ((int64_t)1 << 24) || tokens > 0x7fffffff || (!offsets && tokens != seqs))
    return false;
  c.pages = static_cast<unsigned*>(const_cast<void*>(pages));
  c.page_count = page_count;
  c.page_words = heads * kv_head_words((dim + 63) / 64, page);
  c.heads = heads;
  c.dim = dim;
  c.page = page;
  c.blocks = page / 32;
  c.mag = (unsigned)((((uint64_t)1 << 32) + c.blocks - 1) / c.blocks);
  c.table = table;
  c.table_stride = table_stride;
  c.width = (int)width;
  c.seqs = seqs;
  c.lengths = lengths;
  c.offsets = offsets;
  c.tokens = tokens;
  return true;
}

}  // namespace
