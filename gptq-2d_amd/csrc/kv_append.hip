// Keys and values into the 4-bit cache (append) and back out of it (read).
//
// Both are bound by memory: a token's vectors are read (written) once, and 4.5 bits an element written (read).  A
// workgroup takes one block of 32 tokens of one head, keys or values: the words of V hold eight tokens each, so the block
// is the smallest part that no other workgroup of the call writes.  Eight threads take a token; codes go through LDS
// into the words' order, so that whole blocks are written 16 bytes a thread in order.  In a block that is not all new
// the words of K (one token each) and the scales of the new tokens are written alone, and in the words of V the new
// tokens' nibbles replace the old.
// Measured, 8000 tokens, 8 heads of 128, fp16, keys and values: append 25 us (42 MB: one round of workgroups, each a chain
// of load, maximum, division, LDS and store), read into fp32 19.4 us (74 MB, 3.8 TB/s).  One token of 64 sequences: 6 us
// and 4.
#include "kv_cache.h"

namespace {

constexpr int THREADS = 256;

struct Rows {
  void* k;
  void* v;
  int64_t k_token, k_head, v_token, v_head;  // strides in elements
};

struct BlockIds {
  int64_t b, row0;  // row0: packed row of the block's token 0 (may be before the sequence's first)
  int kb, first, last;  // block of the sequence, and its tokens [first, last) that the call takes
  bool any;
  int64_t t0, none0, none1, t1;  // rows of the sequence, those outside [none0, none1) without a place in the cache
  bool leads;                    // the sequence's first slot
};

// Which block this workgroup takes; `back`: the lengths count the call's tokens already (read), else not (append).
__device__ __forceinline__ BlockIds block_ids(const KvCache& c, int64_t slot, bool back) {
  BlockIds id;
  id.b = c.offsets ? kv_find(c, slot, 1, 32, 2) : slot;
  const int64_t t0 = kv_offset(c, id.b), t1 = kv_offset(c, id.b + 1);
  const int64_t most = (int64_t)c.width * c.page, n = t1 > t0 ? t1 - t0 : 0;
  const int64_t held = c.seqs ? c.lengths[id.b] : 0;
  const int64_t start = back ? held - n : held;  // position of the first token
  const int64_t begin = start < 0 ? 0 : start;
  const int64_t end = start + n < most ? start + n : most;
  const int64_t rel = c.offsets ? slot - kv_first_slot(c, id.b, 1, 32, 2) : 0;  // below 0 before the first sequence
  const int64_t kb = begin / 32 + rel;
  id.any = rel >= 0 && end > begin && kb * 32 < end;
  id.kb = (int)kb;
  id.first = (int)(begin > kb * 32 ? begin - kb * 32 : 0);
  id.last = (int)(end < kb * 32 + 32 ? end - kb * 32 : 32);
  id.row0 = t0 + kb * 32 - start;
  id.t0 = t0, id.t1 = t0 + n;
  id.none0 = end > begin ? t0 + begin - start : id.t1;
  id.none1 = end > begin ? t0 + end - start : id.t1;
  id.leads = rel == 0;
  return id;
}

template <int TYPE, int ND>
__global__ __launch_bounds__(THREADS) void append_kernel(KvCache c, Rows r) {
  typedef typename Elem<TYPE>::T T;
  constexpr int DP = 64 * ND, PER = DP / 8;  // elements of a thread
  alignas(16) __shared__ unsigned words[DP * 4];
  __shared__ unsigned codes[32][DP / 4 + 1];  // V: codes of a token, a byte each
  __shared__ unsigned affine[32];
  const BlockIds id = block_ids(c, blockIdx.x, false);
  if (!id.any) return;
  const int h = blockIdx.y;
  const bool value = blockIdx.z;
  const int hw = (int)kv_head_words(ND, c.page);
  int at;
  unsigned* base = kv_head(c, id.b, id.kb, h, hw, at);
  if (!base) return;
  unsigned* out = base + (value ? (int64_t)c.page * 8 * ND : 0) + at * (DP * 4);
  unsigned* out_affine = base + (int64_t)c.page * (16 * ND + (value ? 1 : 0)) + at * 32;

  const int token = threadIdx.x >> 3, part = threadIdx.x & 7;
  const bool mine = token >= id.first && token < id.last;
  if (mine) {
    const T* row = value ? (const T*)r.v + (id.row0 + token) * r.v_token + h * r.v_head
                         : (const T*)r.k + (id.row0 + token) * r.k_token + h * r.k_head;
    float x[PER];
    load_row<TYPE, PER>(x, row, PER * part, c.dim);
    // extremes; a NaN stays, and makes scale and zero NaN
    float lo = PER * part < c.dim ? x[0] : __builtin_inff();
    float hi = PER * part < c.dim ? x[0] : -__builtin_inff();
#pragma unroll
    for (int i = 1; i < PER; ++i) {
      const bool in = PER * part + i < c.dim;
      lo = in && (x[i] < lo || x[i] != x[i]) ? x[i] : lo;
      hi = in && (x[i] > hi || x[i] != x[i]) ? x[i] : hi;
    }
#pragma unroll
    for (int s = 1; s < 8; s *= 2) {
      const float l2 = __shfl_xor(lo, s), h2 = __shfl_xor(hi, s);
      lo = l2 < lo || l2 != l2 ? l2 : lo;
      hi = h2 > hi || h2 != h2 ? h2 : hi;
    }
    const float step = round_to_bf16((hi - lo) / 15.f), s = step == 0.f ? 1.f : step;
    const float z = round_to_bf16(lo);
    // Without a spread and with codes of 0 (as the largest element's) the vector stands for its zero, and is held with a scale of
    // -0: the scale of 1 would not be its size, and (c - 8) s and z + 8 s would have to cancel (attention holds the first to
    // 11 bits).
    const bool flat = step == 0.f && round_even(hi - z) <= 0.f;
    if (part == 0)
      affine[token] = (flat ? FLAT : __float_as_uint(s) >> 16 & 0x7fffu) | (__float_as_uint(z) & 0xffff0000u);
    // The quotient (x - z) / s as IEEE rounds it, from the correctly rounded 1 / s and one correction with the exact
    // remainder (Markstein's method), where s is in a range in which nothing on the way leaves the normal numbers (the
    // differences are below 2^5 s, and below 2^-24 of s they round to code 0 whatever the remainder); a division otherwise.
    const float rcp = 1.f / s;
    const bool plain = s >= 0x1p-60f && s <= 0x1p60f;
    unsigned code[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float y = x[i] - z, q0 = y * rcp;
      float q = __builtin_fmaf(__builtin_fmaf(-q0, s, y), rcp, q0);
      if (!plain) q = y / s;
      q = __builtin_amdgcn_fmed3f(round_even(q), 0.f, 15.f);
      code[i] = q == q ? (unsigned)q : 0u;
    }
    if (value) {
#pragma unroll
      for (int i = 0; i < PER; i += 4)
        codes[token][(PER * part + i) / 4] = code[i] | code[i + 1] << 8 | code[i + 2] << 16 | code[i + 3] << 24;
    } else {
#pragma unroll
      for (int i = 0; i < PER; i += 8) {
        const int d = PER * part + i, lane = token % 16 + 16 * (d / 8 % 4), W = 2 * ND * (token / 16) + d / 32;
        unsigned w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= code[i + e] << (e / 2 * 4 + e % 2 * 16);
        words[W / 4 * 256 + lane * 4 + W % 4] = w;
      }
    }
  }
  __syncthreads();
  const bool whole = id.first == 0 && id.last == 32;
  if (threadIdx.x < 32 && (int)threadIdx.x >= id.first && (int)threadIdx.x < id.last)
    out_affine[threadIdx.x] = affine[threadIdx.x];
  if (!value) {
    if (whole) {
#pragma unroll
      for (int i = threadIdx.x; i < DP; i += THREADS)
        reinterpret_cast<uint4v*>(out)[i] = reinterpret_cast<const uint4v*>(words)[i];
    } else {
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        const int i = THREADS * j + threadIdx.x, W = i / 256 * 4 + i % 4, key = W / (2 * ND) * 16 + i / 4 % 16;
        if (key >= id.first && key < id.last) out[i] = words[i];
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < ND; ++j) {  // DP * 4 = THREADS * ND words
    const int i = THREADS * j + threadIdx.x, lane = i / 4 % 64, d = 16 * (i / 256 * 4 + i % 4) + lane % 16, g = lane / 16;
    unsigned w = 0, keep = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int token_e = 4 * g + e % 4 + e / 4 * 16, shift = e / 2 * 4 + e % 2 * 16;
      const bool fresh = token_e >= id.first && token_e < id.last;
      const unsigned code = codes[token_e][d / 4] >> (d % 4 * 8) & 15u;  // of an old token: whatever LDS holds
      w |= (fresh ? code : 0u) << shift;
      keep |= (fresh ? 0u : 15u) << shift;
    }
    const unsigned old = whole ? 0u : out[i];
    out[i] = w | (old & keep);
  }
}

// A block's words go through LDS, so that both they and the values lie in order in memory: a thread gives eight elements
// of one token, from one word of K or from one nibble each of eight words of V.
template <int TYPE, int ND>
__global__ __launch_bounds__(THREADS) void read_kernel(KvCache c, Rows r) {
  typedef typename Elem<TYPE>::T T;
  constexpr int DP = 64 * ND, V = 16 / (int)sizeof(T);  // elements of a 16-byte store
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  alignas(16) __shared__ unsigned words[DP * 4];
  __shared__ unsigned affine[32];
  const BlockIds id = block_ids(c, blockIdx.x, true);
  const int h = blockIdx.y;
  const bool value = blockIdx.z;
  T* out = value ? (T*)r.v + h * r.v_head : (T*)r.k + h * r.k_head;
  const int64_t stride = value ? r.v_token : r.k_token;
  if (id.leads && (id.none0 > id.t0 || id.none1 < id.t1)) {  // tokens that the cache cannot hold: zeros
    for (int64_t row = id.t0; row < id.t1; ++row)
      if (row < id.none0 || row >= id.none1)
        for (int d = threadIdx.x; d < c.dim; d += THREADS) out[row * stride + d] = from_f32<TYPE>(0.f);
  }
  // rows that no sequence has: 32 of them a slot before the first one's, and as the last one's that would follow its own
  if (__builtin_expect(c.offsets && ((id.b == 0 && id.t0 > 0) || (id.b + 1 >= c.seqs && id.t1 < c.tokens)), 0)) {
    const int64_t slot = blockIdx.x, rel = slot - kv_first_slot(c, id.b, 1, 32, 2);
    const auto clear = [&](int64_t from, int64_t to, int64_t least, int64_t most) {
      from = from > least ? from : least, to = to < most ? to : most;
      for (int64_t row = from; row < to; ++row)
        for (int d = threadIdx.x; d < c.dim; d += THREADS) out[row * stride + d] = from_f32<TYPE>(0.f);
    };
    if (id.b == 0) clear(32 * slot, 32 * slot + 32, 0, id.t0);
    if (id.b + 1 >= c.seqs && rel >= 0) clear(id.t0 + 32 * rel, id.t0 + 32 * rel + 32, id.t1, c.tokens);
  }
  if (!id.any) return;
  const int hw = (int)kv_head_words(ND, c.page);
  int at;
  const unsigned* base = kv_head(c, id.b, id.kb, h, hw, at);
  if (base) {
    const unsigned* in = base + (value ? (int64_t)c.page * 8 * ND : 0) + at * (DP * 4);
    if (ND % 4 == 0 || threadIdx.x < DP) {
#pragma unroll
      for (int j = 0; j < (ND + 3) / 4; ++j)
        reinterpret_cast<uint4v*>(words)[THREADS * j + threadIdx.x] = reinterpret_cast<const uint4v*>(in)[THREADS * j + threadIdx.x];
    }
    if (threadIdx.x < 32) affine[threadIdx.x] = base[(int64_t)c.page * (16 * ND + (value ? 1 : 0)) + at * 32 + threadIdx.x];
  } else {  // the table's entry is no page: zeros
    for (int i = threadIdx.x; i < DP * 4; i += THREADS) words[i] = 0;
    if (threadIdx.x < 32) affine[threadIdx.x] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ND; ++j) {
    const int i = THREADS * j + threadIdx.x, token = i / (8 * ND), d = i % (8 * ND) * 8;
    const unsigned a = affine[token];
    const float s = __uint_as_float(a << 16), z = __uint_as_float(a & 0xffff0000u);
    unsigned w[8];
    int shift[8];
    if (value) {
      const int e = token % 4 + token / 16 * 4, lane = d % 16 + 16 * (token / 4 % 4), W = d / 16;
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = words[W / 4 * 256 + (lane + k) * 4 + W % 4], shift[k] = e / 2 * 4 + e % 2 * 16;
    } else {
      const int W = 2 * ND * (token / 16) + d / 32;
      w[0] = words[W / 4 * 256 + (token % 16 + 16 * (d / 8 % 4)) * 4 + W % 4];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = w[0], shift[k] = k / 2 * 4 + k % 2 * 16;
    }
    T x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = from_f32<TYPE>(__builtin_fmaf((float)(w[k] >> shift[k] & 15u), s, z));
    T* to = out + (id.row0 + token) * stride + d;
    const bool in = token >= id.first && token < id.last;
    if (in && d + 8 <= c.dim) {
#pragma unroll
      for (int k = 0; k < 8; k += V) {
        vec v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = x[k + e];
        *reinterpret_cast<vec*>(to + k) = v;
      }
    } else if (in) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (d + k < c.dim) to[k] = x[k];
    }
  }
}

template <int TYPE>
int launch(bool back, const KvCache& c, const Rows& r, int nd, hipStream_t st) {
  const int64_t slots = c.offsets ? c.tokens / 32 + 2 * (c.seqs + !c.seqs) : c.seqs;
  if (slots > 0x7fffffff) return GPTQ2D_EUNSUPPORTED;
  const dim3 grid((unsigned)slots, (unsigned)c.heads, 2);
#define GPTQ2D_KV_CASE(ND)                                                             \
  case ND:                                                                             \
    if (back)                                                                          \
      hipLaunchKernelGGL((read_kernel<TYPE, ND>), grid, dim3(THREADS), 0, st, c, r);   \
    else                                                                               \
      hipLaunchKernelGGL((append_kernel<TYPE, ND>), grid, dim3(THREADS), 0, st, c, r); \
    break;
  switch (nd) {
    GPTQ2D_KV_CASE(1)
    GPTQ2D_KV_CASE(2)
    GPTQ2D_KV_CASE(3)
    GPTQ2D_KV_CASE(4)
  }
#undef GPTQ2D_KV_CASE
  return (int)hipGetLastError();
}

int run(bool back, int32_t type, const KvCache& c, const Rows& r, hipStream_t st) {
  const int nd = (c.dim + 63) / 64;
  switch (type) {
    case TYPE_F32:
      return launch<TYPE_F32>(back, c, r, nd, st);
    case TYPE_BF16:
      return launch<TYPE_BF16>(back, c, r, nd, st);
    case TYPE_F16:
      return launch<TYPE_F16>(back, c, r, nd, st);
  }
  return GPTQ2D_EINVAL;
}

}  // namespace

extern "C" {

int64_t gptq2d_kv_page_words(int32_t heads, int32_t dim, int32_t page) {
  if (heads < 1 || heads > 65535 || dim < 1 || dim > 256 || page < 32 || page > 4096 || page % 32) return -1;
  return heads * kv_head_words((dim + 63) / 64, page);
}

int gptq2d_kv_append(void* pages, int64_t page_count, int32_t heads, int32_t dim, int32_t page, const void* k,
                     int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head, int32_t type,
                     const int32_t* table, int64_t seqs, int64_t width, int64_t table_stride, const int32_t* lengths,
                     const int32_t* offsets, int64_t tokens, void* stream) {
  KvCache c;
  if (!make_cache(c, pages, page_count, heads, dim, page, table, seqs, width, table_stride, lengths, offsets, tokens))
    return GPTQ2D_EINVAL;
  if (tokens == 0 || seqs == 0 || width == 0 || page_count == 0) return 0;
  const Rows r = {const_cast<void*>(k), const_cast<void*>(v), k_token, k_head, v_token, v_head};
  return run(false, type, c, r, (hipStream_t)stream);
}

int gptq2d_kv_read(const void* pages, int64_t page_count, int32_t heads, int32_t dim, int32_t page, void* k,
                   int64_t k_token, int64_t k_head, void* v, int64_t v_token, int64_t v_head, int32_t type,
                   const int32_t* table, int64_t seqs, int64_t width, int64_t table_stride, const int32_t* lengths,
                   const int32_t* offsets, int64_t tokens, void* stream) {
  KvCache c;
  if (!make_cache(c, pages, page_count, heads, dim, page, table, seqs, width, table_stride, lengths, offsets, tokens))
    return GPTQ2D_EINVAL;
  if (tokens == 0) return 0;
  const Rows r = {k, v, k_token, k_head, v_token, v_head};
  return run(true, type, c, r, (hipStream_t)stream);
}

}  // extern "C"
