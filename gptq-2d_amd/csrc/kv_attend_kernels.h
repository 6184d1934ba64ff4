// Attention of new tokens over the 4-bit cache.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(t_ij - max_j t_ij) / sum_j exp(...),  t_ij = scale q_i . k_j
// over the keys j that query i sees: j <= position of i and, with a window, j > position - window.  A query that sees
// none gives zeros.  With k = (c - 8) s + (z + 8 s) (kv_cache.h) a score is s (q . (c - 8)) + (z + 8 s) sum q: the matrix
// cores multiply q by whole numbers and a key's two numbers are applied once to the sum.  Likewise
//   o = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (z_j + 8 s_j).
// Operands are fp16.  Codes are exact; a query is scaled by a power of two, its largest finite element to 2^6..2^15, where fp16
// has steps of 2^-24 at the least: an element is held to 22 bits (fp32, in two pieces; those of bf16 and fp16 are all held),
// or to 2^-31 of the query's largest where that is coarser, below the rounding of the score's fp32 sum.  p_j s_j is brought to
// fp16's range by a power of two above the largest s seen (or, where the scales are far apart, p s: SPREAD), and rounded to 11
// bits for bf16 results (which have 8), in two pieces otherwise.  Sums, maxima and rescaling are fp32.
#pragma once

#include "kv_cache.h"
#include "lds_dma.h"

namespace {

constexpr int WAVES = 4, THREADS = 64 * WAVES;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Attend {
  const void* q;
  int64_t q_token, q_head;
  void* out;
  int64_t out_token, out_head;
  float* lse;  // [tokens, query heads], or none
  float* part;  // partial results, or none where one chunk holds all
  float scale;  // times log2 e
  int group;    // query heads of a kv head
  int window;   // 0: none
  int chunk;    // blocks of 32 keys that a workgroup takes
  int chunks;   // of the longest possible range
  const unsigned* seen;  // trees: bits of the nodes that each token sees, `words` of 32 a token
  const int32_t* at;     // and the token's position
  int words;
  int4* list;            // and of many sequences the pieces of the work,
  int pieces, parts;     // those of a head, and of its partial results, at most
};

// What a workgroup's columns (token, query head of the group) are, and the blocks of 32 keys that they see.
struct Tile {
  int64_t b, row;  // first packed row of the sequence
  int col0, cols;  // first column, columns of the sequence
  int pos0;        // position of the sequence's first query
  int kb0, kb1;
  int pos_lo, pos_hi;  // least and largest position of a column; they may lie past the tokens held
  int len;             // tokens that the sequence holds
  int chunks;          // workgroups that share the blocks
};

// Of a tree's nodes (TREE) all see what was held before (but for a window), and none a node past the bits that there are.
template <bool TREE>
__device__ __forceinline__ Tile make_tile(const KvCache& c, const Attend& a, int64_t b, int col0, int CT) {
  Tile t;
  t.b = b;
  const int64_t t0 = kv_offset(c, b), t1 = kv_offset(c, b + 1);
  t.row = t0;
  const int n = t1 > t0 ? (int)(t1 - t0) : 0;
  t.cols = n * a.group;
  t.col0 = col0;
  const int length = c.seqs && c.lengths[b] > 0 ? c.lengths[b] : 0, most = c.width * c.page;
  t.len = length < most ? length : most;  // the table may have no room for all: that bounds the keys, not the positions
  t.pos0 = length - n;
  const int last = t.cols - 1 < col0 + CT - 1 ? t.cols - 1 : col0 + CT - 1;
  if constexpr (TREE) {
    const int nodes = n < 32 * a.words ? n : 32 * a.words;
    t.pos_lo = t.pos0;
    t.pos_hi = t.pos0 + (nodes < 1 ? 0 : nodes - 1);
  } else {
    t.pos_lo = t.pos0 + col0 / a.group;
    t.pos_hi = t.pos0 + (last < 0 ? 0 : last) / a.group;
  }
  const int first = a.window && t.pos_lo - a.window + 1 > 0 ? t.pos_lo - a.window + 1 : 0;
  t.kb0 = first / 32;
  const int end = t.pos_hi < t.len ? t.pos_hi + 1 : t.len;  // of the keys that a column sees
  t.kb1 = end > 0 ? (end - 1) / 32 + 1 : t.kb0;
  if (t.kb1 < t.kb0) t.kb1 = t.kb0;
  t.chunks = t.kb1 - t.kb0 > a.chunk ? (t.kb1 - t.kb0 + a.chunk - 1) / a.chunk : 1;
  return t;
}

// Zeros (and an lse of -inf) in the rows that no sequence has: those of this slot before the first sequence, and those after
// the last one, as the columns (token, query head of the group) that would follow its own.
template <class T>
__device__ __forceinline__ void clear_rows(const KvCache& c, const Attend& a, int head, int64_t from, int64_t to) {
  for (int64_t u = from * c.dim + threadIdx.x; u < to * c.dim; u += blockDim.x) {
    const int64_t col = u / c.dim, row = col / a.group;
    const int d = (int)(u - col * c.dim), hq = head * a.group + (int)(col - row * a.group);
    ((T*)a.out)[row * a.out_token + hq * a.out_head + d] = (T)0;
    if (a.lse && d == 0) a.lse[row * (int64_t)(c.heads * a.group) + hq] = -__builtin_inff();
  }
}
template <class T>
__device__ __forceinline__ void clear_others(const KvCache& c, const Attend& a, int head, int64_t seq, int64_t slot, int64_t first,
                                             int CT) {
  if (!c.offsets || (seq > 0 && seq + 1 < c.seqs)) return;
  const int64_t before = kv_offset(c, 0) * a.group, after = kv_offset(c, c.seqs) * a.group, end = c.tokens * a.group;
  if (__builtin_expect(before == 0 && after == end, 1)) return;
  if (seq == 0) {
    const int64_t begin = slot * CT;
    clear_rows<T>(c, a, head, begin, begin + CT < before ? begin + CT : before);
  }
  if (seq + 1 >= c.seqs && slot >= first) {
    const int64_t begin = kv_offset(c, seq) * a.group + (slot - first) * CT;
    clear_rows<T>(c, a, head, begin > after ? begin : after, begin + CT < end ? begin + CT : end);
  }
}

// A column's position; in a tree the bits of the nodes that it sees, `words` of 32, the first one's position and theirs.
struct Column {
  int pos;
  const unsigned* seen;
  int words, first;
};

// The column of a token of the sequence (any of its columns where there is none: it is not written).
template <bool TREE>
__device__ __forceinline__ Column make_column(const Attend& a, const Tile& t, bool valid, int token) {
  Column c;
  if constexpr (TREE) {
    const int64_t row = t.row + (valid ? token : 0);
    c.pos = a.window ? a.at[row] : 0;
    c.seen = a.seen + row * a.words;
    c.words = a.words;
    c.first = t.pos0;
  } else {
    c.pos = valid ? t.pos0 + token : t.pos_hi;
  }
  return c;
}

// Partial results of (slot, head, chunk): CT columns of DP sums, then CT maxima, then CT sums of weights.

__device__ __forceinline__ float quad_sum(float x) {  // over the four lanes of a column
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

__device__ __forceinline__ floatx4 mfma(half8 a, half8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The queries of NQ x 16 columns as they lie, and each column's largest finite element (0 if it has none).
template <int TYPE, int ND, int NQ>
__device__ __forceinline__ void read_queries(Raw8<TYPE> (&x)[NQ][2 * ND], float (&top)[NQ],
                                             const typename Elem<TYPE>::T* const (&row)[NQ], const bool (&valid)[NQ], int dim) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int s = 0; s < 2 * ND; ++s) x[n][s].load(row[n], 32 * s + 8 * g, valid[n] ? dim : 0);
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    top[n] = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * ND; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_fabsf(x[n][s][e]);
        top[n] = v < __builtin_inff() && v > top[n] ? v : top[n];  // infinities and NaN stay what they are in fp16
      }
    top[n] = quad_max(top[n]);
  }
}

// Queries as B operands, QP pieces, column n times 2^-ex[n]; `sum` is the sum of what a column's operands hold.
template <int TYPE, int ND, int NQ, int QP>
__device__ __forceinline__ void query_operands(half8 (&q)[NQ][2 * ND][QP], float (&sum)[NQ], const Raw8<TYPE> (&x)[NQ][2 * ND],
                                               const int (&ex)[NQ]) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float total = 0.f;
#pragma unroll
    for (int s = 0; s < 2 * ND; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_ldexpf(x[n][s][e], -ex[n]);
        const _Float16 h = (_Float16)v;
        q[n][s][0][e] = h;
        total += (float)h;
        if constexpr (QP == 2) {
          const _Float16 l = (_Float16)(v - (float)h);
          q[n][s][1][e] = l;
          total += (float)l;
        }
      }
    }
    sum[n] = quad_sum(total);
  }
}

// Softmax over a wave's columns, a block of 32 keys at a time.  Bound by vector instructions, so a score takes few: its
// exponent is two fused multiply-adds off a reference that is the maximum of some block before, not of this one -- it moves
// when a score exceeds it by 2^AHEAD, which needs no maximum over the lanes to be seen --, then one each for the exponential,
// its product with the value's scale and the two sums, and half of one each for the comparison and the conversion.
constexpr int AHEAD = 8;  // log2 of how far weights may exceed 1
constexpr int ROOM = 7;   // weights times scales are held as p s 2^(ROOM - shift) <= 2^(ROOM + AHEAD) in fp16: s < 2^shift
// The shift is that of the largest scale seen, common to all columns, whatever little weight its key has.  What p s loses
// below fp16's steps, 2^(shift - 32), is 2^(spread - 32) of what the key of the largest weight adds at least, where no scale
// seen is below 2^(shift - spread).  Where one is, the columns part: each has the shift of the largest p s that it has seen
// (its sums are rescaled every block then: 2048 of 8192 tokens, every 50th value 2^16 times the others, 737 us instead of
// 384; 64 x up to 8000 143 us instead of 114).
template <int PP>
constexpr int SPREAD = PP == 1 ? 14 : 11;

template <int ND, int NQ>
struct State {
  floatx4 o[NQ][4 * ND];        // elements 16 t + 4 g .. + 3 of column l % 16, times 2^(ROOM - shift[n])
  float top[NQ], l[NQ], z[NQ];  // reference; this lane's sums of p and of p (z + 8 s)
  bool fresh[NQ];               // the column has not seen a key: its reference is still to be taken, however low
  int common, shift[NQ];
};

template <int ND, int NQ>
__device__ __forceinline__ void clear(State<ND, NQ>& st) {
  st.common = -1000;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    st.shift[n] = -1000;
    st.top[n] = st.l[n] = st.z[n] = 0.f;
    st.fresh[n] = true;
#pragma unroll
    for (int d = 0; d < 4 * ND; ++d) st.o[n][d] = (floatx4){0.f, 0.f, 0.f, 0.f};
  }
}

// Of the keys key0 .. key0 + 19 those that a tree's column sees: what was held before its nodes (with a window from `from` + 1 on),
// and the nodes that it comes from; keys from `len` on are no tokens.
__device__ __forceinline__ unsigned seen_bits(const Column& c, int key0, int from, int len) {
  const int node = key0 - c.first;  // of the first key
  unsigned bits = 0xffffffffu;
  if (node > -32) {
    const int w = node >> 5, shift = node & 31;  // below 0: from the word before the first one, whose keys all see
    const unsigned low = w < 0 ? 0xffffffffu : w < c.words ? c.seen[w] : 0u;
    const unsigned high = w + 1 < c.words ? c.seen[w + 1] : 0u;
    bits = (unsigned)(((uint64_t)high << 32 | low) >> shift);
  }
  const int hidden = from - key0 + 1, there = len - key0;
  bits = hidden > 0 ? (hidden < 32 ? bits >> hidden << hidden : 0u) : bits;
  return there < 32 ? (there > 0 ? bits & ((1u << there) - 1u) : 0u) : bits;
}

// Exponents e of a block's scores off the reference, and the sums so far brought to the values' new `shift` (apart: to the
// columns' own; vex(i) is the exponent of value i's scale) and, where a column's reference moves, to it -- in one place, so
// that the sums stay in their registers.  key0: this lane's first key
// (keys key0 + 16 (i / 4) + i % 4); len: tokens that the block's page can have (0 without a page); ks, kz: scales and
// zeros with what all columns share in them.
template <bool TREE, int ND, int NQ, class X>
__device__ __forceinline__ void exponents(State<ND, NQ>& st, float (&e)[NQ][8], const floatx4 (&s)[NQ][2], const float (&ks)[8],
                                          const float (&kz)[8], const float (&qsum)[NQ], bool mask, int key0,
                                          const Column (&col)[NQ], int window, int len, int shift, bool apart, X vex) {
  float most[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      e[n][i] = __builtin_fmaf(ks[i], s[n][i / 4][i % 4], __builtin_fmaf(kz[i], qsum[n], -st.top[n]));
  if (__builtin_expect(mask, 0)) {
    asm volatile("");  // a branch, not sixteen selects for every block
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int from = window ? col[n].pos - window : -1, to = col[n].pos < len ? col[n].pos : len - 1;
      unsigned bits = 0;
      if constexpr (TREE) bits = seen_bits(col[n], key0, from, len);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = 16 * (i / 4) + i % 4, key = key0 + at;
        const bool hidden = TREE ? !(bits >> at & 1u) : key > to || key <= from;
        e[n][i] = hidden ? -__builtin_inff() : e[n][i];
      }
    }
  }
  bool move = apart || shift != st.common;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    most[n] = e[n][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most[n] = fmaxf(most[n], e[n][i]);
    move |= most[n] > (st.fresh[n] ? -__builtin_inff() : (float)AHEAD);
  }
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(move) != 0, 0)) {
    st.common = shift;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float m = quad_max(most[n]);
      const float up = st.fresh[n] ? (m == -__builtin_inff() ? 0.f : m) : m > (float)AHEAD ? m : 0.f;
      const float f = st.fresh[n] ? 1.f : __builtin_amdgcn_exp2f(-up);  // sums of 0 stay, however far down it goes
#pragma unroll
      for (int i = 0; i < 8; ++i) e[n][i] -= up;
      int to = shift;
      if (apart) {
        float ps = -1000.f;  // at least the exponent of the largest p s; the sums' own goes down with the reference
#pragma unroll
        for (int i = 0; i < 8; ++i) ps = fmaxf(ps, e[n][i] + (float)vex(i));
        to = (int)__builtin_ceilf(fminf(quad_max(ps), 1000.f)) + ROOM - 15;
        const int was = st.shift[n] - (int)fminf(__builtin_floorf(up), 1000.f);
        to = was > to && !st.fresh[n] ? was : to;
      }
      const int less = st.fresh[n] ? 0 : st.shift[n] - to;  // sums of 0 need no factor, which may be infinite
      st.shift[n] = to;
      st.fresh[n] = st.fresh[n] && m == -__builtin_inff();
      st.top[n] += up;
      st.l[n] *= f;
      st.z[n] *= f;
      const float f2 = __builtin_ldexpf(f, less);
#pragma unroll
      for (int d = 0; d < 4 * ND; ++d) st.o[n][d] *= f2;
    }
  }
}

// The block's weights: p s as B operands in PP pieces, and the sums of p and p (z + 8 s).  shift: what the scales vs are held
// with, where that may not be the columns' (apart).
template <int ND, int NQ, int PP>
__device__ __forceinline__ void weights(State<ND, NQ>& st, half8 (&p)[NQ][PP], const float (&e)[NQ][8], const float (&vs)[8],
                                        const float (&vz)[8], bool mask, bool apart, int shift) {
  float ps[NQ][8];
  if (__builtin_expect(mask || apart, 0)) {  // a scale or zero that is no number must not reach columns that do not see its key
    asm volatile("");
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool hidden = e[n][i] == -__builtin_inff();
        const float w = __builtin_amdgcn_exp2f(e[n][i]), z = w * vz[i];
        ps[n][i] = hidden ? 0.f : __builtin_ldexpf(w * vs[i], apart ? shift - st.shift[n] : 0);
        st.l[n] += w;
        st.z[n] += hidden ? 0.f : z;
      }
  } else {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = __builtin_amdgcn_exp2f(e[n][i]);
        ps[n][i] = w * vs[i];
        st.l[n] += w;
        st.z[n] = __builtin_fmaf(w, vz[i], st.z[n]);
      }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const _Float16 h = (_Float16)ps[n][i];
      p[n][0][i] = h;
      if constexpr (PP == 2) p[n][1][i] = (_Float16)(ps[n][i] - (float)h);
    }
}

// The shift that admits the scales whose largest bits (of 32) this lane found to be `bits`: the present one where it does.
__device__ __forceinline__ int admit(int shift, int bits, const float (&s)[8]) {
  const int limit = shift < -126 ? 0 : (shift + 127) << 23;  // bits of 2^shift
  if (!__builtin_amdgcn_ballot_w64(bits >= limit)) return shift;
  int big = -126;
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // infinities and NaN apart
    const int ex = (int)(__float_as_uint(s[i]) >> 23 & 255u);
    big = ex != 255 && ex - 126 > big ? ex - 126 : big;
  }
  int x = __shfl_xor(big, 16);
  big = x > big ? x : big;
  x = __shfl_xor(big, 32);
  big = __builtin_amdgcn_readfirstlane(x > big ? x : big);
  return big > shift ? big + 2 : shift;  // with room for scales four times as large
}

template <int ND>
struct Words {
  uint4v kw[ND], vw[ND], ka[2], va[2];
};

// Scales and zeros of this lane's eight keys: s and z + 8 s.
__device__ __forceinline__ void unpack_affine(float (&s)[8], float (&z)[8], const uint4v (&w)[2]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned u = w[i / 4][i % 4];
    s[i] = __uint_as_float(u << 16);
    z[i] = __builtin_fmaf(8.f, s[i], __uint_as_float(u & 0xffff0000u));
  }
}

template <bool TREE, int ND, int QP, int PP>  // low: bits of the least scale that this lane has seen
__device__ __forceinline__ void attend_block(State<ND, 1>& st, const half8 (&q)[1][2 * ND][QP], const float (&qsum)[1],
                                             Words<ND>& w, float factor, bool mask, int key0, int len,
                                             const Column (&col)[1], int window, unsigned& low) {
  floatx4 s[1][2];
  s[0][0] = s[0][1] = (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4 * ND; ++i) {
    const int W = i / 2 + i % 2 * (2 * ND);  // the two tiles of keys in turn
    const half8 k = centred_codes(w.kw[W / 4][W % 4]);
#pragma unroll
    for (int p = 0; p < QP; ++p) s[0][i % 2] = mfma(k, q[0][i / 2][p], s[0][i % 2]);
  }
  float ks[8], kz[8], vs[8], vz[8], e[1][8];
  if (mask) {  // beyond the sequence: whatever the page holds
    asm volatile("");
#pragma unroll
    for (int i = 0; i < 8; ++i) w.va[i / 4][i % 4] = key0 + 16 * (i / 4) + i % 4 < len ? w.va[i / 4][i % 4] : FLAT;
  }
  unpack_affine(ks, kz, w.ka);
  unpack_affine(vs, vz, w.va);
  int bits = 0;  // the largest scale's (a NaN's is larger than any); and the least, whose bit of the sign no scale but FLAT's has
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned u = __float_as_uint(vs[i]);
    bits = (int)u > bits ? (int)u : bits;
    low = u < low ? u : low;
    ks[i] *= factor, kz[i] *= factor;
  }
  const int shift = admit(st.common, bits, vs), least = shift - SPREAD<PP>;
  const bool apart = __builtin_amdgcn_ballot_w64(low < (least < -126 ? 0u : (unsigned)(least + 127) << 23));
  exponents<TREE, ND, 1>(st, e, s, ks, kz, qsum, mask, key0, col, window, len, shift, apart,
                         [&](int i) { return (int)(__float_as_uint(vs[i]) >> 23 & 255u) - 126; });
#pragma unroll
  for (int i = 0; i < 8; ++i) vs[i] = __builtin_ldexpf(vs[i], ROOM - st.shift[0]);  // a lane has one column
  half8 p[1][PP];
  weights<ND, 1, PP>(st, p, e, vs, vz, mask, false, 0);
#pragma unroll
  for (int W = 0; W < 4 * ND; ++W) {
    const half8 v = centred_codes(w.vw[W / 4][W % 4]);
#pragma unroll
    for (int r = 0; r < PP; ++r) st.o[0][W] = mfma(v, p[0][r], st.o[0][W]);
  }
}

// A wave's ring of blocks in LDS, each loaded there straight from memory S - 1 blocks ahead: K's and V's words (1 KB a chunk, as the
// lanes read them), then the scales and zeros of 32 keys and 32 values.  Two workgroups of four waves a CU have some 100 KB
// on their way.
template <int ND>
struct Ring {
  static constexpr int STAGE = 2048 * ND + 256, LOADS = 2 * ND + 1;
  static constexpr int S = 20480 / STAGE < 8 ? 20480 / STAGE : 8;
};

// Waits until at most N of this wave's loads are on their way, and until its LDS reads have returned: the stage that they read
// is loaded next, and nothing else orders the two.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt has six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Block `at` of the head's part of a page at `base`; without a page zeros.
template <int ND>
__device__ __forceinline__ void stage_block(char* to, const unsigned* base, int at, int page, int lane) {
  const int words = base ? 1 : 0;
  const auto rsrc = [&](int first, int count) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned*>(base + (base ? first : 0)), (short)0, words * count * 4, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t k = rsrc(at * (256 * ND), 256 * ND), v = rsrc(page * (8 * ND) + at * (256 * ND), 256 * ND);
#pragma unroll
  for (int i = 0; i < ND; ++i) dma_load<4>(k, reinterpret_cast<float*>(to + 1024 * i), 1024 * i + 16 * lane);
#pragma unroll
  for (int i = 0; i < ND; ++i) dma_load<4>(v, reinterpret_cast<float*>(to + 1024 * (ND + i)), 1024 * i + 16 * lane);
  const __amdgpu_buffer_rsrc_t a = rsrc(page * (16 * ND) + at * 32, page + 32);
  dma_load<1>(a, reinterpret_cast<float*>(to + 2048 * ND), (lane < 32 ? lane : page + lane - 32) * 4);
}

template <int ND>
__device__ __forceinline__ void read_block(Words<ND>& w, const char* from, int lane) {
#pragma unroll
  for (int i = 0; i < ND; ++i) w.kw[i] = *reinterpret_cast<const uint4v*>(from + 1024 * i + 16 * lane);
#pragma unroll
  for (int i = 0; i < ND; ++i) w.vw[i] = *reinterpret_cast<const uint4v*>(from + 1024 * (ND + i) + 16 * lane);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    w.ka[t] = *reinterpret_cast<const uint4v*>(from + 2048 * ND + 64 * t + lane / 16 * 16);
    w.va[t] = *reinterpret_cast<const uint4v*>(from + 2048 * ND + 128 + 64 * t + lane / 16 * 16);
  }
}

// Few columns.  A workgroup takes 16 of them and `chunk` blocks of 32 keys, its waves every fourth block each; the waves'
// results are joined through LDS.  Bound by memory for long sequences: 4 of up to 131072 tokens, 8 kv heads of 128, bf16,
// one token each: 156 us, 3.6 TB/s of the cache (a read-only sum: 4.0); by the unequal lengths otherwise: 64 of 300 to 8000
// tokens 115 us, 2.5 TB/s.  Some 300 vector instructions a block and wave, most of them on the 32 keys' scales and codes,
// whatever the columns.  Two tiles of 16 columns a wave, which share them, need registers that leave half of the waves:
// 32 columns of 16 x 4000 tokens 95 us for 55 in two workgroups.
template <bool TREE, int TYPE, int ND>
__global__ __launch_bounds__(THREADS, ND <= 2 ? 2 : 1) void attend_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int CT = 16, DP = 64 * ND, QP = TYPE == TYPE_F32 ? 2 : 1, PP = TYPE == TYPE_BF16 ? 1 : 2;
  typedef Ring<ND> R;
  constexpr int S = R::S;
  static_assert(S * R::STAGE >= 4 * ND * 1024, "a wave's sums fit where its blocks were");
  alignas(16) __shared__ char ring[WAVES][S][R::STAGE];
  __shared__ float tops[WAVES][CT], ls[WAVES][CT];
  const int64_t slot = blockIdx.x;
  const int head = blockIdx.y, chunk = blockIdx.z;
  const int64_t seq = kv_find(c, slot, a.group, CT, 1);
  const int64_t first_slot = kv_first_slot(c, seq, a.group, CT, 1), col0 = (slot - first_slot) * CT;
  if (chunk == 0) clear_others<T>(c, a, head, seq, slot, first_slot, CT);
  if (col0 < 0 || col0 > 0x7fffff00) return;
  const Tile t = make_tile<TREE>(c, a, seq, (int)col0, CT);
  if (t.col0 >= t.cols || chunk >= t.chunks) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;

  const int begin = __builtin_amdgcn_readfirstlane(t.kb0 + chunk * a.chunk);
  const int end = __builtin_amdgcn_readfirstlane(begin + a.chunk < t.kb1 ? begin + a.chunk : t.kb1);
  // all columns see the keys in [all_from, all_to]
  const int all_to = __builtin_amdgcn_readfirstlane((t.pos_lo < t.len ? t.pos_lo : t.len) - (TREE || t.pos_lo >= t.len));
  const int all_from = __builtin_amdgcn_readfirstlane(a.window ? t.pos_hi - a.window + 1 : 0);
  const int hw = (int)kv_head_words(ND, c.page);
  const int64_t b = t.b;
  const int first = begin + wave, count = end > first ? (end - first + WAVES - 1) / WAVES : 0;
  unsigned there = 0;  // bit per stage: the block has a page
  int at = 0;
  const unsigned* base = nullptr;
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < count) {
      base = kv_head(c, b, first + WAVES * i, head, hw, at);
      there |= (base ? 1u : 0u) << i;
      stage_block<ND>(ring[wave][i], base, at, c.page, lane);
    }
  base = S - 1 < count ? kv_head(c, b, first + WAVES * (S - 1), head, hw, at) : nullptr;
  half8 q[1][2 * ND][QP];
  const int col = t.col0 + (lane & 15), token = col / a.group, hq = head * a.group + col % a.group;
  const bool valid[1] = {col < t.cols};
  const Column place[1] = {make_column<TREE>(a, t, valid[0], token)};
  const T* const rows[1] = {(const T*)a.q + (t.row + (valid[0] ? token : 0)) * a.q_token + hq * a.q_head};
  Raw8<TYPE> x[1][2 * ND];
  float top[1], qsum[1];
  read_queries<TYPE, ND, 1>(x, top, rows, valid, c.dim);
  const int ex[1] = {exponent_of(top[0]) - 14};
  query_operands<TYPE, ND, 1, QP>(q, qsum, x, ex);
  const float factor = __builtin_ldexpf(a.scale, ex[0]);  // of the lane's column
  State<ND, 1> st;
  clear(st);
  unsigned low = 0xffffffffu;
  int buf = 0;
  for (int i = 0; i < count; ++i) {
    if (i + S - 1 <= count)
      wait_loads<(S - 2) * R::LOADS>();
    else
      wait_loads<0>();
    const int ahead = buf ? buf - 1 : S - 1;
    if (i + S - 1 < count) {
      there = (there & ~(1u << ahead)) | (base ? 1u : 0u) << ahead;
      stage_block<ND>(ring[wave][ahead], base, at, c.page, lane);
      if (i + S < count) base = kv_head(c, b, first + WAVES * (i + S), head, hw, at);
    }
    Words<ND> w;
    read_block<ND>(w, ring[wave][buf], lane);
    const int kb = first + WAVES * i;
    const bool page = there >> buf & 1u;
    const bool mask = !page || kb * 32 + 31 > all_to || kb * 32 < all_from;
    attend_block<TREE, ND, QP, PP>(st, q, qsum, w, factor, mask, kb * 32 + 4 * g, page ? t.len : 0, place, a.window, low);
    buf = buf + 1 < S ? buf + 1 : 0;
  }
  // the waves' results, brought to one reference, in the place of their own blocks; then every thread adds four elements
  st.l[0] = quad_sum(st.l[0]);
  st.z[0] = quad_sum(st.z[0]);
  if (st.fresh[0] && st.l[0] == 0.f) st.top[0] = -__builtin_inff();  // saw no key; scores that are no numbers stay such
  if (g == 0) {
    tops[wave][lane] = st.top[0];
    ls[wave][lane] = st.l[0];
  }
  __syncthreads();
  floatx4* const mine = reinterpret_cast<floatx4*>(&ring[wave][0][0]);
  float m = -__builtin_inff();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) m = fmaxf(m, tops[w][lane & 15]);
  const float f = st.top[0] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(st.top[0] - m);
  const float f2 = __builtin_ldexpf(f, st.shift[0] - ROOM), z = f * st.z[0];
#pragma unroll
  for (int d = 0; d < 4 * ND; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) st.o[0][d][i] = __builtin_fmaf(f2, st.o[0][d][i], z);
    mine[d * 64 + lane] = st.o[0][d];
  }
  __syncthreads();
  const int cols = t.cols - t.col0 < CT ? t.cols - t.col0 : CT;
  for (int u = threadIdx.x; u < cols * (16 * ND); u += THREADS) {
    const int in = u / (16 * ND), d4 = u % (16 * ND);  // column, four elements
    const int at4 = d4 / 4 * 64 + in + 16 * (d4 % 4);
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    float top = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      v += reinterpret_cast<const floatx4*>(&ring[w][0][0])[at4];
      top = fmaxf(top, tops[w][in]);
    }
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      l += (tops[w][in] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(tops[w][in] - top)) * ls[w][in];
    const bool none = top == -__builtin_inff();
    if (t.chunks > 1) {
      float* out = a.part + ((slot * c.heads + head) * a.chunks + chunk) * (int64_t)(CT * (DP + 2));
      *reinterpret_cast<floatx4*>(out + in * DP + 4 * d4) = v;
      if (d4 == 0) out[CT * DP + in] = top;
      if (d4 == 1) out[CT * (DP + 1) + in] = l;
    } else {
      const int col = t.col0 + in;
      const int64_t row = t.row + col / a.group;
      const int hq = head * a.group + col % a.group;
      const float f = none ? 0.f : 1.f / l;
      T* out = (T*)a.out + row * a.out_token + hq * a.out_head + 4 * d4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T x = from_f32<TYPE>(none ? 0.f : v[i] * f);
        if (4 * d4 + i < c.dim) out[i] = x;
      }
      if (d4 == 0 && a.lse)
        a.lse[row * (int64_t)(c.heads * a.group) + hq] = none ? -__builtin_inff() : (top + __builtin_log2f(l)) * LN2;
    }
  }
}

// Many columns (a prompt's tokens times the heads that share a kv head).  A workgroup takes 32 columns a wave and `chunk` blocks of
// 32 keys; the block's codes are brought to fp16 once, by all waves, into LDS, where they lie as operands (two blocks in
// turn, one barrier a block; the next one's words are in flight meanwhile), and its scales and zeros in fp32 with what all
// columns share already in them.  2048 new tokens of 8192, 32 heads on 8 of 128, bf16: 384 us, 627 TFLOP/s of 240 GFLOP.
// Bound by the two waves a SIMD that its 222 registers allow: of 2050 cycles a block and wave 512 are matrix and about 1000
// vector instructions', one after the other.  64 columns a wave spill (591 us); the next block's scores beside this one's
// weights, which needs half as much LDS again, took 408.
constexpr int PQ = 2, PWAVES = 4;  // columns of a wave: 16 PQ
constexpr int EVEN = 8;            // leaves an element 2^-31 of its own query's largest

template <bool TREE, int ND, int QP, int PP>
__device__ __forceinline__ void prompt_block(State<ND, PQ>& st, const half8 (&q)[PQ][2 * ND][QP], const float (&qsum)[PQ],
                                             const half8 (*kop)[64], const half8 (*vop)[64], const float (*aff)[32], bool mask,
                                             int key0, const Column (&col)[PQ], int window, int len, int shift, bool apart,
                                             bool uneven, int downs) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  floatx4 s[PQ][2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int n = 0; n < PQ; ++n) s[n][t] = (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * ND; ++i) {
      const half8 k = kop[2 * ND * t + i][lane];
#pragma unroll
      for (int n = 0; n < PQ; ++n)
#pragma unroll
        for (int p = 0; p < QP; ++p) s[n][t] = mfma(k, q[n][i][p], s[n][t]);
    }
  }
  float a0[8], a1[8], e[PQ][8];
  auto read = [&](float (&x)[8], int i) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const floatx4 v = *reinterpret_cast<const floatx4*>(&aff[i][16 * t + 4 * g]);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * t + j] = v[j];
    }
  };
  read(a0, 0);
  read(a1, 1);
  if (__builtin_expect(uneven, 0)) {
    asm volatile("" : "+v"(downs));  // a branch, and both exponents in one register outside it
#pragma unroll
    for (int n = 0; n < PQ; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[n][i / 4][i % 4] = __builtin_ldexpf(s[n][i / 4][i % 4], (int16_t)(downs >> 16 * n));
  }
  exponents<TREE, ND, PQ>(st, e, s, a0, a1, qsum, mask, key0, col, window, len, shift, apart, [&](int i) {
    const float x = aff[2][16 * (i / 4) + 4 * g + i % 4];  // s 2^(ROOM - shift)
    return x > 0.f ? exponent_of(x) + 1 - ROOM + shift : -1000;
  });
  half8 p[PQ][PP];
  read(a0, 2);
  read(a1, 3);
  weights<ND, PQ, PP>(st, p, e, a0, a1, mask, apart, shift);
#pragma unroll
  for (int W = 0; W < 4 * ND; ++W) {
    const half8 v = vop[W][lane];
#pragma unroll
    for (int n = 0; n < PQ; ++n)
#pragma unroll
      for (int r = 0; r < PP; ++r) st.o[n][W] = mfma(v, p[n][r], st.o[n][W]);
  }
}

template <bool TREE, int TYPE, int ND>
__global__ __launch_bounds__(64 * PWAVES, ND <= 2 ? 2 : 1) void prompt_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int CT = 16 * PQ * PWAVES, DP = 64 * ND, QP = TYPE == TYPE_F32 ? 2 : 1, PP = TYPE == TYPE_BF16 ? 1 : 2;
  constexpr int CH = (2 * ND + PWAVES - 1) / PWAVES;  // chunks of 1 KB of words of a block that a wave brings
  __shared__ half8 ops[2][8 * ND][64];                // K's operands, then V's
  __shared__ float aff[2][4][32];                     // scale and zero of keys (times what scores share), of values
  __shared__ int shifts[2];  // and whether columns part in the lowest bit
  __shared__ float tops[PWAVES];
  const int head = blockIdx.x, chunk = blockIdx.z;
  const int64_t slot = blockIdx.y + (int64_t)gridDim.y * (blockIdx.z / a.chunks);
  const int part = chunk % a.chunks;
  const int64_t seq = kv_find(c, slot, a.group, CT, 1);
  const int64_t first = kv_first_slot(c, seq, a.group, CT, 1);
  if (part == 0) clear_others<T>(c, a, head, seq, slot, first, CT);
  if (slot < first || (slot - first) * CT > 0x7fffff00) return;
  const Tile t = make_tile<TREE>(c, a, seq, (int)((slot - first) * CT), CT);
  if (t.col0 >= t.cols || part >= t.chunks) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;

  Column place[PQ];
  int row_of[PQ], head_of[PQ];
  bool valid[PQ];
  const T* rows[PQ];
  half8 q[PQ][2 * ND][QP];
  float qsum[PQ];
#pragma unroll
  for (int n = 0; n < PQ; ++n) {
    const int col = t.col0 + 16 * (PQ * wave + n) + (lane & 15), token = col / a.group;
    valid[n] = col < t.cols;
    place[n] = make_column<TREE>(a, t, valid[n], token);
    row_of[n] = token, head_of[n] = head * a.group + col % a.group;
    rows[n] = (const T*)a.q + (t.row + (valid[n] ? token : 0)) * a.q_token + head_of[n] * a.q_head;
  }
  // One exponent for all columns of the workgroup, which the keys' scales in LDS then hold; a wave with a column whose largest
  // element is 2^EVEN below the largest of all gives each its own, and takes its scores to the common one.
  Raw8<TYPE> x[PQ][2 * ND];
  float top[PQ];
  int ex[PQ], down[PQ];
  read_queries<TYPE, ND, PQ>(x, top, rows, valid, c.dim);
  float most = top[0];
#pragma unroll
  for (int n = 1; n < PQ; ++n) most = fmaxf(most, top[n]);
#pragma unroll
  for (int s = 1; s < 16; s *= 2) most = fmaxf(most, __shfl_xor(most, s));
  if (lane == 0) tops[wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < PWAVES; ++w) most = fmaxf(most, tops[w]);
  const int common = __builtin_amdgcn_readfirstlane(exponent_of(most) - 14);
  bool low = false;
#pragma unroll
  for (int n = 0; n < PQ; ++n) {
    down[n] = top[n] > 0.f ? exponent_of(top[n]) - 14 - common : 0;
    low |= down[n] < -EVEN;
  }
  const bool uneven = __builtin_amdgcn_ballot_w64(low);
#pragma unroll
  for (int n = 0; n < PQ; ++n) {
    down[n] = uneven ? down[n] : 0;
    ex[n] = common + down[n];
  }
  query_operands<TYPE, ND, PQ, QP>(q, qsum, x, ex);
#pragma unroll
  for (int n = 0; n < PQ; ++n) qsum[n] = __builtin_ldexpf(qsum[n], down[n]);
  static_assert(PQ == 2, "two columns' exponents in one register");
  const int downs = (down[0] & 0xffff) | down[1] << 16;
  const float factor = __builtin_ldexpf(a.scale, common);
  State<ND, PQ> st;
  clear(st);
  const int begin = __builtin_amdgcn_readfirstlane(t.kb0 + part * a.chunk);
  const int end = __builtin_amdgcn_readfirstlane(begin + a.chunk < t.kb1 ? begin + a.chunk : t.kb1);
  // all columns see the keys in [all_from, all_to]
  const int all_to = __builtin_amdgcn_readfirstlane((t.pos_lo < t.len ? t.pos_lo : t.len) - (TREE || t.pos_lo >= t.len));
  const int all_from = __builtin_amdgcn_readfirstlane(a.window ? t.pos_hi - a.window + 1 : 0);
  const int hw = (int)kv_head_words(ND, c.page), len = t.len;
  const int64_t b = t.b;
  uint4v words[CH];
  unsigned affine = 0;
  int held = -1000, least = -1000;  // the shift that values are staged with; no scale seen is below 2^least
  auto load = [&](const unsigned* base, int at) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int ch = wave + PWAVES * i;  // K's chunks, then V's
      if (ch < 2 * ND)
        words[i] = *reinterpret_cast<const uint4v*>(base + (ch < ND ? 0 : c.page * (8 * ND)) + at * (256 * ND) +
                                                    (ch < ND ? ch : ch - ND) * 256 + lane * 4);
    }
    if (wave == 0) affine = base[c.page * (16 * ND + (lane >> 5)) + at * 32 + (lane & 31)];
  };
  auto put = [&](int kb, int buf, const unsigned* page) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int ch = wave + PWAVES * i;
      if (ch < 2 * ND) {
#pragma unroll
        for (int w = 0; w < 4; ++w) ops[buf][4 * ch + w][lane] = centred_codes(words[i][w]);
      }
    }
    if (wave == 0) {  // lanes 0..31 the keys, 32..63 the values
      unsigned w = page && kb * 32 + (lane & 31) < len ? affine : FLAT;  // beyond the sequence: whatever the page holds
      const float s = __uint_as_float(w << 16), z = __builtin_fmaf(8.f, s, __uint_as_float(w & 0xffff0000u));
      const bool real = lane >= 32 && s > 0.f && s < __builtin_inff();  // -0, infinities and NaN are of no matter
      const int ex = real ? exponent_of(s) + 1 : held;                  // s in [2^(ex - 1), 2^ex), subnormal or not
      if (__builtin_amdgcn_ballot_w64((unsigned)(held - ex) >= (unsigned)(held - least))) {
        int big = real ? ex : -1000, low = real ? ex : 1000;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const int x = __shfl_xor(big, d), y = __shfl_xor(low, d);
          big = x > big ? x : big;
          low = y < low ? y : low;
        }
        big = __builtin_amdgcn_readfirstlane(big), low = __builtin_amdgcn_readfirstlane(low);
        if (big > -1000) {
          least = held == -1000 || low <= least ? low - 2 : least;  // room for half the least scale
          held = big > held ? big + 2 : held;                       // and for four times the largest
        }
      }
      aff[buf][lane >> 5 << 1][lane & 31] = lane < 32 ? s * factor : __builtin_ldexpf(s, ROOM - held);
      aff[buf][(lane >> 5 << 1) + 1][lane & 31] = lane < 32 ? z * factor : z;
      if (lane == 0) shifts[buf] = 2 * held + (least < held - SPREAD<PP>);
    }
  };
  int at = 0, at2 = 0;
  const unsigned* base = begin < end ? kv_head(c, b, begin, head, hw, at) : nullptr;
  if (base) load(base, at);
  const unsigned* next = begin + 1 < end ? kv_head(c, b, begin + 1, head, hw, at2) : nullptr;
  if (begin < end) put(begin, 0, base);
  __syncthreads();
  for (int kb = begin; kb < end; ++kb) {
    const int buf = (kb - begin) & 1;
    if (next) load(next, at2);
    int at3 = 0;
    const unsigned* after = kb + 2 < end ? kv_head(c, b, kb + 2, head, hw, at3) : nullptr;
    const int staged = __builtin_amdgcn_readfirstlane(shifts[buf]), shift = staged >> 1;
    const bool apart = staged & 1;
    const bool mask = !base || kb * 32 + 31 > all_to || kb * 32 < all_from;
    prompt_block<TREE, ND, QP, PP>(st, q, qsum, ops[buf], ops[buf] + 4 * ND, aff[buf], mask, kb * 32 + 4 * g, place, a.window,
                             base ? len : 0, shift, apart, uneven, downs);
    if (kb + 1 < end) put(kb + 1, 1 - buf, next);
    __syncthreads();
    base = next, next = after, at2 = at3;
  }
#pragma unroll
  for (int n = 0; n < PQ; ++n) {
    const float l = quad_sum(st.l[n]), z = quad_sum(st.z[n]);
    const int in = 16 * (PQ * wave + n) + (lane & 15);
    const bool none = st.fresh[n] && l == 0.f;  // scores that are no numbers stay such
    if (t.chunks > 1) {
      float* out = a.part + ((slot * c.heads + head) * a.chunks + part) * (int64_t)(CT * (DP + 2));
#pragma unroll
      for (int d = 0; d < 4 * ND; ++d) {
        floatx4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_ldexpf(st.o[n][d][i], st.shift[n] - ROOM) + z;
        if (valid[n]) *reinterpret_cast<floatx4*>(out + in * DP + 16 * d + 4 * g) = v;
      }
      if (valid[n] && g == 0) {
        out[CT * DP + in] = none ? -__builtin_inff() : st.top[n];
        out[CT * (DP + 1) + in] = l;
      }
    } else {
      const int64_t row = t.row + row_of[n];
      const float f = none ? 0.f : 1.f / l;
      T* out = (T*)a.out + row * a.out_token + head_of[n] * a.out_head;
#pragma unroll
      for (int d = 0; d < 4 * ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = (__builtin_ldexpf(st.o[n][d][i], st.shift[n] - ROOM) + z) * f;
          const T x = from_f32<TYPE>(none ? 0.f : v);
          if (valid[n] && 16 * d + 4 * g + i < c.dim) out[16 * d + 4 * g + i] = x;
        }
      if (valid[n] && a.lse && g == 0)
        a.lse[row * (int64_t)(c.heads * a.group) + head_of[n]] = none ? -__builtin_inff() : (st.top[n] + __builtin_log2f(l)) * LN2;
    }
  }
}

// Joins the chunks' results: a wave a (token, query head), whose chunks are added in their order.  Bound by latency (4 to 7 us).
template <bool TREE, int TYPE, int ND>
__global__ __launch_bounds__(THREADS) void join_kernel(KvCache c, Attend a, int CT) {
  typedef typename Elem<TYPE>::T T;
  constexpr int DP = 64 * ND;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = c.heads * a.group;
  if (item >= c.tokens * heads) return;
  const int64_t row = item / heads;
  const int hq = (int)(item - row * heads), head = hq / a.group;
  const int64_t seq = kv_find(c, row, 1, 1, 0);
  if (row < kv_offset(c, seq) || row >= kv_offset(c, seq + 1)) return;  // no sequence's
  const int col = (int)(row - kv_offset(c, seq)) * a.group + hq % a.group;
  const Tile t = make_tile<TREE>(c, a, seq, col / CT * CT, CT);
  if (t.chunks <= 1) return;
  const int64_t slot = kv_first_slot(c, seq, a.group, CT, 1) + col / CT;
  const int in = col % CT;
  const float* part = a.part + (slot * c.heads + head) * (int64_t)a.chunks * (CT * (DP + 2));
  float top = -__builtin_inff();
  for (int i = lane; i < t.chunks; i += 64) {
    const float x = part[(int64_t)i * (CT * (DP + 2)) + CT * DP + in];
    top = x > top || x != x ? x : top;
  }
#pragma unroll
  for (int s = 1; s < 64; s *= 2) {
    const float x = __shfl_xor(top, s);
    top = x > top || x != x ? x : top;
  }
  float sum[ND], l = 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d) sum[d] = 0.f;
  for (int i0 = 0; i0 < t.chunks; i0 += 64) {  // a lane a chunk's weight, then the chunks' sums, U loads in flight
    constexpr int U = 16 / ND;
    const int n = t.chunks - i0 < 64 ? t.chunks - i0 : 64;
    const float* p = part + (int64_t)i0 * (CT * (DP + 2));
    float f = 0.f;
    if (lane < n) {
      const float* mine = p + (int64_t)lane * (CT * (DP + 2)) + CT * DP + in;
      const float x = mine[0];
      f = x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(x - top);
      l += f * mine[CT];
    }
    for (int i = 0; i < n; i += U) {
      float v[U][ND];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d)
          v[u][d] = p[(int64_t)(i + u < n ? i + u : n - 1) * (CT * (DP + 2)) + in * DP + 64 * d + lane];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = __shfl(f, i + u < n ? i + u : 0);
#pragma unroll
        for (int d = 0; d < ND; ++d) sum[d] += i + u < n ? w * v[u][d] : 0.f;
      }
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s *= 2) l += __shfl_xor(l, s);
  const float f = l == 0.f ? 0.f : 1.f / l;
  T* out = (T*)a.out + row * a.out_token + hq * a.out_head;
#pragma unroll
  for (int d = 0; d < ND; ++d)
    if (64 * d + lane < c.dim) out[64 * d + lane] = from_f32<TYPE>(f == 0.f ? 0.f : sum[d] * f);
  if (a.lse && lane == 0)
    a.lse[row * (int64_t)heads + hq] = l == 0.f ? -__builtin_inff() : (top + __builtin_log2f(l)) * LN2;
}

// How a call is split: columns of a workgroup and blocks of 32 keys of a chunk.
struct Plan {
  bool prompt;
  int nd, ct, chunk, chunks;  // ct: columns of a workgroup
  int64_t slots, part;  // part: floats of the partial results
  int64_t blocks;       // of the longest possible range
  int64_t turns;        // of 65532 slots, where they are not the grid's first axis

  void set_chunks(int heads) {
    chunks = (int)((blocks + chunk - 1) / chunk);
    if (chunks <= 1) chunks = 1;
    part = chunks > 1 ? slots * heads * chunks * (int64_t)(ct * (64 * nd + 2)) : 0;
    turns = (slots + 65531) / 65532;
  }
};

inline Plan make_plan(int64_t tokens, int64_t seqs, int heads, int group, int dim, int64_t most, int64_t window, int64_t nodes = 0) {
  Plan p;
  seqs += !seqs;
  p.nd = (dim + 63) / 64;
  const int64_t columns = tokens * group;
  // From 96 columns a sequence on, a workgroup that brings a block to fp16 once for 128 columns is ahead of workgroups that
  // each do so for their 16 (16 sequences of 4000, 8 kv heads of 128: 64 columns 93 against 90 us, 96 101 against 120, 256
  // 199 against 267).
  p.prompt = columns >= 96 * seqs;
  p.ct = p.prompt ? 16 * PQ * PWAVES : 16;
  p.slots = columns / p.ct + seqs;
  int64_t range = most;
  const int64_t span = nodes ? nodes : p.ct;  // positions of a workgroup's columns
  if (window && window + span < range) range = window + span;
  const int64_t blocks = p.blocks = range / 32 + 2;
  // Chunks as large as leave 768 workgroups, one and a half rounds of two a CU, so that sequences of different lengths end
  // together (one token each, us for 512, 768 and 1024: 64 sequences of up to 8000 tokens 135, 121, 119; 4 of 131072 179,
  // 159, 154; 64 of 4000 94, 86, 91; one of 100000 41, 49, 53); at least two blocks a wave, whose start takes longer than
  // that (one of 16000: 19 us, with one block a wave 29) -- one where that leaves fewer than 256 workgroups, all on the chip
  // at once, and the chunks are joined anyway (both kernels, 8 kv heads of 128, two and one: one of 300 13.1 and 12.2 us, of
  // 1000 13.7 and 12.2, of 2000 13.4 and 12.6, of 4000, 256 workgroups, 13.4 and 13.8; 4 of 200, unjoined, 11.9 and 13.0).
  const int64_t tiles = cdiv(columns, p.ct) > seqs ? cdiv(columns, p.ct) : seqs;  // that hold columns, about
  const int64_t want = cdiv(blocks * tiles * heads, 768);
  const bool few = range > 64 * WAVES && cdiv(blocks, WAVES) * tiles * heads < 256;
  const int64_t least = few ? WAVES : 2 * WAVES;
  if (!p.prompt)
    p.chunk = (int)(want < least ? least : want);
  else  // as many as fill the chip, no more: each writes its columns' sums
    p.chunk = (int)(p.slots * heads >= 256 ? blocks : want < 16 ? 16 : want);
  p.set_chunks(heads);
  return p;
}

template <bool TREE, int TYPE, int ND>
int launch(const KvCache& c, const Attend& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.slots, (unsigned)c.heads, (unsigned)p.chunks), block(THREADS);
  if (p.prompt) {  // heads first: the workgroups of one XCD (every eighth) then read few heads' keys and values
    hipLaunchKernelGGL((prompt_kernel<TREE, TYPE, ND>),
                       dim3((unsigned)c.heads, (unsigned)cdiv(p.slots, p.turns), (unsigned)(p.chunks * p.turns)),
                       dim3(64 * PWAVES), 0, st, c, a);
  } else {
    hipLaunchKernelGGL((attend_kernel<TREE, TYPE, ND>), grid, block, 0, st, c, a);
  }
  if (p.chunks > 1)
    hipLaunchKernelGGL((join_kernel<TREE, TYPE, ND>), dim3((unsigned)cdiv(c.tokens * c.heads * a.group, WAVES)), block, 0, st, c, a,
                       p.ct);
  return (int)hipGetLastError();
}

template <bool TREE, int TYPE>
int launch_type(const KvCache& c, const Attend& a, const Plan& p, hipStream_t st) {
  switch (p.nd) {
    case 1:
      return launch<TREE, TYPE, 1>(c, a, p, st);
    case 2:
      return launch<TREE, TYPE, 2>(c, a, p, st);
    case 3:
      return launch<TREE, TYPE, 3>(c, a, p, st);
    case 4:
      return launch<TREE, TYPE, 4>(c, a, p, st);
  }
  return GPTQ2D_EINVAL;
}

bool attend_ok(int64_t tokens, int64_t seqs, int32_t heads, int32_t group, int32_t dim, int64_t most, int64_t window) {
  return tokens >= 0 && seqs >= 0 && heads >= 1 && group >= 1 && dim >= 1 && dim <= 256 && most >= 0 && window >= 0 &&
         tokens <= 0x7fffffff && seqs <= ((int64_t)1 << 24) && most < ((int64_t)1 << 29) && heads <= 65535 &&
         group <= 65535 && tokens * group < ((int64_t)1 << 31) && window <= 0x3fffffff;
}

// The call's plan and operands in `a`; an error code where they do not do.  first_axis: the slots are the grid's.
inline int set_call(Attend& a, const Plan& p, bool first_axis, const void* q, int64_t q_token, int64_t q_head, int32_t group, double scale,
                    int64_t window, void* out, int64_t out_token, int64_t out_head, float* lse, void* work, int64_t work_bytes) {
  if (p.slots > 0x7fffffff || p.chunks * (first_axis ? 1 : p.turns) > 65535) return GPTQ2D_EUNSUPPORTED;
  if (work_bytes < 4 * p.part || (p.part && (!work || (uintptr_t)work % 16))) return GPTQ2D_ESCRATCH;
  a.q = q, a.q_token = q_token, a.q_head = q_head;
  a.out = out, a.out_token = out_token, a.out_head = out_head;
  a.lse = lse;
  a.part = p.part ? (float*)work : nullptr;
  a.scale = (float)(scale * (double)LOG2E);
  a.group = group;
  a.window = (int)window;
  a.chunk = p.chunk, a.chunks = p.chunks;
  return 0;
}

}  // namespace
