// Attention of new tokens over the 4-bit cache.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(t_ij - max_j t_ij) / sum_j exp(...),  t_ij = scale q_i . k_j
// over the keys j that query i sees: j <= position of i and, with a window, j > position - window.  A query that sees
// none gives zeros.  With k = (c - 8) s + (z + 8 s) (kv_cache.h) a score is s (q . (c - 8)) + (z + 8 s) sum q: the matrix
// cores multiply q by whole numbers and a key's two numbers are applied once to the sum.  Likewise
//   o = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (z_j + 8 s_j).
// Operands are fp16 and exact: codes by nature; a query is scaled by a power of two (its largest element to 2^14..2^15),
// which leaves every bf16 or fp16 element within 2^-38 of the largest as it is, and fp32 ones in two pieces of together 22
// bits.  p_j s_j is brought to fp16's range by a power of two above the largest s seen, and rounded to 11 bits for
// bf16 results (which have 8), in two pieces otherwise.  Sums, maxima and rescaling are fp32.
#include "kv_cache.h"

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
};

// What a workgroup's columns (token, query head of the group) are, and the blocks of 32 keys that they see.
struct Tile {
  int64_t b, row;  // first packed row of the sequence
  int col0, cols;  // first column, columns of the sequence
  int pos0;        // position of the sequence's first query
  int kb0, kb1;
  int pos_lo, pos_hi;  // least and largest position of a column
  int len;             // tokens that the sequence holds
  int chunks;          // workgroups that share the blocks
};

template <int CT>
__device__ __forceinline__ Tile make_tile(const KvCache& c, const Attend& a, int64_t b, int col0) {
  Tile t;
  t.b = b;
  const int64_t t0 = kv_offset(c, b), t1 = kv_offset(c, b + 1);
  t.row = t0;
  const int n = t1 > t0 ? (int)(t1 - t0) : 0;
  t.cols = n * a.group;
  t.col0 = col0;
  t.len = kv_length(c, b);
  t.pos0 = t.len - n;
  const int last = t.cols - 1 < col0 + CT - 1 ? t.cols - 1 : col0 + CT - 1;
  t.pos_lo = t.pos0 + col0 / a.group;
  t.pos_hi = t.pos0 + (last < 0 ? 0 : last) / a.group;
  const int first = a.window && t.pos_lo - a.window + 1 > 0 ? t.pos_lo - a.window + 1 : 0;
  t.kb0 = first / 32;
  t.kb1 = t.pos_hi < 0 ? t.kb0 : t.pos_hi / 32 + 1;
  if (t.kb1 < t.kb0) t.kb1 = t.kb0;
  t.chunks = t.kb1 - t.kb0 > a.chunk ? (t.kb1 - t.kb0 + a.chunk - 1) / a.chunk : 1;
  return t;
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

// A column's query as B operands, QP pieces; `factor` takes the products' sums back to scores, `sum` is the sum of what
// the operands hold.
template <int TYPE, int ND, int QP>
__device__ __forceinline__ void load_query(half8 (&q)[2 * ND][QP], float& factor, float& sum,
                                           const typename Elem<TYPE>::T* row, bool valid, int dim, int g, float scale) {
  float x[2 * ND][8];
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < 2 * ND; ++s) {
    if (valid) {
      load_row<TYPE, 8>(x[s], row, 32 * s + 8 * g, dim);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[s][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __builtin_fabsf(x[s][e]);
      top = v < __builtin_inff() && v > top ? v : top;  // infinities and NaN stay what they are in fp16
    }
  }
  top = quad_max(top);
  const int ex = exponent_of(top) - 14;
  float total = 0.f;
#pragma unroll
  for (int s = 0; s < 2 * ND; ++s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __builtin_ldexpf(x[s][e], -ex);
      const _Float16 h = (_Float16)v;
      q[s][0][e] = h;
      total += (float)h;
      if constexpr (QP == 2) {
        const _Float16 l = (_Float16)(v - (float)h);
        q[s][1][e] = l;
        total += (float)l;
      }
    }
  }
  sum = quad_sum(total);
  factor = __builtin_ldexpf(scale, ex);
}

// Running state of a wave's columns over its keys.
template <int ND, int NQ>
struct State {
  floatx4 o[NQ][4 * ND];  // elements 16 t + 4 g .. + 3 of column l % 16, times 2^(ROOM - shift)
  float top[NQ], l[NQ], z[NQ];  // maximum (all lanes of the column), this lane's sums of p and of p (z + 8 s)
  int shift;                    // p s is held as p s 2^-shift in fp16
};

// p s 2^(ROOM - shift) <= 2^ROOM in fp16: the smaller ones keep their 11 bits down to 2^-28 of that.
constexpr int ROOM = 14;

// One block of 32 keys: kw, vw its codes' words, ka, va its scales and zeros (key 16 t + 4 g + i of this lane).
template <int ND, int NQ, int QP, int PP, bool MASK>
__device__ __forceinline__ void attend_block(State<ND, NQ>& st, const half8 (&q)[NQ][2 * ND][QP], const float (&factor)[NQ],
                                             const float (&qsum)[NQ], const uint4v (&kw)[ND], const uint4v (&vw)[ND],
                                             const uint4v (&ka)[2], const uint4v (&va)[2], int key0, int len,
                                             const int (&pos)[NQ], int window) {
  floatx4 s[NQ][2];
#pragma unroll
  for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int W = 0; W < 4 * ND; ++W) {
    const half8 k = centred_codes(kw[W / 4][W % 4]);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int p = 0; p < QP; ++p) s[n][W / (2 * ND)] = mfma(k, q[n][W % (2 * ND)][p], s[n][W / (2 * ND)]);
  }
  float vs[8], vz[8];
  int big = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned w = va[i / 4][i % 4];
    if (MASK && key0 + 16 * (i / 4) + i % 4 >= len) w = 0;  // beyond the sequence: whatever the page holds
    const int ex = (int)(w >> 7 & 255u);
    if (ex != 255) big = ex > big ? ex : big;
    vs[i] = __uint_as_float(w << 16);
    vz[i] = __builtin_fmaf(8.f, vs[i], __uint_as_float(w & 0xffff0000u));
  }
  // a larger scale than any before: the sums so far move to its range (with room for twice four more)
  if (__builtin_amdgcn_ballot_w64(big - 126 > st.shift)) {
    int most = __shfl_xor(big, 16);
    most = most > big ? most : big;
    const int other = __shfl_xor(most, 32);
    most = most > other ? most : other;
    most = __builtin_amdgcn_readfirstlane(most) - 126 + 2;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int t = 0; t < 4 * ND; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[n][t][i] = __builtin_ldexpf(st.o[n][t][i], st.shift - most);
    st.shift = most;
  }
  half8 p[NQ][PP];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float t[8];
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned w = ka[i / 4][i % 4];
      const float ks = __uint_as_float(w << 16), kz = __builtin_fmaf(8.f, ks, __uint_as_float(w & 0xffff0000u));
      t[i] = __builtin_fmaf(ks, s[n][i / 4][i % 4], kz * qsum[n]) * factor[n];
      if constexpr (MASK) {
        const int key = key0 + 16 * (i / 4) + i % 4;
        if (key > pos[n] || (window && key <= pos[n] - window)) t[i] = -__builtin_inff();
      }
      top = t[i] > top || t[i] != t[i] ? t[i] : top;
    }
    {
      const float a = __shfl_xor(top, 16);
      top = a > top || a != a ? a : top;
      const float b = __shfl_xor(top, 32);
      top = b > top || b != b ? b : top;
    }
    if (__builtin_amdgcn_ballot_w64(top > st.top[n] || top != top)) {
      const float now = top > st.top[n] || top != top ? top : st.top[n];
      const float f = now == st.top[n] ? 1.f : __builtin_amdgcn_exp2f(st.top[n] - now);
      st.top[n] = now;
      st.l[n] *= f;
      st.z[n] *= f;
#pragma unroll
      for (int d = 0; d < 4 * ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[n][d][i] *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float w = __builtin_amdgcn_exp2f(t[i] - st.top[n]);
      float ps = __builtin_ldexpf(w * vs[i], ROOM - st.shift), pz = w * vz[i];
      if constexpr (MASK) {
        const bool hidden = t[i] == -__builtin_inff();
        w = hidden ? 0.f : w, ps = hidden ? 0.f : ps, pz = hidden ? 0.f : pz;
      }
      st.l[n] += w;
      st.z[n] += pz;
      const _Float16 h = (_Float16)ps;
      p[n][0][i] = h;
      if constexpr (PP == 2) p[n][1][i] = (_Float16)(ps - (float)h);
    }
  }
#pragma unroll
  for (int W = 0; W < 4 * ND; ++W) {
    const half8 v = centred_codes(vw[W / 4][W % 4]);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int r = 0; r < PP; ++r) st.o[n][W] = mfma(v, p[n][r], st.o[n][W]);
  }
}

template <int ND>
struct Words {
  uint4v kw[ND], vw[ND], ka[2], va[2];
};

template <int ND>
__device__ __forceinline__ void load_block(Words<ND>& w, const unsigned* base, int at, int page, int lane) {
  const unsigned* k = base + at * (256 * ND) + lane * 4;
  const unsigned* v = k + page * (8 * ND);
  const unsigned* ka = base + page * (16 * ND) + at * 32 + lane / 16 * 4;
  const unsigned* va = ka + page;
#pragma unroll
  for (int i = 0; i < ND; ++i) w.kw[i] = *reinterpret_cast<const uint4v*>(k + 256 * i);
#pragma unroll
  for (int t = 0; t < 2; ++t) w.ka[t] = *reinterpret_cast<const uint4v*>(ka + 16 * t);
#pragma unroll
  for (int i = 0; i < ND; ++i) w.vw[i] = *reinterpret_cast<const uint4v*>(v + 256 * i);
#pragma unroll
  for (int t = 0; t < 2; ++t) w.va[t] = *reinterpret_cast<const uint4v*>(va + 16 * t);
}

// A workgroup takes 16 NQ columns and `chunk` blocks of 32 keys, its waves every fourth block each, the next block's
// words in flight while one is computed; the waves' results are joined through LDS.
template <int TYPE, int ND, int NQ>
__global__ __launch_bounds__(THREADS, ND * NQ <= 2 ? 2 : 1) void attend_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int CT = 16 * NQ, DP = 64 * ND, QP = TYPE == TYPE_F32 ? 2 : 1, PP = TYPE == TYPE_BF16 ? 1 : 2;
  __shared__ floatx4 sums[NQ][4 * ND][64];
  __shared__ float tops[WAVES][CT], ls[WAVES][CT];
  const int64_t slot = blockIdx.x;
  const int head = blockIdx.y, chunk = blockIdx.z;
  const int64_t seq = kv_find(c, slot, a.group, CT, 1);
  const int64_t col0 = (slot - kv_first_slot(c, seq, a.group, CT, 1)) * CT;
  if (col0 > 0x7fffff00) return;
  const Tile t = make_tile<CT>(c, a, seq, (int)col0);
  if (t.col0 >= t.cols || chunk >= t.chunks) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;

  half8 q[NQ][2 * ND][QP];
  float factor[NQ], qsum[NQ];
  int pos[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int col = t.col0 + 16 * n + (lane & 15), token = col / a.group, hq = head * a.group + col % a.group;
    const bool valid = col < t.cols;
    pos[n] = valid ? t.pos0 + token : t.pos_hi;
    load_query<TYPE, ND, QP>(q[n], factor[n], qsum[n],
                             (const T*)a.q + (t.row + token) * a.q_token + hq * a.q_head, valid, c.dim, g, a.scale);
  }
  State<ND, NQ> st;
  st.shift = -1000;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    st.top[n] = -__builtin_inff();
    st.l[n] = st.z[n] = 0.f;
#pragma unroll
    for (int d = 0; d < 4 * ND; ++d) st.o[n][d] = (floatx4){0.f, 0.f, 0.f, 0.f};
  }
  const int begin = __builtin_amdgcn_readfirstlane(t.kb0 + chunk * a.chunk);
  const int end = __builtin_amdgcn_readfirstlane(begin + a.chunk < t.kb1 ? begin + a.chunk : t.kb1);
  const int pos_lo = __builtin_amdgcn_readfirstlane(t.pos_lo), pos_hi = __builtin_amdgcn_readfirstlane(t.pos_hi);
  const int hw = (int)kv_head_words(ND, c.page);
  const int64_t b = t.b;
  Words<ND> cur;
  int at = 0;
  int kb = begin + wave;
  const unsigned* base = kb < end ? kv_head(c, b, kb, head, hw, at) : nullptr;
  if (base) load_block<ND>(cur, base, at, c.page, lane);
  int at2 = 0;
  const unsigned* next = kb + WAVES < end ? kv_head(c, b, kb + WAVES, head, hw, at2) : nullptr;
  for (; kb < end; kb += WAVES) {
    Words<ND> ahead;
    if (next) load_block<ND>(ahead, next, at2, c.page, lane);
    int at3 = 0;
    const unsigned* after = kb + 2 * WAVES < end ? kv_head(c, b, kb + 2 * WAVES, head, hw, at3) : nullptr;
    if (base) {
      const int key0 = kb * 32 + 4 * g;
      if (kb * 32 + 31 <= pos_lo && (!a.window || kb * 32 > pos_hi - a.window))
        attend_block<ND, NQ, QP, PP, false>(st, q, factor, qsum, cur.kw, cur.vw, cur.ka, cur.va, key0, t.len, pos, a.window);
      else
        attend_block<ND, NQ, QP, PP, true>(st, q, factor, qsum, cur.kw, cur.vw, cur.ka, cur.va, key0, t.len, pos, a.window);
    }
    cur = ahead;
    base = next;
    next = after;
    at2 = at3;
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    st.l[n] = quad_sum(st.l[n]);
    st.z[n] = quad_sum(st.z[n]);
    if (g == 0) {
      tops[wave][16 * n + lane] = st.top[n];
      ls[wave][16 * n + lane] = st.l[n];
    }
  }
  __syncthreads();
  float top[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float m = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float x = tops[w][16 * n + (lane & 15)];
      m = x > m || x != x ? x : m;
    }
    top[n] = m;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float x = tops[w][16 * n + (lane & 15)];
      sum += (x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(x - m)) * ls[w][16 * n + (lane & 15)];
    }
    l[n] = sum;
    const float f = st.top[n] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(st.top[n] - m);
#pragma unroll
    for (int d = 0; d < 4 * ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        st.o[n][d][i] = f * (__builtin_ldexpf(st.o[n][d][i], st.shift - ROOM) + st.z[n]);
  }
#pragma unroll
  for (int w = WAVES - 1; w > 0; --w) {
    if (wave == w) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int d = 0; d < 4 * ND; ++d)
          sums[n][d][lane] = w == WAVES - 1 ? st.o[n][d] : sums[n][d][lane] + st.o[n][d];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int in = 16 * n + (lane & 15), col = t.col0 + in;
    const bool valid = col < t.cols;
    if (t.chunks > 1) {
      float* out = a.part + ((slot * c.heads + head) * a.chunks + chunk) * (int64_t)(CT * (DP + 2));
#pragma unroll
      for (int d = 0; d < 4 * ND; ++d) {
        const floatx4 v = sums[n][d][lane] + st.o[n][d];
        if (valid) *reinterpret_cast<floatx4*>(out + in * DP + 16 * d + 4 * g) = v;
      }
      if (valid && g == 0) {
        out[CT * DP + in] = top[n];
        out[CT * (DP + 1) + in] = l[n];
      }
    } else {
      const int64_t row = t.row + col / a.group;
      const int hq = head * a.group + col % a.group;
      const float f = l[n] == 0.f ? 0.f : 1.f / l[n];
      T* out = (T*)a.out + row * a.out_token + hq * a.out_head;
#pragma unroll
      for (int d = 0; d < 4 * ND; ++d) {
        const floatx4 v = sums[n][d][lane] + st.o[n][d];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const typename Elem<TYPE>::T x = from_f32<TYPE>(f == 0.f ? 0.f : v[i] * f);
          if (valid && 16 * d + 4 * g + i < c.dim) out[16 * d + 4 * g + i] = x;
        }
      }
      if (valid && a.lse && g == 0)
        a.lse[row * (int64_t)(c.heads * a.group) + hq] = l[n] == 0.f ? -__builtin_inff() : (top[n] + __builtin_log2f(l[n])) * LN2;
    }
  }
}

// Joins the chunks' results: a wave a (token, query head), whose chunks are added in their order.
template <int TYPE, int ND, int NQ>
__global__ __launch_bounds__(THREADS) void join_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int CT = 16 * NQ, DP = 64 * ND;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = c.heads * a.group;
  if (item >= c.tokens * heads) return;
  const int64_t row = item / heads;
  const int hq = (int)(item - row * heads), head = hq / a.group;
  const int64_t seq = kv_find(c, row, 1, 1, 0);
  const int col = (int)(row - kv_offset(c, seq)) * a.group + hq % a.group;
  const Tile t = make_tile<CT>(c, a, seq, col / CT * CT);
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
#pragma unroll 4
  for (int i = 0; i < t.chunks; ++i) {
    const float* p = part + (int64_t)i * (CT * (DP + 2));
    const float x = p[CT * DP + in];
    const float f = x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(x - top);
    l += f * p[CT * (DP + 1) + in];
#pragma unroll
    for (int d = 0; d < ND; ++d) sum[d] += f * p[in * DP + 64 * d + lane];
  }
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
  int nq, nd, chunk, chunks;
  int64_t slots, part;  // part: floats of the partial results
};

inline Plan make_plan(int64_t tokens, int64_t seqs, int heads, int group, int dim, int64_t most, int64_t window) {
  Plan p;
  p.nd = (dim + 63) / 64;
  p.nq = p.nd > 2 || tokens * group <= 16 * seqs ? 1 : 2;
  const int ct = 16 * p.nq;
  p.slots = tokens * group / ct + seqs;
  int64_t range = most;
  if (window && window + ct < range) range = window + ct;
  const int64_t blocks = range / 32 + 2;
  const int64_t want = (blocks * p.slots * heads + 1023) / 1024;
  p.chunk = (int)(want < 4 ? 4 : want > 64 ? 64 : want);
  p.chunks = (int)((blocks + p.chunk - 1) / p.chunk);
  if (p.chunks <= 1) p.chunks = 1;
  p.part = p.chunks > 1 ? p.slots * heads * p.chunks * (int64_t)(ct * (64 * p.nd + 2)) : 0;
  return p;
}

template <int TYPE, int ND, int NQ>
int launch(const KvCache& c, const Attend& a, const Plan& p, hipStream_t st) {
  hipLaunchKernelGGL((attend_kernel<TYPE, ND, NQ>), dim3((unsigned)p.slots, (unsigned)c.heads, (unsigned)p.chunks),
                     dim3(THREADS), 0, st, c, a);
  if (p.chunks > 1)
    hipLaunchKernelGGL((join_kernel<TYPE, ND, NQ>), dim3((unsigned)cdiv(c.tokens * c.heads * a.group, WAVES)),
                       dim3(THREADS), 0, st, c, a);
  return (int)hipGetLastError();
}

template <int TYPE>
int launch_type(const KvCache& c, const Attend& a, const Plan& p, hipStream_t st) {
  switch (p.nd) {
    case 1:
      return p.nq == 1 ? launch<TYPE, 1, 1>(c, a, p, st) : launch<TYPE, 1, 2>(c, a, p, st);
    case 2:
      return p.nq == 1 ? launch<TYPE, 2, 1>(c, a, p, st) : launch<TYPE, 2, 2>(c, a, p, st);
    case 3:
      return launch<TYPE, 3, 1>(c, a, p, st);
    case 4:
      return launch<TYPE, 4, 1>(c, a, p, st);
  }
  return GPTQ2D_EINVAL;
}

bool attend_ok(int64_t tokens, int64_t seqs, int32_t heads, int32_t group, int32_t dim, int64_t most, int64_t window) {
  return tokens >= 0 && seqs >= 0 && heads >= 1 && group >= 1 && dim >= 1 && dim <= 256 && most >= 0 && window >= 0 &&
         tokens <= 0x7fffffff && seqs <= ((int64_t)1 << 24) && most < ((int64_t)1 << 29) && heads <= 65535 &&
         group <= 65535 && tokens * group < ((int64_t)1 << 31) && window <= 0x3fffffff;
}

}  // namespace

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
  if (!make_cache(c, pages, page_count, heads, dim, page, table, seqs, width, table_stride, lengths, offsets, tokens) ||
      !attend_ok(tokens, seqs, heads, group, dim, width * page, window))
    return GPTQ2D_EINVAL;
  if (tokens == 0 || seqs == 0) return 0;
  const Plan p = make_plan(tokens, seqs, heads, group, dim, width * page, window);
  if (p.slots > 0x7fffffff || p.chunks > 65535) return GPTQ2D_EUNSUPPORTED;
  if (work_bytes < 4 * p.part || (p.part && (!work || (uintptr_t)work % 16))) return GPTQ2D_ESCRATCH;
  Attend a;
  a.q = q, a.q_token = q_token, a.q_head = q_head;
  a.out = out, a.out_token = out_token, a.out_head = out_head;
  a.lse = lse;
  a.part = p.part ? (float*)work : nullptr;
  a.scale = (float)(scale * (double)LOG2E);
  a.group = group;
  a.window = (int)window;
  a.chunk = p.chunk, a.chunks = p.chunks;
  const hipStream_t st = (hipStream_t)stream;
  switch (type) {
    case TYPE_F32:
      return launch_type<TYPE_F32>(c, a, p, st);
    case TYPE_BF16:
      return launch_type<TYPE_BF16>(c, a, p, st);
    case TYPE_F16:
      return launch_type<TYPE_F16>(c, a, p, st);
  }
  return GPTQ2D_EINVAL;
}

}  // extern "C"
