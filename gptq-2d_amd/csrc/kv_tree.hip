// Attention of trees of drafted tokens over the 4-bit cache: gptq2d_kv_attend's formula (kv_attend_kernels.h), each node seeing what
// was held before the nodes, the nodes that it comes from and itself.
#include "kv_attend_kernels.h"

namespace {

// Some columns a sequence (its nodes times the heads that share a kv head).  Bound by vector instructions, so they are shared or
// done without:
//   - two waves share a ring of blocks in LDS, each with 16 columns of its own: a block's words are brought to LDS once, some by
//     each, and its 64 scales and zeros are prepared by one of them, one block ahead, two blocks in turn;
//   - codes are not centred for bf16 (PLAIN): a nibble is an fp16 number as it lies, c 2^-24 or 16 c 2^-24 (subnormal), after one
//     mask: five instructions a word of eight, not nine.  The 16 is divided out of the other operand (of the queries' elements and
//     of the values' scales where e & 2), 2^24 out of the sums.  A key is then (q . c) s + z sum q and a value c s + z.  A query's
//     element is so held to 2^-27 of the largest where that is coarser, and the values' scales may lie 2^4 less apart.  The
//     matrix cores align products by the exponents that operands are written with, so such sums are good to some 17 bits (fp32
//     results measured 1e-5 off that way, 2e-5 with scores of 30; 1e-7 and 2e-6 with centred codes): eight bits finer than bf16,
//     not enough for fp16 and fp32.
// One barrier a block: after it, the stage that was read in the turn before is loaded again.  A workgroup has two rings, with
// every second block each, whose results are joined at the end; four workgroups a CU.
constexpr int COLS = 2, RINGS = 2, SWAVES = COLS * RINGS, SCT = 16 * COLS;  // waves of a ring, rings, columns of a workgroup

template <bool PLAIN>
__device__ __forceinline__ half8 codes_of(unsigned w) {
  if constexpr (!PLAIN) return centred_codes(w);
  union {
    half2v h[4];
    half8 v;
  } r;
  const unsigned x = w >> 8;
  r.h[0] = as_half2(w & 0x000f000fu);
  r.h[1] = as_half2(w & 0x00f000f0u);
  r.h[2] = as_half2(x & 0x000f000fu);
  r.h[3] = as_half2(x & 0x00f000f0u);
  return r.v;
}
// log2 of what a code is held times, and of the 16 of every second pair.
template <bool PLAIN>
constexpr int CODE = PLAIN ? -24 : 0;
template <bool PLAIN>
constexpr int FOLD = PLAIN ? 4 : 0;

template <int ND>
struct Shared {
  static constexpr int STAGE = 2048 * ND + 256, S = ND == 1 ? 6 : 4;  // stages of a ring: 35 KB a workgroup for heads of up to 128
  static constexpr int LOADS[COLS] = {ND + 1, ND};                    // of a stage, by each wave
};

// Until wave `ct`'s loads of the oldest stage on its way have landed, and wave 0's first one, of scales, of the next stage.
template <int ND>
__device__ __forceinline__ void wait_turn(int ct) {
  typedef Shared<ND> R;
  if (ct == 0)
    wait_loads<(R::S - 2) * R::LOADS[0] - 1>();
  else
    wait_loads<(R::S - 2) * R::LOADS[1]>();
}

// As query_operands, with the codes' 16 divided out.
template <bool PLAIN, int TYPE, int ND, int QP>
__device__ __forceinline__ void shared_operands(half8 (&q)[2 * ND][QP], float& sum, const Raw8<TYPE> (&x)[2 * ND], int ex) {
  float total = 0.f;
#pragma unroll
  for (int s = 0; s < 2 * ND; ++s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int fold = e & 2 ? FOLD<PLAIN> : 0;
      const float v = __builtin_ldexpf(x[s][e], -ex - fold), times = (float)(1 << fold);
      const _Float16 h = (_Float16)v;
      q[s][0][e] = h;
      total = __builtin_fmaf((float)h, times, total);
      if constexpr (QP == 2) {
        const _Float16 l = (_Float16)(v - (float)h);
        q[s][1][e] = l;
        total = __builtin_fmaf((float)l, times, total);
      }
    }
  }
  sum = quad_sum(total);
}

template <bool PLAIN, int ND, int QP, int PP>
__device__ __forceinline__ void shared_block(State<ND, 1>& st, const half8 (&q)[2 * ND][QP], const float (&qsum)[1],
                                             const char* stage, const float (*aff)[32], bool mask, int key0,
                                             const Column (&col)[1], int window, int len, int shift, bool apart, bool uneven,
                                             int down) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  floatx4 s[1][2];
  s[0][0] = s[0][1] = (floatx4){0.f, 0.f, 0.f, 0.f};
  {
    uint4v w[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) w[i] = *reinterpret_cast<const uint4v*>(stage + 1024 * i + 16 * lane);
#pragma unroll
    for (int i = 0; i < 4 * ND; ++i) {
      const int W = i / 2 + i % 2 * (2 * ND);  // the two tiles of keys in turn
      const half8 k = codes_of<PLAIN>(w[W / 4][W % 4]);
#pragma unroll
      for (int p = 0; p < QP; ++p) s[0][i % 2] = mfma(k, q[i / 2][p], s[0][i % 2]);
    }
  }
  float a0[8], a1[8], e[1][8];
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
    asm volatile("" : "+v"(down));  // a branch
#pragma unroll
    for (int i = 0; i < 8; ++i) s[0][i / 4][i % 4] = __builtin_ldexpf(s[0][i / 4][i % 4], down);
  }
  exponents<true, ND, 1>(st, e, s, a0, a1, qsum, mask, key0, col, window, len, shift, apart, [&](int i) {
    const float x = aff[2][16 * (i / 4) + 4 * g + i % 4];  // s 2^(ROOM - shift), less the codes' 16
    return x > 0.f ? exponent_of(x) + 1 - ROOM + shift + (i & 2 ? FOLD<PLAIN> : 0) : -1000;
  });
  half8 p[1][PP];
  read(a0, 2);
  read(a1, 3);
  weights<ND, 1, PP>(st, p, e, a0, a1, mask, apart, shift);
  uint4v w[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) w[i] = *reinterpret_cast<const uint4v*>(stage + 1024 * (ND + i) + 16 * lane);
#pragma unroll
  for (int W = 0; W < 4 * ND; ++W) {
    const half8 v = codes_of<PLAIN>(w[W / 4][W % 4]);
#pragma unroll
    for (int r = 0; r < PP; ++r) st.o[0][W] = mfma(v, p[0][r], st.o[0][W]);
  }
}

// The slot of a workgroup of grid (heads, a multiple of 4, ...).  Slots without columns come in patterns (every second one where a
// sequence's columns fill theirs), and neighbours are dealt to the XCD's parts in turn: a quarter of the slots each, or some parts
// would have nothing to do (64 sequences of 32 columns: 185 us, so 145).
__device__ __forceinline__ int64_t slot_of(int turn) {
  return (blockIdx.y & 3) * (gridDim.y >> 2) + (blockIdx.y >> 2) + (int64_t)gridDim.y * turn;
}

template <int TYPE, int ND>
__global__ __launch_bounds__(64 * SWAVES, ND <= 2 && TYPE != TYPE_F32 ? 4 : ND <= 2 ? 3 : 2) void shared_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  typedef Shared<ND> R;
  constexpr int CT = SCT, DP = 64 * ND, QP = TYPE == TYPE_F32 ? 2 : 1, PP = TYPE == TYPE_BF16 ? 1 : 2, S = R::S;
  constexpr bool PLAIN = TYPE == TYPE_BF16;
  alignas(16) __shared__ char ring[RINGS][S][R::STAGE];
  __shared__ float aff[RINGS][2][4][32];  // scale and zero of keys (times what scores share), of values
  __shared__ int shifts[RINGS][2];        // and whether columns part in the lowest bit
  __shared__ float tops[SWAVES][16], ls[COLS][16];
  static_assert(S * R::STAGE >= COLS * 4 * ND * 1024, "a ring's sums fit where its blocks were");
  // heads first: the workgroups of one XCD (every eighth) read few heads' keys and values
  const int head = blockIdx.x, part = blockIdx.z % a.chunks;
  const int64_t slot = slot_of(blockIdx.z / a.chunks);
  const int64_t seq = kv_find(c, slot, a.group, CT, 1);
  const int64_t first_slot = kv_first_slot(c, seq, a.group, CT, 1);
  if (part == 0) clear_others<T>(c, a, head, seq, slot, first_slot, CT);
  if (slot < first_slot || (slot - first_slot) * CT > 0x7fffff00) return;
  const Tile t = make_tile<true>(c, a, seq, (int)((slot - first_slot) * CT), CT);
  if (t.col0 >= t.cols || part >= t.chunks) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int mine = wave / COLS, ct = wave % COLS;  // the wave's ring, and its tile of columns
  const int begin = __builtin_amdgcn_readfirstlane(t.kb0 + part * a.chunk);
  const int end = __builtin_amdgcn_readfirstlane(begin + a.chunk < t.kb1 ? begin + a.chunk : t.kb1);
  // all columns see the keys in [all_from, all_to]
  const int all_to = __builtin_amdgcn_readfirstlane((t.pos_lo < t.len ? t.pos_lo : t.len) - 1);
  const int all_from = __builtin_amdgcn_readfirstlane(a.window ? t.pos_hi - a.window + 1 : 0);
  const int hw = (int)kv_head_words(ND, c.page), len = t.len;
  const int64_t b = t.b;
  const int first = begin + mine, count = end > first ? (end - first + RINGS - 1) / RINGS : 0;
  const int turns = end > begin ? (end - begin + RINGS - 1) / RINGS : 0;  // of the ring that has most

  unsigned there = 0;  // bit per stage: the block has a page
  auto load = [&](int stage, const unsigned* base, int at) {
    there = (there & ~(1u << stage)) | (base ? 1u : 0u) << stage;
    char* const to = ring[mine][stage];
    const auto rsrc = [&](int from, int words) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned*>(base + (base ? from : 0)), (short)0, base ? words * 4 : 0,
                                               0x00020000);
    };
    if (ct == 0)
      dma_load<1>(rsrc(c.page * (16 * ND) + at * 32, c.page + 32), reinterpret_cast<float*>(to + 2048 * ND),
                  (lane < 32 ? lane : c.page + lane - 32) * 4);
    const __amdgpu_buffer_rsrc_t k = rsrc(at * (256 * ND), 256 * ND), v = rsrc(c.page * (8 * ND) + at * (256 * ND), 256 * ND);
#pragma unroll
    for (int i = 0; i < 2 * ND; ++i)
      if (i % COLS == ct) dma_load<4>(i < ND ? k : v, reinterpret_cast<float*>(to + 1024 * i), 1024 * (i % ND) + 16 * lane);
  };
  int at = 0;
  const unsigned* base = nullptr;
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < count) {
      base = kv_head(c, b, first + RINGS * i, head, hw, at);
      load(i, base, at);
    }
  base = S - 1 < count ? kv_head(c, b, first + RINGS * (S - 1), head, hw, at) : nullptr;

  const int col = t.col0 + 16 * ct + (lane & 15), token = col / a.group, hq = head * a.group + col % a.group;
  const bool valid = col < t.cols, active = t.col0 + 16 * ct < t.cols;  // the lane has a column, the wave any
  const Column place[1] = {make_column<true>(a, t, valid, token)};
  const T* const rows[1] = {(const T*)a.q + (t.row + (valid ? token : 0)) * a.q_token + hq * a.q_head};
  // One exponent for all columns of the workgroup; a wave with a column whose largest element is 2^EVEN below the largest of all
  // gives each its own, and takes its scores to the common one.
  Raw8<TYPE> x[1][2 * ND];
  half8 q[2 * ND][QP];
  float top[1], qsum[1];
  read_queries<TYPE, ND, 1>(x, top, rows, {valid}, c.dim);
  float most = top[0];
#pragma unroll
  for (int s = 1; s < 16; s *= 2) most = fmaxf(most, __shfl_xor(most, s));
  if (lane == 0) tops[wave][0] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SWAVES; ++w) most = fmaxf(most, tops[w][0]);
  const int common = __builtin_amdgcn_readfirstlane(exponent_of(most) - 14);
  int down = top[0] > 0.f ? exponent_of(top[0]) - 14 - common : 0;
  const bool uneven = __builtin_amdgcn_ballot_w64(down < -EVEN);
  down = uneven ? down : 0;
  shared_operands<PLAIN, TYPE, ND, QP>(q, qsum[0], x[0], common + down);
  qsum[0] = __builtin_ldexpf(qsum[0], down);
  const float factor = __builtin_ldexpf(a.scale, common);
  State<ND, 1> st;
  clear(st);

  int held = -1000, least = -1000;  // the shift that values are staged with; no scale seen is below 2^least
  auto prepare = [&](int kb, int stage, int buf) {  // lanes 0..31 the keys, 32..63 the values
    const unsigned affine = *reinterpret_cast<const unsigned*>(ring[mine][stage] + 2048 * ND + 4 * lane);
    const unsigned w = (there >> stage & 1u) && kb * 32 + (lane & 31) < len ? affine : FLAT;  // beyond the sequence: whatever the page holds
    const float s = __uint_as_float(w << 16), zero = __uint_as_float(w & 0xffff0000u), z = PLAIN ? zero : __builtin_fmaf(8.f, s, zero);
    const unsigned bits = (w >> 7 & 255u) - 1;  // zeros, subnormal numbers, infinities and NaN are of no matter
    const bool real = lane >= 32 && bits < 254u;
    const int ex = real ? (int)bits - 125 : held;  // s in [2^(ex - 1), 2^ex)
    if (__builtin_amdgcn_ballot_w64((unsigned)(held - ex) >= (unsigned)(held - least))) {
      int big = real ? ex : -1000, low = real ? ex : 1000;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int u = __shfl_xor(big, d), v = __shfl_xor(low, d);
        big = u > big ? u : big;
        low = v < low ? v : low;
      }
      big = __builtin_amdgcn_readfirstlane(big), low = __builtin_amdgcn_readfirstlane(low);
      if (big > -1000) {
        least = held == -1000 || low <= least ? low - 2 : least;  // room for half the least scale
        held = big > held ? big + 2 : held;                       // and for four times the largest
      }
    }
    float(*const to)[32] = aff[mine][buf];
    to[lane >> 5 << 1][lane & 31] = lane < 32 ? __builtin_ldexpf(s * factor, -CODE<PLAIN>)
                                                  : __builtin_ldexpf(s, ROOM - held - (lane & 2 ? FOLD<PLAIN> : 0));
    to[(lane >> 5 << 1) + 1][lane & 31] = lane < 32 ? z * factor : z;
    if (lane == 0) shifts[mine][buf] = 2 * held + (least < held - SPREAD<PP> + FOLD<PLAIN>);
  };
  if (ct == 0 && count) {
    if (S - 1 <= count)
      wait_loads<(S - 1) * R::LOADS[0] - 1>();
    else
      wait_loads<0>();
    prepare(first, 0, 0);
  }
  int buf = 0;
  for (int i = 0; i < turns; ++i) {
    if (i + S - 1 <= count)
      wait_turn<ND>(ct);
    else
      wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int ahead = buf ? buf - 1 : S - 1, next = buf + 1 < S ? buf + 1 : 0;
    if (i + S - 1 < count) {
      load(ahead, base, at);
      if (i + S < count) base = kv_head(c, b, first + RINGS * (i + S), head, hw, at);
    }
    const int kb = first + RINGS * i;
    if (ct == 0 && i + 1 < count) prepare(kb + RINGS, next, 1 - i % 2);
    if (active && i < count) {
      const int staged = __builtin_amdgcn_readfirstlane(shifts[mine][i % 2]), shift = staged >> 1;
      const bool page = there >> buf & 1u;
      const bool mask = !page || kb * 32 + 31 > all_to || kb * 32 < all_from;
      shared_block<PLAIN, ND, QP, PP>(st, q, qsum, ring[mine][buf], aff[mine][i % 2], mask, kb * 32 + 4 * g, place, a.window,
                               page ? len : 0, shift, staged & 1, uneven, down);
    }
    buf = next;
  }
  // the second ring's results go through LDS, where its blocks were, and are brought to one reference with the first one's
  float l = quad_sum(st.l[0]), m = st.top[0];
  const float z = quad_sum(st.z[0]);
  if (st.fresh[0] && l == 0.f) m = -__builtin_inff();  // saw no key; scores that are no numbers stay such
#pragma unroll
  for (int d = 0; d < 4 * ND; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) st.o[0][d][i] = __builtin_ldexpf(st.o[0][d][i], st.shift[0] - ROOM - CODE<PLAIN>) + z;
  floatx4* const other = reinterpret_cast<floatx4*>(&ring[1][0][0]) + ct * (4 * ND * 64);
  __syncthreads();
  if (mine == 1) {
#pragma unroll
    for (int d = 0; d < 4 * ND; ++d) other[d * 64 + lane] = st.o[0][d];
    if (g == 0) tops[ct][lane] = m, ls[ct][lane] = l;
  }
  __syncthreads();
  if (mine == 1 || !valid) return;
  {
    const float m0 = m, m1 = tops[ct][lane & 15];
    m = m0 > m1 || m0 != m0 ? m0 : m1;
    const float f0 = m0 == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m0 - m);
    const float f1 = m1 == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
#pragma unroll
    for (int d = 0; d < 4 * ND; ++d) st.o[0][d] = st.o[0][d] * f0 + other[d * 64 + lane] * f1;
    l = l * f0 + ls[ct][lane & 15] * f1;
  }
  const bool none = m == -__builtin_inff();
  const int in = 16 * ct + (lane & 15);
  if (t.chunks > 1) {
    float* out = a.part + ((slot * c.heads + head) * a.chunks + part) * (int64_t)(CT * (DP + 2));
#pragma unroll
    for (int d = 0; d < 4 * ND; ++d) *reinterpret_cast<floatx4*>(out + in * DP + 16 * d + 4 * g) = st.o[0][d];
    if (g == 0) {
      out[CT * DP + in] = m;
      out[CT * (DP + 1) + in] = l;
    }
  } else {
    const int64_t row = t.row + token;
    const float f = none ? 0.f : 1.f / l;
    T* out = (T*)a.out + row * a.out_token + hq * a.out_head;
#pragma unroll
    for (int d = 0; d < 4 * ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T x = from_f32<TYPE>(none ? 0.f : st.o[0][d][i] * f);
        if (16 * d + 4 * g + i < c.dim) out[16 * d + 4 * g + i] = x;
      }
    if (a.lse && g == 0)
      a.lse[row * (int64_t)(c.heads * a.group) + hq] = none ? -__builtin_inff() : (m + __builtin_log2f(l)) * LN2;
  }
}

// Joins the chunks' results of shared_kernel: a workgroup a slot and head, its 32 columns at once, so that what is looked up (the
// sequence, its chunks, their maxima) is looked up once.  64 sequences of 8 nodes, 32 heads of 128, up to 6 chunks: 9 us (a wave
// a column, as join_kernel, 19).
template <int TYPE, int ND>
__global__ __launch_bounds__(THREADS) void join_tile_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int CT = SCT, DP = 64 * ND, SIZE = CT * (DP + 2), PER = THREADS / CT, ITEMS = CT * 16 * ND / THREADS, PIECE = 32;
  __shared__ float factors[PIECE][CT], tops[CT], sums[CT];
  const int head = blockIdx.x;
  const int64_t slot = slot_of(blockIdx.z);
  const int64_t seq = kv_find(c, slot, a.group, CT, 1), first_slot = kv_first_slot(c, seq, a.group, CT, 1);
  if (slot < first_slot || (slot - first_slot) * CT > 0x7fffff00) return;
  const Tile t = make_tile<true>(c, a, seq, (int)((slot - first_slot) * CT), CT);
  if (t.col0 >= t.cols || t.chunks <= 1) return;
  const float* part = a.part + (slot * c.heads + head) * (int64_t)a.chunks * SIZE;
  const int cols = t.cols - t.col0 < CT ? t.cols - t.col0 : CT;
  // the largest of each column's references, by PER threads
  const int col = threadIdx.x / PER, j = threadIdx.x % PER;
  const float* mine = part + CT * DP + (col < cols ? col : 0);
  float top = -__builtin_inff(), l = 0.f;
  for (int i = j; i < t.chunks; i += PER) {
    const float x = mine[(int64_t)i * SIZE];
    top = x > top || x != x ? x : top;
  }
#pragma unroll
  for (int s = 1; s < PER; s *= 2) {
    const float x = __shfl_xor(top, s);
    top = x > top || x != x ? x : top;
  }
  floatx4 sum[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) sum[k] = (floatx4){0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < t.chunks; i0 += PIECE) {
    const int n = t.chunks - i0 < PIECE ? t.chunks - i0 : PIECE;
    for (int i = j; i < n; i += PER) {
      const float* at = mine + (int64_t)(i0 + i) * SIZE;
      const float x = at[0], f = x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(x - top);
      l += f * at[CT];
      factors[i][col] = f;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const floatx4* from = reinterpret_cast<const floatx4*>(part + (int64_t)(i0 + i) * SIZE);
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {  // columns past the sequence's are not written: the first one's in their place
        const int u = threadIdx.x + THREADS * k, in = u / (16 * ND);
        sum[k] += factors[i][in] * from[in < cols ? u : u % (16 * ND)];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int s = 1; s < PER; s *= 2) l += __shfl_xor(l, s);
  if (j == 0) tops[col] = top, sums[col] = l;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int u = threadIdx.x + THREADS * k, in = u / (16 * ND), d = 4 * (u % (16 * ND));
    if (in >= cols) continue;
    const int at = t.col0 + in, hq = head * a.group + at % a.group;
    const int64_t row = t.row + at / a.group;
    const float total = sums[in], f = total == 0.f ? 0.f : 1.f / total;
    T* out = (T*)a.out + row * a.out_token + hq * a.out_head + d;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < c.dim) out[i] = from_f32<TYPE>(f == 0.f ? 0.f : sum[k][i] * f);
    if (a.lse && d == 0)
      a.lse[row * (int64_t)(c.heads * a.group) + hq] = total == 0.f ? -__builtin_inff() : (tops[in] + __builtin_log2f(total)) * LN2;
  }
}

// How a call is split: by attend_kernel or prompt_kernel as gptq2d_kv_attend's, or by shared_kernel.
struct TreePlan : Plan {
  bool shared;
};

inline TreePlan make_tree_plan(int64_t tokens, int64_t seqs, int heads, int group, int dim, int64_t most, int64_t window,
                               int64_t nodes) {
  TreePlan p;
  static_cast<Plan&>(p) = make_plan(tokens, seqs, heads, group, dim, most, window, nodes);
  seqs += !seqs;
  const int64_t columns = tokens * group, tiles = cdiv(columns, SCT) > seqs ? cdiv(columns, SCT) : seqs;
  const int64_t total = p.blocks * tiles * heads;
  // Fewer blocks than workgroups of shared_kernel fit at once: the call is its start, which attend_kernel's waves, each alone,
  // do sooner (8 kv heads of 128, 4 heads each, us of both kernels and the join, attend and shared: 7 nodes of one sequence of
  // 100 tokens 10 and 15, of 1000 14 and 15, of 4000 16 and 22; of 4 of 1000 19 and 18, of 32 of 300 36 and 29, of 16 of 4000 55
  // and 45).  From 384 columns a sequence on prompt_kernel, which brings codes to fp16 once for 128 columns (prompt and shared:
  // 16 x 4000, 512 columns 209 and 313; one of 8000, 512 columns 53 and 67; 4 x 30000, 256 columns 252 and 256; 64 of up to 8000,
  // 256 columns 635 and 569, 128 columns 567 and 344).
  p.shared = total >= 1024 && columns < 384 * seqs;
  if (!p.shared) return p;
  p.prompt = false;
  p.ct = SCT;
  p.slots = columns / SCT + seqs;
  // Three rounds of four workgroups a CU, or chunks of 24 blocks, whose starts and joining take longer than uneven ends, or one
  // round; two blocks a ring at least.
  const int64_t thirds = cdiv(total, 3072), once = cdiv(total, 1024), least = once < 24 ? once : 24;
  p.chunk = (int)(thirds > least ? thirds : least < 4 ? 4 : least);
  p.set_chunks(heads);
  return p;
}

template <int TYPE, int ND>
int launch_shared(const KvCache& c, const Attend& a, const TreePlan& p, hipStream_t st) {
  const dim3 grid((unsigned)c.heads, (unsigned)(4 * cdiv(p.slots, 4 * p.turns)), (unsigned)(p.chunks * p.turns));
  hipLaunchKernelGGL((shared_kernel<TYPE, ND>), grid, dim3(64 * SWAVES), 0, st, c, a);
  if (p.chunks > 1)
    hipLaunchKernelGGL((join_tile_kernel<TYPE, ND>), dim3(grid.x, grid.y, (unsigned)p.turns),
                       dim3(THREADS), 0, st, c, a);
  return (int)hipGetLastError();
}

template <int TYPE>
int launch_tree(const KvCache& c, const Attend& a, const TreePlan& p, hipStream_t st) {
  if (!p.shared) return launch_type<true, TYPE>(c, a, p, st);
  switch (p.nd) {
    case 1:
      return launch_shared<TYPE, 1>(c, a, p, st);
    case 2:
      return launch_shared<TYPE, 2>(c, a, p, st);
    case 3:
      return launch_shared<TYPE, 3>(c, a, p, st);
    case 4:
      return launch_shared<TYPE, 4>(c, a, p, st);
  }
  return GPTQ2D_EINVAL;
}

bool tree_ok(int64_t nodes, int64_t window) {
  return nodes >= 1 && nodes <= 512 && (window == 0 || window >= nodes);
}

}  // namespace

extern "C" {

int64_t gptq2d_kv_attend_tree_workspace(int64_t tokens, int64_t seqs, int32_t heads, int32_t group, int32_t dim, int64_t most,
                                        int64_t window, int64_t nodes) {
  if (!attend_ok(tokens, seqs, heads, group, dim, most, window) || !tree_ok(nodes, window)) return -1;
  return 4 * make_tree_plan(tokens, seqs, heads, group, dim, most, window, (nodes + 31) / 32 * 32).part;
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
  const int64_t most = (int64_t)c.width * c.page;
  if (!attend_ok(tokens, seqs, heads, group, dim, most, window)) return GPTQ2D_EINVAL;
  if (tokens == 0) return 0;
  Attend a = {};
  a.seen = ancestors, a.at = positions, a.words = (int)((nodes + 31) / 32);
  const TreePlan p = make_tree_plan(tokens, seqs, heads, group, dim, most, window, 32 * (int64_t)a.words);
  const int rc = set_call(a, p, !p.prompt && !p.shared, q, q_token, q_head, group, scale, window, out, out_token, out_head, lse, work, work_bytes);
  if (rc) return rc;
  switch (type) {
    case TYPE_F32:
      return launch_tree<TYPE_F32>(c, a, p, (hipStream_t)stream);
    case TYPE_BF16:
      return launch_tree<TYPE_BF16>(c, a, p, (hipStream_t)stream);
    case TYPE_F16:
      return launch_tree<TYPE_F16>(c, a, p, (hipStream_t)stream);
  }
  return GPTQ2D_EINVAL;
}

}  // extern "C"
