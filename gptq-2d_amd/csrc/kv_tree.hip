// Attention of trees of drafted tokens over the 4-bit cache: gptq2d_kv_attend's formula (kv_attend_kernels.h), each node seeing what
// was held before the nodes, the nodes that it comes from and itself.
#include "kv_attend_kernels.h"

namespace {

// Some columns a sequence (its nodes times the heads that share a kv head).  Bound by vector instructions, so they are shared: two
// waves share a ring of blocks in LDS, each with 16 columns of its own.  A block's words are brought to LDS once, some by each,
// and its 64 scales and zeros are prepared by one of them, one block ahead, two blocks in turn.  Operands are attend_kernel's.
// One barrier a block: after it, the stage that was read in the turn before is loaded again.  A workgroup has two rings, with
// every second block each, whose results are joined at the end; four workgroups a CU.
// Of up to 16 columns a sequence a ring has one wave (COLS): 64 sequences of 2 nodes and up to 8000 tokens 99 us (with two, one of
// them without columns, 111), 100 of 4 nodes and 1000 51 (60).
constexpr int RINGS = 2;

template <int ND, int COLS>
struct Shared {
  static constexpr int STAGE = 2048 * ND + 256, S = ND == 1 ? 6 : 4;  // stages of a ring: 35 KB a workgroup for heads of up to 128
  static constexpr int LOADS[2] = {COLS == 2 ? ND + 1 : 2 * ND + 1, ND};  // of a stage, by each wave
};

// Until wave `ct`'s loads of the oldest stage on its way have landed, and wave 0's first one, of scales, of the next stage.
template <int ND, int COLS>
__device__ __forceinline__ void wait_turn(int ct) {
  typedef Shared<ND, COLS> R;
  if (COLS == 1 || ct == 0)
    wait_loads<(R::S - 2) * R::LOADS[0] - 1>();
  else
    wait_loads<(R::S - 2) * R::LOADS[1]>();
}

template <int ND, int QP, int PP>
__device__ __forceinline__ void shared_block(State<ND, 1>& st, const half8 (&q)[1][2 * ND][QP], const float (&qsum)[1],
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
      const half8 k = centred_codes(w[W / 4][W % 4]);
#pragma unroll
      for (int p = 0; p < QP; ++p) s[0][i % 2] = mfma(k, q[0][i / 2][p], s[0][i % 2]);
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
    const float x = aff[2][16 * (i / 4) + 4 * g + i % 4];  // s 2^(ROOM - shift)
    return x > 0.f ? exponent_of(x) + 1 - ROOM + shift : -1000;
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
    const half8 v = centred_codes(w[W / 4][W % 4]);
#pragma unroll
    for (int r = 0; r < PP; ++r) st.o[0][W] = mfma(v, p[0][r], st.o[0][W]);
  }
}

// How a call's work is dealt.  A sequence has a tile for every CT (32 or 16) of its columns, and its keys are cut into as many
// chunks as the lengths that there are make right, whatever the table has room for (chunks made for a table's room, four times the
// longest of 64 sequences: half as long again); a piece is a chunk of a tile.  Pieces lie side by side, a chunk's tiles next to each
// other, and the workgroups without one behind them: neighbours are dealt to an XCD's shader engines in turn, and engines without
// work are what pieces that may or may not be there lead to (every second one of no columns: 1.7 times the time; 64 empty sequences
// behind 64 others: 1.4).  Up to 64 sequences every workgroup looks at all of them, a lane each, and finds its own piece; more are
// looked at by one workgroup beforehand, which lists the pieces (some 5 us a call; done by every workgroup, 256 sequences take 1.4
// times as long, 4096 13 times).
struct Work {
  bool any;
  int tile, tiles, chunk, chunks;  // of the sequence: the tile, how many; the chunk, how many
  int first;                       // the sequence's first partial result, where it has some (chunks)
  int idle;                        // none: how many of these are before this one
  Tile t;
};

// Three rounds of the workgroups that fit at once.  Of less work than makes chunks of 32 blocks so, whose starts and joining take
// longer than uneven ends, half a round, of still less chunks of 8 or a quarter of a round; two blocks a ring at least (a round:
// 32 sequences of 300 tokens, 7 nodes, 32 heads of 128, 26 us, so 21, 32 of 1000 36 and 34).  `total`: blocks of all tiles and heads.
constexpr int ROUND = 1024;  // four a CU
__device__ __forceinline__ int chunk_size(float total) {
  const int thirds = 1 + (int)(total * (1.0001f / (3 * ROUND))), half = (int)(total * (2.f / ROUND));
  const int few = half < 2 ? 4 : half < 4 ? 2 * half : 8, least = half < few ? few : half < 32 ? half : 32;
  return thirds > least ? thirds : least;
}
// A head's blocks are so this many chunks at most, its pieces as many and the tiles, and those of tiles of two chunks or more
// (of 3/4 of the size at least) 4/3 of it.
inline int64_t most_chunks(int heads) { return 3 * ROUND / heads + 1; }

// The sum of the lanes up to this one.
template <class N>
__device__ __forceinline__ N lanes_before(N x) {
#define STEP(dpp, rows)                                                                                              \
  {                                                                                                                  \
    union { N n; int i; } u, v;                                                                                      \
    u.n = x;                                                                                                         \
    v.i = __builtin_amdgcn_update_dpp(0, u.i, dpp, rows, 0xf, false);                                                \
    x += v.n;                                                                                                        \
  }
  STEP(0x111, 0xf)  // from 1, 2, 4, 8 lanes before in a row of 16
  STEP(0x112, 0xf)
  STEP(0x114, 0xf)
  STEP(0x118, 0xf)
  STEP(0x142, 0xa)  // a row's last lane to the next row
  STEP(0x143, 0xc)  // the first half's to the second
#undef STEP
  return x;
}

struct Shape {
  Tile t;
  int tiles, blocks, chunks;
  __device__ __forceinline__ Shape(const KvCache& c, const Attend& a, int64_t b, int CT) {
    const bool valid = b < c.seqs;
    t = make_tile<true>(c, a, valid ? b : 0, 0, CT);
    tiles = valid ? (int)(((int64_t)t.cols + CT - 1) / CT) : 0;
    blocks = valid ? t.kb1 - t.kb0 : 0;
  }
  __device__ __forceinline__ float work() const { return (float)tiles * (float)blocks; }
  // some `size` blocks a chunk: up to half as many again where it is one
  __device__ __forceinline__ void cut(int size) { chunks = 2 * blocks >= 3 * size ? (2 * blocks + size) / (2 * size) : 1; }
  __device__ __forceinline__ int pieces() const { return tiles * chunks; }
  __device__ __forceinline__ int parts() const { return chunks > 1 ? tiles * chunks : 0; }
};

// The list: int4 {blocks of a chunk, pieces, tiles}, then {sequence, tile, chunk, the sequence's first partial result} for
// a.pieces pieces, then the same for the tiles.
constexpr int LISTING = 1024;
__global__ __launch_bounds__(LISTING) void list_kernel(KvCache c, Attend a, int most_tiles, int CT) {
  constexpr int WAVES = LISTING / 64;
  __shared__ float works[WAVES];
  __shared__ int sums[3][WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float work = 0.f;
  for (int64_t b = threadIdx.x; b < c.seqs; b += LISTING) work += Shape(c, a, b, CT).work();
  work = lanes_before(work);
  if (lane == 63) works[wave] = work;
  __syncthreads();
  float total = 0.f;
  for (int w = 0; w < WAVES; ++w) total += works[w];
  const int size = chunk_size(total * (float)c.heads);
  int4 *const piece_at = a.list + 1, *const tile_at = piece_at + a.pieces;
  int before[3] = {0, 0, 0};  // pieces, tiles, partial results of the sequences before these
  for (int64_t b0 = 0; b0 < c.seqs; b0 += LISTING) {
    Shape s(c, a, b0 + threadIdx.x, CT);
    s.cut(size);
    const int count[3] = {s.pieces(), s.tiles, s.parts()};
    int first[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      first[i] = lanes_before(count[i]);
      if (lane == 63) sums[i][wave] = first[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      first[i] += before[i] - count[i];
      for (int w = 0; w < WAVES; ++w) {
        const int n = sums[i][w];
        first[i] += w < wave ? n : 0;
        before[i] += n;
      }
    }
    const int seq = (int)(b0 + threadIdx.x);
    // none past the list's ends, where offsets that do not ascend would lead
    for (int i = 0; i < s.tiles && (unsigned)(first[1] + i) < (unsigned)most_tiles; ++i)
      tile_at[first[1] + i] = make_int4(seq, i, 0, first[2]);
    for (int k = 0, at = first[0]; k < s.chunks; ++k)
      for (int i = 0; i < s.tiles && (unsigned)at < (unsigned)a.pieces; ++i, ++at) piece_at[at] = make_int4(seq, i, k, first[2]);
    __syncthreads();
  }
  if (threadIdx.x == 0)
    *a.list = make_int4(size, before[0] < a.pieces ? before[0] : a.pieces, before[1] < most_tiles ? before[1] : most_tiles, 0);
}

// Piece number `at`, or (of_tiles) tile number `at`.
template <bool of_tiles, int CT>
__device__ __forceinline__ Work find_work(const KvCache& c, const Attend& a, int at) {
  Work w;
  if (a.list) {
    const int4 head = *a.list;
    w.idle = at - head.y;
    w.any = at < (of_tiles ? head.z : head.y);
    if (!w.any) return w;
    const int4 mine = a.list[1 + at + (of_tiles ? a.pieces : 0)];
    Shape s(c, a, mine.x, CT);
    s.cut(head.x);
    w.t = s.t, w.t.col0 = CT * mine.y;
    w.tile = mine.y, w.chunk = mine.z, w.first = mine.w, w.tiles = s.tiles, w.chunks = s.chunks;
    return w;
  }
  Shape s(c, a, threadIdx.x & 63, CT);
  const int size = chunk_size(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(lanes_before(s.work())), 63)) * (float)c.heads);
  s.cut(size);
  const int count = of_tiles ? s.tiles : s.pieces(), to = lanes_before(count), from = to - count;
  const int first = lanes_before(s.parts()) - s.parts();
  const uint64_t here = __builtin_amdgcn_ballot_w64(from <= at && at < to);
  w.any = here != 0;
  w.idle = at - __builtin_amdgcn_readlane(to, 63);
  if (!w.any) return w;
  const int l = __builtin_ctzll(here);
  const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
  w.tiles = of(s.tiles), w.chunks = of(s.chunks), w.first = of(first);
  const int in = at - of(from);
  w.chunk = of_tiles ? 0 : in / w.tiles;
  w.tile = of_tiles ? in : in - w.chunk * w.tiles;
  w.t.b = l;
  w.t.row = (int64_t)((uint64_t)(unsigned)of((int)(s.t.row >> 32)) << 32 | (unsigned)of((int)s.t.row));
  w.t.col0 = CT * w.tile, w.t.cols = of(s.t.cols), w.t.pos0 = of(s.t.pos0);
  w.t.kb0 = of(s.t.kb0), w.t.kb1 = of(s.t.kb1), w.t.pos_lo = of(s.t.pos_lo), w.t.pos_hi = of(s.t.pos_hi), w.t.len = of(s.t.len);
  return w;
}

// Zeros (and an lse of -inf) in the rows that no sequence has, of one head, by the workgroups without a piece.
template <class T>
__device__ __forceinline__ void clear_idle(const KvCache& c, const Attend& a, int head, int idle, int idles) {
  const int64_t before = kv_offset(c, 0), after = c.seqs ? kv_offset(c, c.seqs) : before;
  if (__builtin_expect(before == 0 && after == c.tokens && c.seqs, 1)) return;
  const int64_t from = c.seqs ? after : 0, end = c.seqs ? before : 0;  // [0, end) and [from, tokens)
  const int64_t rows = end + c.tokens - from, per = (rows + idles - 1) / idles;
  for (int64_t u = idle * per; u < (idle + 1) * per && u < rows; ++u) {
    const int64_t row = u < end ? u : from + u - end;
    clear_rows<T>(c, a, head, row * a.group, (row + 1) * a.group);
  }
}

// (Workgroups a CU as registers are dealt: with one column tile four, as there is LDS for, made the compiler move sums to and fro,
// 104 us for 99 with 64 sequences of 2 nodes.)
template <int TYPE, int ND, int COLS>
__global__ __launch_bounds__(64 * COLS * RINGS, COLS == 1 ? 2 : ND <= 2 && TYPE != TYPE_F32 ? 4 : ND <= 2 ? 3 : 2) void
shared_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  typedef Shared<ND, COLS> R;
  constexpr int SWAVES = COLS * RINGS, CT = 16 * COLS, DP = 64 * ND, QP = TYPE == TYPE_F32 ? 2 : 1, PP = TYPE == TYPE_BF16 ? 1 : 2, S = R::S;
  alignas(16) __shared__ char ring[RINGS][S][R::STAGE];
  __shared__ float aff[RINGS][2][4][32];  // scale and zero of keys (times what scores share), of values
  __shared__ int shifts[RINGS][2];        // and whether columns part in the lowest bit
  __shared__ float tops[SWAVES][16], ls[COLS][16];
  static_assert(S * R::STAGE >= COLS * 4 * ND * 1024, "a ring's sums fit where its blocks were");
  // heads first: the workgroups of one XCD (every eighth) read few heads' keys and values
  const int head = blockIdx.x, piece = (int)(blockIdx.y + gridDim.y * blockIdx.z);
  const Work work = find_work<false, CT>(c, a, piece);
  if (!work.any) {
    clear_idle<T>(c, a, head, work.idle, (int)(gridDim.y * gridDim.z) - (piece - work.idle));
    return;
  }
  const Tile& t = work.t;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int mine = wave / COLS, ct = wave % COLS;  // the wave's ring, and its tile of columns
  const int blocks = t.kb1 - t.kb0, size = blocks / work.chunks, more = blocks - size * work.chunks;  // one more in some
  const int begin = __builtin_amdgcn_readfirstlane(t.kb0 + work.chunk * size + (work.chunk < more ? work.chunk : more));
  const int end = __builtin_amdgcn_readfirstlane(begin + size + (work.chunk < more));
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
  half8 q[1][2 * ND][QP];
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
  query_operands<TYPE, ND, 1, QP>(q, qsum, x, {common + down});
  qsum[0] = __builtin_ldexpf(qsum[0], down);
  const float factor = __builtin_ldexpf(a.scale, common);
  State<ND, 1> st;
  clear(st);

  int held = -1000, least = -1000;  // the shift that values are staged with; no scale seen is below 2^least
  auto prepare = [&](int kb, int stage, int buf) {  // lanes 0..31 the keys, 32..63 the values
    const unsigned affine = *reinterpret_cast<const unsigned*>(ring[mine][stage] + 2048 * ND + 4 * lane);
    const unsigned w = (there >> stage & 1u) && kb * 32 + (lane & 31) < len ? affine : FLAT;  // beyond the sequence: whatever the page holds
    const float s = __uint_as_float(w << 16), z = __builtin_fmaf(8.f, s, __uint_as_float(w & 0xffff0000u));
    const bool real = lane >= 32 && s > 0.f && s < __builtin_inff();  // -0, infinities and NaN are of no matter
    const int ex = real ? exponent_of(s) + 1 : held;                  // s in [2^(ex - 1), 2^ex), subnormal or not
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
    to[lane >> 5 << 1][lane & 31] = lane < 32 ? s * factor : __builtin_ldexpf(s, ROOM - held);
    to[(lane >> 5 << 1) + 1][lane & 31] = lane < 32 ? z * factor : z;
    if (lane == 0) shifts[mine][buf] = 2 * held + (least < held - SPREAD<PP>);
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
      wait_turn<ND, COLS>(ct);
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
      shared_block<ND, QP, PP>(st, q, qsum, ring[mine][buf], aff[mine][i % 2], mask, kb * 32 + 4 * g, place, a.window,
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
    for (int i = 0; i < 4; ++i) st.o[0][d][i] = __builtin_ldexpf(st.o[0][d][i], st.shift[0] - ROOM) + z;
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
  if (work.chunks > 1) {
    const int at = work.first + work.chunk * work.tiles + work.tile;
    if ((unsigned)at >= (unsigned)a.parts) return;  // offsets that do not ascend
    float* out = a.part + ((int64_t)at * c.heads + head) * (int64_t)(CT * (DP + 2));
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

// Joins the chunks' results of shared_kernel: a workgroup 8 columns of a tile and head, a wave's loads of 16 chunks on their way at
// once: of few tiles, that many chunks share, it is the joining that is waited for.  All kernels, bf16, 8 kv heads of 128, 4 heads
// each (in brackets: a workgroup all 32 columns, 4 loads at once): 7 nodes of one sequence of 8000 tokens 22 us (28), of 4 of 131000
// 220 (230), 8 of 64 of up to 8000 127 (126); 8 heads each, 32 of one of 8000 42 (44).
constexpr int CJ = 8;
template <int TYPE, int ND, int CT>
__global__ __launch_bounds__(THREADS) void join_tile_kernel(KvCache c, Attend a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int DP = 64 * ND, SIZE = CT * (DP + 2), PER = THREADS / CJ, PIECE = 32;
  constexpr int VECTORS = CJ * 16 * ND, ITEMS = (VECTORS + THREADS - 1) / THREADS, UNROLL = ITEMS < 4 ? 16 / ITEMS : 4;
  __shared__ float factors[PIECE][CJ], tops[CJ], sums[CJ];
  const int head = blockIdx.x % c.heads, col0 = blockIdx.x / c.heads * CJ;
  const Work work = find_work<true, CT>(c, a, (int)(blockIdx.y + gridDim.y * blockIdx.z));
  if (!work.any || work.chunks <= 1) return;
  const int last = work.first + (work.chunks - 1) * work.tiles + work.tile;
  if (work.first < 0 || (unsigned)last >= (unsigned)a.parts) return;  // offsets that do not ascend
  const Tile& t = work.t;
  const float* part = a.part + ((int64_t)(work.first + work.tile) * c.heads + head) * SIZE;
  const int64_t stride = (int64_t)work.tiles * c.heads * SIZE;  // from chunk to chunk
  const int cols = (t.cols - t.col0 < CT ? t.cols - t.col0 : CT) - col0;  // of these that there are
  if (cols <= 0) return;
  // the largest of each column's references, by PER threads
  const int col = threadIdx.x / PER, j = threadIdx.x % PER;
  const float* mine = part + CT * DP + col0 + (col < cols ? col : 0);
  float top = -__builtin_inff(), l = 0.f;
  for (int i = j; i < work.chunks; i += PER) {
    const float x = mine[i * stride];
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
  for (int i0 = 0; i0 < work.chunks; i0 += PIECE) {
    const int n = work.chunks - i0 < PIECE ? work.chunks - i0 : PIECE;
    for (int i = j; i < n; i += PER) {
      const float* at = mine + (i0 + i) * stride;
      const float x = at[0], f = x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(x - top);
      l += f * at[CT];
      factors[i][col] = f;
    }
    __syncthreads();
#pragma unroll UNROLL
    for (int i = 0; i < n; ++i) {
      const floatx4* from = reinterpret_cast<const floatx4*>(part + (i0 + i) * stride + col0 * DP);
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {  // columns past the sequence's are not written: the first one's in their place
        const int u = threadIdx.x + THREADS * k, in = u / (16 * ND) % CJ;
        sum[k] += factors[i][in] * from[in < cols ? u % VECTORS : u % (16 * ND)];
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
    if (in >= cols || u >= VECTORS) continue;
    const int at = t.col0 + col0 + in, hq = head * a.group + at % a.group;
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
  int64_t pieces, parts;  // of shared_kernel's work and of its partial results, for a head, at most
  int64_t list;           // floats of the list of pieces, before the partial results
};

inline TreePlan make_tree_plan(int64_t tokens, int64_t seqs, int heads, int group, int dim, int64_t most, int64_t window,
                               int64_t nodes) {
  TreePlan p;
  static_cast<Plan&>(p) = make_plan(tokens, seqs, heads, group, dim, most, window, nodes);
  seqs += !seqs;
  const int64_t columns = tokens * group, tiles = cdiv(columns, 32) > seqs ? cdiv(columns, 32) : seqs;
  const int64_t total = p.blocks * tiles * heads;
  // Few columns, and fewer blocks than workgroups of shared_kernel fit at once: the call is its start, which attend_kernel's waves,
  // each alone, do sooner (bf16, 8 kv heads of 128, 4 heads each, us of all kernels, attend and shared: 7 nodes of one sequence of
  // 100 tokens 10 and 15, of 1000 14 and 16, of 8000 23 and 23; of 4 of 1000 19 and 17, of 32 of 300 37 and 21, of 16 of 4000 56
  // and 44; where pieces are listed, 2 nodes of 65 of 100 18 and 21, of 100 of 100 22 and 23, 4 of 100 of 300 43 and 30).  Up to 8
  // columns a sequence attend_kernel is ahead of more work too where lengths are alike (2 nodes of one of 8000 16 and 20, of 100 of
  // 4000 123 and 140, of 256 of 2000 149 and 170), which a call does not know, and behind where they differ (300 to 8000: 64
  // sequences 122 and 94, 100 165 and 142, 256 365 and 331; 300 to 4000: 65 63 and 73, 256 193 and 187).
  // Many columns and more blocks than fit at a time: prompt_kernel, which brings codes to fp16 once for 128 columns (shared and
  // prompt: 24 nodes of 100 tokens 14 and 20; 128 of 1000 25 and 36, of 4000 42 and 47, of 8 of 300 43 and 46, of 16 of 300 73 and
  // 50; of 64 of up to 8000 32 366 and 560, 48 538 and 597, 64 697 and 603, 80 838 and 757; of 16 of 2000 48 92 and 112, 64 117 and
  // 115, 80 141 and 116; 32 of 4 of 131000, 8 heads each, 1151 and 989.  fp16 and fp32 64 of 16 of 2000 128 and 141, 142 and 154, else
  // alike).  Heads past 128 leave it a wave a SIMD (of 256, 16 of 3000: 64 nodes 300 and 490, 96 414 and 502).
  const int64_t many = p.nd <= 2 ? 256 : 384;
  p.shared = p.prompt ? columns < many * seqs || total < 16384 : total >= (seqs > 64 ? 4096 : 1024);
  if (!p.shared) return p;
  p.prompt = false;
  p.ct = columns <= 16 * seqs ? 16 : 32;
  p.slots = columns / p.ct + seqs;  // tiles at most
  p.pieces = p.slots + most_chunks(heads);
  p.parts = p.blocks > 5 ? (4 * most_chunks(heads) + 2) / 3 : 0;
  p.turns = cdiv(p.pieces + 1, 65535);  // one more, for the rows that no sequence has
  p.chunks = 1;
  p.list = seqs > 64 ? 4 * (1 + p.pieces + p.slots) : 0;
  p.part = p.list + p.parts * heads * (int64_t)(p.ct * (64 * p.nd + 2));
  return p;
}

template <int TYPE, int ND, int COLS>
void launch_cols(const KvCache& c, const Attend& a, const TreePlan& p, hipStream_t st) {
  const auto grid = [&](int64_t x, int64_t y) { return dim3((unsigned)x, (unsigned)cdiv(y, p.turns), (unsigned)p.turns); };
  hipLaunchKernelGGL((shared_kernel<TYPE, ND, COLS>), grid(c.heads, p.pieces + 1), dim3(64 * COLS * RINGS), 0, st, c, a);
  if (p.parts)
    hipLaunchKernelGGL((join_tile_kernel<TYPE, ND, 16 * COLS>), grid(16 * COLS / CJ * c.heads, p.slots), dim3(THREADS), 0, st, c, a);
}

template <int TYPE, int ND>
int launch_shared(const KvCache& c, Attend a, const TreePlan& p, hipStream_t st) {
  a.pieces = (int)p.pieces, a.parts = (int)p.parts;
  if (p.list) {
    a.list = reinterpret_cast<int4*>(a.part);
    a.part += p.list;
    hipLaunchKernelGGL(list_kernel, dim3(1), dim3(LISTING), 0, st, c, a, (int)p.slots, p.ct);
  }
  if (p.ct == 16)
    launch_cols<TYPE, ND, 1>(c, a, p, st);
  else
    launch_cols<TYPE, ND, 2>(c, a, p, st);
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
