// Products with a packed INT layer, with the low-rank adapters of many requests beside them (packed_linear.h for the
// formulas).  A call is two launches, three where the columns are dealt to several workgroups:
//   prepare_kernel: a workgroup a token brings the activations to fp16 (and sums groups of them for the zero points);
//                   others, beside them, multiply 16 tokens by one adapter's A over a chunk of columns;
//   stream_kernel (up to 64 tokens) or tile_kernel (more): the product, with B and the bias in its epilogue;
//   finish_kernel: adds the parts of a row that several workgroups summed.
// Measured: prepare_kernel 5.4 us for one token (launch and two latencies), 2048 x 8192 bf16 22 us (67 MB, 3.1 TB/s), 42
// with four adapters of rank 64 beside them (their loads' latency: two CU-fulls of workgroups); finish_kernel 4 to 5 us.
#include "packed_linear.h"

namespace {

constexpr int PREP = 512;

template <int TYPE>
__device__ __forceinline__ void prepare_token(const Linear& p, int t, int pieces) {
  typedef typename Elem<TYPE>::T T;
  constexpr int U = 4;  // loads in flight
  __shared__ float tops[PREP / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* row = static_cast<const T*>(p.x) + (int64_t)t * p.x_token;
  const bool held = p.n <= 8 * PREP * U;  // the row stays in registers
  Raw8<TYPE> x[U];
  float top = 0.f;
  for (int d0 = 8 * tid; d0 < p.n; d0 += 8 * PREP * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(row, d0 + 8 * PREP * u, p.n);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_fabsf(x[u][e]);
        top = v < __builtin_inff() && v > top ? v : top;  // infinities and NaN stay what they are in fp16
      }
  }
#pragma unroll
  for (int s = 1; s < 64; s *= 2) top = fmaxf(top, __shfl_xor(top, s));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < PREP / 64; ++w) top = fmaxf(top, tops[w]);
  // At least -126, so that the factor back is a normal number; the smallest fp32 numbers are then multiples of 2^-23, which
  // fp16 holds.
  const int ex = exponent_of(top) - 14 > -126 ? exponent_of(top) - 14 : -126;
  _Float16* out = p.xp + (int64_t)t * (128 * p.blocks);
  const bool by_lanes = p.corrected && p.group <= 512 && (p.group & (p.group - 1)) == 0;  // a group is 4 to 64 lanes' runs
  float all = 0.f;
  for (int d0 = 8 * tid; d0 - 8 * tid < 128 * p.blocks; d0 += 8 * PREP * U) {
    if (!held || d0 >= p.n)
#pragma unroll
      for (int u = 0; u < U; ++u) x[u].load(row, d0 + 8 * PREP * u, p.n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (d0 - 8 * tid + 8 * PREP * u >= 128 * p.blocks) break;
      const int d = d0 + 8 * PREP * u;
      half8 h, l;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_ldexpf(x[u][e / 2 + e % 2 * 4], -ex);
        sum += v;
        h[e] = (_Float16)v;
        l[e] = __builtin_fabsf(v) < __builtin_inff() ? (_Float16)(v - (float)h[e]) : (_Float16)0.f;
      }
      if (d < 128 * p.blocks) {
        *reinterpret_cast<half8*>(out + d) = h;
        if (pieces == 2) *reinterpret_cast<half8*>(out + p.piece + d) = l;
      }
      all += sum;
      if (by_lanes) {
        for (int s = 1; s < p.group / 8; s *= 2) sum += __shfl_xor(sum, s);
        if (d < p.n && d % p.group == 0) p.sums[d / p.group * p.sums_row + t] = sum;
      }
    }
  }
  if (tid == 0) p.factor[t] = __builtin_ldexpf(1.f, ex);
  if (!p.corrected || by_lanes) return;
  if (p.groups == 1) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) all += __shfl_xor(all, s);
    __syncthreads();
    if (lane == 0) tops[wave] = all;
    __syncthreads();
    all = 0.f;
#pragma unroll
    for (int w = 0; w < PREP / 64; ++w) all += tops[w];
    if (tid == 0) p.sums[t] = all;
  } else {  // other groups: a wave each
    for (int k = wave; k < p.groups; k += PREP / 64) {
      float sum = 0.f;
      for (int d = k * p.group + 8 * lane; d < (k + 1) * p.group; d += 512) {
        Raw8<TYPE> x;
        x.load(row, d, p.n);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += __builtin_ldexpf(x[e], -ex);
      }
#pragma unroll
      for (int s = 1; s < 64; s *= 2) sum += __shfl_xor(sum, s);
      if (lane == 0) p.sums[k * p.sums_row + t] = sum;
    }
  }
}

template <int TYPE>
struct Operand {  // eight elements as an operand: fp16 and bf16 as they are, fp32 in three bf16 pieces
  bf16x8 p[3];
  __device__ __forceinline__ explicit Operand(const Raw8<TYPE>& r) {
    if constexpr (TYPE == TYPE_F32) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = r[e];
      split8(x, p);
    } else {
      p[0] = __builtin_bit_cast(bf16x8, r.v[0]);
    }
  }
};

template <int TYPE>
__device__ __forceinline__ floatx4 multiply(const Operand<TYPE>& a, const Operand<TYPE>& b, floatx4 c) {
  if constexpr (TYPE == TYPE_F16) {
    c = mma(__builtin_bit_cast(half8, a.p[0]), __builtin_bit_cast(half8, b.p[0]), c);
  } else if constexpr (TYPE == TYPE_BF16) {
    c = mma(a.p[0], b.p[0], c);
  } else {
#pragma unroll
    for (int q = 0; q < NPROD; ++q) c = mma(a.p[prod_a[q]], b.p[prod_b[q]], c);
  }
  return c;
}

// V[chunk, t, j] = sum over the chunk's columns of x[t, k] A[a, j, k], for those of a tile's 16 tokens (bits `same`) that have
// adapter a.  The eight waves take every eighth step of 32 columns, two or four steps' loads in flight; ranks
// j0 .. j0 + 31 (64 take so many registers that a CU holds one workgroup, with nothing beside it).
template <int TYPE>
__device__ __forceinline__ void shrink_one(const Linear& p, int tile, int chunk, int a, unsigned same, int j0, int k0, int k1,
                                           floatx4 (*parts)[2][64]) {
  typedef typename Elem<TYPE>::T T;
  constexpr int W = PREP / 64, U = TYPE == TYPE_F32 ? 2 : 4;  // steps whose loads are in flight
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const bool match = same >> (lane & 15) & 1u;
  const T* row = static_cast<const T*>(p.x) + (int64_t)(match ? 16 * tile + (lane & 15) : 0) * p.x_token;
  floatx4 acc[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) acc[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
  const T* w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = j0 + 16 * j + (lane & 15);
    w[j] = static_cast<const T*>(p.a) + ((int64_t)a * p.rank + (r < p.rank ? r : p.rank - 1)) * p.n;
  }
  const int tiles16 = p.rank - j0 > 16 ? 2 : 1;
  for (int k = k0 + 32 * wave; k < k1; k += 32 * W * U) {
    Raw8<TYPE> x[U], b[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // past the chunk's end: nothing
      const int d = k + 32 * W * u + 8 * g, n = k + 32 * W * u < k1 ? p.n : 0;
      x[u].load(row, d, match ? n : 0);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (j < tiles16) b[u][j].load(w[j], d, n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Operand<TYPE> xo(x[u]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (j < tiles16) acc[j] = multiply<TYPE>(xo, Operand<TYPE>(b[u][j]), acc[j]);
    }
  }
  if (wave) {
#pragma unroll
    for (int j = 0; j < 2; ++j) parts[wave - 1][j][lane] = acc[j];
  }
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      floatx4 v = acc[j];
#pragma unroll
      for (int w = 0; w < W - 1; ++w) v += parts[w][j][lane];
      const int r = j0 + 16 * j + (lane & 15);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int in = 4 * g + i;
        const float out = r < p.rank ? v[i] : 0.f;
        if (r < p.rank_pad && same >> in & 1u) p.v[((int64_t)chunk * p.tokens + 16 * tile + in) * p.rank_pad + r] = out;
      }
    }
  }
  __syncthreads();
}

// Workgroup `slot` of a tile of 16 tokens, 32 ranks and a chunk of columns takes every slots-th of the tile's distinct adapters.
template <int TYPE>
__device__ __forceinline__ void shrink(const Linear& p, int item) {
  __shared__ floatx4 parts[PREP / 64 - 1][2][64];
  const int ranks = p.rank_pad / 32, tiles = (p.tokens + 15) / 16;
  const int slot = item % p.slots, j0 = item / p.slots % ranks * 32, rest = item / p.slots / ranks;
  const int tile = rest % tiles, chunk = rest / tiles;
  const int mine = adapter_of(p, 16 * tile + (threadIdx.x & 15));
  const int k0 = chunk * p.chunk, k1 = k0 + p.chunk < p.n ? k0 + p.chunk : p.n;
  unsigned pending = (unsigned)__builtin_amdgcn_ballot_w64(mine >= 0) & 0xffffu;
  for (int s = 0; pending; ++s) {
    const int a = __builtin_amdgcn_readlane(mine, __builtin_ctz(pending));
    const unsigned same = (unsigned)__builtin_amdgcn_ballot_w64(mine == a) & 0xffffu;
    pending &= ~same;
    if (s % p.slots == slot) shrink_one<TYPE>(p, tile, chunk, a, same, j0, k0, k1, parts);
  }
}

template <int TYPE>
__global__ __launch_bounds__(PREP, 4) void prepare_kernel(Linear p, int shrinks, int pieces) {
  if ((int)blockIdx.x < shrinks)  // first: they take longer
    shrink<TYPE>(p, blockIdx.x);
  else
    prepare_token<TYPE>(p, blockIdx.x - shrinks, pieces);
}

// y = the splits' parts added in their order, and the bias.
__global__ __launch_bounds__(256) void finish_kernel(Linear p) {
  const int r = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (r >= p.m) return;
  float sum = p.bias ? load_any(p.bias, r, p.type) : 0.f;
  const float* part = p.part + (int64_t)t * p.m + r;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) sum += part[(int64_t)s * p.tokens * p.m];
  store_any(p.y, (int64_t)t * p.y_token + r, p.type, sum);
}

inline int64_t align4(int64_t n) { return (n + 3) / 4 * 4; }

inline bool make_plan(Plan& q, int64_t tokens, int64_t m, int64_t n, int bits, int64_t group, bool zero, int type,
                      int64_t adapters, int64_t rank) {
  if (tokens < 0 || m < 1 || n < 1 || tokens > ((int64_t)1 << 24) || m >= ((int64_t)1 << 26) || n >= ((int64_t)1 << 21) ||
      (bits != 2 && bits != 3 && bits != 4 && bits != 8) || group < 0 || group % 32 || type < 0 ||
      type > 2 || adapters < 0 || adapters > (1 << 24) || (adapters > 0 && (rank < 1 || rank > 4096)))
    return false;
  const int64_t blocks = cdiv(n, 128);
  if (group >= n) group = 0;
  q.pieces = type == TYPE_F32 ? 2 : 1;
  q.mode = group == 0 ? ROWS : (group % 128 == 0 ? WIDE : NARROW) | (zero ? ZEROS : 0);
  q.groups = group ? cdiv(n, group) : 1;
  // Rows and tokens of a workgroup (fp32, whose activations are two pieces, stays with small tiles).  Measured, us, bf16:
  //   up to 4 tokens 16 rows of W, else 64: 4096 x 4096, 1 token 18.5 against 21.0; 8192 x 28672, 4 tokens 37.8 against 39.3;
  //   up to 64 tokens stream_kernel, more tile_kernel: 64 tokens, 14336 x 4096 33.9 against 38.1; 128 tokens, 8192 x 28672
  //   101 against 92; and 65 to 128 tokens of a layer that tile_kernel makes fewer than 256 workgroups of: 128 tokens,
  //   4096 x 4096 25.0 against 34.9.
  int64_t wgs, least, enough;  // workgroups without splits, blocks of a split at least, workgroups that need no splits
  const bool small = cdiv(m, 128) * cdiv(blocks, 8) < 256;
  if (tokens <= 4) {
    q.tile = 16, q.rows = 16, least = 16, enough = 192;
  } else if (tokens <= 64 || q.pieces == 2 || (tokens <= 128 && small)) {
    q.tile = tokens <= 16 ? 16 : tokens <= 32 || q.pieces == 2 ? 32 : 64;
    q.rows = tokens <= 16 || q.pieces == 2 ? 64 : 128, least = 8, enough = 192;
  } else {
    q.tile = 128, q.rows = 128, least = 8, enough = 384;
  }
  wgs = cdiv(m, q.rows) * cdiv(tokens + !tokens, q.tile);
  // Columns are split where the workgroups leave CUs idle, at the price of finish_kernel: 16 tokens, 8192 x 8192 (128
  // workgroups) 22.5 us in four parts, 25.3 in one; 14336 x 4096 (224) 21.9 and 19.2.
  int64_t splits = wgs >= enough ? 1 : cdiv(512, wgs);
  if (splits > cdiv(blocks, least)) splits = cdiv(blocks, least);
  if (splits > 64) splits = 64;
  q.split_blocks = (int)cdiv(blocks, splits);
  q.splits = (int)cdiv(blocks, q.split_blocks);
  q.rank_pad = adapters ? (int)((rank + 31) / 32 * 32) : 0;
  // the adapters' columns in chunks: a workgroup for each CU where 16 tokens share an adapter, a chunk at least 1024 columns
  // and at most 8 of them (32 tokens, 8 adapters, 28672 columns: with at most 4 the whole call takes 89 us for 80, with 16 the
  // same); 16 tokens may have 16 adapters, which as many workgroups take as find room beside each other
  const int64_t tiles = cdiv(tokens + !tokens, 16);
  int64_t chunks = cdiv(256, tiles);
  chunks = chunks > 8 ? 8 : chunks;
  q.chunk = (int)(cdiv(cdiv(n, chunks), 128) * 128);
  if (q.chunk < 1024) q.chunk = 1024;
  q.chunks = (int)cdiv(n, q.chunk);
  const int64_t slots = cdiv(512, tiles * q.chunks * (q.rank_pad / 32 + !q.rank_pad)), most = adapters < 16 ? adapters : 16;
  q.slots = (int)(slots < most ? slots : most);
  q.sums_row = cdiv(tokens, 16) * 16 + 128;  // a tile's reads past the last token stay inside
  int64_t at = 0;
  q.xp = at, at += align4(q.pieces * tokens * blocks * 64);
  q.factor = at, at += align4(tokens);
  q.sums = at, at += q.groups * q.sums_row;
  q.v = at, at += adapters ? q.chunks * tokens * q.rank_pad : 0;
  q.part = at, at += q.splits > 1 ? align4((int64_t)q.splits * tokens * m) : 0;
  q.total = at;
  return true;
}

}  // namespace

extern "C" {

int64_t gptq2d_packed_linear_workspace(int64_t tokens, int64_t m, int64_t n, int32_t bits, int64_t group, int32_t type,
                                       int64_t adapters, int64_t rank) {
  Plan q;
  return make_plan(q, tokens, m, n, bits, group, false, type, adapters, rank) ? 4 * q.total : -1;
}

int gptq2d_packed_linear(const void* x, int64_t x_token, int32_t type, int64_t tokens, const uint32_t* words, int64_t m,
                         int64_t n, int64_t row_words, int32_t bits, const float* scale, int64_t scale_row,
                         int64_t scale_col, const float* zero, int64_t zero_row, int64_t zero_col, double qmin,
                         int64_t group, const void* bias, const void* a, const void* b, const float* scaling,
                         const int32_t* index, int64_t adapters, int64_t rank, void* y, int64_t y_token, void* work,
                         int64_t work_bytes, void* stream) {
  Plan q;
  if (!index || adapters == 0) adapters = 0, rank = 0, index = nullptr;
  if (qmin != __builtin_rint(qmin) || __builtin_fabs(qmin) > 1e9) return GPTQ2D_EINVAL;
  const double offset = -qmin - (double)(1 << (bits & 15) >> 1);  // 0 for the symmetric bounds of a whole bit field
  const bool shifted = zero || __builtin_fabs(offset) > 512.;
  if (!make_plan(q, tokens, m, n, bits, group, shifted, type, adapters, rank)) return GPTQ2D_EINVAL;
  if (row_words < cdiv(n * bits, 32)) return GPTQ2D_EINVAL;
  const int64_t far = (m < 128 ? m : 128) - 1, limit = (int64_t)1 << 28;  // a workgroup's byte offsets have 31 bits
  if (far * row_words > limit || far * scale_row + q.groups * scale_col > limit || far * zero_row + q.groups * zero_col > limit)
    return GPTQ2D_EUNSUPPORTED;
  if (tokens == 0) return 0;
  if (!work || (uintptr_t)work % 16 || work_bytes < 4 * q.total) return GPTQ2D_ESCRATCH;
  if (group >= n) group = 0;
  Linear p = {};
  p.tokens = (int)tokens, p.m = (int)m, p.n = (int)n, p.blocks = (int)cdiv(n, 128);
  p.words = words, p.row_words = row_words;
  p.scale = scale, p.scale_row = scale_row, p.scale_col = scale_col;
  p.zero = zero, p.zero_row = zero_row, p.zero_col = zero_col;
  p.offset = (float)offset;
  p.group = group ? (int)group : 128 * p.blocks;
  p.steps = (unsigned)(narrow(q.mode) ? p.group / 32 : p.group / 128);
  p.mag = (unsigned)((((uint64_t)1 << 32) + p.steps - 1) / p.steps);
  p.need_words = cdiv(n * bits, 32);
  p.whole = (int)(p.need_words / (4 * bits));
  p.corrected = shifted;
  p.x = x, p.x_token = x_token, p.type = type;
  float* w = static_cast<float*>(work);
  p.xp = reinterpret_cast<_Float16*>(w + q.xp);
  p.piece = tokens * 128 * p.blocks;
  p.factor = w + q.factor;
  p.sums = w + q.sums, p.sums_row = q.sums_row, p.groups = (int)q.groups;
  p.a = a, p.b = b, p.scaling = scaling, p.index = index;
  p.adapters = (int)adapters, p.rank = (int)rank, p.rank_pad = q.rank_pad, p.slots = q.slots, p.chunks = q.chunks, p.chunk = q.chunk;
  p.v = w + q.v;
  p.y = y, p.y_token = y_token, p.bias = bias;
  p.splits = q.splits, p.split_blocks = q.split_blocks, p.part = w + q.part;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t shrinks = index ? q.slots * (q.rank_pad / 32) * cdiv(tokens, 16) * q.chunks : 0, prep = tokens + shrinks;
  if (prep > 0x7fffffff || (q.tile && cdiv(tokens, q.tile) > 65535)) return GPTQ2D_EUNSUPPORTED;
  const dim3 grid((unsigned)prep), block(PREP);
  if (type == TYPE_F32)
    hipLaunchKernelGGL((prepare_kernel<TYPE_F32>), grid, block, 0, st, p, (int)shrinks, q.pieces);
  else if (type == TYPE_BF16)
    hipLaunchKernelGGL((prepare_kernel<TYPE_BF16>), grid, block, 0, st, p, (int)shrinks, q.pieces);
  else
    hipLaunchKernelGGL((prepare_kernel<TYPE_F16>), grid, block, 0, st, p, (int)shrinks, q.pieces);
  const int rc = bits == 2   ? packed_product_bits2(&p, &q, st)
                 : bits == 3 ? packed_product_bits3(&p, &q, st)
                 : bits == 4 ? packed_product_bits4(&p, &q, st)
                             : packed_product_bits8(&p, &q, st);
  if (rc) return rc;
  if (q.splits > 1)  // of fewer than 384 workgroups of up to 128 tokens: few enough for the grid's second axis
    hipLaunchKernelGGL(finish_kernel, dim3((unsigned)cdiv(m, 256), (unsigned)tokens), dim3(256), 0, st, p);
  return (int)hipGetLastError();
}

}  // extern "C"
