// Products with a packed INT layer, with the low-rank adapters of many requests beside them (packed_linear.h for the
// formulas).  A call is two launches, three where the columns are dealt to several workgroups:
//   prepare_kernel: a workgroup a token brings the activations to fp16 (and sums groups of them for the zero points);
//                   others, beside them, multiply 16 tokens by one adapter's A over a chunk of columns;
//   stream_kernel (up to 16 tokens) or tile_kernel (more): the product, with B and the bias in its epilogue;
//   finish_kernel: adds the parts of a row that several workgroups summed.
#include "packed_linear.h"

namespace {

constexpr int PREP = 256;

template <int TYPE>
__device__ __forceinline__ void prepare_token(const Linear& p, int pieces) {
  typedef typename Elem<TYPE>::T T;
  __shared__ float tops[PREP / 64];
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* row = static_cast<const T*>(p.x) + (int64_t)t * p.x_token;
  float top = 0.f;
  for (int d = 8 * tid; d < p.n; d += 8 * PREP) {
    float x[8];
    load_row<TYPE, 8>(x, row, d, p.n);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __builtin_fabsf(x[e]);
      top = v < __builtin_inff() && v > top ? v : top;  // infinities and NaN stay what they are in fp16
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s *= 2) top = fmaxf(top, __shfl_xor(top, s));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < PREP / 64; ++w) top = fmaxf(top, tops[w]);
  const int ex = exponent_of(top) - 14;
  _Float16* out = p.xp + (int64_t)t * (128 * p.blocks);
  float sum = 0.f;
  for (int d = 8 * tid; d < 128 * p.blocks; d += 8 * PREP) {
    float x[8];
    load_row<TYPE, 8>(x, row, d, p.n);
    half8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __builtin_ldexpf(x[e / 2 + e % 2 * 4], -ex);
      sum += v;
      h[e] = (_Float16)v;
      l[e] = __builtin_fabsf(v) < __builtin_inff() ? (_Float16)(v - (float)h[e]) : (_Float16)0.f;
    }
    *reinterpret_cast<half8*>(out + d) = h;
    if (pieces == 2) *reinterpret_cast<half8*>(out + p.piece + d) = l;
  }
  if (tid == 0) p.factor[t] = __builtin_ldexpf(1.f, ex);
  if (!p.corrected) return;
  if (p.groups == 1) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) sum += __shfl_xor(sum, s);
    __syncthreads();
    if (lane == 0) tops[wave] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < PREP / 64; ++w) sum += tops[w];
    if (tid == 0) p.sums[t] = sum;
  } else if (p.group <= 256) {  // a thread a group
    for (int k = tid; k < p.groups; k += PREP) {
      sum = 0.f;
      for (int d = k * p.group; d < (k + 1) * p.group; d += 8) {
        float x[8];
        load_row<TYPE, 8>(x, row, d, p.n);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += __builtin_ldexpf(x[e], -ex);
      }
      p.sums[k * p.sums_row + t] = sum;
    }
  } else {  // a wave a group
    for (int k = wave; k < p.groups; k += PREP / 64) {
      sum = 0.f;
      for (int d = k * p.group + 8 * lane; d < (k + 1) * p.group; d += 512) {
        float x[8];
        load_row<TYPE, 8>(x, row, d, p.n);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += __builtin_ldexpf(x[e], -ex);
      }
#pragma unroll
      for (int s = 1; s < 64; s *= 2) sum += __shfl_xor(sum, s);
      if (lane == 0) p.sums[k * p.sums_row + t] = sum;
    }
  }
}

// V[chunk, t, j] = sum over the chunk's columns of x[t, k] A[a, j, k], for the 16 tokens of a tile that have one adapter:
// workgroup `slot` of the tile takes the adapter of its token `slot`, where no earlier token has the same.  The four waves
// take every fourth step of 32 columns; 64 ranks at a time.
template <int TYPE>
__device__ __forceinline__ void shrink(const Linear& p, int item) {
  typedef typename Elem<TYPE>::T T;
  __shared__ floatx4 parts[3][4][64];
  const int slot = item % 16, rest = item / 16, tiles = (p.tokens + 15) / 16, tile = rest % tiles, chunk = rest / tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int t = 16 * tile + (lane & 15), mine = adapter_of(p, t);
  const int a = __builtin_amdgcn_readlane(mine, slot);
  const unsigned same = (unsigned)__builtin_amdgcn_ballot_w64(mine == a) & 0xffffu;
  if (a < 0 || __builtin_ctz(same) != slot) return;
  const T* row = static_cast<const T*>(p.x) + (int64_t)t * p.x_token;
  const int k0 = chunk * p.chunk, k1 = k0 + p.chunk < p.n ? k0 + p.chunk : p.n;
  for (int j0 = 0; j0 < p.rank_pad; j0 += 64) {
    floatx4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    for (int k = k0 + 32 * wave; k < k1; k += 128) {
      float x[8] = {};
      if (mine == a) load_row<TYPE, 8>(x, row, k + 8 * g, p.n);
      float w[4][8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j0 + 16 * j + (lane & 15);
        if (j0 + 16 * j < p.rank)
          load_row<TYPE, 8>(w[j], static_cast<const T*>(p.a) + ((int64_t)a * p.rank + (r < p.rank ? r : p.rank - 1)) * p.n,
                            k + 8 * g, p.n);
      }
      if constexpr (TYPE == TYPE_F16) {
        half8 xh;
#pragma unroll
        for (int e = 0; e < 8; ++e) xh[e] = (_Float16)x[e];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j0 + 16 * j < p.rank) {
            half8 wh;
#pragma unroll
            for (int e = 0; e < 8; ++e) wh[e] = (_Float16)w[j][e];
            acc[j] = mma(xh, wh, acc[j]);
          }
        }
      } else {
        bf16x8 xp[3], wp[3];
        split8(x, xp);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j0 + 16 * j < p.rank) {
            split8(w[j], wp);
            if constexpr (TYPE == TYPE_BF16) {
              acc[j] = mma(xp[0], wp[0], acc[j]);
            } else {
#pragma unroll
              for (int q = 0; q < NPROD; ++q) acc[j] = mma(xp[prod_a[q]], wp[prod_b[q]], acc[j]);
            }
          }
        }
      }
    }
    if (wave) {
#pragma unroll
      for (int j = 0; j < 4; ++j) parts[wave - 1][j][lane] = acc[j];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const floatx4 v = acc[j] + parts[0][j][lane] + parts[1][j][lane] + parts[2][j][lane];
        const int r = j0 + 16 * j + (lane & 15);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int in = 4 * g + i;
          if (r < p.rank_pad && same >> in & 1u)
            p.v[((int64_t)chunk * p.tokens + 16 * tile + in) * p.rank_pad + r] = r < p.rank ? v[i] : 0.f;
        }
      }
    }
    __syncthreads();
  }
}

template <int TYPE>
__global__ __launch_bounds__(PREP) void prepare_kernel(Linear p, int pieces) {
  if ((int)blockIdx.x < p.tokens)
    prepare_token<TYPE>(p, pieces);
  else
    shrink<TYPE>(p, blockIdx.x - p.tokens);
}

// Scale (and what the zero point differs from the middle code by) of row r in group k.
__device__ __forceinline__ float scale_of(const Linear& p, int r, int k) {
  return p.scale[r * p.scale_row + k * p.scale_col];
}
__device__ __forceinline__ float shift_of(const Linear& p, int r, int k) {
  return p.zero ? p.zero[r * p.zero_row + k * p.zero_col] + p.offset : p.offset;
}

enum { ROWS = 0, WIDE = 1, NARROW = 2 };  // groups: whole rows, multiples of 128 columns, other multiples of 32

// Adds the finished sums `acc` of tokens t0 + 16 n + 4 g .. + 3 and row r of W in group k to `tot`.
template <int NT>
__device__ __forceinline__ void add_group(floatx4 (&tot)[NT], floatx4 (&acc)[NT], const Linear& p, int t0, int r, int k,
                                          bool correct) {
  const float s = scale_of(p, r, k);
#pragma unroll
  for (int n = 0; n < NT; ++n) tot[n] += acc[n] * s;
  if (correct && p.corrected) {
    const float f = -s * shift_of(p, r, k);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(p.sums + k * p.sums_row + t0 + 16 * n + 4 * (threadIdx.x >> 4 & 3));
      tot[n] += x * f;
    }
  }
}

// A block's products into tot (and acc, the running sums of a group that is not finished): o[j] its operands of rows
// r0 + 16 j, x(n, i, q) the activations' operand of tokens 16 n, step i, piece q.
template <int MODE, int NT, int MR, int NP, class X>
__device__ __forceinline__ void block_products(floatx4 (&tot)[MR][NT], floatx4 (&acc)[MR][NT], const half8 (&o)[MR][4], X x,
                                               const Linear& p, int kb, int kb_last, int t0, int r0) {
  const int row = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (MODE == NARROW) {
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const half8 a = x(n, i, q);
#pragma unroll
        for (int j = 0; j < MR; ++j) acc[j][n] = mma(a, o[j][i], acc[j][n]);
      }
    }
    if constexpr (MODE == NARROW) {
      const int step = 4 * kb + i;
      if (32 * step < p.n) {
        const int k = p.steps == 1 ? step : (int)__umulhi((unsigned)step, p.mag);
        const bool ends = step + 1 == (int)((k + 1) * p.steps) || 32 * (step + 1) >= p.n;
#pragma unroll
        for (int j = 0; j < MR; ++j) {
          const int r = r0 + 16 * j + row;
          add_group<NT>(tot[j], acc[j], p, t0, r < p.m ? r : p.m - 1, k, ends);
        }
      }
    }
  }
  if constexpr (MODE != NARROW) {
    const int k = MODE == ROWS ? 0 : p.steps == 1 ? kb : (int)__umulhi((unsigned)kb, p.mag);
    const bool ends = MODE == ROWS ? kb + 1 == p.blocks : kb + 1 == (int)((k + 1) * p.steps) || kb + 1 == p.blocks;
    if (ends || kb == kb_last) {
#pragma unroll
      for (int j = 0; j < MR; ++j) {
        const int r = r0 + 16 * j + row;
        add_group<NT>(tot[j], acc[j], p, t0, r < p.m ? r : p.m - 1, k, ends);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
      }
    }
  }
}

// The result of 16 tokens from t0 and the rows r0 + 16 j, or this split's part of it.
template <int MR>
__device__ __forceinline__ void finish_tile(floatx4 (&tot)[MR], const Linear& p, int t0, int r0, int split) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  floatx4 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = t0 + 4 * g + i < p.tokens ? p.factor[t0 + 4 * g + i] : 0.f;
#pragma unroll
  for (int j = 0; j < MR; ++j) tot[j] *= f;
  if (p.index && split == 0) add_adapters<MR>(tot, p, t0, r0);
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    const int r = r0 + 16 * j + (lane & 15);
    const float bias = p.bias && r < p.m && p.splits == 1 ? load_any(p.bias, r, p.type) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + 4 * g + i;
      const bool in = t < p.tokens && r < p.m;
      if (p.splits > 1) {
        if (in) p.part[((int64_t)split * p.tokens + t) * p.m + r] = tot[j][i];
      } else {
        if (in) store_any(p.y, (int64_t)t * p.y_token + r, p.type, tot[j][i] + bias);
      }
    }
  }
}

// Up to 16 tokens: a workgroup takes 16 MR rows of W over the split's columns, its eight waves a run of blocks each; a
// wave reads its activations and codes as operands from memory, and the waves' sums are joined through LDS.
template <int BITS, int MODE, int MR, int NP>
__global__ __launch_bounds__(512) void stream_kernel(Linear p) {
  constexpr int W = 8;
  __shared__ floatx4 sums[W - 1][MR][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int r0 = blockIdx.x * (16 * MR), split = blockIdx.y;
  const int b0 = split * p.split_blocks, b1 = b0 + p.split_blocks < p.blocks ? b0 + p.split_blocks : p.blocks;
  const int per = (b1 - b0 + W - 1) / W;
  const int begin = b0 + wave * per, end = begin + per < b1 ? begin + per : b1;
  const unsigned* row[MR];
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    const int r = r0 + 16 * j + (lane & 15);
    row[j] = p.words + (r < p.m ? r : p.m - 1) * p.row_words;
  }
  const int t = lane & 15;
  const bool valid = t < p.tokens;
  const _Float16* x = p.xp + (int64_t)(valid ? t : 0) * (128 * p.blocks);
  floatx4 tot[MR][1], acc[MR][1];
#pragma unroll
  for (int j = 0; j < MR; ++j) tot[j][0] = acc[j][0] = (floatx4){0.f, 0.f, 0.f, 0.f};
  const half8 none = {};
  for (int kb = begin; kb < end; ++kb) {
    Codes<BITS> c[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) load_codes<BITS>(c[j], row[j], (4 * kb + g) * BITS, (int)p.row_words);
    half8 xs[4][NP];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const half8 v = *reinterpret_cast<const half8*>(x + q * p.piece + 128 * kb + (MODE == NARROW ? 32 * i + 8 * g : 32 * g + 8 * i));
        xs[i][q] = valid ? v : none;
      }
    half8 o[MR][4];
#pragma unroll
    for (int j = 0; j < MR; ++j) operands<BITS, MODE != NARROW>(o[j], c[j]);
    block_products<MODE, 1, MR, NP>(tot, acc, o, [&](int, int i, int q) { return xs[i][q]; }, p, kb, end - 1, 0, r0);
  }
  if (wave) {
#pragma unroll
    for (int j = 0; j < MR; ++j) sums[wave - 1][j][lane] = tot[j][0];
  }
  __syncthreads();
  if (wave) return;
  floatx4 out[MR];
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    out[j] = tot[j][0];
#pragma unroll
    for (int w = 0; w < W - 1; ++w) out[j] += sums[w][j][lane];
  }
  finish_tile<MR>(out, p, 0, r0, split);
}

// More tokens: 256 threads take 16 NT WT tokens and 16 MR (4 / WT) rows of W, each wave 16 NT tokens and 16 MR rows.  The
// activations of a block of 128 columns go to LDS straight from memory, two blocks in turn; the codes from memory to the
// operands of the wave that multiplies by them, a block ahead.  In LDS a token's 16 pieces of 16 bytes lie at piece ^ token,
// so that the 16 tokens of an operand read lie in different banks.
template <int BITS, int MODE, int NT, int MR, int WT, int NP>
__global__ __launch_bounds__(256) void tile_kernel(Linear p) {
  constexpr int TOK = 16 * NT * WT;
  extern __shared__ float4 lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
  const int wt = wave % WT, wr = wave / WT;
  const int tile_t = blockIdx.y * TOK, t0 = tile_t + 16 * NT * wt, r0 = blockIdx.x * (16 * MR * (4 / WT)) + 16 * MR * wr;
  const int split = blockIdx.z;
  const int b0 = split * p.split_blocks, b1 = b0 + p.split_blocks < p.blocks ? b0 + p.split_blocks : p.blocks;
  const int pitch = 256 * p.blocks;  // bytes of a token
  const int rows = p.tokens - tile_t < TOK ? p.tokens - tile_t : TOK;
  __amdgpu_buffer_rsrc_t rsrc[NP];
#pragma unroll
  for (int q = 0; q < NP; ++q)
    rsrc[q] = __builtin_amdgcn_make_buffer_rsrc(p.xp + q * p.piece + (int64_t)tile_t * (128 * p.blocks), (short)0,
                                                rows * pitch, 0x00020000);
  // 1 KB = four tokens a load: lane l brings piece (l % 16) ^ token of token l / 16 of the four
  constexpr int LOADS = TOK / 4 / 4;  // of a wave, a piece
  int off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int token = 4 * (wave * LOADS + i) + g;
    off[i] = token < rows ? token * pitch + 16 * (c16 ^ (token & 15)) : OOB;
  }
  auto stage = [&](int kb, int buf) {
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        dma_load<4>(rsrc[q], reinterpret_cast<float*>(lds + (buf * NP + q) * (TOK * 16) + (wave * LOADS + i) * 64),
                    off[i] == OOB ? OOB : off[i] + 256 * kb);
  };
  const unsigned* row[MR];
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    const int r = r0 + 16 * j + c16;
    row[j] = p.words + (r < p.m ? r : p.m - 1) * p.row_words;
  }
  floatx4 tot[MR][NT], acc[MR][NT];
#pragma unroll
  for (int j = 0; j < MR; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) tot[j][n] = acc[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
  Codes<BITS> c[MR];
  stage(b0, 0);
#pragma unroll
  for (int j = 0; j < MR; ++j) load_codes<BITS>(c[j], row[j], (4 * b0 + g) * BITS, (int)p.row_words);
  for (int kb = b0; kb < b1; ++kb) {
    const int buf = (kb - b0) & 1;
    wait_dma();
    __syncthreads();  // buffer `buf` is whole, the other no longer read
    half8 o[MR][4];
#pragma unroll
    for (int j = 0; j < MR; ++j) operands<BITS, MODE != NARROW>(o[j], c[j]);
    if (kb + 1 < b1) {
      stage(kb + 1, 1 - buf);
#pragma unroll
      for (int j = 0; j < MR; ++j) load_codes<BITS>(c[j], row[j], (4 * (kb + 1) + g) * BITS, (int)p.row_words);
    }
    const float4* in = lds + buf * NP * (TOK * 16);
    block_products<MODE, NT, MR, NP>(
        tot, acc, o,
        [&](int n, int i, int q) {
          const int token = 16 * (NT * wt + n) + c16, piece = MODE == NARROW ? 4 * i + g : 4 * g + i;
          return __builtin_bit_cast(half8, in[q * (TOK * 16) + token * 16 + (piece ^ c16)]);
        },
        p, kb, b1 - 1, t0, r0);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (t0 + 16 * n < p.tokens) {
      floatx4 out[MR];
#pragma unroll
      for (int j = 0; j < MR; ++j) out[j] = tot[j][n];
      finish_tile<MR>(out, p, t0 + 16 * n, r0, split);
    }
  }
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

// How a call is computed: tile (0: stream_kernel, else tokens of a tile), rows of a workgroup, splits of the columns, and
// where its workspace holds what (floats).
struct Plan {
  int pieces, tile, rows, splits, split_blocks, mode, bits, rank_pad, chunks, chunk;
  int64_t groups, sums_row, xp, factor, sums, v, part, total;  // offsets; total: floats
};

inline int64_t align4(int64_t n) { return (n + 3) / 4 * 4; }

inline bool make_plan(Plan& q, int64_t tokens, int64_t m, int64_t n, int bits, int64_t group, int type, int64_t adapters,
                      int64_t rank) {
  if (tokens < 0 || m < 1 || n < 1 || tokens > ((int64_t)1 << 24) || m >= ((int64_t)1 << 26) || n >= ((int64_t)1 << 21) ||
      (bits != 2 && bits != 3 && bits != 4 && bits != 8) || group < 0 || group % 32 || type < 0 ||
      type > 2 || adapters < 0 || adapters > (1 << 24) || (adapters > 0 && (rank < 1 || rank > 4096)))
    return false;
  const int64_t blocks = cdiv(n, 128);
  if (group >= n) group = 0;
  q.bits = bits;
  q.pieces = type == TYPE_F32 ? 2 : 1;
  q.mode = group == 0 ? ROWS : group % 128 == 0 ? WIDE : NARROW;
  q.groups = group ? cdiv(n, group) : 1;
  int64_t wgs;
  if (tokens <= 16) {
    q.tile = 0;
    q.rows = 16;
    wgs = cdiv(m, q.rows);
  } else {
    q.tile = q.pieces == 2 || tokens <= 32 ? 32 : tokens <= 64 ? 64 : 128;
    q.rows = 128;
    wgs = cdiv(m, q.rows) * cdiv(tokens, q.tile);
  }
  const int64_t least = q.tile ? 4 : 8;  // blocks of a split, at least
  int64_t splits = wgs >= 384 ? 1 : cdiv(512, wgs);
  if (splits > cdiv(blocks, least)) splits = cdiv(blocks, least);
  if (splits > 64) splits = 64;
  q.split_blocks = (int)cdiv(blocks, splits);
  q.splits = (int)cdiv(blocks, q.split_blocks);
  q.rank_pad = adapters ? (int)((rank + 31) / 32 * 32) : 0;
  q.chunk = (int)(cdiv(cdiv(n, 16), 128) * 128);
  if (q.chunk < 512) q.chunk = 512;
  q.chunks = (int)cdiv(n, q.chunk);
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

template <int BITS, int MODE>
int launch_product(const Linear& p, const Plan& q, hipStream_t st) {
  const dim3 stream_grid((unsigned)cdiv(p.m, 16), (unsigned)q.splits);
  const dim3 grid((unsigned)cdiv(p.m, 128), q.tile ? (unsigned)cdiv(p.tokens, q.tile) : 1, (unsigned)q.splits);
  const size_t lds = (size_t)q.tile * 512 * q.pieces;
#define GPTQ2D_TILE(...)                                                                                              \
  do {                                                                                                                \
    static const int ready = (int)hipFuncSetAttribute(reinterpret_cast<const void*>(&tile_kernel<__VA_ARGS__>),       \
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, 163840);            \
    if (ready) return ready;                                                                                          \
    hipLaunchKernelGGL((tile_kernel<__VA_ARGS__>), grid, dim3(256), lds, st, p);                                      \
  } while (0)
  if (q.pieces == 2) {
    if (q.tile == 0)
      hipLaunchKernelGGL((stream_kernel<BITS, MODE, 1, 2>), stream_grid, dim3(512), 0, st, p);
    else
      GPTQ2D_TILE(BITS, MODE, 2, 2, 1, 2);
  } else if (q.tile == 0) {
    hipLaunchKernelGGL((stream_kernel<BITS, MODE, 1, 1>), stream_grid, dim3(512), 0, st, p);
  } else if (q.tile == 32) {
    GPTQ2D_TILE(BITS, MODE, 2, 2, 1, 1);
  } else if (q.tile == 64) {
    GPTQ2D_TILE(BITS, MODE, 4, 2, 1, 1);
  } else {
    GPTQ2D_TILE(BITS, MODE, 4, 4, 2, 1);
  }
#undef GPTQ2D_TILE
  return (int)hipGetLastError();
}

template <int BITS>
int launch_mode(const Linear& p, const Plan& q, hipStream_t st) {
  return q.mode == ROWS ? launch_product<BITS, ROWS>(p, q, st)
                        : q.mode == WIDE ? launch_product<BITS, WIDE>(p, q, st) : launch_product<BITS, NARROW>(p, q, st);
}

}  // namespace

extern "C" {

int64_t gptq2d_packed_linear_workspace(int64_t tokens, int64_t m, int64_t n, int32_t bits, int64_t group, int32_t type,
                                       int64_t adapters, int64_t rank) {
  Plan q;
  return make_plan(q, tokens, m, n, bits, group, type, adapters, rank) ? 4 * q.total : -1;
}

int gptq2d_packed_linear(const void* x, int64_t x_token, int32_t type, int64_t tokens, const uint32_t* words, int64_t m,
                         int64_t n, int64_t row_words, int32_t bits, const float* scale, int64_t scale_row,
                         int64_t scale_col, const float* zero, int64_t zero_row, int64_t zero_col, double qmin,
                         int64_t group, const void* bias, const void* a, const void* b, const float* scaling,
                         const int32_t* index, int64_t adapters, int64_t rank, void* y, int64_t y_token, void* work,
                         int64_t work_bytes, void* stream) {
  Plan q;
  if (!index || adapters == 0) adapters = 0, rank = 0, index = nullptr;
  if (!make_plan(q, tokens, m, n, bits, group, type, adapters, rank)) return GPTQ2D_EINVAL;
  if (row_words < cdiv(n * bits, 32)) return GPTQ2D_EINVAL;
  if (tokens == 0) return 0;
  if (!work || (uintptr_t)work % 16 || work_bytes < 4 * q.total) return GPTQ2D_ESCRATCH;
  if (group >= n) group = 0;
  Linear p = {};
  p.tokens = (int)tokens, p.m = (int)m, p.n = (int)n, p.blocks = (int)cdiv(n, 128);
  p.words = words, p.row_words = row_words;
  p.scale = scale, p.scale_row = scale_row, p.scale_col = scale_col;
  p.zero = zero, p.zero_row = zero_row, p.zero_col = zero_col;
  p.qmin = (float)qmin;
  p.offset = (float)(-qmin - (double)(1 << (bits - 1)));
  p.group = group ? (int)group : 128 * p.blocks;
  p.steps = (unsigned)(q.mode == NARROW ? p.group / 32 : p.group / 128);
  p.mag = (unsigned)((((uint64_t)1 << 32) + p.steps - 1) / p.steps);
  p.corrected = zero || p.offset != 0.f;
  p.x = x, p.x_token = x_token, p.type = type;
  float* w = static_cast<float*>(work);
  p.xp = reinterpret_cast<_Float16*>(w + q.xp);
  p.piece = tokens * 128 * p.blocks;
  p.factor = w + q.factor;
  p.sums = w + q.sums, p.sums_row = q.sums_row, p.groups = (int)q.groups;
  p.a = a, p.b = b, p.scaling = scaling, p.index = index;
  p.adapters = (int)adapters, p.rank = (int)rank, p.rank_pad = q.rank_pad, p.chunks = q.chunks, p.chunk = q.chunk;
  p.v = w + q.v;
  p.y = y, p.y_token = y_token, p.bias = bias;
  p.splits = q.splits, p.split_blocks = q.split_blocks, p.part = w + q.part;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t prep = tokens + (index ? 16 * cdiv(tokens, 16) * q.chunks : 0);
  if (prep > 0x7fffffff || (q.tile && cdiv(tokens, q.tile) > 65535)) return GPTQ2D_EUNSUPPORTED;
  const dim3 grid((unsigned)prep), block(PREP);
  if (type == TYPE_F32)
    hipLaunchKernelGGL((prepare_kernel<TYPE_F32>), grid, block, 0, st, p, q.pieces);
  else if (type == TYPE_BF16)
    hipLaunchKernelGGL((prepare_kernel<TYPE_BF16>), grid, block, 0, st, p, q.pieces);
  else
    hipLaunchKernelGGL((prepare_kernel<TYPE_F16>), grid, block, 0, st, p, q.pieces);
  int rc = bits == 2 ? launch_mode<2>(p, q, st)
                     : bits == 3 ? launch_mode<3>(p, q, st) : bits == 4 ? launch_mode<4>(p, q, st) : launch_mode<8>(p, q, st);
  if (rc) return rc;
  if (q.splits > 1) {
    if (tokens > 65535) return GPTQ2D_EUNSUPPORTED;
    hipLaunchKernelGGL(finish_kernel, dim3((unsigned)cdiv(m, 256), (unsigned)tokens), dim3(256), 0, st, p);
  }
  return (int)hipGetLastError();
}

}  // extern "C"
