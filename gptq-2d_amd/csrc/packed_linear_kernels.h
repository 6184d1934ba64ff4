// The product's kernels for one width of the codes (each width is a source file of its own: packed_linear_bits*.hip).
#pragma once

#include "lds_limit.h"
#include "packed_linear.h"

namespace {

// Scales and zero points of a block of 128 columns for a lane's row in MR tiles of rows (NARROW: of its four steps).
template <int MODE, int MR>
struct Affine {
  static constexpr int N = narrow(MODE) ? 4 : 1;
  float s[MR][N], z[MR][N];
};

template <int MODE>
__device__ __forceinline__ int group_of(const Linear& p, int kb, int i) {
  const int step = narrow(MODE) ? 4 * kb + i : kb;
  const int k = p.steps == 1 ? step : (int)__umulhi((unsigned)step, p.mag);
  return k < p.groups ? k : p.groups - 1;  // steps past the row's end
}

// Whole rows': read once.
template <int MR>
__device__ __forceinline__ void load_affine(Affine<ROWS, MR>& f, const Linear& p, const int (&row)[MR]) {
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    f.s[j][0] = p.scale[row[j] * p.scale_row];
    f.z[j][0] = p.zero ? p.zero[row[j] * p.zero_row] : 0.f;
  }
}

// Where a group ends: tot -= s rest times the sums of its activations (tokens t0 + 16 n + 4 g .. + 3), in the rows with a
// rest: the sums may be infinite or NaN, which times 0 would be NaN in rows that only share the wave with such a row.
template <int NT>
__device__ __forceinline__ void add_rest(floatx4 (&tot)[NT], const Linear& p, int t0, int k, float s, float rest) {
  if (!p.corrected || !__builtin_amdgcn_ballot_w64(rest != 0.f)) return;
  const float f = -s * rest;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const floatx4 x = *reinterpret_cast<const floatx4*>(p.sums + k * p.sums_row + t0 + 16 * n + 4 * (threadIdx.x >> 4 & 3));
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[n][i] = rest != 0.f ? __builtin_fmaf(x[i], f, tot[n][i]) : tot[n][i];
  }
}

// A block's products into tot, times their scales where there are groups: c its codes of MR tiles of 16 rows, f their scales and zero
// points, x(n, i, q) the activations' operand of tokens 16 n, step i, piece q.
template <int BITS, int MODE, int NT, int MR, int NP, class X>
__device__ __forceinline__ void block_products(floatx4 (&tot)[MR][NT], const Codes<BITS> (&c)[MR],
                                               const Affine<MODE, MR>& f, X x, const Linear& p, int kb, int t0) {
  Run<BITS> runs[MR][4];
#pragma unroll
  for (int j = 0; j < MR; ++j) step_runs<BITS, !narrow(MODE)>(runs[j], c[j]);
  Middle<BITS> mid[MR];
  float rest[MR];
  if constexpr (!narrow(MODE)) {  // all steps of a tile of tokens in turn: a group's sums live no longer than the block
    half8 o[MR][4];
#pragma unroll
    for (int j = 0; j < MR; ++j) {
      rest[j] = split_shift<BITS>(mid[j], f.z[j][0] + p.offset);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = centred<BITS>(runs[j][i], mid[j]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      floatx4 part[MR];
#pragma unroll
      for (int j = 0; j < MR; ++j) part[j] = MODE == ROWS ? tot[j][n] : (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          const half8 a = x(n, i, q);
#pragma unroll
          for (int j = 0; j < MR; ++j) part[j] = mma(a, o[j][i], part[j]);
        }
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          tot[j][n][e] = MODE == ROWS ? part[j][e] : __builtin_fmaf(part[j][e], f.s[j][0], tot[j][n][e]);
      if (MR > 1) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (zeros(MODE)) {
      const int k = group_of<MODE>(p, kb, 0);
      if (kb + 1 == (int)((k + 1) * p.steps) || kb + 1 == p.blocks)
#pragma unroll
        for (int j = 0; j < MR; ++j) add_rest<NT>(tot[j], p, t0, k, f.s[j][0], rest[j]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (zeros(MODE) || i == 0) {
#pragma unroll
      for (int j = 0; j < MR; ++j) rest[j] = split_shift<BITS>(mid[j], f.z[j][i] + p.offset);
    }
    half8 o[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) o[j] = centred<BITS>(runs[j][i], mid[j]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      floatx4 part[MR];
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const half8 a = x(n, i, q);
#pragma unroll
        for (int j = 0; j < MR; ++j) part[j] = mma(a, o[j], q ? part[j] : (floatx4){0.f, 0.f, 0.f, 0.f});
      }
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) tot[j][n][e] = __builtin_fmaf(part[j][e], f.s[j][i], tot[j][n][e]);
    }
    if constexpr (zeros(MODE)) {
      const int step = 4 * kb + i, k = group_of<MODE>(p, kb, i);
      if (32 * step < p.n && (step + 1 == (int)((k + 1) * p.steps) || 32 * (step + 1) >= p.n))
#pragma unroll
        for (int j = 0; j < MR; ++j) add_rest<NT>(tot[j], p, t0, k, f.s[j][i], rest[j]);
    }
  }
}

// After the last block [.., kb_end) of whole rows: their scales.
template <int BITS, int MODE, int NT, int MR>
__device__ __forceinline__ void end_rows(floatx4 (&tot)[MR][NT], const Affine<MODE, MR>& f, const Linear& p, int kb_end, int t0) {
  if constexpr (MODE == ROWS) {
#pragma unroll
    for (int j = 0; j < MR; ++j) {
      Middle<BITS> mid;
      const float rest = split_shift<BITS>(mid, f.z[j][0] + p.offset);
#pragma unroll
      for (int n = 0; n < NT; ++n) tot[j][n] *= f.s[j][0];
      if (kb_end == p.blocks) add_rest<NT>(tot[j], p, t0, 0, f.s[j][0], rest);
    }
  }
}

// The factors that bring the sums of tokens t0 + 4 g .. + 3 back.
__device__ __forceinline__ floatx4 factors(const Linear& p, int t0) {
  const int t = t0 + 4 * (threadIdx.x >> 4 & 3);
  floatx4 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = p.factor[t + i < p.tokens ? t + i : p.tokens - 1];
  return f;
}

// The result of 16 tokens from t0 and the rows r0 + 16 j, or this split's part of it.
template <int MR>
__device__ __forceinline__ void store_tile(const floatx4 (&tot)[MR], const Linear& p, int t0, int r0, int split) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
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

// Waits until at most N of this wave's loads are on their way (they return in order), and until its LDS reads have returned:
// the stage that they read is loaded next, and a wave alone with its stages has no barrier between the two.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt has six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Up to 64 tokens, where the codes' bytes are the bound.  A workgroup takes 16 NT tokens and 16 MR WR rows of W: WR waves beside
// each other in the rows (which share the activations), WK such groups, each with a run of the split's blocks, whose sums
// are joined through LDS at the end (so that no part of a row is left for another launch to add).  All that a block of
// 128 columns needs -- activations, codes, scales, zero points -- is loaded straight into LDS, S - 1 blocks ahead, without a
// register; every wave issues the same number of loads a block and waits for its own by count.  In LDS a token's 16 pieces
// of 16 bytes lie at piece ^ token, so that the 16 tokens of an operand read lie in different banks; codes and scales lie
// as the lanes read them.  TQ: quads of tokens that are staged.
// Measured, INT4: 14336 x 4096 in groups of 128, 16 tokens 18.5 us (1.9 TB/s: seven blocks a wave, of which the ring's
// first fill and the sums' joining take half); 8192 x 28672 in groups of 32, 32 tokens 50 us (3.0 TB/s; 64 fused multiply-adds and
// 40 conversions a block for 16 products); 4096 x 4096, one token 7 us.
template <int BITS, int MODE, int NT, int TQ, int MR, int WR, int WK, int NP>
struct Ring {
  static constexpr int X = NP * TQ;                              // loads of 1 KB: activations
  static constexpr int CW = BITS == 8 ? 2 : BITS == 4 ? 1 : BITS;  // loads of codes of 16 rows (16 bytes a lane, or 4)
  static constexpr int CB = BITS * 256;                            // their bytes
  static constexpr int A = MODE == ROWS ? 0 : wide(MODE) ? 1 : MR;  // loads of 256 bytes: scales; as many zero points
  static constexpr int AZ = zeros(MODE) ? 2 * A : A;
  static constexpr int PART = MR * CB + AZ * 256;  // bytes of a wave's own part
  static constexpr int STAGE = X * 1024 + WR * PART;                  // of a group of waves
  static constexpr int LOADS = X / WR + MR * CW + AZ;              // of a wave
  static constexpr int FIT = 81920 / (WK * STAGE);                    // two workgroups a CU
  static constexpr int COUNT = 63 / LOADS + 2;
  static constexpr int S = FIT < COUNT ? (FIT < 8 ? FIT : 8) : (COUNT < 8 ? COUNT : 8);
  static constexpr int BYTES = S * WK * STAGE;
  static_assert(S >= 2 && X % WR == 0 && WK * WR * MR * NT * 1024 <= BYTES, "a block fits twice, and the groups' sums");
};

template <int BITS, int MODE, int NT, int TQ, int MR, int WR, int WK, int NP>
__global__ __launch_bounds__(64 * WR * WK, WR * WK / 2) void stream_kernel(Linear p) {
  typedef Ring<BITS, MODE, NT, TQ, MR, WR, WK, NP> R;
  constexpr int S = R::S;
  extern __shared__ float4 lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
  const int wr = wave % WR, wk = wave / WR;
  const int t0 = blockIdx.y * (16 * NT), r0 = (blockIdx.x * WR + wr) * (16 * MR);
  const int split = blockIdx.z;
  const int s0 = split * p.split_blocks, s1 = s0 + p.split_blocks < p.blocks ? s0 + p.split_blocks : p.blocks;
  const int per = (s1 - s0 + WK - 1) / WK, b0 = s0 + wk * per;
  const int count = s1 - b0 < per ? (s1 - b0 > 0 ? s1 - b0 : 0) : per;  // blocks of this group; the others may have one more
  char* const base = reinterpret_cast<char*>(lds) + wk * (S * R::STAGE);
  const int own = R::X * 1024 + wr * R::PART;  // this wave's part of a stage

  // activations: 1 KB = four tokens a load, lane l brings piece (l % 16) ^ token of token l / 16 of the four
  constexpr int XL = TQ / WR;
  const int pitch = 256 * p.blocks, tokens = p.tokens - t0 < 4 * TQ ? p.tokens - t0 : 4 * TQ;
  const _Float16* const xb = p.xp + (int64_t)t0 * (128 * p.blocks);
  int xo[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int token = 4 * (wr * XL + i) + g;
    xo[i] = token < tokens ? token * pitch + 16 * (c16 ^ (token & 15)) : OOB;
  }
  // codes: of lane l, those of row l % 16 that its part g multiplies; the extent ends with the last row's words
  const int first = r0 < p.m ? r0 : p.m - 1, rows = p.m - first < 16 * MR ? p.m - first : 16 * MR;
  const unsigned* const cb = p.words + first * p.row_words;
  const int extent = (int)(((rows - 1) * p.row_words + p.need_words) * 4);
  int co[MR];
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    const int r = 16 * j + c16;
    co[j] = (int)((r < rows ? r : rows - 1) * p.row_words * 4) + g * BITS * 4;
  }
  // scales: WIDE lane l brings row l % 16 of tile l / 16, NARROW row l / 4 of a tile in step l % 4
  const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p.scale) + first * p.scale_row,
                                                                     (short)0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t zr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<float*>(p.zero) + (p.zero ? first * p.zero_row : 0), (short)0, p.zero ? 0x7fffffff : 0, 0x00020000);
  int so[R::A ? R::A : 1], zo[R::A ? R::A : 1];
#pragma unroll
  for (int j = 0; j < R::A; ++j) {
    const int r = wide(MODE) ? lane : 16 * j + lane / 4;
    so[j] = (int)((r < rows ? r : rows - 1) * p.scale_row * 4);
    zo[j] = (int)((r < rows ? r : rows - 1) * p.zero_row * 4);
  }
  auto stage = [&](int kb, int buf) {
    char* const at = base + buf * R::STAGE;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<_Float16*>(xb + q * p.piece + 128 * kb), (short)0, tokens * pitch - 256 * kb, 0x00020000);
#pragma unroll
      for (int i = 0; i < XL; ++i) dma_load<4>(xr, reinterpret_cast<float*>(at + (q * TQ + wr * XL + i) * 1024), xo[i]);
    }
    char* const mine = at + own;
    const __amdgpu_buffer_rsrc_t cr = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned*>(cb + kb * (4 * BITS)), (short)0,
                                                                       extent - kb * (16 * BITS), 0x00020000);
#pragma unroll
    for (int j = 0; j < MR; ++j)
#pragma unroll
      for (int i = 0; i < R::CW; ++i) {
        if constexpr (BITS >= 4)
          dma_load<4>(cr, reinterpret_cast<float*>(mine + j * R::CB + i * 1024), co[j] + 16 * i);
        else
          dma_load<1>(cr, reinterpret_cast<float*>(mine + j * R::CB + i * 256), co[j] + 4 * i);
      }
    if constexpr (MODE != ROWS) {
      const int k = wide(MODE) ? group_of<MODE>(p, kb, 0) : group_of<MODE>(p, kb, lane & 3);
#pragma unroll
      for (int j = 0; j < R::A; ++j) {
        dma_load<1>(sr, reinterpret_cast<float*>(mine + MR * R::CB + j * 256), so[j] + k * (int)p.scale_col * 4);
        if constexpr (zeros(MODE)) dma_load<1>(zr, reinterpret_cast<float*>(mine + MR * R::CB + (R::A + j) * 256), zo[j] + k * (int)p.zero_col * 4);
      }
    }
  };
  floatx4 tot[MR][NT], low[MR][NT];
#pragma unroll
  for (int j = 0; j < MR; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) tot[j][n] = low[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
  Affine<MODE, MR> f;
  if constexpr (MODE == ROWS) {
    int row[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) row[j] = first + (16 * j + c16 < rows ? 16 * j + c16 : rows - 1);
    load_affine<MR>(f, p, row);
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < count) stage(b0 + s, s);
  if (p.index) {
#pragma unroll
    for (int j = 0; j < MR; ++j)
      add_own_adapters<NT, NP>(low[j], p, t0, r0 + 16 * j + c16, split * WK + wk, p.splits * WK);
  }
  int buf = 0;
  for (int it = 0; it < per; ++it) {
    if (it + S - 1 <= count)
      wait_loads<(S - 2) * R::LOADS>();
    else
      wait_loads<0>();
    if constexpr (WR > 1) __syncthreads();  // every wave's part of the stage is there, the stage before is no longer read
    const int ahead = buf ? buf - 1 : S - 1;
    if (it + S - 1 < count) stage(b0 + it + S - 1, ahead);
    if (it < count) {
      const char* const at = base + buf * R::STAGE;
      const char* const mine = at + own;
      Codes<BITS> c[MR];
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int i = 0; i < R::CW; ++i) {
          if constexpr (BITS >= 4) {
            const uint4v v = *reinterpret_cast<const uint4v*>(mine + j * R::CB + i * 1024 + lane * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) c[j].w[4 * i + e] = v[e];
          } else {
            c[j].w[i] = *reinterpret_cast<const unsigned*>(mine + j * R::CB + i * 256 + lane * 4);
          }
        }
      if constexpr (MODE != ROWS) {
        const float* const s = reinterpret_cast<const float*>(mine + MR * R::CB);
#pragma unroll
        for (int j = 0; j < MR; ++j)
#pragma unroll
          for (int i = 0; i < Affine<MODE, MR>::N; ++i) {
            const int e = wide(MODE) ? 16 * j + c16 : 64 * j + 4 * c16 + i;
            f.s[j][i] = s[e];
            f.z[j][i] = zeros(MODE) ? s[64 * R::A + e] : 0.f;
          }
      }
      block_products<BITS, MODE, NT, MR, NP>(
          tot, c, f,
          [&](int n, int i, int q) {
            const int token = (16 * n + c16) % (4 * TQ), piece = narrow(MODE) ? 4 * i + g : 4 * g + i;
            return *reinterpret_cast<const half8*>(at + q * (TQ * 1024) + token * 256 + (piece ^ (token & 15)) * 16);
          },
          p, b0 + it, t0);
    }
    buf = buf + 1 < S ? buf + 1 : 0;
  }
  if (count) end_rows<BITS, MODE, NT, MR>(tot, f, p, b0 + count, t0);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const floatx4 f4 = factors(p, t0 + 16 * n);
#pragma unroll
    for (int j = 0; j < MR; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) low[j][n][i] = __builtin_fmaf(tot[j][n][i], f4[i], low[j][n][i]);
  }
  if constexpr (WK > 1) {
    floatx4* const sums = reinterpret_cast<floatx4*>(lds);
    __syncthreads();  // no wave reads its stages any more
    if (wk) {
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) sums[((wave * MR + j) * NT + n) * 64 + lane] = low[j][n];
    }
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int w = 1; w < WK; ++w)
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) low[j][n] += sums[(((w * WR + wr) * MR + j) * NT + n) * 64 + lane];
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    floatx4 out[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) out[j] = low[j][n];
    if (t0 + 16 * n < p.tokens) store_tile<MR>(out, p, t0 + 16 * n, r0, split);
  }
}

// More tokens: 256 threads take 16 NT WT tokens and 16 MR (4 / WT) rows of W, each wave 16 NT tokens and 16 MR rows.  The
// activations of a block of 128 columns, scales and zero points go to LDS straight from memory, two blocks in turn; the codes
// from memory to the wave that multiplies by them, a block ahead.  In LDS a token's 16 pieces of 16 bytes lie at piece ^ token, so that
// the 16 tokens of an operand read lie in different banks.
// Measured, INT4, 2048 tokens x 8192 x 8192: rows 296 us, groups of 128 300 us (916 TFLOP/s; a library's fp16 product of that size
// takes 221 us), with zero points 320, groups of 32 with zero points 505.
// Bound by the two waves a SIMD that 255 registers leave: 1024 cycles of matrix and some 850 of vector instructions a block
// and wave overlap only between them.
template <int BITS, int MODE, int NT, int MR, int WT>
__global__ __launch_bounds__(256, 2) void tile_kernel(Linear p) {
  constexpr int TOK = 16 * NT * WT, ROWS_OF = 16 * MR * (4 / WT), N = Affine<MODE, MR>::N;
  extern __shared__ float4 lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
  const int wt = wave % WT, wr = wave / WT;
  const int tile_t = blockIdx.y * TOK, t0 = tile_t + 16 * NT * wt, tile_r = blockIdx.x * ROWS_OF, r0 = tile_r + 16 * MR * wr;
  const int split = blockIdx.z;
  const int b0 = split * p.split_blocks, b1 = b0 + p.split_blocks < p.blocks ? b0 + p.split_blocks : p.blocks;
  const int pitch = 256 * p.blocks;  // bytes of a token
  const int rows = p.tokens - tile_t < TOK ? p.tokens - tile_t : TOK;
  const __amdgpu_buffer_rsrc_t rsrc =
      __builtin_amdgcn_make_buffer_rsrc(p.xp + (int64_t)tile_t * (128 * p.blocks), (short)0, rows * pitch, 0x00020000);
  // 1 KB = four tokens a load: lane l brings piece (l % 16) ^ token of token l / 16 of the four
  constexpr int LOADS = TOK / 4 / 4;  // of a wave
  int off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int token = 4 * (wave * LOADS + i) + g;
    off[i] = token < rows ? token * pitch + 16 * (c16 ^ (token & 15)) : OOB;
  }
  auto stage = [&](int kb, int buf) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      dma_load<4>(rsrc, reinterpret_cast<float*>(lds + buf * (TOK * 16) + (wave * LOADS + i) * 64),
                  off[i] == OOB ? OOB : off[i] + 256 * kb);
  };
  // scales, then zero points: of row i / N in step i % N, 64 of them a load.  (Loaded by the lanes that use them they are 4
  // to 32 loads a wave and block, each of 16 lines, and their registers: 2048 tokens x 8192 x 8192, with zero points, groups
  // of 128 482 us for 342, groups of 32 1500 us for 536.)
  constexpr int AL = ROWS_OF * N / 64, ALL = zeros(MODE) ? 2 * AL : AL;
  const int rows_w = p.m - tile_r < ROWS_OF ? p.m - tile_r : ROWS_OF;
  float* const affine = reinterpret_cast<float*>(lds + 2 * TOK * 16);
  [[maybe_unused]] auto stage_affine = [&](int kb, int buf) {
    const int k = narrow(MODE) ? group_of<MODE>(p, kb, lane & 3) : group_of<MODE>(p, kb, 0);
#pragma unroll
    for (int i = 0; i < ALL; i += 4) {
      const int load = i + wave, part = load % AL;
      if (load >= ALL) break;
      const bool z = load >= AL;
      const int r = (64 * part + lane) / N, at = r < rows_w ? r : rows_w - 1;
      const int64_t first = tile_r * (z ? p.zero_row : p.scale_row);
      const float* const from = z ? p.zero + (p.zero ? first : 0) : p.scale + first;
      const __amdgpu_buffer_rsrc_t ar = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(from), (short)0,
                                                                         from ? 0x7fffffff : 0, 0x00020000);
      dma_load<1>(ar, affine + (buf * ALL + load) * 64,
                  at * (int)(z ? p.zero_row : p.scale_row) * 4 + k * (int)(z ? p.zero_col : p.scale_col) * 4);
    }
  };
  int row[MR];
  const unsigned* words[MR];
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    const int r = r0 + 16 * j + c16;
    row[j] = r < p.m ? r : p.m - 1;
    words[j] = p.words + row[j] * p.row_words;
  }
  floatx4 tot[MR][NT];
#pragma unroll
  for (int j = 0; j < MR; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) tot[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
  Codes<BITS> c[MR];
  Affine<MODE, MR> f;
  auto load = [&](int kb) {
    if (kb < p.whole) {
#pragma unroll
      for (int j = 0; j < MR; ++j) load_codes<BITS, false>(c[j], words[j], (4 * kb + g) * BITS, (int)p.need_words);
    } else {
#pragma unroll
      for (int j = 0; j < MR; ++j) load_codes<BITS, true>(c[j], words[j], (4 * kb + g) * BITS, (int)p.need_words);
    }
    if constexpr (MODE != ROWS) stage_affine(kb, (kb - b0) & 1);
  };
  if constexpr (MODE == ROWS) load_affine<MR>(f, p, row);
  stage(b0, 0);
  load(b0);
  for (int kb = b0; kb < b1; ++kb) {
    const int buf = (kb - b0) & 1;
    wait_dma();
    __syncthreads();  // buffer `buf` is whole, the other no longer read
    Codes<BITS> now[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) now[j] = c[j];
    if (kb + 1 < b1) {
      stage(kb + 1, 1 - buf);
      load(kb + 1);
    }
    if constexpr (MODE != ROWS) {
      const float* const at = affine + buf * (ALL * 64) + (16 * MR * wr + c16) * N;
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          f.s[j][i] = at[16 * N * j + i];
          f.z[j][i] = zeros(MODE) ? at[AL * 64 + 16 * N * j + i] : 0.f;
        }
    }
    const float4* in = lds + buf * (TOK * 16);
    block_products<BITS, MODE, NT, MR, 1>(
        tot, now, f,
        [&](int n, int i, int) {
          const int token = 16 * (NT * wt + n) + c16, piece = narrow(MODE) ? 4 * i + g : 4 * g + i;
          return __builtin_bit_cast(half8, in[token * 16 + (piece ^ c16)]);
        },
        p, kb, t0);
  }
  end_rows<BITS, MODE, NT, MR>(tot, f, p, b1, t0);
  if (t0 >= p.tokens) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const floatx4 back = factors(p, t0 + 16 * n);
#pragma unroll
    for (int j = 0; j < MR; ++j) tot[j][n] *= back;
  }
  if (p.index && split == 0) add_adapters<MR, NT>(tot, p, t0, r0);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    floatx4 out[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) out[j] = tot[j][n];
    store_tile<MR>(out, p, t0 + 16 * n, r0, split);
  }
}

template <int BITS, int MODE, int NT, int TQ, int MR, int WR, int WK, int NP>
int launch_stream(const Linear& p, const Plan& q, hipStream_t st) {
  constexpr auto kernel = stream_kernel<BITS, MODE, NT, TQ, MR, WR, WK, NP>;
  if (const int rc = allow_lds<kernel>()) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(p.m, 16 * MR * WR), (unsigned)cdiv(p.tokens, q.tile), (unsigned)q.splits),
                     dim3(64 * WR * WK), (Ring<BITS, MODE, NT, TQ, MR, WR, WK, NP>::BYTES), st, p);
  return (int)hipGetLastError();
}

template <int BITS, int MODE>
int launch_product(const Linear& p, const Plan& q, hipStream_t st) {
  if (q.pieces == 2)
    return q.rows == 16 ? launch_stream<BITS, MODE, 1, 1, 1, 1, 8, 2>(p, q, st)
                        : q.tile == 16 ? launch_stream<BITS, MODE, 1, 4, 1, 4, 2, 2>(p, q, st)
                                       : launch_stream<BITS, MODE, 2, 8, 1, 4, 1, 2>(p, q, st);
  if (q.rows == 16) return launch_stream<BITS, MODE, 1, 1, 1, 1, 8, 1>(p, q, st);
  if (q.tile == 16) return launch_stream<BITS, MODE, 1, 4, 1, 4, 2, 1>(p, q, st);
  if (q.tile == 32) return launch_stream<BITS, MODE, 2, 8, 1, 8, 1, 1>(p, q, st);
  if (q.tile == 64) return launch_stream<BITS, MODE, 4, 16, 1, 8, 1, 1>(p, q, st);
  constexpr int affine = MODE == ROWS ? 0 : 128 * (narrow(MODE) ? 4 : 1) * (zeros(MODE) ? 2 : 1);  // floats of a block
  constexpr auto kernel = tile_kernel<BITS, MODE, 4, 4, 2>;
  if (const int rc = allow_lds<kernel>()) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(p.m, q.rows), (unsigned)cdiv(p.tokens, q.tile), (unsigned)q.splits), dim3(256),
                     (size_t)q.tile * 512 + 8 * affine, st, p);
  return (int)hipGetLastError();
}

template <int BITS>
int launch_mode(const Linear& p, const Plan& q, hipStream_t st) {
  switch (q.mode) {
    case ROWS:
      return launch_product<BITS, ROWS>(p, q, st);
    case WIDE:
      return launch_product<BITS, WIDE>(p, q, st);
    case NARROW:
      return launch_product<BITS, NARROW>(p, q, st);
    case WIDE | ZEROS:
      return launch_product<BITS, WIDE | ZEROS>(p, q, st);
  }
  return launch_product<BITS, NARROW | ZEROS>(p, q, st);
}

}  // namespace
