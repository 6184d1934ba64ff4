// Products with a packed INT layer, with the low-rank adapters of many requests beside them (packed_linear.h for the
// formulas).  A call is two launches, three where the columns are dealt to several workgroups:
//   prepare_kernel: a workgroup a token brings the activations to fp16 (and sums groups of them for the zero points);
//                   others, beside them, multiply 16 tokens by one adapter's A over a chunk of columns;
//   stream_kernel (up to 64 tokens) or tile_kernel (more): the product, with B and the bias in its epilogue;
//   finish_kernel: adds the parts of a row that several workgroups summed.
#include "packed_linear.h"

#include <atomic>

namespace {

constexpr int PREP = 512;

// Eight consecutive elements as they lie, 0 past the row's end; loads only, so that several can be in flight.
template <int TYPE>
struct Raw8 {
  typedef typename Elem<TYPE>::T T;
  static constexpr int V = 16 / (int)sizeof(T);  // elements of a 16-byte load
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec v[8 / V];
  __device__ __forceinline__ void load(const T* __restrict__ row, int d, int n) {
    if (d + 8 <= n) {
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) v[i] = *reinterpret_cast<const vec*>(row + d + V * i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i / V][i % V] = d + i < n ? row[d + i] : (T)0;
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32<TYPE>(v[i / V][i % V]); }
};

template <int TYPE>
__device__ __forceinline__ void prepare_token(const Linear& p, int pieces) {
  typedef typename Elem<TYPE>::T T;
  constexpr int U = 2;  // loads in flight
  __shared__ float tops[PREP / 64];
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* row = static_cast<const T*>(p.x) + (int64_t)t * p.x_token;
  float top = 0.f;
  for (int d0 = 8 * tid; d0 < p.n; d0 += 8 * PREP * U) {
    Raw8<TYPE> x[U];
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
  const int ex = exponent_of(top) - 14;
  _Float16* out = p.xp + (int64_t)t * (128 * p.blocks);
  const bool by_lanes = p.corrected && p.group <= 512 && (p.group & (p.group - 1)) == 0;  // a group is 4 to 64 lanes' runs
  float all = 0.f;
  for (int d0 = 8 * tid; d0 - 8 * tid < 128 * p.blocks; d0 += 8 * PREP * U) {
    Raw8<TYPE> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(row, d0 + 8 * PREP * u, p.n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
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

// V[chunk, t, j] = sum over the chunk's columns of x[t, k] A[a, j, k], for the 16 tokens of a tile that have one adapter:
// workgroup `slot` of the tile takes its slot-th distinct one.  The eight waves take every eighth step of 32 columns, two
// steps' loads in flight; 64 ranks at a time.
template <int TYPE>
__device__ __forceinline__ void shrink(const Linear& p, int item) {
  typedef typename Elem<TYPE>::T T;
  constexpr int W = PREP / 64;
  __shared__ floatx4 parts[W - 1][4][64];
  const int slot = item % p.slots, rest = item / p.slots, tiles = (p.tokens + 15) / 16, tile = rest % tiles, chunk = rest / tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const int t = 16 * tile + (lane & 15), mine = adapter_of(p, t);
  unsigned pending = (unsigned)__builtin_amdgcn_ballot_w64(mine >= 0) & 0xffffu, same = 0;
  int a = -1;
  for (int s = 0; s <= slot; ++s) {
    if (!pending) return;
    a = __builtin_amdgcn_readlane(mine, __builtin_ctz(pending));
    same = (unsigned)__builtin_amdgcn_ballot_w64(mine == a) & 0xffffu;
    pending &= ~same;
  }
  const bool match = mine == a;
  const T* row = static_cast<const T*>(p.x) + (int64_t)(match ? t : 0) * p.x_token;
  const int k0 = chunk * p.chunk, k1 = k0 + p.chunk < p.n ? k0 + p.chunk : p.n;
  for (int j0 = 0; j0 < p.rank_pad; j0 += 64) {
    floatx4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    const T* w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = j0 + 16 * j + (lane & 15);
      w[j] = static_cast<const T*>(p.a) + ((int64_t)a * p.rank + (r < p.rank ? r : p.rank - 1)) * p.n;
    }
    const int tiles16 = p.rank - j0 > 48 ? 4 : p.rank - j0 > 32 ? 3 : p.rank - j0 > 16 ? 2 : 1;
    for (int k = k0 + 32 * wave; k < k1; k += 64 * W) {
      Raw8<TYPE> x[2], b[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {  // past the chunk's end: nothing
        const int d = k + 32 * W * u + 8 * g, n = k + 32 * W * u < k1 ? p.n : 0;
        x[u].load(row, d, match ? n : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < tiles16) b[u][j].load(w[j], d, n);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const Operand<TYPE> xo(x[u]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < tiles16) acc[j] = multiply<TYPE>(xo, Operand<TYPE>(b[u][j]), acc[j]);
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
}

template <int TYPE>
__global__ __launch_bounds__(PREP) void prepare_kernel(Linear p, int pieces) {
  if ((int)blockIdx.x < p.tokens)
    prepare_token<TYPE>(p, pieces);
  else
    shrink<TYPE>(p, blockIdx.x - p.tokens);
}

enum { ROWS = 0, WIDE = 1, NARROW = 2 };  // groups: whole rows, multiples of 128 columns, other multiples of 32

// Scales and zero points of a block of 128 columns for a lane's row in MR tiles of rows (NARROW: of its four steps).
template <int MODE, int MR>
struct Affine {
  static constexpr int N = MODE == NARROW ? 4 : 1;
  float s[MR][N], z[MR][N];
};

template <int MODE>
__device__ __forceinline__ int group_of(const Linear& p, int kb, int i) {
  if constexpr (MODE == ROWS) return 0;
  const int step = MODE == NARROW ? 4 * kb + i : kb;
  const int k = p.steps == 1 ? step : (int)__umulhi((unsigned)step, p.mag);
  return k < p.groups ? k : p.groups - 1;  // steps past the row's end
}

template <int MODE, int MR>
__device__ __forceinline__ void load_affine(Affine<MODE, MR>& f, const Linear& p, const int (&row)[MR], int kb) {
#pragma unroll
  for (int i = 0; i < Affine<MODE, MR>::N; ++i) {
    const int k = group_of<MODE>(p, kb, i);
#pragma unroll
    for (int j = 0; j < MR; ++j) f.s[j][i] = p.scale[row[j] * p.scale_row + k * p.scale_col];
    if (p.zero) {
#pragma unroll
      for (int j = 0; j < MR; ++j) f.z[j][i] = p.zero[row[j] * p.zero_row + k * p.zero_col];
    } else {
#pragma unroll
      for (int j = 0; j < MR; ++j) f.z[j][i] = 0.f;
    }
  }
}

// tot += s acc, and where the group ends here s rest times the sums of its activations (tokens t0 + 16 n + 4 g .. + 3).
template <int NT>
__device__ __forceinline__ void add_group(floatx4 (&tot)[NT], const floatx4 (&acc)[NT], const Linear& p, int t0, int k, float s,
                                          float rest, bool ends) {
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[n][i] = __builtin_fmaf(acc[n][i], s, tot[n][i]);
  if (p.corrected && ends && __builtin_amdgcn_ballot_w64(rest != 0.f)) {
    const float f = -s * rest;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(p.sums + k * p.sums_row + t0 + 16 * n + 4 * (threadIdx.x >> 4 & 3));
#pragma unroll
      for (int i = 0; i < 4; ++i) tot[n][i] = __builtin_fmaf(x[i], f, tot[n][i]);
    }
  }
}

// A block's products into tot, or acc where its group goes on: c its codes of MR tiles of 16 rows, f their scales and zero
// points, x(n, i, q) the activations' operand of tokens 16 n, step i, piece q.
template <int BITS, int MODE, int NT, int MR, int NP, class X>
__device__ __forceinline__ void block_products(floatx4 (&tot)[MR][NT], floatx4 (&acc)[MR][NT], const Codes<BITS> (&c)[MR],
                                               const Affine<MODE, MR>& f, X x, const Linear& p, int kb, int kb_last, int t0) {
  Run<BITS> runs[MR][4];
#pragma unroll
  for (int j = 0; j < MR; ++j) step_runs<BITS, MODE != NARROW>(runs[j], c[j]);
  Middle<BITS> mid[MR];
  float rest[MR];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (MODE == NARROW || i == 0) {
#pragma unroll
      for (int j = 0; j < MR; ++j) rest[j] = split_shift<BITS>(mid[j], f.z[j][MODE == NARROW ? i : 0] + p.offset);
    }
    half8 o[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) o[j] = centred<BITS>(runs[j][i], mid[j]);
    if constexpr (MODE == NARROW) {
      floatx4 part[MR][NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          const half8 a = x(n, i, q);
#pragma unroll
          for (int j = 0; j < MR; ++j) part[j][n] = mma(a, o[j], q ? part[j][n] : (floatx4){0.f, 0.f, 0.f, 0.f});
        }
      }
      const int step = 4 * kb + i, k = group_of<MODE>(p, kb, i);
      const bool ends = 32 * step < p.n && (step + 1 == (int)((k + 1) * p.steps) || 32 * (step + 1) >= p.n);
#pragma unroll
      for (int j = 0; j < MR; ++j) add_group<NT>(tot[j], part[j], p, t0, k, f.s[j][i], rest[j], ends);
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          const half8 a = x(n, i, q);
#pragma unroll
          for (int j = 0; j < MR; ++j) acc[j][n] = mma(a, o[j], acc[j][n]);
        }
      }
    }
  }
  if constexpr (MODE == WIDE) {
    const int k = group_of<MODE>(p, kb, 0);
    const bool ends = kb + 1 == (int)((k + 1) * p.steps) || kb + 1 == p.blocks;
    if (ends || kb == kb_last) {
#pragma unroll
      for (int j = 0; j < MR; ++j) {
        add_group<NT>(tot[j], acc[j], p, t0, k, f.s[j][0], rest[j], ends);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
      }
    }
  }
}

// After the last block [.., kb_end): whole rows' sums.
template <int BITS, int MODE, int NT, int MR>
__device__ __forceinline__ void end_rows(floatx4 (&tot)[MR][NT], const floatx4 (&acc)[MR][NT], const Affine<MODE, MR>& f,
                                         const Linear& p, int kb_end, int t0) {
  if constexpr (MODE == ROWS) {
#pragma unroll
    for (int j = 0; j < MR; ++j) {
      Middle<BITS> mid;
      const float rest = split_shift<BITS>(mid, f.z[j][0] + p.offset);
#pragma unroll
      for (int n = 0; n < NT; ++n) tot[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
      add_group<NT>(tot[j], acc[j], p, t0, 0, f.s[j][0], rest, kb_end == p.blocks);
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

// Waits until at most N of this wave's loads are on their way (they return in order).
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt has six bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Up to 64 tokens, where the codes' bytes are the bound.  A workgroup of four waves takes 16 NT tokens and 16 MR rows of W a
// wave (WK 1), or 16 MR rows whose blocks the waves take in turn (WK 4; few tokens or few rows: no part of a row is then
// left for another launch to add).  All that a block of 128 columns needs -- activations, codes, scales, zero points -- is
// loaded straight into LDS, S - 1 blocks ahead: 4 to 8 KB of codes a block and workgroup, so that a CU has 30 to 60 KB
// on their way without a register.  Every wave issues the same number of loads a block and waits for its own by count.
// In LDS a token's 16 pieces of 16 bytes lie at piece ^ token, so that the 16 tokens of an operand read lie in different
// banks; codes and scales lie as the lanes read them.  TQ: quads of tokens that are staged.
template <int BITS, int MODE, int NT, int TQ, int MR, int WK, int NP>
struct Ring {
  static constexpr int X = NP * TQ;                              // loads of 1 KB: activations
  static constexpr int CW = BITS == 8 ? 2 : BITS == 4 ? 1 : BITS;  // loads of codes of 16 rows (16 bytes a lane, or 4)
  static constexpr int CB = BITS * 256;                            // their bytes
  static constexpr int A = MODE == ROWS ? 0 : MODE == WIDE ? 1 : MR;  // loads of 256 bytes: scales; as many zero points
  static constexpr int PART = MR * CB + 2 * A * 256;                  // bytes of a wave's own part
  static constexpr int STAGE = WK == 1 ? X * 1024 + 4 * PART : 4 * (X * 1024 + PART);
  static constexpr int LOADS = (WK == 1 ? X / 4 : X) + MR * CW + 2 * A;  // of a wave
  static constexpr int FIT = 81920 / STAGE;  // two workgroups a CU
  static constexpr int COUNT = 63 / LOADS + 2;
  static constexpr int S = FIT < COUNT ? (FIT < 8 ? FIT : 8) : (COUNT < 8 ? COUNT : 8);
  static constexpr int BYTES = S * STAGE;
  static_assert(S >= 2, "a block fits twice");
};

template <int BITS, int MODE, int NT, int TQ, int MR, int WK, int NP>
__global__ __launch_bounds__(256, 2) void stream_kernel(Linear p) {
  typedef Ring<BITS, MODE, NT, TQ, MR, WK, NP> R;
  constexpr int S = R::S;
  extern __shared__ float4 lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
  const int t0 = blockIdx.y * (16 * NT), r0 = (blockIdx.x * (WK == 1 ? 4 : 1) + (WK == 1 ? wave : 0)) * (16 * MR);
  const int split = blockIdx.z;
  const int s0 = split * p.split_blocks, s1 = s0 + p.split_blocks < p.blocks ? s0 + p.split_blocks : p.blocks;
  const int per = (s1 - s0 + WK - 1) / WK;
  const int b0 = WK == 1 ? s0 : s0 + wave * per, b1 = WK == 1 ? s1 : b0 + per < s1 ? b0 + per : s1;
  char* const base = reinterpret_cast<char*>(lds) + (WK == 1 ? 0 : wave * (R::X * 1024 + R::PART) * S);
  constexpr int STEP = WK == 1 ? R::STAGE : R::X * 1024 + R::PART;  // from a stage to the next
  const int own = R::X * 1024 + (WK == 1 ? wave * R::PART : 0);     // this wave's part of a stage

  // activations: 1 KB = four tokens a load, lane l brings piece (l % 16) ^ token of token l / 16 of the four
  const int pitch = 256 * p.blocks, tokens = p.tokens - t0 < 4 * TQ ? p.tokens - t0 : 4 * TQ;
  constexpr int XL = WK == 1 ? TQ / 4 : TQ;
  __amdgpu_buffer_rsrc_t xr[NP];
#pragma unroll
  for (int q = 0; q < NP; ++q)
    xr[q] = __builtin_amdgcn_make_buffer_rsrc(p.xp + q * p.piece + (int64_t)t0 * (128 * p.blocks), (short)0, tokens * pitch,
                                              0x00020000);
  int xo[XL];
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int token = 4 * ((WK == 1 ? wave * XL : 0) + i) + g;
    xo[i] = token < tokens ? token * pitch + 16 * (c16 ^ (token & 15)) : -1;
  }
  // codes: of lane l, those of row l % 16 that its part g multiplies; the extent ends with the last row's words
  const int first = r0 < p.m ? r0 : p.m - 1, rows = p.m - first < 16 * MR ? p.m - first : 16 * MR;
  const __amdgpu_buffer_rsrc_t cr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned*>(p.words) + first * p.row_words, (short)0,
      (int)(((rows - 1) * p.row_words + p.need_words) * 4), 0x00020000);
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
    const int r = MODE == WIDE ? lane : 16 * j + lane / 4;
    so[j] = (int)((r < rows ? r : rows - 1) * p.scale_row * 4);
    zo[j] = (int)((r < rows ? r : rows - 1) * p.zero_row * 4);
  }
  auto stage = [&](int kb, int buf) {
    char* const at = base + buf * STEP;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int i = 0; i < XL; ++i)
        dma_load<4>(xr[q], reinterpret_cast<float*>(at + (q * TQ + (WK == 1 ? wave * XL : 0) + i) * 1024),
                    xo[i] < 0 ? OOB : xo[i] + 256 * kb);
    char* const mine = at + own;
#pragma unroll
    for (int j = 0; j < MR; ++j) {
      const int off = co[j] + kb * (16 * BITS);
      if constexpr (BITS >= 4) {
#pragma unroll
        for (int i = 0; i < R::CW; ++i) dma_load<4>(cr, reinterpret_cast<float*>(mine + j * R::CB + i * 1024), off + 16 * i);
      } else {
#pragma unroll
        for (int i = 0; i < R::CW; ++i) dma_load<1>(cr, reinterpret_cast<float*>(mine + j * R::CB + i * 256), off + 4 * i);
      }
    }
    if constexpr (MODE != ROWS) {
      const int k = MODE == WIDE ? group_of<MODE>(p, kb, 0) : group_of<MODE>(p, kb, lane & 3);
#pragma unroll
      for (int j = 0; j < R::A; ++j) {
        dma_load<1>(sr, reinterpret_cast<float*>(mine + MR * R::CB + j * 256), so[j] + k * (int)p.scale_col * 4);
        dma_load<1>(zr, reinterpret_cast<float*>(mine + MR * R::CB + (R::A + j) * 256), zo[j] + k * (int)p.zero_col * 4);
      }
    }
  };
  floatx4 tot[MR][NT], acc[MR][NT], low[MR][NT];
#pragma unroll
  for (int j = 0; j < MR; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) tot[j][n] = acc[j][n] = low[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
  Affine<MODE, MR> f;
  if constexpr (MODE == ROWS) {
    int row[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) row[j] = first + (16 * j + c16 < rows ? 16 * j + c16 : rows - 1);
    load_affine<MODE, MR>(f, p, row, 0);
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (b0 + s < b1) stage(b0 + s, s);
  if (p.index) {
    const int share = WK == 1 ? split : split * WK + wave;
#pragma unroll
    for (int j = 0; j < MR; ++j) add_own_adapters<NT>(low[j], p, t0, r0 + 16 * j + c16, share, p.splits * WK);
  }
  int buf = 0;
  for (int kb = b0; kb < b1; ++kb) {
    if (kb + S - 1 <= b1)
      wait_loads<(S - 2) * R::LOADS>();
    else
      wait_loads<0>();
    if constexpr (WK == 1) __syncthreads();  // every wave's part of the stage is there, the stage before is no longer read
    const int ahead = buf ? buf - 1 : S - 1;
    if (kb + S - 1 < b1) stage(kb + S - 1, ahead);
    const char* const at = base + buf * STEP;
    const char* const mine = at + own;
    Codes<BITS> c[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) {
      if constexpr (BITS >= 4) {
#pragma unroll
        for (int i = 0; i < R::CW; ++i) {
          const uint4v v = *reinterpret_cast<const uint4v*>(mine + j * R::CB + i * 1024 + lane * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) c[j].w[4 * i + e] = v[e];
        }
      } else {
#pragma unroll
        for (int i = 0; i < R::CW; ++i) c[j].w[i] = *reinterpret_cast<const unsigned*>(mine + j * R::CB + i * 256 + lane * 4);
      }
    }
    if constexpr (MODE != ROWS) {
      const float* const s = reinterpret_cast<const float*>(mine + MR * R::CB);
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int i = 0; i < Affine<MODE, MR>::N; ++i) {
          const int e = MODE == WIDE ? 16 * j + c16 : 64 * j + 4 * c16 + i;
          f.s[j][i] = s[e];
          f.z[j][i] = s[64 * R::A + e];
        }
    }
    block_products<BITS, MODE, NT, MR, NP>(
        tot, acc, c, f,
        [&](int n, int i, int q) {
          const int token = (16 * n + c16) % (4 * TQ), piece = MODE == NARROW ? 4 * i + g : 4 * g + i;
          return *reinterpret_cast<const half8*>(at + q * (TQ * 1024) + token * 256 + (piece ^ (token & 15)) * 16);
        },
        p, kb, b1 - 1, t0);
    buf = buf + 1 < S ? buf + 1 : 0;
  }
  if (b0 < b1) end_rows<BITS, MODE, NT, MR>(tot, acc, f, p, b1, t0);
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
    if (wave) {
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) sums[(((wave - 1) * MR + j) * NT + n) * 64 + lane] = low[j][n];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WK; ++w)
#pragma unroll
      for (int j = 0; j < MR; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) low[j][n] += sums[(((w - 1) * MR + j) * NT + n) * 64 + lane];
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
// activations of a block of 128 columns go to LDS straight from memory, two blocks in turn; the codes and scales from memory
// to the wave that multiplies by them, a block ahead.  In LDS a token's 16 pieces of 16 bytes lie at piece ^ token, so that
// the 16 tokens of an operand read lie in different banks.
template <int BITS, int MODE, int NT, int MR, int WT, int NP>
__global__ __launch_bounds__(256, 2) void tile_kernel(Linear p) {
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
  int row[MR];
  const unsigned* words[MR];
#pragma unroll
  for (int j = 0; j < MR; ++j) {
    const int r = r0 + 16 * j + c16;
    row[j] = r < p.m ? r : p.m - 1;
    words[j] = p.words + row[j] * p.row_words;
  }
  floatx4 tot[MR][NT], acc[MR][NT];
#pragma unroll
  for (int j = 0; j < MR; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) tot[j][n] = acc[j][n] = (floatx4){0.f, 0.f, 0.f, 0.f};
  Codes<BITS> c[MR];
  Affine<MODE, MR> f;
  auto load = [&](int kb) {
    if (kb < p.whole) {
#pragma unroll
      for (int j = 0; j < MR; ++j) load_codes<BITS, false>(c[j], words[j], (4 * kb + g) * BITS, (int)p.row_words);
    } else {
#pragma unroll
      for (int j = 0; j < MR; ++j) load_codes<BITS, true>(c[j], words[j], (4 * kb + g) * BITS, (int)p.row_words);
    }
    if (MODE != ROWS || kb == b0) load_affine<MODE, MR>(f, p, row, kb);
  };
  stage(b0, 0);
  load(b0);
  for (int kb = b0; kb < b1; ++kb) {
    const int buf = (kb - b0) & 1;
    wait_dma();
    __syncthreads();  // buffer `buf` is whole, the other no longer read
    Codes<BITS> now[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) now[j] = c[j];
    const Affine<MODE, MR> nowf = f;
    if (kb + 1 < b1) {
      stage(kb + 1, 1 - buf);
      load(kb + 1);
    }
    const float4* in = lds + buf * NP * (TOK * 16);
    block_products<BITS, MODE, NT, MR, NP>(
        tot, acc, now, nowf,
        [&](int n, int i, int q) {
          const int token = 16 * (NT * wt + n) + c16, piece = MODE == NARROW ? 4 * i + g : 4 * g + i;
          return __builtin_bit_cast(half8, in[q * (TOK * 16) + token * 16 + (piece ^ c16)]);
        },
        p, kb, b1 - 1, t0);
  }
  end_rows<BITS, MODE, NT, MR>(tot, acc, f, p, b1, t0);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (t0 + 16 * n < p.tokens) {
      const floatx4 f = factors(p, t0 + 16 * n);
      floatx4 out[MR];
#pragma unroll
      for (int j = 0; j < MR; ++j) out[j] = tot[j][n] * f;
      if (p.index && split == 0) add_adapters<MR>(out, p, t0 + 16 * n, r0);
      store_tile<MR>(out, p, t0 + 16 * n, r0, split);
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

// How a call is computed: tile (tokens of a workgroup; up to 64 stream_kernel, 128 tile_kernel), rows of a workgroup, waves
// along the columns, splits of the columns, and where its workspace holds what (floats).
struct Plan {
  int pieces, tile, rows, along, splits, split_blocks, mode, bits, rank_pad, slots, chunks, chunk;
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
  int64_t wgs, least;  // workgroups without splits, blocks of a split at least
  if (tokens <= 4 || (tokens <= 16 && q.pieces == 1 && cdiv(m, 64) < 192)) {
    q.tile = 16, q.rows = 16, q.along = 4, least = 16;
    wgs = cdiv(m, q.rows);
  } else if (tokens <= 64 || q.pieces == 2) {
    q.tile = tokens <= 16 ? 16 : tokens <= 32 || q.pieces == 2 ? 32 : 64;
    q.rows = 64, q.along = 1, least = 8;
    wgs = cdiv(m, q.rows) * cdiv(tokens, q.tile);
  } else {
    q.tile = 128, q.rows = 128, q.along = 1, least = 8;
    wgs = cdiv(m, q.rows) * cdiv(tokens, q.tile);
  }
  int64_t splits = wgs >= 192 ? 1 : cdiv(512, wgs);
  if (splits > cdiv(blocks, least)) splits = cdiv(blocks, least);
  if (splits > 64) splits = 64;
  q.split_blocks = (int)cdiv(blocks, splits);
  q.splits = (int)cdiv(blocks, q.split_blocks);
  q.rank_pad = adapters ? (int)((rank + 31) / 32 * 32) : 0;
  // the adapters' columns in chunks: about 512 workgroups, a chunk at least 1024 columns and at most 8 of them
  q.slots = adapters < 16 ? (int)adapters : 16;
  int64_t chunks = adapters ? cdiv(512, cdiv(tokens, 16) * q.slots) : 1;
  chunks = chunks > 8 ? 8 : chunks;
  q.chunk = (int)(cdiv(cdiv(n, chunks), 128) * 128);
  if (q.chunk < 1024) q.chunk = 1024;
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

// A kernel that may use all of a CU's LDS: said once for each device (the attribute is per device).
template <class K>
int allow_lds(K kernel) {
  static std::atomic<uint64_t> told{0};
  int dev = 0;
  const int rc = (int)hipGetDevice(&dev);
  if (rc) return rc;
  if (dev < 64 && told.load(std::memory_order_relaxed) >> dev & 1) return 0;
  const int set = (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           163840);
  if (!set && dev < 64) told.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  return set;
}

template <int BITS, int MODE, int NT, int TQ, int MR, int WK, int NP>
int launch_stream(const Linear& p, const Plan& q, hipStream_t st) {
  const auto kernel = stream_kernel<BITS, MODE, NT, TQ, MR, WK, NP>;
  if (const int rc = allow_lds(kernel)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(p.m, q.rows), (unsigned)cdiv(p.tokens, q.tile), (unsigned)q.splits), dim3(256),
                     (Ring<BITS, MODE, NT, TQ, MR, WK, NP>::BYTES), st, p);
  return (int)hipGetLastError();
}

template <int BITS, int MODE>
int launch_product(const Linear& p, const Plan& q, hipStream_t st) {
  if (q.pieces == 2)
    return q.along == 4 ? launch_stream<BITS, MODE, 1, 1, 1, 4, 2>(p, q, st)
                        : q.tile == 16 ? launch_stream<BITS, MODE, 1, 4, 1, 1, 2>(p, q, st)
                                       : launch_stream<BITS, MODE, 2, 8, 1, 1, 2>(p, q, st);
  if (q.along == 4)
    return p.tokens <= 4 ? launch_stream<BITS, MODE, 1, 1, 1, 4, 1>(p, q, st)
                         : launch_stream<BITS, MODE, 1, 4, 1, 4, 1>(p, q, st);
  if (q.tile == 16) return launch_stream<BITS, MODE, 1, 4, 1, 1, 1>(p, q, st);
  if (q.tile == 32) return launch_stream<BITS, MODE, 2, 8, 1, 1, 1>(p, q, st);
  if (q.tile == 64) return launch_stream<BITS, MODE, 4, 16, 1, 1, 1>(p, q, st);
  const auto kernel = tile_kernel<BITS, MODE, 4, 4, 2, 1>;
  if (const int rc = allow_lds(kernel)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(p.m, q.rows), (unsigned)cdiv(p.tokens, q.tile), (unsigned)q.splits), dim3(256),
                     (size_t)q.tile * 512, st, p);
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
  p.need_words = cdiv(n * bits, 32);
  p.whole = (int)(p.need_words / (4 * bits));
  p.corrected = zero || p.offset != __builtin_rintf(p.offset) || __builtin_fabsf(p.offset) > 512.f;
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
  const int64_t prep = tokens + (index ? q.slots * cdiv(tokens, 16) * q.chunks : 0);
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
