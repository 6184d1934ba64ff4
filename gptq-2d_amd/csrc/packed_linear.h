// Products with a packed INT layer: what the kernels of packed_linear.hip share.
//
//   y[t, i] = sum_k x[t, k] (u[i, k] - w[i, k / group]) s[i, k / group],  w = zero point - qmin,
// u the code in the layer's bit field (pack.hip).  The matrix cores multiply fp16 activations by u - 2^(bits - 1), which
// fp16 holds exactly, less the nearest whole number to what w differs from that; a group's products are summed in fp32 and
// then multiplied by its scale, and the rest of w (0 for whole zero points) is taken off through the sum of the group's
// activations.  Activations are scaled by a power of two per token, the largest finite element to 2^14..2^15, where fp16 has
// steps of 2^-24 at the least: an element is held to 22 bits (fp32, in two pieces; those of bf16 and fp16 are all held), or to
// 2^-39 of the token's largest where that is coarser -- below an fp32 sum's rounding, unless the largest element's weight is 0.
// So no weight is rounded, whatever its scale, and a whole zero point costs nothing.
#pragma once

#include "elements.h"
#include "lds_dma.h"
#include "split_mma.h"

namespace {

// Order of a run of eight activations in memory: element j and j + 4 side by side, as the codes' pairs come out.
// Operands: lane l holds row (token) or column (row of W) l % 16 and the eight k of its part g = l / 16 of a step.
// WIDE (groups that a block of 128 columns does not cut): in step i part g holds k = 32 g + 8 i .. + 7 of the block, so that a
// lane's 32 codes are one run of its row.  Otherwise k = 32 i + 8 g .. + 7, so that a step stays inside a group; the
// words change places between the four parts for that (four permlane swaps for 32 codes).

// The codes of 128 columns of 16 rows, as loaded: this lane's 32 (BITS words).
template <int BITS>
struct Codes {
  unsigned w[BITS];
};

// Words at .. at + BITS - 1 of a row (vector loads need only a word's own alignment); GUARD: zeros from word `end` on, the
// end of those that hold codes (the next row may begin anywhere after it, the last one has nothing behind it), where the
// activations are zeros.
template <int BITS, bool GUARD>
__device__ __forceinline__ void load_codes(Codes<BITS>& c, const unsigned* row, int at, int end) {
  typedef unsigned vec4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef unsigned vec3 __attribute__((ext_vector_type(3), aligned(4)));
  typedef unsigned vec2 __attribute__((ext_vector_type(2), aligned(4)));
  if constexpr (GUARD) {
#pragma unroll
    for (int i = 0; i < BITS; ++i) {
      c.w[i] = 0;
      if (at + i < end) c.w[i] = row[at + i];
    }
  } else if constexpr (BITS == 2) {
    const vec2 v = *reinterpret_cast<const vec2*>(row + at);
    c.w[0] = v[0], c.w[1] = v[1];
  } else if constexpr (BITS == 3) {
    const vec3 v = *reinterpret_cast<const vec3*>(row + at);
    c.w[0] = v[0], c.w[1] = v[1], c.w[2] = v[2];
  } else {
#pragma unroll
    for (int i = 0; i < BITS; i += 4) {
      const vec4 v = *reinterpret_cast<const vec4*>(row + at + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) c.w[i + j] = v[j];
    }
  }
}

// Step i's eight codes of the lane, as they lie: 8 BITS bits in one word (two for 8 bits).
template <int BITS>
struct Run {
  unsigned w[BITS == 8 ? 2 : 1];
};

template <int BITS>
__device__ __forceinline__ void split_runs(Run<BITS> (&r)[4], const Codes<BITS>& c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BITS == 8) {
      r[i].w[0] = c.w[2 * i], r[i].w[1] = c.w[2 * i + 1];
    } else if constexpr (BITS == 4) {
      r[i].w[0] = c.w[i];
    } else if constexpr (BITS == 3) {
      r[i].w[0] = i == 0 ? c.w[0]
                         : i == 1 ? __builtin_amdgcn_alignbit(c.w[1], c.w[0], 24)
                                  : i == 2 ? __builtin_amdgcn_alignbit(c.w[2], c.w[1], 16) : c.w[2] >> 8;
    } else {
      r[i].w[0] = i % 2 ? c.w[i / 2] >> 16 : c.w[i / 2];
    }
  }
}

// r[i] of part g becomes r[g] of part i: 4 x 4 words exchanged between the lanes l, l + 16, l + 32, l + 48.
__device__ __forceinline__ void swap_parts(unsigned& a, unsigned& b, unsigned& c, unsigned& d) {
  typedef unsigned pair __attribute__((ext_vector_type(2)));
  pair p = __builtin_amdgcn_permlane32_swap(a, c, false, false);
  a = p[0], c = p[1];
  p = __builtin_amdgcn_permlane32_swap(b, d, false, false);
  b = p[0], d = p[1];
  p = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = p[0], b = p[1];
  p = __builtin_amdgcn_permlane16_swap(c, d, false, false);
  c = p[0], d = p[1];
}

// What is taken off the codes of a row's group: 2^(BITS - 1) and, where the zero point is that far from it, the whole number
// nearest to the rest; the rest of the rest (0 for zero points that are whole) goes through the activations' sum.
template <int BITS>
struct Middle {
  half2v k[BITS == 8 ? 1 : BITS == 4 ? 2 : BITS == 3 ? 3 : 4];
};

template <int BITS>
__device__ __forceinline__ float split_shift(Middle<BITS>& m, float shift) {
  float whole = round_even(shift);
  whole = __builtin_fabsf(whole) <= 512.f ? whole : 0.f;  // fp16 holds 1024 + 128 + 512; also for a NaN
  const half2v w = both(whole);
  if constexpr (BITS == 8) {
    m.k[0] = both(-1152.f) - w;
  } else if constexpr (BITS == 4) {
    m.k[0] = both(-1032.f) - w, m.k[1] = both(-72.f) - w;
  } else if constexpr (BITS == 3) {
    m.k[0] = both(-1028.f) - w, m.k[1] = both(-132.f) - w, m.k[2] = both(-20.f) - w;
  } else {
    m.k[0] = both(-1026.f) - w, m.k[1] = both(-258.f) - w, m.k[2] = both(-66.f) - w, m.k[3] = both(-18.f) - w;
  }
  return shift - whole;
}

// The eight codes of a run less their middle, in fp16 in the activations' order.  1024 + c 2^p is an fp16 number with the
// code in its low bits: a mask brings two codes of a word whose halves hold four each, one packed operation takes 1024,
// the factor and the middle away, exactly: nine instructions for eight 4-bit codes.
template <int BITS>
__device__ __forceinline__ half8 centred(const Run<BITS>& r, const Middle<BITS>& m) {
  union {
    half2v h[4];
    half8 v;
  } o;
  if constexpr (BITS == 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o.h[j] = as_half2(__builtin_amdgcn_perm(r.w[1], r.w[0], 0x0c040c00u + j * 0x00010001u) | 0x64006400u) + m.k[0];
  } else if constexpr (BITS == 4) {
    const unsigned a = r.w[0], b = a >> 8;
    o.h[0] = codes_at(a, 0x000f000fu) + m.k[0];
    o.h[1] = __builtin_elementwise_fma(codes_at(a, 0x00f000f0u), both(0.0625f), m.k[1]);
    o.h[2] = codes_at(b, 0x000f000fu) + m.k[0];
    o.h[3] = __builtin_elementwise_fma(codes_at(b, 0x00f000f0u), both(0.0625f), m.k[1]);
  } else if constexpr (BITS == 3) {
    const unsigned a = (r.w[0] & 0xfffu) | (r.w[0] << 4 & 0x0fff0000u), b = a >> 3;
    o.h[0] = codes_at(a, 0x00070007u) + m.k[0];
    o.h[1] = __builtin_elementwise_fma(codes_at(a, 0x00380038u), both(0.125f), m.k[1]);
    o.h[2] = __builtin_elementwise_fma(codes_at(a, 0x01c001c0u), both(0.015625f), m.k[2]);
    o.h[3] = __builtin_elementwise_fma(codes_at(b, 0x01c001c0u), both(0.015625f), m.k[2]);
  } else {
    const unsigned a = (r.w[0] & 0xffu) | (r.w[0] << 8 & 0x00ff0000u);
    o.h[0] = codes_at(a, 0x00030003u) + m.k[0];
    o.h[1] = __builtin_elementwise_fma(codes_at(a, 0x000c000cu), both(0.25f), m.k[1]);
    o.h[2] = __builtin_elementwise_fma(codes_at(a, 0x00300030u), both(0.0625f), m.k[2]);
    o.h[3] = __builtin_elementwise_fma(codes_at(a, 0x00c000c0u), both(0.015625f), m.k[3]);
  }
  return o.v;
}

// The four steps' runs of a block of 128 columns.
template <int BITS, bool WIDE>
__device__ __forceinline__ void step_runs(Run<BITS> (&r)[4], const Codes<BITS>& c) {
  split_runs<BITS>(r, c);
  if constexpr (!WIDE) {
    swap_parts(r[0].w[0], r[1].w[0], r[2].w[0], r[3].w[0]);
    if constexpr (BITS == 8) swap_parts(r[0].w[1], r[1].w[1], r[2].w[1], r[3].w[1]);
  }
}

__device__ __forceinline__ floatx4 mma(half8 a, half8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mma(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A call, as its kernels take it.
struct Linear {
  int tokens, m, n, blocks;  // blocks of 128 columns
  int whole;                 // of which a row's words hold all
  int64_t need_words;        // of a row
  // layer
  const unsigned* words;
  int64_t row_words;
  const float* scale;
  const float* zero;  // or none: `offset` everywhere
  int64_t scale_row, scale_col, zero_row, zero_col;
  float offset;    // -qmin - 2^(bits - 1)
  int group;       // columns of a group, a multiple of 32 (whole rows: 128 blocks)
  unsigned steps;  // group / 32 (not WIDE: steps of 32 columns of a group) or group / 128
  unsigned mag;    // of the division by `steps`
  bool corrected;  // zero points, or an offset that is no whole number
  // activations
  const void* x;
  int64_t x_token;
  int type;
  _Float16* xp;  // [pieces][tokens][128 blocks], their factor back [tokens], sums of groups [groups][tokens to 16]
  int64_t piece;
  float* factor;
  float* sums;
  int64_t sums_row;
  int groups;
  // adapters, or none (index null)
  const void* a;
  const void* b;
  const float* scaling;
  const int32_t* index;
  int adapters, rank, rank_pad, slots, chunks, chunk;  // v: [chunks][tokens][rank_pad]; columns of a chunk
  float* v;
  // result
  void* y;
  int64_t y_token;
  const void* bias;
  int splits, split_blocks;
  float* part;  // [splits][tokens][m] where splits > 1
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int type) {
  if (type == TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == TYPE_BF16) return to_f32<TYPE_BF16>(static_cast<const uint16_t*>(p)[i]);
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int type, float x) {
  if (type == TYPE_F32)
    static_cast<float*>(p)[i] = x;
  else if (type == TYPE_BF16)
    static_cast<uint16_t*>(p)[i] = from_f32<TYPE_BF16>(x);
  else
    static_cast<_Float16*>(p)[i] = (_Float16)x;
}
// The index of the adapter of token t, -1 for none.
__device__ __forceinline__ int adapter_of(const Linear& p, int t) {
  const int a = t < p.tokens ? p.index[t] : -1;
  return a >= 0 && a < p.adapters ? a : -1;
}

// tot[j][n] += V B^T for the 16 NT tokens from t0 and the rows r0 + 16 j of W, one distinct adapter of the tokens after the
// other; its B is read once for all of them.  The other tokens' rows of V are zeros, and what they make of B is dropped: an
// infinity or NaN in one request's adapter stays in its own tokens.  V (fp32) and B (fp16 or bf16) are taken in bf16
// pieces: six products, 2^-23 of the result; of bf16 adapters B is one piece, and two of V leave out 2^-17.  For long
// batches, where a wave's tokens have few adapters.
template <int MR, int NT>
__device__ __forceinline__ void add_adapters(floatx4 (&tot)[MR][NT], const Linear& p, int t0, int r0) {
  static_assert(16 * NT <= 64, "a lane a token");
  const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const int mine = lane < 16 * NT ? adapter_of(p, t0 + lane) : -1;
  uint64_t pending = __builtin_amdgcn_ballot_w64(mine >= 0);
  while (pending) {
    const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(pending));
    const uint64_t same = __builtin_amdgcn_ballot_w64(mine == a);
    pending &= ~same;
    const float c = p.scaling ? p.scaling[a] : 1.f;
    for (int j0 = 0; j0 < p.rank_pad; j0 += 32) {
      Raw8<TYPE_BF16> b[MR];  // the bits of either type
#pragma unroll
      for (int j = 0; j < MR; ++j) {
        const int r = r0 + 16 * j + c16;
        b[j].load(static_cast<const uint16_t*>(p.b) + ((int64_t)a * p.m + (r < p.m ? r : p.m - 1)) * p.rank, j0 + 8 * g, p.rank);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const unsigned these = (unsigned)(same >> (16 * n)) & 0xffffu;
        if (!these) continue;
        float v[8] = {};
        if (these >> c16 & 1u) {
          const float* row = p.v + (int64_t)(t0 + 16 * n + c16) * p.rank_pad + j0 + 8 * g;
#pragma unroll 2
          for (int k = 0; k < p.chunks; ++k) {
            const float4 lo = *reinterpret_cast<const float4*>(row), hi = *reinterpret_cast<const float4*>(row + 4);
            v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
            v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
            row += (int64_t)p.tokens * p.rank_pad;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= c;
        }
        bf16x8 vp[3];
        split8(v, vp);
        floatx4 before[MR];
#pragma unroll
        for (int j = 0; j < MR; ++j) before[j] = tot[j][n];
        if (p.type == TYPE_BF16) {
#pragma unroll
          for (int q = 1; q >= 0; --q)
#pragma unroll
            for (int j = 0; j < MR; ++j) tot[j][n] = mma(vp[q], __builtin_bit_cast(bf16x8, b[j].v[0]), tot[j][n]);
        } else {
#pragma unroll
          for (int j = 0; j < MR; ++j) {
            const half8 h = __builtin_bit_cast(half8, b[j].v[0]);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
            bf16x8 bp[3];
            split8(x, bp);
#pragma unroll
            for (int q = 0; q < NPROD; ++q) tot[j][n] = mma(vp[prod_a[q]], bp[prod_b[q]], tot[j][n]);
          }
        }
        if (these != 0xffffu) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < MR; ++j) tot[j][n][i] = these >> (4 * g + i) & 1u ? tot[j][n][i] : before[j][i];
        }
      }
    }
  }
}

// acc[n] += V B^T for the tokens t0 + 16 n + 4 g .. + 3 and the lane's row r of W, each token with its own adapter: for short
// batches, where every token may have another one.  Eight ranks at a time, dealt to `shares` waves that sum apart; the
// loads of four tokens are in flight together.  NP: fp32 elements where 2.
template <int NT, int NP>
__device__ __forceinline__ void add_own_adapters(floatx4 (&acc)[NT], const Linear& p, int t0, int r, int share, int shares) {
  typedef unsigned vec __attribute__((ext_vector_type(4), aligned(2)));
  const int g = threadIdx.x >> 4 & 3, row = r < p.m ? r : p.m - 1;
  if (8 * share >= p.rank) return;
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {
    const int t = t0 + 16 * n + 4 * g;
    int a[4];
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = adapter_of(p, t + i);
    if (!__builtin_amdgcn_ballot_w64(a[0] >= 0 || a[1] >= 0 || a[2] >= 0 || a[3] >= 0)) continue;
    for (int j = 8 * share; j < p.rank; j += 8 * shares) {
      vec b[4][NP];
      const bool whole = j + 8 <= p.rank;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* at = static_cast<const char*>(p.b) + (((int64_t)(a[i] < 0 ? 0 : a[i]) * p.m + row) * p.rank + j) * (2 * NP);
        if (whole) {
#pragma unroll
          for (int q = 0; q < NP; ++q) b[i][q] = *reinterpret_cast<const vec*>(at + 16 * q);
        } else {
          typedef typename std::conditional<NP == 2, unsigned, uint16_t>::type E;
          union {
            E e[8];
            unsigned u[4 * NP];
          } x;
#pragma unroll
          for (int e = 0; e < 8; ++e) x.e[e] = j + e < p.rank ? reinterpret_cast<const E*>(at)[e] : (E)0;
#pragma unroll
          for (int e = 0; e < 4 * NP; ++e) b[i][e / 4][e % 4] = x.u[e];
        }
      }
      float v[4][8] = {};
      const float* at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) at[i] = p.v + (int64_t)(a[i] < 0 ? 0 : t + i) * p.rank_pad + j;
#pragma unroll 1
      for (int k = 0; k < p.chunks; ++k) {
        float4 x[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i][0] = *reinterpret_cast<const float4*>(at[i]), x[i][1] = *reinterpret_cast<const float4*>(at[i] + 4);
          at[i] += (int64_t)p.tokens * p.rank_pad;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            v[i][4 * h] += x[i][h].x, v[i][4 * h + 1] += x[i][h].y, v[i][4 * h + 2] += x[i][h].z, v[i][4 * h + 3] += x[i][h].w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float add = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float w;
          if constexpr (NP == 2) {
            w = __uint_as_float(b[i][e / 4][e % 4]);
          } else {
            const unsigned u = b[i][0][e / 2] >> (e % 2 * 16) & 0xffffu;
            w = p.type == TYPE_BF16 ? __uint_as_float(u << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)u);
          }
          add = __builtin_fmaf(v[i][e], w, add);
        }
        sum[i] += a[i] < 0 ? 0.f : add;  // without an adapter whatever was read
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (a[i] >= 0 && p.scaling) sum[i] *= p.scaling[a[i]];
#pragma unroll
    for (int m = 0; m < NT; ++m)
      if (m == n) acc[m] += sum;
  }
}

// Groups: whole rows, multiples of 128 columns, other multiples of 32; the last two with zero points or without.
enum { ROWS = 0, WIDE = 1, NARROW = 2, ZEROS = 4 };
__host__ __device__ constexpr bool narrow(int mode) { return (mode & 3) == NARROW; }
__host__ __device__ constexpr bool wide(int mode) { return (mode & 3) == WIDE; }
__host__ __device__ constexpr bool zeros(int mode) { return mode & ZEROS; }

// How a call is computed: tile (tokens of a workgroup; up to 64 stream_kernel, 128 tile_kernel), rows of a workgroup, splits
// of the columns, and where its workspace holds what (floats).
struct Plan {
  int pieces, tile, rows, splits, split_blocks, mode, rank_pad, slots, chunks, chunk;
  int64_t groups, sums_row, xp, factor, sums, v, part, total;  // offsets; total: floats
};

}  // namespace

// launch_mode<BITS> of a Linear and a Plan, one source file each.
#define GPTQ2D_PACKED_PRODUCT(BITS) \
  __attribute__((visibility("hidden"))) int packed_product_bits##BITS(const void* linear, const void* plan, hipStream_t st)
GPTQ2D_PACKED_PRODUCT(2);
GPTQ2D_PACKED_PRODUCT(3);
GPTQ2D_PACKED_PRODUCT(4);
GPTQ2D_PACKED_PRODUCT(8);
