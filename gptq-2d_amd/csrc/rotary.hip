// Rotation of queries and keys by their positions, one launch for both; the gradient is the rotation back.
//
// Of a head's first r elements pair i, (x[i], x[i + r/2]) or interleaved (x[2 i], x[2 i + 1]), is turned by the angle t = p f_i:
//   y1 = a (x1 cos t - x2 sin t),  y2 = a (x2 cos t + x1 sin t);  its transpose turns by -t.
// The elements from r on are passed on.
//
// Frequencies are held as turns a position, in fp64: the product with a position leaves the fraction of a turn good to 2^-51 of
// the turns made (three roundings, the frequency's among them: 10^-6 of a radian at a position of 2^31 and f_i = 1), where fp32 would
// leave nothing of far positions.  The fraction is brought to an eighth of
// a turn around the nearest quarter, exactly, and only then rounded to fp32, for which the Taylor series of sine (to x^9) and
// cosine (to x^10) are good to 2^-28.  So an angle costs some 40 instructions and no memory (a table of 131072 positions and
// 64 pairs is 64 MB, and as many reads a head's worth each token).
//
// Bound by memory.  A workgroup takes a few tokens: it puts their cosines and sines into LDS, then walks over their heads, each
// thread with V pairs of a head (two loads of 16 bytes), BATCH heads in flight; neighbours take the next pairs, then the next
// heads, then the next token, so that it reads and writes in the order of memory.  16384 tokens, 40 heads of 128, inputs not in a
// cache: bf16 71 us, 4.7 TB/s (a large copy: 5.4; with cosines for each thread's own heads of one token, whose loads then lie a
// row apart, 80 us); 8 + 8 heads, fp32 55 us, 4.9 TB/s.
#include "elements.h"

namespace {

constexpr int THREADS = 256, BATCH = 4, PARTS = 2, DIM = 1024, PAIRS = 4096;  // the longest head; pairs of a workgroup's tokens

struct Part {
  const void* x;
  void* y;
  int heads;
  int64_t x_outer, x_token, x_head, y_outer, y_token, y_head;
};

struct Rotate {
  Part part[PARTS];
  int heads;     // of all parts
  unsigned mag;  // ceil(2^32 / heads): row / heads = umulhi(row, mag) for rows below 2^16
  int64_t inner;
  int blocks;  // workgroups of an outer index
  int tokens;  // of a workgroup
  int dim, rotated, turned, units;  // units of V pairs that turn, units of a row
  const double* turns;
  float amplitude;
  const void* positions;
  int64_t pos_outer, pos_inner;
  bool wide, back;
};

// cos and sin of `part` turns, any of them: |part| below 2^52.
__device__ __forceinline__ void cos_sin(double part, float& c, float& s) {
  const double r = part - __builtin_rint(part), q = __builtin_rint(4. * r);
  const float x = (float)(6.283185307179586 * __builtin_fma(-0.25, q, r)), x2 = x * x;  // [-pi/4, pi/4]
  float a = __builtin_fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);
  a = __builtin_fmaf(x2, a, 8.3333333e-3f);
  a = __builtin_fmaf(x2, a, -1.6666667e-1f);
  a = __builtin_fmaf(x * x2, a, x);
  float b = __builtin_fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
  b = __builtin_fmaf(x2, b, -1.3888889e-3f);
  b = __builtin_fmaf(x2, b, 4.1666667e-2f);
  b = __builtin_fmaf(x2, b, -0.5f);
  b = __builtin_fmaf(x2, b, 1.f);
  const int quarter = (int)q;  // -2 .. 2
  const float cc = quarter & 1 ? a : b, ss = quarter & 1 ? b : a;
  c = (quarter + 1) & 2 ? -cc : cc;
  s = quarter & 2 ? -ss : ss;
}

template <int TYPE>
__device__ __forceinline__ void round_all(typename Elem<TYPE>::T (&to)[16 / sizeof(typename Elem<TYPE>::T)],
                                          const float (&x)[16 / sizeof(typename Elem<TYPE>::T)]) {
  constexpr int V = 16 / sizeof(typename Elem<TYPE>::T);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (TYPE == TYPE_BF16) {
      to[i] = __builtin_bit_cast(uint16_t, (__bf16)x[i]);  // to nearest even, one instruction a pair
    } else {
      float y = x[i];
      if constexpr (TYPE == TYPE_F16) asm("" : "+v"(y));  // rounded to fp32 first everywhere, or the same row's bits vary with its place
      to[i] = (typename Elem<TYPE>::T)y;
    }
  }
}

template <int TYPE, bool INTERLEAVED>
__global__ __launch_bounds__(THREADS) void rotary_kernel(Rotate a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int V = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  alignas(16) __shared__ float cosines[PAIRS], sines[PAIRS];
  const int64_t o = blockIdx.x / a.blocks, first = (int64_t)(blockIdx.x - o * a.blocks) * a.tokens;
  const int tokens = (int)(a.inner - first < a.tokens ? a.inner - first : a.tokens);
  const int half = a.rotated / 2, pairs = a.turned * V;
  for (int u = threadIdx.x; u < tokens * pairs; u += THREADS) {
    const int t = u / pairs, i = u - t * pairs;
    const int64_t at = o * a.pos_outer + (first + t) * a.pos_inner;
    const double p = a.wide ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
    float c, s;
    cos_sin(p * a.turns[i < half ? i : half - 1], c, s);
    cosines[u] = c * a.amplitude;
    sines[u] = s * (a.back ? -a.amplitude : a.amplitude);
  }
  __syncthreads();
  // this thread's unit of a row, and its rows: (token, head) numbers from row0 on, `step` apart
  const int row0 = threadIdx.x / a.units, unit = threadIdx.x - row0 * a.units, step = THREADS / a.units, rows = tokens * a.heads;
  if (row0 >= step) return;
  const bool turned = unit < a.turned;
  int d0, d1, n0, n1;  // the unit's two runs of V elements, and how many of each there are
  if (turned) {
    const int i0 = unit * V, n = half - i0 < V ? half - i0 : V;
    if (INTERLEAVED) {
      d0 = 2 * i0, d1 = d0 + V;
      n0 = 2 * n < V ? 2 * n : V, n1 = 2 * n - n0;
    } else {
      d0 = i0, d1 = half + i0;
      n0 = n1 = n;
    }
  } else {
    d0 = a.rotated + (unit - a.turned) * 2 * V, d1 = d0 + V;
    n0 = a.dim - d0 < V ? a.dim - d0 : V;
    n1 = a.dim - d1 < 0 ? 0 : a.dim - d1 < V ? a.dim - d1 : V;
  }
  const bool whole = n0 == V && n1 == V;
  for (int r = row0; r < rows; r += step * BATCH) {
    vec u[BATCH], w[BATCH];
    T* to[BATCH];
    int token[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int row = r + b * step < rows ? r + b * step : rows - 1, t = a.heads > 1 ? (int)__umulhi((unsigned)row, a.mag) : row;
      const int g = row - t * a.heads, second = g >= a.part[0].heads;
      const Part& part = a.part[second];
      const int head = second ? g - a.part[0].heads : g;
      const T* from = (const T*)part.x + o * part.x_outer + (first + t) * part.x_token + head * part.x_head;
      to[b] = (T*)part.y + o * part.y_outer + (first + t) * part.y_token + head * part.y_head;
      token[b] = t;
      if (whole) {
        u[b] = *reinterpret_cast<const vec*>(from + d0);
        w[b] = *reinterpret_cast<const vec*>(from + d1);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          u[b][i] = i < n0 ? from[d0 + i] : (T)0;
          w[b][i] = i < n1 ? from[d1 + i] : (T)0;
        }
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (r + b * step >= rows) break;
      if (turned) {
        float c[V], s[V], y0[V], y1[V];
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const floatx4 cc = *reinterpret_cast<const floatx4*>(&cosines[token[b] * pairs + unit * V + i]);
          const floatx4 ss = *reinterpret_cast<const floatx4*>(&sines[token[b] * pairs + unit * V + i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) c[i + j] = cc[j], s[i + j] = ss[j];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // pair i of the unit: elements of the two runs, or neighbours in the 2 V of both
          if (INTERLEAVED) {
            const int j = 2 * i;
            const float x1 = to_f32<TYPE>(j < V ? u[b][j % V] : w[b][j % V]);
            const float x2 = to_f32<TYPE>(j < V ? u[b][(j + 1) % V] : w[b][(j + 1) % V]);
            const float r1 = __builtin_fmaf(x1, c[i], -x2 * s[i]), r2 = __builtin_fmaf(x2, c[i], x1 * s[i]);
            (j < V ? y0 : y1)[j % V] = r1;
            (j < V ? y0 : y1)[(j + 1) % V] = r2;
          } else {
            const float x1 = to_f32<TYPE>(u[b][i]), x2 = to_f32<TYPE>(w[b][i]);
            y0[i] = __builtin_fmaf(x1, c[i], -x2 * s[i]);
            y1[i] = __builtin_fmaf(x2, c[i], x1 * s[i]);
          }
        }
        T r0[V], r1[V];
        round_all<TYPE>(r0, y0);
        round_all<TYPE>(r1, y1);
#pragma unroll
        for (int i = 0; i < V; ++i) u[b][i] = r0[i], w[b][i] = r1[i];
      }
      if (whole) {
        *reinterpret_cast<vec*>(to[b] + d0) = u[b];
        *reinterpret_cast<vec*>(to[b] + d1) = w[b];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (i < n0) to[b][d0 + i] = u[b][i];
          if (i < n1) to[b][d1 + i] = w[b][i];
        }
      }
    }
  }
}

// Tokens of a workgroup: as many as give every thread BATCH rows, but no more than leave two workgroups a CU, and a row each at
// least (40 heads of 128, bf16, 1, 2, 4, 8 and 16 tokens: 64 tokens 14.4, 14.0, 14.4, 14.5, 15.8 us with the call; 4096 31, 23, 23,
// 24, 31; 16384 101, 71, 73, 72, 73).
inline int tokens_of(const Rotate& a, int64_t outer, int V) {
  const int64_t step = THREADS / a.units, least = (step + a.heads - 1) / a.heads;
  int64_t t = (step * BATCH + a.heads - 1) / a.heads;
  while (t > least && outer * ((a.inner + t - 1) / t) < 512) t /= 2;
  const int64_t most = PAIRS / (a.turned * V);
  t = t < least ? least : t;
  t = t < most ? t : most;
  while (t > 1 && t * a.heads > 0xffff) t /= 2;
  return (int)t;
}

template <int TYPE>
int launch(Rotate& a, int64_t outer, bool interleaved, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(typename Elem<TYPE>::T);
  a.turned = (a.rotated / 2 + V - 1) / V;
  a.units = a.turned + (a.dim - a.rotated + 2 * V - 1) / (2 * V);
  static_assert(DIM / 2 / 4 + 1 <= THREADS && DIM / 2 + 4 <= PAIRS, "a row's units have a thread each, a token's pairs their place");
  a.tokens = tokens_of(a, outer, V);
  const int64_t blocks = (a.inner + a.tokens - 1) / a.tokens;
  if (outer * blocks > 0xffffff) return GPTQ2D_EUNSUPPORTED;  // 2^32 threads
  a.blocks = (int)blocks;
  const dim3 grid((unsigned)(outer * blocks));
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<TYPE, true>), grid, dim3(THREADS), 0, st, a);
  else
    hipLaunchKernelGGL((rotary_kernel<TYPE, false>), grid, dim3(THREADS), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int gptq2d_rotary(const void* x0, int64_t x0_outer, int64_t x0_token, int64_t x0_head, void* y0, int64_t y0_outer,
                             int64_t y0_token, int64_t y0_head, int32_t heads0, const void* x1, int64_t x1_outer,
                             int64_t x1_token, int64_t x1_head, void* y1, int64_t y1_outer, int64_t y1_token, int64_t y1_head,
                             int32_t heads1, int32_t type, int64_t outer, int64_t inner, int32_t dim, int32_t rotated,
                             int32_t interleaved, const double* turns, double amplitude, const void* positions, int32_t wide,
                             int64_t pos_outer, int64_t pos_inner, int32_t back, void* stream) {
  if (heads0 < 0 || heads0 > 0x7fff || heads1 < 0 || heads1 > 0x7fff || outer < 0 || inner < 0 || dim < 2 || dim > DIM || rotated < 2 || rotated > dim ||
      rotated % 2)
    return GPTQ2D_EINVAL;
  if (outer > 0x7fffffff || inner > 0x7fffffff) return GPTQ2D_EUNSUPPORTED;
  Rotate a = {};
  a.part[0] = {x0, y0, heads0, x0_outer, x0_token, x0_head, y0_outer, y0_token, y0_head};
  a.part[1] = {x1, y1, heads1, x1_outer, x1_token, x1_head, y1_outer, y1_token, y1_head};
  if (outer * inner == 0 || heads0 + heads1 == 0) return 0;
  a.heads = heads0 + heads1;
  a.mag = (unsigned)((((uint64_t)1 << 32) + a.heads - 1) / a.heads);
  a.inner = inner, a.dim = dim, a.rotated = rotated;
  a.turns = turns, a.amplitude = (float)amplitude;
  a.positions = positions, a.wide = wide != 0, a.pos_outer = pos_outer, a.pos_inner = pos_inner;
  a.back = back != 0;
  const hipStream_t st = (hipStream_t)stream;
  switch (type) {
    case TYPE_F32:
      return launch<TYPE_F32>(a, outer, interleaved != 0, st);
    case TYPE_BF16:
      return launch<TYPE_BF16>(a, outer, interleaved != 0, st);
    case TYPE_F16:
      return launch<TYPE_F16>(a, outer, interleaved != 0, st);
  }
  return GPTQ2D_EINVAL;
}
