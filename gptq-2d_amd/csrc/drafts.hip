// Trees of drafted tokens: who comes from whom, which of them are accepted, and the accepted ones' entries in the 4-bit cache.
//
// A sequence's nodes are numbered from 0 on, each after the one that it follows (its parent; -1 or anything else that is no earlier node:
// none).  All of these calls are bound by latency: a workgroup or a wave a sequence, no step longer than the tree is deep.
#include "kv_cache.h"

namespace {

constexpr int MOST = 512, THREADS = 256;  // nodes of a tree

struct Nodes {
  const int32_t* parents;
  const int32_t* offsets;
  int64_t seqs, tokens;
  int nodes, words;
};

__device__ __forceinline__ int64_t row_of(const Nodes& t, int64_t b) {
  const int64_t o = t.offsets[b];
  return o < 0 ? 0 : o > t.tokens ? t.tokens : o;
}

// Each node's ancestors and itself as bits, and its position.  Pointers are doubled: with the ancestors of up to 2^k steps and
// the one 2^k steps away known of all, a node's next 2^k are those of the latter, so a tree of depth d takes log2 d rounds.
// (A round reads sets that others of it may have widened already: by ancestors all the same.)  64 trees of 24 nodes: 5 us.
__global__ __launch_bounds__(THREADS) void tree_kernel(Nodes t, const int32_t* held, unsigned* ancestors, int32_t* positions) {
  __shared__ unsigned bits[MOST * (MOST / 32)];
  __shared__ int jump[MOST];
  const int64_t b = blockIdx.x;
  if (b == t.seqs) {  // rows that no sequence has
    const int64_t first = t.seqs ? row_of(t, 0) : 0, end = t.seqs ? row_of(t, t.seqs) : 0;
    for (int64_t r = threadIdx.x; r < t.tokens; r += THREADS) {
      if (r >= first && r < end) r += (end - r - 1) / THREADS * THREADS;  // past those of the sequences
      if (r < first || r >= end) {
        positions[r] = 0;
        for (int w = 0; w < t.words; ++w) ancestors[r * t.words + w] = 0;
      }
    }
    return;
  }
  const int64_t row = row_of(t, b), all = row_of(t, b + 1) - row;
  const int n = (int)(all < t.nodes ? (all > 0 ? all : 0) : t.nodes), words = t.words, start = held[b];
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int p = t.parents[row + i];
    jump[i] = p >= 0 && p < i ? p : -1;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < n * words; u += THREADS) {
    const int i = u / words, w = u - i * words, p = jump[i];
    bits[u] = (i / 32 == w ? 1u << i % 32 : 0u) | (p >= 0 && p / 32 == w ? 1u << p % 32 : 0u);
  }
  for (;;) {
    __syncthreads();
    for (int u = threadIdx.x; u < n * words; u += THREADS) {
      const int i = u / words, j = jump[i];
      if (j >= 0) bits[u] |= bits[j * words + (u - i * words)];
    }
    int next[MOST / THREADS];
#pragma unroll
    for (int k = 0; k < MOST / THREADS; ++k) {
      const int i = threadIdx.x + k * THREADS, j = i < n ? jump[i] : -1;
      next[k] = j >= 0 ? jump[j] : -1;
    }
    __syncthreads();
    bool more = false;
#pragma unroll
    for (int k = 0; k < MOST / THREADS; ++k) {
      const int i = threadIdx.x + k * THREADS;
      if (i < n) jump[i] = next[k];
      more |= next[k] >= 0;
    }
    if (!__syncthreads_or(more)) break;
  }
  for (int u = threadIdx.x; u < n * words; u += THREADS) ancestors[row * words + u] = bits[u];
  for (int i = threadIdx.x; i < n; i += THREADS) {
    int depth = -1;
    for (int w = 0; w < words; ++w) depth += __popc(bits[i * words + w]);
    positions[row + i] = start + depth;
  }
  for (int64_t i = n + threadIdx.x; i < all; i += THREADS) {  // more nodes than there may be: they see what was held
    positions[row + i] = start;
    for (int w = 0; w < words; ++w) ancestors[(row + i) * words + w] = 0;
  }
}

// From node 0, the one that needs no accepting, to the first child whose token was chosen, and on from there.  A wave a tree:
// a lane looks at every 64th node.
template <class T>
__global__ __launch_bounds__(64) void accept_kernel(Nodes t, const T* drafted, const T* chosen, int32_t* path, int32_t* counts,
                                                    T* last) {
  __shared__ int follows[MOST];  // the parent whose chosen token the node is, or none
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x;
  const int64_t row = row_of(t, b), all = row_of(t, b + 1) - row;
  const int n = (int)(all < t.nodes ? (all > 0 ? all : 0) : t.nodes);
  for (int i = lane; i < n; i += 64) {
    const int p = t.parents[row + i];
    follows[i] = p >= 0 && p < i && drafted[row + i] == chosen[row + p] ? p : -1;
  }
  __syncthreads();
  int count = 0, node = 0;
  int32_t* mine = path + b * t.nodes;
  if (n > 0) {
    for (;;) {
      if (lane == 0) mine[count] = node;
      ++count;
      int child = -1;
      for (int i = node + 1; i < n; i += 64) {
        const uint64_t found = __builtin_amdgcn_ballot_w64(i + lane < n && follows[i + lane] == node);
        if (found) {
          child = i + __builtin_ctzll(found);
          break;
        }
      }
      if (child < 0) break;
      node = child;
    }
  }
  for (int i = count + lane; i < t.nodes; i += 64) mine[i] = -1;
  if (lane == 0) {
    counts[b] = count;
    last[b] = n > 0 ? chosen[row + node] : (T)-1;
  }
}

// The entries of the nodes path[0] < path[1] < ... of a sequence (its last tokens) to the places of its nodes 0, 1, ...
//
// A workgroup takes one head's keys or values of one sequence, a block of 32 places at a time: all of its sources are read
// before any of its places is written, and the sources of later places lie behind them, since the path ascends.  Words of K
// hold one token and move whole; those of V hold eight, whose nibbles go through LDS, and the others' stay.
template <int ND>
__global__ __launch_bounds__(THREADS) void keep_kernel(KvCache c, const int32_t* path, int64_t path_stride, int most,
                                                       const int32_t* counts) {
  constexpr int DP = 64 * ND;
  __shared__ unsigned codes[32][DP / 4 + 1];  // V: codes of a token, a byte each
  const int64_t b = blockIdx.x;
  const int h = blockIdx.y;
  const bool value = blockIdx.z;
  const int64_t t0 = kv_offset(c, b), t1 = kv_offset(c, b + 1), n = t1 - t0;
  const int64_t start = (int64_t)c.lengths[b] - n, room = (int64_t)c.width * c.page;
  const int32_t* mine = path + b * path_stride;
  const int lane = threadIdx.x & 63;
  int count = counts[b] < most ? counts[b] : most;
  for (int i = 0; i < count; i += 64) {  // as far as it ascends among the sequence's nodes
    const int at = i + lane;
    const bool bad = at < count && (mine[at] >= n || mine[at] <= (at ? mine[at - 1] : -1));
    const uint64_t found = __builtin_amdgcn_ballot_w64(bad);
    if (found) {
      count = i + __builtin_ctzll(found);
      break;
    }
  }
  if (count <= 0 || n <= 0) return;
  const int64_t head = (int64_t)h * kv_head_words(ND, c.page);
  const int token = threadIdx.x >> 3, part = threadIdx.x & 7;
  // the page's part that holds a position, for this head
  const auto words_of = [&](int64_t position) -> unsigned* {
    if (position < 0 || position >= room) return nullptr;
    const int64_t id = c.table[b * c.table_stride + position / c.page];
    return id < 0 || id >= c.page_count ? nullptr : c.pages + id * c.page_words + head;
  };
  const int64_t first = start > 0 ? start : 0, end = start + count < room ? start + count : room;
  for (int64_t kb = first / 32; kb * 32 < end; ++kb) {
    const int64_t place = kb * 32 + token, i = place - start;
    const bool in = i >= 0 && i < count && place < room && mine[i] != i;
    if (!__syncthreads_or(in)) continue;  // and the last block's codes have been read
    const int64_t from = in ? start + mine[i] : 0;
    const unsigned* source = in ? words_of(from) : nullptr;
    unsigned* to = words_of(kb * 32);  // a block lies in one page
    const bool moves = source && to;
    const int s = (int)(from % 32), blocks = (int)(from % c.page / 32);
    unsigned word[ND], affine = 0;
    if (moves) {
      const unsigned* in_block = source + (value ? (int64_t)c.page * 8 * ND : 0) + blocks * (DP * 4);
      if (part == 0) affine = source[(int64_t)c.page * (16 * ND + (value ? 1 : 0)) + blocks * 32 + s];
      if (!value) {
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          const int d8 = part * ND + j, W = 2 * ND * (s / 16) + d8 / 4;
          word[j] = in_block[W / 4 * 256 + (s % 16 + 16 * (d8 % 4)) * 4 + W % 4];
        }
      } else {
        const int e = s % 4 + s / 16 * 4, shift = e / 2 * 4 + e % 2 * 16, g = s / 4 % 4;
#pragma unroll
        for (int j = 0; j < 2 * ND; ++j) {
          unsigned four = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int d = (part * 2 * ND + j) * 4 + k, W = d / 16;
            four |= (in_block[W / 4 * 256 + (d % 16 + 16 * g) * 4 + W % 4] >> shift & 15u) << 8 * k;
          }
          codes[token][part * 2 * ND + j] = four;
        }
      }
    }
    // which of the block's tokens are written; and every source has been read
    __shared__ unsigned written[THREADS / 64];
    const uint64_t lanes = __builtin_amdgcn_ballot_w64(moves && part == 0);
    if (lane == 0) {
      unsigned bits = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) bits |= (unsigned)(lanes >> 8 * k & 1) << k;
      written[threadIdx.x / 64] = bits;
    }
    __syncthreads();
    if (!to) continue;
    const int at = (int)(kb * 32 % c.page / 32);
    unsigned* out = to + (value ? (int64_t)c.page * 8 * ND : 0) + at * (DP * 4);
    if (moves && part == 0) to[(int64_t)c.page * (16 * ND + (value ? 1 : 0)) + at * 32 + token] = affine;
    if (!value) {
      if (moves) {
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          const int d8 = part * ND + j, W = 2 * ND * (token / 16) + d8 / 4;
          out[W / 4 * 256 + (token % 16 + 16 * (d8 % 4)) * 4 + W % 4] = word[j];
        }
      }
    } else {
      const unsigned fresh = written[0] | written[1] << 8 | written[2] << 16 | written[3] << 24;
#pragma unroll
      for (int j = 0; j < ND; ++j) {  // DP * 4 = THREADS * ND words
        const int u = THREADS * j + threadIdx.x, l = u / 4 % 64, d = 16 * (u / 256 * 4 + u % 4) + l % 16, g = l / 16;
        unsigned w = 0, keep = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int token_e = 4 * g + e % 4 + e / 4 * 16, shift = e / 2 * 4 + e % 2 * 16;
          const bool now = fresh >> token_e & 1u;
          const unsigned code = codes[token_e][d / 4] >> (d % 4 * 8) & 15u;  // of another token: whatever LDS holds
          w |= (now ? code : 0u) << shift;
          keep |= (now ? 0u : 15u) << shift;
        }
        out[u] = w | (out[u] & keep);
      }
    }
  }
}

bool nodes_ok(int64_t seqs, int64_t tokens, int64_t nodes) {
  return seqs >= 0 && seqs <= (int64_t)1 << 24 && tokens >= 0 && tokens <= 0x7fffffff && nodes >= 1 && nodes <= MOST;
}

}  // namespace

extern "C" {

int gptq2d_draft_tree(const int32_t* parents, const int32_t* offsets, const int32_t* held, int64_t seqs, int64_t tokens,
                      int64_t nodes, uint32_t* ancestors, int32_t* positions, void* stream) {
  if (!nodes_ok(seqs, tokens, nodes)) return GPTQ2D_EINVAL;
  if (tokens == 0) return 0;
  const Nodes t = {parents, offsets, seqs, tokens, (int)nodes, (int)((nodes + 31) / 32)};
  hipLaunchKernelGGL(tree_kernel, dim3((unsigned)(seqs + 1)), dim3(THREADS), 0, (hipStream_t)stream, t, held, ancestors, positions);
  return (int)hipGetLastError();
}

int gptq2d_draft_accept(const int32_t* parents, const int32_t* offsets, int64_t seqs, int64_t tokens, int64_t nodes,
                        const void* drafted, const void* chosen, int32_t wide, int32_t* path, int32_t* counts, void* last,
                        void* stream) {
  if (!nodes_ok(seqs, tokens, nodes)) return GPTQ2D_EINVAL;
  if (seqs == 0) return 0;
  const Nodes t = {parents, offsets, seqs, tokens, (int)nodes, (int)((nodes + 31) / 32)};
  const dim3 grid((unsigned)seqs);
  const hipStream_t st = (hipStream_t)stream;
  if (wide)
    hipLaunchKernelGGL((accept_kernel<int64_t>), grid, dim3(64), 0, st, t, (const int64_t*)drafted, (const int64_t*)chosen, path,
                       counts, (int64_t*)last);
  else
    hipLaunchKernelGGL((accept_kernel<int32_t>), grid, dim3(64), 0, st, t, (const int32_t*)drafted, (const int32_t*)chosen, path,
                       counts, (int32_t*)last);
  return (int)hipGetLastError();
}

int gptq2d_kv_keep(void* pages, int64_t page_count, int32_t heads, int32_t dim, int32_t page, const int32_t* table, int64_t seqs,
                   int64_t width, int64_t table_stride, const int32_t* lengths, const int32_t* offsets, int64_t tokens,
                   const int32_t* path, int64_t path_stride, int64_t most, const int32_t* counts, void* stream) {
  KvCache c;
  if (!make_cache(c, pages, page_count, heads, dim, page, table, seqs, width, table_stride, lengths, offsets, tokens) ||
      !offsets || path_stride < 0 || most < 0 || most > 0x7fffffff)
    return GPTQ2D_EINVAL;
  if (seqs == 0 || width == 0 || page_count == 0 || most == 0) return 0;
  const dim3 grid((unsigned)seqs, (unsigned)heads, 2);
  const hipStream_t st = (hipStream_t)stream;
  switch ((dim + 63) / 64) {
    case 1:
      hipLaunchKernelGGL((keep_kernel<1>), grid, dim3(THREADS), 0, st, c, path, path_stride, (int)most, counts);
      break;
    case 2:
      hipLaunchKernelGGL((keep_kernel<2>), grid, dim3(THREADS), 0, st, c, path, path_stride, (int)most, counts);
      break;
    case 3:
      hipLaunchKernelGGL((keep_kernel<3>), grid, dim3(THREADS), 0, st, c, path, path_stride, (int)most, counts);
      break;
    case 4:
      hipLaunchKernelGGL((keep_kernel<4>), grid, dim3(THREADS), 0, st, c, path, path_stride, (int)most, counts);
      break;
  }
  return (int)hipGetLastError();
}

}  // extern "C"
