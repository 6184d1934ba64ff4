// The pages of a cache dealt to sequences, and where new tokens go.
//
// Sequence b has the first owned[b] entries of its table's row; the pages that no sequence has are a stack.  A call says how many
// tokens each sequence is to hold, so how many pages it wants: min(ceil(length / page), width).  Whole numbers only:
//   the entries [want, owned) of all sequences, in order, are given back, the last one first, each on the stack's top;
//   the entries [owned, want) of all sequences, in order, then take from the top while there are pages.
// So a step taken back gives the pages to where the next step's tokens will find them.  With e the place of an entry among all
// that are given (taken) and G their number: the given one goes to stack place left + G - 1 - e, the taken one comes from there.
// Three inclusive sums over the sequences -- entries given, taken, and new tokens -- decide everything; an entry or a row finds
// its sequence in them by bisection.
//
// Bound by latency.  Up to SMALL rows and sequences one workgroup does it all, with the sums in LDS; more take a second
// launch, between the pages that come back and those that go out, and every workgroup of the first sums for itself.  No
// kernel waits for another workgroup.  The cache's kernels read the table in a way that sees earlier launches only (kv_head of
// kv_cache.h): pages are dealt in launches of their own.
#include "common.h"

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64, SMALL = 2048;
constexpr int MOST = 1 << 30;  // tokens of a sequence

struct Pool {
  int32_t* table;
  int64_t table_stride;
  int seqs, width, page, pages;
  int32_t *owned, *lengths, *missing, *free, *left;
  const int32_t* request;  // lengths, or (extend) new tokens
  bool extend;
  int64_t tokens;
  int32_t *offsets, *held, *positions;
  int64_t* slots;
  int32_t* work;
};

// What the scan leaves: of each sequence, and the stack's height before and after the gifts.
struct Sums {
  int32_t *given, *taken, *rows;  // inclusive sums
  int32_t *keep, *base, *length;  // entries that stay, tokens held before, tokens to be held
};
constexpr int ARRAYS = 6;
__device__ __forceinline__ Sums sums_at(int32_t* p, int seqs) {
  return {p, p + seqs, p + 2 * seqs, p + 3 * seqs, p + 4 * seqs, p + 5 * seqs};
}
__device__ __forceinline__ int before(const int32_t* sums, int b) { return b ? sums[b - 1] : 0; }

// First b with sums[b] > e, in [lo, hi); hi where there is none.
__device__ __forceinline__ int bisect(const int32_t* sums, int lo, int hi, int e) {
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (sums[mid] > e)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int64_t add_up(int64_t x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(x, d);
    x += lane >= d ? y : 0;
  }
  return x;
}

// The sums over all sequences, left in `s` for those in [from, to); by all threads of a workgroup, ended by a barrier.  Returns the entries given.
__device__ __forceinline__ int scan(const Pool& p, const Sums& s, int from, int to) {
  __shared__ int64_t pages_of[WAVES], rows_of[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t pages = 0, rows = 0;  // given in the low half, taken in the high one; both below 2^31
  for (int b0 = 0; b0 < p.seqs; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    int64_t x = 0, n = 0;
    int keep = 0, base = 0, length = 0;
    if (b < p.seqs) {
      const int request = p.request[b] > 0 ? p.request[b] : 0, had = p.owned[b], was = p.lengths[b];
      const int owned = had < 0 ? 0 : had < p.width ? had : p.width;
      base = was < 0 ? 0 : was < MOST ? was : MOST;
      length = p.extend ? (request < MOST - base ? base + request : MOST) : request < MOST ? request : MOST;
      n = p.extend ? request : 0;
      const int wish = (length + p.page - 1) / p.page, want = wish < p.width ? wish : p.width;
      keep = owned < want ? owned : want;
      x = (int64_t)(want - keep) << 32 | (owned - keep);
    }
    const int64_t xs = add_up(x, lane), ns = add_up(n, lane);
    if (lane == 63) pages_of[wave] = xs, rows_of[wave] = ns;
    __syncthreads();
    int64_t xb = pages, nb = rows;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const int64_t xw = pages_of[w], nw = rows_of[w];
      xb += w < wave ? xw : 0, nb += w < wave ? nw : 0;
      pages += xw, rows += nw;
    }
    if (b + 1 >= from && b < to) {  // and the one before its own, whose sums it starts from
      s.given[b] = (int32_t)(uint32_t)(xb + xs);
      s.taken[b] = (int32_t)((xb + xs) >> 32);
      s.rows[b] = (int32_t)(nb + ns < p.tokens ? nb + ns : p.tokens);
      s.keep[b] = keep, s.base[b] = base, s.length[b] = length;
    }
    __syncthreads();
  }
  return (int)(uint32_t)pages;
}

__device__ __forceinline__ int stack_height(const Pool& p) {
  const int left = p.left[0];
  return left < 0 ? 0 : left < p.pages ? left : p.pages;
}

// Entries given back by the sequences [from, to), `all` by all of them, onto a stack of `left` pages.
__device__ __forceinline__ void give(const Pool& p, const Sums& s, int from, int to, int left, int all) {
  if (from >= to) return;
  const int end = s.given[to - 1];
  for (int e = before(s.given, from) + (int)threadIdx.x; e < end; e += THREADS) {
    const int b = bisect(s.given, from, to, e);
    int32_t* entry = p.table + b * p.table_stride + s.keep[b] + (e - before(s.given, b));
    const int64_t place = (int64_t)left + all - 1 - e;
    if (place < p.pages) p.free[place] = *entry;
    *entry = -1;
  }
}

// Page that entry number `e` of those that are taken gets, from a stack of `top` pages: -1 where it is empty.
__device__ __forceinline__ int taken_page(const Pool& p, int64_t top, int e) {
  const int64_t place = top - 1 - e;
  return place >= 0 && place < p.pages ? p.free[place] : -1;
}

// Entries that are taken, the rows of new tokens, and the sequences' state; thread `first` of `step`.
__device__ __forceinline__ void take(const Pool& p, const Sums& s, int left, int all, int64_t first, int64_t step) {
  const int64_t top = (int64_t)left + all;
  const int n = p.seqs, taken = n ? s.taken[n - 1] : 0;
  for (int64_t e = first; e < taken && e < top; e += step) {  // an entry that gets none is -1 already
    const int b = bisect(s.taken, 0, n, (int)e);
    p.table[b * p.table_stride + s.keep[b] + ((int)e - before(s.taken, b))] = taken_page(p, top, (int)e);
  }
  for (int64_t r = first; r < p.tokens; r += step) {
    const int b = bisect(s.rows, 0, n, (int)r);
    int position = 0;
    int64_t slot = -1;
    if (b < n) {
      const int64_t row = (int64_t)s.base[b] + (r - before(s.rows, b));  // of more rows than a sequence may hold past 32 bits
      position = row < MOST ? (int)row : MOST;
      if (row < MOST) {
        const int at = position / p.page, fresh = at - s.keep[b], count = s.taken[b] - before(s.taken, b);
        // an entry that this call takes may not be in the table yet
        const int page = fresh < 0 ? p.table[b * p.table_stride + at]
                                   : fresh < count ? taken_page(p, top, before(s.taken, b) + fresh) : -1;
        if (page >= 0) slot = (int64_t)page * p.page + position % p.page;
      }
    }
    if (p.positions) p.positions[r] = position;
    if (p.slots) p.slots[r] = slot;
  }
  for (int64_t b = first; b < n; b += step) {
    const int start = before(s.taken, (int)b), count = s.taken[b] - start;
    const int64_t there = top - start;
    const int got = there < 0 ? 0 : there < count ? (int)there : count;
    p.owned[b] = s.keep[b] + got;
    p.missing[b] = count - got;
    p.lengths[b] = s.length[b];
    if (p.held) p.held[b] = s.base[b];
    if (p.offsets) p.offsets[b + 1] = s.rows[b];
  }
  if (first == 0) {
    p.left[0] = (int)(top > taken ? top - taken : 0);
    if (p.offsets) p.offsets[0] = 0;
  }
}

__global__ __launch_bounds__(THREADS) void small_kernel(Pool p) {
  __shared__ int32_t sums[ARRAYS * SMALL];
  const Sums s = sums_at(sums, p.seqs);
  const int left = stack_height(p);
  const int all = scan(p, s, 0, p.seqs);
  give(p, s, 0, p.seqs, left, all);
  __syncthreads();  // the stack's new pages are there
  take(p, s, left, all, threadIdx.x, THREADS);
}

// A workgroup sums over all sequences and deals with the gifts of its own ones.
__global__ __launch_bounds__(THREADS) void give_kernel(Pool p) {
  const Sums s = sums_at(p.work, p.seqs);
  const int per = (p.seqs + gridDim.x - 1) / gridDim.x;
  const int from = blockIdx.x * per < p.seqs ? blockIdx.x * per : p.seqs, to = from + per < p.seqs ? from + per : p.seqs;
  const int left = stack_height(p);
  const int all = scan(p, s, from, to);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.work[ARRAYS * p.seqs] = left, p.work[ARRAYS * p.seqs + 1] = all;
  give(p, s, from, to, left, all);
}

__global__ __launch_bounds__(THREADS) void take_kernel(Pool p) {
  const Sums s = sums_at(p.work, p.seqs);
  take(p, s, p.work[ARRAYS * p.seqs], p.work[ARRAYS * p.seqs + 1], (int64_t)blockIdx.x * THREADS + threadIdx.x,
       (int64_t)gridDim.x * THREADS);
}

// Positions of packed rows: held[b] + row - offsets[b], 0 for rows that no sequence has.
__global__ __launch_bounds__(256) void positions_kernel(const int32_t* held, const int32_t* offsets, int seqs, int tokens,
                                                        int32_t* positions) {
  const int r = (int)(blockIdx.x * 256 + threadIdx.x);
  if (r >= tokens) return;
  const int b = bisect(offsets, 0, seqs + 1, r) - 1;  // the last one that begins at r or before
  positions[r] = b < 0 || b >= seqs ? 0 : held[b] + (r - offsets[b]);
}

bool pool_ok(int64_t seqs, int64_t width, int32_t page, int64_t pages, int64_t tokens) {
  return seqs >= 0 && width >= 0 && page >= 1 && page <= 1 << 20 && pages >= 0 && tokens >= 0 && pages < (int64_t)1 << 31 &&
         tokens < (int64_t)1 << 31 && seqs <= (int64_t)1 << 24 && width < (int64_t)1 << 31 &&
         seqs * width < (int64_t)1 << 31;
}
bool one_workgroup(int64_t seqs, int64_t tokens) { return seqs <= SMALL && tokens <= SMALL; }

}  // namespace

extern "C" {

int64_t gptq2d_page_pool_workspace(int64_t seqs) {
  return seqs < 0 || seqs > (int64_t)1 << 24 ? -1 : 4 * (ARRAYS * seqs + 2);
}

int gptq2d_page_pool(int32_t* table, int64_t seqs, int64_t width, int64_t table_stride, int32_t page, int64_t pages,
                     int32_t* owned, int32_t* lengths, int32_t* missing, int32_t* free, int32_t* left, const int32_t* request,
                     int32_t extend, int64_t tokens, int32_t* offsets, int32_t* held, int32_t* positions, int64_t* slots,
                     void* work, int64_t work_bytes, void* stream) {
  if (!pool_ok(seqs, width, page, pages, tokens) || table_stride < 0) return GPTQ2D_EINVAL;
  if (work_bytes < gptq2d_page_pool_workspace(seqs) || !work || (uintptr_t)work % 4) return GPTQ2D_ESCRATCH;
  Pool p;
  p.table = table, p.table_stride = table_stride;
  p.seqs = (int)seqs, p.width = (int)width, p.page = page, p.pages = (int)pages;
  p.owned = owned, p.lengths = lengths, p.missing = missing, p.free = free, p.left = left;
  p.request = request, p.extend = extend != 0;
  p.tokens = extend ? tokens : 0;
  p.offsets = offsets, p.held = held, p.positions = positions, p.slots = slots;
  p.work = (int32_t*)work;
  const hipStream_t st = (hipStream_t)stream;
  if (one_workgroup(seqs, p.tokens)) {
    hipLaunchKernelGGL(small_kernel, dim3(1), dim3(THREADS), 0, st, p);
  } else {
    const int64_t shares = seqs / 16 + 1, rows = (p.tokens + seqs) / THREADS + 1;
    hipLaunchKernelGGL(give_kernel, dim3((unsigned)(shares < 256 ? shares : 256)), dim3(THREADS), 0, st, p);
    hipLaunchKernelGGL(take_kernel, dim3((unsigned)(rows < 512 ? rows : 512)), dim3(THREADS), 0, st, p);
  }
  return (int)hipGetLastError();
}

int gptq2d_row_positions(const int32_t* held, const int32_t* offsets, int64_t seqs, int64_t tokens, int32_t* positions,
                         void* stream) {
  if (seqs < 0 || seqs > (int64_t)1 << 24 || tokens < 0 || tokens >= (int64_t)1 << 31) return GPTQ2D_EINVAL;
  if (tokens == 0) return 0;
  hipLaunchKernelGGL(positions_kernel, dim3((unsigned)((tokens + 255) / 256)), dim3(256), 0, (hipStream_t)stream, held, offsets,
                     (int)seqs, (int)tokens, positions);
  return (int)hipGetLastError();
}

}  // extern "C"
