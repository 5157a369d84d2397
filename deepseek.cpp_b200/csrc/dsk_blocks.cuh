// dsk_blocks.cuh — which blocks of a cache are whose, on the GPU: places for tokens that join sequences, blocks that come back.
//
// Free blocks are a stack.  A sequence of len tokens holds the first ceil(len / block) entries of its row of the table; count more tokens need
// ceil((len + count) / block) - ceil(len / block) blocks.  With exclusive sums over the sequences in order (needs: n_b, tokens: s_b), block j of sequence b is
// free[top - 1 - n_b - (j - ceil(len / block))], and token s_b + i of the packed ones has position t = len + i and slot (number of block t / block) x block + t % block: every token's
// place follows from sums over at most 1024 sequences and one look at the stack or the table, without any order among threads.  Blocks come back in the reverse of that order, so that
// what was taken last lies on top again, as it did.
// Bound: two dependent loads behind a launch (lengths, then a block's number); every CTA makes the sums anew (1024 sequences: four a thread), which costs less than a launch between.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dsk {
namespace blocks {

constexpr int kMaxBatch = 1024, kThreads = 256, kEach = kMaxBatch / kThreads, kWarps = kThreads / 32, kCutThreads = 1024;
enum { ST_PAGE = 1, ST_RANGE = 2, ST_SHORT = 8, ST_TWICE = 16 };   // a number that is no block; tokens outside the table; blocks or rows ran out; more blocks came back than there are

struct Pool { int *free, *top, *status; int n_blocks, shift; };   // top: how many are free, and a word that counts CTAs (0 between calls)
struct Extend {
  Pool P;
  int* table;
  long long pitch;
  const int *lens, *count;
  int *starts, *lens_out, *positions, *slots;
  int4* pieces;                                              // (first row, rows, block, place in the block)
  int table_blocks, batch, rows, n_pieces;
};
struct Cut {
  Pool P;
  int* table;
  long long pitch;
  const int *lens, *keep;
  int table_blocks, batch;
};

__device__ __forceinline__ void note(const Pool& P, int bit) { if (P.status) atomicOr(P.status, bit); }

// Sums over what lies ahead of a thread's value, for three values at a time; `all` gets the sums over all threads
template <int WARPS> __device__ __forceinline__ void sums_ahead(int (&v)[3], int (&all)[3], int (*of_warp)[WARPS]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int own[3];
#pragma unroll
  for (int u = 0; u < 3; u++) {
    own[u] = v[u];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, v[u], o);
      if (lane >= o) v[u] += x;
    }
    if (lane == 31) of_warp[u][warp] = v[u];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 3; u++) {
    int ahead = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const int x = of_warp[u][w];
      if (w < warp) ahead += x;
      sum += x;
    }
    v[u] += ahead - own[u];
    all[u] = sum;
  }
}

__global__ void __launch_bounds__(kThreads) extend(const Extend A) {
  __shared__ int start[kMaxBatch + 1], len[kMaxBatch], taken[kMaxBatch], piece[kMaxBatch], of_warp[3][kWarps], free_now, served[2];
  const int shift = A.P.shift, block = 1 << shift, b0 = threadIdx.x * kEach;
  if (threadIdx.x == 0) { free_now = min(max(*A.P.top, 0), A.P.n_blocks); served[0] = served[1] = 0; }
  const long long room = (long long)A.table_blocks << shift;
  int l[kEach], c[kEach], need[kEach], pieces[kEach], sum[3] = {0, 0, 0}, all[3];
#pragma unroll
  for (int k = 0; k < kEach; k++) {
    l[k] = c[k] = need[k] = pieces[k] = 0;
    const int b = b0 + k;
    if (b >= A.batch) continue;
    l[k] = A.lens[b];
    const int n = A.count[b];
    if (l[k] < 0 || (long long)l[k] + max(n, 0) > room) {    // gets nothing and stays what it is
      if (blockIdx.x == 0) note(A.P, ST_RANGE);
      continue;
    }
    c[k] = min(max(n, 0), A.rows + 1);                       // (one row more than there are is refused as well; sums stay below 2^31)
    need[k] = (int)(((long long)l[k] + c[k] + block - 1) >> shift) - (int)(((long long)l[k] + block - 1) >> shift);
    pieces[k] = c[k] ? ((l[k] + c[k] - 1) >> shift) - (l[k] >> shift) + 1 : 0;
    sum[0] += c[k]; sum[1] += need[k]; sum[2] += pieces[k];
  }
  sums_ahead<kWarps>(sum, all, of_warp);
  const int have = free_now;
  bool refused = false;
  int rows_end = 0, taken_end = 0;                           // behind the last served one of this thread
#pragma unroll
  for (int k = 0; k < kEach; k++) {
    const int b = b0 + k;
    if (b < A.batch) {
      const bool fits = sum[0] + c[k] <= A.rows && sum[1] + need[k] <= have;   // (sums only grow: behind the first that does not fit, none does)
      start[b] = fits ? sum[0] : 0x7fffffff;
      len[b] = l[k];
      taken[b] = sum[1];
      piece[b] = sum[2];
      if (fits) { rows_end = sum[0] + c[k]; taken_end = sum[1] + need[k]; }
      else refused |= c[k] > 0;
      if (blockIdx.x == 0) A.lens_out[b] = l[k] + (fits ? c[k] : 0);
    }
    sum[0] += c[k]; sum[1] += need[k]; sum[2] += pieces[k];
  }
  rows_end = __reduce_max_sync(0xffffffffu, rows_end);
  taken_end = __reduce_max_sync(0xffffffffu, taken_end);
  if ((threadIdx.x & 31) == 0 && rows_end + taken_end > 0) { atomicMax(&served[0], rows_end); atomicMax(&served[1], taken_end); }
  __syncthreads();
  const int total = served[0];
#pragma unroll
  for (int k = 0; k < kEach; k++) {
    const int b = b0 + k;
    if (b >= A.batch) break;
    const int s = min(start[b], total);
    start[b] = s;
    if (blockIdx.x == 0) A.starts[b] = s;
  }
  if (threadIdx.x == 0) {
    start[A.batch] = total;
    if (blockIdx.x == 0) A.starts[A.batch] = total;
  }
  if (blockIdx.x == 0 && refused) note(A.P, ST_SHORT);
  __syncthreads();
  // places: four neighbouring tokens a thread
  const bool wide = ((reinterpret_cast<uintptr_t>(A.positions) | reinterpret_cast<uintptr_t>(A.slots)) & 15) == 0;
  for (int i0 = 4 * (blockIdx.x * kThreads + threadIdx.x); i0 < A.rows; i0 += 4 * gridDim.x * kThreads) {
    int at[4], slot[4], b = 0;
    if (i0 < total) {
      for (int step = kMaxBatch / 2; step; step >>= 1) if (b + step < A.batch && start[b + step] <= i0) b += step;   // the last sequence that starts at or ahead of i0: it has a token there
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int i = i0 + k;
      at[k] = slot[k] = -1;
      if (i >= total) continue;
      while (start[b + 1] <= i) b++;
      const int t = len[b] + i - start[b], j = t >> shift, had = (int)(((long long)len[b] + block - 1) >> shift), in = t & (block - 1);
      int* entry = A.table + b * A.pitch + j;
      const bool fresh = j >= had;
      const int p = fresh ? A.P.free[have - 1 - taken[b] - (j - had)] : *entry;
      const bool known = (unsigned)p < (unsigned)A.P.n_blocks;
      if (!known) note(A.P, ST_PAGE);
      if (fresh && in == 0) *entry = p;
      at[k] = t;
      if (known) slot[k] = p << shift | in;
      if (in == 0 || i == start[b]) {
        const int n = piece[b] + j - (len[b] >> shift);
        if (n < A.n_pieces) A.pieces[n] = make_int4(i, known ? min(block - in, start[b + 1] - i) : 0, p, in);
      }
    }
    if (wide && i0 + 4 <= A.rows) {
      *reinterpret_cast<int4*>(A.positions + i0) = make_int4(at[0], at[1], at[2], at[3]);
      *reinterpret_cast<int4*>(A.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) if (i0 + k < A.rows) { A.positions[i0 + k] = at[k]; A.slots[i0 + k] = slot[k]; }
    }
  }
  // pieces behind the last one: none of the served sequences has them
  int n = 0;
  if (total) {
    int b = 0;
    for (int step = kMaxBatch / 2; step; step >>= 1) if (b + step < A.batch && start[b + step] < total) b += step;
    n = piece[b] + ((len[b] + total - 1 - start[b]) >> shift) - (len[b] >> shift) + 1;
  }
  for (int i = n + blockIdx.x * kThreads + threadIdx.x; i < A.n_pieces; i += gridDim.x * kThreads) A.pieces[i] = make_int4(0, 0, -1, 0);
  if (threadIdx.x == 0) {                                    // the last CTA that has read the stack's height sets it
    if (gridDim.x == 1) *A.P.top = have - served[1];
    else {
      __threadfence();
      if (atomicAdd(A.P.top + 1, 1) == (int)gridDim.x - 1) { A.P.top[1] = 0; *A.P.top = have - served[1]; }
    }
  }
}

// One CTA.  A thread has one sequence's count of entries, a warp walks a sequence's entries: numbers that are no blocks do not go back, so they are counted first.
// MANY: the table has 2^31 entries or more, and if they repeat as many may come back: two sums, of 16 and 11 bits of each count (4.1 us for a call that has nothing to do, 3.1 with one sum).  What comes back
// beyond the stack's end, which has at most 2^27 places, goes nowhere: a sum beyond is taken as one more than those.
template <bool MANY> __global__ void __launch_bounds__(kCutThreads) cut(const Cut A) {
  constexpr int WARPS = kCutThreads / 32;
  __shared__ int low[kMaxBatch], high[kMaxBatch], good[kMaxBatch], of_warp[3][WARPS], height;
  const int shift = A.P.shift, block = 1 << shift, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = threadIdx.x;
  if (threadIdx.x == 0) height = min(max(*A.P.top, 0), A.P.n_blocks);
  if (b < A.batch) {
    const int l = A.lens[b], k = A.keep[b];
    const bool fine = k >= 0 && k <= l && (long long)l <= (long long)A.table_blocks << shift;
    if (!fine) note(A.P, ST_RANGE);
    low[b] = fine ? (int)(((long long)k + block - 1) >> shift) : 0;
    high[b] = fine ? (int)(((long long)l + block - 1) >> shift) : 0;
  }
  __syncthreads();
  for (int s = warp; s < A.batch; s += WARPS) {
    const int* row = A.table + s * A.pitch;
    int n = 0;
    for (int j = low[s] + lane; j < high[s]; j += 32) n += (unsigned)row[j] < (unsigned)A.P.n_blocks;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) good[s] = n;
  }
  __syncthreads();
  const int from = A.batch - 1 - b, count = b < A.batch ? good[from] : 0;   // sums over the sequences behind a thread's own: the last one's blocks go first
  int sum[3] = {MANY ? count & 0xffff : count, MANY ? count >> 16 : 0, 0}, all[3];
  const bool lost = b < A.batch && count < high[from] - low[from];
  sums_ahead<WARPS>(sum, all, of_warp);
  auto whole = [&](const int (&x)[3]) { return min(MANY ? (min(x[1], 1 << 12) << 16) + x[0] : x[0], A.P.n_blocks + 1); };
  if (b < A.batch) good[from] = whole(sum);
  if (lost) note(A.P, ST_PAGE);
  const int have = height, back = whole(all);
  __syncthreads();
  for (int s = warp; s < A.batch; s += WARPS) {
    int* row = A.table + s * A.pitch;
    int to = have + good[s];
    for (int j0 = high[s] - 1; j0 >= low[s]; j0 -= 32) {
      const int j = j0 - lane, p = j >= low[s] ? row[j] : -1;
      const bool known = (unsigned)p < (unsigned)A.P.n_blocks;
      const unsigned there = __ballot_sync(0xffffffffu, known);
      const int place = to + __popc(there & ((1u << lane) - 1));
      if (known && place < A.P.n_blocks) A.P.free[place] = p;
      if (j >= low[s]) row[j] = -1;
      to += __popc(there);
    }
  }
  if (threadIdx.x == 0) {
    if (have + back > A.P.n_blocks) note(A.P, ST_TWICE);
    *A.P.top = min(have + back, A.P.n_blocks);
  }
}

}  // namespace blocks
}  // namespace dsk
