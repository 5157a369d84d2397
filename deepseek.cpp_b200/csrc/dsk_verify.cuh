// dsk_verify.cuh — verification of drafted tokens by speculative sampling, from uniform numbers that the caller gives.
//
// p_i = softmax(logits_i / temperature).  Draft x_i is accepted while coin_i q_i(x_i) < p_i(x_i); the first one that is not is replaced by a draw from max(p_i - q_i, 0), and
// behind accepted ones the next token is drawn from p.  Both draws take the lowest index whose running sum is over (last coin) x (whole sum).
// Two kernels: row_stats reads every row of logits once (maximum and sum of a piece of 1024 per warp, in fp32); pick has a cluster of CTAs for each sequence, which decides
// on the drafts and draws from one row.  A draw's result hangs on sums of up to the whole vocabulary next to a border, so pick takes exponentials, sums and differences
// of that row in 64 bits: in 32 one draw in some thousands of a flat row would take a neighbour.  Where coin x q is within 1e-4 of p, the row's sum is taken again in 64 bits as well.
// Bound: row_stats by the bytes of the logits; pick by the latency of three walks over a row that L2 holds, with a cluster's barrier behind two of them.
#pragma once

#include <cooperative_groups.h>

#include "dsk_kv8.cuh"

namespace dsk {
namespace verify {

constexpr int kThreads = 256, kWarps = kThreads / 32, kPiece = 1024, kMaxDrafts = 127, kMaxCluster = 16;

struct Params {
  const void* logits;
  long long l_batch, l_row;              // pitches, in elements
  const float* probs;                    // nullable: drafts are certain
  long long p_batch, p_row;
  const int *drafts, *count;             // [batch][n]; nullable
  const float* coins;                    // [batch][n + 1]
  float2* part;                          // [batch][n + 1][pieces]: maximum and sum (greedy: maximum and index bits)
  int *accepted, *tokens;
  int batch, n, vocab, pieces, cluster, wide_l, wide_p;
  double slope;                          // log2(e) / temperature; 0: greedy
};

template <typename T> __device__ __forceinline__ float value(T x) { return (float)x; }
__device__ __forceinline__ int drafts_of(const Params& P, int b) { return P.count ? min(max(P.count[b], 0), P.n) : P.n; }
// four values of a row from index i on; behind the row's end -inf
template <typename T> __device__ __forceinline__ void four(const T* row, int i, int vocab, bool wide, float (&x)[4]) {
  if (wide && i + 4 <= vocab) {
    T t[4];
    if (sizeof(T) == 4) *reinterpret_cast<uint4*>(t) = __ldg(reinterpret_cast<const uint4*>(row + i));
    else *reinterpret_cast<uint2*>(t) = __ldg(reinterpret_cast<const uint2*>(row + i));
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = value(t[u]);
  } else {
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = i + u < vocab ? value(row[i + u]) : -INFINITY;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) row_stats(const Params P) {
  grid_release();
  const int warp = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31, r = blockIdx.y, b = blockIdx.z;
  if (warp >= P.pieces || r > drafts_of(P, b)) return;
  const T* row = static_cast<const T*>(P.logits) + b * P.l_batch + r * P.l_row;
  float x[kPiece / 128][4], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPiece / 128; i++) four(row, warp * kPiece + i * 128 + lane * 4, P.vocab, P.wide_l, x[i]);
#pragma unroll
  for (int i = 0; i < kPiece / 128; i++)
#pragma unroll
    for (int u = 0; u < 4; u++) m = fmaxf(m, x[i][u]);
  float2* out = P.part + ((size_t)b * (P.n + 1) + r) * P.pieces + warp;
  const float top = warp_max(m);
  if (P.slope == 0.0) {                                      // lowest index of the maximum; a NaN anywhere shows as one in the maximum's place
    int at = 0x7fffffff;
    bool nan = false;
#pragma unroll
    for (int i = kPiece / 128 - 1; i >= 0; i--)
#pragma unroll
      for (int u = 3; u >= 0; u--) {
        if (x[i][u] == top) at = warp * kPiece + i * 128 + lane * 4 + u;
        nan |= x[i][u] != x[i][u];
      }
    at = (int)__reduce_min_sync(0xffffffffu, (unsigned)at);
    nan = __any_sync(0xffffffffu, nan);
    if (lane == 0) *out = make_float2(nan ? NAN : top, __int_as_float(at));
    return;
  }
  const float from = top == -INFINITY ? 0.f : top, slope = (float)P.slope;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kPiece / 128; i++)
#pragma unroll
    for (int u = 0; u < 4; u++) s += exp2f((x[i][u] - from) * slope);
  s = warp_sum(s);
  if (lane == 0) *out = make_float2(top, s);
}

// 2^y for y <= 0 in 64 bits: 2^(k / 64) from a table, the rest of at most 1/128 by the series of e^z (z^6 / 720 < 4e-17); Tang, "Table-driven implementation of the exponential
// function in IEEE floating-point arithmetic" (1989)
__device__ __forceinline__ double power(double y, const double* table) {
  const double magic = 6755399441055744.0, t = fma(y, 64.0, magic);   // 1.5 x 2^52: the integer next to 64 y stands in the low bits
  const int k = __double2loint(t);
  const double z = fma(t - magic, -1.0 / 64.0, y) * 0.693147180559945309417;
  double p = fma(z, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(z, p, 1.0 / 6.0);
  p = fma(z, p, 0.5);
  p = fma(z, p, 1.0);
  p = fma(z, p, 1.0);
  const double r = table[k & 63] * p;
  return y > -1000.0 ? __hiloint2double(__double2hiint(r) + ((k >> 6) << 20), __double2loint(r)) : (y <= -1000.0 ? 0.0 : y);
}
__device__ __forceinline__ double sum64(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pick(const Params P) {
  namespace cg = cooperative_groups;
  __shared__ double table[64], ends[kMaxCluster * kWarps], sums[2][kWarps], row_sum[kMaxDrafts + 1];
  __shared__ float row_max[kMaxDrafts + 1];
  __shared__ int flag[kMaxDrafts + 1], top_at[kMaxDrafts + 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / P.cluster, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < 64) table[tid] = exp2(tid / 64.0);
  grid_wait();
  __syncthreads();
  const int n = drafts_of(P, b), V = P.vocab;
  const bool greedy = P.slope == 0.0;
  const T* logits = static_cast<const T*>(P.logits) + b * P.l_batch;
  const int* drafts = P.drafts + (size_t)b * P.n;
  const float* coins = P.coins + (size_t)b * (P.n + 1);
  // rows: maximum and sum of the pieces; 0: refused, 1: accepted, 2: next to the border, 4: not a distribution (a NaN, +inf or nothing but -inf)
  for (int r = warp; r <= n; r += kWarps) {
    const float2* part = P.part + ((size_t)b * (P.n + 1) + r) * P.pieces;
    float m = -INFINITY;
    bool nan = false;
    for (int i = lane; i < P.pieces; i += 32) { const float t = part[i].x; m = fmaxf(m, t); nan |= t != t; }
    m = warp_max(m);
    nan = __any_sync(0xffffffffu, nan);
    int x = r < n ? drafts[r] : -1;
    if ((unsigned)x >= (unsigned)V) x = -1;
    if (greedy) {
      unsigned at = 0x7fffffffu;
      for (int i = lane; i < P.pieces; i += 32) if (part[i].x == m) at = min(at, (unsigned)__float_as_int(part[i].y));
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0) { flag[r] = nan || m == -INFINITY ? 4 : x == (int)at ? 1 : 0; top_at[r] = (int)at; }
      continue;
    }
    double s = 0.0;
    for (int i = lane; i < P.pieces; i += 32) { const float2 t = part[i]; s += t.x == -INFINITY ? (double)t.y : (double)t.y * power(((double)t.x - m) * P.slope, table); }
    s = sum64(s);
    if (lane == 0) {
      int f = 0;
      if (!(m > -INFINITY && m < INFINITY) || !(s < INFINITY)) f = 4;
      else if (x >= 0) {
        const double p = power(((double)value(logits[r * P.l_row + x]) - m) * P.slope, table) / s, q = P.probs ? (double)P.probs[b * P.p_batch + r * P.p_row + x] : 1.0, want = (double)coins[r] * q;
        f = fabs(want - p) <= 1e-4 * p && p > 0.0 ? 2 : want < p ? 1 : 0;
      }
      flag[r] = f; row_max[r] = m; row_sum[r] = s;
    }
  }
  __syncthreads();
  auto walk = [&](int r, int from, int to, double m) {       // sum of a row's exponentials over indices from .. to - 1 (from a multiple of four), by a warp
    const T* row = logits + r * P.l_row;
    double s = 0.0;
    for (int i = from + lane * 4; i < to; i += 512) {
      float x[4][4];
#pragma unroll
      for (int u = 0; u < 4; u++) four(row, i + u * 128, i + u * 128 < to ? V : 0, P.wide_l, x[u]);
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int w = 0; w < 4; w++) s += power(((double)x[u][w] - m) * P.slope, table);
    }
    return sum64(s);
  };
  const int all = P.cluster * kWarps, share = ((V + all - 1) / all + 127) / 128 * 128, mine = rank * kWarps + warp;   // a warp's indices of the row that is drawn from
  const int from = min(V, mine * share), to = min(V, from + share);
  int r = 0;                                                 // (the same in every CTA of the cluster)
  for (; r < n; r++) {
    int f = flag[r];
    if (f == 2) {
      const int each = ((V + kWarps - 1) / kWarps + 3) / 4 * 4;
      const double s = walk(r, min(V, warp * each), min(V, (warp + 1) * each), row_max[r]);
      if (lane == 0) sums[0][warp] = s;
      __syncthreads();
      double whole = 0.0;
      for (int w = 0; w < kWarps; w++) whole += sums[0][w];
      __syncthreads();
      const int x = drafts[r];
      const double p = power(((double)value(logits[r * P.l_row + x]) - row_max[r]) * P.slope, table) / whole, q = P.probs ? (double)P.probs[b * P.p_batch + r * P.p_row + x] : 1.0;
      f = (double)coins[r] * q < p;
    }
    if (f != 1) break;
  }
  int token = -1;
  int* out = P.tokens + (size_t)b * (P.n + 1);
  if (rank == 0) {
    for (int i = tid; i <= P.n; i += kThreads) if (i != r) out[i] = i < r ? drafts[i] : -1;
    if (tid == 0) P.accepted[b] = r;
  }
  if (greedy || flag[r] == 4) {
    if (rank == 0 && tid == 0) out[r] = flag[r] == 4 ? -1 : top_at[r];
    return;                                                  // (the whole cluster)
  }
  const double m = row_max[r];
  {
    const double s = walk(r, from, to, m);
    if (lane == 0) sums[0][warp] = s;
  }
  cluster.sync();
  auto gather = [&](int which) {                             // sums of all warps of the cluster, in order
    if (tid < all) ends[tid] = *cluster.map_shared_rank(&sums[which][tid % kWarps], tid / kWarps);
    __syncthreads();
  };
  gather(0);
  double whole = 0.0;
  for (int i = lane; i < all; i += 32) whole += ends[i];
  whole = sum64(whole);
  const double inv = 1.0 / whole;
  const bool drafted = r < n;
  const T* row = logits + r * P.l_row;
  const float* q = drafted && P.probs ? P.probs + b * P.p_batch + r * P.p_row : nullptr;
  const int certain = drafted && !P.probs ? drafts[r] : -1;
  auto left = [&](int i, double (&d)[4]) {                   // what four indices have in the draw
    float x[4], y[4] = {0.f, 0.f, 0.f, 0.f};
    four(row, i, i < to ? V : 0, P.wide_l, x);
    if (q && i < to) four(q, i, V, P.wide_p, y);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const double p = power(((double)x[u] - m) * P.slope, table) * inv;
      d[u] = i + u >= to ? 0.0 : q ? fmax(p - (double)y[u], 0.0) : i + u == certain ? 0.0 : p;
    }
  };
  {
    double s = 0.0;
    for (int i = from + lane * 4; i < to; i += 256) {
      double d[2][4];
      left(i, d[0]);
      left(i + 128, d[1]);
#pragma unroll
      for (int u = 0; u < 4; u++) s += d[0][u] + d[1][u];
    }
    s = sum64(s);
    if (lane == 0) sums[1][warp] = s;
  }
  cluster.sync();
  gather(1);
  if (warp == 0) {                                           // running sums of the warps, in order
    double run = 0.0;
    for (int i0 = 0; i0 < all; i0 += 32) {
      double v = i0 + lane < all ? ends[i0 + lane] : 0.0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const double t = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += t; }
      if (i0 + lane < all) ends[i0 + lane] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const double total = ends[all - 1], want = (double)coins[P.n] * total;
  int owner = -1;                                            // the first warp whose running sum is over it; behind all of them (a coin of one, rounding) the last that has anything
  for (int i0 = 0; i0 < all && owner < 0; i0 += 32) {
    const uint32_t over = __ballot_sync(0xffffffffu, i0 + lane < all && ends[i0 + lane] > want);
    if (over) owner = i0 + __ffs(over) - 1;
  }
  for (int i = all - 1; i >= 0 && owner < 0; i--) if (ends[i] > (i ? ends[i - 1] : 0.0)) owner = i;
  if (owner < 0 && mine == 0 && lane == 0) out[r] = -1;      // nothing is left
  if (mine == owner) {
    double run = owner ? ends[owner - 1] : 0.0;
    int last = -1;
    for (int i0 = from; i0 < to && token < 0; i0 += 128) {
      double d[4];
      left(i0 + lane * 4, d);
      double v = d[0] + d[1] + d[2] + d[3];
      const double own = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const double t = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += t; }
      const uint32_t over = __ballot_sync(0xffffffffu, run + v > want && own > 0.0), some = __ballot_sync(0xffffffffu, own > 0.0);
      const int hit = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
      int at = -1, latest = -1;
      double c = run + v - own;
#pragma unroll
      for (int u = 0; u < 4; u++) {
        c += d[u];
        if (d[u] > 0.0) { latest = i0 + lane * 4 + u; if (at < 0 && c > want) at = latest; }
      }
      if (at < 0) at = latest;
      const int found = __shfl_sync(0xffffffffu, at, max(hit, 0));
      if (over) token = found;
      else if (some) last = __shfl_sync(0xffffffffu, latest, hit);
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (token < 0) token = last;
    if (lane == 0) out[r] = token;
  }
  cluster.sync();                                            // nobody's shared memory is read any more
}

}  // namespace verify
}  // namespace dsk
