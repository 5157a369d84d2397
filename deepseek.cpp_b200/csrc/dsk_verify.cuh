// dsk_verify.cuh — verification of drafted tokens by speculative sampling, from uniform numbers that the caller gives.
//
// p_i = softmax(logits_i / temperature).  Draft x_i is accepted while coin_i q_i(x_i) < p_i(x_i); the first one that is not is replaced by a draw from max(p_i - q_i, 0), and
// behind accepted ones the next token is drawn from p.  Both draws take the lowest index whose running sum is over (last coin) x (whole sum).
// Two kernels: row_stats reads every row of logits once (maximum and sum of a piece of 1024 per warp, in fp32); pick has a cluster of CTAs for each sequence, which decides
// on the drafts and draws from one row.  A draw's result hangs on sums of up to the whole vocabulary next to a border: in fp32 one draw in some thousands of a flat row would take a
// neighbour.  pick takes that row's exponentials in two fp32 parts, good to 2^-36 of each, as whole numbers of 2^-61 of the power of two above the row's sum, whose sums are the same in
// any order and miss at most 2^-40 of the row by what each loses below one (2^20 entries; as multiples of a fixed 2^-45 at least one each, the tail of a row weighed up to 2^-28 of it, where
// it should have had 2^-32); p and q meet as such numbers too.  Where coin x q is within 1e-4 of p, the row's sum is taken that way as well.
// Bound: row_stats by the bytes of the logits; pick by the instructions of its exponentials (some 86 each, all that a value takes included) where sequences are many, otherwise by the latency of its steps, two walks over a row
// that L2 holds and a cluster's barrier behind each among them.  Seven drafts of 32 sequences over 129280 tokens: 48 us, 14.5 of them row_stats (exponentials in fp64: 71); four drafts of
// one over 32000: 14 us (15.7 with the statistics in pick's clusters instead of a launch of their own).
#pragma once

#include <cooperative_groups.h>

#include "dsk_kv8.cuh"

namespace dsk {
namespace verify {

constexpr int kStatThreads = 256, kStatWarps = kStatThreads / 32, kThreads = 512, kWarps = kThreads / 32, kPiece = 1024, kMaxDrafts = 127, kMaxCluster = 8;

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
__global__ void __launch_bounds__(kStatThreads) row_stats(const Params P) {
  grid_release();
  const int warp = blockIdx.x * kStatWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31, r = blockIdx.y, b = blockIdx.z;
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

// 2^y in fp64, for the few values that drafts are judged by
__device__ __forceinline__ double power(double y) { return y > -1000.0 ? exp2(y) : y <= -1000.0 ? 0.0 : y; }

// 2^y of many values as whole numbers of 2^(down - kBits) (table and series: Tang, "Table-driven implementation of the exponential function in IEEE floating-point arithmetic", 1989).  y = 64 (l - m) / temperature log2(e) in two parts, its integer part k looks up 2^(k mod 64 / 64), the rest f gives e^(f ln2 / 64) - 1
// in two parts, of at most 0.0055; relative error 2^-36 (two roundings to 2^-39, 2^-37.5 for the first bits of the table's entry, less for the series).
constexpr int kBits = 61;                                    // 2^0 is 2^(kBits - down); a row's sum stays below 2^62 where 2^down is above the row's sum
struct Slope { float hi, lo; int down; };                    // 64 log2(e) / temperature; the row's shift
__device__ __forceinline__ uint64_t whole_power(float l, float m, Slope s, const uint4* table) {
  constexpr float C = 0.010830424726009369f, C_LO = -2.976022e-11f;   // ln 2 / 64 in two parts
  const float d = l - m, b = d - l, d_lo = (l - (d - b)) - (m + b);   // l - m exactly
  float y = d * s.hi;
  const bool none = !(y > -4000.f);                          // below 2^-62 (-inf among them)
  const float e = fmaf(d_lo, s.hi, fmaf(d, s.lo, fmaf(d, s.hi, -y)));
  const float t = y + 12582912.f, f0 = y - (t - 12582912.f), f = f0 + e, f_lo = (f0 - f) + e;
  const float z = f * C, z_lo = fmaf(f_lo, C, fmaf(f, C_LO, fmaf(f, C, -z)));
  const float r = fmaf(z * z, fmaf(z, fmaf(z, 1.f / 24.f, 1.f / 6.f), 0.5f), z_lo);
  const int q = __float2int_rn(z * 274877906944.f) + __float2int_rn(r * 274877906944.f);   // 2^38
  const int n = __float_as_int(t) - 0x4b400000;
  const uint4 p = table[n & 63];                             // 2^kBits to 2^(kBits + 1), and its first 31 bits
  const uint64_t v = (((uint64_t)p.y << 32) | p.x) + (uint64_t)(((int64_t)(int)p.z * q) >> (68 - kBits));
  return none ? 0 : v >> min(s.down - (n >> 6), 63);
}
__device__ __forceinline__ uint64_t sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t running(uint64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const uint64_t t = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += t; }
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) pick(const Params P) {
  namespace cg = cooperative_groups;
  __shared__ uint4 table[64];
  __shared__ uint64_t ends[kMaxCluster * kWarps], sums[2][kWarps];
  __shared__ double row_sum[kMaxDrafts + 1];
  __shared__ float row_max[kMaxDrafts + 1];
  __shared__ int flag[kMaxDrafts + 1], top_at[kMaxDrafts + 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / P.cluster, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = drafts_of(P, b), V = P.vocab;
  const bool greedy = P.slope == 0.0;
  const T* logits = static_cast<const T*>(P.logits) + b * P.l_batch;
  const int* drafts = P.drafts + (size_t)b * P.n;
  const float* coins = P.coins + (size_t)b * (P.n + 1);
  const double slope64 = 64.0 * P.slope;
  Slope slope{(float)slope64, (float)(slope64 - (float)slope64), 0};
  if (tid < 64) {
    const uint64_t p = (uint64_t)__double2ll_rn(exp2(tid / 64.0 + kBits));
    table[tid] = make_uint4((uint32_t)p, (uint32_t)(p >> 32), (uint32_t)(p >> (kBits - 30)), 0);
  }
  // what drafts are judged by does not wait for the kernel ahead, which only reads it
  struct Row { int x; float l, q, coin; };
  auto look = [&](int r) {
    Row w{r < n ? drafts[r] : -1, 0.f, 1.f, coins[min(r, P.n)]};
    if ((unsigned)w.x >= (unsigned)V) w.x = -1;
    else { w.l = value(logits[r * P.l_row + w.x]); if (P.probs) w.q = P.probs[b * P.p_batch + r * P.p_row + w.x]; }
    return w;
  };
  Row w = look(warp <= n ? warp : n);
  const float last_coin = coins[P.n];
  grid_wait();
  // rows: maximum and sum of the pieces; 0: refused, 1: accepted, 2: next to the border, 4: not a distribution (a NaN, +inf or nothing but -inf)
  for (int r = warp; r <= n; r += kWarps) {
    if (r != warp) w = look(r);
    const float2* part = P.part + ((size_t)b * (P.n + 1) + r) * P.pieces;
    float m = -INFINITY;
    bool nan = false;
    for (int i = lane; i < P.pieces; i += 32) { const float t = part[i].x; m = fmaxf(m, t); nan |= t != t; }
    m = warp_max(m);
    nan = __any_sync(0xffffffffu, nan);
    if (greedy) {
      unsigned at = 0x7fffffffu;
      for (int i = lane; i < P.pieces; i += 32) if (part[i].x == m) at = min(at, (unsigned)__float_as_int(part[i].y));
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0) { flag[r] = nan || m == -INFINITY ? 4 : w.x == (int)at ? 1 : 0; top_at[r] = (int)at; }
      continue;
    }
    float s = 0.f;                                           // (to 1e-5; what hangs on more is taken again)
    for (int i = lane; i < P.pieces; i += 32) { const float2 t = part[i]; s += t.x == -INFINITY ? t.y : t.y * exp2f((t.x - m) * (float)P.slope); }
    s = warp_sum(s);
    if (lane == 0) {
      int f = 0;
      if (!(m > -INFINITY && m < INFINITY) || !(s < INFINITY)) f = 4;
      else if (w.x >= 0) {
        const double p = power(((double)w.l - m) * P.slope) / s, want = (double)w.coin * w.q;
        f = fabs(want - p) <= 1e-4 * p && p > 0.0 ? 2 : want < p ? 1 : 0;
      }
      flag[r] = f; row_max[r] = m; row_sum[r] = s;
    }
  }
  __syncthreads();
  auto walk = [&](int r, int from, int to, float m) {        // sum of a row's exponentials over indices from .. to - 1 (from a multiple of four), by a warp
    const T* row = logits + r * P.l_row;
    uint64_t s = 0;
    for (int i = from + lane * 4; i < to; i += 512) {
      float x[4][4];
#pragma unroll
      for (int u = 0; u < 4; u++) four(row, i + u * 128, i + u * 128 < to ? V : 0, P.wide_l, x[u]);
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int k = 0; k < 4; k++) s += whole_power(x[u][k], m, slope, table);
    }
    return sum64(s);
  };
  auto down_of = [&](int r) { return (__float_as_int((float)row_sum[r]) >> 23) - 126; };   // (the sum is at least 1, and known to 1e-5 of it)
  const int all = P.cluster * kWarps, share = ((V + all - 1) / all + 127) / 128 * 128, mine = rank * kWarps + warp;   // a warp's indices of the row that is drawn from
  const int from = min(V, mine * share), to = min(V, from + share);
  int r = 0;                                                 // (the same in every CTA of the cluster)
  for (; r < n; r++) {
    int f = flag[r];
    if (f == 2) {
      const int each = ((V + kWarps - 1) / kWarps + 3) / 4 * 4;
      slope.down = down_of(r);
      const uint64_t s = walk(r, min(V, warp * each), min(V, (warp + 1) * each), row_max[r]);
      if (lane == 0) sums[0][warp] = s;
      __syncthreads();
      uint64_t whole = 0;
      for (int k = 0; k < kWarps; k++) whole += sums[0][k];
      __syncthreads();
      const Row y = look(r);
      f = (double)y.coin * y.q < power(((double)y.l - row_max[r]) * P.slope) / ((double)whole * exp2((double)(slope.down - kBits)));
    }
    if (f != 1) break;
  }
  int* out = P.tokens + (size_t)b * (P.n + 1);
  if (rank == 0) {
    for (int i = tid; i <= P.n; i += kThreads) if (i != r) out[i] = i < r ? drafts[i] : -1;
    if (tid == 0) P.accepted[b] = r;
  }
  if (greedy || flag[r] == 4) {
    if (rank == 0 && tid == 0) out[r] = flag[r] == 4 ? -1 : top_at[r];
    return;                                                  // (the whole cluster)
  }
  const float m = row_max[r];
  slope.down = down_of(r);
  const bool drafted = r < n;
  const float* q = drafted && P.probs ? P.probs + b * P.p_batch + r * P.p_row : nullptr;
  auto gather = [&](int which) {                             // sums of all warps of the cluster, in order
    if (tid < all) ends[tid] = *cluster.map_shared_rank(&sums[which][tid % kWarps], tid / kWarps);
    __syncthreads();
  };
  uint64_t whole = 0;
  if (q) {                                                   // (a row that is drawn from by itself needs no sum ahead of its draw)
    const uint64_t s = walk(r, from, to, m);
    if (lane == 0) sums[0][warp] = s;
    cluster.sync();
    gather(0);
    for (int i = lane; i < all; i += 32) whole += ends[i];
    whole = sum64(whole);
  }
  const uint32_t whole_hi = (uint32_t)(whole >> 31), whole_lo = (uint32_t)(whole << 1);   // twice the sum (below 2^63)
  const T* row = logits + r * P.l_row;
  const int certain = drafted && !P.probs ? drafts[r] : -1;
  auto left = [&](int i, int end, uint64_t (&d)[4]) {        // what four indices have in the draw: (p - q) x (sum of the row), none below zero
    float x[4], y[4] = {0.f, 0.f, 0.f, 0.f};
    four(row, i, i < end ? V : 0, P.wide_l, x);
    if (q && i < end) four(q, i, V, P.wide_p, y);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint64_t p = whole_power(x[u], m, slope, table);
      if (!q) { d[u] = i + u >= end || i + u == certain ? 0 : p; continue; }
      const uint32_t bits = __float_as_uint(y[u] + 0.f);     // (-0 is 0; nothing is left where q is negative or not a number; numbers below 2^-126 count as none)
      const int ex = (int)(bits >> 23), by = 127 - ex;
      const uint32_t q32 = (bits & 0x7fffffu) << 8 | 0x80000000u;            // q = q32 2^(ex - 158)
      const uint64_t t = (uint64_t)whole_hi * q32 + __umulhi(whole_lo, q32);   // q x sum x 2^by, cut to a whole number (of 32 bits of the sum alone: off by up to 2^-31 of q)
      const uint64_t other = by < 0 ? p : ex == 0 || by > 63 ? 0 : t >> by;
      d[u] = i + u >= end || other >= p ? 0 : p - other;
    }
  };
  {
    uint64_t s = 0;
#pragma unroll 2
    for (int i = from + lane * 4; i < to; i += 128) {
      uint64_t d[4];
      left(i, to, d);
      s += (d[0] + d[1]) + (d[2] + d[3]);
    }
    s = sum64(s);
    if (lane == 0) sums[1][warp] = s;
  }
  cluster.sync();
  gather(1);
  if (warp == 0) {                                           // running sums of the warps, in order
    uint64_t run = 0;
    for (int i0 = 0; i0 < all; i0 += 32) {
      const uint64_t v = running(i0 + lane < all ? ends[i0 + lane] : 0, lane);
      if (i0 + lane < all) ends[i0 + lane] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const uint64_t total = ends[all - 1], want = min((uint64_t)((double)last_coin * (double)total), total ? total - 1 : 0);   // (behind all: the last index that has anything)
  int owner = -1;                                            // the warp whose indices hold the border
  for (int i0 = 0; i0 < all && owner < 0; i0 += 32) {
    const uint32_t over = __ballot_sync(0xffffffffu, i0 + lane < all && ends[i0 + lane] > want);
    if (over) owner = i0 + __ffs(over) - 1;
  }
  if (owner < 0) {                                           // nothing is left
    if (mine == 0 && lane == 0) out[r] = -1;
  } else if (owner / kWarps == rank) {                       // its CTA takes 128 indices a warp at a time
    const int begin = min(V, owner * share), end = min(V, begin + share);
    uint64_t run = owner ? ends[owner - 1] : 0;
    for (int i0 = begin; i0 < end; i0 += kWarps * 128) {
      uint64_t d[4];
      const int i = i0 + warp * 128 + lane * 4;
      left(i, end, d);
      const uint64_t own = d[0] + d[1] + d[2] + d[3], v = running(own, lane);
      if (lane == 31) sums[0][warp] = v;
      __syncthreads();
      uint64_t before = run, next = run;
#pragma unroll
      for (int k = 0; k < kWarps; k++) { if (k < warp) before += sums[0][k]; next += sums[0][k]; }
      uint64_t c = before + v - own;
      if (c <= want && c + own > want) {                     // (one lane)
        int at = 0;
#pragma unroll
        for (int u = 0; u < 3; u++) { c += d[u]; if (c <= want) at = u + 1; }
        out[r] = i + at;
      }
      if (next > want) break;
      run = next;
      __syncthreads();
    }
  }
  cluster.sync();                                            // nobody's shared memory is read any more
}

}  // namespace verify
}  // namespace dsk
