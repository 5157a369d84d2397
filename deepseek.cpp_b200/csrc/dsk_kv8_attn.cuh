// dsk_kv8_attn.cuh — softmax attention of decoded tokens and drafts over the 8-bit cache (dsk_kv8.cuh).
//
// The queries of a key head are its query heads' queries, `group` heads x `rows` tokens, in tiles of 8.  Products run on mma.sync with keys and values as the left operand:
// scores (16 keys x 8 queries) = K Q^T, results (16 entries x 8 queries) = V^T W; a left operand is converted once whatever the number of query tiles (1 to 3), and no row of a product is
// empty with the few queries of decoding.  An E4M3 code is exact in fp16, so keys and values go from their codes to operands by a conversion alone; a query is divided by a power
// of two that puts its largest entry near 2^10 (what that leaves below fp16's range is 2^-24 of it).  The scales are applied around the products: the key block's to the
// scores, the value block's inside the softmax, w_j = 2^(t_j - m) with t_j = score_j + log2(value scale), so that a weight with its scale is one fp16 number of at most 2^kSlack
// and the sum takes w_j / (value scale).  Rounding: the weights to fp16, 2^-11 of each, and 2^-31 of the row's largest for those below 2^-20 of it: a reference m lies kLift below the largest
// t_j that it was taken from (at that itself, fp16 ends at 2^-25 of the largest weight: of a long tail behind one large weight the sum kept what the results lost, 2^-9 of a row at 131072 keys
// and all of an entry that the large one has as zero); queries in fp16 or bf16 are exact.
// Work: the steps (32 keys, 16 where heads have 256 entries) of all sequences, key heads and query tiles lie in one line that the CTAs share out evenly, four steps to a unit, whatever the lengths; a CTA that has
// a whole (sequence, head, tile) stores it, pieces are joined by `join`.  Every warp has every fourth step, with stages of its own that cp.async fills: no barrier but where
// a piece ends, and the copies run on across pieces.
// A call of few pieces has clusters instead of the line (SHARED).
// Bound: in large calls the dependent instructions of a step (some 560 for 32 keys and a tile of 8 queries: conversions, fragments, products, softmax; steps of 16 keys spend more of
// them on what a step does once) at 8 warps an SM, which leave 64 % of the issue slots empty; in small calls the chain of a step and the joins.  64 sequences of up to 16000 tokens, 16 heads of 128 over 4: 107 us (533 MB: 5.0 TB/s; a measured copy 6.5);
// a token and four drafts of 16 sequences, window 1024: 18 us; one token behind 1000: 8.6 us.  With queries as the left operand, half of whose rows were empty: 295 us for the first.
// Fragments come from shared memory as whole 16-byte pieces, entries and keys permuted alike on both sides of a product: a quarter warp's lanes (two
// keys x four pieces) are keys j and j + 4, whose rows lie 16 banks apart.
#pragma once

#include <cooperative_groups.h>

#include "dsk_kv8.cuh"
#include "dsk_tmem.cuh"

namespace dsk {
namespace kv8 {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kMaxBatch = 1024;
__host__ __device__ constexpr int step_of(int dv) { return dv < 256 ? 32 : 16; }   // keys of a warp's step (as two CTAs of an SM have registers and stages for)
__device__ __forceinline__ long long quotient(long long a, long long b) { return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b; }   // (of numbers >= 0)
constexpr float kLowest = -3e38f;                            // a maximum ahead of the first score (finite: no difference of infinities)
constexpr float kFar = 16777216.f;                           // scores beyond it are rounded ahead of the subtraction: what fma keeps of a product that its reference does not would be exponents
constexpr float kLift = 7.f, kSlack = 15.f;                  // the reference of a row's weights is taken kLift below its maximum, and follows once that is kSlack ahead (fp16 ends at 2^16)

struct Attn {
  Cache C;
  Rows S;                                                    // first: tokens of a sequence in the cache, its queries the last ones
  const void* q;
  void* out;
  Pitch pq, po;
  int heads, group, row_tiles, bf16, wide_q, wide_o, window, keep, cluster;   // cluster: CTAs that share a (sequence, head, tile), 0: the line
  float scale;                                               // times log2(e)
  float* part;                                               // workspace: pieces
};

// What a sequence has: visible steps are the first `kept` ones and those from `low` on
struct Seq { int len, count, kept, low, steps, units, first, last; };   // first, last: positions of the queries
template <int STEP> __device__ __forceinline__ Seq sequence(const Attn& P, int b) {
  Seq q;
  const long long room = (long long)P.S.table_blocks << P.C.shift;
  const int len = max(P.S.first[b], -1);                     // (positions of the queries do not wrap)
  q.count = P.S.count ? min(max(P.S.count[b], 0), P.S.rows) : P.S.rows;
  q.len = (int)min((long long)max(len, 0), room);
  const long long first = (long long)len - q.count + 1 - P.window;
  q.low = P.window > 0 && first > 0 ? (int)min(first, (long long)q.len) / STEP : 0;
  q.kept = P.window > 0 ? min((min(P.keep, q.len) + STEP - 1) / STEP, q.low) : 0;
  q.steps = q.kept + (q.len + STEP - 1) / STEP - q.low;
  q.units = q.count ? max(1, (q.steps + kWarps - 1) / kWarps) : 0;
  q.last = len - 1;
  q.first = len - q.count;
  return q;
}

template <int DK, int DV, int QT> __host__ __device__ constexpr int stages() {   // as many as two CTAs of an SM have room for
  return DK == 64 ? 3 : 2;
}
template <int DK, int DV> __host__ __device__ constexpr int stage_bytes(int step) { return step * (DK + 16 + DV + 32) + 16; }
template <int DK, int DV, int QT> __host__ __device__ constexpr int attn_smem() {
  return kWarps * stages<DK, DV, QT>() * stage_bytes<DK, DV>(step_of(DV)) + QT * 8 * (2 * DK + 16) + 2 * QT * DV / 4 * 128 + (2 * kWarps + 1) * QT * 8 * 4;
}

template <int to, int from> __device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(to), "n"(from) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// pieces J .. N - 1 of a lane, 512 bytes apart where they come from; they go to place[j] of the u-th 16 rows
template <int N, int J, int HALF> __device__ __forceinline__ void copy_rows(uint32_t to, const uint32_t (&place)[N], const unsigned char* from, int u) {
  if constexpr (J < N) {
    if (u == 0) copy16<0, J * 512>(to + place[J], from); else copy16<HALF, J * 512>(to + place[J], from);
    copy_rows<N, J + 1, HALF>(to, place, from, u);
  }
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {     // an 8 x 8 matrix of 16-bit entries (row lane / 4, two entries a lane), transposed
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {   // 0xff where a byte is NaN
  return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

// CTAs that share the line out: where each (sequence, head, tile) has several, as many to each, so that those of equal length have whole pieces
__device__ __forceinline__ long long ctas_of(int grid, long long total, long long each) {
  const long long n = 2 * each <= grid ? grid / (int)each * each : grid;
  return min(n, total);
}

// A place in the line of units
template <int STEP> struct Place {
  Seq q;
  int b, head, tile, unit;
  const int* table;                                          // the sequence's row
  __device__ __forceinline__ void find(const Attn& P, const long long* ends, long long x, int per) {   // per: heads x row tiles
    int lo = 0, hi = P.S.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (ends[mid] * per <= x) lo = mid; else hi = mid - 1;
    }
    b = lo;
    table = P.S.table + b * P.S.table_pitch;
    q = sequence<STEP>(P, b);
    const long long in = x - ends[b] * per;
    const int hr = (int)quotient(in, q.units);
    unit = (int)(in - (long long)hr * q.units);
    head = hr / P.row_tiles;
    tile = hr - head * P.row_tiles;
  }
  __device__ __forceinline__ void next(const Attn& P) {
    if (++unit < q.units) return;
    unit = 0;
    if (++tile < P.row_tiles) return;
    tile = 0;
    if (++head < P.C.heads) return;
    head = 0;
    do {
      if (++b >= P.S.batch) return;
      table += P.S.table_pitch;
      q = sequence<STEP>(P, b);
    } while (q.units == 0);
  }
};

// Rows of a tile: row r of a key head is token r / group, head r % group
struct Out {
  __device__ static __forceinline__ void store(const Attn& P, const Seq& q, int b, int head, int row, int d0, int n, const float* x, float inv) {   // n values (8 or 16) from entry d0 on
    const int i = row / P.group, dim = P.C.dim[1];
    if (i >= q.count || d0 >= dim) return;
    const long long at = b * P.po.batch + i * P.po.row + (long long)(head * P.group + row - i * P.group) * P.po.head + d0;
    uint16_t o[16];
#pragma unroll
    for (int k = 0; k < 16; k++)
      if (k < n) o[k] = P.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x[k] * inv)) : __half_as_ushort(__float2half_rn(x[k] * inv));
    uint16_t* p = static_cast<uint16_t*>(P.out) + at;
#pragma unroll
    for (int k = 0; k < 16; k += 8)
      if (k < n) {
        if (P.wide_o) *reinterpret_cast<uint4*>(p + k) = make_uint4(o[k] | (uint32_t)o[k + 1] << 16, o[k + 2] | (uint32_t)o[k + 3] << 16, o[k + 4] | (uint32_t)o[k + 5] << 16, o[k + 6] | (uint32_t)o[k + 7] << 16);
        else
#pragma unroll
          for (int u = 0; u < 8; u++) p[k + u] = o[k + u];
      }
  }
};

// Joins n pieces of a (sequence, head, query tiles), piece(i): [accumulator][lane], maxima, sums.  A warp has eight entries of one of every lane's two queries: warp `task` of QT DV / 32.
template <int DV, int QT, typename F>
__device__ __forceinline__ void join_pieces(const Attn& P, const Seq& q, int b, int head, int row0, int task, int lane, int n, F piece) {
  constexpr int NO = DV / 16, VCH = DV >= 128 ? 16 : 8;
  const int r = lane >> 2, c = lane & 3, e = task & 1;
  task >>= 1;
  const int k0 = (task % (DV / 64)) * 8, t = task / (DV / 64), row = t * 8 + 2 * c + e;   // k0: of a lane's DV / 8 entries
  float x[16], m = kLowest, l = 0.f;
#pragma unroll
  for (int k = 0; k < 8; k++) x[k] = 0.f;
  constexpr int AT = 8;                                      // pieces under way
  for (int i = 0; i < n; i += AT) {
    float pm[AT], pl[AT], px[AT][8], to = m;
#pragma unroll
    for (int u = 0; u < AT; u++) {
      if (i + u >= n) { pm[u] = -INFINITY; continue; }
      const float* from = piece(i + u);
      pm[u] = from[QT * NO * 128 + row];
      pl[u] = from[QT * NO * 128 + QT * 8 + row];
#pragma unroll
      for (int k = 0; k < 8; k++) px[u][k] = from[((t * NO + (k0 + k) / 2) * 4 + 2 * (k & 1) + e) * 32 + lane];
    }
#pragma unroll
    for (int u = 0; u < AT; u++) to = fmaxf(to, pm[u]);
    const float f = exp2_fast(m - to);
    m = to;
    l *= f;
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] *= f;
#pragma unroll
    for (int u = 0; u < AT; u++) {
      if (i + u >= n) break;
      const float g = exp2_fast(pm[u] - m);
      l = fmaf(pl[u], g, l);
#pragma unroll
      for (int k = 0; k < 8; k++) x[k] = fmaf(px[u][k], g, x[k]);
    }
  }
  Out::store(P, q, b, head, row0 + row, k0 / VCH * 128 + r * VCH + k0 % VCH, 8, x, l == 0.f ? 0.f : 1.f / l);
}

// DK, DV: entries of keys and values, rounded up; QT: tiles of 8 queries.  SHARED: P.cluster CTAs have one (sequence, head, tile) and join their pieces in one another's shared memory
// (one token behind 1000, 16 heads over 4: 8.7 us, 9.2 by the line with its second launch, whose call takes the host 14 us instead of 9).
template <int DK, int DV, int QT, bool SHARED>
__global__ void __launch_bounds__(kThreads) attend_tokens(const Attn P) {
  constexpr int NST = stages<DK, DV, QT>(), KS = DK + 16, VS = DV + 32, STEP = step_of(DV), HV = STEP / 16, SB = stage_bytes<DK, DV>(STEP), QS = 2 * DK + 16, VCH = DV >= 128 ? 16 : 8,
                HF = DV / (8 * VCH), NO = DV / 16;           // NO: tiles of 16 entries; a lane's entries are VCH neighbours, two to a tile
  constexpr bool QREG = QT * DK <= 256;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ long long warp_sums[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, B = P.S.batch;
  unsigned char* q_raw = raw + kWarps * NST * SB;
  float* turn = reinterpret_cast<float*>(q_raw + QT * 8 * QS);           // [2][accumulators][lane]
  float* row_m = turn + 2 * QT * NO * 4 * 32;                            // [warp][query]
  float* row_l = row_m + kWarps * QT * 8;
  float* row_q = row_l + kWarps * QT * 8;                                // factor of a query's scores
  long long* ends = reinterpret_cast<long long*>(raw + ((attn_smem<DK, DV, QT>() + 7) & ~7));
  const uint32_t stage0 = smem_u32(raw) + warp * NST * SB, q0 = smem_u32(q_raw);
  const int per = P.C.heads * P.row_tiles;
  int mine, rank = 0;                                        // units of this CTA
  Place<STEP> at;                                            // of the next copies
  if (P.C.dim[0] < DK || P.C.dim[1] < DV)
    for (int i = threadIdx.x; i < NST * SB * kWarps / 16; i += kThreads) reinterpret_cast<uint4*>(raw)[i] = make_uint4(0, 0, 0, 0);   // (entries behind the last one stay zero)
  if constexpr (SHARED) {
    const int u = blockIdx.x / P.cluster, hr = u % per;
    rank = blockIdx.x - u * P.cluster;
    at.b = u / per;
    at.q = sequence<STEP>(P, at.b);
    if (rank == 0 && hr == 0 && threadIdx.x == 0) {
      const long long len = P.S.first[at.b];
      if (len < 0 || len > (long long)P.S.table_blocks << P.C.shift) note(P.C, ST_RANGE);
    }
    if (at.q.count == 0) return;                             // (the whole cluster)
    at.head = hr / P.row_tiles;
    at.tile = hr - at.head * P.row_tiles;
    at.table = P.S.table + at.b * P.S.table_pitch;
    at.unit = (int)((long long)at.q.units * rank / P.cluster);
    mine = (int)((long long)at.q.units * (rank + 1) / P.cluster) - at.unit;
    __syncthreads();
  } else {
    grid_release();
    // line of units: running sums over the sequences
    long long run = 0;
    for (int b0 = 0; b0 < B; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const long long own = b < B ? sequence<STEP>(P, b).units : 0;
      long long v = own;
  #pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += t; }
      if (lane == 31) warp_sums[warp] = v;
      __syncthreads();
      long long before = run, all = run;
  #pragma unroll
      for (int w = 0; w < kWarps; w++) { if (w < warp) before += warp_sums[w]; all += warp_sums[w]; }
      if (b < B) ends[b] = before + v - own;
      run = all;
      __syncthreads();
    }
    const long long total = run * per, N = ctas_of(gridDim.x, total, (long long)B * per);
    if (blockIdx.x == 0) {
      for (int b = threadIdx.x; b < B; b += kThreads) {
        const long long len = P.S.first[b];
        if (len < 0 || len > (long long)P.S.table_blocks << P.C.shift) note(P.C, ST_RANGE);
      }
    }
    if ((long long)blockIdx.x >= N) return;
    const long long x0 = quotient(blockIdx.x * total, N), x1 = quotient((blockIdx.x + 1) * total, N);
    mine = (int)(x1 - x0);
    __syncthreads();
    at.find(P, ends, x0, per);
  }
  const int dk = P.C.dim[0], dv = P.C.dim[1], dk16 = dk / 16, dv16 = dv / 16;
  const bool exact = dk == DK && dv == DV;
  const uint32_t head_k = P.C.block * dk, head_v = P.C.block * dv, block_k = P.C.heads * head_k, block_v = P.C.heads * head_v;   // bytes of a head and of a block (at most 2^30)
  const float* my_scale = P.C.scale[lane & 1];

  // copies: a step of this warp to a unit, from a block whose number was looked up a unit ahead; 16-byte pieces lane, lane + 32, .. of a step's rows, which lie side by side
  uint32_t to_k[DK / 32], to_v[DV / 32];
  {
    int row = lane / dk16, col = lane - row * dk16;
    const int dr = 32 / dk16, dc = 32 - dr * dk16;
#pragma unroll
    for (int j = 0; j < DK / 32; j++) { to_k[j] = row * KS + col * 16; row += dr; col += dc; if (col >= dk16) { col -= dk16; row++; } }
  }
  {
    int row = lane / dv16, col = lane - row * dv16;
    const int dr = 32 / dv16, dc = 32 - dr * dv16;
#pragma unroll
    for (int j = 0; j < DV / 32; j++) { to_v[j] = STEP * KS + row * VS + col * 16; row += dr; col += dc; if (col >= dv16) { col -= dv16; row++; } }
  }
  int ahead = mine, page[HV], key = -1;                      // units that are not under way yet; the next step's blocks (of 16 keys each) and first key (-1: this warp has none)
  auto look = [&]() {
    const int s = at.unit * kWarps + warp;
    key = -1;
    if (ahead > 0 && s < at.q.steps) {
      key = (s < at.q.kept ? s : at.q.low + s - at.q.kept) * STEP;
      page[0] = __ldg(at.table + (key >> P.C.shift));
      if (HV == 2) page[HV - 1] = P.C.shift > 4 ? page[0] : key + 16 < at.q.len ? __ldg(at.table + (key >> 4) + 1) : -1;   // (-1: behind the last key)
    }
  };
  auto fetch = [&](int stage) {
    if (key >= 0) {
      const uint32_t to = stage0 + stage * SB;
#pragma unroll
      for (int u = 0; u < HV; u++) {
        const bool ok = (unsigned)page[u] < (unsigned)P.C.n_blocks;
        const uint32_t at_page = ok ? page[u] : 0, row0 = (key + 16 * u) & (P.C.block - 1);
        const unsigned char* k = P.C.code[0] + ((uint64_t)at_page * block_k + (at.head * head_k + row0 * dk + lane * 16));
        const unsigned char* v = P.C.code[1] + ((uint64_t)at_page * block_v + (at.head * head_v + row0 * dv + lane * 16));
        const float* scale = my_scale + ((uint64_t)at_page * (uint32_t)P.C.heads + at.head);
        if (ok && exact && key + 16 * u + 16 <= at.q.len) {
          copy_rows<DK / 32, 0, 16 * KS>(to, to_k, k, u);
          copy_rows<DV / 32, 0, 16 * VS>(to, to_v, v, u);
          if (lane < 2) copy4(to + STEP * (KS + VS) + u * 8 + lane * 4, scale, 4);
        } else {                                             // what is behind the last key, or in a block outside the cache, comes as zeros, its scales too where the block is nobody's
          if (!ok && lane == 0 && key + 16 * u < at.q.len) note(P.C, ST_PAGE);
          const int there = ok ? at.q.len - key - 16 * u : 0;
          for (int i = lane; i < dk; i += 32) { const int row = i / dk16; copy16_or_zero(to + (u * 16 + row) * KS + (i - row * dk16) * 16, row < there ? k + (i - lane) * 16 : P.C.code[0], row < there); }
          for (int i = lane; i < dv; i += 32) { const int row = i / dv16; copy16_or_zero(to + STEP * KS + (u * 16 + row) * VS + (i - row * dv16) * 16, row < there ? v + (i - lane) * 16 : P.C.code[1], row < there); }
          if (lane < 2) copy4(to + STEP * (KS + VS) + u * 8 + lane * 4, ok ? scale : P.C.scale[0], ok ? 4 : 0);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (--ahead > 0) at.next(P);
    look();
  };
  look();
  Place<STEP> pl = at;                                       // of the step that is computed
  uint32_t qv[QT * 2][DK / 64];                              // a piece's query rows on their way, two entries a lane
  auto load_queries = [&]() {
#pragma unroll
    for (int u = 0; u < QT * 2; u++) {
      const int row = pl.tile * QT * 8 + u * kWarps + warp, i = row / P.group;
      const uint16_t* src = static_cast<const uint16_t*>(P.q) + pl.b * P.pq.batch + i * P.pq.row + (long long)(pl.head * P.group + row - i * P.group) * P.pq.head + lane * 2;
#pragma unroll
      for (int k = 0; k < DK / 64; k++) {
        qv[u][k] = 0;
        if (i < pl.q.count && k * 64 + lane * 2 < dk) qv[u][k] = P.wide_q ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 64)) : src[k * 64] | (uint32_t)src[k * 64 + 1] << 16;
      }
    }
  };
  load_queries();
#pragma unroll 1
  for (int i = 0; i < NST - 1; i++) fetch(i);

  float o[QT][NO][4], m[QT][2], l[QT][2], fq[QT][2];         // a lane's queries: 2 c and 2 c + 1 of a tile; fq: factor of their scores
  uint32_t qf[QREG ? QT : 1][QREG ? DK / 16 : 1][2];
  int begun = pl.unit, stage = 0;                            // the piece's first unit
  bool fresh = true;
#pragma unroll 1
  for (int y = 0; y < mine; y++) {
    const Seq& q = pl.q;
    const int head = pl.head, row0 = pl.tile * QT * 8;
    if (fresh) {                                             // query rows as fp16, each by its own power of two
      __syncthreads();
      if (y > 0) load_queries();
#pragma unroll
      for (int u = 0; u < QT * 2; u++) {
        const int row = u * kWarps + warp;
        float v[DK / 32], top = 0.f;
#pragma unroll
        for (int k = 0; k < DK / 64; k++) {
          const float2 f = P.bf16 ? make_float2(__uint_as_float(qv[u][k] << 16), __uint_as_float(qv[u][k] & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&qv[u][k]));
          v[2 * k] = f.x; v[2 * k + 1] = f.y;
          const float x = fabsf(f.x), y = fabsf(f.y);
          top = fmaxf(top, fmaxf(x < INFINITY ? x : 0.f, y < INFINITY ? y : 0.f));
        }
        top = warp_max(top);
        const int e = top > 0.f ? max(-100, min(120, (int)(__float_as_uint(top) >> 23) - 127 - 10)) : 0;
        const float by = P.scale < 0.f ? -pow2(-e) : pow2(-e);               // (factors of scores are positive)
#pragma unroll
        for (int k = 0; k < DK / 64; k++) *reinterpret_cast<uint32_t*>(q_raw + row * QS + (k * 64 + lane * 2) * 2) = halves(v[2 * k] * by, v[2 * k + 1] * by);
        if (lane == 0) row_q[row] = pow2(e) * fabsf(P.scale);
      }
      __syncthreads();
      if constexpr (QREG) {
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int i = 0; i < DK / 32; i++) {
            const uint4 a = lds128(q0 + (t * 8 + r) * QS + (i / 2 * 64 + 16 * c + 8 * (i & 1)) * 2);
            qf[t][2 * i][0] = a.x; qf[t][2 * i][1] = a.y; qf[t][2 * i + 1][0] = a.z; qf[t][2 * i + 1][1] = a.w;
          }
      }
#pragma unroll
      for (int t = 0; t < QT; t++) {
#pragma unroll
        for (int e = 0; e < 2; e++) { m[t][e] = kLowest; l[t][e] = 0.f; fq[t][e] = row_q[t * 8 + 2 * c + e]; }
#pragma unroll
        for (int k = 0; k < NO; k++)
#pragma unroll
          for (int u = 0; u < 4; u++) o[t][k][u] = 0.f;
      }
      fresh = false;
    }
    fetch(stage == 0 ? NST - 1 : stage - 1);                 // (the stage read last)
    asm volatile("cp.async.wait_group %0;" ::"n"(NST - 1) : "memory");
    __syncwarp();
    const int step = pl.unit * kWarps + warp;
    if (step < q.steps) {
      const uint32_t from = stage0 + stage * SB;
      const int key0 = (step < q.kept ? step : q.low + step - q.kept) * STEP;
      float ks[HV], lift[HV], back[HV];                      // scales: of keys; of values as exponent and reciprocal
      bool gone = false;
#pragma unroll
      for (int u = 0; u < HV; u++) {
        ks[u] = __uint_as_float(lds32(from + STEP * (KS + VS) + u * 8));
        const float vs = __uint_as_float(lds32(from + STEP * (KS + VS) + u * 8 + 4));
        lift[u] = (float)((int)(__float_as_uint(vs) >> 23) - 127);
        back[u] = pow2(-(int)lift[u]);
        if (vs == 0.f) { back[u] = 0.f; gone = true; }
      }
      float s[QT][HV][4];                                    // keys r, r + 8 (permuted) x queries 2 c, 2 c + 1
#pragma unroll
      for (int t = 0; t < QT; t++)
#pragma unroll
        for (int u = 0; u < HV; u++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[t][u][i] = 0.f;
      const int turn_r = (r >> 1) + 4 * (r & 1);
      const uint32_t krow = from + turn_r * KS + c * 16;
#pragma unroll
      for (int g = 0; g < DK / 64; g++) {
        uint32_t kw[HV][2][4];
#pragma unroll
        for (int u = 0; u < HV; u++)
#pragma unroll
          for (int e = 0; e < 2; e++) { const uint4 x = lds128(krow + (u * 16 + e * 8) * KS + g * 64); kw[u][e][0] = x.x; kw[u][e][1] = x.y; kw[u][e][2] = x.z; kw[u][e][3] = x.w; }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t a[HV][2][4];
#pragma unroll
          for (int u = 0; u < HV; u++)
#pragma unroll
            for (int x = 0; x < 2; x++) { four_halves(kw[u][0][2 * h + x], a[u][x][0], a[u][x][2]); four_halves(kw[u][1][2 * h + x], a[u][x][1], a[u][x][3]); }
#pragma unroll
          for (int t = 0; t < QT; t++) {
            uint32_t b[2][2];
            if constexpr (QREG) {
#pragma unroll
              for (int x = 0; x < 2; x++) { b[x][0] = qf[t][g * 4 + 2 * h + x][0]; b[x][1] = qf[t][g * 4 + 2 * h + x][1]; }
            } else {
              const uint4 y = lds128(q0 + (t * 8 + r) * QS + (g * 64 + 16 * c + 8 * h) * 2);
              b[0][0] = y.x; b[0][1] = y.y; b[1][0] = y.z; b[1][1] = y.w;
            }
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
              for (int u = 0; u < HV; u++) mma16(s[t][u], a[u][x], b[x][0], b[x][1]);
          }
        }
      }
      // a step that every query sees needs no mask
      const bool masked = key0 + STEP - 1 > q.first || (P.window > 0 && q.last - key0 >= P.window && key0 + STEP > P.keep) || gone;
      // keys that a query sees, a bit each: not behind its own, in the window or among the first, in the cache
      auto sees = [&](int t, int e) {
        const int pos = q.first + (row0 + t * 8 + 2 * c + e) / P.group;
        uint32_t see = lower_bits(pos + 1 - key0);
        if (P.window > 0) see &= ~lower_bits(pos - P.window + 1 - key0) | lower_bits(P.keep - key0);
        see &= lower_bits(q.len - key0);
        if (back[0] == 0.f) see &= ~0xffffu;
        if (HV == 2 && back[HV - 1] == 0.f) see &= 0xffffu;
        return see >> turn_r;                                // (bit 16 u + 8 h: key of score [u][h])
      };
      if (masked) {
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t see = sees(t, e);
#pragma unroll
            for (int u = 0; u < HV; u++)
#pragma unroll
              for (int h = 0; h < 2; h++) if (!(see >> (16 * u + 8 * h) & 1)) s[t][u][2 * h + e] = -INFINITY;
          }
      }
      uint32_t w[QT][HV][2];                                 // weights as right operands: [query r][keys 2 c, 2 c + 1]
#pragma unroll
      for (int t = 0; t < QT; t++) {
        float f[2][HV], mx[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          mx[e] = -INFINITY;
#pragma unroll
          for (int u = 0; u < HV; u++) {
            f[e][u] = fmaxf(fq[t][e] * ks[u], 1.17549435e-38f);      // (positive: -inf stays what it is)
            mx[e] = fmaxf(mx[e], fmaf(fmaxf(s[t][u][e], s[t][u][2 + e]), f[e][u], lift[u]));
          }
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[t][0] + kSlack || mx[1] > m[t][1] + kSlack || fmaxf(fabsf(mx[0]), fabsf(mx[1])) > kFar)) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int u = 0; u < HV; u++)
              if (fabsf(mx[e]) > kFar) {
                s[t][u][e] = fmaf(s[t][u][e], f[e][u], lift[u]) - lift[u];
                s[t][u][2 + e] = fmaf(s[t][u][2 + e], f[e][u], lift[u]) - lift[u];
                f[e][u] = 1.f;
              }
            const float to = fmaxf(m[t][e], fabsf(mx[e]) > kFar ? mx[e] : mx[e] - kLift), by = exp2_fast(m[t][e] - to);
            m[t][e] = to;
            l[t][e] *= by;
#pragma unroll
            for (int k = 0; k < NO; k++) { o[t][k][e] *= by; o[t][k][2 + e] *= by; }
          }
        }
#pragma unroll
        for (int u = 0; u < HV; u++) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float off = lift[u] - m[t][e];
            p[e] = exp2_fast(fmaf(s[t][u][e], f[e][u], off));
            p[2 + e] = exp2_fast(fmaf(s[t][u][2 + e], f[e][u], off));
            l[t][e] = fmaf(p[e] + p[2 + e], back[u], l[t][e]);
          }
          w[t][u][0] = turned(halves(p[0], p[1]));
          w[t][u][1] = turned(halves(p[2], p[3]));
        }
      }
      const uint32_t vrow = from + STEP * KS + c * VS + r * VCH;
      auto values = [&](int hf, int key, uint32_t (&x)[VCH / 4]) {
        if constexpr (VCH == 16) { const uint4 y = lds128(vrow + key * VS + hf * 128); x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w; }
        else { const uint2 y = lds64(vrow + key * VS); x[0] = y.x; x[1] = y.y; }
      };
      bool nan = false;
      // a NaN among values that some query does not see must not reach that query, whose weight for it is zero (behind the last key there are zeros)
      if (masked && (min(key0 + STEP, q.len) - 1 > q.first || (P.window > 0 && q.last - key0 >= P.window))) {
#pragma unroll 1
        for (int hf = 0; hf < HF; hf++)
#pragma unroll 4
          for (int k = 0; k < STEP / 4; k++) {
            uint32_t x[VCH / 4];
            values(hf, k * 4, x);
#pragma unroll
            for (int u = 0; u < VCH / 4; u++) nan |= nan_bytes(x[u]) != 0;
          }
        nan = __any_sync(0xffffffffu, nan);
      }
#pragma unroll
      for (int y = 0; y < HV * HF; y++) {
        const int hf = y % HF, sub = y / HF;                 // (constants once unrolled)
        uint32_t x[4][VCH / 4];
        values(hf, sub * 16, x[0]); values(hf, sub * 16 + 4, x[1]); values(hf, sub * 16 + 8, x[2]); values(hf, sub * 16 + 12, x[3]);
        if (nan) {                                           // counts of the NaN that a query sees, two entries at a time, then numbers alone
          uint32_t see[QT][2];
#pragma unroll
          for (int t = 0; t < QT; t++) {
            const uint32_t see0 = sees(t, 0), see1 = sees(t, 1);
#pragma unroll
            for (int h = 0; h < 2; h++) see[t][h] = turned(((see0 >> (16 * sub + 8 * h)) & 1 ? 0x3c00u : 0u) | ((see1 >> (16 * sub + 8 * h)) & 1 ? 0x3c000000u : 0u));
          }
#pragma unroll
          for (int k = 0; k < VCH / 2; k++) {
            uint32_t a[4];
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
              for (int h = 0; h < 2; h++) {
                const int byte = 8 * ((2 * k + e) & 3);
                a[2 * h + e] = ((nan_bytes(x[2 * h][(2 * k + e) / 4]) >> byte) & 1 ? 0x3c00u : 0u) | ((nan_bytes(x[2 * h + 1][(2 * k + e) / 4]) >> byte) & 1 ? 0x3c000000u : 0u);
              }
#pragma unroll
            for (int t = 0; t < QT; t++) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
              mma16(d, a, see[t][0], see[t][1]);
#pragma unroll
              for (int i = 0; i < 4; i++) if (d[i] > 0.f) o[t][hf * VCH / 2 + k][i] = NAN;
            }
          }
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int u = 0; u < VCH / 4; u++) x[k][u] &= ~nan_bytes(x[k][u]);
        }
#pragma unroll
        for (int u = 0; u < VCH / 4; u++) {                  // four entries: two tiles, whose rows r and r + 8 are neighbouring entries
          const uint32_t lo0 = __byte_perm(x[0][u], x[1][u], 0x5140), hi0 = __byte_perm(x[0][u], x[1][u], 0x7362);
          const uint32_t lo1 = __byte_perm(x[2][u], x[3][u], 0x5140), hi1 = __byte_perm(x[2][u], x[3][u], 0x7362);
          uint32_t a[2][4];
          four_halves(lo0, a[0][0], a[0][1]);
          four_halves(lo1, a[0][2], a[0][3]);
          four_halves(hi0, a[1][0], a[1][1]);
          four_halves(hi1, a[1][2], a[1][3]);
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int t = 0; t < QT; t++) mma16(o[t][hf * VCH / 2 + u * 2 + k], a[k], w[t][sub][0], w[t][sub][1]);
        }
      }
    }
    __syncwarp();                                            // the stage is read
    if (++stage == NST) stage = 0;
    // where the piece ends: the warps' sums in one
    const bool whole_end = pl.unit + 1 == q.units;
    if (whole_end || y + 1 == mine) {
#pragma unroll
      for (int t = 0; t < QT; t++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], x);
          if (r == 0) { row_m[warp * QT * 8 + t * 8 + 2 * c + e] = m[t][e]; row_l[warp * QT * 8 + t * 8 + 2 * c + e] = l[t][e]; }
        }
      __syncthreads();
      float top[QT][2], sum[QT][2];
#pragma unroll
      for (int t = 0; t < QT; t++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int row = t * 8 + 2 * c + e;
          top[t][e] = row_m[row];
#pragma unroll
          for (int w = 1; w < kWarps; w++) top[t][e] = fmaxf(top[t][e], row_m[w * QT * 8 + row]);
          sum[t][e] = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; w++) sum[t][e] += row_l[w * QT * 8 + row] * exp2_fast(row_m[w * QT * 8 + row] - top[t][e]);
          const float f = exp2_fast(m[t][e] - top[t][e]);
#pragma unroll
          for (int k = 0; k < NO; k++) { o[t][k][e] *= f; o[t][k][2 + e] *= f; }
        }
      float* mine_at = turn + (warp & 1) * QT * NO * 128 + lane;
      auto put = [&]() {
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int k = 0; k < NO; k++)
#pragma unroll
            for (int u = 0; u < 4; u++) mine_at[((t * NO + k) * 4 + u) * 32] = o[t][k][u];
      };
      auto add = [&](const float* other) {
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
          for (int k = 0; k < NO; k++)
#pragma unroll
            for (int u = 0; u < 4; u++) o[t][k][u] += other[((t * NO + k) * 4 + u) * 32];
      };
      if (warp >= 2) put();
      __syncthreads();
      if (warp < 2) add(mine_at);
      if (warp == 1) put();
      __syncthreads();
      if (warp == 0) {
        add(turn + QT * NO * 128 + lane);
        __syncwarp();
        if (!SHARED && begun == 0 && whole_end) {
#pragma unroll
          for (int t = 0; t < QT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float inv = sum[t][e] == 0.f ? 0.f : 1.f / sum[t][e];        // (a query that sees nothing: zeros)
#pragma unroll
              for (int hf = 0; hf < HF; hf++) {
                float x[16];
#pragma unroll
                for (int k = 0; k < VCH; k++) x[k] = o[t][hf * VCH / 2 + k / 2][2 * (k & 1) + e];
                Out::store(P, q, pl.b, head, row0 + t * 8 + 2 * c + e, hf * 128 + r * VCH, VCH, x, inv);
              }
            }
        } else {                                             // a piece: [accumulator][lane], then maxima and sums of the queries
          float* to = SHARED ? turn : P.part + (size_t)(2 * blockIdx.x + (y == pl.unit - begun ? 0 : 1)) * (QT * (NO * 128 + 16));
#pragma unroll
          for (int t = 0; t < QT; t++) {
#pragma unroll
            for (int k = 0; k < NO; k++)
#pragma unroll
              for (int u = 0; u < 4; u++) to[((t * NO + k) * 4 + u) * 32 + lane] = o[t][k][u];
            if (r == 0)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                to[QT * NO * 128 + t * 8 + 2 * c + e] = top[t][e];
                to[QT * NO * 128 + QT * 8 + t * 8 + 2 * c + e] = sum[t][e];
              }
          }
        }
      }
      fresh = true;
    }
    pl.next(P);
    if (fresh) begun = pl.unit;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if constexpr (SHARED) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (mine == 0) {                                         // (more CTAs than units)
      for (int i = threadIdx.x; i < QT * NO * 128; i += kThreads) turn[i] = 0.f;
      for (int i = threadIdx.x; i < QT * 8; i += kThreads) { turn[QT * NO * 128 + i] = kLowest; turn[QT * NO * 128 + QT * 8 + i] = 0.f; }
    }
    cluster.sync();
    for (int task = rank * kWarps + warp; task < QT * DV / 32; task += P.cluster * kWarps)
      join_pieces<DV, QT>(P, at.q, at.b, at.head, at.tile * QT * 8, task, lane, P.cluster, [&](int i) { return (const float*)cluster.map_shared_rank(turn, i); });
    cluster.sync();                                          // nobody's shared memory is read any more
  }
}

// Joins the pieces that several CTAs of the line had
template <int DV, int QT>
__global__ void __launch_bounds__(QT * DV) join(const Attn P, int ctas) {
  constexpr int NO = DV / 16;
  // who had what is known without the kernel ahead
  __shared__ long long sums[2][QT * DV / 32];
  const int b = blockIdx.y, hr = blockIdx.x, per = gridDim.x;
  long long before = 0, all = 0;
  for (int i = threadIdx.x; i < P.S.batch; i += QT * DV) { const int u = sequence<step_of(DV)>(P, i).units; all += u; if (i < b) before += u; }
#pragma unroll
  for (int o = 16; o; o >>= 1) { before += __shfl_xor_sync(0xffffffffu, before, o); all += __shfl_xor_sync(0xffffffffu, all, o); }
  if ((threadIdx.x & 31) == 0) { sums[0][threadIdx.x >> 5] = before; sums[1][threadIdx.x >> 5] = all; }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int i = 0; i < QT * DV / 32; i++) { before += sums[0][i]; all += sums[1][i]; }
  const Seq q = sequence<step_of(DV)>(P, b);
  const long long units = q.units, total = all * per, N = ctas_of(ctas, total, (long long)P.S.batch * per), u0 = before * per + hr * units;
  const int i0 = units ? (int)quotient((u0 + 1) * N + total - 1, total) - 1 : 0, i1 = units ? (int)quotient((u0 + units) * N + total - 1, total) - 1 : 0;   // the CTAs of its first and last unit
  grid_wait();                                               // (every thread: what follows this kernel then follows the one ahead as well)
  if (i0 == i1) return;
  const int own = quotient(i0 * total, N) >= u0 ? 0 : 1;     // the first one's piece: its first or its last (the others' pieces are their first)
  const int head = hr / P.row_tiles;
  join_pieces<DV, QT>(P, q, b, head, (hr - head * P.row_tiles) * QT * 8, threadIdx.x >> 5, threadIdx.x & 31, i1 - i0 + 1,
                      [&](int i) { return (const float*)P.part + (size_t)(2 * (i0 + i) + (i == 0 ? own : 0)) * (QT * (NO * 128 + 16)); });
}

}  // namespace kv8
}  // namespace dsk
