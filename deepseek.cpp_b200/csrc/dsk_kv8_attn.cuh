// dsk_kv8_attn.cuh — softmax attention of decoded tokens and drafts over the 8-bit cache (dsk_kv8.cuh).
//
// The rows of a key head are its query heads' queries, `group` heads x `rows` tokens; a tile of 16 (two tiles: 32) meets the keys in steps of 16 on mma.sync, fp16 operands
// and fp32 sums.  An E4M3 code is exact in fp16, so keys and values go from their codes to operands by a conversion alone; a query row is divided by a power of two that
// puts its largest entry near 2^10 (what that leaves below fp16's range is 2^-24 of the row).  The scales are applied around the products: the key block's to the scores, and the value block's
// inside the softmax, w_j = 2^(t_j - m) with t_j = score_j + log2(value scale), so that a weight with its scale is one fp16 number of at most 2^kSlack and the sum takes w_j / (value scale).
// Rounding: the weights to fp16, 2^-11 of each; queries in fp16 or bf16 are exact.
// Work: the steps of all sequences, key heads and row tiles lie in one line that the CTAs share out evenly (four steps, 64 keys, to a unit), whatever the lengths; a CTA that has a
// whole (sequence, head, row tile) stores it, pieces are joined by `join`.  Every warp has every fourth step, with stages of its own that cp.async fills: no barrier but where
// a piece ends, and the copies run on across pieces.
// Bound: bytes of the cache.  Fragments come from shared memory as whole 16-byte pieces, entries and keys permuted alike on both sides of a product: a quarter warp's lanes (two
// keys x four pieces) are keys j and j + 4, whose rows lie 16 banks apart.
#pragma once

#include "dsk_kv8.cuh"

namespace dsk {
namespace kv8 {

constexpr int kStep = 16, kWarps = 4, kUnit = kStep * kWarps, kThreads = 32 * kWarps, kMaxBatch = 1024;
constexpr float kSlack = 8.f;                                // the reference of a row's weights follows its maximum once that is 2^8 ahead

struct Attn {
  Cache C;
  Rows S;                                                    // first: tokens of a sequence in the cache, its queries the last ones
  const void* q;
  void* out;
  Pitch pq, po;
  int heads, group, row_tiles, bf16, wide_q, wide_o, window, keep;
  float scale;                                               // times log2(e)
  long long* ends;                                           // workspace: [batch + 1] first units of the sequences (a head's row tile), and pieces
  float* part;
};

// What a sequence has: visible steps are the first `kept` ones and those from `low` on
struct Seq { int len, count, kept, low, steps, units; };
__device__ __forceinline__ Seq sequence(const Attn& P, int b) {
  Seq q;
  const long long room = (long long)P.S.table_blocks * P.C.block;
  const int len = P.S.first[b];
  q.count = P.S.count ? min(max(P.S.count[b], 0), P.S.rows) : P.S.rows;
  q.len = (int)min((long long)max(len, 0), room);
  const long long first = (long long)len - q.count + 1 - P.window;
  q.low = P.window > 0 && first > 0 ? (int)min(first, (long long)q.len) / kStep : 0;
  q.kept = P.window > 0 ? min((min(P.keep, q.len) + kStep - 1) / kStep, q.low) : 0;
  q.steps = q.kept + (q.len + kStep - 1) / kStep - q.low;
  q.units = q.count ? max(1, (q.steps + kWarps - 1) / kWarps) : 0;
  return q;
}

template <int DK, int DV, int MT> __host__ __device__ constexpr int stages() {   // as many as two CTAs of an SM have room for
  return DK == 64 ? 6 : DK == 128 ? (MT == 1 ? 4 : 3) : DK == 192 ? (MT == 1 ? 3 : 2) : 2;
}
template <int DK, int DV> __host__ __device__ constexpr int stage_bytes() { return kStep * (DK + 16 + DV + 32) + 16; }
template <int DK, int DV, int MT> __host__ __device__ constexpr int attn_smem() {
  return kWarps * stages<DK, DV, MT>() * stage_bytes<DK, DV>() + MT * 16 * (2 * DK + 16) + 2 * MT * DV / 8 * 4 * 128 + (2 * kWarps + 1) * MT * 16 * 4;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
__device__ __forceinline__ float exp2_fast(float x) {        // 2 ulp, results below 2^-126 are zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// E4M3 pairs: NaN as zero, and where the NaN are as ones
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {   // 0xff where a byte is NaN
  return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

// A place in the line of units
struct Place {
  Seq q;
  int b, hr, unit;
  __device__ __forceinline__ void find(const Attn& P, const long long* ends, long long x, int per) {   // per: heads x row tiles
    int lo = 0, hi = P.S.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (ends[mid] * per <= x) lo = mid; else hi = mid - 1;
    }
    b = lo;
    q = sequence(P, b);
    const long long in = x - ends[b] * per;
    hr = (int)(in / q.units);
    unit = (int)(in - (long long)hr * q.units);
  }
  __device__ __forceinline__ void next(const Attn& P, int per) {
    if (++unit < q.units) return;
    unit = 0;
    if (++hr < per) return;
    hr = 0;
    do {
      if (++b >= P.S.batch) return;
      q = sequence(P, b);
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

// DK, DV: entries of keys and values, rounded up; MT: tiles of 16 rows
template <int DK, int DV, int MT>
__global__ void __launch_bounds__(kThreads) attend_tokens(const Attn P) {
  constexpr int NST = stages<DK, DV, MT>(), KS = DK + 16, VS = DV + 32, SB = stage_bytes<DK, DV>(), QS = 2 * DK + 16, NT = DV / 8, VCH = DV >= 128 ? 16 : 8, HF = DV / (8 * VCH);
  constexpr bool QREG = MT == 1 && DK <= 128;
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ long long warp_sums[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, B = P.S.batch;
  unsigned char* q_raw = raw + kWarps * NST * SB;
  float* turn = reinterpret_cast<float*>(q_raw + MT * 16 * QS);          // [2][accumulators][lane]
  float* row_m = turn + 2 * MT * NT * 4 * 32;                            // [warp][row]
  float* row_l = row_m + kWarps * MT * 16;
  float* row_q = row_l + kWarps * MT * 16;                               // factor of a row's scores
  long long* ends = reinterpret_cast<long long*>(raw + ((attn_smem<DK, DV, MT>() + 7) & ~7));
  const uint32_t stage0 = smem_u32(raw) + warp * NST * SB, q0 = smem_u32(q_raw);
  grid_release();
  // line of units: running sums over the sequences
  for (int i = threadIdx.x; i < NST * SB * kWarps / 16; i += kThreads) reinterpret_cast<uint4*>(raw)[i] = make_uint4(0, 0, 0, 0);   // (entries behind the last one stay zero)
  long long run = 0;
  for (int b0 = 0; b0 < B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const long long own = b < B ? sequence(P, b).units : 0;
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
  const int per = P.C.heads * P.row_tiles;
  const long long total = run * per, N = min((long long)gridDim.x, total);
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < B; b += kThreads) {
      P.ends[b] = ends[b];
      const long long len = P.S.first[b];
      if (len < 0 || len > (long long)P.S.table_blocks * P.C.block) note(P.C, ST_RANGE);
    }
    if (threadIdx.x == 0) P.ends[B] = run;
  }
  if ((long long)blockIdx.x >= N) return;
  const long long x0 = blockIdx.x * total / N, x1 = (blockIdx.x + 1) * total / N;
  __syncthreads();
  const int dk = P.C.dim[0], dv = P.C.dim[1], dk16 = dk / 16, dv16 = dv / 16;
  const size_t block_k = (size_t)P.C.block * dk, block_v = (size_t)P.C.block * dv;

  // copies: a step of this warp to a unit, from a block whose number was looked up a unit ahead
  Place at;                                                  // of the next copies
  at.find(P, ends, x0, per);
  long long x = x0;
  int page = -1, key = 0;
  auto look = [&]() {
    page = -1;
    const int s = at.unit * kWarps + warp;
    if (x < x1 && s < at.q.steps) {
      key = (s < at.q.kept ? s : at.q.low + s - at.q.kept) * kStep;
      page = __ldg(P.S.table + at.b * P.S.table_pitch + key / P.C.block);
    }
  };
  auto fetch = [&](int stage) {
    const int s = at.unit * kWarps + warp;
    if (x < x1 && s < at.q.steps) {
      const bool ok = (unsigned)page < (unsigned)P.C.n_blocks;
      if (!ok && lane == 0) note(P.C, ST_PAGE);
      const size_t slot = ok ? (size_t)page * P.C.heads + at.hr / P.row_tiles : 0;
      const int there = ok ? at.q.len - key : 0, row0 = key % P.C.block;     // (what is behind the last key comes as zeros)
      const unsigned char* k = P.C.code[0] + slot * block_k + row0 * dk;
      const unsigned char* v = P.C.code[1] + slot * block_v + row0 * dv;
      const uint32_t to = stage0 + stage * SB;
      for (int i = lane; i < dk; i += 32) { const int row = i / dk16; copy16(to + row * KS + (i - row * dk16) * 16, row < there ? k + i * 16 : k, row < there ? 16 : 0); }
      for (int i = lane; i < dv; i += 32) { const int row = i / dv16; copy16(to + kStep * KS + row * VS + (i - row * dv16) * 16, row < there ? v + i * 16 : v, row < there ? 16 : 0); }
      if (lane < 2) copy4(to + kStep * (KS + VS) + lane * 4, P.C.scale[lane] + slot, ok ? 4 : 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (x < x1) { at.next(P, per); x++; }
    look();
  };
  look();
#pragma unroll 1
  for (int i = 0; i < NST - 1; i++) fetch(i);

  float o[MT][NT][4], m[MT][2], l[MT][2];
  uint32_t qf[QREG ? DK / 16 : 1][4];
  Place pl;
  pl.find(P, ends, x0, per);
  int begun = pl.unit, stage = 0;                            // the piece's first unit
  bool fresh = true;
#pragma unroll 1
  for (long long y = x0; y < x1; y++) {
    const Seq q = pl.q;
    const int head = pl.hr / P.row_tiles, row0 = (pl.hr - head * P.row_tiles) * MT * 16;
    if (fresh) {                                             // query rows as fp16, each by its own power of two
      __syncthreads();
      for (int row = warp; row < MT * 16; row += kWarps) {
        const int i = (row0 + row) / P.group;
        const uint16_t* src = static_cast<const uint16_t*>(P.q) + pl.b * P.pq.batch + i * P.pq.row + (long long)(head * P.group + row0 + row - i * P.group) * P.pq.head;
        float v[DK / 32], top = 0.f;
#pragma unroll
        for (int k = 0; k < DK / 64; k++)
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const int d = k * 64 + lane * 2 + u;
            float f = 0.f;
            if (i < q.count && d < dk) f = P.bf16 ? __bfloat162float(__ushort_as_bfloat16(src[d])) : __half2float(__ushort_as_half(src[d]));
            v[2 * k + u] = f;
            const float a = fabsf(f);
            top = fmaxf(top, a < INFINITY ? a : 0.f);
          }
        top = warp_max(top);
        const int e = top > 0.f ? max(-100, min(100, (int)(__float_as_uint(top) >> 23) - 127 - 10)) : 0;
        const float by = pow2(-e);
#pragma unroll
        for (int k = 0; k < DK / 64; k++) *reinterpret_cast<uint32_t*>(q_raw + row * QS + (k * 64 + lane * 2) * 2) = halves(v[2 * k] * by, v[2 * k + 1] * by);
        if (lane == 0) row_q[row] = pow2(e) * P.scale;
      }
      __syncthreads();
      if constexpr (QREG) {
#pragma unroll
        for (int g = 0; g < DK / 64; g++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint4 a = lds128(q0 + r * QS + (g * 64 + 16 * c + 8 * h) * 2), b = lds128(q0 + (r + 8) * QS + (g * 64 + 16 * c + 8 * h) * 2);
            uint32_t* f = qf[g * 4 + 2 * h];
            f[0] = a.x; f[1] = b.x; f[2] = a.y; f[3] = b.y;
            f = qf[g * 4 + 2 * h + 1];
            f[0] = a.z; f[1] = b.z; f[2] = a.w; f[3] = b.w;
          }
      }
#pragma unroll
      for (int t = 0; t < MT; t++) {
        m[t][0] = m[t][1] = -1e30f;
        l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int k = 0; k < NT; k++)
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
      const int key0 = (step < q.kept ? step : q.low + step - q.kept) * kStep;
      const float ks = __uint_as_float(lds32(from + kStep * (KS + VS))), vs = __uint_as_float(lds32(from + kStep * (KS + VS) + 4));
      const float lift = (float)((int)(__float_as_uint(vs) >> 23) - 127), back = vs > 0.f ? 1.f / vs : 0.f;
      float s[MT][2][4];
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int u = 0; u < 4; u++) s[t][0][u] = s[t][1][u] = 0.f;
      const uint32_t krow = from + ((r >> 1) + 4 * (r & 1)) * KS + c * 16;
#pragma unroll
      for (int g = 0; g < DK / 64; g++) {
        const uint4 k0 = lds128(krow + g * 64), k1 = lds128(krow + 8 * KS + g * 64);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t a[MT][2][4];
          if constexpr (QREG) {
#pragma unroll
            for (int u = 0; u < 4; u++) { a[0][0][u] = qf[g * 4 + 2 * h][u]; a[0][1][u] = qf[g * 4 + 2 * h + 1][u]; }
          } else {
#pragma unroll
            for (int t = 0; t < MT; t++) {
              const uint4 x = lds128(q0 + (t * 16 + r) * QS + (g * 64 + 16 * c + 8 * h) * 2), y = lds128(q0 + (t * 16 + r + 8) * QS + (g * 64 + 16 * c + 8 * h) * 2);
              a[t][0][0] = x.x; a[t][0][1] = y.x; a[t][0][2] = x.y; a[t][0][3] = y.y;
              a[t][1][0] = x.z; a[t][1][1] = y.z; a[t][1][2] = x.w; a[t][1][3] = y.w;
            }
          }
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t b0 = two_halves(w0[2 * h + e]), b1 = two_halves(w0[2 * h + e] >> 16), b2 = two_halves(w1[2 * h + e]), b3 = two_halves(w1[2 * h + e] >> 16);
#pragma unroll
            for (int t = 0; t < MT; t++) { mma16(s[t][0], a[t][e], b0, b1); mma16(s[t][1], a[t][e], b2, b3); }
          }
        }
      }
      // a step that every row sees needs no mask
      const int last = P.S.first[pl.b] - 1, first = last + 1 - q.count;    // positions of the last and first query
      const bool masked = key0 + kStep - 1 > first || (P.window > 0 && last - key0 >= P.window && key0 + kStep > P.keep) || vs == 0.f;
      uint32_t pf[MT][4], seen[MT] = {};                     // weights as fp16; keys that this lane's rows see: a bit to a score
#pragma unroll
      for (int t = 0; t < MT; t++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float f = row_q[t * 16 + r + 8 * h] * ks;
#pragma unroll
          for (int g = 0; g < 2; g++)
#pragma unroll
            for (int e = 0; e < 2; e++) s[t][g][2 * h + e] = fmaf(s[t][g][2 * h + e], f, lift);
          if (masked) {
            const int pos = first + (row0 + t * 16 + r + 8 * h) / P.group;
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const int j = key0 + 8 * g + c + 4 * e;
                const bool ok = vs != 0.f && j < q.len && j <= pos && (P.window <= 0 || pos - j < P.window || j < P.keep);
                if (ok) seen[t] |= 1u << (g * 4 + 2 * h + e); else s[t][g][2 * h + e] = -INFINITY;
              }
          }
        }
        float mx[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          mx[h] = fmaxf(fmaxf(s[t][0][2 * h], s[t][0][2 * h + 1]), fmaxf(s[t][1][2 * h], s[t][1][2 * h + 1]));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[t][0] + kSlack || mx[1] > m[t][1] + kSlack)) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const float to = fmaxf(m[t][h], mx[h]), f = exp2_fast(m[t][h] - to);
            m[t][h] = to;
            l[t][h] *= f;
#pragma unroll
            for (int k = 0; k < NT; k++) { o[t][k][2 * h] *= f; o[t][k][2 * h + 1] *= f; }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float sum = 0.f;
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const float p0 = exp2_fast(s[t][g][2 * h] - m[t][h]), p1 = exp2_fast(s[t][g][2 * h + 1] - m[t][h]);
            sum += p0 + p1;
            pf[t][2 * g + h] = halves(p0, p1);
          }
          l[t][h] = fmaf(sum, back, l[t][h]);
        }
      }
      const uint32_t vrow = from + kStep * KS + c * VS + r * VCH;
      auto values = [&](int hf, int key, uint32_t (&w)[VCH / 4]) {
        if constexpr (VCH == 16) { const uint4 x = lds128(vrow + key * VS + hf * 128); w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; }
        else { const uint2 x = lds64(vrow + key * VS); w[0] = x.x; w[1] = x.y; }
      };
      bool nan = false;
      if (masked) {                                          // a NaN among values that some row does not see must not reach that row, whose weight for it is zero
#pragma unroll
        for (int hf = 0; hf < HF; hf++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            uint32_t w[VCH / 4];
            values(hf, (k & 1) * 4 + (k >> 1) * 8, w);
#pragma unroll
            for (int u = 0; u < VCH / 4; u++) nan |= nan_bytes(w[u]) != 0;
          }
        nan = __any_sync(0xffffffffu, nan);
      }
#pragma unroll
      for (int hf = 0; hf < HF; hf++) {
        uint32_t w[4][VCH / 4];
        values(hf, 0, w[0]); values(hf, 4, w[1]); values(hf, 8, w[2]); values(hf, 12, w[3]);
        if (nan) {                                           // counts of the NaN that a row sees, entry by entry, then numbers alone
#pragma unroll 1
          for (int u = 0; u < VCH; u++) {
            uint32_t b[2];
#pragma unroll
            for (int g = 0; g < 2; g++) {
              uint32_t n0 = 0, n1 = 0;
#pragma unroll
              for (int k = 0; k < VCH / 4; k++) if (k == u >> 2) { n0 = nan_bytes(w[2 * g][k]); n1 = nan_bytes(w[2 * g + 1][k]); }
              b[g] = ((n0 >> (8 * (u & 3))) & 1 ? 0x3c00u : 0u) | ((n1 >> (8 * (u & 3))) & 1 ? 0x3c000000u : 0u);
            }
#pragma unroll
            for (int t = 0; t < MT; t++) {
              uint32_t a[4];
#pragma unroll
              for (int g = 0; g < 2; g++)
#pragma unroll
                for (int h = 0; h < 2; h++) a[2 * g + h] = ((seen[t] >> (g * 4 + 2 * h)) & 1 ? 0x3c00u : 0u) | ((seen[t] >> (g * 4 + 2 * h + 1)) & 1 ? 0x3c000000u : 0u);
              float d[4] = {0.f, 0.f, 0.f, 0.f};
              mma16(d, a, b[0], b[1]);
#pragma unroll
              for (int k = 0; k < VCH; k++)
                if (k == u)
#pragma unroll
                  for (int e = 0; e < 4; e++) if (d[e] > 0.f) o[t][hf * VCH + k][e] = NAN;
            }
          }
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int u = 0; u < VCH / 4; u++) w[k][u] &= ~nan_bytes(w[k][u]);
        }
#pragma unroll
        for (int u = 0; u < VCH / 4; u++) {
          const uint32_t lo0 = __byte_perm(w[0][u], w[1][u], 0x5140), hi0 = __byte_perm(w[0][u], w[1][u], 0x7362);
          const uint32_t lo1 = __byte_perm(w[2][u], w[3][u], 0x5140), hi1 = __byte_perm(w[2][u], w[3][u], 0x7362);
          const uint32_t b[4][2] = {{two_halves(lo0), two_halves(lo1)}, {two_halves(lo0 >> 16), two_halves(lo1 >> 16)}, {two_halves(hi0), two_halves(hi1)}, {two_halves(hi0 >> 16), two_halves(hi1 >> 16)}};
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int t = 0; t < MT; t++) mma16(o[t][hf * VCH + u * 4 + e], pf[t], b[e][0], b[e][1]);
        }
      }
    }
    __syncwarp();                                            // the stage is read
    if (++stage == NST) stage = 0;
    // where the piece ends: the warps' sums in one
    const bool whole_end = pl.unit + 1 == q.units;
    if (whole_end || y + 1 == x1) {
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          l[t][h] += __shfl_xor_sync(0xffffffffu, l[t][h], 1);
          l[t][h] += __shfl_xor_sync(0xffffffffu, l[t][h], 2);
          if (c == 0) { row_m[warp * MT * 16 + t * 16 + r + 8 * h] = m[t][h]; row_l[warp * MT * 16 + t * 16 + r + 8 * h] = l[t][h]; }
        }
      __syncthreads();
      float top[MT][2], sum[MT][2];
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int row = t * 16 + r + 8 * h;
          top[t][h] = row_m[row];
#pragma unroll
          for (int w = 1; w < kWarps; w++) top[t][h] = fmaxf(top[t][h], row_m[w * MT * 16 + row]);
          sum[t][h] = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; w++) sum[t][h] += row_l[w * MT * 16 + row] * exp2_fast(row_m[w * MT * 16 + row] - top[t][h]);
          const float f = exp2_fast(m[t][h] - top[t][h]);
#pragma unroll
          for (int k = 0; k < NT; k++) { o[t][k][2 * h] *= f; o[t][k][2 * h + 1] *= f; }
        }
      float* mine = turn + (warp & 1) * MT * NT * 128 + lane;
      auto put = [&]() {
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int k = 0; k < NT; k++)
#pragma unroll
            for (int u = 0; u < 4; u++) mine[((t * NT + k) * 4 + u) * 32] = o[t][k][u];
      };
      auto add = [&](const float* from) {
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int k = 0; k < NT; k++)
#pragma unroll
            for (int u = 0; u < 4; u++) o[t][k][u] += from[((t * NT + k) * 4 + u) * 32];
      };
      if (warp >= 2) put();
      __syncthreads();
      if (warp < 2) add(mine);
      if (warp == 1) put();
      __syncthreads();
      if (warp == 0) {
        add(turn + MT * NT * 128 + lane);
        if (begun == 0 && whole_end) {
#pragma unroll
          for (int t = 0; t < MT; t++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int row = row0 + t * 16 + r + 8 * h;
              const float inv = sum[t][h] == 0.f ? 0.f : 1.f / sum[t][h];        // (a row that sees nothing: zeros)
#pragma unroll
              for (int hf = 0; hf < HF; hf++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  float x[16];
#pragma unroll
                  for (int k = 0; k < VCH; k++) x[k] = o[t][hf * VCH + k][2 * h + e];
                  Out::store(P, q, pl.b, head, row, hf * 128 + (2 * c + e) * VCH, VCH, x, inv);
                }
            }
        } else {                                             // a piece: [accumulator][lane], then maxima and sums of the rows
          float* to = P.part + (size_t)(2 * blockIdx.x + (y + 1 - x0 == pl.unit - begun + 1 ? 0 : 1)) * (MT * (NT * 128 + 32));
#pragma unroll
          for (int t = 0; t < MT; t++) {
#pragma unroll
            for (int k = 0; k < NT; k++)
#pragma unroll
              for (int u = 0; u < 4; u++) to[((t * NT + k) * 4 + u) * 32 + lane] = o[t][k][u];
            if (c == 0)
#pragma unroll
              for (int h = 0; h < 2; h++) {
                to[MT * NT * 128 + t * 16 + r + 8 * h] = top[t][h];
                to[MT * NT * 128 + MT * 16 + t * 16 + r + 8 * h] = sum[t][h];
              }
          }
        }
      }
      fresh = true;
    }
    pl.next(P, per);
    if (fresh) begun = pl.unit;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Joins the pieces of a (sequence, head, row tile) that several CTAs of attend_tokens had: a warp has eight entries of every lane's row
template <int DV, int MT>
__global__ void __launch_bounds__(MT * DV / 16 * 32) join(const Attn P, int ctas) {
  constexpr int NT = DV / 8, VCH = DV >= 128 ? 16 : 8;
  grid_wait();
  const int b = blockIdx.y, hr = blockIdx.x, per = gridDim.x;
  const long long total = P.ends[P.S.batch] * per, units = P.ends[b + 1] - P.ends[b];
  if (units == 0) return;
  const long long N = min((long long)ctas, total), u0 = P.ends[b] * per + hr * units;
  const int i0 = (int)(((u0 + 1) * N + total - 1) / total) - 1, i1 = (int)(((u0 + units) * N + total - 1) / total) - 1;   // the CTAs of its first and last unit
  if (i0 == i1) return;
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  int w = threadIdx.x >> 5;
  const int e = w & 1, h = (w >> 1) & 1;
  w >>= 2;
  const int k0 = (w % (NT / 8)) * 8, t = w / (NT / 8), row = t * 16 + r + 8 * h;
  float x[8], m = -1e30f, l = 0.f;
#pragma unroll
  for (int k = 0; k < 8; k++) x[k] = 0.f;
  for (int i = i0; i <= i1; i += 4) {
    float pm[4], pl[4], px[4][8];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if (i + u > i1) { pm[u] = -INFINITY; continue; }
      const float* from = P.part + (size_t)(2 * (i + u) + ((i + u) * total / N >= u0 ? 0 : 1)) * (MT * (NT * 128 + 32));
      pm[u] = from[MT * NT * 128 + row];
      pl[u] = from[MT * NT * 128 + MT * 16 + row];
#pragma unroll
      for (int k = 0; k < 8; k++) px[u][k] = from[((t * NT + k0 + k) * 4 + 2 * h + e) * 32 + lane];
    }
    const float to = fmaxf(m, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]))), f = exp2_fast(m - to);
    m = to;
    l *= f;
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] *= f;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if (i + u > i1) break;
      const float g = exp2_fast(pm[u] - m);
      l = fmaf(pl[u], g, l);
#pragma unroll
      for (int k = 0; k < 8; k++) x[k] = fmaf(px[u][k], g, x[k]);
    }
  }
  const int head = hr / P.row_tiles, row0 = (hr - head * P.row_tiles) * MT * 16;
  const int hf = k0 / VCH;
  float y[16];
#pragma unroll
  for (int k = 0; k < 8; k++) y[k] = x[k];
  Out::store(P, sequence(P, b), b, head, row0 + row, hf * 128 + (2 * c + e) * VCH + k0 % VCH, 8, y, l == 0.f ? 0.f : 1.f / l);
}

}  // namespace kv8
}  // namespace dsk
