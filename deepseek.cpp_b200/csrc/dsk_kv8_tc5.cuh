// dsk_kv8_tc5.cuh — softmax attention of portions (many query rows to a key head) over the 8-bit cache on the 5th-generation tensor cores, keys up to 192 entries, values up to 128.
//
// A CTA has 256 query rows of a key head (its query heads' rows one behind the other, so that all of them share the keys), two tiles of 128, and walks the keys that they see in tiles
// of 128.  Roles: four warps bring codes from the cache, turn them into fp16 (exact) and store them as swizzled operands, so that the cache crosses HBM and L2 as bytes; one thread
// issues the products, scores into TMEM, weights from TMEM; two groups of four warps have the softmax, a thread to a row, each for its own tile, so that one tile's products run under the
// other one's softmax.  Scales and weights as in dsk_kv8_attn.cuh: key scales on the scores, value scales inside the exponent, fp16 weights of at most 2^kSlack.
// The results stay in TMEM; they are scaled again only where a row's maximum has moved by more than 2^kSlack, by the thread that has the row.  Weights lie where the scores were:
// a tile's next scores wait for the product that reads its weights.
// NaN among values: a tile that some row does not see whole goes to the products with zeros in their place, and rows that do see one get it back at the end.
#pragma once

#include "dsk_kv8_attn.cuh"
#include "dsk_tcprim.cuh"

namespace dsk {
namespace kv8 {

constexpr int kTile = 128, kRows = 256, kRowThreads = 512, kSlots = 4;       // keys of a tile; rows and threads of a CTA; tiles whose scales are held

struct Portion {
  Attn A;                                                    // row_tiles: of kRows rows
  int shares;                                                // of a row tile's keys (CTAs), joined by join_rows where there are several
};

template <int DK, int DV> __host__ __device__ constexpr int k_stages() { return DK == 64 ? 3 : 2; }
template <int DK, int DV> __host__ __device__ constexpr int v_stages() { return DK == 192 ? 1 : DK == 64 ? 3 : 2; }
template <int DK, int DV> __host__ __device__ constexpr int rows_smem() {
  return 1024 + kRows * DK * 2 + k_stages<DK, DV>() * kTile * DK * 2 + v_stages<DK, DV>() * kTile * DV * 2 + kSlots * 3 * 8 * 4 + 256;
}

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const Cache& C) {   // bounded; every lane of a warp gets the same answer
  if (hy::tc_poll(bar, parity)) return true;
  const long long from = clock64();
  do {
    if (hy::tc_poll(bar, parity)) return true;
  } while (clock64() - from < hy::kTcWaitCycles);
  note(C, ST_WAIT);
  return false;
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, const Cache& C) { return __all_sync(0xffffffffu, wait_bar(bar, parity, C)); }
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_read64(uint32_t addr, uint32_t (&r)[64]) {   // loaded when it returns
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_read32(uint32_t addr, uint32_t (&r)[32]) {   // loaded when it returns
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_read16(uint32_t addr, uint32_t (&r)[16]) {   // loaded when it returns
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// operand whose rows are the depth: 64 columns to a swizzled 128-byte row, groups of eight rows 1024 bytes apart, the next 64 columns kTile rows behind
__device__ __forceinline__ uint64_t value_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(kTile * 128 >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// The keys of a CTA's rows, tile by tile: the first `kept` tiles, then those from `low` on; a share's are begin .. end - 1
struct Walk { int len, count, first, kept, low, begin, end, i0, i1; };   // first: position of the sequence's first query; i0, i1: tokens of the CTA's first and last row
__device__ __forceinline__ Walk walk_of(const Portion& P, int b, int row0, int share) {
  const Attn& A = P.A;
  Walk w;
  const long long room = (long long)A.S.table_blocks << A.shift;
  const int len = A.S.first[b];
  w.count = A.S.count ? min(max(A.S.count[b], 0), A.S.rows) : A.S.rows;
  w.first = len - w.count;
  w.i0 = row0 / A.group;
  w.i1 = min((row0 + kRows - 1) / A.group, w.count - 1);
  w.len = (int)min((long long)max(w.first + w.i1 + 1, 0), room);                 // (what the CTA's last row sees)
  const long long lo = (long long)w.first + w.i0 + 1 - A.window;
  w.low = A.window > 0 && lo > 0 ? (int)min(lo, (long long)w.len) / kTile : 0;
  w.kept = A.window > 0 ? min((min(A.keep, w.len) + kTile - 1) / kTile, w.low) : 0;
  const int n = w.kept + (w.len + kTile - 1) / kTile - w.low;
  w.begin = (int)((long long)n * share / P.shares);
  w.end = (int)((long long)n * (share + 1) / P.shares);
  return w;
}
__device__ __forceinline__ int key_of(const Walk& w, int tile) { return (tile < w.kept ? tile : w.low + tile - w.kept) * kTile; }
// whether rows i0 .. i1 see all of a tile
__device__ __forceinline__ bool sees_all(const Attn& A, const Walk& w, int i0, int i1, int key0) {
  return key0 + kTile - 1 <= w.first + i0 && (A.window <= 0 || w.first + i1 - key0 < A.window || key0 + kTile <= A.keep);
}

template <int DK, int DV>
__global__ void __launch_bounds__(kRowThreads, 1) attend_rows(const __grid_constant__ Portion P) {
  constexpr int KST = k_stages<DK, DV>(), VST = v_stages<DK, DV>(), KB = kTile * DK * 2, VB = kTile * DV * 2;
  extern __shared__ unsigned char raw[];
  __shared__ uint32_t tmem_slot;
  __shared__ int nan_seen;
  const Attn& A = P.A;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gbase = raw + (base - smem_u32(raw));
  const uint32_t qs = base, ks = qs + kRows * DK * 2, vs = ks + KST * KB, cs = vs + VST * VB, bars = cs + kSlots * 3 * 8 * 4;
  float* scales = reinterpret_cast<float*>(gbase + (cs - base));          // [slot][key scale | exponent of the value scale | its reciprocal, zero: not there][16 keys]
  const uint32_t kfull = bars, kempty = bars + 24, vfull = bars + 48, vempty = bars + 72, sfull = bars + 96, pfull = bars + 112, pvdone = bars + 128, cfull = bars + 144, cdone = bars + 176, flushed = bars + 184;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x / P.shares, share = blockIdx.x - h * P.shares, b = blockIdx.z, row0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * kRows;   // late rows, which see most, first
  const Walk w = walk_of(P, b, row0, share);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    const long long len = A.S.first[b];
    if (len < 0 || len > (long long)A.S.table_blocks << A.shift) note(A.C, ST_RANGE);
  }
  if (w.i0 >= w.count) return;                               // (the whole CTA: none of its rows exists)
  const int n = w.end - w.begin;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; i++) { mbar_init(kfull + 8 * i, 4); mbar_init(kempty + 8 * i, 1); mbar_init(vfull + 8 * i, 4); mbar_init(vempty + 8 * i, 1); }
    for (int i = 0; i < 2; i++) { mbar_init(sfull + 8 * i, 1); mbar_init(pfull + 8 * i, 4); mbar_init(pvdone + 8 * i, 1); }
    for (int i = 0; i < kSlots; i++) mbar_init(cfull + 8 * i, 1);
    mbar_init(cdone, 4);
    mbar_init(flushed, 1);
    nan_seen = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int dk = A.C.dim[0], dv = A.C.dim[1];
  if (dk < DK || dv < DV)                                    // entries behind the last one stay zero
    for (int i = threadIdx.x; i < (KST * KB + VST * VB) / 16; i += kRowThreads) sts128(ks + i * 16, 0, 0, 0, 0);
  // query rows as fp16, two threads to a row, each by its own power of two (dsk_kv8_attn.cuh)
  float row_scale = 0.f;                                     // of the row that this thread has in the softmax
  {
    const int row = threadIdx.x >> 1, half = threadIdx.x & 1, i = (row0 + row) / A.group;
    const uint16_t* src = static_cast<const uint16_t*>(A.q) + b * A.pq.batch + (long long)i * A.pq.row + (long long)(h * A.group + row0 + row - i * A.group) * A.pq.head;
    const bool there = i < w.count;
    float top = 0.f;
    auto eight = [&](int d, uint32_t (&x)[4]) {
      x[0] = x[1] = x[2] = x[3] = 0;
      if (there && d < dk) {
        if (A.wide_q) { const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + d)); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
        else
#pragma unroll
          for (int u = 0; u < 4; u++) x[u] = src[d + 2 * u] | (uint32_t)src[d + 2 * u + 1] << 16;
      }
    };
    auto pair = [&](uint32_t x) { return A.bf16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&x)); };
    for (int d = half * 8; d < DK; d += 16) {
      uint32_t x[4];
      eight(d, x);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const float2 f = pair(x[u]);
        const float a = fabsf(f.x), c = fabsf(f.y);
        top = fmaxf(top, fmaxf(a < INFINITY ? a : 0.f, c < INFINITY ? c : 0.f));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const int e = top > 0.f ? max(-100, min(100, (int)(__float_as_uint(top) >> 23) - 127 - 10)) : 0;
    const float by = A.scale < 0.f ? -pow2(-e) : pow2(-e);
    for (int d = half * 8; d < DK; d += 16) {
      uint32_t x[4];
      eight(d, x);
#pragma unroll
      for (int u = 0; u < 4; u++) { const float2 f = pair(x[u]); x[u] = halves(f.x * by, f.y * by); }
      const int tile = row >> 7, rr = row & 127;             // [tile][64 entries][row], 16-byte pieces swizzled
      sts128(qs + tile * (kTile * DK * 2) + (d >> 6) * (kTile * 128) + rr * 128 + ((((d & 63) >> 3) ^ (rr & 7)) << 4), x[0], x[1], x[2], x[3]);
    }
    // thread t of the softmax has row t: its factor comes from threads 2 t, 2 t + 1 (through the scales' memory, which nobody uses yet)
    __syncthreads();
    float* f = reinterpret_cast<float*>(gbase + (vs - base));               // (the first values come behind the barrier below)
    if (half == 0) f[row] = pow2(e) * fabsf(A.scale);
    __syncthreads();
    if (threadIdx.x < kRows) row_scale = f[threadIdx.x];
    __syncthreads();
    if (dv < DV && half == 0) f[row] = 0.f;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot, o_at = tmem + 256;        // columns: scores (then weights) [2][128], results [2][128]

  if (warp >= 12) {
    if (warp == 12 && hy::tc_elect()) {
      const uint32_t idesc = (1u << 4) | ((uint32_t)(kTile / 16) << 24);       // fp32 sums, fp16 x fp16, 128 rows
      const uint32_t sdesc = idesc | ((uint32_t)(kTile / 8) << 17), pdesc = idesc | (1u << 16) | ((uint32_t)(DV / 8) << 17);
      auto score = [&](int t, int stage) {
        const uint64_t a = hy::tc_desc(qs + t * (kTile * DK * 2)), k = hy::tc_desc(ks + stage * KB);
#pragma unroll
        for (int g = 0; g < DK / 64; g++)
#pragma unroll
          for (int u = 0; u < 4; u++) hy::tc_mma(tmem + t * 128, a + g * (kTile * 128 >> 4) + 2 * u, k + g * (kTile * 128 >> 4) + 2 * u, sdesc, g > 0 || u > 0);
        hy::tc_commit(sfull + 8 * t);
      };
      bool alive = n > 0 && wait_bar(kfull, 0, A.C);
      if (alive) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        score(0, 0);
        score(1, 0);
        hy::tc_commit(kempty);
      }
      int kst = 0, vst = 0;
      uint32_t kturn = 0, vturn = 0;                         // the stage that was read last, parity of its tile
      for (int i = 0; i < n && alive; i++) {
        alive = wait_bar(vfull + 8 * vst, vturn, A.C);
        if (!alive) break;
        const uint64_t v = value_desc(vs + vst * VB);
        const bool more = i + 1 < n;
        if (more && ++kst == KST) { kst = 0; kturn ^= 1; }
        for (int t = 0; t < 2 && alive; t++) {
          alive = wait_bar(pfull + 8 * t, i & 1, A.C);
          if (!alive) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int u = 0; u < kTile / 16; u++) hy::tc_mma_ta(o_at + t * 128, tmem + t * 128 + (u >> 2) * 64 + (u & 3) * 8, v + u * 128, pdesc, i > 0 || u > 0);
          hy::tc_commit(pvdone + 8 * t);
          if (t == 1) hy::tc_commit(vempty + 8 * vst);
          if (!more) continue;
          if (t == 0) { alive = wait_bar(kfull + 8 * kst, kturn, A.C); if (!alive) break; }
          alive = wait_bar(pvdone + 8 * t, i & 1, A.C);      // the weights are read: their columns may have the next scores
          if (!alive) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          score(t, kst);
          if (t == 1) hy::tc_commit(kempty + 8 * kst);
        }
        if (++vst == VST) { vst = 0; vturn ^= 1; }
      }
      hy::tc_commit(flushed);                                // no product is under way when TMEM is given back
      wait_bar(flushed, 0, A.C);
    }
    __syncwarp();
  } else if (warp >= 8) {
    // codes to operands: 16-byte pieces tid, tid + 128, .. of a tile's rows, keys and values in turn, the next piece's load under way
    const int tid = threadIdx.x - 256;
    const uint32_t head_k = A.C.block * dk, head_v = A.C.block * dv, block_k = A.C.heads * head_k, block_v = A.C.heads * head_v;
    int page = 0, next_page = -1;                            // lane g < 8: block of keys 16 g .. of the tile
    auto look = [&](int i) {                                 // (-1: behind the last key)
      int p = -1;
      if (i < n && lane < 8) {
        const int key = key_of(w, w.begin + i) + 16 * lane;
        if (key < w.len) { p = __ldg(A.S.table + b * A.S.table_pitch + (key >> A.shift)); if ((unsigned)p >= (unsigned)A.C.n_blocks) { if (tid < 32) note(A.C, ST_PAGE); p = -1; } }
      }
      return p;
    };
    uint4 kx[DK / 16], vx[DV / 16];
    auto load = [&](auto& x, int per, const unsigned char* code, uint32_t head, uint32_t block, int dim, int key0) {
      int row = tid / per, col = tid - row * per;
      const int dr = 128 / per, dc = 128 - dr * per;
#pragma unroll
      for (int j = 0; j < (int)(sizeof(x) / sizeof(uint4)); j++) {
        if (j >= per) break;
        const int p = __shfl_sync(0xffffffffu, page, row >> 4);
        x[j] = make_uint4(0, 0, 0, 0);
        if (p >= 0 && key0 + row < w.len) x[j] = __ldg(reinterpret_cast<const uint4*>(code + ((uint64_t)(uint32_t)p * block + (h * head + ((key0 + row) & (A.C.block - 1)) * dim + col * 16))));
        row += dr; col += dc;
        if (col >= per) { col -= per; row++; }
      }
    };
    auto store = [&](const auto& x, int per, uint32_t to, bool clean) {
      int row = tid / per, col = tid - row * per;
      const int dr = 128 / per, dc = 128 - dr * per;
      uint32_t found = 0;
#pragma unroll
      for (int j = 0; j < (int)(sizeof(x) / sizeof(uint4)); j++) {
        if (j >= per) break;
        uint32_t c[4] = {x[j].x, x[j].y, x[j].z, x[j].w}, f[8];
        if (clean)
#pragma unroll
          for (int u = 0; u < 4; u++) { const uint32_t z = nan_bytes(c[u]); found |= z; c[u] &= ~z; }
#pragma unroll
        for (int u = 0; u < 4; u++) four_halves(c[u], f[2 * u], f[2 * u + 1]);
        const uint32_t at = to + (col >> 2) * (kTile * 128) + row * 128, p0 = ((col & 3) * 2) ^ (row & 7);
        // two 16-byte pieces; lanes of odd 64-entry blocks begin with the second one: eight lanes never meet a bank twice
        if ((col >> 2) & 1) { sts128(at + ((p0 ^ 1) << 4), f[4], f[5], f[6], f[7]); sts128(at + (p0 << 4), f[0], f[1], f[2], f[3]); }
        else { sts128(at + (p0 << 4), f[0], f[1], f[2], f[3]); sts128(at + ((p0 ^ 1) << 4), f[4], f[5], f[6], f[7]); }
        row += dr; col += dc;
        if (col >= per) { col -= per; row++; }
      }
      return found;
    };
    const int pk = dk / 16, pv = dv / 16;
    int kst = 0, vst = 0;
    uint32_t kturn = 1, vturn = 1;
    bool alive = true;
    next_page = look(0);
    page = next_page;
    if (n > 0) load(kx, pk, A.C.code[0], head_k, block_k, dk, key_of(w, w.begin));
    for (int i = 0; i < n && alive; i++) {
      const int key0 = key_of(w, w.begin + i);
      next_page = look(i + 1);
      float k_scale = 0.f, v_scale = 0.f;
      if (warp == 8 && lane < 8 && page >= 0) {
        const uint64_t slot = (uint64_t)(uint32_t)page * (uint32_t)A.C.heads + h;
        k_scale = __ldg(A.C.scale[0] + slot);
        v_scale = __ldg(A.C.scale[1] + slot);
      }
      load(vx, pv, A.C.code[1], head_v, block_v, dv, key0);
      alive = wait_warp(kempty + 8 * kst, kturn, A.C);
      if (!alive) break;
      if (warp == 8) {
        if (lane < 8) {
          float* to = scales + (i % kSlots) * 24 + lane;
          const int e = (int)(__float_as_uint(v_scale) >> 23) - 127;
          to[0] = k_scale;
          to[8] = page >= 0 ? (float)e : 0.f;
          to[16] = page >= 0 ? pow2(-e) : 0.f;
        }
        __syncwarp();
        if (lane == 0) hy::tc_arrive(cfull + 8 * (i % kSlots));
      }
      store(kx, pk, ks + kst * KB, false);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) hy::tc_arrive(kfull + 8 * kst);
      if (++kst == KST) { kst = 0; kturn ^= 1; }
      page = next_page;
      if (i + 1 < n) load(kx, pk, A.C.code[0], head_k, block_k, dk, key_of(w, w.begin + i + 1));
      alive = wait_warp(vempty + 8 * vst, vturn, A.C);
      if (!alive) break;
      if (store(vx, pv, vs + vst * VB, !sees_all(A, w, w.i0, w.i1, key0))) nan_seen = 1;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) hy::tc_arrive(vfull + 8 * vst);
      if (++vst == VST) { vst = 0; vturn ^= 1; }
    }
    __syncwarp();
    if (lane == 0) hy::tc_arrive(cdone);
  } else {
    const int t = warp >> 2, quad = warp & 3, row = row0 + threadIdx.x, i_row = row / A.group, pos = w.first + i_row;
    const int r_first = (row0 + t * 128) / A.group, r_last = min((row0 + t * 128 + 127) / A.group, w.i1);   // tokens of the tile's rows
    const uint32_t lanes = (uint32_t)(quad * 32) << 16, s_at = tmem + t * 128 + lanes, res = o_at + t * 128 + lanes;
    float m = -1e30f, l = 0.f;
    bool ok = true;
    for (int i = 0; i < n; i++) {
      const int slot = i % kSlots, key0 = key_of(w, w.begin + i);
      ok = wait_warp(cfull + 8 * slot, (i / kSlots) & 1, A.C) && wait_warp(sfull + 8 * t, i & 1, A.C);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float* sc = scales + slot * 24;
      bool gone = false;
#pragma unroll
      for (int g = 0; g < 8; g++) gone |= sc[16 + g] == 0.f;
      const bool masked = gone || !sees_all(A, w, r_first, r_last, key0);
      // half a row of scores in registers at a time: both halves for the maximum, the second one stays, the first one is read again
      float s[64], top = -INFINITY;
      auto half = [&](int c) {
        uint32_t x[64];
        tmem_read64(s_at + c, x);
#pragma unroll
        for (int k = 0; k < 64; k++) s[k] = __uint_as_float(x[k]);
        if (masked) {
#pragma unroll
          for (int k = 0; k < 64; k++) {
            const int j = key0 + c + k;
            if (sc[16 + (c + k) / 16] == 0.f || j > pos || (A.window > 0 && pos - j >= A.window && j >= A.keep)) s[k] = -INFINITY;
          }
        }
      };
      auto highest = [&](int c) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
          float x = s[16 * g];
#pragma unroll
          for (int k = 1; k < 16; k++) x = fmaxf(x, s[16 * g + k]);
          top = fmaxf(top, fmaf(x, fmaxf(row_scale * sc[c / 16 + g], 1.17549435e-38f), sc[8 + c / 16 + g]));
        }
      };
      half(0);
      highest(0);
      half(64);
      highest(64);
      if (__any_sync(0xffffffffu, top > m + kSlack)) {
        const float to = fmaxf(m, top), by = exp2_fast(m - to);
        m = to;
        l *= by;
        if (i > 0) {                                         // (the tile's last product was through ahead of these scores)
#pragma unroll 1
          for (int c = 0; c < DV; c += 16) {
            uint32_t x[16];
            tmem_read16(res + c, x);
#pragma unroll
            for (int k = 0; k < 16; k++) x[k] = __float_as_uint(__uint_as_float(x[k]) * by);
            tmem_store16(res + c, x);
          }
        }
      }
      auto weigh = [&](int c) {                              // weights of a half lie in the first 32 of its columns
        uint32_t x[32];
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const float f = fmaxf(row_scale * sc[c / 16 + g], 1.17549435e-38f), off = sc[8 + c / 16 + g] - m;
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const float p0 = exp2_fast(fmaf(s[16 * g + 2 * k], f, off)), p1 = exp2_fast(fmaf(s[16 * g + 2 * k + 1], f, off));
            sum += p0 + p1;
            x[8 * g + k] = halves(p0, p1);
          }
          l = fmaf(sum, sc[16 + c / 16 + g], l);
        }
        tmem_store32(s_at + c, x);
      };
      weigh(64);
      half(0);
      weigh(0);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) hy::tc_arrive(pfull + 8 * t);
    }
    ok = ok && wait_warp(cdone, 0, A.C) && (n == 0 || wait_warp(pvdone + 8 * t, (n - 1) & 1, A.C));
    if (ok) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint32_t lost[DV / 32] = {};                           // entries of this row that see a NaN
      if (nan_seen && i_row < w.count) {
        for (int i = 0; i < n; i++) {
          const int key0 = key_of(w, w.begin + i);
          if (sees_all(A, w, w.i0, w.i1, key0)) continue;
          for (int j = key0; j < min(key0 + kTile, min(w.len, pos + 1)); j++) {
            if (A.window > 0 && pos - j >= A.window && j >= A.keep) continue;
            const int page = A.S.table[b * A.S.table_pitch + (j >> A.shift)];
            if ((unsigned)page >= (unsigned)A.C.n_blocks) continue;
            const uint32_t* code = reinterpret_cast<const uint32_t*>(A.C.code[1] + (((size_t)page * A.C.heads + h) * A.C.block + (j & (A.C.block - 1))) * dv);
            for (int d = 0; d < dv / 4; d++) {
              const uint32_t z = nan_bytes(code[d]), bits = (z & 1) | (z >> 7 & 2) | (z >> 14 & 4) | (z >> 21 & 8);
#pragma unroll
              for (int u = 0; u < DV / 32; u++) if (u == d >> 3) lost[u] |= bits << (4 * (d & 7));
            }
          }
        }
      }
      const float inv = P.shares > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      float* part = A.part + ((((size_t)b * A.C.heads + h) * gridDim.y + (gridDim.y - 1 - blockIdx.y)) * P.shares + share) * kRows * (DV + 2);
#pragma unroll
      for (int c = 0; c < DV; c += 32) {
        uint32_t x[32];
        if (n > 0) tmem_read32(res + c, x);
        float f[32];
#pragma unroll
        for (int k = 0; k < 32; k++) f[k] = n == 0 ? 0.f : (lost[c / 32] >> k) & 1 ? NAN : __uint_as_float(x[k]);
        if (P.shares > 1) {                                  // [entry][row]: neighbouring threads side by side
#pragma unroll
          for (int k = 0; k < 32; k++) part[(c + k) * kRows + threadIdx.x] = f[k];
        } else {
          Out::store(A, Seq{w.len, w.count, 0, 0, 0, 0, 0, 0}, b, h, row, c, 16, f, inv);
          Out::store(A, Seq{w.len, w.count, 0, 0, 0, 0, 0, 0}, b, h, row, c + 16, 16, f + 16, inv);
        }
      }
      if (P.shares > 1) { part[DV * kRows + threadIdx.x] = m; part[(DV + 1) * kRows + threadIdx.x] = l; }
    }
  }
  __syncthreads();
  if (warp == 12) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Joins the shares of a row tile's keys: a thread has 16 entries of a row
template <int DV>
__global__ void __launch_bounds__(kRows) join_rows(const __grid_constant__ Portion P) {
  grid_wait();
  const Attn& A = P.A;
  const int h = blockIdx.x / (DV / 16), d0 = blockIdx.x % (DV / 16) * 16, tile = blockIdx.y, b = blockIdx.z, row = tile * kRows + threadIdx.x;
  const Walk w = walk_of(P, b, tile * kRows, 0);
  if (w.i0 >= w.count || row / A.group >= w.count) return;
  const float* part = A.part + (((size_t)b * A.C.heads + h) * gridDim.y + tile) * P.shares * kRows * (DV + 2);
  float m = -1e30f, l = 0.f, x[16];
#pragma unroll
  for (int k = 0; k < 16; k++) x[k] = 0.f;
  for (int s = 0; s < P.shares; s++) {
    const float* from = part + (size_t)s * kRows * (DV + 2) + threadIdx.x;
    const float pm = from[DV * kRows], pl = from[(DV + 1) * kRows], to = fmaxf(m, pm), f = exp2_fast(m - to), g = exp2_fast(pm - to);
    m = to;
    l = l * f + pl * g;
#pragma unroll
    for (int k = 0; k < 16; k++) x[k] = x[k] * f + from[(d0 + k) * kRows] * g;
  }
  Out::store(A, Seq{w.len, w.count, 0, 0, 0, 0, 0, 0}, b, h, row, d0, 16, x, l == 0.f ? 0.f : 1.f / l);
}

}  // namespace kv8
}  // namespace dsk
