// dsk_kv8_tc5.cuh — softmax attention of portions (many query rows to a key head) over the 8-bit cache on the 5th-generation tensor cores.
//
// A CTA has query rows of a key head (its query heads' rows one behind the other, so that all of them share the keys), two tiles of 128 or one (up to 128 rows; heads of 256 entries, whose
// queries, keys and values fill shared memory), and walks the keys that they see in tiles of 128.  Roles: seven or eight warps bring codes from the cache, four the keys' and three or four the
// values', turn them into fp16 (exact) and store them as swizzled operands, so that the cache crosses HBM and L2 as bytes; one thread issues the products, scores into TMEM, weights from TMEM;
// a group of four warps for each tile of rows has the softmax, a thread to a row.  Two tiles: one's products run under the other's softmax, weights lie where the scores were, and a
// tile's next scores wait for the product that reads its weights.  One tile: scores lie in two places in turn, and the next tile's products run under this one's softmax.
// Scales and weights as in dsk_kv8_attn.cuh: key scales on the scores, value scales inside the exponent, fp16 weights of at most 2^kSlack, references kLift below a maximum, as whole numbers.
// The results stay in TMEM; they are scaled again only where a row's maximum is kSlack ahead of the reference of its weights, by the thread that has the row.
// NaN among values: a tile that some row does not see whole goes to the products with zeros in their place, and rows that do see one get it back at the end.
// Bound: the softmax.  Of some 4500 cycles for 256 rows and 128 keys of 192 + 128 entries the weights of one group take 1500 (1024 of the exponentials' pipe), its maxima 500, the products
// 2560 of the tensor pipe, and a group's products and the way there and back stand 1700 behind its weights.  2048 queries behind 3952 tokens, 16 heads of 192 + 128: 137 us (104 GFLOP:
// 760 TFLOP/s; a measured product of matrices 1638), heads of 256: 240 us (167 GFLOP: 695), 3 x 777 queries of 16 heads of 64 over 4 with a window of 512: 27 us.
#pragma once

#include "dsk_kv8_attn.cuh"
#include "dsk_tcprim.cuh"

namespace dsk {
namespace kv8 {

constexpr int kTile = 128, kRowThreads = 512, kSlots = 4;    // keys of a tile; threads of a CTA; tiles whose scales are held

struct Portion {
  Attn A;                                                    // row_tiles: of a CTA's rows
  int shares;                                                // of a row tile's keys (CTAs), joined by join_rows where there are several
};

// TILES: tiles of 128 query rows of a CTA (256 entries: its shared memory and TMEM are full with one)
template <int DK, int DV, int TILES> __host__ __device__ constexpr int k_stages() { return DK == 64 && TILES == 2 ? 3 : DK == 256 ? 1 : 2; }   // (one tile of rows: keys three tiles ahead would bring scales over those that a softmax may still read)
template <int DK, int DV, int TILES> __host__ __device__ constexpr int v_stages() { return DK == 256 || (DK == 192 && TILES == 2) ? 1 : DK == 64 ? 3 : 2; }
template <int DK, int DV, int TILES> __host__ __device__ constexpr int rows_smem() {
  return 1024 + 128 * TILES * DK * 2 + k_stages<DK, DV, TILES>() * kTile * DK * 2 + v_stages<DK, DV, TILES>() * kTile * DV * 2 + kSlots * 3 * 8 * 4 + 256;
}

// Bounded.  (Polls that are given a time to sleep wake some 100 cycles late.)
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, int* status) {
  const long long from = clock64();
  do {
    if (hy::tc_poll(bar, parity)) return true;
  } while (clock64() - from < hy::kTcWaitCycles);
  if (status) atomicOr(status, ST_WAIT);
  return false;
}
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const Cache& C) { return hy::tc_poll(bar, parity) || wait_long(bar, parity, C.status); }
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
__device__ __forceinline__ void tmem_read16(uint32_t addr, uint32_t (&r)[16]) {   // loaded when it returns
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr) : "memory");
}
// two fp32 operations at a time
__device__ __forceinline__ uint64_t both(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void fma2(uint32_t x0, uint32_t x1, uint64_t f, uint64_t a, float& y0, float& y1) {
  asm("{\n\t.reg .b64 x;\n\tmov.b64 x, {%2, %3};\n\tfma.rn.f32x2 x, x, %4, %5;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(y0), "=f"(y1) : "r"(x0), "r"(x1), "l"(f), "l"(a));
}
__device__ __forceinline__ void add2(uint64_t& s, float y0, float y1) {
  asm("{\n\t.reg .b64 y;\n\tmov.b64 y, {%1, %2};\n\tadd.rn.f32x2 %0, %0, y;\n\t}" : "+l"(s) : "f"(y0), "f"(y1));
}
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return r;
}
// Products and commits of one lane of a warp whose lanes all run the same code: descriptors then stay in uniform registers, where a branch to that lane would have them copied there
// for every product
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead) {
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead) {   // A in TMEM
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t lead) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
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
__device__ __forceinline__ Walk walk_of(const Portion& P, int b, int row0, int rows, int share) {
  const Attn& A = P.A;
  Walk w;
  const long long room = (long long)A.S.table_blocks << A.C.shift;
  const int len = max(A.S.first[b], -1);                     // (positions do not wrap)
  w.count = A.S.count ? min(max(A.S.count[b], 0), A.S.rows) : A.S.rows;
  w.first = len - w.count;
  w.i0 = row0 / A.group;
  w.i1 = min((row0 + rows - 1) / A.group, w.count - 1);
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

// Codes to operands, keys or values of all tiles, by WARPS warps: a thread has the c-th 16 entries of every 64 of rows r0, r0 + 8 WARPS, ..  (G of them).  A warp's loads are 64 bytes
// of eight rows, its stores meet no bank twice (neighbouring rows are swizzled to even and odd pieces), and places in shared memory differ by constants.  A tile's codes are
// loaded a tile ahead, with its scales, and the numbers of its blocks two tiles ahead.
template <int D, int G, int WARPS>
__device__ __forceinline__ void bring(const Attn& A, const Walk& w, int b, int h, int which, int warp, int lane, uint32_t ring, uint32_t stage_bytes, int stages, uint32_t full, uint32_t empty,
                                      uint32_t scaled, float* scales, int* nan_seen) {
  constexpr int NB = D / 64;
  const int n = w.end - w.begin, dim = A.C.dim[which], r0 = warp * 8 + (lane >> 2), c0 = lane & 3;
  const uint32_t head = A.C.block * dim, block = A.C.heads * head, place = r0 * 128 + (((c0 * 2) ^ (r0 & 7)) << 4);
  const unsigned char* code = A.C.code[which];
  const int* table = A.S.table + b * A.S.table_pitch;
  const bool scaling = which == 0 && warp == 0;
  auto look = [&](int i) {                                   // lane g < 8: block of keys 16 g .. of a tile (-1: behind the last key, or outside the cache)
    int p = -1;
    if (i < n && lane < 8) {
      const int key = key_of(w, w.begin + i) + 16 * lane;
      if (key < w.len) p = __ldg(table + (key >> A.C.shift));
    }
    return p;
  };
  auto checked = [&](int p, int i) {
    const bool bad = i < n && lane < 8 && (unsigned)p >= (unsigned)A.C.n_blocks;
    if (bad && scaling && key_of(w, w.begin + i) + 16 * lane < w.len) note(A.C, ST_PAGE);
    return bad ? -1 : p;
  };
  float k_scale = 0.f, v_scale = 0.f;
  auto look_scales = [&](int p) {
    if (scaling && p >= 0) {
      const uint64_t slot = (uint64_t)(uint32_t)p * (uint32_t)A.C.heads + h;
      k_scale = __ldg(A.C.scale[0] + slot);
      v_scale = __ldg(A.C.scale[1] + slot);
    }
  };
  uint4 x[G * NB];
  const bool exact = dim == D;
  auto load = [&](int i, int page) {
    const int key0 = key_of(w, w.begin + i);
    if (exact && key0 + kTile <= w.len && __all_sync(0xffffffffu, lane >= 8 || page >= 0)) {   // a whole tile
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int at = min(g * WARPS * 8 + r0, kTile - 1);   // (G x 8 x WARPS rows may be more than a tile has)
        const uint32_t p = __shfl_sync(0xffffffffu, page, at >> 4);
        const unsigned char* from = code + ((uint64_t)p * block + (h * head + ((key0 + at) & (A.C.block - 1)) * D + c0 * 16));
#pragma unroll
        for (int k = 0; k < NB; k++) x[g * NB + k] = __ldg(reinterpret_cast<const uint4*>(from + k * 64));
      }
      return;
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int at = g * WARPS * 8 + r0, row = key0 + at, p = __shfl_sync(0xffffffffu, page, at >> 4);
      const bool there = at < kTile && p >= 0 && row < w.len;
      const unsigned char* from = code + ((uint64_t)(uint32_t)max(p, 0) * block + (h * head + (row & (A.C.block - 1)) * dim + c0 * 16));
#pragma unroll
      for (int k = 0; k < NB; k++) {
        x[g * NB + k] = make_uint4(0, 0, 0, 0);
        if (there && k * 64 + c0 * 16 < dim) x[g * NB + k] = __ldg(reinterpret_cast<const uint4*>(from + k * 64));
      }
    }
  };
  int stage = 0, page = checked(look(0), 0);
  uint32_t turn = 1;
  if (n > 0) load(0, page);
  look_scales(page);
  int next = look(1);
  for (int i = 0; i < n; i++) {
    if (!wait_warp(empty + 8 * stage, turn, A.C)) break;
    if (scaling) {
      if (lane < 8) {
        float* to = scales + (i % kSlots) * 24 + lane;
        const int e = (int)(__float_as_uint(v_scale) >> 23) - 127;
        to[0] = page >= 0 ? k_scale : 0.f;
        to[8] = page >= 0 ? (float)e : 0.f;
        to[16] = page >= 0 ? pow2(-e) : 0.f;
      }
      __syncwarp();
      if (lane == 0) hy::tc_arrive(scaled + 8 * (i % kSlots));
    }
    if (which == 1 && !sees_all(A, w, w.i0, w.i1, key_of(w, w.begin + i))) {   // NaN become zeros
      uint32_t found = 0;
#pragma unroll
      for (int j = 0; j < G * NB; j++) {
        uint32_t* c = reinterpret_cast<uint32_t*>(&x[j]);
#pragma unroll
        for (int u = 0; u < 4; u++) { const uint32_t z = nan_bytes(c[u]); found |= z; c[u] &= ~z; }
      }
      if (found) *nan_seen = 1;
    }
    const uint32_t to = ring + stage * stage_bytes + place, to_other = ring + stage * stage_bytes + (place ^ 16);
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int k = 0; k < NB; k++) {
        const uint4 c = x[g * NB + k];
        uint32_t f[8];
        four_halves(c.x, f[0], f[1]);
        four_halves(c.y, f[2], f[3]);
        four_halves(c.z, f[4], f[5]);
        four_halves(c.w, f[6], f[7]);
        const uint32_t at = k * (kTile * 128) + g * WARPS * 8 * 128;
        if (kTile % (WARPS * 8) == 0 || g * WARPS * 8 + r0 < kTile) { sts128(to + at, f[0], f[1], f[2], f[3]); sts128(to_other + at, f[4], f[5], f[6], f[7]); }
      }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) hy::tc_arrive(full + 8 * stage);
    if (++stage == stages) { stage = 0; turn ^= 1; }
    page = checked(next, i + 1);
    if (i + 1 < n) load(i + 1, page);
    look_scales(page);
    next = look(i + 2);
  }
  __syncwarp();
}

template <int DK, int DV, int TILES>
__global__ void __launch_bounds__(kRowThreads, 1) attend_rows(const __grid_constant__ Portion P) {
  constexpr int KST = k_stages<DK, DV, TILES>(), VST = v_stages<DK, DV, TILES>(), KB = kTile * DK * 2, VB = kTile * DV * 2, ROWS = 128 * TILES, VW = TILES == 2 ? 3 : 4;   // VW: warps that bring values
  extern __shared__ unsigned char raw[];
  __shared__ uint32_t tmem_slot;
  __shared__ int nan_seen;
  const Attn& A = P.A;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gbase = raw + (base - smem_u32(raw));
  const uint32_t qs = base, ks = qs + ROWS * DK * 2, vs = ks + KST * KB, cs = vs + VST * VB, bars = cs + kSlots * 3 * 8 * 4;
  float* scales = reinterpret_cast<float*>(gbase + (cs - base));          // [slot][key scale | exponent of the value scale | its reciprocal, zero: not there][16 keys]
  const uint32_t kfull = bars, kempty = bars + 24, vfull = bars + 48, vempty = bars + 72, sfull = bars + 96, pfull = bars + 112, pvdone = bars + 128, cfull = bars + 144, cdone = bars + 176, flushed = bars + 184, qfull = bars + 192;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int h = blockIdx.x / P.shares, share = blockIdx.x - h * P.shares, b = blockIdx.z, row0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * ROWS;   // late rows, which see most, first
  const Walk w = walk_of(P, b, row0, ROWS, share);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    const long long len = A.S.first[b];
    if (len < 0 || len > (long long)A.S.table_blocks << A.C.shift) note(A.C, ST_RANGE);
  }
  if (w.i0 >= w.count) return;                               // (the whole CTA: none of its rows exists)
  const int n = w.end - w.begin;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; i++) { mbar_init(kfull + 8 * i, 4); mbar_init(kempty + 8 * i, 1); mbar_init(vfull + 8 * i, VW); mbar_init(vempty + 8 * i, 1); }
    for (int i = 0; i < 2; i++) { mbar_init(sfull + 8 * i, 1); mbar_init(pfull + 8 * i, 4); mbar_init(pvdone + 8 * i, 1); }
    for (int i = 0; i < kSlots; i++) mbar_init(cfull + 8 * i, 1);
    mbar_init(cdone, VW);
    mbar_init(qfull, 4 * TILES);
    mbar_init(flushed, 1);
    nan_seen = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int dk = A.C.dim[0], dv = A.C.dim[1];
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot, o_at = tmem + 256;        // columns: scores (then weights) [2][128], results [tile][DV]

  if (warp >= 12) {
    if (warp == 12) {
      const uint32_t lead = hy::tc_elect();
      const uint32_t idesc = (1u << 4) | ((uint32_t)(kTile / 16) << 24);       // fp32 sums, fp16 x fp16, 128 rows
      const uint32_t sdesc = idesc | ((uint32_t)(kTile / 8) << 17), pdesc = idesc | (1u << 16) | ((uint32_t)(DV / 8) << 17);
      auto score = [&](int t, int stage) {                   // one tile of rows: into alternate columns
        const uint64_t a = hy::tc_desc(qs + (TILES == 2 ? t * (kTile * DK * 2) : 0)), k = hy::tc_desc(ks + stage * KB);
#pragma unroll
        for (int g = 0; g < DK / 64; g++)
#pragma unroll
          for (int u = 0; u < 4; u++) mma_ss(tmem + t * 128, a + g * (kTile * 128 >> 4) + 2 * u, k + g * (kTile * 128 >> 4) + 2 * u, sdesc, g > 0 || u > 0, lead);
        commit(sfull + 8 * t, lead);
      };
      bool alive = n > 0 && wait_warp(qfull, 0, A.C) && wait_warp(kfull, 0, A.C);
      if (alive) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        score(0, 0);
        if (TILES == 2) score(1, 0);
        commit(kempty, lead);
      }
      int kst = 0, vst = 0;
      uint32_t kturn = 0, vturn = 0;                         // the stage that was read last, parity of its tile
      for (int i = 0; i < n && alive; i++) {
        const uint64_t v = value_desc(vs + vst * VB);
        const bool more = i + 1 < n;
        if (more && ++kst == KST) { kst = 0; kturn ^= 1; }
        if constexpr (TILES == 1) {                          // the next scores' products run under this tile's softmax, where the weights of the tile ahead were read
          if (more) {
            alive = wait_warp(kfull + 8 * kst, kturn, A.C) && (i == 0 || wait_warp(pvdone, (i - 1) & 1, A.C));
            if (!alive) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            score((i + 1) & 1, kst);
            commit(kempty + 8 * kst, lead);
          }
          alive = wait_warp(vfull + 8 * vst, vturn, A.C) && wait_warp(pfull + 8 * (i & 1), (i >> 1) & 1, A.C);
          if (!alive) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int u = 0; u < kTile / 16; u++) mma_ts(o_at, tmem + (i & 1) * 128 + (u >> 2) * 64 + (u & 3) * 8, v + u * 128, pdesc, i > 0 || u > 0, lead);
          commit(pvdone, lead);
          commit(vempty + 8 * vst, lead);
        } else {
          alive = wait_warp(vfull + 8 * vst, vturn, A.C);
          if (!alive) break;
#pragma unroll
          for (int t = 0; t < 2; t++) {
            if (!alive) continue;
            alive = wait_warp(pfull + 8 * t, i & 1, A.C);
            if (!alive) continue;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int u = 0; u < kTile / 16; u++) mma_ts(o_at + t * 128, tmem + t * 128 + (u >> 2) * 64 + (u & 3) * 8, v + u * 128, pdesc, i > 0 || u > 0, lead);
            commit(pvdone + 8 * t, lead);
            if (t == 1) commit(vempty + 8 * vst, lead);
            if (!more) continue;
            if (t == 0) { alive = wait_warp(kfull + 8 * kst, kturn, A.C); if (!alive) continue; }
            alive = wait_warp(pvdone + 8 * t, i & 1, A.C);   // the weights are read: their columns may have the next scores
            if (!alive) continue;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            score(t, kst);
            if (t == 1) commit(kempty + 8 * kst, lead);
          }
        }
        if (++vst == VST) { vst = 0; vturn ^= 1; }
      }
      commit(flushed, lead);                                 // no product is under way when TMEM is given back
      wait_warp(flushed, 0, A.C);
    }
    __syncwarp();
    if (TILES == 2 && warp > 12) {
      bring<DV, (kTile + 8 * VW - 1) / (8 * VW), VW>(A, w, b, h, 1, warp - 13, lane, vs, VB, VST, vfull, vempty, 0, nullptr, &nan_seen);
      if (lane == 0) hy::tc_arrive(cdone);
    }
  } else if (warp >= 8) {
    bring<DK, kTile / 32, 4>(A, w, b, h, 0, warp - 8, lane, ks, KB, KST, kfull, kempty, cfull, scales, &nan_seen);
  } else if (TILES == 1 && warp >= 4) {
    bring<DV, kTile / (8 * VW), VW>(A, w, b, h, 1, warp - 4, lane, vs, VB, VST, vfull, vempty, 0, nullptr, &nan_seen);
    if (lane == 0) hy::tc_arrive(cdone);
  } else {
    const int t = warp >> 2, quad = warp & 3, row = row0 + threadIdx.x, i_row = row / A.group, pos = w.first + i_row;
    const int r_first = (row0 + t * 128) / A.group, r_last = min((row0 + t * 128 + 127) / A.group, w.i1);   // tokens of the tile's rows
    const uint32_t lanes = (uint32_t)(quad * 32) << 16, s_0 = tmem + t * 128 + lanes, res = o_at + t * 128 + lanes;
    // the thread's query row as fp16, by a power of two of its own (dsk_kv8_attn.cuh), while the first keys are brought: [tile][64 entries][row], 16-byte pieces swizzled
    float row_scale;
    {
      const uint16_t* src = static_cast<const uint16_t*>(A.q) + b * A.pq.batch + (long long)i_row * A.pq.row + (long long)(h * A.group + row - i_row * A.group) * A.pq.head;
      const bool there = i_row < w.count;
      uint4 x[DK / 8];
#pragma unroll
      for (int d = 0; d < DK / 8; d++) {
        x[d] = make_uint4(0, 0, 0, 0);
        if (there && d * 8 < dk) {
          if (A.wide_q) x[d] = __ldg(reinterpret_cast<const uint4*>(src) + d);
          else x[d] = make_uint4(src[8 * d] | (uint32_t)src[8 * d + 1] << 16, src[8 * d + 2] | (uint32_t)src[8 * d + 3] << 16, src[8 * d + 4] | (uint32_t)src[8 * d + 5] << 16,
                                 src[8 * d + 6] | (uint32_t)src[8 * d + 7] << 16);
        }
      }
      uint32_t top = 0;                                      // the largest number's bits, whose order is that of the magnitudes
      const uint32_t inf = A.bf16 ? 0x7f80u : 0x7c00u;
#pragma unroll
      for (int d = 0; d < DK / 8; d++) {
        const uint32_t y[4] = {x[d].x, x[d].y, x[d].z, x[d].w};
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const uint32_t lo = y[u] & 0x7fffu, hi = (y[u] >> 16) & 0x7fffu;
          top = max(top, max(lo < inf ? lo : 0u, hi < inf ? hi : 0u));
        }
      }
      const float most = A.bf16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half((unsigned short)top));
      const int e = most > 0.f ? max(-100, min(120, (int)(__float_as_uint(most) >> 23) - 127 - 10)) : 0;
      const float by = A.scale < 0.f ? -pow2(-e) : pow2(-e);                 // (factors of scores are positive)
      row_scale = pow2(e) * fabsf(A.scale);
      const uint32_t to = qs + t * (kTile * DK * 2) + (threadIdx.x & 127) * 128;
#pragma unroll
      for (int d = 0; d < DK / 8; d++) {
        uint32_t y[4] = {x[d].x, x[d].y, x[d].z, x[d].w};
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const float2 f = A.bf16 ? make_float2(__uint_as_float(y[u] << 16), __uint_as_float(y[u] & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&y[u]));
          y[u] = halves(f.x * by, f.y * by);
        }
        sts128(to + (d >> 3) * (kTile * 128) + (((d & 7) ^ (threadIdx.x & 7)) << 4), y[0], y[1], y[2], y[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) hy::tc_arrive(qfull);
    }
    auto factor = [&](float key_scale) { return fmaxf(row_scale * key_scale, 1.17549435e-38f); };   // (positive: -inf stays what it is)
    float m = kLowest, l = 0.f, limit = -INFINITY;             // limit: where a maximum moves the reference; any does while that is beyond kFar
    bool ok = true;
    // A wait by parity is right while the barrier is in the phase asked for or the one behind it.  With one tile, scores i are issued behind product i - 2 alone: product i - 1 is waited for by
    // whoever reads results of tile i, and ahead of handing over the last weights, without which product n - 1 cannot be through; then the wait for that one is right as well.
    auto product_ahead = [&](int i) {
      if (TILES == 1 && i > 0 && i + 1 == n) ok = wait_warp(pvdone, (i - 1) & 1, A.C) && ok;
    };
    const bool idle = (row0 + warp * 32) / A.group >= w.count;              // none of the warp's rows exists
    for (int i = 0; i < n; i++) {
      const int slot = i % kSlots, key0 = key_of(w, w.begin + i);
      ok = wait_warp(cfull + 8 * slot, (i / kSlots) & 1, A.C);
      const float4* sc = reinterpret_cast<const float4*>(scales + slot * 24);   // key scales of 16 keys each [8], exponents of their value scales [8], reciprocals of those [8] (zero: not there)
      const float4 there[2] = {sc[4], sc[5]};
      const bool masked = there[0].x == 0.f || there[0].y == 0.f || there[0].z == 0.f || there[0].w == 0.f || there[1].x == 0.f || there[1].y == 0.f || there[1].z == 0.f || there[1].w == 0.f ||
                          !sees_all(A, w, r_first, r_last, key0);
      float fs[4], lift[4];
      auto scales_of = [&](int half) {
        const float4 k4 = sc[half], l4 = sc[2 + half];
        fs[0] = factor(k4.x); fs[1] = factor(k4.y); fs[2] = factor(k4.z); fs[3] = factor(k4.w);
        lift[0] = l4.x; lift[1] = l4.y; lift[2] = l4.z; lift[3] = l4.w;
      };
      scales_of(1);
      const uint32_t s_at = TILES == 2 ? s_0 : s_0 + (i & 1) * 128;
      ok = ok && (TILES == 2 ? wait_warp(sfull + 8 * t, i & 1, A.C) : wait_warp(sfull + 8 * (i & 1), (i >> 1) & 1, A.C));
      if (!ok) break;
      if (idle) {                                            // (its rows' results are whatever comes of the scores as weights, and go nowhere)
        product_ahead(i);
        __syncwarp();
        if (lane == 0) hy::tc_arrive(TILES == 2 ? pfull + 8 * t : pfull + 8 * (i & 1));
        continue;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // Half a row of scores in registers at a time, each read once: the reference may lag behind the maximum by kSlack, within fp16's range, so that the first half's weights do not wait for
      // the second half's maximum; where that moves the reference after all, weights that are stored already are scaled again, by a power of two since references are whole numbers: exactly, but
      // for what comes below 2^-14, where fp16 has multiples of 2^-24.
#pragma unroll 1
      for (int half = 1; half >= 0; half--) {
        const int c = half * 64;
        uint32_t x[64];
        tmem_read64(s_at + c, x);
        if (masked) {                                        // keys that the row sees, a bit each: not behind its own, in the window or among the first, in the cache
          const float4 back = half ? there[1] : there[0];
#pragma unroll
          for (int u = 0; u < 64; u += 32) {
            const int j = key0 + c + u, window = A.window > 0 ? pos - A.window + 1 - j : 0;
            uint32_t see = lower_bits(pos + 1 - j) & (~lower_bits(window) | lower_bits(A.keep - j));
            if ((u ? back.z : back.x) == 0.f) see &= 0xffff0000u;
            if ((u ? back.w : back.y) == 0.f) see &= 0xffffu;
#pragma unroll
            for (int k = 0; k < 32; k++) if (!(see >> k & 1)) x[u + k] = 0xff800000u;
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          float y[5];
#pragma unroll
          for (int k = 0; k < 5; k++) y[k] = max3(x[16 * g + 3 * k], x[16 * g + 3 * k + 1], x[16 * g + 3 * k + 2]);
          const float z = max3(__float_as_uint(max3(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]))), __float_as_uint(fmaxf(y[3], y[4])), x[16 * g + 15]);
          top = fmaxf(top, fmaf(z, fs[g], lift[g]));
        }
        if (__any_sync(0xffffffffu, top > limit)) {
          const float c_top = ceilf(top), to = fmaxf(m, fabsf(c_top) > kFar ? c_top : c_top - kLift), by = exp2_fast(m - to);
          m = to;
          l *= by;
          const bool far = fabsf(m) > kFar;
          limit = far ? -INFINITY : m + kSlack;
          if (__any_sync(0xffffffffu, far)) {                // (maxima beyond it under a reference that is not have weights of zero as they are)
#pragma unroll
            for (int g = 0; g < 4; g++) {
#pragma unroll
              for (int k = 0; k < 16; k++) x[16 * g + k] = __float_as_uint(fmaf(__uint_as_float(x[16 * g + k]), fs[g], lift[g]) - lift[g]);
              fs[g] = 1.f;
            }
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");   // what the tile's newer half stored, weights and results, is read back: a load is not behind a store by itself
          if (i > 0) {                                       // (two tiles of rows: the tile's last product was through ahead of these scores)
            if (TILES == 1) {
              ok = wait_warp(pvdone, (i - 1) & 1, A.C);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
#pragma unroll 1
            for (int d = 0; d < DV; d += 16) {
              uint32_t y[16];
              tmem_read16(res + d, y);
#pragma unroll
              for (int k = 0; k < 16; k++) y[k] = __float_as_uint(__uint_as_float(y[k]) * by);
              tmem_store16(res + d, y);
            }
          }
          if (half == 0) {
#pragma unroll 1
            for (int d = 0; d < 32; d += 16) {
              uint32_t y[16];
              tmem_read16(s_at + 64 + d, y);
#pragma unroll
              for (int k = 0; k < 16; k++) { const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&y[k])); y[k] = halves(v.x * by, v.y * by); }   // (fp16 has no factor below 2^-24)
              tmem_store16(s_at + 64 + d, y);
            }
          }
        }
        const float4 b4 = half ? there[1] : there[0];
        const float back[4] = {b4.x, b4.y, b4.z, b4.w};
        uint32_t p[32];                                      // weights of a half lie in the first 32 of its columns
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const uint64_t f = both(fs[g], fs[g]), off = both(lift[g] - m, lift[g] - m);
          uint64_t sum = 0;
#pragma unroll
          for (int k = 0; k < 8; k++) {
            float y0, y1;
            fma2(x[16 * g + 2 * k], x[16 * g + 2 * k + 1], f, off, y0, y1);
            y0 = exp2_fast(y0);
            y1 = exp2_fast(y1);
            add2(sum, y0, y1);
            p[8 * g + k] = halves(y0, y1);
          }
          l = fmaf(__uint_as_float((uint32_t)sum) + __uint_as_float((uint32_t)(sum >> 32)), back[g], l);
        }
        tmem_store32(s_at + c, p);
        if (half) scales_of(0);
      }
      product_ahead(i);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) hy::tc_arrive(TILES == 2 ? pfull + 8 * t : pfull + 8 * (i & 1));
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
            const int page = A.S.table[b * A.S.table_pitch + (j >> A.C.shift)];
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
      float* part = A.part + ((((size_t)b * A.C.heads + h) * gridDim.y + (gridDim.y - 1 - blockIdx.y)) * P.shares + share) * ROWS * (DV + 2) + threadIdx.x;
#pragma unroll
      for (int c = 0; c < DV; c += 16) {
        uint32_t x[16];
        if (n > 0) tmem_read16(res + c, x);
        float f[16];
#pragma unroll
        for (int k = 0; k < 16; k++) f[k] = n == 0 ? 0.f : (lost[c / 32] >> ((c & 31) + k)) & 1 ? NAN : __uint_as_float(x[k]);
        if (P.shares > 1) {                                  // [entry][row]: neighbouring threads side by side
#pragma unroll
          for (int k = 0; k < 16; k++) if (i_row < w.count) part[(c + k) * ROWS] = f[k];
        } else Out::store(A, Seq{w.len, w.count, 0, 0, 0, 0, 0, 0}, b, h, row, c, 16, f, inv);
      }
      if (P.shares > 1 && i_row < w.count) { part[DV * ROWS] = m; part[(DV + 1) * ROWS] = l; }
    }
  }
  __syncthreads();
  if (warp == 12) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Joins the shares of a row tile's keys, eight at a time: a thread has 16 entries of a row
template <int DV, int TILES>
__global__ void __launch_bounds__(128 * TILES) join_rows(const __grid_constant__ Portion P) {
  constexpr int ROWS = 128 * TILES, AT = 8;
  const Attn& A = P.A;
  const int h = blockIdx.x / (DV / 16), d0 = blockIdx.x % (DV / 16) * 16, tile = blockIdx.y, b = blockIdx.z, row = tile * ROWS + threadIdx.x;
  const Walk w = walk_of(P, b, tile * ROWS, ROWS, 0);
  grid_wait();                                               // (every thread: what follows this kernel then follows the one ahead as well)
  if (w.i0 >= w.count || row / A.group >= w.count) return;
  const float* part = A.part + (((size_t)b * A.C.heads + h) * gridDim.y + tile) * P.shares * ROWS * (DV + 2) + threadIdx.x;
  float m = kLowest, l = 0.f, x[16];
#pragma unroll
  for (int k = 0; k < 16; k++) x[k] = 0.f;
  for (int s = 0; s < P.shares; s += AT) {
    float pm[AT], pl[AT], px[AT][16], to = m;
#pragma unroll
    for (int u = 0; u < AT; u++) {
      pm[u] = -INFINITY;
      if (s + u >= P.shares) continue;
      const float* from = part + (size_t)(s + u) * ROWS * (DV + 2);
      pm[u] = from[DV * ROWS];
      pl[u] = from[(DV + 1) * ROWS];
#pragma unroll
      for (int k = 0; k < 16; k++) px[u][k] = from[(d0 + k) * ROWS];
    }
#pragma unroll
    for (int u = 0; u < AT; u++) to = fmaxf(to, pm[u]);
    const float f = exp2_fast(m - to);
    m = to;
    l *= f;
#pragma unroll
    for (int k = 0; k < 16; k++) x[k] *= f;
#pragma unroll
    for (int u = 0; u < AT; u++) {
      if (s + u >= P.shares) break;
      const float g = exp2_fast(pm[u] - m);
      l = fmaf(pl[u], g, l);
#pragma unroll
      for (int k = 0; k < 16; k++) x[k] = fmaf(px[u][k], g, x[k]);
    }
  }
  Out::store(A, Seq{w.len, w.count, 0, 0, 0, 0, 0, 0}, b, h, row, d0, 16, x, l == 0.f ? 0.f : 1.f / l);
}

}  // namespace kv8
}  // namespace dsk
