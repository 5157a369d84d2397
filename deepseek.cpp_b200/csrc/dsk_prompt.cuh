// dsk_prompt.cuh — causal softmax attention of packed prompts on the 5th-generation tensor cores: o_i = sum_j p_ij v_j, p_i = softmax over j of scale q_i k_j, j <= i, in a window or
// among the first tokens.
//
// Query rows of a key head lie token by token, the heads that share it side by side, so that a tile of 128 rows has few tokens and its keys end close behind the rows' own.  A CTA has two
// tiles (one where heads have more than 192 + 128 entries) and walks their keys in tiles of 128; tensor-map copies bring queries, keys and values as swizzled operands, in units of 16 KB that
// are given back as soon as their product is through.  Roles: a warp for the copies of keys and queries, one for the values, one that issues each row tile's products (scores into TMEM, weights
// from TMEM), four softmax warps for each row tile, a thread to a row, one that deals out the work, three that look at values of tiles which some row does not see whole.
// Weights: y = f s - m in one fused operation, f = scale log2(e); the reference m is a whole number that may lag behind the maximum, so that the results in TMEM are scaled again, by
// powers of two, where a maximum has moved far (the thread that has the row does it).  bf16 weights have fp32's range: references lead by 2^40, so that no sum of weights x values exceeds the
// largest value; fp16 weights lie between 2^-24 and 2^14, references 2^7 below the maximum.
// Infinities and NaN among values that a row does not see must not reach it as 0 x inf: in tiles that some row does not see whole they go to the products as zeros, and rows that do see
// one get it back at the end.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "dsk_tmem.cuh"

namespace dsk {
namespace prompt {

constexpr int kThreads = 512, kTile = 128, kUnit = 16384, kMaxBatch = 1024, kHeld = 8, kAhead = 4;   // keys of a tile; bytes of a copied unit; sequences whose tiles a lane of the dealing warp keeps in registers; tiles of keys under way
constexpr int ST_WAIT = 4;                                   // a wait that gave up
constexpr float kLowest = -3e38f;                            // a maximum ahead of the first score (finite: no difference of infinities)
constexpr float kFar = 16777216.f;                           // scores beyond it are rounded ahead of the subtraction: what fma keeps of a product that its reference does not would be exponents

struct Params {
  CUtensorMap q, k, v;                                       // [row][head][entry]: boxes of 64 entries of (heads of a tile, its tokens), (one head, 128 keys), (one head, the keys of a unit)
  const int* starts;                                         // [batch + 1]
  int* status;
  const void* values;
  void* out;
  long long v_row, v_head, o_row, o_head;
  int rows, batch, group, pack, subs, tokens, units;         // pack: heads of a row tile; subs: group / pack; tokens: of a row tile; units: key heads x subs
  int dk, dv, window, keep, wide_o;
  float f;                                                   // scale x log2(e), positive
};

template <int DK, int DV> __host__ __device__ constexpr int tiles() { return DV == 256 ? 1 : 2; }
template <int DK, int DV> __host__ __device__ constexpr int k_units() { return DK == 192 ? 5 : 6; }
template <int DK, int DV> __host__ __device__ constexpr int v_units() { return DK == 192 ? 3 : DK == 64 ? 5 : 4; }
template <int DK, int DV> __host__ __device__ constexpr int smem_bytes() { return 1024 + 128 * tiles<DK, DV>() * DK * 2 + (k_units<DK, DV>() + v_units<DK, DV>()) * kUnit; }

// Bounded, in line: a call would cost what the wait itself does
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* status) {
  bool ok = hy::tc_poll(bar, parity);
  if (!ok) {
    const uint32_t from = clock();
    do ok = hy::tc_poll(bar, parity); while (!ok && (uint32_t)clock() - from < 1u << 31);
    if (!ok && status) atomicOr(status, ST_WAIT);
  }
  return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int entry, int head, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(entry), "r"(head), "r"(row) : "memory");
}
// operand whose rows are the depth, `keys` of them: 64 columns to a swizzled 128-byte row, groups of eight rows 1024 bytes apart, the next 64 columns `keys` rows behind
__device__ __forceinline__ uint64_t value_desc(uint32_t addr, int keys) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(keys * 128 >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
template <bool BF16> __device__ __forceinline__ uint32_t pair(float lo, float hi) {
  if (!BF16) return halves(lo, hi);
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// What a CTA has at a time: row tiles from token `tok` on of a sequence whose rows begin at `row`, for the heads `unit`; len 0: nothing more
struct Item { int row, len, tok, unit; };
// The keys that its rows see, in tiles: the first `kept` ones, then those from `low` on
struct Walk { int t1, low, kept, n; };
__device__ __forceinline__ Walk walk_of(const Params& P, const Item& w, int tokens) {
  Walk k;
  k.t1 = min(w.tok + tokens, w.len);
  k.low = P.window > 0 ? max(0, w.tok + 1 - P.window) / kTile : 0;
  k.kept = P.window > 0 ? min((min(P.keep, k.t1) + kTile - 1) / kTile, k.low) : 0;
  k.n = k.kept + (k.t1 + kTile - 1) / kTile - k.low;
  return k;
}
__device__ __forceinline__ int key_of(const Walk& k, int i) { return (i < k.kept ? i : k.low + i - k.kept) * kTile; }
// whether tokens a .. b see all of a tile of keys; any of it
__device__ __forceinline__ bool sees_all(const Params& P, int a, int b, int key0) {
  return key0 + kTile - 1 <= a && (P.window <= 0 || b - key0 < P.window || key0 + kTile <= P.keep);
}
__device__ __forceinline__ bool sees_some(const Params& P, int a, int b, int key0) {
  return key0 <= b && (P.window <= 0 || a - key0 - kTile + 1 < P.window || key0 < P.keep);
}

// Infinities and NaN among the values that a row sees in tiles where they went to the products as zeros: its results c .. c + 15 become what they make of them
template <bool BF16> __device__ __noinline__ void give_back(const Params& P, const Item& w, const Walk& k, int pos, int head, int c, uint32_t (&x)[16]) {
  for (int i = 0; i < k.n; i++) {
    const int key0 = key_of(k, i);
    if (sees_all(P, w.tok, k.t1 - 1, key0)) continue;
    for (int j = key0; j < min(key0 + kTile, pos + 1); j++) {
      if (P.window > 0 && pos - j >= P.window && j >= P.keep) continue;
      const uint16_t* v = static_cast<const uint16_t*>(P.values) + (long long)(w.row + j) * P.v_row + (long long)head * P.v_head + c;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const uint32_t u = v[e];
        if (BF16 ? (u & 0x7f80u) == 0x7f80u : (u & 0x7c00u) == 0x7c00u) x[e] = __float_as_uint(__uint_as_float(x[e]) + (BF16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((unsigned short)u))));
      }
    }
  }
}

template <int DK, int DV, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) attend_packed(const __grid_constant__ Params P) {
  constexpr int TILES = tiles<DK, DV>(), KU = k_units<DK, DV>(), VU = v_units<DK, DV>(), VK = kUnit / (2 * DV), STEPS = VK / 16, SOFT = 4 * TILES, USERS = SOFT + 7;   // VK: keys of a unit of values
  constexpr float LEAD = BF16 ? 40.f : -7.f, ROOM = BF16 ? -26.f : 14.f;       // a reference is taken LEAD above its maximum, and follows once that is above m + ROOM
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[50];
  __shared__ int4 items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int odd_values;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u, qs = base, ks = qs + 128 * TILES * DK * 2, vs = ks + KU * kUnit, b0 = smem_u32(bars);
  const uint32_t kfull = b0, kempty = b0 + 32, vfull = b0 + 64, vempty = b0 + 104, vok = b0 + 144, vraw = b0 + 184, qfull = b0 + 224, qempty = b0 + 240, sfull = b0 + 256, pfull = b0 + 272,
                 pvdone = b0 + 304, odone = b0 + 320, ifull = b0 + 336, iempty = b0 + 352, flushed = b0 + 368, turns = b0 + 384;   // keys: a barrier for each of kAhead tiles; vraw: where values land that are looked at ahead of their products
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, tokens = TILES * P.tokens;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kAhead; i++) { mbar_init(kfull + 8 * i, 1); mbar_init(kempty + 8 * i, TILES); }
    for (int i = 0; i < 5; i++) { mbar_init(vfull + 8 * i, 1); mbar_init(vempty + 8 * i, TILES); mbar_init(vok + 8 * i, 3); mbar_init(vraw + 8 * i, 1); }
    for (int i = 0; i < 2; i++) {
      mbar_init(qfull + 8 * i, 1); mbar_init(qempty + 8 * i, 1); mbar_init(sfull + 8 * i, 1); mbar_init(pfull + 16 * i, 4); mbar_init(pfull + 16 * i + 8, 4);
      mbar_init(pvdone + 8 * i, 1); mbar_init(odone + 8 * i, 1); mbar_init(ifull + 8 * i, 1); mbar_init(iempty + 8 * i, USERS); mbar_init(flushed + 8 * i, 1); mbar_init(turns + 8 * i, 4);
    }
    odd_values = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot, o_at = tmem + 256;        // columns: scores (then weights) [2][128], results [tile][DV]

  // 512 threads have 128 registers each; a softmax thread holds a row of scores, the others little
  constexpr int MANY = 192, FEW = 64;

  uint32_t turn = 0;                                         // items that this warp has taken
  auto take = [&](Item& w) {                                 // the next item, in every lane
    const uint32_t slot = turn & 1;
    const bool ok = wait_warp(ifull + 8 * slot, (turn >> 1) & 1, P.status);
    const int4 x = items[slot];
    __syncwarp();
    if (lane == 0) hy::tc_arrive(iempty + 8 * slot);
    turn++;
    w = Item{x.x, x.y, x.z, x.w};
    return ok && w.len > 0;
  };

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW));
  if (warp == 8 || warp == 9) {                              // products: of row tile warp - 8 (one row tile: scores, results)
    const int t = warp - 8;
    const uint32_t lead = hy::tc_elect();
    const uint32_t idesc = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (8u << 24);         // fp32 sums of bf16 or fp16, 128 rows
    const uint32_t pdesc = idesc | (1u << 16) | ((uint32_t)(P.dv / 8) << 17);
    const int chunks = (P.dk + 63) / 64, ksteps = P.dk / 16;
    uint32_t kt = 0, kn = 0, vn = 0, vpar[2] = {0, 0}, passed = 0, took = 0;   // tiles of keys behind, places in the rings, parities of values (a bit for each place: as they came, looked at), tiles of this row tile, items that had rows
    int pend = -1;                                           // a unit of values whose product is issued and that is to be given back
    auto keys_there = [&] { return wait_warp(kfull + 8 * (kt % kAhead), (kt / kAhead) & 1, P.status); };
    auto scores = [&](uint32_t to, int n, uint32_t full) {   // of the next tile of keys, of which the rows see the first 16 n
      const uint64_t a = hy::tc_desc(qs + (TILES == 2 ? t * (kTile * DK * 2) : 0));
      const uint32_t sdesc = idesc | (uint32_t)(2 * n) << 17;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
      for (int c = 0; c < DK / 64; c++) {
        if (c >= chunks) break;
        const uint64_t k = hy::tc_desc(ks + (kn + c < KU ? kn + c : kn + c - KU) * kUnit);
#pragma unroll
        for (int u = 0; u < 4; u++) if (4 * c + u < ksteps) mma_ss(to, a + c * (kTile * 128 >> 4) + 2 * u, k + 2 * u, sdesc, c > 0 || u > 0, lead);
      }
      commit(full, lead);
      commit(kempty + 8 * (kt % kAhead), lead);
    };
    auto next_keys = [&] {
      kt++;
      kn += chunks;
      if (kn >= KU) kn -= KU;
    };
    auto values_there = [&](const bool masked) {
      uint32_t at = vn;
#pragma unroll
      for (int u = 0; u < kTile / VK; u++) {
        if (!wait_warp((masked ? vok : vfull) + 8 * at, (masked ? vpar[1] : vpar[0]) >> at & 1, P.status)) return false;
        if (masked) vpar[1] ^= 1u << at; else vpar[0] ^= 1u << at;
        if (++at == VU) at = 0;
      }
      return true;
    };
    auto results = [&](uint32_t weights, uint32_t to, uint32_t full, uint32_t parity, int n, const bool add, uint32_t done) {
#pragma unroll
      for (int u = 0; u < kTile / 16; u++) {
        if (u % 4 == 0) {
          if (!wait_warp(full + (u / 4) * 8, parity, P.status)) return false;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        if (u < n) mma_ts(to, weights + u * 8, value_desc(vs + vn * kUnit, VK) + (u % STEPS) * 128, pdesc, add || u > 0, lead);
        if (u == kTile / 16 - 1) commit(done, lead);
        if (u % STEPS == STEPS - 1) {
          if (TILES == 2 && u == kTile / 16 - 1) pend = vn;  // (given back behind the next scores, which wait for this product and not for that)
          else commit(vempty + 8 * vn, lead);
          if (++vn == VU) vn = 0;
        }
      }
      return true;
    };
    Item w;
    bool alive = true;
    while (alive && take(w)) {
      const Walk k = walk_of(P, w, tokens);
      const int a = w.tok + (TILES == 2 ? t * P.tokens : 0), b = min(a + (TILES == 2 ? P.tokens : tokens), w.len) - 1;
      const bool there = a < w.len;
      bool any = false;
      if (TILES == 2) {
        alive = (!there || wait_warp(qfull + 8 * t, took & 1, P.status)) && keys_there();
        for (int i = 0; i < k.n && alive; i++) {
          const int key0 = key_of(k, i), n = min(8, (b - key0 + 16) / 16);
          const bool mine = there && sees_some(P, a, b, key0), masked = !sees_all(P, w.tok, k.t1 - 1, key0);
          if (mine) {
            if (passed) alive = wait_warp(pvdone + 8 * t, (passed - 1) & 1, P.status);   // the weights are read: their columns may have the next scores
            if (!alive) break;
            scores(tmem + t * 128, n, sfull + 8 * t);
          } else if (lead) hy::tc_arrive(kempty + 8 * (kt % kAhead));
          if (pend >= 0) { commit(vempty + 8 * pend, lead); pend = -1; }
          next_keys();
          if (i + 1 < k.n) alive = keys_there();
          else if (there) commit(qempty + 8 * t, lead);
          alive = alive && values_there(masked);
          if (!alive) break;
          if (mine) {
            alive = results(tmem + t * 128, o_at + t * 128, pfull + 16 * t, passed & 1, n, any, pvdone + 8 * t);
            passed++;
            any = true;
          } else {
#pragma unroll
            for (int u = 0; u < kTile / VK; u++) {
              if (lead) hy::tc_arrive(vempty + 8 * vn);
              if (++vn == VU) vn = 0;
            }
          }
        }
        if (there && alive) { commit(odone + 8 * t, lead); took++; }
        if (pend >= 0) { commit(vempty + 8 * pend, lead); pend = -1; }
      } else if (t == 0) {                                   // scores lie in two places in turn
        alive = wait_warp(qfull, took & 1, P.status);
        for (int i = 0; i < k.n && alive; i++, passed++) {
          const uint32_t s = passed & 1;
          alive = keys_there() && (passed < 2 || wait_warp(pvdone + 8 * s, ((passed >> 1) - 1) & 1, P.status));
          if (!alive) break;
          scores(tmem + s * 128, min(8, (b - key_of(k, i) + 16) / 16), sfull + 8 * s);
          next_keys();
        }
        if (alive) { commit(qempty, lead); took++; }
      } else {
        for (int i = 0; i < k.n && alive; i++, passed++) {
          const uint32_t s = passed & 1;
          const int key0 = key_of(k, i);
          alive = values_there(!sees_all(P, w.tok, k.t1 - 1, key0)) && results(tmem + s * 128, o_at, pfull + 16 * s, (passed >> 1) & 1, min(8, (b - key0 + 16) / 16), i > 0, pvdone + 8 * s);
        }
        if (alive) commit(odone, lead);
      }
    }
    commit(flushed + 8 * t, lead);                           // no product is under way when TMEM is given back
    wait_warp(flushed + 8 * t, 0, P.status);
  } else if (warp == 10 || warp == 11) {                     // copies: keys and queries, values
    Item w;
    const int chunks = (P.dk + 63) / 64, boxes = (P.dv + 63) / 64;
    uint32_t n = 0, par = 0, took[2] = {0, 0}, vpar[2] = {0, 0}, vsent[2] = {0, 0};
    int tile = 0, freed = 0, sent = 0;                       // tiles of keys begun and given back, units sent
    bool alive = true;
    auto keys = [&](const Item& w, int key0, int head) {
      for (int c = 0; c < chunks; c++) {
        while (freed + kAhead <= tile || freed * chunks + KU <= sent) {   // the barrier's last tile, and the unit that lies where this one goes
          alive = wait_warp(kempty + 8 * (freed % kAhead), (freed / kAhead) & 1, P.status);
          if (!alive) return;
          freed++;
        }
        if (lane == 0) {
          if (c == 0) mbar_expect_tx(kfull + 8 * (tile % kAhead), chunks * kUnit);
          copy_box(ks + n * kUnit, &P.k, 64 * c, head, w.row + key0, kfull + 8 * (tile % kAhead));
        }
        sent++;
        if (++n == KU) n = 0;
      }
      tile++;
    };
    if (warp == 10) {
      while (alive && take(w)) {
        const Walk k = walk_of(P, w, tokens);
        const int head = w.unit / P.subs, q_head = head * P.group + (w.unit - head * P.subs) * P.pack;
        keys(w, key_of(k, 0), head);
        for (int t = 0; t < TILES && alive; t++) {
          if (w.tok + t * P.tokens >= w.len) continue;
          alive = wait_warp(qempty + 8 * t, (took[t] & 1) ^ 1, P.status);
          if (!alive) break;
          if (lane == 0) {
            mbar_expect_tx(qfull + 8 * t, chunks * P.tokens * P.pack * 128);
            for (int c = 0; c < chunks; c++) copy_box(qs + t * (kTile * DK * 2) + c * (kTile * 128), &P.q, 64 * c, q_head, w.row + w.tok + t * P.tokens, qfull + 8 * t);
          }
          took[t]++;
        }
        for (int i = 1; i < k.n && alive; i++) keys(w, key_of(k, i), head);
      }
      for (int t = 0; t < TILES; t++) if (took[t]) wait_warp(qfull + 8 * t, (took[t] - 1) & 1, P.status);   // no copy is under way at the end, whatever happened
      for (int s = max(0, tile - kAhead); s < tile; s++) wait_warp(kfull + 8 * (s % kAhead), (s / kAhead) & 1, P.status);
    } else {
      while (alive && take(w)) {
        const Walk k = walk_of(P, w, tokens);
        const int head = w.unit / P.subs;
        for (int i = 0; i < k.n && alive; i++) {
          const int key0 = key_of(k, i);
          const bool masked = !sees_all(P, w.tok, k.t1 - 1, key0);
          const uint32_t full = masked ? vraw : vfull;
          for (int u = 0; u < kTile / VK && alive; u++) {
            alive = wait_warp(vempty + 8 * n, par ^ 1, P.status);
            if (!alive) break;
            if (lane == 0) {
              mbar_expect_tx(full + 8 * n, boxes * VK * 128);
              for (int c = 0; c < boxes; c++) copy_box(vs + n * kUnit + c * (VK * 128), &P.v, 64 * c, head, w.row + key0 + u * VK, full + 8 * n);
            }
            vpar[masked] ^= 1u << n;
            vsent[masked] |= 1u << n;
            if (++n == VU) { n = 0; par ^= 1; }
          }
        }
      }
      for (uint32_t s = 0; s < 2 * VU; s++)                  // no copy is under way at the end, whatever happened
        if (vsent[s & 1] >> (s >> 1) & 1) wait_warp((s & 1 ? vraw : vfull) + 8 * (s >> 1), ~(vpar[s & 1] >> (s >> 1)) & 1, P.status);
    }
  } else if (warp == 15) {                                   // deals out the work: rows with most keys first, so that the short ones fill the gaps
    int held[kHeld];                                         // row tiles of sequences lane, lane + 32, ..
    auto tiles_of = [&](int b) {
      if (b >= P.batch) return 0;
      const int from = min(max(P.starts[b], 0), P.rows), to = min(max(P.starts[b + 1], from), P.rows);
      return (to - from + tokens - 1) / tokens;
    };
    int most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; i++) { held[i] = tiles_of(lane + 32 * i); most = max(most, held[i]); }
    for (int b = lane + 32 * kHeld; b < P.batch; b += 32) most = max(most, tiles_of(b));
    most = __reduce_max_sync(0xffffffffu, most);
    auto from_level = [&](int j) {                           // row tiles that are the j-th or a later one of their sequence
      int n = 0;
#pragma unroll
      for (int i = 0; i < kHeld; i++) n += max(held[i] - j, 0);
      for (int b = lane + 32 * kHeld; b < P.batch; b += 32) n += max(tiles_of(b) - j, 0);
      return __reduce_add_sync(0xffffffffu, n);
    };
    const int all = from_level(0);
    uint32_t par = 0, round = 0;
    for (long long at = blockIdx.x;; at += gridDim.x, round++) {
      int4 item = make_int4(0, 0, 0, 0);
      const int k = (int)(at / P.units);
      if (at < (long long)all * P.units) {
        int lo = 0, hi = most - 1;                           // the level j with from_level(j + 1) <= k < from_level(j)
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (from_level(mid) > k) lo = mid; else hi = mid - 1;
        }
        most = lo + 1;                                       // (later ones lie no higher)
        int rank = k - from_level(lo + 1), b = -1;
        for (int c = 0; b < 0 && c < P.batch; c += 32) {
          bool has = tiles_of(c + lane) > lo;
          const uint32_t mask = __ballot_sync(0xffffffffu, has);
          const uint32_t hit = __ballot_sync(0xffffffffu, has && __popc(mask & ((1u << lane) - 1)) == rank);
          if (hit) b = c + __ffs(hit) - 1;
          rank -= __popc(mask);
        }
        if (b >= 0) {
          const int from = min(max(P.starts[b], 0), P.rows), to = min(max(P.starts[b + 1], from), P.rows);
          item = make_int4(from, to - from, lo * tokens, (int)(at - (long long)k * P.units));
        }
      }
      const uint32_t slot = round & 1;
      if (!wait_warp(iempty + 8 * slot, par ^ 1, P.status)) break;
      if (lane == 0) { items[slot] = item; hy::tc_arrive(ifull + 8 * slot); }
      if (slot) par ^= 1;
      if (item.y <= 0) break;
    }
  } else {                                                   // values of tiles that some row does not see whole: rows behind the sequence, infinities and NaN become zeros
    Item w;
    const int me = threadIdx.x - 12 * 32, boxes = (P.dv + 63) / 64;
    const uint32_t inf = BF16 ? 0x7f807f80u : 0x7c007c00u;
    uint32_t n = 0, par = 0;                                 // par: a bit for each place
    bool alive = true;
    while (alive && take(w)) {
      const Walk k = walk_of(P, w, tokens);
      for (int i = 0; i < k.n && alive; i++) {
        const int key0 = key_of(k, i);
        const bool masked = !sees_all(P, w.tok, k.t1 - 1, key0);
        for (int u = 0; u < kTile / VK && alive; u++) {
          if (masked) {
            alive = wait_warp(vraw + 8 * n, par >> n & 1, P.status);
            par ^= 1u << n;
            const int first = key0 + u * VK;
            bool odd = false;
            for (int p = me; p < boxes * VK * 8; p += 96) {  // 16-byte pieces: eight to a row of 64 columns
              const int row = first + ((p >> 3) & (VK - 1));
              const uint32_t at = vs + n * kUnit + p * 16;
              const uint4 x = lds128(at);
              uint32_t y[4] = {x.x, x.y, x.z, x.w}, z[4], hit = 0;
#pragma unroll
              for (int e = 0; e < 4; e++) { z[e] = row < w.len ? __vcmpeq2(y[e] & inf, inf) : 0xffffffffu; hit |= z[e]; y[e] &= ~z[e]; }
              if (hit) { sts128(at, y[0], y[1], y[2], y[3]); odd |= row < w.len; }
            }
            if (odd) odd_values = 1;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) hy::tc_arrive(vok + 8 * n);
          }
          if (++n == VU) n = 0;
        }
      }
    }
  }
  } else if (warp < SOFT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY));
    const int t = warp >> 2, quad = warp & 3, r = threadIdx.x & 127, tok_of = r / P.pack;       // the thread's row: token tok_of of the tile, head r % pack
    const bool exists = r < P.tokens * P.pack;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16, res = o_at + t * 128 + lanes;
    uint32_t passed = 0, took = 0, gated = 0;                // gated: tiles that both groups have
    Item w;
    bool ok = true;
    while (ok && take(w)) {
      const int a = w.tok + t * P.tokens, b = min(a + P.tokens, w.len) - 1, other = w.tok + (t ^ 1) * P.tokens;
      if (a >= w.len) continue;
      const Walk k = walk_of(P, w, tokens);
      const int pos = exists ? a + tok_of : 0x3fffffff;
      const bool mine = pos < w.len, idle = !__any_sync(0xffffffffu, mine);
      float m = kLowest, l = 0.f, limit = -INFINITY;         // limit: where a maximum moves the reference; any does while that is beyond kFar
      bool any = false;
      for (int i = 0; i < k.n; i++) {
        const int key0 = key_of(k, i);
        if (!sees_some(P, a, b, key0)) continue;
        const uint32_t buf = TILES == 2 ? t : passed & 1, par = TILES == 2 ? passed & 1 : (passed >> 1) & 1, s_at = tmem + buf * 128 + lanes;
        const bool masked = !sees_all(P, a, b, key0);
        // The two groups' exponentials take turns: one's products then run under the other's, where both at a time would wait for the exponentials' pipe and leave the tensor pipe idle
        const bool gate = TILES == 2 && other < w.len && sees_some(P, other, min(other + P.tokens, w.len) - 1, key0);
        const uint32_t turn_of = turns + 8 * t, turn_par = (gated - 1 + t) & 1;
        ok = wait_warp(sfull + 8 * buf, par, P.status);
        if (!ok) break;
        if (idle) {                                          // (its rows' results are whatever comes of the scores as weights, and go nowhere)
          __syncwarp();
          if (lane < 2) hy::tc_arrive(pfull + 16 * buf + 8 * lane);
          if (gate) { if (lane == 0) hy::tc_arrive(turns + 8 * (t ^ 1)); gated++; }
          passed++;
          any = true;
          continue;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const bool go = !gate || gated + t == 0 || hy::tc_poll(turn_of, turn_par);   // (asked ahead of the maxima, which the answer then comes under)
        uint32_t x[128];                                     // the whole row: its weights then lie where the scores were
        tmem_row(s_at, x);
        if (masked) {                                        // keys that the row sees, a bit each: not behind its own, in the window or among the first
#pragma unroll
          for (int u = 0; u < 128; u += 32) {
            const int j = key0 + u;
            uint32_t see = lower_bits(pos + 1 - j);
            if (P.window > 0) see &= ~lower_bits(pos - P.window + 1 - j) | lower_bits(P.keep - j);
#pragma unroll
            for (int e = 0; e < 32; e++) if (!(see >> e & 1)) x[u + e] = 0xff800000u;
          }
        }
        float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 128; e += 8)
#pragma unroll
          for (int g = 0; g < 4; g++) y[g] = max3(__float_as_uint(y[g]), x[e + 2 * g], x[e + 2 * g + 1]);
        const float top = mine ? fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) * P.f : -INFINITY;
        float f = P.f;
        if (__any_sync(0xffffffffu, top > limit)) {
          const float c_top = ceilf(top), to = fmaxf(m, fabsf(c_top) > kFar ? c_top : c_top + LEAD), by = exp2_fast(m - to);
          m = to;
          l *= by;
          const bool far = fabsf(m) > kFar;
          limit = far ? -INFINITY : m + ROOM;
          if (__any_sync(0xffffffffu, far)) {
#pragma unroll
            for (int e = 0; e < 128; e++) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
            f = 1.f;
          }
          if (any) {                                         // (two row tiles: the last product was through ahead of these scores)
            // A wait by parity is right while the barrier is in the phase asked for or the one behind it: these scores waited for the product before the one ahead
            if (TILES == 1) ok = wait_warp(pvdone + 8 * (buf ^ 1), ((passed - 1) >> 1) & 1, P.status);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int d = 0; d < P.dv; d += 16) {
              uint32_t z[16];
              tmem_read16(res + d, z);
#pragma unroll
              for (int e = 0; e < 16; e++) z[e] = __float_as_uint(__uint_as_float(z[e]) * by);
              tmem_store16(res + d, z);
            }
          }
        }
        if (!__all_sync(0xffffffffu, go)) ok = wait_warp(turn_of, turn_par, P.status) && ok;
        const uint64_t f2 = both(f, f), off = both(-m, -m);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int u = 0; u < 4; u++) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            float y0, y1;
            fma2(x[32 * u + 2 * e], x[32 * u + 2 * e + 1], f2, off, y0, y1);
            y0 = exp2_fast(y0);
            y1 = exp2_fast(y1);
            add2(sum[e & 1], y0, y1);
            p[e] = pair<BF16>(y0, y1);
          }
          if (u == 3 && gate) {
            __syncwarp();
            if (lane == 0) hy::tc_arrive(turns + 8 * (t ^ 1));
            gated++;
          }
          tmem_store16(s_at + 16 * u, p);
          if (u & 1) {                                       // a half of the weights: its product starts
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) hy::tc_arrive(pfull + 16 * buf + 8 * (u >> 1));
          }
        }
        l += (__uint_as_float((uint32_t)sum[0]) + __uint_as_float((uint32_t)(sum[0] >> 32))) + (__uint_as_float((uint32_t)sum[1]) + __uint_as_float((uint32_t)(sum[1] >> 32)));
        passed++;
        any = true;
      }
      ok = ok && wait_warp(odone + 8 * (TILES == 2 ? t : 0), took & 1, P.status);
      took++;
      if (!ok || idle) continue;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int odd = odd_values, head = w.unit / P.subs, q_head = head * P.group + (w.unit - head * P.subs) * P.pack + r - tok_of * P.pack;
      uint16_t* to = static_cast<uint16_t*>(P.out) + (long long)(w.row + pos) * P.o_row + (long long)q_head * P.o_head;
#pragma unroll 1
      for (int c = 0; c < P.dv; c += 16) {
        uint32_t x[16];
        tmem_read16(res + c, x);
        if (!mine) continue;
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = __float_as_uint(__uint_as_float(x[e]) * inv);
        if (odd) give_back<BF16>(P, w, k, pos, head, c, x);
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = pair<BF16>(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        if (P.wide_o) {
          uint4* at = reinterpret_cast<uint4*>(to + c);
          at[0] = make_uint4(y[0], y[1], y[2], y[3]);
          at[1] = make_uint4(y[4], y[5], y[6], y[7]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) { to[c + 2 * e] = (uint16_t)y[e]; to[c + 2 * e + 1] = (uint16_t)(y[e] >> 16); }
        }
      }
    }
  }
  __syncthreads();
  if (warp == 8) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

}  // namespace prompt
}  // namespace dsk
