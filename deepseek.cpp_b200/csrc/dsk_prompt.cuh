// dsk_prompt.cuh — causal softmax attention of packed prompts on the 5th-generation tensor cores: o_i = sum_j p_ij v_j, p_i = softmax over j of scale q_i k_j, j <= i, in a window or
// among the first tokens.
//
// Query rows of a key head lie token by token, the heads that share it side by side, so that a tile of 128 rows has few tokens and its keys end close behind the rows' own.  A CTA has two row
// tiles (one where heads have more than 192 + 128 entries) and walks their keys in tiles of 64; tensor-map copies bring queries, keys and values as swizzled operands into rings whose places are
// given back as soon as their products are through.  Roles: a warp for the copies of keys and queries, one for those of values; for each row tile one that issues products of scores, one that issues
// products with the values (scores lie in TMEM, weights where the scores were) and four for the softmax, a thread to a row; one that deals out the work, one that looks at values of tiles which
// some row does not see whole.  A row tile has scores in two places, so that the products and the way there and back (1400 cycles a tile) come under the softmax of the tile ahead.
// Weights: y = f s - m in one fused operation, f = scale log2(e); the reference m is a maximum, moved by a power of two, that may lag behind, so that the results in TMEM are scaled
// again where a maximum has moved far (the thread that has the row does it).  A weight that is the row's largest when its reference is taken is that power of two, which its rounding leaves as it is: a row
// that sees one key has its value, bit for bit (with references that are whole numbers it was off by half a step).  bf16 weights have fp32's range: references lead by 2^40, so that no sum of weights x values
// exceeds the largest value; fp16 weights lie between 2^-24 and 2^14, references 2^7 below the maximum.  Sums are of the weights ahead of their rounding, which is off by half a step of the type at most.
// Infinities and NaN among values that a row does not see must not reach it as 0 x inf: in tiles that some row does not see whole they go to the products as zeros, and rows that do see
// one get it back at the end.
// Few rows: both row tiles of a CTA have the same rows, each every second tile of their keys (joint; the second one's results are added in the reference of both, from its half of TMEM, at the end).
// Work: pieces are dealt out with the longest walks first; CTAs take over pieces of CTAs that have not started (clusterlaunchcontrol), so that nothing but starts is needed to balance them.
// Short prompts: a piece of one tile runs through the code of every role once, and what does not fit the instruction cache is fetched each time (39 % of its lines, a softmax of one tile 4500 cycles
// where it has 1350 by itself).  So the code that pieces run through is kept small: walks are worked out by the warp that deals, one form of each product, one place that counts levels, waits that
// note in a register that they gave up (222 prompts of 60 tokens, 8 heads over 8: 43 us where it was 60; 64 prompts of 1 to 200: 26, was 31).
// Bound: between tensor pipe and softmax.  Of 1505 cycles for 256 rows and 64 keys of 128 + 128 entries the tensor pipe has 1280 (products of 64 keys read their operands from shared memory in 48 cycles
// for 32 of work; tiles of 128 keys, whose products are whole, leave one place for scores: 1860 for as many keys), the exponentials' pipe 1024.  16384 tokens of 16 heads over 4, 128 + 128: 957 us
// one call behind another (1.15 PFLOP/s; a measured product of matrices 1.41 so), 828 us in a few of them (1.33, of 1.68), at 1.65 GHz: the power limit has both.  32 heads of 192 + 128, 8 prompts of up to
// 5001 tokens: 872 and 752 us (0.94, 1.09), 2000 cycles; 256 + 256: 107 and 94 us (0.75, 0.85), 2155 cycles for 128 rows; 64 + 64, windowed: 141 and 151 us, 1835 cycles.
// Taken back: four softmax warps more that share the columns of a row (1300 us where it was 1080), shares of the exponentials as polynomials (850 to 870 where it was 820), maxima only
// where the sum of a tile's weights asks for them (910), sums of rounded weights (937; the error against 64 bits is 0.0021 in bf16, the plain form's 0.0016).
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "dsk_tmem.cuh"

namespace dsk {
namespace prompt {

constexpr int kThreads = 512, kRows = 128, kTile = 64;       // rows of a row tile, keys of a tile
constexpr int kMaxBatch = 1024, kHeld = 8, kEarly = 8;       // sequences; those whose rows a lane of the dealing warp keeps in registers; tiles ahead of the end at which more work is asked for
constexpr int ST_WAIT = 4;                                   // a wait that gave up
constexpr float kLowest = -3e38f;                            // a maximum ahead of the first score (finite: no difference of infinities)
constexpr float kFar = 16777216.f;                           // scores beyond it are rounded ahead of the subtraction: what fma keeps of a product that its reference does not would be exponents

struct Params {
  CUtensorMap q, k, v;                                       // [row][head][entry]: boxes of 64 entries of (heads of a row tile, its tokens), (one head, a tile of keys) for both others
  const int* starts;                                         // [batch + 1]
  int* status;
  const void* values;
  void* out;
  long long v_row, v_head, o_row, o_head;
  int rows, batch, group, pack, subs, tokens, units, span;   // pack: heads of a row tile; subs: group / pack; tokens: of a row tile; units: key heads x subs; span: units that are worked on at a time
  int dk, dv, window, keep, wide_o;                          // wide_o: rows of results lie on 32 bytes (2), on 16
  float f;                                                   // scale x log2(e), positive
};

template <int DK, int DV> __host__ __device__ constexpr int tiles() { return DV == 256 ? 1 : 2; }
// tiles of keys and of values that shared memory has room for beside the queries
template <int DK, int DV> __host__ __device__ constexpr int k_places() { return DK == 64 ? 8 : DK == 128 ? 6 : DK == 192 ? 3 : 2; }
template <int DK, int DV> __host__ __device__ constexpr int v_places() { return DK == 64 ? 8 : DK == 128 ? 4 : 3; }
template <int DK, int DV> __host__ __device__ constexpr int smem_bytes() {
  return 1024 + kRows * tiles<DK, DV>() * DK * 2 + k_places<DK, DV>() * kTile * DK * 2 + v_places<DK, DV>() * kTile * DV * 2;
}

// Bounded (a poll that fails has waited some microseconds), in line: a call would cost what the wait itself does
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, bool& lost) {
  bool ok = hy::tc_poll(bar, parity);
#pragma unroll 1
  for (int i = 0; i < 1 << 20 && !ok; i++) ok = hy::tc_poll(bar, parity);
  ok = __all_sync(0xffffffffu, ok);
  lost |= !ok;
  return ok;
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int entry, int head, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(entry), "r"(head), "r"(row) : "memory");
}
// operand whose rows are the depth, a tile of keys: 64 columns to a swizzled 128-byte row, groups of eight rows 1024 bytes apart, the next 64 columns kTile rows behind
__device__ __forceinline__ uint64_t value_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(kTile * 128 >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
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
// What tokens a .. b see of them, found once: something of those ahead of upto that have kept keys (the first `kept`, among them some that the walk has for its window) or come behind some, everything of
// those from all to end - 1 (and perhaps of kept ones)
struct Seen {
  int kept, some, upto, all, end;
  __device__ __forceinline__ bool any_of(int i) const { return (i < upto) & ((i < kept) | (i >= some)); }
  __device__ __forceinline__ bool all_of(int i) const { return (i >= all) & (i < end); }
};
__device__ __forceinline__ Seen seen_by(const Params& P, const Walk& k, int a, int b) {
  const int at = k.kept - k.low;                             // from a tile's number to its place in the walk
  const bool windowed = P.window > 0;
  return Seen{windowed ? (min(P.keep, k.t1) + kTile - 1) / kTile : 0, windowed ? max(0, a + 1 - P.window) / kTile + at : 0, b / kTile + 1 + at, windowed ? max((max(0, b + 1 - P.window) + kTile - 1) / kTile + at, k.kept) : 0, (a + 1) / kTile + at};
}

// Infinities and NaN among the values that a row sees in tiles where they went to the products as zeros: its results c .. c + 15 become what they make of them
template <bool BF16> __device__ __noinline__ void give_back(const Params& P, const Item& w, const Walk& k, int pos, int head, int c, float (&x)[16]) {
  const Seen cta = seen_by(P, k, w.tok, k.t1 - 1);
  for (int i = 0; i < k.n; i++) {
    const int key0 = key_of(k, i);
    if (cta.all_of(i)) continue;
    for (int j = key0; j < min(key0 + kTile, pos + 1); j++) {
      if (P.window > 0 && pos - j >= P.window && j >= P.keep) continue;
      const uint16_t* v = static_cast<const uint16_t*>(P.values) + (long long)(w.row + j) * P.v_row + (long long)head * P.v_head + c;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const uint32_t u = v[e];
        if (BF16 ? (u & 0x7f80u) == 0x7f80u : (u & 0x7c00u) == 0x7c00u) x[e] += BF16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((unsigned short)u));
      }
    }
  }
}

template <int DK, int DV, bool BF16, int joint>              // joint: 1: both row tiles have the same rows
__global__ void __launch_bounds__(kThreads, 1) attend_packed(const __grid_constant__ Params P) {
  constexpr int TILES = tiles<DK, DV>(), KP = k_places<DK, DV>(), VP = v_places<DK, DV>(), KB = kTile * DK * 2, VB = kTile * DV * 2, SOFT = 4 * TILES, USERS = SOFT + 2 * TILES + 3;
  constexpr float LEAD = BF16 ? 40.f : -7.f, ROOM = BF16 ? -26.f : 14.f;       // a reference is taken LEAD above its maximum, and follows once that is above m + ROOM
  constexpr int MANY = 192, FEW = 64;                        // registers of a softmax thread and of another one: 512 threads have 128 each
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[78];
  __shared__ int4 items[2][4];                               // [slot][item, walk, what its rows see (and the end of that)]
  __shared__ __align__(16) uint4 claim;
  __shared__ uint32_t tmem_slot;
  __shared__ int odd_values, pieces;
  __shared__ float2 halves[TILES == 2 ? kRows : 1];          // reference and sum of the second row tile's rows, where both have the same (0 and no weight: it had no tile)
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u, qs = base, ks = qs + kRows * TILES * DK * 2, vs = ks + KP * KB, b0 = smem_u32(bars);
  const uint32_t kfull = b0, kempty = b0 + 64, vfull = b0 + 128, vempty = b0 + 192, vok = b0 + 256, vraw = b0 + 320, sfull = b0 + 384, pfull = b0 + 416, pvdone = b0 + 448, flushed = b0 + 480,
                 qfull = b0 + 512, qempty = b0 + 528, odone = b0 + 544, ifull = b0 + 560, iempty = b0 + 576, want = b0 + 592, claimed = b0 + 600, joined = b0 + 608, joint_read = b0 + 616;
  // keys and values: for each place (vraw: where values land that are looked at ahead of their products); scores, weights, products: [row tile][place]
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, tokens = TILES == 2 && !joint ? 2 * P.tokens : P.tokens, apart = joint ? 0 : P.tokens;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; i++) {
      mbar_init(kfull + 8 * i, 1); mbar_init(kempty + 8 * i, TILES); mbar_init(vfull + 8 * i, 1); mbar_init(vempty + 8 * i, TILES); mbar_init(vok + 8 * i, 1); mbar_init(vraw + 8 * i, 1);
    }
    for (int i = 0; i < 4; i++) { mbar_init(sfull + 8 * i, 1); mbar_init(pfull + 8 * i, 4); mbar_init(pvdone + 8 * i, 1); mbar_init(flushed + 8 * i, 1); }
    for (int i = 0; i < 2; i++) { mbar_init(qfull + 8 * i, 1); mbar_init(qempty + 8 * i, 1 + joint); mbar_init(odone + 8 * i, 1); mbar_init(ifull + 8 * i, 1); mbar_init(iempty + 8 * i, USERS); }
    mbar_init(want, 1);
    mbar_init(joined, 4); mbar_init(joint_read, 4);
    mbar_init(claimed, 1);
    odd_values = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // How many pieces of work there are: row tiles that are the j-th or a later one of their sequence, of all sequences
  int first[kHeld], size[kHeld], held[kHeld], most = 0;      // (the dealing warp's: first row, rows and row tiles of sequences lane, lane + 32, ..)
  // A start that falls is taken as the highest one ahead of it: no two sequences share a row, and there are no more pieces than the host allows for.  Sequences that are not held take a scan then, in
  // loops of their own (a scan in the others, behind a branch: 423 us for 1000 prompts of 50 tokens, 211 so; 192 and 142 for 1024 of one)
  bool falls = false;
  int ahead = 0;                                             // of lane c, where some start falls: the highest one ahead of sequence 32 c
  auto rows_of = [&](int b, int& from) {                     // whatever starts say, inside
    from = b < P.batch ? min(max(P.starts[b], 0), P.rows) : 0;
    return b < P.batch ? min(max(P.starts[b + 1], from), P.rows) - from : 0;
  };
  auto rows_risen = [&](int c, int& from) {                  // of sequence 32 c + lane, by the highest starts
    const int end = rows_of(32 * c + lane, from) + from;     // (not below the sequence's own start)
    from = max(from, __shfl_sync(0xffffffffu, ahead, c));
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, from, o);
      if (lane >= o) from = max(from, x);
    }
    return max(end, from) - from;
  };
  auto tiles_of = [&](int rows) { return (rows + tokens - 1) / tokens; };
  auto from_level = [&](int j) {
    int n = 0, from;
#pragma unroll
    for (int i = 0; i < kHeld; i++) n += max(held[i] - j, 0);
    if (!falls) {
      for (int b = lane + 32 * kHeld; b < P.batch; b += 32) n += max(tiles_of(rows_of(b, from)) - j, 0);
    } else {
#pragma unroll 1
      for (int c = kHeld; 32 * c < P.batch; c++) n += max(tiles_of(rows_risen(c, from)) - j, 0);
    }
    return __reduce_add_sync(0xffffffffu, n);
  };
  if (warp == 15) {
    bool fall = false;
    auto falls_behind = [&](int b, int from) { return b < P.batch && max(P.starts[b + 1], 0) < from; };
#pragma unroll
    for (int i = 0; i < kHeld; i++) { size[i] = rows_of(lane + 32 * i, first[i]); fall |= falls_behind(lane + 32 * i, first[i]); }
    for (int b = lane + 32 * kHeld; b < P.batch; b += 32) {
      int from;
      most = max(most, tiles_of(rows_of(b, from)));          // (where starts fall, too many: that is steps of a search and no more)
      fall |= falls_behind(b, from);
    }
    falls = __any_sync(0xffffffffu, fall);
    if (falls) {
      int top = 0;
#pragma unroll 1
      for (int c = 0; 32 * c < P.batch; c++) {
        if (lane == c) ahead = top;
        int from;
        const int rows = rows_risen(c, from);
        top = __shfl_sync(0xffffffffu, from, 31);
#pragma unroll
        for (int i = 0; i < kHeld; i++) if (i == c) { first[i] = from; size[i] = rows; }
      }
    }
#pragma unroll
    for (int i = 0; i < kHeld; i++) {
      held[i] = tiles_of(size[i]);
      most = max(most, held[i]);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    const int n = from_level(0);
    if (lane == 0) pieces = n;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot, o_at = tmem + 256;        // columns: scores (then weights) [row tile][place][64], results [tile][DV]
  const int all = pieces * P.units;

  bool lost = false;                                         // a wait of this warp gave up
  uint32_t turn = 0;                                         // items that this warp has taken
  auto take = [&](Item& w, Walk& k, Seen& cta) {             // the next item, the walk of its keys and what all its rows see of them, in every lane
    const uint32_t slot = turn & 1;
    const bool ok = wait_warp(ifull + 8 * slot, (turn >> 1) & 1, lost);
    const int4 x = items[slot][0], y = items[slot][1], z = items[slot][2];
    const int last = items[slot][3].x;
    __syncwarp();
    if (lane == 0) hy::tc_arrive(iempty + 8 * slot);
    turn++;
    w = Item{x.x, x.y, x.z, x.w};
    k = Walk{y.x, y.y, y.z, y.w};
    cta = Seen{z.x, z.y, z.z, z.w, last};
    return ok && w.len > 0;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW));
    const bool scoring = warp < 8 + TILES, adding = warp == 11 || warp == 10 + TILES;
    if (scoring || adding) {                                 // products of a row tile: scores, or weights x values.  (A warp for each: neither waits behind the other's)
      const int t = scoring ? warp - 8 : warp - 11;
      const uint32_t lead = hy::tc_elect();
      const uint32_t idesc = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (8u << 24);         // fp32 sums of bf16 or fp16, 128 rows
      const uint32_t s_at = tmem + t * 2 * kTile, done_at = pvdone + 16 * t;
      uint32_t passed = 0, took = 0, n = 0, par[2] = {0, 0};  // tiles behind that the row tile sees, items that had rows; the next tile's place and its parities (values: a bit for each place, as they came and looked at)
      Item w;
      Walk k;
      Seen cta;
      bool alive = true;
      while (alive && take(w, k, cta)) {
        const int a = w.tok + t * apart, b = min(a + P.tokens, w.len) - 1;
        const bool there = a < w.len;
        const Seen mine = seen_by(P, k, a, b);
        auto sixteenths = [&](int i) { return there && mine.any_of(i) && !(joint & (i ^ t)) ? mine.all_of(i) ? kTile / 16 : min(kTile / 16, (b - key_of(k, i) + 16) / 16) : 0; };   // those of a tile that some row sees
        if (scoring) {
          const int from = joint ? 0 : t;                    // the row tile whose queries these are
          const uint64_t q_desc = hy::tc_desc(qs + from * (kRows * DK * 2));
          const int ksteps = P.dk / 16;
          alive = !there || wait_warp(qfull + 8 * from, took & 1, lost);
          for (int i = 0; i < k.n && alive; i++) {
            const int see = sixteenths(i);
            const uint64_t k_desc = hy::tc_desc(ks + n * KB);
            alive = wait_warp(kfull + 8 * n, par[0], lost);
            if (see && alive) {
              const uint32_t place = passed & 1, at = s_at + place * kTile, sdesc = idesc | (uint32_t)(2 * see) << 17;
              if (passed > 1) alive = wait_warp(done_at + 8 * place, ((passed >> 1) - 1) & 1, lost);   // the weights that lie there are read
              if (!alive) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
              for (int u = 0; u < DK / 16; u++) if (u < ksteps) mma_ss(at, q_desc + (u >> 2) * (kRows * 128 >> 4) + 2 * (u & 3), k_desc + (u >> 2) * (kTile * 128 >> 4) + 2 * (u & 3), sdesc, u > 0, lead);
              commit(sfull + 16 * t + 8 * place, lead);
              passed++;
            }
            if (there) commit(kempty + 8 * n, lead);         // (stands for all products ahead of it)
            else if (lead) hy::tc_arrive(kempty + 8 * n);
            if (++n == KP) { n = 0; par[0] ^= 1; }
          }
          if (there && alive) { commit(qempty + 8 * from, lead); took++; }
        } else {
          const uint32_t pdesc = idesc | (1u << 16) | ((uint32_t)(P.dv / 8) << 17), to = o_at + t * 128;
          bool any = false;
          for (int i = 0; i < k.n && alive; i++) {
            const int see = sixteenths(i);
            const bool masked = !cta.all_of(i);
            const uint64_t v_desc = value_desc(vs + n * VB);
            alive = wait_warp((masked ? vok : vfull) + 8 * n, (masked ? par[1] : par[0]) >> n & 1, lost);
            if (masked) par[1] ^= 1u << n; else par[0] ^= 1u << n;
            if (see && alive) {
              const uint32_t place = passed & 1, weights = s_at + place * kTile;
              alive = wait_warp(pfull + 16 * t + 8 * place, (passed >> 1) & 1, lost);
              if (!alive) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
              for (int u = 0; u < kTile / 16; u++) if (u < see) mma_ts(to, weights + u * 8, v_desc + u * 128, pdesc, any || u > 0, lead);
              commit(done_at + 8 * place, lead);
              passed++;
              any = true;
            }
            if (there) commit(vempty + 8 * n, lead);
            else if (lead) hy::tc_arrive(vempty + 8 * n);
            if (++n == VP) n = 0;
          }
          if (any && alive) commit(odone + 8 * t, lead);
        }
      }
      const uint32_t last = flushed + 16 * t + (scoring ? 0 : 8);
      commit(last, lead);                                    // no product is under way when TMEM is given back
      wait_warp(last, 0, lost);
    } else if (warp == 10) {                                 // copies of keys and queries
      Item w;
      Walk k;
      Seen cta;
      const int chunks = (P.dk + 63) / 64;
      uint32_t n = 0, par = 0, took = 0, asked = 0, sent = 0;  // took, asked: a bit for each row tile (its next copy's parity; there was one)
      bool alive = true;
      while (alive && take(w, k, cta)) {
        const int head = w.unit / P.subs, q_head = head * P.group + (w.unit - head * P.subs) * P.pack;
        for (int i = 0; i < k.n && alive; i++) {
          alive = wait_warp(kempty + 8 * n, par ^ 1, lost);
          if (!alive) break;
          if (lane == 0) {
            mbar_expect_tx(kfull + 8 * n, chunks * kTile * 128);
#pragma unroll 1
            for (int c = 0; c < chunks; c++) copy_box(ks + n * KB + c * (kTile * 128), &P.k, 64 * c, head, w.row + key_of(k, i), kfull + 8 * n);
          }
          sent |= 1u << n;
          if (++n == KP) { n = 0; par ^= 1; }
          if (i == max(0, k.n - kEarly) && lane == 0) hy::tc_arrive(want);
#pragma unroll 1
          for (int t = 0; t < TILES && alive && i == 0; t++) {
            if (w.tok + t * apart >= w.len || (joint & t)) continue;
            alive = wait_warp(qempty + 8 * t, (took >> t & 1) ^ 1, lost);
            if (!alive) break;
            if (lane == 0) {
              mbar_expect_tx(qfull + 8 * t, chunks * P.tokens * P.pack * 128);
#pragma unroll 1
              for (int c = 0; c < chunks; c++) copy_box(qs + t * (kRows * DK * 2) + c * (kRows * 128), &P.q, 64 * c, q_head, w.row + w.tok + t * apart, qfull + 8 * t);
            }
            took ^= 1u << t;
            asked |= 1u << t;
          }
        }
      }
      for (int t = 0; t < TILES; t++) if (asked >> t & 1) wait_warp(qfull + 8 * t, (took >> t & 1) ^ 1, lost);   // no copy is under way at the end, whatever happened
      for (uint32_t s = 0; s < KP; s++) if (sent >> s & 1) wait_warp(kfull + 8 * s, s < n ? par : par ^ 1, lost);
    } else if (warp == 13) {                                 // copies of values
      Item w;
      Walk k;
      Seen cta;
      const int boxes = (P.dv + 63) / 64;
      uint32_t n = 0, par = 0, vpar[2] = {0, 0}, sent[2] = {0, 0};
      bool alive = true;
      while (alive && take(w, k, cta)) {
        const int head = w.unit / P.subs;
        for (int i = 0; i < k.n && alive; i++) {
          const int key0 = key_of(k, i);
          const bool masked = !cta.all_of(i);
          const uint32_t full = masked ? vraw : vfull;
          alive = wait_warp(vempty + 8 * n, par ^ 1, lost);
          if (!alive) break;
          if (lane == 0) {
            mbar_expect_tx(full + 8 * n, boxes * kTile * 128);
#pragma unroll 1
            for (int c = 0; c < boxes; c++) copy_box(vs + n * VB + c * (kTile * 128), &P.v, 64 * c, head, w.row + key0, full + 8 * n);
          }
          vpar[masked] ^= 1u << n;
          sent[masked] |= 1u << n;
          if (++n == VP) { n = 0; par ^= 1; }
        }
      }
      for (uint32_t s = 0; s < 2 * VP; s++)                  // no copy is under way at the end, whatever happened
        if (sent[s & 1] >> (s >> 1) & 1) wait_warp((s & 1 ? vraw : vfull) + 8 * (s >> 1), ~(vpar[s & 1] >> (s >> 1)) & 1, lost);
    } else if (warp == 15) {                                 // deals out the work: rows with most keys first, so that the short ones fill the gaps, of as many heads at a time as the L2 holds
      // CTAs take over work of CTAs that have not started yet, each when its copies near the end of what it has.  The grid is launched for as many pieces as there may be: CTAs that have none are
      // taken over one behind the other, without a start (37 tokens in 65536 rows, 901 sequences, 16 heads over 4: 20 us where each started and ended 157)
      uint32_t claims = 0;
      auto take_over = [&] {                                 // the CTA whose work is taken over, -1: none is left (and no other may be asked for)
        if (lane == 0) {
          mbar_expect_tx(claimed, 16);
          asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(&claim)), "r"(claimed) : "memory");
        }
        if (!wait_warp(claimed, claims++ & 1, lost)) return -1;
        uint32_t got, next;
        asm volatile("{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tld.shared.b128 h, [%2];\n\tclusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                     "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}" : "=r"(got), "=r"(next) : "r"(smem_u32(&claim)) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (read ahead of the next claim's write)
        __syncwarp();
        return got ? (int)next : -1;
      };
      int at = blockIdx.x;
      bool asks = false;
      for (uint32_t round = 0;; round++) {
        int4 item = make_int4(0, 0, 0, 0);
#pragma unroll 1
        while (asks || at >= all) { at = take_over(); asks = false; }
        if (at >= 0) {
          const int block = (uint32_t)at / (uint32_t)(pieces * P.span), wide = min(P.span, P.units - block * P.span), in = at - block * pieces * P.span, k = (uint32_t)in / (uint32_t)wide;
          int lo = 0, hi = most - 1, rank, from = 0, len = 0;          // the level lo with from_level(lo + 1) <= k < from_level(lo); the rank-th sequence with more than lo row tiles
          for (;;) {
            const int mid = lo < hi ? (lo + hi + 1) >> 1 : lo + 1, n = from_level(mid);
            if (lo >= hi) { rank = k - n; break; }
            if (n > k) lo = mid; else hi = mid - 1;
          }
          bool found = false;
          auto among = [&](bool has, int row, int rows) {
            const uint32_t mask = __ballot_sync(0xffffffffu, has), hit = __ballot_sync(0xffffffffu, has && __popc(mask & ((1u << lane) - 1)) == rank);
            if (!found && hit) {
              from = __shfl_sync(0xffffffffu, row, __ffs(hit) - 1);
              len = __shfl_sync(0xffffffffu, rows, __ffs(hit) - 1);
              found = true;
            }
            rank -= __popc(mask);
          };
#pragma unroll
          for (int i = 0; i < kHeld; i++) if (!found && 32 * i < P.batch) among(held[i] > lo, first[i], size[i]);
          if (!falls) {
            for (int c = 32 * kHeld; c < P.batch && !found; c += 32) {
              int row;
              const int rows = rows_of(c + lane, row);
              among(tiles_of(rows) > lo, row, rows);
            }
          } else {
#pragma unroll 1
            for (int c = kHeld; 32 * c < P.batch && !found; c++) {
              int row;
              const int rows = rows_risen(c, row);
              among(tiles_of(rows) > lo, row, rows);
            }
          }
          if (found) item = make_int4(from, len, lo * tokens, block * P.span + in - k * wide);
        }
        const uint32_t slot = round & 1;
        if (!wait_warp(iempty + 8 * slot, (round >> 1 & 1) ^ 1, lost)) break;
        if (lane == 0) {
          const Item w{item.x, item.y, item.z, item.w};
          const Walk k = walk_of(P, w, tokens);
          const Seen cta = seen_by(P, k, w.tok, k.t1 - 1);
          items[slot][0] = item;
          items[slot][1] = make_int4(k.t1, k.low, k.kept, k.n);
          items[slot][2] = make_int4(cta.kept, cta.some, cta.upto, cta.all);
          items[slot][3].x = cta.end;
          hy::tc_arrive(ifull + 8 * slot);
        }
        if (item.y <= 0 || !wait_warp(want, round & 1, lost)) break;
        asks = true;
      }
    } else if (warp == 14) {                                 // values of tiles that some row does not see whole: rows behind the sequence, infinities and NaN become zeros
      Item w;
      Walk k;
      Seen cta;
      const int boxes = (P.dv + 63) / 64;
      const uint32_t inf = BF16 ? 0x7f807f80u : 0x7c007c00u;
      uint32_t n = 0, par = 0;                               // par: a bit for each place
      bool alive = true;
      while (alive && take(w, k, cta)) {
        for (int i = 0; i < k.n && alive; i++, n = n + 1 == VP ? 0 : n + 1) {
          if (cta.all_of(i)) continue;
          const int key0 = key_of(k, i);
          alive = wait_warp(vraw + 8 * n, par >> n & 1, lost);
          par ^= 1u << n;
          bool odd = false;
#pragma unroll 4
          for (int p = lane; p < boxes * kTile * 8; p += 32) {   // 16-byte pieces: eight to a row of 64 columns
            const int row = key0 + ((p >> 3) & (kTile - 1));
            const uint32_t at = vs + n * VB + p * 16;
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
      }
    }
  } else if (warp < SOFT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY));
    const int t = warp >> 2, quad = warp & 3, r = threadIdx.x & 127, tok_of = r / P.pack;       // the thread's row: token tok_of of the tile, head r % pack
    const bool exists = r < P.tokens * P.pack;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16, res = o_at + t * 128 + lanes;
    uint32_t passed = 0, took = 0, pairs = 0;                // pairs: items whose rows both row tiles had
    Item w;
    Walk k;
    Seen cta;
    bool ok = true;
    while (ok && take(w, k, cta)) {
      const int a = w.tok + t * apart, b = min(a + P.tokens, w.len) - 1;
      if (a >= w.len) continue;
      const int pos = exists ? a + tok_of : 0x3fffffff;
      const bool mine = pos < w.len, idle = !__any_sync(0xffffffffu, mine);
      float m = kLowest, l = 0.f, limit = -INFINITY;         // limit: where a maximum moves the reference; any does while that is beyond kFar
      bool any = false, there = false;
      const Seen tile = seen_by(P, k, a, b);
      for (int i = 0; i < k.n; i++) {
        if (!tile.any_of(i) || (joint & (i ^ t))) continue;
        there = true;
        const int key0 = key_of(k, i);
        const uint32_t place = passed & 1, s_at = tmem + (2 * t + place) * kTile + lanes, p_bar = pfull + 16 * t + 8 * place;
        const bool masked = !tile.all_of(i);
        ok = wait_warp(sfull + 16 * t + 8 * place, (passed >> 1) & 1, lost);
        if (!ok) break;
        if (idle) {                                          // (its rows' results are whatever comes of the scores as weights, and go nowhere)
          __syncwarp();
          if (lane == 0) hy::tc_arrive(p_bar);
          passed++;
          continue;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t x[kTile];
        tmem_ask<0, kTile>(s_at, x);
        tmem_got<0, kTile>(x);
        if (masked) {                                        // keys that the row sees, a bit each: not behind its own, in the window or among the first
#pragma unroll
          for (int u = 0; u < kTile; u += 32) {
            const int j = key0 + u;
            uint32_t see = lower_bits(pos + 1 - j);
            if (P.window > 0) see &= ~lower_bits(pos - P.window + 1 - j) | lower_bits(P.keep - j);
#pragma unroll
            for (int e = 0; e < 32; e++) if (!(see >> e & 1)) x[u + e] = 0xff800000u;
          }
        }
        float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kTile; e += 8)
#pragma unroll
          for (int g = 0; g < 4; g++) y[g] = max3(__float_as_uint(y[g]), x[e + 2 * g], x[e + 2 * g + 1]);
        const float top = mine ? fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) * P.f : -INFINITY;
        float f = P.f;
        if (__any_sync(0xffffffffu, top > limit)) {
          const float to = fmaxf(m, fabsf(top) > kFar ? top : top + LEAD), by = exp2_fast(m - to);
          m = to;
          l *= by;
          const bool far = fabsf(m) > kFar;
          limit = far ? -INFINITY : m + ROOM;
          if (__any_sync(0xffffffffu, far)) {
#pragma unroll
            for (int e = 0; e < kTile; e++) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
            f = 1.f;
          }
          if (any) {
            // The product ahead must be through.  A wait by parity is right while the barrier is in the phase asked for or the one behind it: these scores waited for the product before that one
            ok = wait_warp(pvdone + 16 * t + 8 * (place ^ 1), ((passed - 1) >> 1) & 1, lost);
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
        const uint64_t f2 = both(f, f), off = both(-m, -m);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int u = 0; u < kTile / 32; u++) {
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
          tmem_store16(s_at + 16 * u, p);
        }
        l += (__uint_as_float((uint32_t)sum[0]) + __uint_as_float((uint32_t)(sum[0] >> 32))) + (__uint_as_float((uint32_t)sum[1]) + __uint_as_float((uint32_t)(sum[1] >> 32)));
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) hy::tc_arrive(p_bar);
        passed++;
        any = true;
      }
      if (there) {
        ok = ok && wait_warp(odone + 8 * t, took & 1, lost);
        took++;
      }
      float mine_by = 1.f, other_by = 0.f;                   // what becomes of the results of the two row tiles, in one reference
      if (joint && ok) {
        if (t) {
          halves[r] = make_float2(m, l);
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) hy::tc_arrive(joined);
          ok = wait_warp(joint_read, pairs++ & 1, lost);     // (its results and halves are free again)
          continue;
        }
        ok = wait_warp(joined, pairs++ & 1, lost);
        const float2 other = halves[r];
        const float to = fmaxf(m, other.x);
        mine_by = exp2_fast(m - to);
        other_by = k.n > 1 ? exp2_fast(other.x - to) : 0.f;  // (a walk of one tile leaves the second row tile none)
        l = l * mine_by + other.y * other_by;
      }
      if (!ok || idle) {
        __syncwarp();
        if (joint && lane == 0) hy::tc_arrive(joint_read);
        continue;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int odd = odd_values, head = w.unit / P.subs, q_head = head * P.group + (w.unit - head * P.subs) * P.pack + r - tok_of * P.pack;
      uint16_t* to = static_cast<uint16_t*>(P.out) + (long long)(w.row + pos) * P.o_row + (long long)q_head * P.o_head;
      mine_by *= inv;
      other_by *= inv;
#pragma unroll 1
      for (int c = 0; c < P.dv; c += 16) {                   // (64 columns at a time: as long, and more code, which a short prompt waits for)
        uint32_t x[16];
        tmem_read16(res + c, x);
        float z[16];
#pragma unroll
        for (int e = 0; e < 16; e++) z[e] = __uint_as_float(x[e]) * mine_by;
        if (joint && k.n > 1) {
          tmem_read16(res + 128 + c, x);
#pragma unroll
          for (int e = 0; e < 16; e++) z[e] = fmaf(__uint_as_float(x[e]), other_by, z[e]);
        }
        if (!mine) continue;
        if (odd) {                                           // (a copy: what a call is given by address lies in memory)
          float d[16];
#pragma unroll
          for (int e = 0; e < 16; e++) d[e] = z[e];
          give_back<BF16>(P, w, k, pos, head, c, d);
#pragma unroll
          for (int e = 0; e < 16; e++) z[e] = d[e];
        }
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = pair<BF16>(z[2 * e], z[2 * e + 1]);
        if (P.wide_o == 2) {                                 // (whole sectors: in two pieces of 16 bytes they took twice as long)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to + c), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7]) : "memory");
        } else if (P.wide_o) {
          uint4* at = reinterpret_cast<uint4*>(to + c);
          at[0] = make_uint4(y[0], y[1], y[2], y[3]);
          at[1] = make_uint4(y[4], y[5], y[6], y[7]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) { to[c + 2 * e] = (uint16_t)y[e]; to[c + 2 * e + 1] = (uint16_t)(y[e] >> 16); }
        }
      }
      if (joint) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) hy::tc_arrive(joint_read);
      }
    }
  }
  if (lost && lane == 0 && P.status) atomicOr(P.status, ST_WAIT);
  __syncthreads();
  if (warp == 8) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

}  // namespace prompt
}  // namespace dsk
