// dsk_kv8.cuh — a key / value cache held in 8 bits: writing (quantising) and reading back.
//
// The cache is made of blocks of `block` tokens, [block][head][token][entry] E4M3 codes and one fp32 scale for every block and head: value = code x scale.
// Scales are powers of two, the smallest s with amax <= 448 s: multiplying by one is exact, so that a value is rounded once, by the conversion to E4M3
// (at most half a step, 2^-4 of it, or 2^-10 s below 2^-6 s), whatever else the block holds.  A float code keeps its relative accuracy at any scale within its range, so
// the up to one bit of range that a power of two leaves unused costs nothing but there.  A block is written in several calls: its scale never falls while it holds rows
// of earlier ones, and where it grows, their codes are rounded again, which changes those alone that leave the normal range.  Exponents stay within +-kExp,
// so that attention's sums of weights over scales stay in fp32's range (dsk_kv8_attn.cuh).
// Bound of both kernels: bytes; small calls by the chain of dependent loads (first token, block, rows).  Four prompts of up to 8191 tokens, 16 heads of 192 + 128 entries in bf16 are written in
// 79 us (409 MB: 5.2 TB/s; a measured copy 6.5), 8 x 8000 tokens of 4 heads of 128 + 128 read in 32 us (160 MB: 5.0 TB/s), one token written in 2.2 us, 161 read in 2.3.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "dsk_async.cuh"

namespace dsk {
namespace kv8 {

constexpr int kExp = 40;                                     // exponents of scales
enum { ST_PAGE = 1, ST_RANGE = 2, ST_WAIT = 4 };             // bits of Cache::status: a block outside the cache, tokens outside the table, a wait that gave up

struct Cache {
  unsigned char* code[2];                                    // keys, values
  float* scale[2];
  int* status;                                               // nullable
  int n_blocks, block, heads, dim[2], shift;                 // shift: log2 of block
};
struct Rows {                                                // rows of a padded batch, and where their sequences lie in the cache
  const int* table;                                          // [batch] rows of table_blocks, table_pitch apart
  long long table_pitch;
  const int *first, *count;                                  // (first: what the operator says; count nullable: all rows)
  int table_blocks, batch, rows;
};
struct Pitch { long long batch, row, head; };                // in elements; entries of a head lie side by side

__device__ __forceinline__ void note(const Cache& C, int bit) { if (C.status) atomicOr(C.status, bit); }

// eight values as they lie in memory
template <typename T> struct Eight { uint4 q[sizeof(T) / 2]; };
template <typename T, bool WIDE> __device__ __forceinline__ Eight<T> load_eight(const T* p) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; i++) {
    if (WIDE) e.q[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    else if constexpr (sizeof(T) == 4) e.q[i] = make_uint4(__float_as_uint(p[4 * i]), __float_as_uint(p[4 * i + 1]), __float_as_uint(p[4 * i + 2]), __float_as_uint(p[4 * i + 3]));
    else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
      e.q[i] = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
    }
  }
  return e;
}
__device__ __forceinline__ void floats(const Eight<float>& e, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; i++) { x[4 * i] = __uint_as_float(e.q[i].x); x[4 * i + 1] = __uint_as_float(e.q[i].y); x[4 * i + 2] = __uint_as_float(e.q[i].z); x[4 * i + 3] = __uint_as_float(e.q[i].w); }
}
__device__ __forceinline__ void floats(const Eight<__half>& e, float (&x)[8]) {
  const uint32_t w[4] = {e.q[0].x, e.q[0].y, e.q[0].z, e.q[0].w};
#pragma unroll
  for (int i = 0; i < 4; i++) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i])); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
__device__ __forceinline__ void floats(const Eight<__nv_bfloat16>& e, float (&x)[8]) {
  const uint32_t w[4] = {e.q[0].x, e.q[0].y, e.q[0].z, e.q[0].w};
#pragma unroll
  for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
// the largest magnitudes so far (16-bit types: of the even and of the odd values; NaN are passed over), and the larger one
template <typename T> struct Highest { uint32_t v = 0; };
__device__ __forceinline__ void higher(Highest<float>& top, const Eight<float>& e) {
  float m = __uint_as_float(top.v);
#pragma unroll
  for (int i = 0; i < 2; i++) m = fmaxf(fmaxf(fmaxf(m, fabsf(__uint_as_float(e.q[i].x))), fabsf(__uint_as_float(e.q[i].y))), fmaxf(fabsf(__uint_as_float(e.q[i].z)), fabsf(__uint_as_float(e.q[i].w))));
  top.v = __float_as_uint(m);
}
template <typename T2> __device__ __forceinline__ uint32_t higher_pair(uint32_t a, uint32_t b) {
  const T2 r = __hmax2(*reinterpret_cast<const T2*>(&a), __habs2(*reinterpret_cast<const T2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void higher(Highest<__half>& top, const Eight<__half>& e) {
  top.v = higher_pair<__half2>(higher_pair<__half2>(higher_pair<__half2>(higher_pair<__half2>(top.v, e.q[0].x), e.q[0].y), e.q[0].z), e.q[0].w);
}
__device__ __forceinline__ void higher(Highest<__nv_bfloat16>& top, const Eight<__nv_bfloat16>& e) {
  top.v = higher_pair<__nv_bfloat162>(higher_pair<__nv_bfloat162>(higher_pair<__nv_bfloat162>(higher_pair<__nv_bfloat162>(top.v, e.q[0].x), e.q[0].y), e.q[0].z), e.q[0].w);
}
// the same, slower, of numbers alone (as bits, whose order is that of the magnitudes)
template <typename T> __device__ __forceinline__ void highest_number(Highest<T>& top, const Eight<T>& e) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; i++) {
    const uint32_t w[4] = {e.q[i].x, e.q[i].y, e.q[i].z, e.q[i].w};
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if constexpr (sizeof(T) == 4) { const uint32_t a = w[u] & 0x7fffffffu; top.v = max(top.v, a < 0x7f800000u ? a : 0u); }
      else {
        constexpr uint32_t inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
        const uint32_t a = w[u] & 0x7fffu, b = (w[u] >> 16) & 0x7fffu;
        top.v = max(top.v, max(a < inf ? a : 0u, b < inf ? b : 0u));
      }
    }
  }
}
__device__ __forceinline__ float magnitude(Highest<float> top) { return __uint_as_float(top.v); }
__device__ __forceinline__ float magnitude(Highest<__half> top) { return __half2float(__ushort_as_half(max(top.v & 0xffffu, top.v >> 16))); }
__device__ __forceinline__ float magnitude(Highest<__nv_bfloat16> top) { return __uint_as_float(max(top.v << 16, top.v & 0xffff0000u)); }
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {   // round to nearest even, infinities to +-448, NaN stays
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}" : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ uint32_t two_halves(uint32_t codes) {                       // two codes (the low 16 bits) as fp16, exact
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ void four_halves(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float2 two_values(uint32_t codes) {
  const uint32_t h = two_halves(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// exponent of the smallest power of two s with amax <= 448 s (448 = 1.75 x 2^8)
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
  return max(-kExp, min(kExp, e));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// What a CTA has of a sequence: rows lo .. hi - 1 (tokens) of the blockIdx.x-th block that its rows touch
struct Piece { int page, kept, rows; long long from; };      // kept: the first row's place in the block; from: the first row's place among the new ones; page: checked by `known`
__device__ __forceinline__ bool known(const Cache& C, const Piece& p) {
  if ((unsigned)p.page < (unsigned)C.n_blocks) return true;
  if (threadIdx.x == 0) note(C, ST_PAGE);
  return false;
}
__device__ __forceinline__ bool piece(const Cache& C, const Rows& S, int b, Piece& p) {
  const long long start = S.first[b], n = S.count ? min(max(S.count[b], 0), S.rows) : S.rows, room = (long long)S.table_blocks << C.shift;
  const bool outside = n > 0 && (start < 0 || start + n > room);
  if (outside && blockIdx.x == 0 && threadIdx.x == 0) note(C, ST_RANGE);
  if (start < 0 || start >= room) return false;
  const long long j = (start >> C.shift) + blockIdx.x, lo = max(start, j << C.shift), hi = min(min(start + n, room), (j + 1) << C.shift);   // (64-bit divisions were a third of all instructions)
  if (lo >= hi) return false;
  p.page = S.table[b * S.table_pitch + j];
  p.kept = (int)(lo - (j << C.shift));
  p.rows = (int)(hi - lo);
  p.from = lo - start;
  return true;
}

// A CTA of TH threads writes one block of one head, keys or values; its values stay in registers between the maximum and the codes (R eights a thread).
template <typename T, int TH, int R, bool WIDE>
__global__ void __launch_bounds__(TH) write_rows(const Cache C, const Rows S, const T* k, const T* v, const Pitch pk, const Pitch pv) {
  __shared__ uint32_t most[TH / 32];
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1;
  Piece p;
  if (!piece(C, S, b, p)) return;
  const int dim = C.dim[which], per = dim / 8, total = p.rows * per;
  const Pitch at = which ? pv : pk;
  const T* src = (which ? v : k) + b * at.batch + p.from * at.row + h * at.head;
  Eight<T> x[R];
  const int dr = TH / per, dc = TH - dr * per, row = threadIdx.x / per, mine = ((int)threadIdx.x < total) + (total - 1 - (int)threadIdx.x) / TH;   // mine: eights of this thread
  int col = threadIdx.x - row * per;
  const long long step = dr * at.row + dc * 8, wrap = at.row - per * 8;
  src += row * at.row + col * 8;
#pragma unroll
  for (int i = 0; i < R; i++) {
    if (i < mine) x[i] = load_eight<T, WIDE>(src);
    src += step; col += dc;
    if (col >= per) { col -= per; src += wrap; }
  }
  if (!known(C, p)) return;                                  // (the rows do not wait for the block's number)
  float* scale = C.scale[which] + (size_t)p.page * C.heads + h;
  unsigned char* dst = C.code[which] + ((size_t)p.page * C.heads + h) * C.block * dim;
  const float old = p.kept ? *scale : 0.f;
  // the largest magnitude; where that is an infinity, which makes no scale, once more without
  Highest<T> top;
#pragma unroll
  for (int i = 0; i < R; i++) if (i < mine) higher(top, x[i]);
  float m = magnitude(top);
  if (!(m < INFINITY)) {
    top.v = 0;
#pragma unroll
    for (int i = 0; i < R; i++) if (i < mine) highest_number(top, x[i]);
    m = magnitude(top);
  }
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
  if (TH > 32) {
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TH / 32; i++) bits = max(bits, most[i]);
  }
  const float need = pow2(scale_exponent(__uint_as_float(bits))), now = p.kept ? fmaxf(old, need) : need, inv = __uint_as_float((254u << 23) - __float_as_uint(now));   // (powers of two)
  if (threadIdx.x == 0) *scale = now;                        // (every thread has read the old one ahead of the maximum)
  if (p.kept && old != now) {                                // rows of earlier calls, in the new scale
    const float ratio = old * inv;
    for (int i = threadIdx.x; i < p.kept * dim / 16; i += TH) {
      uint4 c = reinterpret_cast<uint4*>(dst)[i];
      uint32_t* w = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const float2 lo = two_values(w[u]), hi = two_values(w[u] >> 16);
        w[u] = four_codes(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
      }
      reinterpret_cast<uint4*>(dst)[i] = c;
    }
  }
  uint2* to = reinterpret_cast<uint2*>(dst + p.kept * dim) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < R; i++)
    if (i < mine) {
      float f[8];
      floats(x[i], f);
      uint2 c;
      c.x = four_codes(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
      c.y = four_codes(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
      to[i * TH] = c;
    }
}

template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }
template <> __device__ __forceinline__ __half rounded<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// A CTA reads one block of one head, keys or values: a lane has as many codes as give it 16 bytes of result, so that a warp's stores lie side by side (with 16 codes to a lane they were
// half sectors: 37 us for 8 x 8000 tokens), four loads under way.
constexpr int kReadThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kReadThreads) read_rows(const Cache C, const Rows S, T* k, T* v, const Pitch pk, const Pitch pv, int wide) {
  constexpr int N = 16 / (int)sizeof(T), W = N / 4, AT_A_TIME = 8 / W;
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1;
  Piece p;
  if (!piece(C, S, b, p) || !known(C, p)) return;
  const int dim = C.dim[which], per = dim / N, total = p.rows * per;
  const Pitch at = which ? pv : pk;
  T* dst = (which ? v : k) + b * at.batch + p.from * at.row + h * at.head;
  const float scale = C.scale[which][(size_t)p.page * C.heads + h];
  const uint32_t* src = reinterpret_cast<const uint32_t*>(C.code[which] + (((size_t)p.page * C.heads + h) * C.block + p.kept) * dim);
  const int dr = kReadThreads / per, dc = kReadThreads - dr * per;
  int row = threadIdx.x / per, col = threadIdx.x - row * per;
  for (int i0 = threadIdx.x; i0 < total; i0 += AT_A_TIME * kReadThreads) {
    uint32_t c[AT_A_TIME][W];
#pragma unroll
    for (int u = 0; u < AT_A_TIME; u++)
      if (i0 + u * kReadThreads < total) {
        if constexpr (W == 2) { const uint2 x = __ldg(reinterpret_cast<const uint2*>(src) + i0 + u * kReadThreads); c[u][0] = x.x; c[u][1] = x.y; }
        else c[u][0] = __ldg(src + i0 + u * kReadThreads);
      }
#pragma unroll
    for (int u = 0; u < AT_A_TIME; u++) {
      if (i0 + u * kReadThreads >= total) break;
      __align__(16) T o[N];
#pragma unroll
      for (int q = 0; q < W; q++) {
        const float2 lo = two_values(c[u][q]), hi = two_values(c[u][q] >> 16);
        o[4 * q] = rounded<T>(lo.x * scale); o[4 * q + 1] = rounded<T>(lo.y * scale); o[4 * q + 2] = rounded<T>(hi.x * scale); o[4 * q + 3] = rounded<T>(hi.y * scale);
      }
      T* to = dst + row * at.row + col * N;
      if (wide) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(o);
      else
#pragma unroll
        for (int q = 0; q < N; q++) to[q] = o[q];
      row += dr; col += dc;
      if (col >= per) { col -= per; row++; }
    }
  }
}

}  // namespace kv8
}  // namespace dsk
