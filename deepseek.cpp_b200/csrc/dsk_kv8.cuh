// dsk_kv8.cuh — a key / value cache held in 8 bits: writing (quantising) and reading back.
//
// The cache is made of blocks of `block` tokens, [block][head][token][entry] E4M3 codes and one fp32 scale for every block and head: value = code x scale.
// Scales are powers of two, the smallest s with amax <= 448 s: multiplying by one is exact, so that a value is rounded once, by the conversion to E4M3
// (at most half a step, 2^-4 of it, or 2^-10 s below 2^-6 s), whatever else the block holds.  A float code keeps its relative accuracy at any scale within its range, so
// the up to one bit of range that a power of two leaves unused costs nothing but there.  A block is written in several calls: its scale never falls while it holds rows
// of earlier ones, and where it grows, their codes are rounded again, which changes those alone that leave the normal range.  Exponents stay within +-kExp:
// attention keeps weights times scales in fp32 (dsk_kv8_attn.cuh).
// Bound of both kernels: bytes; small calls by the chain of dependent loads (first token, block, rows).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "dsk_async.cuh"

namespace dsk {
namespace kv8 {

constexpr int kExp = 40;                                     // exponents of scales
enum { ST_PAGE = 1, ST_RANGE = 2, ST_WAIT = 4 };             // bits of Cache::status: a block outside the cache, tokens outside the table, a wait that gave up

struct Cache {
  unsigned char* code[2];                                    // keys, values
  float* scale[2];
  int* status;                                               // nullable
  int n_blocks, block, heads, dim[2];
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
template <typename T> __device__ __forceinline__ Eight<T> load_eight(const T* p, bool wide) {
  Eight<T> e;
  if (wide) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) e.q[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
    T* x = reinterpret_cast<T*>(&e);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = p[i];
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
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {   // round to nearest even, infinities to +-448, NaN stays
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
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
struct Piece { int page, kept, rows; long long from; };      // kept: the first row's place in the block; from: the first row's place among the new ones
__device__ __forceinline__ bool piece(const Cache& C, const Rows& S, int b, Piece& p) {
  const long long start = S.first[b], n = S.count ? min(max(S.count[b], 0), S.rows) : S.rows, room = (long long)S.table_blocks * C.block;
  const bool outside = n > 0 && (start < 0 || start + n > room);
  if (outside && blockIdx.x == 0 && threadIdx.x == 0) note(C, ST_RANGE);
  if (start < 0 || start >= room) return false;
  const long long j = start / C.block + blockIdx.x, lo = max(start, j * C.block), hi = min(min(start + n, room), (j + 1) * C.block);
  if (lo >= hi) return false;
  p.page = S.table[b * S.table_pitch + j];
  if ((unsigned)p.page >= (unsigned)C.n_blocks) {
    if (threadIdx.x == 0) note(C, ST_PAGE);
    return false;
  }
  p.kept = (int)(lo - j * C.block);
  p.rows = (int)(hi - lo);
  p.from = lo - start;
  return true;
}

// A CTA of TH threads writes one block of one head, keys or values; its values stay in registers between the maximum and the codes (R eights a thread).
template <typename T, int TH, int R>
__global__ void __launch_bounds__(TH) write_rows(const Cache C, const Rows S, const T* k, const T* v, const Pitch pk, const Pitch pv, int wide) {
  __shared__ uint32_t most[TH / 32];
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1;
  Piece p;
  if (!piece(C, S, b, p)) return;
  const int dim = C.dim[which], per = dim / 8, total = p.rows * per;
  const Pitch at = which ? pv : pk;
  const T* src = (which ? v : k) + b * at.batch + p.from * at.row + h * at.head;
  float* scale = C.scale[which] + (size_t)p.page * C.heads + h;
  unsigned char* dst = C.code[which] + ((size_t)p.page * C.heads + h) * C.block * dim;
  const float old = p.kept ? *scale : 0.f;
  Eight<T> x[R];
  const int dr = TH / per, dc = TH - dr * per;
  int row = threadIdx.x / per, col = threadIdx.x - row * per;
#pragma unroll
  for (int i = 0; i < R; i++) {
    if (i * TH + (int)threadIdx.x < total) x[i] = load_eight(src + row * at.row + col * 8, wide);
    row += dr; col += dc;
    if (col >= per) { col -= per; row++; }
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++)
    if (i * TH + (int)threadIdx.x < total) {
      float f[8];
      floats(x[i], f);
#pragma unroll
      for (int u = 0; u < 8; u++) { const float a = fabsf(f[u]); m = fmaxf(m, a < INFINITY ? a : 0.f); }   // (neither infinities nor NaN make a scale)
    }
  uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
  if (TH > 32) {
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TH / 32; i++) bits = max(bits, most[i]);
  }
  const float need = pow2(scale_exponent(__uint_as_float(bits))), now = p.kept ? fmaxf(old, need) : need, inv = 1.f / now;
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
  dst += p.kept * dim;
#pragma unroll
  for (int i = 0; i < R; i++)
    if (i * TH + (int)threadIdx.x < total) {
      float f[8];
      floats(x[i], f);
      uint2 c;
      c.x = four_codes(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
      c.y = four_codes(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
      reinterpret_cast<uint2*>(dst)[i * TH + threadIdx.x] = c;
    }
}

__device__ __forceinline__ void store_sixteen(float* p, const float (&x)[16], bool wide) {
  if (wide)
#pragma unroll
    for (int i = 0; i < 4; i++) reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  else
#pragma unroll
    for (int i = 0; i < 16; i++) p[i] = x[i];
}
template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }
template <> __device__ __forceinline__ __half rounded<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <typename T> __device__ __forceinline__ void store_sixteen(T* p, const float (&x)[16], bool wide) {   // 16-bit types
  T o[16];
#pragma unroll
  for (int i = 0; i < 16; i++) o[i] = rounded<T>(x[i]);
  if (wide) {
    reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<uint4*>(o)[0];
    reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<uint4*>(o)[1];
  } else
#pragma unroll
    for (int i = 0; i < 16; i++) p[i] = o[i];
}

// A CTA reads one block of one head, keys or values, sixteen codes a thread at a time, four loads under way.
constexpr int kReadThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kReadThreads) read_rows(const Cache C, const Rows S, T* k, T* v, const Pitch pk, const Pitch pv, int wide) {
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1;
  Piece p;
  if (!piece(C, S, b, p)) return;
  const int dim = C.dim[which], per = dim / 16, total = p.rows * per;
  const Pitch at = which ? pv : pk;
  T* dst = (which ? v : k) + b * at.batch + p.from * at.row + h * at.head;
  const float scale = C.scale[which][(size_t)p.page * C.heads + h];
  const uint4* src = reinterpret_cast<const uint4*>(C.code[which] + (((size_t)p.page * C.heads + h) * C.block + p.kept) * dim);
  for (int i0 = threadIdx.x; i0 < total; i0 += 4 * kReadThreads) {
    uint4 c[4];
#pragma unroll
    for (int u = 0; u < 4; u++) if (i0 + u * kReadThreads < total) c[u] = __ldg(src + i0 + u * kReadThreads);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int i = i0 + u * kReadThreads, row = i / per;
      if (i >= total) break;
      const uint32_t w[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
      float x[16];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const float2 lo = two_values(w[q]), hi = two_values(w[q] >> 16);
        x[4 * q] = lo.x * scale; x[4 * q + 1] = lo.y * scale; x[4 * q + 2] = hi.x * scale; x[4 * q + 3] = hi.y * scale;
      }
      store_sixteen(dst + row * at.row + (i - row * per) * 16, x, wide);
    }
  }
}

}  // namespace kv8
}  // namespace dsk
