// dsk_serve_host.cuh — what the C entry points of the operators on device memory share on the host: errors, devices, launches, checks of caches and views.
#pragma once

#include "../../include/dsk.h"

#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdio>
#include <mutex>

#include "dsk_host.h"
#include "dsk_kv8.cuh"

using namespace dsk;

static int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  fail_text(code, fmt, ap);
  va_end(ap);
  return code;
}
#define CK(call)                                                                                   \
  do {                                                                                             \
    cudaError_t e_ = (call);                                                                       \
    if (e_ != cudaSuccess) { cudaGetLastError(); return fail(-2, "%s failed: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__); } \
  } while (0)

namespace {
constexpr int kMaxDevices = 64;

// The caller's current device comes back at the end of a call.
struct OnDevice {
  int before = -1, device;
  cudaError_t error;
  explicit OnDevice(int d) : device(d) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && before != d) error = cudaSetDevice(d);
  }
  ~OnDevice() { if (before >= 0 && before != device) cudaSetDevice(before); }
};
int multiprocessors(int device) {
  static std::mutex lock;
  static int known[kMaxDevices];
  std::lock_guard<std::mutex> hold(lock);
  if (!known[device] && cudaDeviceGetAttribute(&known[device], cudaDevAttrMultiProcessorCount, device) != cudaSuccess) { cudaGetLastError(); known[device] = 0; }
  return known[device];
}
// Shared memory beyond 48 KB, granted once for a kernel and device.
template <auto KERNEL> cudaError_t allow(int device, int bytes) {
  static std::mutex lock;
  static int granted[kMaxDevices];
  std::lock_guard<std::mutex> hold(lock);
  if (granted[device] >= bytes) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) granted[device] = bytes;
  return e;
}
// A launch behind another one of the same call: its CTAs may come up under the kernel ahead and wait there (grid_wait).
template <typename... KA, typename... A>
cudaError_t launch_behind(void (*kernel)(KA...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, int cluster, A... a) {   // cluster < 0: clusters of -cluster, not behind anything
  cudaLaunchConfig_t c{};
  cudaLaunchAttribute at[2];
  c.gridDim = grid; c.blockDim = block; c.dynamicSmemBytes = smem; c.stream = stream; c.attrs = at; c.numAttrs = 0;
  if (cluster > 0) {
    at[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[c.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1 || cluster < -1) {
    at[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[c.numAttrs].val.clusterDim.x = std::abs(cluster); at[c.numAttrs].val.clusterDim.y = 1; at[c.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&c, kernel, static_cast<KA>(a)...);
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int size_of(int dtype) { return dtype == DSK_DT_F32 ? 4 : 2; }

int check_device(int device) {
  static std::atomic<int> known{0};                          // (devices do not come and go within a process)
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    const cudaError_t e = cudaGetDeviceCount(&n);
    if (e != cudaSuccess || n == 0) { cudaGetLastError(); return fail(-1, "no CUDA device available (%s) — libdsk has no CPU fallback", cudaGetErrorString(e)); }
    known.store(n, std::memory_order_relaxed);
  }
  if (device < 0 || device >= n || device >= kMaxDevices) return fail(-1, "device %d out of range (have %d)", device, n);
  return 0;
}
int check_cache(const dsk_kv8* c) {
  if (!c) return fail(-1, "null cache or rows");
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return fail(-4, "blocks of %d tokens: 16, 32, 64 or 128 are supported", c->block);
  if (c->n_blocks <= 0 || c->kv_heads <= 0 || c->kv_heads > 32767) return fail(-4, "%d blocks of %d key heads: both must be positive, heads at most 32767", c->n_blocks, c->kv_heads);
  for (int d : {c->dim_k, c->dim_v})
    if (d <= 0 || d % 16 || d > 256) return fail(-4, "heads of %d entries: a multiple of 16 up to 256 is needed", d);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(-1, "cache: null memory");
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->status, 4)) return fail(-1, "cache: codes need 16-byte alignment, scales and status 4");
  return 0;
}
int check_cache(const dsk_kv8* c, const dsk_kv8_rows* s) {
  if (!c || !s) return fail(-1, "null cache or rows");
  if (const int code = check_cache(c)) return code;
  if (s->batch < 0 || s->rows < 0 || s->batch > 65535 || s->table_blocks < 0 || s->table_blocks > (1 << 30) / c->block)
    return fail(-4, "batch %d (at most 65535), %d rows, tables of %d blocks (2^30 tokens at most)", s->batch, s->rows, s->table_blocks);
  if (s->batch && s->rows && (!s->table || !s->first || s->table_blocks == 0)) return fail(-1, "rows: null or empty table, or null first");
  if (!aligned(s->table, 4) || !aligned(s->first, 4) || !aligned(s->count, 4)) return fail(-1, "rows: table, first and count need 4-byte alignment");
  return check_device(c->device);
}
int check_view(const char* what, const dsk_view* v, int dtype) {
  if (!v || !v->data) return fail(-1, "%s: null", what);
  if (v->dtype != dtype) return fail(-4, "%s: element type %d where %d is needed", what, v->dtype, dtype);
  if (!aligned(v->data, size_of(dtype))) return fail(-1, "%s: memory is not aligned to its element", what);
  return 0;
}
bool wide(const dsk_view* v) {
  const int n = 16 / size_of(v->dtype);
  return aligned(v->data, 16) && v->batch % n == 0 && v->row % n == 0 && v->head % n == 0;
}
kv8::Cache cache_of(const dsk_kv8* c) {
  return kv8::Cache{{static_cast<unsigned char*>(c->k), static_cast<unsigned char*>(c->v)}, {c->k_scale, c->v_scale}, c->status, c->n_blocks, c->block, c->kv_heads, {c->dim_k, c->dim_v}, c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7};
}
kv8::Rows rows_of(const dsk_kv8_rows* s) { return kv8::Rows{s->table, s->table_pitch, s->first, s->count, s->table_blocks, s->batch, s->rows}; }
kv8::Pitch pitch_of(const dsk_view* v) { return kv8::Pitch{v->batch, v->row, v->head}; }

// Rows to the cache: `most` rows at most of a block, `where` says which (kv8::piece)
template <typename T, bool WIDE, typename Where> int write_as(const dsk_kv8* c, const Where& where, dim3 grid, int most, const dsk_view* k, const dsk_view* v, cudaStream_t stream) {
  const T *pk = static_cast<const T*>(k->data), *pv = static_cast<const T*>(v->data);
  const int eights = most * (c->dim_k > c->dim_v ? c->dim_k : c->dim_v) / 8;
  // a CTA's values stay in registers: a warp of four eights a lane for a few rows (no barrier), otherwise few threads with many (what a thread does once, addresses for the most part,
  // is 200 instructions; twice the threads with half the eights: 98 us for four prompts of 8191 tokens)
#define WRITE(TH, R) kv8::write_rows<T, TH, R, WIDE, Where><<<grid, TH, 0, stream>>>(cache_of(c), where, pk, pv, pitch_of(k), pitch_of(v))
  if (eights <= 128) WRITE(32, 4);
  else if (eights <= 512) WRITE(64, 8);
  else if (eights <= 1024) WRITE(64, 16);
  else if (eights <= 2048) WRITE(128, 16);
  else WRITE(256, 16);
#undef WRITE
  CK(cudaGetLastError());
  return 0;
}
template <typename T, typename Where> int write_as(const dsk_kv8* c, const Where& where, dim3 grid, int most, const dsk_view* k, const dsk_view* v, cudaStream_t stream) {
  return wide(k) && wide(v) ? write_as<T, true>(c, where, grid, most, k, v, stream) : write_as<T, false>(c, where, grid, most, k, v, stream);
}
template <typename Where> int write_all(const dsk_kv8* c, const Where& where, dim3 grid, int most, const dsk_view* k, const dsk_view* v, cudaStream_t stream) {
  return k->dtype == DSK_DT_F32 ? write_as<float>(c, where, grid, most, k, v, stream) : k->dtype == DSK_DT_F16 ? write_as<__half>(c, where, grid, most, k, v, stream)
                                                                                                                : write_as<__nv_bfloat16>(c, where, grid, most, k, v, stream);
}
}  // namespace
