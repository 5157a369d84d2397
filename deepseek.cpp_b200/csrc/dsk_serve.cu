// dsk_serve.cu — C-ABI (include/dsk.h) of the operators on device memory: the 8-bit key / value cache (write, read, attention) and the verification of
// drafted tokens.  They belong to no model: the caller gives memory, workspace, device and stream; nothing is allocated, waited for or kept, so that calls can be
// captured into graphs and run on several streams and devices at a time.

#include "../../include/dsk.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <mutex>

#include "dsk_host.h"
#include "dsk_kv8.cuh"
#include "dsk_kv8_attn.cuh"
#include "dsk_kv8_tc5.cuh"
#include "dsk_verify.cuh"

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
int check_cache(const dsk_kv8* c, const dsk_kv8_rows* s) {
  if (!c || !s) return fail(-1, "null cache or rows");
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return fail(-4, "blocks of %d tokens: 16, 32, 64 or 128 are supported", c->block);
  if (c->n_blocks <= 0 || c->kv_heads <= 0 || c->kv_heads > 32767) return fail(-4, "%d blocks of %d key heads: both must be positive, heads at most 32767", c->n_blocks, c->kv_heads);
  for (int d : {c->dim_k, c->dim_v})
    if (d <= 0 || d % 16 || d > 256) return fail(-4, "heads of %d entries: a multiple of 16 up to 256 is needed", d);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(-1, "cache: null memory");
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->status, 4)) return fail(-1, "cache: codes need 16-byte alignment, scales and status 4");
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
// blocks that the rows of one sequence may touch
unsigned touched(const dsk_kv8* c, const dsk_kv8_rows* s) {
  return (unsigned)std::min<long long>(s->table_blocks, ((long long)s->rows + c->block - 2) / c->block + 1);
}

template <typename T, bool WIDE> int write_as(const dsk_kv8* c, const dsk_kv8_rows* s, const dsk_view* k, const dsk_view* v, cudaStream_t stream) {
  const dim3 grid(touched(c, s), 2 * c->kv_heads, s->batch);
  const T *pk = static_cast<const T*>(k->data), *pv = static_cast<const T*>(v->data);
  const int eights = std::min(s->rows, c->block) * std::max(c->dim_k, c->dim_v) / 8;
  // a CTA's values stay in registers: a warp of four eights a lane for a few rows (no barrier), otherwise few threads with many (what a thread does once, addresses for the most part,
  // is 200 instructions; twice the threads with half the eights: 98 us for four prompts of 8191 tokens)
#define WRITE(TH, R) kv8::write_rows<T, TH, R, WIDE><<<grid, TH, 0, stream>>>(cache_of(c), rows_of(s), pk, pv, pitch_of(k), pitch_of(v))
  if (eights <= 128) WRITE(32, 4);
  else if (eights <= 512) WRITE(64, 8);
  else if (eights <= 1024) WRITE(64, 16);
  else if (eights <= 2048) WRITE(128, 16);
  else WRITE(256, 16);
#undef WRITE
  CK(cudaGetLastError());
  return 0;
}
template <typename T> int write_as(const dsk_kv8* c, const dsk_kv8_rows* s, const dsk_view* k, const dsk_view* v, cudaStream_t stream) {
  return wide(k) && wide(v) ? write_as<T, true>(c, s, k, v, stream) : write_as<T, false>(c, s, k, v, stream);
}
template <typename T> int read_as(const dsk_kv8* c, const dsk_kv8_rows* s, const dsk_view* k, const dsk_view* v, cudaStream_t stream) {
  const dim3 grid(touched(c, s), 2 * c->kv_heads, s->batch);
  kv8::read_rows<T><<<grid, kv8::kReadThreads, 0, stream>>>(cache_of(c), rows_of(s), static_cast<T*>(k->data), static_cast<T*>(v->data), pitch_of(k), pitch_of(v), wide(k) && wide(v));
  CK(cudaGetLastError());
  return 0;
}

// How an attention call is laid out
struct Layout { int shape, tiles, row_tiles, ctas, shares, cluster; size_t bytes; };   // shares > 0: attend_rows
// Query rows of a key head up to which attend_tokens has them, attend_rows behind that.  us for 16 sequences of 4000 tokens, 4 key heads, attend_tokens / attend_rows: 128 entries,
// 24 rows 31 / 38, 32 rows 46 / 38; 192, 16 rows 44 / 41, 24 rows 54 / 41 (one sequence 17 / 20); 64, 24 rows 24 / 33, 32 rows 30 / 33; 256, 16 rows 44 / 80, 32 rows (two tiles twice) 72 / 80.
constexpr int kPortionRows = 24, kWidePortionRows = 32;
constexpr int kShapes[4][2] = {{64, 64}, {128, 128}, {192, 128}, {256, 256}};
int window_of(int window) { return window >= 1 << 30 ? 0 : window; }   // (no table has more tokens)
int layout_of(const dsk_kv8* c, const dsk_kv8_rows* s, int heads, int window, int keep_first, Layout* L) {
  if (window < 0 || keep_first < 0) return fail(-4, "window %d and keep_first %d must not be negative", window, keep_first);
  window = window_of(window);
  if (heads <= 0 || heads % c->kv_heads) return fail(-4, "%d query heads over %d key heads: a multiple is needed", heads, c->kv_heads);
  if (s->batch > kv8::kMaxBatch) return fail(-4, "attention over %d sequences: at most %d a call", s->batch, kv8::kMaxBatch);
  const long long rows = (long long)(heads / c->kv_heads) * s->rows;
  if (rows > (1 << 22)) return fail(-4, "%lld query rows of a key head: at most 2^22", rows);
  for (L->shape = 0; c->dim_k > kShapes[L->shape][0] || c->dim_v > kShapes[L->shape][1];) L->shape++;
  if (!rows || !s->batch) { *L = Layout{}; return 0; }      // (nothing to lay out)
  const int sms = multiprocessors(c->device);
  if (!sms) return fail(-2, "device %d: no attributes", c->device);
  const long long keys = (long long)s->table_blocks * c->block;
  L->shares = L->cluster = 0;
  if (rows > (L->shape < 3 ? kPortionRows : kWidePortionRows)) {
    L->tiles = rows > 128 && L->shape < 3 ? 2 : 1;           // (16 sequences of 4000, 40 rows of 128 entries: 54 us with tiles of rows that do not exist, 38 without)
    const int each = 128 * L->tiles;
    L->row_tiles = (int)((rows + each - 1) / each);
    const long long tiles = (long long)s->batch * c->kv_heads * L->row_tiles;
    // Keys are shared out where that is expected to pay: waves of CTAs x (their tiles of keys, and what a CTA does once), and the pieces through memory (ns, from the cases below).  us with
    // one share / with what the rule takes: 700 queries of 32 heads over 8 behind 7300 tokens 161 / 131 (three shares), 3 x 777 of 16 heads of 64 over 4, 4000 tokens, 127 / 114; with one,
    // which the rule takes / with two: 2048 queries of 16 heads behind 3952 tokens 137 / 160, 1500 of 24 heads behind 1500 74 / 90, 500 queries of 64 heads over 8, two sequences of 3000
    // tokens, 134 / 181.  A table that has room for more than its sequence is priced as if that were there: 2048 tokens of 32 heads over 8 take 64 us, 159 behind a table for 32768.
    const int tile = L->shape == 3 ? 3500 : L->tiles == 2 ? 2400 : 1800, group = heads / c->kv_heads, cols = kShapes[L->shape][1] + 2;
    const long long seen = window ? std::min(keys, (long long)window + each / group + keep_first + kv8::kTile) : keys, key_tiles = std::max(1ll, (seen + kv8::kTile - 1) / kv8::kTile);
    long long best = -1;
    for (long long n = 1; n <= std::min(key_tiles, std::max(4ll, sms / tiles)); n += std::max(1ll, n / 8)) {
      const long long ns = (tiles * n + sms - 1) / sms * ((key_tiles + n - 1) / n * tile + 10000) + (n > 1 ? 3000 + tiles * n * each * cols * 8 / 5000 : 0);
      if (best < 0 || ns < best) { best = ns; L->shares = (int)n; }
    }
    L->bytes = L->shares > 1 ? (size_t)tiles * L->shares * each * cols * sizeof(float) : 0;
    return 0;
  }
  L->tiles = rows <= 8 ? 1 : rows <= 16 || L->shape == 3 ? 2 : 3;       // (tiles of 8 queries; 256 entries: the results of two fill the registers)
  L->row_tiles = (int)((rows + 8 * L->tiles - 1) / (8 * L->tiles));
  const int unit = kv8::kWarps * kv8::step_of(kShapes[L->shape][1]);
  const long long units = (long long)s->batch * c->kv_heads * L->row_tiles * ((keys + unit - 1) / unit + 1);
  // A cluster to each (sequence, head, tile) where its CTAs have at most four units each: one launch, no workspace.  Otherwise the line: any number of CTAs to a head, whatever the lengths.
  // us by clusters / by the line, 128 entries, a token of 16 heads over 4: one sequence of 1000 tokens 8.7 / 9.2, of 4000 11.2 / 11.2, of 8000 (eight units) 16.6 / 15.5, 8 of 4000
  // 13.9 / 15.1, 16 with a window of 1024 10.0 / 10.9, 18 of 4000 (288 CTAs: clusters do not find all places) 33 / 21.
  const long long each = (long long)s->batch * c->kv_heads * L->row_tiles, most = window ? std::min(keys, (long long)window + s->rows + keep_first) : keys, longest = (most + unit - 1) / unit + (window ? 2 : 0);
  for (int k = 8; k >= 2 && !L->cluster; k /= 2)
    if (each * k <= 7 * sms / 4 && longest <= 4 * k) L->cluster = k;
  if (L->cluster) { L->ctas = (int)each * L->cluster; L->bytes = 0; return 0; }
  L->ctas = (int)std::min<long long>(2 * sms, std::max<long long>(1, units));
  L->bytes = (size_t)2 * L->ctas * L->tiles * (kShapes[L->shape][1] / 16 * 128 + 16) * sizeof(float);
  return 0;
}
template <int DK, int DV, int QT> int attend_as(const kv8::Attn& P, const Layout& L, int device, cudaStream_t stream) {
  if (L.cluster) {
    CK((allow<kv8::attend_tokens<DK, DV, QT, true>>(device, kv8::attn_smem<DK, DV, QT>())));
    CK(launch_behind(kv8::attend_tokens<DK, DV, QT, true>, dim3(L.ctas), dim3(kv8::kThreads), kv8::attn_smem<DK, DV, QT>(), stream, -L.cluster, P));
    return 0;
  }
  const int smem = kv8::attn_smem<DK, DV, QT>() + 8 + 8 * P.S.batch;
  CK((allow<kv8::attend_tokens<DK, DV, QT, false>>(device, kv8::attn_smem<DK, DV, QT>() + 8 + 8 * kv8::kMaxBatch)));
  kv8::attend_tokens<DK, DV, QT, false><<<L.ctas, kv8::kThreads, smem, stream>>>(P);
  CK(cudaGetLastError());
  CK(launch_behind(kv8::join<DV, QT>, dim3(P.C.heads * P.row_tiles, P.S.batch), dim3(QT * DV), 0, stream, 1, P, L.ctas));
  return 0;
}
template <int DK, int DV, int TILES> int attend_portion(const kv8::Attn& A, const Layout& L, int device, cudaStream_t stream) {
  const kv8::Portion P{A, L.shares};
  CK((allow<kv8::attend_rows<DK, DV, TILES>>(device, kv8::rows_smem<DK, DV, TILES>())));
  kv8::attend_rows<DK, DV, TILES><<<dim3(A.C.heads * L.shares, L.row_tiles, A.S.batch), kv8::kRowThreads, kv8::rows_smem<DK, DV, TILES>(), stream>>>(P);
  CK(cudaGetLastError());
  if (L.shares > 1) CK(launch_behind(kv8::join_rows<DV, TILES>, dim3(A.C.heads * (DV / 16), L.row_tiles, A.S.batch), dim3(128 * TILES), 0, stream, 1, P));
  return 0;
}
template <int DK, int DV> int attend_tiles(const kv8::Attn& P, const Layout& L, int device, cudaStream_t stream) {
  if (L.shares) {
    if constexpr (DV < 256) if (L.tiles == 2) return attend_portion<DK, DV, 2>(P, L, device, stream);
    return attend_portion<DK, DV, 1>(P, L, device, stream);
  }
  if (L.tiles == 1) return attend_as<DK, DV, 1>(P, L, device, stream);
  if constexpr (DV < 256) {
    if (L.tiles == 3) return attend_as<DK, DV, 3>(P, L, device, stream);
  }
  return attend_as<DK, DV, 2>(P, L, device, stream);
}
}  // namespace

extern "C" int dsk_kv8_write(const dsk_kv8* c, const dsk_kv8_rows* s, const dsk_view* k, const dsk_view* v, void* stream) {
  if (const int code = check_cache(c, s)) return code;
  const int dt = k ? k->dtype : -1;
  if (dt != DSK_DT_F32 && dt != DSK_DT_F16 && dt != DSK_DT_BF16) return fail(-4, "dsk_kv8_write: keys and values are F32, F16 or BF16");
  if (!s->batch || !s->rows) return 0;
  if (const int code = check_view("keys", k, dt)) return code;
  if (const int code = check_view("values", v, dt)) return code;
  OnDevice on(c->device);
  CK(on.error);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dt == DSK_DT_F32 ? write_as<float>(c, s, k, v, st) : dt == DSK_DT_F16 ? write_as<__half>(c, s, k, v, st) : write_as<__nv_bfloat16>(c, s, k, v, st);
}

extern "C" int dsk_kv8_read(const dsk_kv8* c, const dsk_kv8_rows* s, const dsk_view* k, const dsk_view* v, void* stream) {
  if (const int code = check_cache(c, s)) return code;
  const int dt = k ? k->dtype : -1;
  if (dt != DSK_DT_F32 && dt != DSK_DT_F16 && dt != DSK_DT_BF16) return fail(-4, "dsk_kv8_read: keys and values are F32, F16 or BF16");
  if (!s->batch || !s->rows) return 0;
  if (const int code = check_view("keys", k, dt)) return code;
  if (const int code = check_view("values", v, dt)) return code;
  OnDevice on(c->device);
  CK(on.error);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dt == DSK_DT_F32 ? read_as<float>(c, s, k, v, st) : dt == DSK_DT_F16 ? read_as<__half>(c, s, k, v, st) : read_as<__nv_bfloat16>(c, s, k, v, st);
}

extern "C" int dsk_kv8_attn_workspace(const dsk_kv8* c, const dsk_kv8_rows* s, int heads, int window, int keep_first, size_t* bytes) {
  if (!bytes) return fail(-1, "bad arguments");
  if (const int code = check_cache(c, s)) return code;
  Layout L{};
  if (const int code = layout_of(c, s, heads, window, keep_first, &L)) return code;
  *bytes = L.bytes;
  return 0;
}

extern "C" int dsk_kv8_attn(const dsk_kv8* c, const dsk_kv8_rows* s, const dsk_view* q, const dsk_view* out, int heads, float scale, int window, int keep_first, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (const int code = check_cache(c, s)) return code;
  const int dt = q ? q->dtype : -1;
  if (dt != DSK_DT_F16 && dt != DSK_DT_BF16) return fail(-4, "dsk_kv8_attn: queries are F16 or BF16");
  if (!(std::fabs(scale) < INFINITY)) return fail(-4, "dsk_kv8_attn: the scale is not a number");
  if (window < 0 || keep_first < 0) return fail(-4, "window %d and keep_first %d must not be negative", window, keep_first);
  if (heads <= 0 || heads % c->kv_heads) return fail(-4, "%d query heads over %d key heads: a multiple is needed", heads, c->kv_heads);
  if (!s->batch || !s->rows) return 0;
  if (const int code = check_view("queries", q, dt)) return code;
  if (const int code = check_view("output", out, dt)) return code;
  Layout L{};
  if (const int code = layout_of(c, s, heads, window, keep_first, &L)) return code;
  if (L.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < L.bytes)) return fail(-1, "dsk_kv8_attn: a workspace of %zu bytes is needed, 16-byte aligned (%zu given)", L.bytes, workspace_bytes);
  OnDevice on(c->device);
  CK(on.error);
  kv8::Attn P;
  P.C = cache_of(c); P.S = rows_of(s);
  P.q = q->data; P.out = out->data; P.pq = pitch_of(q); P.po = pitch_of(out);
  P.heads = heads; P.group = heads / c->kv_heads; P.row_tiles = L.row_tiles; P.bf16 = dt == DSK_DT_BF16; P.wide_q = wide(q); P.wide_o = wide(out);
  P.window = window_of(window); P.keep = keep_first;
  P.scale = scale * 1.44269504088896340736f;
  P.part = static_cast<float*>(workspace);
  P.cluster = L.cluster;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (L.shape) {
    case 0: return attend_tiles<64, 64>(P, L, c->device, st);
    case 1: return attend_tiles<128, 128>(P, L, c->device, st);
    case 2: return attend_tiles<192, 128>(P, L, c->device, st);
    default: return attend_tiles<256, 256>(P, L, c->device, st);
  }
}

static int check_verify(const dsk_verify_args* a) {
  if (!a) return fail(-1, "null arguments");
  if (a->batch < 0 || a->batch > 65535 || a->drafts < 0 || a->drafts > verify::kMaxDrafts || a->vocab <= 0 || a->vocab > (1 << 20))
    return fail(-4, "batch %d (at most 65535), %d drafts (at most %d), vocabulary %d (at most 2^20)", a->batch, a->drafts, verify::kMaxDrafts, a->vocab);
  return 0;
}
static int pieces_of(const dsk_verify_args* a) { return (a->vocab + verify::kPiece - 1) / verify::kPiece; }

extern "C" int dsk_verify_workspace(const dsk_verify_args* a, size_t* bytes) {
  if (!bytes) return fail(-1, "bad arguments");
  if (const int code = check_verify(a)) return code;
  *bytes = (size_t)a->batch * (a->drafts + 1) * pieces_of(a) * sizeof(float2);
  return 0;
}

template <typename T> static int verify_as(const verify::Params& P, cudaStream_t stream) {
  verify::row_stats<T><<<dim3((P.pieces + verify::kStatWarps - 1) / verify::kStatWarps, P.n + 1, P.batch), verify::kStatThreads, 0, stream>>>(P);
  CK(cudaGetLastError());
  CK(launch_behind(verify::pick<T>, dim3(P.batch * P.cluster), dim3(verify::kThreads), 0, stream, P.cluster, P));
  return 0;
}

extern "C" int dsk_verify(const dsk_verify_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int code = check_verify(a)) return code;
  if (a->logits_dtype != DSK_DT_F32 && a->logits_dtype != DSK_DT_F16 && a->logits_dtype != DSK_DT_BF16) return fail(-4, "dsk_verify: logits are F32, F16 or BF16");
  if (!(a->temperature >= 0.f && a->temperature < INFINITY)) return fail(-4, "temperature must be >= 0");
  if (a->temperature > 0.f && a->temperature < 0x1p-120f) return fail(-4, "a temperature of %g: 0 or at least 2^-120 is needed", (double)a->temperature);   // (64 log2(e) / temperature is an fp32 number)
  if (!a->batch) return 0;
  if (!a->logits || !a->coins || !a->accepted || !a->tokens || (a->drafts && !a->draft_tokens)) return fail(-1, "dsk_verify: null memory");
  size_t need = 0;
  if (const int code = dsk_verify_workspace(a, &need)) return code;
  if (!workspace || !aligned(workspace, 8) || workspace_bytes < need) return fail(-1, "dsk_verify: a workspace of %zu bytes is needed, 8-byte aligned (%zu given)", need, workspace_bytes);
  if (!aligned(a->logits, size_of(a->logits_dtype)) || !aligned(a->draft_probs, 4) || !aligned(a->draft_tokens, 4) || !aligned(a->count, 4) || !aligned(a->coins, 4) || !aligned(a->accepted, 4) || !aligned(a->tokens, 4)) return fail(-1, "dsk_verify: memory is not aligned to its element");
  if (const int code = check_device(a->device)) return code;
  OnDevice on(a->device);
  CK(on.error);
  verify::Params P;
  const int size = size_of(a->logits_dtype);
  P.logits = a->logits; P.l_batch = a->logits_batch; P.l_row = a->logits_row;
  P.probs = a->draft_probs; P.p_batch = a->probs_batch; P.p_row = a->probs_row;
  P.drafts = a->draft_tokens; P.count = a->count; P.coins = a->coins; P.part = static_cast<float2*>(workspace); P.accepted = a->accepted; P.tokens = a->tokens;
  P.batch = a->batch; P.n = a->drafts; P.vocab = a->vocab; P.pieces = pieces_of(a);
  P.wide_l = aligned(a->logits, 4 * size) && a->logits_batch % 4 == 0 && a->logits_row % 4 == 0;
  P.wide_p = aligned(a->draft_probs, 16) && a->probs_batch % 4 == 0 && a->probs_row % 4 == 0;
  P.slope = a->temperature == 0.f ? 0.0 : 1.44269504088896340736 / (double)a->temperature;
  P.cluster = 8;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->logits_dtype == DSK_DT_F32 ? verify_as<float>(P, st) : a->logits_dtype == DSK_DT_F16 ? verify_as<__half>(P, st) : verify_as<__nv_bfloat16>(P, st);
}
