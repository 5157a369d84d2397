// dsk_packed.cu — C-ABI (include/dsk.h) of the operators on packed rows, several sequences one behind the other: places in a cache for tokens that join (and blocks that come
// back), packed rows into the 8-bit cache, attention of whole prompts.  As in dsk_serve.cu nothing is allocated, waited for or kept.

#include "dsk_serve_host.cuh"

#include <algorithm>
#include <cstring>

#include "dsk_blocks.cuh"
#include "dsk_prompt.cuh"

namespace {
constexpr int kMaxRows = 1 << 20;

int check_pool(const dsk_blocks* p, const int32_t* table, int64_t pitch, int table_blocks, int batch) {
  if (!p) return fail(-1, "null blocks");
  if (p->block != 16 && p->block != 32 && p->block != 64 && p->block != 128) return fail(-4, "blocks of %d tokens: 16, 32, 64 or 128 are supported", p->block);
  if (p->n_blocks <= 0 || p->n_blocks > INT32_MAX / p->block) return fail(-4, "%d blocks of %d tokens: at least one, and less than 2^31 tokens", p->n_blocks, p->block);
  if (batch < 0 || batch > blocks::kMaxBatch) return fail(-4, "%d sequences: at most %d a call", batch, blocks::kMaxBatch);
  if (table_blocks < 0 || table_blocks > (1 << 30) / p->block) return fail(-4, "tables of %d blocks (2^30 tokens at most)", table_blocks);
  if (batch > 1 && pitch < table_blocks) return fail(-4, "rows of %d blocks %lld apart: they must not overlap", table_blocks, (long long)pitch);
  if (!p->free || !p->n_free) return fail(-1, "blocks: null memory");
  if (!aligned(p->free, 4) || !aligned(p->n_free, 4) || !aligned(p->status, 4)) return fail(-1, "blocks: memory needs 4-byte alignment");
  if (batch && (!table || !aligned(table, 4) || !table_blocks)) return fail(-1, "null, empty or unaligned table");
  return 0;
}
blocks::Pool pool_of(const dsk_blocks* p) { return blocks::Pool{p->free, p->n_free, p->status, p->n_blocks, p->block == 16 ? 4 : p->block == 32 ? 5 : p->block == 64 ? 6 : 7}; }
int check_packed(const dsk_packed* s) {
  if (!s) return fail(-1, "null packed rows");
  if (s->batch < 0 || s->batch > prompt::kMaxBatch || s->rows < 0 || s->rows > kMaxRows) return fail(-4, "%d sequences (at most %d a call) in %d packed rows (at most 2^20)", s->batch, prompt::kMaxBatch, s->rows);
  if (!s->starts || !aligned(s->starts, 4) || !aligned(s->status, 4)) return fail(-1, "packed rows: starts are null or unaligned");
  return 0;
}
int check_pieces(const dsk_packed* s, int block) {
  const int most = std::min(s->rows, s->rows / block + 2 * s->batch);
  if (s->n_pieces < most) return fail(-4, "room for %d pieces where %d rows of %d sequences may have %d", s->n_pieces, s->rows, s->batch, most);
  if (s->n_pieces && (!s->pieces || !aligned(s->pieces, 16))) return fail(-1, "packed rows: pieces are null or not 16-byte aligned");
  return 0;
}
}  // namespace

extern "C" int dsk_blocks_extend(const dsk_blocks* p, int32_t* table, int64_t table_pitch, int table_blocks, const int32_t* lens, const int32_t* count, const dsk_packed* s, void* stream) {
  if (const int code = check_packed(s)) return code;
  if (const int code = check_pool(p, table, table_pitch, table_blocks, s->batch)) return code;
  if (s->block != p->block) return fail(-4, "packed rows for blocks of %d tokens, blocks of %d", s->block, p->block);
  if (const int code = check_pieces(s, p->block)) return code;
  if (s->batch && (!lens || !count || !s->lens || !aligned(lens, 4) || !aligned(count, 4) || !aligned(s->lens, 4))) return fail(-1, "dsk_blocks_extend: lengths or counts are null or unaligned");
  if (s->batch && s->lens < lens + s->batch && lens < s->lens + s->batch) return fail(-1, "dsk_blocks_extend: the new lengths must not lie over the old ones");
  if (s->batch && s->lens < count + s->batch && count < s->lens + s->batch) return fail(-1, "dsk_blocks_extend: the new lengths must not lie over the counts");
  if (s->rows && (!s->positions || !s->slots || !aligned(s->positions, 4) || !aligned(s->slots, 4))) return fail(-1, "dsk_blocks_extend: positions or slots are null or unaligned");
  if (const int code = check_device(p->device)) return code;
  if (s->device != p->device) return fail(-1, "packed rows on device %d, blocks on %d", s->device, p->device);
  OnDevice on(p->device);
  CK(on.error);
  blocks::Extend A;
  A.P = pool_of(p);
  A.table = table; A.pitch = table_pitch; A.lens = lens; A.count = count;
  A.starts = s->starts; A.lens_out = s->lens; A.positions = s->positions; A.slots = s->slots; A.pieces = reinterpret_cast<int4*>(s->pieces);
  A.table_blocks = table_blocks; A.batch = s->batch; A.rows = s->rows; A.n_pieces = s->n_pieces;
  const int ctas = std::max(1, std::min(148, (s->rows + 4 * blocks::kThreads - 1) / (4 * blocks::kThreads)));
  blocks::extend<<<ctas, blocks::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(A);
  CK(cudaGetLastError());
  return 0;
}

extern "C" int dsk_blocks_cut(const dsk_blocks* p, int32_t* table, int64_t table_pitch, int table_blocks, const int32_t* lens, const int32_t* keep, int batch, void* stream) {
  if (const int code = check_pool(p, table, table_pitch, table_blocks, batch)) return code;
  if (!batch) return 0;
  if (!lens || !keep || !aligned(lens, 4) || !aligned(keep, 4)) return fail(-1, "dsk_blocks_cut: lengths are null or unaligned");
  if (const int code = check_device(p->device)) return code;
  OnDevice on(p->device);
  CK(on.error);
  const blocks::Cut A{pool_of(p), table, table_pitch, lens, keep, table_blocks, batch};
  if ((long long)batch * table_blocks > INT32_MAX) blocks::cut<true><<<1, blocks::kCutThreads, 0, static_cast<cudaStream_t>(stream)>>>(A);
  else blocks::cut<false><<<1, blocks::kCutThreads, 0, static_cast<cudaStream_t>(stream)>>>(A);
  CK(cudaGetLastError());
  return 0;
}

namespace {
template <typename T> int write_few(const dsk_kv8* c, const kv8::Pieces& at, dim3 grid, const dsk_view* k, const dsk_view* v, cudaStream_t stream) {
  const T *pk = static_cast<const T*>(k->data), *pv = static_cast<const T*>(v->data);
  if (wide(k) && wide(v)) kv8::write_few<T, true><<<grid, 64, 0, stream>>>(cache_of(c), at, pk, pv, pitch_of(k), pitch_of(v));
  else kv8::write_few<T, false><<<grid, 64, 0, stream>>>(cache_of(c), at, pk, pv, pitch_of(k), pitch_of(v));
  CK(cudaGetLastError());
  return 0;
}
}  // namespace

extern "C" int dsk_kv8_append(const dsk_kv8* c, const dsk_packed* s, const dsk_view* k, const dsk_view* v, void* stream) {
  if (const int code = check_cache(c)) return code;
  if (const int code = check_packed(s)) return code;
  if (s->block != c->block) return fail(-4, "packed rows for blocks of %d tokens, a cache of %d", s->block, c->block);
  if (const int code = check_pieces(s, c->block)) return code;
  const int dt = k ? k->dtype : -1;
  if (dt != DSK_DT_F32 && dt != DSK_DT_F16 && dt != DSK_DT_BF16) return fail(-4, "dsk_kv8_append: keys and values are F32, F16 or BF16");
  if (!s->batch || !s->rows) return 0;
  if (const int code = check_view("keys", k, dt)) return code;
  if (const int code = check_view("values", v, dt)) return code;
  if (const int code = check_device(c->device)) return code;
  if (s->device != c->device) return fail(-1, "packed rows on device %d, a cache on %d", s->device, c->device);
  OnDevice on(c->device);
  CK(on.error);
  const kv8::Pieces at{reinterpret_cast<const int4*>(s->pieces), s->rows};
  const dim3 grid(s->n_pieces, 2 * c->kv_heads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Fewer than 32 rows to a sequence, and blocks that take more than a warp or two: 64 threads read their values twice (211 sequences of one token, 8 heads of 192 + 128, blocks of 128: 4.9 us where a
  // CTA with registers for the whole block takes 26; 200 of one and one of 2000: 16 for 33; 100 of 32: 9.1 for 20.5; but 31 of one and one of 1000, 32 on average: 9.8 for 8.6)
  if (s->rows / s->batch < 32 && std::min(s->rows, c->block) * std::max(c->dim_k, c->dim_v) / 8 > 512)
    return dt == DSK_DT_F32 ? write_few<float>(c, at, grid, k, v, st) : dt == DSK_DT_F16 ? write_few<__half>(c, at, grid, k, v, st) : write_few<__nv_bfloat16>(c, at, grid, k, v, st);
  return write_all(c, at, grid, std::min(s->rows, c->block), k, v, st);
}

namespace {
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) { cudaGetLastError(); p = nullptr; }
    return (EncodeTiledFn)p;
  }();
  return fn;
}
// [row][head][entry] of 16-bit entries, copied in boxes of 64 entries of box_heads heads of box_rows rows (what lies outside reads as zeros)
int rows_map(CUtensorMap* m, const char* what, const dsk_view* v, int dim, int heads, int rows, int box_heads, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? v->head * 2 : 16), (cuuint64_t)(rows > 1 ? v->row * 2 : 16)};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows}, one[3] = {1, 1, 1};
  const CUresult r = encode_tiled()(m, v->dtype == DSK_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, v->data, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : fail(-4, "%s: no tensor map for %d rows of %d heads of %d entries, rows %lld and heads %lld entries apart (error %d)", what, rows, heads, dim, (long long)v->row, (long long)v->head, (int)r);
}
// rows that tensor-map copies can read: 16-byte pieces
int check_rows(const char* what, const dsk_view* v, int heads, int rows) {
  if (!aligned(v->data, 16)) return fail(-4, "%s: memory needs 16-byte alignment", what);
  for (const auto& d : {std::pair<int, int64_t>{heads, v->head}, {rows, v->row}})
    if (d.first > 1 && (d.second <= 0 || d.second % 8 || d.second >= (1ll << 39))) return fail(-4, "%s: rows and heads must lie a positive multiple of 8 entries apart, got %lld and %lld", what, (long long)v->row, (long long)v->head);
  return 0;
}
template <int DK, int DV, bool BF16, int JOINT> int attend_as(const prompt::Params& P, int ctas, int device, cudaStream_t stream) {
  static std::atomic<int> registers{0};                      // of a thread at launch: what its warps give and take adds up to that, or they wait for good
  if (registers.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes at{};
    CK((cudaFuncGetAttributes(&at, prompt::attend_packed<DK, DV, BF16, JOINT>)));
    registers.store(at.numRegs, std::memory_order_relaxed);
  }
  if (registers.load(std::memory_order_relaxed) != 65536 / prompt::kThreads) return fail(-2, "dsk_packed_attn: built with %d registers a thread where %d are needed", registers.load(), 65536 / prompt::kThreads);
  CK((allow<prompt::attend_packed<DK, DV, BF16, JOINT>>(device, prompt::smem_bytes<DK, DV>())));
  prompt::attend_packed<DK, DV, BF16, JOINT><<<ctas, prompt::kThreads, prompt::smem_bytes<DK, DV>(), stream>>>(P);
  CK(cudaGetLastError());
  return 0;
}
template <int DK, int DV> int attend_as(const prompt::Params& P, bool bf16, bool joint, int ctas, int device, cudaStream_t stream) {
  if constexpr (prompt::tiles<DK, DV>() == 2)
    if (joint) return bf16 ? attend_as<DK, DV, true, 1>(P, ctas, device, stream) : attend_as<DK, DV, false, 1>(P, ctas, device, stream);
  return bf16 ? attend_as<DK, DV, true, 0>(P, ctas, device, stream) : attend_as<DK, DV, false, 0>(P, ctas, device, stream);
}
}  // namespace

extern "C" int dsk_packed_attn(const dsk_packed* s, const dsk_view* q, const dsk_view* k, const dsk_view* v, const dsk_view* out, int heads, int kv_heads, int dim_k, int dim_v, float scale,
                               int window, int keep_first, void* stream) {
  if (const int code = check_packed(s)) return code;
  const int dt = q ? q->dtype : -1;
  if (dt != DSK_DT_F16 && dt != DSK_DT_BF16) return fail(-4, "dsk_packed_attn: queries, keys and values are F16 or BF16");
  for (int d : {dim_k, dim_v})
    if (d <= 0 || d % 16 || d > 256) return fail(-4, "heads of %d entries: a multiple of 16 up to 256 is needed", d);
  if (kv_heads <= 0 || heads <= 0 || heads > 32767 || heads % kv_heads) return fail(-4, "%d query heads over %d key heads: a multiple is needed, at most 32767", heads, kv_heads);
  if (!(scale >= 0.f && scale < INFINITY)) return fail(-4, "dsk_packed_attn: the scale must be a number that is not negative");
  if (window < 0 || keep_first < 0) return fail(-4, "window %d and keep_first %d must not be negative", window, keep_first);
  if (!s->batch || !s->rows) return 0;
  for (const auto& x : {std::pair<const char*, const dsk_view*>{"queries", q}, {"keys", k}, {"values", v}, {"output", out}})
    if (const int code = check_view(x.first, x.second, dt)) return code;
  if (const int code = check_rows("queries", q, heads, s->rows)) return code;
  if (const int code = check_rows("keys", k, kv_heads, s->rows)) return code;
  if (const int code = check_rows("values", v, kv_heads, s->rows)) return code;
  if (const int code = check_device(s->device)) return code;
  if (!encode_tiled()) return fail(-2, "the driver has no cuTensorMapEncodeTiled");
  OnDevice on(s->device);
  CK(on.error);
  prompt::Params P;
  P.group = heads / kv_heads;
  // Heads of a row tile, a divisor of the group: with more of them a tile has fewer tokens, whose keys end close together, and short prompts make fewer pieces.  The most that fill all 128 rows,
  // if those are four or more; else the most that leave at most 8 of them empty (us, packed / a head by itself or in pairs: 7 heads, 222 prompts of 60 tokens 35 / 86, 8192 tokens 211 / 210; 3: 18 / 34,
  // 119 / 122; 6: 28 / 40, 178 / 174; 12 in fours 30, 170, all together 27, 180)
  P.pack = 1;
  for (int n = 2; n <= std::min(P.group, 128); n++)
    if (P.group % n == 0 && 128 % n == 0) P.pack = n;
  if (P.pack < 4)
    for (int n = P.pack + 1; n <= std::min(P.group, 128); n++)
      if (P.group % n == 0 && 128 % n <= 8) P.pack = n;
  P.tokens = 128 / P.pack; P.subs = P.group / P.pack; P.units = kv_heads * P.subs;
  // Key heads that are worked on at a time: those whose keys and values take half of the L2, so that later rows find there what earlier ones read (32 heads of 192 + 128 entries, 22508 rows:
  // 870 us with all at a time, at 1420 MHz under the power limit; 774 with 4, 789 with 8); with fewer than that the last ones leave gaps (16 heads of 128, 8192 rows: 147 with all, 150 with 4)
  P.span = (int)std::max<long long>(1, std::min<long long>(kv_heads, (64ll << 20) / (2ll * s->rows * (dim_k + dim_v)))) * P.subs;
  constexpr int kShapes[4][2] = {{64, 64}, {128, 128}, {192, 128}, {256, 256}};
  int shape = 0;
  while (dim_k > kShapes[shape][0] || dim_v > kShapes[shape][1]) shape++;
  if (const int code = rows_map(&P.q, "queries", q, dim_k, heads, s->rows, P.pack, P.tokens)) return code;
  if (const int code = rows_map(&P.k, "keys", k, dim_k, kv_heads, s->rows, 1, prompt::kTile)) return code;
  if (const int code = rows_map(&P.v, "values", v, dim_v, kv_heads, s->rows, 1, prompt::kTile)) return code;
  P.starts = s->starts; P.status = s->status;
  P.values = v->data; P.v_row = v->row; P.v_head = v->head;
  P.out = out->data; P.o_row = out->row; P.o_head = out->head;
  P.wide_o = aligned(out->data, 32) && out->row % 16 == 0 && out->head % 16 == 0 ? 2 : aligned(out->data, 16) && out->row % 8 == 0 && out->head % 8 == 0;
  P.rows = s->rows; P.batch = s->batch; P.dk = dim_k; P.dv = dim_v;
  P.window = window >= s->rows ? 0 : window; P.keep = keep_first;
  // Positive, so that -inf stays what it is: scale 0 becomes the smallest number there is, 2^-149, with which no finite score reaches 2^-21.  By its bits: a host that takes such numbers for zero gives no
  // other way
  P.f = scale * 1.44269504088896340736f;
  uint32_t bits;
  std::memcpy(&bits, &P.f, 4);
  if (!(bits & 0x7fffffffu)) bits = 1;
  std::memcpy(&P.f, &bits, 4);
  // Few pieces: both row tiles of a CTA have the same rows, each every second tile of its keys, so that the longest walk takes half the time and there are twice the pieces.  Where pieces of two row
  // tiles would not fill the GPU (one prompt of 8192 tokens, 4 heads over 1: 69 us for 115; 20 prompts of 60, 16 over 4: 11.2 for 10.4); beyond, keys and values are read twice as often (four
  // prompts of 4096 tokens: 73 us for 65).  By rows alone, what a captured call has to spare among them: one prompt of 9600 tokens, 4 heads over 1, takes 147 us where 9472 take 84
  const bool joint = shape != 3 && s->rows / (2ll * P.tokens) * P.units <= multiprocessors(s->device);
  const int tokens = P.tokens * (shape == 3 || joint ? 1 : 2);
  const long long items = ((long long)s->rows / tokens + std::min(s->batch, s->rows)) * P.units;   // at most, whatever the lengths
  if (items > INT32_MAX) return fail(-4, "%lld pieces of work: at most 2^31", items);
  const int ctas = (int)items;                               // (those that are running take over the others)
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = dt == DSK_DT_BF16;
  switch (shape) {
    case 0: return attend_as<64, 64>(P, bf16, joint, ctas, s->device, st);
    case 1: return attend_as<128, 128>(P, bf16, joint, ctas, s->device, st);
    case 2: return attend_as<192, 128>(P, bf16, joint, ctas, s->device, st);
    default: return attend_as<256, 256>(P, bf16, joint, ctas, s->device, st);
  }
}
