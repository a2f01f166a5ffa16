// C ABI of the batch-serving operators: the paged 8-bit K/V cache (block tables, append, read back,
// attention) and the token scorer. Device pointers and a stream from the caller, no allocation.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "attention_q8.cuh"
#include "attention_q8_tiles.cuh"
#include "capi_common.h"
#include "kvcache.cuh"
#include "logprobs.cuh"

using namespace drt;

namespace {

template <typename... P, typename... Args>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl ? attr : nullptr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// SM count of the current device; 0 with an error recorded.
int current_sms(int* device) {
  static std::atomic<int> cache[64];
  if (cudaGetDevice(device) != cudaSuccess || *device < 0 || *device >= 64) return 0;
  int n = cache[*device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *device) != cudaSuccess) return 0;
    cache[*device].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Allows Kernel its dynamic shared memory on the current device (the attribute is per device).
template <auto Kernel>
cudaError_t allow_smem(int device, size_t bytes) {
  static std::atomic<uint64_t> done{0};
  if (done.load(std::memory_order_acquire) >> device & 1) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess) done.fetch_or(1ull << device, std::memory_order_release);
  return e;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool block_ok(int b) { return b == 16 || b == 32 || b == 64 || b == 128; }

}  // namespace

// ======================================================================= block tables and slot maps
extern "C" int drt_cache_plan(const int32_t* start, const int32_t* count, const int32_t* held_in, int32_t* held_out,
                              int32_t requests, int32_t* tables, int64_t ld_tables, int32_t width, int32_t block,
                              int32_t* ring, int32_t ring_size, const int32_t* ring_in, int32_t* ring_out,
                              int32_t* row_start, int32_t* slots, int32_t* positions, int32_t max_rows, int32_t* lengths,
                              int32_t* status, void* stream) {
  REQUIRE(requests >= 0 && requests <= (1 << 20), "requests outside [0, 2^20]");
  REQUIRE(row_start && ring && ring_in && ring_out && status, "null argument");
  REQUIRE(requests == 0 || (start && count && held_in && held_out && tables && lengths), "null argument");
  REQUIRE(max_rows >= 0 && (max_rows == 0 || (slots && positions)), "max_rows needs slots and positions");
  REQUIRE(block >= 1 && width >= 1 && ld_tables >= width, "bad table geometry");
  REQUIRE(static_cast<int64_t>(width) * block <= INT32_MAX, "a request's tokens exceed 2^31 - 1");
  REQUIRE(ring_size >= 1, "the ring needs a capacity");
  PlanArgs a;
  memset(&a, 0, sizeof(a));
  a.start = start;
  a.count = count;
  a.held_in = held_in;
  a.held_out = held_out;
  a.requests = requests;
  a.tables = tables;
  a.ld_tables = ld_tables;
  a.width = width;
  a.block = block;
  a.ring = ring;
  a.ring_size = ring_size;
  a.ring_in = ring_in;
  a.ring_out = ring_out;
  a.row_start = row_start;
  a.slots = slots;
  a.positions = positions;
  a.max_rows = max_rows;
  a.lengths = lengths;
  a.status = status;
  // A token a request: the thread that plans a request writes its slot too (64 requests: 4.9 us in one launch, 6.2 in
  // two). More: one CTA would write them all, so a second launch does (64 x 8 rows: 13.1 us in one, 7.4 in two).
  a.fill_slots = max_rows <= requests;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CK(launch(plan_cache_kernel, dim3(1), dim3(kPlanThreads), 0, st, false, a));
  if (!a.fill_slots)
    CK(launch(plan_slots_kernel, dim3((max_rows + kPlanSlotRows - 1) / kPlanSlotRows), dim3(256), 0, st, true, a));
  return DRT_OK;
}

// ======================================================================= append and read back
namespace {
int check_cache(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale, int64_t blocks,
                int32_t heads, int32_t block, int32_t dim, int32_t code) {
  REQUIRE(k_cache && v_cache && k_scale && v_scale, "null argument");
  REQUIRE(blocks >= 1 && heads >= 1 && heads <= 65535, "bad cache geometry");
  REQUIRE(block_ok(block), "a block holds 16, 32, 64 or 128 tokens (got %d)", block);
  REQUIRE(blocks * block <= INT32_MAX, "slots exceed 2^31 - 1");
  if (dim != 64 && dim != 128) return set_error(DRT_UNSUPPORTED, "head dim %d: 64 and 128 are served", dim);
  REQUIRE(code == DRT_CODE_INT8 || code == DRT_CODE_E4M3, "unknown code type %d", code);
  REQUIRE(aligned16(k_cache) && aligned16(v_cache), "the caches must be 16-byte aligned");
  return DRT_OK;
}

template <typename T, int kDim, int kCode>
cudaError_t run_append(const AppendArgs& a, cudaStream_t st) {
  return launch(append_cache_kernel<T, kDim, kCode>, dim3((a.rows + a.group - 1) / a.group, a.heads, 2), dim3(kAppendThreads),
                0, st, false, a);
}
template <typename T, int kDim, int kCode>
cudaError_t run_read(const ReadArgs& a, cudaStream_t st) {
  return launch(read_cache_kernel<T, kDim, kCode>, dim3((a.rows + kReadRows - 1) / kReadRows, a.heads), dim3(kReadThreads), 0,
                st, false, a);
}
}  // namespace

#define DRT_DISPATCH_DIM_CODE(fn, T, ...)                                                      \
  (dim == 128 ? (code == DRT_CODE_INT8 ? fn<T, 128, CACHE_INT8>(__VA_ARGS__) : fn<T, 128, CACHE_E4M3>(__VA_ARGS__)) \
              : (code == DRT_CODE_INT8 ? fn<T, 64, CACHE_INT8>(__VA_ARGS__) : fn<T, 64, CACHE_E4M3>(__VA_ARGS__)))

extern "C" int drt_cache_append(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                                int32_t dtype, int32_t rows, const int32_t* slots, void* k_cache, void* v_cache,
                                float* k_scale, float* v_scale, int64_t blocks, int32_t heads, int32_t block, int32_t dim,
                                int32_t code, void* stream) {
  REQUIRE(rows >= 0, "rows must be >= 0");
  TRY(check_cache(k_cache, v_cache, k_scale, v_scale, blocks, heads, block, dim, code));
  REQUIRE(dtype == DRT_TYPE_BF16 || dtype == DRT_TYPE_F16, "k and v must be bf16 or f16");
  if (rows == 0) return DRT_OK;
  REQUIRE(k && v && slots, "null argument");
  AppendArgs a;
  memset(&a, 0, sizeof(a));
  a.k = k;
  a.v = v;
  a.k_row = k_row;
  a.k_head = k_head;
  a.v_row = v_row;
  a.v_head = v_head;
  a.slots = slots;
  a.rows = rows;
  a.heads = heads;
  a.block = block;
  a.group = rows <= kAppendFewRows ? kAppendThreads / 32 : kAppendGroup;
  a.blocks = blocks;
  a.k_cache = static_cast<uint8_t*>(k_cache);
  a.v_cache = static_cast<uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.vec = aligned16(k) && aligned16(v) && (k_row | k_head | v_row | v_head) % 8 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CK(dtype == DRT_TYPE_BF16 ? DRT_DISPATCH_DIM_CODE(run_append, __nv_bfloat16, a, st)
                            : DRT_DISPATCH_DIM_CODE(run_append, __half, a, st));
  return DRT_OK;
}

extern "C" int drt_cache_read(const int32_t* slots, int32_t rows, const void* k_cache, const void* v_cache,
                              const float* k_scale, const float* v_scale, int64_t blocks, int32_t heads, int32_t block,
                              int32_t dim, int32_t code, void* k_out, void* v_out, int32_t dtype, void* stream) {
  REQUIRE(rows >= 0, "rows must be >= 0");
  TRY(check_cache(k_cache, v_cache, k_scale, v_scale, blocks, heads, block, dim, code));
  REQUIRE(dtype == DRT_TYPE_BF16 || dtype == DRT_TYPE_F16 || dtype == DRT_TYPE_F32, "values are read as bf16, f16 or f32");
  if (rows == 0) return DRT_OK;
  REQUIRE(slots && k_out && v_out, "null argument");
  REQUIRE(aligned16(k_out) && aligned16(v_out), "the outputs must be 16-byte aligned");
  ReadArgs a;
  memset(&a, 0, sizeof(a));
  a.slots = slots;
  a.rows = rows;
  a.heads = heads;
  a.block = block;
  a.blocks = blocks;
  a.k_cache = static_cast<const uint8_t*>(k_cache);
  a.v_cache = static_cast<const uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.k_out = k_out;
  a.v_out = v_out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CK(dtype == DRT_TYPE_BF16  ? DRT_DISPATCH_DIM_CODE(run_read, __nv_bfloat16, a, st)
     : dtype == DRT_TYPE_F16 ? DRT_DISPATCH_DIM_CODE(run_read, __half, a, st)
                             : DRT_DISPATCH_DIM_CODE(run_read, float, a, st));
  return DRT_OK;
}

// ======================================================================= attention over the cache
namespace {
// The kernel over few rows reads a unit's keys once for 8 or 16 rows, the one over many once for up to 256 but no
// faster for one row than for 128. Rows of a kv head against us, 64 requests of 2,048 tokens in int8, 8 kv heads of 128:
//   8: 64 (few), 177 (many)   16: 85, 184   32: 146, 185   64: 256, 190   128: 476, 200
// and one request of 32,768 tokens: 25, 47   32, 49   43, 49   68, 50   119, 55.
constexpr int kFewRows = 32;

constexpr size_t up256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// Lays a call's scratch out from `base` and returns its size: the cut units' parts of every warp and CTA, for the
// launch over few rows (`few`) and the one over many.
size_t attend_scratch(int sms, int dim, uint8_t* base, CacheAttnArgs* few, CacheAttnArgs* many) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base + at;
    at += up256(bytes);
    return p;
  };
  const size_t warp_rows = static_cast<size_t>(sms) * kQrMaxParts;
  few->part = reinterpret_cast<float*>(take(warp_rows * dim * 4));
  few->stat = reinterpret_cast<float4*>(take(warp_rows * 16));
  auto ctas = [&](CacheAttnArgs* a, int tile_rows) {
    const size_t rows = static_cast<size_t>(sms) * 2 * tile_rows;
    a->cta_part = reinterpret_cast<float*>(take(rows * dim * 4));
    a->cta_stat = reinterpret_cast<float4*>(take(rows * 16));
    a->desc = reinterpret_cast<int4*>(take(static_cast<size_t>(sms) * 16));
  };
  ctas(few, kQrMaxRows);
  ctas(many, kQtRows);
  return at;
}

template <typename T, int kDim, int kRows>
cudaError_t run_merge(const CacheAttnArgs& a, int grid, int64_t rows, cudaStream_t st) {
  // two rows to a CTA where the units are so many that most have few parts, else one: a long unit takes the whole CTA
  const int64_t units = (static_cast<int64_t>(a.q_rows) * a.group / kRows + a.requests) * a.heads;
  const int step = units * kQmAlone >= grid ? 2 : 1;
  return launch(cache_attn_merge_kernel<T, kDim, kRows>,
                dim3((grid + kQmWarps - 1) / kQmWarps, static_cast<unsigned>((std::min<int64_t>(rows, kRows) + step - 1) / step)),
                dim3(kQmThreads), 0, st, true, a, grid, step);
}

// rows: the most rows of one kv head's queries in a request; tiles: an upper bound on the key tiles of all units;
// deep: a unit's, 1 if nothing can be cut.
template <typename T, int kDim, int kCode, int kNT>
cudaError_t run_rows_nt(const CacheAttnArgs& a, int device, int sms, int64_t rows, int64_t tiles, int64_t deep, cudaStream_t st) {
  using Cfg = QrCfg<kDim, kNT>;
  const int grid = static_cast<int>(std::min<int64_t>(sms, tiles));
  cudaError_t e = allow_smem<cache_attn_rows_kernel<T, kDim, kCode, kNT>>(device, Cfg::kSmem);
  if (e == cudaSuccess)
    e = launch(cache_attn_rows_kernel<T, kDim, kCode, kNT>, dim3(grid), dim3(Cfg::kThreads), Cfg::kSmem, st, false, a);
  if (e == cudaSuccess && deep > 1) e = run_merge<T, kDim, Cfg::kRows>(a, grid, rows, st);
  return e;
}

template <typename T, int kDim, int kCode>
cudaError_t run_attend(const CacheAttnArgs& few, const CacheAttnArgs& many, int device, int sms, int64_t rows, int64_t width,
                       cudaStream_t st) {
  const int64_t total = static_cast<int64_t>(few.q_rows) * few.group;
  auto tiles = [&](int tile_rows, int64_t deep) { return (total / tile_rows + few.requests) * few.heads * deep; };
  cudaError_t e = cudaSuccess;
  if (few.rows_from <= few.rows_to) {
    // eight rows to a tile where the caller's bound says that a kv head's rows fit, else sixteen
    const int64_t deep = (width + kQrTile - 1) / kQrTile;
    e = rows <= 8 ? run_rows_nt<T, kDim, kCode, 1>(few, device, sms, rows, tiles(8, deep), deep, st)
                  : run_rows_nt<T, kDim, kCode, 2>(few, device, sms, rows, tiles(16, deep), deep, st);
  }
  if (e == cudaSuccess && many.rows_from <= many.rows_to) {
    const int64_t deep = (width + kQtKeys - 1) / kQtKeys;
    const int grid = static_cast<int>(std::min<int64_t>(sms, tiles(kQtRows, deep)));
    e = allow_smem<cache_attn_tiles_kernel<T, kDim, kCode>>(device, QtCfg<kDim>::kSmem);
    if (e == cudaSuccess)
      e = launch(cache_attn_tiles_kernel<T, kDim, kCode>, dim3(grid), dim3(kQtThreads), QtCfg<kDim>::kSmem, st, false, many);
    if (e == cudaSuccess && deep > 1) e = run_merge<T, kDim, kQtRows>(many, grid, rows, st);
  }
  return e;
}
}  // namespace

extern "C" size_t drt_cache_attend_scratch_bytes(int32_t dim) {
  int device = 0;
  const int sms = current_sms(&device);
  CacheAttnArgs a, b;
  return attend_scratch(sms > 0 ? sms : 148, dim, nullptr, &a, &b);
}

extern "C" int drt_cache_attend(const drt_cache_attend_args* p, void* stream) {
  REQUIRE(p, "null argument");
  TRY(check_cache(p->k_cache, p->v_cache, p->k_scale, p->v_scale, p->blocks, p->kv_heads, p->block, p->dim, p->code));
  REQUIRE(p->dtype == DRT_TYPE_BF16 || p->dtype == DRT_TYPE_F16, "q and out must be bf16 or f16");
  REQUIRE(p->heads >= 1 && p->heads % p->kv_heads == 0, "query heads must be a multiple of the K/V heads");
  REQUIRE(p->q_rows >= 0 && p->requests >= 0 && p->requests <= kQrMaxRequests, "requests outside [0, %d]", kQrMaxRequests);
  REQUIRE(static_cast<int64_t>(p->q_rows) * p->heads <= INT32_MAX, "rows times heads exceed 2^31 - 1");
  REQUIRE(p->width >= 1 && p->ld_tables >= p->width && static_cast<int64_t>(p->width) * p->block <= INT32_MAX,
          "bad table geometry");
  REQUIRE(p->mask_block >= 0 && p->mask_block <= (1 << 24), "mask_block outside [0, 2^24]");
  REQUIRE(std::isfinite(p->scale) && p->scale >= 0.0f, "scale must be finite and >= 0");
  if (p->q_rows == 0 || p->requests == 0) return DRT_OK;
  REQUIRE(p->q && p->out && p->tables && p->lengths && p->row_start && p->scratch, "null argument");
  REQUIRE(reinterpret_cast<uintptr_t>(p->out) % 4 == 0 && (p->out_row | p->out_head) % 2 == 0, "out rows must be 4-byte aligned");
  REQUIRE(aligned16(p->scratch), "scratch must be 16-byte aligned");
  int device = 0;
  const int sms = current_sms(&device);
  if (sms == 0) return set_error(DRT_INTERNAL_ERROR, "no current CUDA device");
  CacheAttnArgs a;
  memset(&a, 0, sizeof(a));
  a.q = p->q;
  a.q_row = p->q_row;
  a.q_head = p->q_head;
  a.q_rows = p->q_rows;
  a.k_cache = static_cast<const uint8_t*>(p->k_cache);
  a.v_cache = static_cast<const uint8_t*>(p->v_cache);
  a.k_scale = p->k_scale;
  a.v_scale = p->v_scale;
  a.blocks = p->blocks;
  a.block = p->block;
  a.heads = p->kv_heads;
  a.group = p->heads / p->kv_heads;
  a.tables = p->tables;
  a.ld_tables = p->ld_tables;
  a.width = p->width;
  a.lengths = p->lengths;
  a.row_start = p->row_start;
  a.origin = p->origin;
  a.requests = p->requests;
  a.mask_block = p->mask_block;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.out = p->out;
  a.out_row = p->out_row;
  a.out_head = p->out_head;
  a.lse = p->lse;
  a.vec = aligned16(p->q) && (p->q_row | p->q_head) % 8 == 0;
  a.out_vec = aligned16(p->out) && (p->out_row | p->out_head) % 8 == 0;
  // Rows of one kv head in a request: up to kFewRows go to the kernel for few, the rest to the one for many; either
  // serves any count. One launch where the caller's bound leaves nothing to the other kernel, or where the average is
  // so near the bound that no more than 3 requests in 8 can be small: a launch that finds nothing costs 9 us (32 requests
  // of 8 tokens x 8 heads: 113 us in two, 104 in one), while 64 requests of 2,048 tokens, of which a half (a quarter)
  // have one row and the rest 64, take 313 us in two and 345 in one (with a quarter of one row and the rest 16: 197, 196).
  CacheAttnArgs b = a;
  attend_scratch(sms, p->dim, static_cast<uint8_t*>(p->scratch), &a, &b);
  const int max_rows = p->max_rows > 0 ? std::min(p->max_rows, p->q_rows) : p->q_rows;
  const int64_t rows = static_cast<int64_t>(max_rows) * a.group;
  const int64_t average = static_cast<int64_t>(p->q_rows) * a.group / p->requests;
  const bool only_few = rows <= kFewRows, only_many = !only_few && average * 8 >= rows * 5;
  a.rows_from = only_many ? 1 : 0;
  a.rows_to = only_many ? 0 : only_few ? INT32_MAX : kFewRows;
  b.rows_from = only_few ? 1 : only_many ? 0 : kFewRows + 1;
  b.rows_to = only_few ? 0 : INT32_MAX;
  const int dim = p->dim, code = p->code;
  const int64_t width = static_cast<int64_t>(p->width) * p->block;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CK(p->dtype == DRT_TYPE_BF16 ? DRT_DISPATCH_DIM_CODE(run_attend, __nv_bfloat16, a, b, device, sms, rows, width, st)
                               : DRT_DISPATCH_DIM_CODE(run_attend, __half, a, b, device, sms, rows, width, st));
  return DRT_OK;
}

// ======================================================================= token scores
namespace {
struct LpPlan {
  int segs, slices, per;
};
LpPlan logprob_plan(int rows, int vocab, int type, int sms) {
  const int elem = type == LOGIT_F32 ? 4 : 2;
  const int seg = 4096 / elem;
  LpPlan p;
  p.segs = (vocab + 16 / elem - 1 + seg - 1) / seg;  // a row may begin inside a 16-byte vector
  const int64_t total = static_cast<int64_t>(p.segs) * rows;
  const int64_t want = total / (static_cast<int64_t>(sms) * kLpCtasPerSm);
  p.per = static_cast<int>(std::min<int64_t>(std::max<int64_t>(want, kLpWarps), kLpMaxSliceSegs));
  p.per = std::min(p.per, p.segs);
  p.slices = (p.segs + p.per - 1) / p.per;
  p.per = (p.segs + p.slices - 1) / p.slices;
  return p;
}

template <typename T>
cudaError_t run_logprobs(const LogprobArgs& a, cudaStream_t st) {
  cudaError_t e = launch(logprob_stats_kernel<T>, dim3(static_cast<unsigned>(a.rows) * a.slices), dim3(kLpThreads), 0, st, false, a);
  if (e != cudaSuccess) return e;
  const size_t smem = a.top > 0 ? kLpCands * 8 + static_cast<size_t>(a.segs) * 4 : 0;
  return launch(logprob_finish_kernel<T>, dim3(a.rows), dim3(a.rows <= kLpFinFewRows ? kLpFinFew : kLpFinMany), smem, st, true, a);
}
}  // namespace

extern "C" size_t drt_selector_logprobs_scratch_bytes(int32_t rows, int32_t vocab, int32_t dtype) {
  if (rows <= 0 || vocab <= 0) return 0;
  int device = 0;
  const int sms = current_sms(&device);
  const LpPlan p = logprob_plan(rows, vocab, dtype, sms > 0 ? sms : 148);
  return up256(static_cast<size_t>(rows) * p.slices * 16) + up256(static_cast<size_t>(rows) * p.segs * 4);
}

extern "C" int drt_selector_logprobs(const void* logits, int32_t dtype, int64_t ld, int32_t logit_rows,
                                     const int32_t* row_index, int32_t rows, int32_t vocab, const int32_t* tokens,
                                     double temperature, int32_t exclude_token, int32_t top, void* scratch, float* logprob,
                                     float* entropy, int32_t* rank, int32_t* top_token, float* top_logprob, void* stream) {
  REQUIRE(rows >= 0 && vocab >= 1 && ld >= vocab, "bad selector geometry");
  REQUIRE(logit_rows >= (row_index ? 1 : rows) || rows == 0, "more rows than logits");
  REQUIRE(dtype == DRT_TYPE_F32 || dtype == DRT_TYPE_BF16 || dtype == DRT_TYPE_F16, "logits must be f32, bf16 or f16");
  REQUIRE(top >= 0 && top <= kLpMaxTop, "top must be in [0, %d]", kLpMaxTop);
  REQUIRE(std::isfinite(temperature) && (temperature <= 0.0 || temperature >= 1e-30),
          "temperature must be finite, and at least 1e-30 if positive");
  REQUIRE(exclude_token >= -1 && exclude_token < vocab, "exclude_token outside the vocabulary");
  if (rows == 0) return DRT_OK;
  REQUIRE(logits && scratch && (top == 0 || (top_token && top_logprob)), "null argument");
  REQUIRE(tokens || (!logprob && !rank), "logprob and rank need tokens");
  REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == DRT_TYPE_F32 ? 4 : 2) == 0 && aligned16(scratch),
          "logits or scratch misaligned");
  int device = 0;
  const int sms = current_sms(&device);
  if (sms == 0) return set_error(DRT_INTERNAL_ERROR, "no current CUDA device");
  const LpPlan p = logprob_plan(rows, vocab, dtype, sms);
  REQUIRE(p.segs <= kLpMaxSegs, "rows of at most %d logits", kLpMaxSegs * (dtype == DRT_TYPE_F32 ? 1024 : 2048) - 8);
  REQUIRE(static_cast<int64_t>(rows) * p.slices <= INT32_MAX, "too many rows");
  LogprobArgs a;
  memset(&a, 0, sizeof(a));
  a.logits = logits;
  a.ld = ld;
  a.row_index = row_index;
  a.tokens = tokens;
  a.rows = rows;
  a.logit_rows = logit_rows;
  a.vocab = vocab;
  a.top = top;
  a.exclude = exclude_token;
  a.unit_log2 = static_cast<float>(1.4426950408889634 / (temperature > 0.0 ? temperature : 1.0));
  a.segs = p.segs;
  a.slices = p.slices;
  a.segs_per_slice = p.per;
  a.part = static_cast<float4*>(scratch);
  a.seg_max = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + up256(static_cast<size_t>(rows) * p.slices * 16));
  a.logprob = logprob;
  a.entropy = entropy;
  a.rank = rank;
  a.top_token = top_token;
  a.top_logprob = top_logprob;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CK(dtype == DRT_TYPE_F32    ? run_logprobs<float>(a, st)
     : dtype == DRT_TYPE_BF16 ? run_logprobs<__nv_bfloat16>(a, st)
                              : run_logprobs<__half>(a, st));
  return DRT_OK;
}
