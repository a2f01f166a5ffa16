// Attention over the paged 8-bit K/V cache (kvcache.cuh) for the rows of many requests.
//
//   o_i = sum_j p_ij vs_b(j) v_j,   p_ij = softmax over j < limit(i) of  scale * ks_b(j) <q_i, k_j>
// with k, v the 8-bit codes and ks, vs their blocks' scales. Row i of a request with n rows and `len` cached
// tokens stands at position p = len - n + i (the step's own tokens are in the cache already) and sees
//   mask_block b >= 1: keys below origin + ((p - origin) / b + 1) b, below origin where p < origin
//   mask_block 0: every key
// and never a key at len or behind it; a row with p < 0 or len = 0 sees none and gets zeros and lse -inf.
// b = 1 is the causal mask, a block size with the prompt as origin the d2f_hybrid mask of attention.cuh.
//
// Codes go to the matrix units exactly: an int8 or e4m3 code is an f16 number, so <q, k> is exact up to its
// f32 sum (a bf16 row of q is brought into f16's range by a power of two, which the scale takes back). The
// scales stay outside: ks multiplies the f32 score; vs joins the probability before it is rounded to f16,
//   w_ij = 2^(s_ij - m_i) vs_j / 2^(M_i - m_i),  m_i = running max s,  M_i = running max (s + log2 vs)
// so the largest weight of a row is 1 whatever the spread of the scales, and a weight is off by 2^-11 of
// itself or 2^-25 of the row's largest. The sum of the probabilities keeps its own maximum m and f32.
//
// Work is counted in key tiles of 64: a unit (request, row tile, kv head) has as many as its last row sees.
// All tiles of all units lie on one axis that is cut into equal shares, so a batch of unequal lengths, one
// long request and many short ones all fill the GPU; a unit cut between shares leaves partial sums that a
// second kernel joins in the order of the shares.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "kvcache.cuh"

namespace drt {

struct CacheAttnArgs {
  const void* q;
  int64_t q_row, q_head;      // strides in elements
  int q_rows;                 // rows of q and out
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  int64_t blocks;
  int block, heads, group;    // kv heads; query heads per kv head
  const int* tables;
  int64_t ld_tables;
  int width;
  const int *lengths, *row_start, *origin;
  int requests, mask_block;
  float scale_log2;           // scale * log2(e)
  void* out;
  int64_t out_row, out_head;
  float* lse;                 // [q_rows][heads * group] or null
  int vec, out_vec;           // rows of q and of out start on 16-byte boundaries
  int rows_from, rows_to;     // the requests whose rows times group lie in between are this launch's
  // parts of cut units: per warp and per CTA a front and a tail, [rows of a tile][dim] sums and their (m, M, l)
  float *part, *cta_part;
  float4 *stat, *cta_stat;
  int4* desc;                 // [CTAs] rows | last CTA << 9, request, row tile, head of the unit that the CTA begins
};

struct CacheReq {
  int row0, n, len, origin;
};

// Request r as this launch sees it (n = 0: nothing to do).
__device__ __forceinline__ CacheReq cache_request(const CacheAttnArgs& a, int r) {
  CacheReq q;
  q.row0 = min(max(a.row_start[r], 0), a.q_rows);
  q.n = max(0, min(a.row_start[r + 1], a.q_rows) - q.row0);
  if (q.n * a.group < a.rows_from || q.n * a.group > a.rows_to) q.n = 0;  // another launch's
  q.len = static_cast<int>(min(static_cast<int64_t>(max(a.lengths[r], 0)), static_cast<int64_t>(a.width) * a.block));
  q.origin = a.origin ? max(a.origin[r], 0) : 0;
  return q;
}

// Keys that row i of the request sees; never falls with i.
__device__ __forceinline__ int cache_limit(const CacheAttnArgs& a, const CacheReq& q, int i) {
  const int p = q.len - q.n + i;
  if (p < 0) return 0;
  if (a.mask_block == 0) return q.len;
  if (p < q.origin) return min(q.origin, q.len);
  const int64_t lim = q.origin + (static_cast<int64_t>((p - q.origin) / a.mask_block) + 1) * a.mask_block;
  return static_cast<int>(min(lim, static_cast<int64_t>(q.len)));
}

__device__ __forceinline__ float qa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four codes of a 32-bit word as two f16 pairs, exact.
template <int kCode>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kCode == CACHE_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // code + 128 as the low mantissa byte of 1024 gives f16 1152 + code
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 base = __half2half2(__ushort_as_half(0x6480));  // 1152
    const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), base);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&y), base);
    lo = *reinterpret_cast<const uint32_t*>(&p);
    hi = *reinterpret_cast<const uint32_t*>(&r);
  }
}

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word_of(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// Transposed 8 x 8 matrix of f16 spread over the warp (a lane holds row lane / 4, columns 2 (lane % 4), + 1).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t f16_pair(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Untiled bulk copy of `bytes` (a multiple of 16, both ends 16-byte aligned) into shared memory.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ---------------------------------------------------------------- few rows: one warp, one share
// A warp owns a share. Its unit is a row tile of 8 kNT rows (row = position * group + query head, so a kv head's
// keys serve all of its query heads) and it computes the transposed products on mma.sync m16n8k16,
//   S^T [keys x rows] = K Q^T,   O^T [dims x rows] += V^T W^T,
// with the codes as the 16-row operand: eight rows, the query heads of one token in a GQA model, then waste
// nothing, and each code is expanded to f16 once, in the registers of the lane that read it. A key costs 2 kDim bytes
// and 16 kNT kDim multiply-adds, 8 kNT a byte, far below what the SM's mma.sync can do at the memory's rate, so the
// bytes bound a long call; tcgen05 would need the expanded codes written to shared memory first.
// Measured (dim 128): 64 requests of 8,192 tokens, 8 kv heads, 1.07 GB of codes: 176 us for 2 query heads each, 188 for
// 8 (6.1 and 5.7 TB/s); 16 of 65,536, 4 kv heads of 7: 174 us. A start costs about 5 us (lengths, shares, first
// tiles), the join in the CTA 3, the join's launch 4: one request of 130,001 tokens, 133 MB, takes 39 us (3.4 TB/s), one
// of 4,096 tokens 15. Twelve warps to a CTA with two tiles in flight each were slower than eight with three.
//
// Lanes (g = lane / 4, q = lane % 4). The contracted index may be taken in any order that both operands share:
//   K: a lane reads 16 bytes of a key's row, dimensions 16 (q + 4 half) .., four k-steps' worth of its fragment;
//   V: a lane reads the 16 tokens of group q of one dimension, four k-steps' worth; so k-step s of the 64 keys
//      contracts tokens 16 q + 4 s + {0, 1} and + {2, 3} of each lane group q, and K's fragment s holds the same
//      tokens in its rows: row g token 16 (g / 2) + 4 s + g % 2, row g + 8 the token two behind.
// A lane's keys are all of group g / 2, hence of one block (a block holds whole groups): one ks, one vs per
// lane and tile. movmatrix turns W^T's accumulator layout into the operand's.
//
// The warps do not wait for one another until their shares are done: each issues its own copies (2 KB per 16-token
// group) into its own ring of K and V tiles, on into its next unit, whose table entries it has read by then. At the
// end the CTA joins what its warps' borders cut, so that a long unit leaves one part per CTA and not one per warp.
constexpr int kQrTile = 64;        // keys
constexpr int kQrMaxRequests = 16384;

template <int kDim, int kNT>
struct QrCfg {
  static constexpr int kRows = 8 * kNT;
  static constexpr int kWarps = 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kGroupBytes = 16 * kDim;
  static constexpr int kGroupPitch = kGroupBytes + 32;  // V reads of the four groups fall into different banks
  static constexpr int kSlot = 4 * kGroupPitch;
  static constexpr int kSlots = 3 * (128 / kDim);
  static constexpr int kRing = kSlots * kSlot;
  static constexpr size_t kSmem = static_cast<size_t>(kWarps) * kRing + kWarps * kSlots * 8;
  static_assert(kWarps * kRing >= (kQrMaxRequests + 1) * 8, "the requests' places stand in the rings' memory first");
};
constexpr int kQrMaxRows = 16;                 // of a tile
constexpr int kQrMaxParts = 8 * 2 * kQrMaxRows;  // rows of the parts of a CTA's warps

// A unit: row tile t of request r with kv head h. lim: the keys that its last row sees, L: their tiles (at least one).
struct QaUnit {
  CacheReq q;
  int r, t, h, lim, L;
};

template <int kRows, int kTile>
__device__ __forceinline__ void qa_size(const CacheAttnArgs& a, QaUnit& u) {
  u.lim = cache_limit(a, u.q, (min(u.q.n * a.group, (u.t + 1) * kRows) - 1) / a.group);
  u.L = max(1, (u.lim + kTile - 1) / kTile);
}
// The unit behind u; there is one.
template <int kRows, int kTile>
__device__ __forceinline__ void qa_next(const CacheAttnArgs& a, QaUnit& u) {
  if (++u.h < a.heads) return;
  u.h = 0;
  if (++u.t * kRows >= u.q.n * a.group) {
    u.t = 0;
    do u.q = cache_request(a, ++u.r);
    while (u.q.n == 0);
  }
  qa_size<kRows, kTile>(a, u);
}

// The axis of `total` places cut into `shares`: each has `each` places, the first `more` of them one more.
struct QaCut {
  int64_t each;
  int more;
  __device__ __forceinline__ QaCut(int64_t total, int shares) {
    each = total >> 31 ? total / shares : static_cast<uint32_t>(total) / static_cast<uint32_t>(shares);
    more = static_cast<int>(total - each * shares);
  }
  __device__ __forceinline__ int64_t begin(int w) const { return each * w + min(w, more); }
  // The share that holds place x.
  __device__ __forceinline__ int owner(int64_t x) const {
    const int64_t wide = (each + 1) * more;
    return static_cast<int>(x < wide ? x / (each + 1) : more + (x - wide) / each);
  }
};

// What a unit costs beside its tiles, in tiles: the reads of its queries and table, its softmax's start and its output.
// A unit takes so many places on the axis before its first tile, so that the shares of many short units are not
// longer than those of one long one.
constexpr int kQaUnitCost = 2;

// Exclusive sums of the requests' places on the axis into prefix[0 .. requests], by the whole CTA.
template <int kRows, int kTile, int kThreads>
__device__ __forceinline__ int64_t qa_prefix(const CacheAttnArgs& a, int64_t* prefix) {
  __shared__ int64_t wsum[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t base = 0;
  for (int r0 = 0; r0 < a.requests; r0 += kThreads) {
    const int r = r0 + tid;
    int64_t v = 0;
    if (r < a.requests) {
      const CacheReq q = cache_request(a, r);
      const int nt = (q.n * a.group + kRows - 1) / kRows;
      QaUnit u;
      u.q = q;
      for (u.t = 0; u.t < nt; ++u.t) {
        qa_size<kRows, kTile>(a, u);
        v += u.L + kQaUnitCost;
      }
      v *= a.heads;
    }
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    int64_t add = base, all = base;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) add += wsum[w];
      all += wsum[w];
    }
    if (r < a.requests) prefix[r] = add + x - v;
    base = all;
    __syncthreads();
  }
  if (tid == 0) prefix[a.requests] = base;
  __syncthreads();
  return base;
}

template <typename T>
__device__ __forceinline__ void qa_store2(T* p, float x, float y);
template <>
__device__ __forceinline__ void qa_store2<__half>(__half* p, float x, float y) {
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y);
}
template <>
__device__ __forceinline__ void qa_store2<__nv_bfloat16>(__nv_bfloat16* p, float x, float y) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
}

// What a warp's share cuts: its front (a unit begun in an earlier share) and its tail (one that ends in a later).
enum : int { QR_FRONT = 1, QR_FRONT_ENDS = 2, QR_TAIL = 4 };
struct QrEnd {
  int flags, rows, front_rows, busy, r, t, h, last;
};

template <int kE>
__device__ __forceinline__ void qa_load(float* v, const float* src) {
  if constexpr (kE == 4) {
    const float4 x = *reinterpret_cast<const float4*>(src);
    v[0] = x.x;
    v[1] = x.y;
    v[2] = x.z;
    v[3] = x.w;
  } else {
    const float2 x = *reinterpret_cast<const float2*>(src);
    v[0] = x.x;
    v[1] = x.y;
  }
}

// A finished row by one warp: kE dimensions a lane, sums against the references z (of l) and Z (of acc).
template <typename T, int kE>
__device__ __forceinline__ void qa_put(const CacheAttnArgs& a, int r, int row, int h, int lane, float z, float Z, float m,
                                       float l, const float* acc) {
  const int i = row / a.group, hq = h * a.group + row - i * a.group;
  const int64_t out_row = min(max(a.row_start[r], 0), a.q_rows) + i;
  const float n = l == 0.0f ? 0.0f : qa_ex2(Z - z) / l;
  T* dst = static_cast<T*>(a.out) + out_row * a.out_row + hq * a.out_head + lane * kE;
#pragma unroll
  for (int e = 0; e < kE; e += 2) qa_store2<T>(dst + e, acc[e] * n, acc[e + 1] * n);
  if (lane == 0 && a.lse) a.lse[out_row * a.heads * a.group + hq] = (m + log2f(l)) * 0.6931471805599453f;
}

template <typename T, int kDim, int kCode, int kNT>
__global__ void __launch_bounds__(QrCfg<kDim, kNT>::kThreads, 1) cache_attn_rows_kernel(const CacheAttnArgs a) {
  using Cfg = QrCfg<kDim, kNT>;
  constexpr int kRows = Cfg::kRows;
  constexpr int kHalves = kDim / 64;   // 16-byte reads of a key's row per lane
  constexpr int kMT = kDim / 16;       // 16-dimension tiles of O^T
  extern __shared__ __align__(128) uint8_t qr_smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(qr_smem + Cfg::kWarps * Cfg::kRing);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, tq = lane & 3;
  uint8_t* ring = qr_smem + warp * Cfg::kRing;
  uint64_t* full = bars + warp * Cfg::kSlots;
  if (lane == 0)
    for (int i = 0; i < Cfg::kSlots; ++i) mbar_init(&full[i], 1);
  fence_mbar_init();

  griddep_launch_dependents();  // the join's CTAs may take what is left of the SMs; they wait for this grid's end
  // the table entries on their way to L2 while the lengths are read
  for (int64_t i = blockIdx.x * Cfg::kThreads + tid; i * 32 < static_cast<int64_t>(a.requests) * a.width && i < 65536;
       i += gridDim.x * Cfg::kThreads) {
    const int64_t e = i * 32, r = e / a.width;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(a.tables + r * a.ld_tables + (e - r * a.width)));
  }
  __shared__ QrEnd ends[Cfg::kWarps];
  int64_t* prefix = reinterpret_cast<int64_t*>(qr_smem);
  const int64_t total = qa_prefix<kRows, kQrTile, Cfg::kThreads>(a, prefix);
  const int ctas = static_cast<int>(min(total, static_cast<int64_t>(gridDim.x)));
  int64_t x = 0, x_end = 0;
  QaUnit cur = {};
  const QaCut cut(total, max(ctas, 1));
  if (blockIdx.x < ctas) {
    const int64_t c0 = cut.begin(blockIdx.x), n = cut.begin(blockIdx.x + 1) - c0;
    x = c0 + n * warp / Cfg::kWarps;
    x_end = c0 + n * (warp + 1) / Cfg::kWarps;
    int hi = a.requests;
    while (hi - cur.r > 1) {
      const int mid = (cur.r + hi) >> 1;
      if (prefix[mid] <= x) cur.r = mid;
      else hi = mid;
    }
  }
  int64_t rem = x - prefix[cur.r];
  __syncthreads();           // prefix is done with: its memory becomes the rings
  fence_proxy_async_smem();

  int kt = 0;                // first key tile of the segment: what this share holds of the unit
  uint32_t seq_used = 0;     // ring entries consumed in earlier segments
  uint32_t issued = 0;       // entries asked for, counted from the segment's first
  bool failed = false;
  const int block_shift = 31 - __clz(a.block);
  if (x < x_end) {
    cur.q = cache_request(a, cur.r);
    qa_size<kRows, kQrTile>(a, cur);
    while (rem >= static_cast<int64_t>(cur.L + kQaUnitCost) * a.heads) {
      rem -= static_cast<int64_t>(cur.L + kQaUnitCost) * a.heads;
      ++cur.t;
      qa_size<kRows, kQrTile>(a, cur);
    }
    const int per = cur.L + kQaUnitCost;
    cur.h = rem >> 31 ? static_cast<int>(rem / per) : static_cast<int>(rem) / per;
    kt = static_cast<int>(rem - static_cast<int64_t>(cur.h) * per) - kQaUnitCost;
    if (kt < 0) {            // the share begins before the unit's first tile
      x -= kt;
      kt = 0;
    }
  }
  QrEnd end;
  end.flags = end.rows = end.front_rows = end.r = end.t = end.h = end.last = 0;
  end.busy = x < x_end;
  // tables and scales of eight tiles at a time: lane = tile * 4 + group
  struct Meta {
    int page;
    float ks, vs;
  };
  auto table_entry = [&](const QaUnit& u, int tile0) {
    const int tok = (tile0 + (lane >> 2)) * kQrTile + (lane & 3) * 16;
    return tok < u.lim ? a.tables[u.r * a.ld_tables + (tok >> block_shift)] : -1;
  };
  auto scales_of = [&](int id, int h) {
    Meta d = {-1, 0.0f, 0.0f};
    if (id >= 0 && id < a.blocks) {
      d.page = id;
      d.ks = a.k_scale[static_cast<int64_t>(id) * a.heads + h];
      d.vs = a.v_scale[static_cast<int64_t>(id) * a.heads + h];
    }
    return d;
  };
  int tiles = static_cast<int>(min(static_cast<int64_t>(cur.L - kt), x_end - x));
  QaUnit nxt = cur;
  Meta now = {-1, 0.0f, 0.0f}, then = now, ahead = now;
  if (x < x_end) now = scales_of(table_entry(cur, kt), cur.h);

  while (x < x_end && !failed) {
    const int entries = 2 * tiles;
    const int tiles_nxt = [&] {
      if (x + tiles + kQaUnitCost >= x_end) return 0;
      qa_next<kRows, kQrTile>(a, nxt);
      return static_cast<int>(min(static_cast<int64_t>(nxt.L), x_end - x - tiles - kQaUnitCost));
    }();
    // Asks for the next ring entry (even: K, odd: V) of this segment or the one behind it; `done` tiles are consumed.
    auto issue = [&](int done) -> bool {
      int s = issued, base = kt, h = cur.h, pg;
      if (s < entries) {
        const int tile = s >> 1;
        pg = __shfl_sync(~0u, (tile >> 3) != (done >> 3) ? then.page : now.page, (tile & 7) * 4 + (lane & 3));
      } else {
        s -= entries;
        if (s >= 2 * tiles_nxt || s >= 16) return false;
        base = 0;
        h = nxt.h;
        pg = __shfl_sync(~0u, ahead.page, (s >> 1) * 4 + (lane & 3));
      }
      const uint32_t slot = (seq_used + issued++) % Cfg::kSlots;
      const uint32_t have = __ballot_sync(~0u, pg >= 0) & 15u;
      if (lane == 0) mbar_expect_tx(&full[slot], __popc(have) * Cfg::kGroupBytes);
      __syncwarp();
      if (lane < 4 && pg >= 0) {
        const int tok = (base + (s >> 1)) * kQrTile + lane * 16;
        const uint8_t* src = ((s & 1) ? a.v_cache : a.k_cache) +
                             (((static_cast<int64_t>(pg) * a.heads + h) << block_shift) + (tok & (a.block - 1))) * kDim;
        bulk_load(smem_u32(ring + slot * Cfg::kSlot + lane * Cfg::kGroupPitch), src, Cfg::kGroupBytes, &full[slot]);
      }
      return true;
    };
    while (issued < Cfg::kSlots && issued < entries) issue(0);
    // asked for here, looked at behind the first K tile's products
    int then_id = tiles > 8 ? table_entry(cur, kt + 8) : -1;
    const int ahead_id = tiles_nxt > 0 ? table_entry(nxt, 0) : -1;
    const int rows_all = cur.q.n * a.group, row0 = cur.t * kRows, lim = cur.lim;
    if (tiles_nxt > 0) {     // the next unit's rows of Q on their way to L2
      const int row = min(nxt.t * kRows + g, nxt.q.n * a.group - 1), i = row / a.group;
      const T* src = static_cast<const T*>(a.q) + (nxt.q.row0 + i) * a.q_row + (nxt.h * a.group + row - i * a.group) * a.q_head;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(src + tq * (kDim / 4)));
    }

    // ---- Q^T fragments: lane holds dimensions 16 (q + 4 half) .. + 15 of row g of each row group
    uint32_t qf[kNT][kHalves * 4][2];
    float f[kNT];             // takes the power of two of row g back
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int row = min(row0 + n * 8 + g, rows_all - 1), i = row / a.group;
      const T* src = static_cast<const T*>(a.q) + (cur.q.row0 + i) * a.q_row + (cur.h * a.group + row - i * a.group) * a.q_head;
      __align__(16) T v[kHalves * 16];
#pragma unroll
      for (int hh = 0; hh < kHalves; ++hh) {
        const T* p = src + 16 * (tq + 4 * hh);
        if (a.vec) {
          reinterpret_cast<uint4*>(v)[hh * 2] = reinterpret_cast<const uint4*>(p)[0];
          reinterpret_cast<uint4*>(v)[hh * 2 + 1] = reinterpret_cast<const uint4*>(p)[1];
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[hh * 16 + e] = p[e];
        }
      }
      float up = 1.0f;
      f[n] = a.scale_log2;
      if constexpr (!std::is_same<T, __half>::value) {
        float mx = 0.0f;
#pragma unroll
        for (int e = 0; e < kHalves * 16; ++e) mx = fmaxf(mx, fabsf(cache_in_f32(v[e])));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
        // the largest magnitude to [2^14, 2^15)
        const int e = mx > 0.0f && mx <= 3.402823466e38f ? max(-100, static_cast<int>((__float_as_uint(mx) >> 23) & 255) - 127) : 14;
        up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
        f[n] *= __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
      }
#pragma unroll
      for (int st = 0; st < kHalves * 4; ++st) {
        qf[n][st][0] = f16_pair(cache_in_f32(v[st * 4]) * up, cache_in_f32(v[st * 4 + 1]) * up);
        qf[n][st][1] = f16_pair(cache_in_f32(v[st * 4 + 2]) * up, cache_in_f32(v[st * 4 + 3]) * up);
      }
    }
    // of the rows that this lane's accumulators hold: 2 q and 2 q + 1 of each row group
    float fr[kNT][2];
    int lr[kNT][2], lim_low = lim;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        fr[n][e] = __shfl_sync(~0u, f[n], (2 * tq + e) * 4);
        lr[n][e] = cache_limit(a, cur.q, min(row0 + n * 8 + 2 * tq + e, rows_all - 1) / a.group);
        lim_low = min(lim_low, lr[n][e]);
      }

    float o[kNT][kMT][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < kMT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
    float m[kNT][2], M[kNT][2], l[kNT][2];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = M[n][e] = -INFINITY;
        l[n][e] = 0.0f;
      }

    for (int j = 0; j < tiles; ++j) {
      if (j > 0 && (j & 7) == 0) {
        now = then;
        then_id = j + 8 < tiles ? table_entry(cur, kt + j + 8) : -1;
      }
      const int key0 = (kt + j) * kQrTile;

      // ---- S^T = K Q^T
      float s[kNT][4][4];
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i][0] = s[n][i][1] = s[n][i][2] = s[n][i][3] = 0.0f;
      {
        const uint32_t e = seq_used + 2 * j;
        if (!failed) failed = __any_sync(~0u, !mbar_wait(&full[e % Cfg::kSlots], (e / Cfg::kSlots) & 1));
        const uint8_t* kb = ring + (e % Cfg::kSlots) * Cfg::kSlot + (g >> 1) * Cfg::kGroupPitch + (g & 1) * kDim + tq * 16;
        // four keys' fragments side by side: their products do not wait for one another
#pragma unroll
        for (int hh = 0; hh < kHalves; ++hh) {
          uint4 u[4], u2[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[i] = *reinterpret_cast<const uint4*>(kb + 4 * i * kDim + hh * 64);
            u2[i] = *reinterpret_cast<const uint4*>(kb + (4 * i + 2) * kDim + hh * 64);
          }
#pragma unroll
          for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t af[4];
              codes_to_f16<kCode>(word_of(u[i], st), af[0], af[2]);
              codes_to_f16<kCode>(word_of(u2[i], st), af[1], af[3]);
#pragma unroll
              for (int n = 0; n < kNT; ++n) mma_f16(s[n][i], af, qf[n][hh * 4 + st][0], qf[n][hh * 4 + st][1]);
            }
        }
        __syncwarp();
        if ((j & 7) == 0) then = scales_of(then_id, cur.h);
        if (j == 0) ahead = scales_of(ahead_id, nxt.h);
        while (!failed && issued < 2 * j + 1 + Cfg::kSlots && issue(j)) {}
      }

      // ---- softmax over this lane's eight keys, then over the lanes g of a row
      const int src_lane = (j & 7) * 4 + (g >> 1);
      const float k_mul = __shfl_sync(~0u, now.ks, src_lane), lv = __log2f(__shfl_sync(~0u, now.vs, src_lane));
      const bool here = __shfl_sync(~0u, now.page, src_lane) >= 0;
      const int first = key0 + (g >> 1) * 16 + (g & 1);  // the lane's keys: first + 4 i, + 2
      const bool edge = __any_sync(~0u, key0 + kQrTile > lim_low || !here);
      uint32_t pf[kNT][4][2];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        float tm[2], um[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float c = k_mul * fr[n][e];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[n][i][e] *= c;
            s[n][i][2 + e] *= c;
          }
          if (edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (!(here && first + 4 * i < lr[n][e])) s[n][i][e] = -INFINITY;
              if (!(here && first + 4 * i + 2 < lr[n][e])) s[n][i][2 + e] = -INFINITY;
            }
          }
          tm[e] = fmaxf(s[n][0][e], s[n][0][2 + e]);
#pragma unroll
          for (int i = 1; i < 4; ++i) tm[e] = fmaxf(tm[e], fmaxf(s[n][i][e], s[n][i][2 + e]));
          um[e] = here ? tm[e] + lv : -INFINITY;
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            tm[e] = fmaxf(tm[e], __shfl_xor_sync(~0u, tm[e], d));
            um[e] = fmaxf(um[e], __shfl_xor_sync(~0u, um[e], d));
          }
        float z[2], w[2], k[2];
        bool moved = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float nm = fmaxf(m[n][e], tm[e]), nM = fmaxf(M[n][e], um[e]);
          // a row that has seen nothing yet keeps zeros: its reference is 0 and every term 2^-inf
          z[e] = nm == -INFINITY ? 0.0f : nm;
          const float Z = nM == -INFINITY ? 0.0f : nM;
          l[n][e] *= qa_ex2(m[n][e] - z[e]);
          k[e] = qa_ex2(M[n][e] - Z);
          moved = moved || nM != M[n][e];
          m[n][e] = nm;
          M[n][e] = nM;
          // weight = p vs / 2^(M - m): at most 1 where p is not 0; the factor alone may leave f32's range
          w[e] = here ? qa_ex2(fminf(lv + (z[e] - Z), 120.0f)) : 0.0f;
        }
        if (__any_sync(~0u, moved)) {
#pragma unroll
          for (int i = 0; i < kMT; ++i) {
            o[n][i][0] *= k[0];
            o[n][i][1] *= k[1];
            o[n][i][2] *= k[0];
            o[n][i][3] *= k[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = qa_ex2(s[n][i][0] - z[0]), p1 = qa_ex2(s[n][i][1] - z[1]);
          const float p2 = qa_ex2(s[n][i][2] - z[0]), p3 = qa_ex2(s[n][i][3] - z[1]);
          l[n][0] += p0 + p2;
          l[n][1] += p1 + p3;
          pf[n][i][0] = transpose8(f16_pair(p0 * w[0], p1 * w[1]));
          pf[n][i][1] = transpose8(f16_pair(p2 * w[0], p3 * w[1]));
        }
      }

      // ---- O^T += V^T W^T
      {
        const uint32_t e = seq_used + 2 * j + 1;
        if (!failed) failed = __any_sync(~0u, !mbar_wait(&full[e % Cfg::kSlots], (e / Cfg::kSlots) & 1));
        const uint8_t* vb = ring + (e % Cfg::kSlots) * Cfg::kSlot + tq * Cfg::kGroupPitch + g * 16;
        // tokens nobody sees hold anything: their codes are cleared, since 0 times a NaN code is not 0
        uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
        if (edge) {
          const bool mine = __shfl_sync(~0u, now.page, (j & 7) * 4 + tq) >= 0;
          const int live = mine ? min(16, max(0, lim - key0 - tq * 16)) : 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = min(4, max(0, live - 4 * i));
            keep[i] = c >= 4 ? ~0u : (1u << (8 * c)) - 1u;
          }
        }
#pragma unroll
        for (int i0 = 0; i0 < kMT; i0 += 4) {
          uint4 u[4], u2[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[i] = *reinterpret_cast<const uint4*>(vb + (i0 + i) * 256);
            u2[i] = *reinterpret_cast<const uint4*>(vb + (i0 + i) * 256 + 128);
          }
          if (edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              u[i] = make_uint4(u[i].x & keep[0], u[i].y & keep[1], u[i].z & keep[2], u[i].w & keep[3]);
              u2[i] = make_uint4(u2[i].x & keep[0], u2[i].y & keep[1], u2[i].z & keep[2], u2[i].w & keep[3]);
            }
          }
#pragma unroll
          for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t af[4];
              codes_to_f16<kCode>(word_of(u[i], st), af[0], af[2]);
              codes_to_f16<kCode>(word_of(u2[i], st), af[1], af[3]);
#pragma unroll
              for (int n = 0; n < kNT; ++n) mma_f16(o[n][i0 + i], af, pf[n][st][0], pf[n][st][1]);
            }
        }
        __syncwarp();
        while (!failed && issued < 2 * j + 2 + Cfg::kSlots && issue(j)) {}
      }
    }

    const bool begins = kt == 0, whole = begins && tiles == cur.L;
    const int64_t at = (static_cast<int64_t>(blockIdx.x * Cfg::kWarps + warp) * 2 + (begins ? 1 : 0)) * kRows;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(~0u, l[n][e], d);
        if (failed) l[n][e] = NAN;  // a copy did not arrive in time: the rows read as NaN
        const int rt = n * 8 + 2 * tq + e, row = row0 + rt;
        if (row >= rows_all) continue;
        if (whole) {
          const int i = row / a.group, hq = cur.h * a.group + row - i * a.group;
          const float inv = l[n][e] == 0.0f ? 0.0f : qa_ex2(M[n][e] - m[n][e]) / l[n][e];
          T* dst = static_cast<T*>(a.out) + (cur.q.row0 + i) * a.out_row + hq * a.out_head + g;
#pragma unroll
          for (int d = 0; d < kMT; ++d) {
            dst[d * 16] = cache_out<T>(o[n][d][e] * inv);
            dst[d * 16 + 8] = cache_out<T>(o[n][d][2 + e] * inv);
          }
          if (a.lse && g == 0)
            a.lse[(cur.q.row0 + i) * static_cast<int64_t>(a.heads) * a.group + hq] =
                (m[n][e] + log2f(l[n][e])) * 0.6931471805599453f;
        } else {
          float* dst = a.part + (at + rt) * kDim + g;
#pragma unroll
          for (int d = 0; d < kMT; ++d) {
            dst[d * 16] = o[n][d][e];
            dst[d * 16 + 8] = o[n][d][2 + e];
          }
          if (g == 0) a.stat[at + rt] = make_float4(m[n][e], M[n][e], l[n][e], 0.0f);
        }
      }
    if (!whole) {
      end.flags |= begins ? QR_TAIL : kt + tiles == cur.L ? QR_FRONT | QR_FRONT_ENDS : QR_FRONT;
      end.rows = min(kRows, rows_all - row0);  // of the last cut unit: the tail's, or a front that fills the share
      if (!begins) end.front_rows = end.rows;
      if (begins) {
        end.r = cur.r;
        end.t = cur.t;
        end.h = cur.h;
        end.last = cut.owner(x + cur.L - 1);
      }
    }
    x = tiles_nxt > 0 ? x + tiles + kQaUnitCost : x_end;
    if (x < x_end && !failed) {
      seq_used += entries;
      issued -= min(issued, static_cast<uint32_t>(entries));
      cur = nxt;
      tiles = tiles_nxt;
      kt = 0;
      now = ahead;
    }
  }
  if (failed) {  // the copies still under way land (bounded waits) before the shared memory is given up
    const uint32_t all = seq_used + issued;
    for (uint32_t e = all > Cfg::kSlots ? all - Cfg::kSlots : 0; e < all; ++e)
      mbar_wait(&full[e % Cfg::kSlots], (e / Cfg::kSlots) & 1);
  }

  // ---- the CTA joins the parts that its warps' borders cut: a chain is the tail of one warp, or the front of the
  // first, and the fronts behind it up to the one that ends the unit. Items (chain, row) are dealt to the warps.
  if (lane == 0) ends[warp] = end;
  __syncthreads();
  int item = 0;
  for (int s = -1; s < Cfg::kWarps; ++s) {
    // chain s: begins with warp s's tail, -1: with the front of the CTA's first busy warp
    int w = s, rows;
    bool done = false;
    if (s < 0) {
      for (w = 0; w < Cfg::kWarps && !ends[w].busy; ++w) {}
      if (w == Cfg::kWarps || !(ends[w].flags & QR_FRONT)) continue;
      rows = ends[w].front_rows;
      done = ends[w].flags & QR_FRONT_ENDS;
    } else {
      if (!(ends[w].flags & QR_TAIL)) continue;
      rows = ends[w].rows;
    }
    int last = w;
    for (int v = w + 1; v < Cfg::kWarps && !done; ++v)
      if (ends[v].flags & QR_FRONT) {
        last = v;
        done = ends[v].flags & QR_FRONT_ENDS;
      }
    for (int row = 0; row < rows; ++row, ++item) {
      if (item % Cfg::kWarps != warp) continue;
      auto slot = [&](int v) {
        return (static_cast<int64_t>(blockIdx.x * Cfg::kWarps + v) * 2 + (v == s ? 1 : 0)) * kRows + row;
      };
      const bool has = lane >= w && lane <= last && (lane == s || (ends[min(lane, Cfg::kWarps - 1)].flags & QR_FRONT));
      const uint32_t who = __ballot_sync(~0u, has);
      constexpr int kE = kDim / 32;
      float part[Cfg::kWarps][kE];
#pragma unroll
      for (int v = 0; v < Cfg::kWarps; ++v)  // all loads at once; a warp without a part gives the first one's, times 0
        qa_load<kE>(part[v], a.part + slot(who >> v & 1 ? v : w) * kDim + lane * kE);
      float4 st = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
      if (has) st = a.stat[slot(lane)];
      float m = st.x, M = st.y;
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
        M = fmaxf(M, __shfl_xor_sync(~0u, M, d));
      }
      const float z = m == -INFINITY ? 0.0f : m, Z = M == -INFINITY ? 0.0f : M;
      const float fM = has ? qa_ex2(st.y - Z) : 0.0f;
      float l = has ? st.z * qa_ex2(st.x - z) : 0.0f;
#pragma unroll
      for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
      float acc[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[e] = 0.0f;
#pragma unroll
      for (int v = 0; v < Cfg::kWarps; ++v) {
        const float f = __shfl_sync(~0u, fM, v);
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] += part[v][e] * f;
      }
      if (s >= 0 && done) {
        qa_put<T, kE>(a, ends[s].r, ends[s].t * kRows + row, ends[s].h, lane, z, Z, m, l, acc);
      } else {
        const int64_t at = (static_cast<int64_t>(blockIdx.x) * 2 + (s < 0 ? 0 : 1)) * kRows + row;
        float* dst = a.cta_part + at * kDim + lane * kE;
#pragma unroll
        for (int e = 0; e < kE; e += 2) *reinterpret_cast<float2*>(dst + e) = make_float2(acc[e], acc[e + 1]);
        if (lane == 0) a.cta_stat[at] = make_float4(m, M, l, 0.0f);
      }
    }
    if (s >= 0 && !done && tid == 0)  // cut at the CTA's end: its owner's descriptor
      a.desc[blockIdx.x] = make_int4(rows | ends[s].last << 9, ends[s].r, ends[s].t, ends[s].h);
    if (s >= 0 && !done) return;      // the last chain
  }
  if (tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
}

// Joins the parts of the units that CTAs' shares cut: the CTA in which a unit begins names it (tail part), its later
// parts are the front parts of the CTAs up to the last. CTA (four owners, `step` rows of the tile): half a warp joins a row
// of a unit of up to kQmAlone parts, all of them read at once, the whole CTA a row of the longer ones, their parts dealt to
// the warps; either order is fixed by the shares.
// Bound by the latency of dependent reads (owner, then statistics, parts and the request's place): 2.5 to 6 us after the
// kernel over few rows; 13 us after the one over many for two prompts, whose 148 cut units leave 40 MB. A warp to a row with
// its parts read in turn took 1.3 and 6 us more; as many CTAs as are resident, each through several rows, 3 us more.
constexpr int kQmThreads = 128;  // with their registers they fit beside a CTA of the rows kernel
constexpr int kQmWarps = kQmThreads / 32;
constexpr int kQmAlone = 4;

template <typename T, int kDim, int kRows>
__global__ void __launch_bounds__(kQmThreads) cache_attn_merge_kernel(const CacheAttnArgs a, int ctas, int step) {
  constexpr int kE = kDim / 32;  // dimensions per lane
  constexpr int kE2 = kDim / 16; // with half a warp to a row
  __shared__ float red[kQmWarps][kDim];
  __shared__ float red_s[kQmWarps];
  griddep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = blockIdx.x * kQmWarps;
  int4 mine = make_int4(0, 0, 0, 0);  // lane i of every warp holds owner base + i
  if (lane < kQmWarps && base + lane < ctas) mine = a.desc[base + lane];
  const int my_parts = (mine.x >> 9) - (base + lane) + 1, my_rows = mine.x & 511;
  for (int row = blockIdx.y * step; row < kRows; row += gridDim.y * step) {
    const uint32_t alone = __ballot_sync(~0u, row < my_rows && my_parts <= kQmAlone);
    if (__ballot_sync(~0u, row < my_rows) == 0) break;  // later rows have no owner either
    if (alone >> warp & 1) {
      const int parts = __shfl_sync(~0u, my_parts, warp), rows = __shfl_sync(~0u, my_rows, warp);
      const int r = __shfl_sync(~0u, mine.y, warp), t = __shfl_sync(~0u, mine.z, warp), h = __shfl_sync(~0u, mine.w, warp);
      const int own = row + (lane >> 4), at_dim = (lane & 15) * kE2;
      if ((lane >> 4) < step && own < rows) {
        float4 s[kQmAlone];
        float v[kQmAlone][kE2];
#pragma unroll
        for (int p = 0; p < kQmAlone; ++p) {
          s[p] = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
          if (p < parts) {
            const int64_t at = (static_cast<int64_t>(base + warp + p) * 2 + (p == 0 ? 1 : 0)) * kRows + own;
            s[p] = a.cta_stat[at];
#pragma unroll
            for (int e = 0; e < kE2; e += 4) qa_load<4>(v[p] + e, a.cta_part + at * kDim + at_dim + e);
          }
        }
        float m = -INFINITY, M = -INFINITY, l = 0.0f, acc[kE2];
#pragma unroll
        for (int p = 0; p < kQmAlone; ++p) {
          m = fmaxf(m, s[p].x);
          M = fmaxf(M, s[p].y);
        }
        const float z = m == -INFINITY ? 0.0f : m, Z = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int e = 0; e < kE2; ++e) acc[e] = 0.0f;
#pragma unroll
        for (int p = 0; p < kQmAlone; ++p) {
          if (p >= parts) break;
          const float f = qa_ex2(s[p].y - Z);
          l += s[p].z * qa_ex2(s[p].x - z);
#pragma unroll
          for (int e = 0; e < kE2; ++e) acc[e] += v[p][e] * f;
        }
        qa_put<T, kE2>(a, r, t * kRows + own, h, lane & 15, z, Z, m, l, acc);
      }
      __syncwarp();
    }
  }
  for (int first = blockIdx.y * step, k = 0; first + k < kRows; k + 1 < step ? ++k : (k = 0, first += gridDim.y * step)) {
    const int row = first + k;
    uint32_t many = __ballot_sync(~0u, row < my_rows && my_parts > kQmAlone);
    if (many == 0) return;
    auto slot = [&](int c0, int p) { return (static_cast<int64_t>(c0 + p) * 2 + (p == 0 ? 1 : 0)) * kRows + row; };
    auto maxima = [&](int c0, int parts, int p0, int step, float& m, float& M) {
      for (int p = p0; p < parts; p += step) {
        const float4 s = a.cta_stat[slot(c0, p)];
        m = fmaxf(m, s.x);
        M = fmaxf(M, s.y);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
      }
    };
    // sums of the parts p0, p0 + step, ... against the maxima z, Z
    auto add = [&](int c0, int parts, int p0, int step, float z, float Z, float* acc, float& l) {
#pragma unroll 5
      for (int p = p0; p < parts; p += step) {
        const int64_t at = slot(c0, p);
        const float4 s = a.cta_stat[at];
        float part[kE];
        qa_load<kE>(part, a.cta_part + at * kDim + lane * kE);
        const float f = qa_ex2(s.y - Z);
        l += s.z * qa_ex2(s.x - z);
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] += part[e] * f;
      }
    };
    for (; many; many &= many - 1) {
      const int i = __ffs(many) - 1;
      const int parts = __shfl_sync(~0u, my_parts, i);
      float m = -INFINITY, M = -INFINITY, l = 0.0f, acc[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[e] = 0.0f;
      maxima(base + i, parts, lane, 32, m, M);  // by every warp for itself: the parts are at most one per SM
      const float z = m == -INFINITY ? 0.0f : m, Z = M == -INFINITY ? 0.0f : M;
      add(base + i, parts, warp, kQmWarps, z, Z, acc, l);
      __syncthreads();  // the last unit's sums have been read
#pragma unroll
      for (int e = 0; e < kE; ++e) red[warp][lane * kE + e] = acc[e];
      if (lane == 0) red_s[warp] = l;
      __syncthreads();
      if (warp == 0) {
        l = 0.0f;
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < kQmWarps; ++w) {
          l += red_s[w];
#pragma unroll
          for (int e = 0; e < kE; ++e) acc[e] += red[w][lane * kE + e];
        }
        qa_put<T, kE>(a, __shfl_sync(~0u, mine.y, i), __shfl_sync(~0u, mine.z, i) * kRows + row,
                      __shfl_sync(~0u, mine.w, i), lane, z, Z, m, l, acc);
      }
    }
  }
}

}  // namespace drt
