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
  int vec;                    // q rows start on 16-byte boundaries
  // partial sums of units cut between shares
  float* part;                // [workers][2][rows of a tile][dim]
  float4* stat;               // [workers][2][rows of a tile]: m, M, l
  int4* desc;                 // [workers][2]
};

struct CacheReq {
  int row0, n, len, origin;
};

__device__ __forceinline__ CacheReq cache_request(const CacheAttnArgs& a, int r) {
  CacheReq q;
  q.row0 = min(max(a.row_start[r], 0), a.q_rows);
  q.n = max(0, min(a.row_start[r + 1], a.q_rows) - q.row0);
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// A warp owns a share: row tiles of 16 (row = position * group + query head, so a kv head's keys serve all
// of its query heads), mma.sync m16n8k16 with the codes read from its own ring of key and value tiles in
// shared memory. With 16 rows the tiles are bound by their bytes (256 B per key and head against 8 kFLOP),
// and the legacy matrix instruction needs no staging of expanded tiles: the codes become f16 operands in
// the registers of the lane that read them. tcgen05 would need them expanded in shared memory first.
//
// Lanes (g = lane / 4, q = lane % 4). The contracted dimension may be taken in any order that both operands
// share, so a lane's 16-byte read of a key's row is four k-steps' worth of its B fragment, and key n of score
// tile j is token 16 (n / 2) + 2 j + n % 2 of the 64: then the score columns that a lane holds (2q, 2q + 1 of
// each j) are tokens 16 q .. 16 q + 15, one 16-token group of V, whose codes are again one 16-byte read per
// dimension, and one block (a block holds whole groups), so a lane needs one ks and one vs per tile.
//
// The warps do not wait for one another: each issues its own copies (2 KB per group), three tiles of K or V
// ahead, and 8 warps keep about 130 KB of copies in flight per SM.
constexpr int kQrWarps = 8;
constexpr int kQrThreads = kQrWarps * 32;
constexpr int kQrRows = 16;
constexpr int kQrTile = 64;        // keys
constexpr int kQrMaxRequests = 16384;

template <int kDim>
struct QrCfg {
  static constexpr int kGroupBytes = 16 * kDim;
  static constexpr int kGroupPitch = kGroupBytes + 32;  // V reads of the four groups fall into different banks
  static constexpr int kSlot = 4 * kGroupPitch;
  static constexpr int kSlots = kDim == 128 ? 3 : 6;
  static constexpr int kRing = kSlots * kSlot;
  static constexpr size_t kSmem = static_cast<size_t>(kQrWarps) * kRing + kQrWarps * kSlots * 8;
};

// Key tiles of row tile t.
template <int kRows, int kTile>
__device__ __forceinline__ int qa_tiles(const CacheAttnArgs& a, const CacheReq& q, int t) {
  const int last = min(q.n * a.group, (t + 1) * kRows) - 1;
  return max(1, (cache_limit(a, q, last / a.group) + kTile - 1) / kTile);
}

__device__ __forceinline__ int64_t qa_share(int64_t total, int workers, int w) { return total * w / workers; }
// The share that holds tile x.
__device__ __forceinline__ int qa_owner(int64_t total, int workers, int64_t x) {
  int w = static_cast<int>(x * workers / total);
  while (w + 1 < workers && qa_share(total, workers, w + 1) <= x) ++w;
  while (w > 0 && qa_share(total, workers, w) > x) --w;
  return w;
}

// Exclusive sums of the requests' tile counts into prefix[0 .. requests], by the whole CTA.
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
      for (int t = 0; t < nt; ++t) v += qa_tiles<kRows, kTile>(a, q, t);
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

template <typename T, int kDim, int kCode>
__global__ void __launch_bounds__(kQrThreads, 1) cache_attn_rows_kernel(const CacheAttnArgs a) {
  using Cfg = QrCfg<kDim>;
  constexpr int kHalves = kDim / 64;   // 16-byte reads of a key's row per lane
  constexpr int kDTiles = kDim / 8;
  extern __shared__ __align__(128) uint8_t qr_smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(qr_smem + kQrWarps * Cfg::kRing);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, tq = lane & 3;
  uint8_t* ring = qr_smem + warp * Cfg::kRing;
  uint64_t* full = bars + warp * Cfg::kSlots;
  if (lane == 0)
    for (int i = 0; i < Cfg::kSlots; ++i) mbar_init(&full[i], 1);
  fence_mbar_init();

  int64_t* prefix = reinterpret_cast<int64_t*>(qr_smem);
  const int64_t total = qa_prefix<kQrRows, kQrTile, kQrThreads>(a, prefix);
  const int workers = static_cast<int>(min(total, static_cast<int64_t>(gridDim.x) * kQrWarps));
  const int me = warp * gridDim.x + blockIdx.x;   // few tiles spread over the CTAs first
  int64_t x = 0, x_end = 0;
  int r = 0;
  if (me < workers) {
    x = qa_share(total, workers, me);
    x_end = qa_share(total, workers, me + 1);
    int hi = a.requests;
    while (hi - r > 1) {
      const int mid = (r + hi) >> 1;
      if (prefix[mid] <= x) r = mid;
      else hi = mid;
    }
  }
  const int64_t r_first = prefix[r];
  __syncthreads();           // prefix is done with: its memory becomes the rings
  fence_proxy_async_smem();
  if (me >= workers) {
    if (lane == 0) a.desc[me * 2] = make_int4(0, 0, 0, 0);
    return;
  }

  CacheReq rq = cache_request(a, r);
  int t = 0, L = qa_tiles<kQrRows, kQrTile>(a, rq, 0);
  int64_t rem = x - r_first;
  while (rem >= static_cast<int64_t>(L) * a.heads) {
    rem -= static_cast<int64_t>(L) * a.heads;
    L = qa_tiles<kQrRows, kQrTile>(a, rq, ++t);
  }
  int h = static_cast<int>(rem / L), kt = static_cast<int>(rem % L);
  uint32_t seq_used = 0;     // ring entries consumed so far
  int4 owner = make_int4(0, 0, 0, 0), owner2 = owner;
  uint32_t issued = 0;       // ring entries asked for so far
  bool failed = false;

  while (x < x_end && !failed) {
    const int tiles = static_cast<int>(min(static_cast<int64_t>(L - kt), x_end - x));
    const int rows_all = rq.n * a.group;
    const int row_a = t * kQrRows + g, row_b = row_a + 8;
    const bool ok_a = row_a < rows_all, ok_b = row_b < rows_all;
    const int i_a = min(row_a, rows_all - 1) / a.group, i_b = min(row_b, rows_all - 1) / a.group;
    const int lim_a = cache_limit(a, rq, i_a), lim_b = cache_limit(a, rq, i_b);
    const int lim = cache_limit(a, rq, (min(rows_all, (t + 1) * kQrRows) - 1) / a.group);  // the tile's largest
    const int hq_a = h * a.group + min(row_a, rows_all - 1) - i_a * a.group;
    const int hq_b = h * a.group + min(row_b, rows_all - 1) - i_b * a.group;

    // ---- tables and scales of eight tiles at a time: lane = tile * 4 + group
    int page, page_n;
    float ks, lv, ks_n, lv_n;
    const int* table = a.tables + r * a.ld_tables;
    auto load_meta = [&](int tile0, int& pg, float& k, float& l) {
      const int tok = (tile0 + (lane >> 2)) * kQrTile + (lane & 3) * 16;
      pg = -1;
      k = 0.0f;
      l = -INFINITY;
      if (tok < lim) {
        const int id = table[tok / a.block];
        if (id >= 0 && id < a.blocks) {
          pg = id;
          k = a.k_scale[static_cast<int64_t>(id) * a.heads + h] * a.scale_log2;
          l = log2f(a.v_scale[static_cast<int64_t>(id) * a.heads + h]);
        }
      }
    };
    load_meta(kt, page, ks, lv);
    load_meta(kt + 8, page_n, ks_n, lv_n);

    auto issue = [&](int s, int done) {  // ring entry s of this segment (even: K, odd: V); `done` tiles consumed
      const int tile = s >> 1;
      const bool next = (tile >> 3) != (done >> 3);
      const int pg = __shfl_sync(~0u, next ? page_n : page, (tile & 7) * 4 + (lane & 3));
      const uint32_t e = seq_used + s;
      const int slot = e % Cfg::kSlots;
      issued = e + 1;
      const uint32_t have = __ballot_sync(~0u, pg >= 0) & 15u;
      if (lane == 0) mbar_expect_tx(&full[slot], __popc(have) * Cfg::kGroupBytes);
      __syncwarp();
      if (lane < 4 && pg >= 0) {
        const int tok = (kt + tile) * kQrTile + lane * 16;
        const uint8_t* src = ((s & 1) ? a.v_cache : a.k_cache) +
                             ((static_cast<int64_t>(pg) * a.heads + h) * a.block + tok % a.block) * kDim;
        bulk_load(smem_u32(ring + slot * Cfg::kSlot + lane * Cfg::kGroupPitch), src, Cfg::kGroupBytes, &full[slot]);
      }
    };
    const int entries = 2 * tiles;
    for (int s = 0; s < min(Cfg::kSlots, entries); ++s) issue(s, 0);

    // ---- Q fragments: lane holds dimensions 16 (q + 4 half) .. + 15 of rows g and g + 8
    uint32_t qf[kHalves * 4][4];
    float f_a = 1.0f, f_b = 1.0f;  // takes a bf16 row's power of two back
    {
      const T* qa = static_cast<const T*>(a.q) + (rq.row0 + i_a) * a.q_row + hq_a * a.q_head;
      const T* qb = static_cast<const T*>(a.q) + (rq.row0 + i_b) * a.q_row + hq_b * a.q_head;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const T* src = side ? qb : qa;
        __align__(16) T v[kHalves * 16];
#pragma unroll
        for (int hh = 0; hh < kHalves; ++hh) {
          const T* p = src + 16 * (tq + 4 * hh);
          if (a.vec) {
            reinterpret_cast<uint4*>(v)[hh * 2] = reinterpret_cast<const uint4*>(p)[0];
            reinterpret_cast<uint4*>(v)[hh * 2 + 1] = reinterpret_cast<const uint4*>(p)[1];
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[hh * 16 + i] = p[i];
          }
        }
        float up = 1.0f;
        if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
          float mx = 0.0f;
#pragma unroll
          for (int i = 0; i < kHalves * 16; ++i) mx = fmaxf(mx, fabsf(cache_in_f32(v[i])));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
          // the largest magnitude to [2^14, 2^15)
          const int e = mx > 0.0f && mx <= 3.402823466e38f ? max(-100, static_cast<int>((__float_as_uint(mx) >> 23) & 255) - 127) : 14;
          up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
          const float down = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
          if (side) f_b = down;
          else f_a = down;
        }
#pragma unroll
        for (int st = 0; st < kHalves * 4; ++st) {
          qf[st][side] = f16_pair(cache_in_f32(v[st * 4]) * up, cache_in_f32(v[st * 4 + 1]) * up);
          qf[st][2 + side] = f16_pair(cache_in_f32(v[st * 4 + 2]) * up, cache_in_f32(v[st * 4 + 3]) * up);
        }
      }
    }

    float o[kDTiles][4];
#pragma unroll
    for (int i = 0; i < kDTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m_a = -INFINITY, m_b = -INFINITY, M_a = -INFINITY, M_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;

    for (int j = 0; j < tiles; ++j) {
      if (j > 0 && (j & 7) == 0) {
        page = page_n;
        ks = ks_n;
        lv = lv_n;
        load_meta(kt + j + 8, page_n, ks_n, lv_n);
      }
      const int src_lane = (j & 7) * 4 + tq;
      const float k_mul = __shfl_sync(~0u, ks, src_lane), lv_g = __shfl_sync(~0u, lv, src_lane);
      const bool here = __shfl_sync(~0u, page, src_lane) >= 0;
      const int key0 = (kt + j) * kQrTile;

      // ---- S = Q K^T
      float s[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
      {
        const uint32_t e = seq_used + 2 * j;
        if (!failed) failed = __any_sync(~0u, !mbar_wait(&full[e % Cfg::kSlots], (e / Cfg::kSlots) & 1));
        const uint8_t* kb = ring + (e % Cfg::kSlots) * Cfg::kSlot + (g >> 1) * Cfg::kGroupPitch + (g & 1) * kDim + tq * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int hh = 0; hh < kHalves; ++hh) {
            const uint4 u = *reinterpret_cast<const uint4*>(kb + 2 * i * kDim + hh * 64);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
              uint32_t b0, b1;
              codes_to_f16<kCode>(w[st], b0, b1);
              mma_f16(s[i], qf[hh * 4 + st], b0, b1);
            }
          }
        }
        __syncwarp();
        if (!failed && 2 * j + Cfg::kSlots < entries) issue(2 * j + Cfg::kSlots, j);
      }

      // ---- softmax
      const float c_a = k_mul * f_a, c_b = k_mul * f_b;
      const int first = key0 + tq * 16;
      if (__any_sync(~0u, key0 + kQrTile > min(lim_a, lim_b) || !here)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[i][e] = here && first + 2 * i + e < lim_a ? s[i][e] * c_a : -INFINITY;
            s[i][2 + e] = here && first + 2 * i + e < lim_b ? s[i][2 + e] * c_b : -INFINITY;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[i][0] *= c_a;
          s[i][1] *= c_a;
          s[i][2] *= c_b;
          s[i][3] *= c_b;
        }
      }
      float t_a = s[0][0], t_b = s[0][2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t_a = fmaxf(t_a, fmaxf(s[i][0], s[i][1]));
        t_b = fmaxf(t_b, fmaxf(s[i][2], s[i][3]));
      }
      float u_a = t_a + lv_g, u_b = t_b + lv_g;
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        t_a = fmaxf(t_a, __shfl_xor_sync(~0u, t_a, d));
        t_b = fmaxf(t_b, __shfl_xor_sync(~0u, t_b, d));
        u_a = fmaxf(u_a, __shfl_xor_sync(~0u, u_a, d));
        u_b = fmaxf(u_b, __shfl_xor_sync(~0u, u_b, d));
      }
      const float nm_a = fmaxf(m_a, t_a), nm_b = fmaxf(m_b, t_b);
      const float nM_a = fmaxf(M_a, u_a), nM_b = fmaxf(M_b, u_b);
      // a row that has seen nothing yet keeps zeros: its reference is 0 and every term 2^-inf
      const float z_a = nm_a == -INFINITY ? 0.0f : nm_a, z_b = nm_b == -INFINITY ? 0.0f : nm_b;
      const float Z_a = nM_a == -INFINITY ? 0.0f : nM_a, Z_b = nM_b == -INFINITY ? 0.0f : nM_b;
      l_a *= qa_ex2(m_a - z_a);
      l_b *= qa_ex2(m_b - z_b);
      if (__any_sync(~0u, nM_a != M_a || nM_b != M_b)) {
        const float k_a = qa_ex2(M_a - Z_a), k_b = qa_ex2(M_b - Z_b);
#pragma unroll
        for (int i = 0; i < kDTiles; ++i) {
          o[i][0] *= k_a;
          o[i][1] *= k_a;
          o[i][2] *= k_b;
          o[i][3] *= k_b;
        }
      }
      m_a = nm_a;
      m_b = nm_b;
      M_a = nM_a;
      M_b = nM_b;
      // w = p vs / 2^(M - m): at most 1 where p is not 0; the factor alone may leave f32's range
      const float w_a = qa_ex2(fminf(lv_g + (z_a - Z_a), 120.0f)), w_b = qa_ex2(fminf(lv_g + (z_b - Z_b), 120.0f));
      uint32_t pf[4][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = qa_ex2(s[i][0] - z_a), p1 = qa_ex2(s[i][1] - z_a);
        const float p2 = qa_ex2(s[i][2] - z_b), p3 = qa_ex2(s[i][3] - z_b);
        l_a += p0 + p1;
        l_b += p2 + p3;
        pf[i >> 1][(i & 1) * 2] = f16_pair(p0 * w_a, p1 * w_a);
        pf[i >> 1][(i & 1) * 2 + 1] = f16_pair(p2 * w_b, p3 * w_b);
      }

      // ---- O += W V
      {
        const uint32_t e = seq_used + 2 * j + 1;
        if (!failed) failed = __any_sync(~0u, !mbar_wait(&full[e % Cfg::kSlots], (e / Cfg::kSlots) & 1));
        const uint8_t* vb = ring + (e % Cfg::kSlots) * Cfg::kSlot + tq * Cfg::kGroupPitch + g * 16;
        // tokens nobody sees hold anything: their codes are cleared, since 0 times a NaN code is not 0
        const int live = here ? min(16, max(0, lim - first)) : 0;
        uint32_t keep[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = min(4, max(0, live - 4 * i));
          keep[i] = n >= 4 ? ~0u : (1u << (8 * n)) - 1u;
        }
#pragma unroll
        for (int i = 0; i < kDTiles; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(vb + i * 128);
          const uint32_t w[4] = {u.x & keep[0], u.y & keep[1], u.z & keep[2], u.w & keep[3]};
#pragma unroll
          for (int st = 0; st < 4; ++st) {
            uint32_t b0, b1;
            codes_to_f16<kCode>(w[st], b0, b1);
            mma_f16(o[i], pf[st], b0, b1);
          }
        }
        __syncwarp();
        if (!failed && 2 * j + 1 + Cfg::kSlots < entries) issue(2 * j + 1 + Cfg::kSlots, j);
      }
    }
    seq_used += entries;
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      l_a += __shfl_xor_sync(~0u, l_a, d);
      l_b += __shfl_xor_sync(~0u, l_b, d);
    }
    if (failed) l_a = l_b = NAN;  // a copy did not arrive in time: the rows read as NaN

    const bool begins = kt == 0, ends = kt + tiles == L;
    if (begins && ends) {
      T* out = static_cast<T*>(a.out);
      const float n_a = l_a == 0.0f ? 0.0f : qa_ex2(M_a - m_a) / l_a, n_b = l_b == 0.0f ? 0.0f : qa_ex2(M_b - m_b) / l_b;
      T* pa = out + (rq.row0 + i_a) * a.out_row + hq_a * a.out_head + 2 * tq;
      T* pb = out + (rq.row0 + i_b) * a.out_row + hq_b * a.out_head + 2 * tq;
#pragma unroll
      for (int i = 0; i < kDTiles; ++i) {
        if (ok_a) qa_store2<T>(pa + i * 8, o[i][0] * n_a, o[i][1] * n_a);
        if (ok_b) qa_store2<T>(pb + i * 8, o[i][2] * n_b, o[i][3] * n_b);
      }
      if (a.lse && tq == 0) {
        const int64_t hq = static_cast<int64_t>(a.heads) * a.group;
        if (ok_a) a.lse[(rq.row0 + i_a) * hq + hq_a] = (m_a + log2f(l_a)) * 0.6931471805599453f;
        if (ok_b) a.lse[(rq.row0 + i_b) * hq + hq_b] = (m_b + log2f(l_b)) * 0.6931471805599453f;
      }
    } else {
      const int64_t at = (static_cast<int64_t>(me) * 2 + (begins ? 1 : 0)) * kQrRows;
      float* pa = a.part + (at + g) * kDim + 2 * tq;
      float* pb = pa + 8 * kDim;
#pragma unroll
      for (int i = 0; i < kDTiles; ++i) {
        if (ok_a) *reinterpret_cast<float2*>(pa + i * 8) = make_float2(o[i][0], o[i][1]);
        if (ok_b) *reinterpret_cast<float2*>(pb + i * 8) = make_float2(o[i][2], o[i][3]);
      }
      if (tq == 0) {
        if (ok_a) a.stat[at + g] = make_float4(m_a, M_a, l_a, 0.0f);
        if (ok_b) a.stat[at + g + 8] = make_float4(m_b, M_b, l_b, 0.0f);
      }
      if (begins) {
        owner = make_int4(min(kQrRows, rows_all - t * kQrRows), r, t, h);  // rows, request, row tile, head
        owner2.x = qa_owner(total, workers, x - kt + L - 1);
      }
    }
    x += tiles;
    kt = 0;
    if (x < x_end && ++h == a.heads) {
      h = 0;
      ++t;
      if (t * kQrRows >= rq.n * a.group) {
        t = 0;
        do rq = cache_request(a, ++r);
        while (rq.n == 0);
      }
      L = qa_tiles<kQrRows, kQrTile>(a, rq, t);
    }
  }
  if (lane == 0) {
    a.desc[me * 2] = owner;
    a.desc[me * 2 + 1] = owner2;
  }
  if (failed)  // the copies still under way land (bounded waits) before the shared memory is given up
    for (uint32_t e = issued > Cfg::kSlots ? issued - Cfg::kSlots : 0; e < issued; ++e)
      mbar_wait(&full[e % Cfg::kSlots], (e / Cfg::kSlots) & 1);
}

// Joins the partial sums of the units that shares cut: the share in which a unit begins names it, its later
// parts lie in the first slots of the shares up to the last. CTA (eight shares, rows of the tile): a warp joins
// a unit of up to kQmAlone parts, the whole CTA the longer ones, the parts dealt to its warps; either order
// is fixed by the shares alone.
constexpr int kQmThreads = 256;
constexpr int kQmWarps = kQmThreads / 32;
constexpr int kQmAlone = 16;

template <typename T, int kDim, int kRows>
__global__ void __launch_bounds__(kQmThreads) cache_attn_merge_kernel(const CacheAttnArgs a, int shares) {
  constexpr int kE = kDim / 32;  // dimensions per lane
  __shared__ float red[kQmWarps][kDim];
  __shared__ float red_s[kQmWarps][3];
  griddep_wait();
  int row = 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = blockIdx.x * kQmWarps;
  auto slot = [&](int w0, int p) { return (static_cast<int64_t>(w0 + p) * 2 + (p == 0 ? 1 : 0)) * kRows + row; };
  // sums of the parts p0, p0 + step, ... against the maxima z, Z
  auto add = [&](int w0, int parts, int p0, int step, float z, float Z, float* acc, float& l) {
#pragma unroll 4
    for (int p = p0; p < parts; p += step) {
      const int64_t at = slot(w0, p);
      const float4 s = a.stat[at];
      const float f = qa_ex2(s.y - Z);
      l += s.z * qa_ex2(s.x - z);
      const float* src = a.part + at * kDim + lane * kE;
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[e] += src[e] * f;
    }
  };
  auto put = [&](const int4& u, float z, float Z, float m, float l, const float* acc) {
    const int rr = u.z * kRows + row;
    const int i = rr / a.group, hq = u.w * a.group + rr - i * a.group;
    const int64_t out_row = min(max(a.row_start[u.y], 0), a.q_rows) + i;
    const float n = l == 0.0f ? 0.0f : qa_ex2(Z - z) / l;
    T* dst = static_cast<T*>(a.out) + out_row * a.out_row + hq * a.out_head + lane * kE;
#pragma unroll
    for (int e = 0; e < kE; e += 2) qa_store2<T>(dst + e, acc[e] * n, acc[e + 1] * n);
    if (lane == 0 && a.lse) a.lse[out_row * a.heads * a.group + hq] = (m + log2f(l)) * 0.6931471805599453f;
  };
  auto maxima = [&](int w0, int parts, int p0, int step, float& m, float& M) {
    for (int p = p0; p < parts; p += step) {
      const float4 s = a.stat[slot(w0, p)];
      m = fmaxf(m, s.x);
      M = fmaxf(M, s.y);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
      M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    }
  };
  for (row = blockIdx.y; row < kRows; row += gridDim.y) {
    if (base + warp < shares) {
      const int w0 = base + warp;
      const int4 u = a.desc[w0 * 2];
      const int parts = row < u.x ? a.desc[w0 * 2 + 1].x - w0 + 1 : 0;
      if (parts > 0 && parts <= kQmAlone) {
        float m = -INFINITY, M = -INFINITY, l = 0.0f, acc[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] = 0.0f;
        maxima(w0, parts, lane, 32, m, M);
        const float z = m == -INFINITY ? 0.0f : m, Z = M == -INFINITY ? 0.0f : M;
        add(w0, parts, 0, 1, z, Z, acc, l);
        put(u, z, Z, m, l, acc);
      }
    }
    for (int w0 = base; w0 < min(base + kQmWarps, shares); ++w0) {
      const int4 u = a.desc[w0 * 2];
      const int parts = row < u.x ? a.desc[w0 * 2 + 1].x - w0 + 1 : 0;
      if (parts <= kQmAlone) continue;
      float m = -INFINITY, M = -INFINITY, l = 0.0f, acc[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[e] = 0.0f;
      maxima(w0, parts, tid, kQmThreads, m, M);
      __syncthreads();  // the last unit's sums have been read
      if (lane == 0) {
        red_s[warp][0] = m;
        red_s[warp][1] = M;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kQmWarps; ++i) {
        m = fmaxf(m, red_s[i][0]);
        M = fmaxf(M, red_s[i][1]);
      }
      const float z = m == -INFINITY ? 0.0f : m, Z = M == -INFINITY ? 0.0f : M;
      add(w0, parts, warp, kQmWarps, z, Z, acc, l);
#pragma unroll
      for (int e = 0; e < kE; ++e) red[warp][lane * kE + e] = acc[e];
      if (lane == 0) red_s[warp][2] = l;
      __syncthreads();
      if (warp == 0) {
        l = 0.0f;
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < kQmWarps; ++w) {
          l += red_s[w][2];
#pragma unroll
          for (int e = 0; e < kE; ++e) acc[e] += red[w][lane * kE + e];
        }
        put(u, z, Z, m, l, acc);
      }
    }
  }
}

}  // namespace drt
