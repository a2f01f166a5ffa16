// Paged 8-bit K/V cache: block tables and slot maps from request lengths, rows appended under a scale
// per (block, head), and rows read back.
//
// Layout (a block holds `block` tokens, a multiple of 16, of one cache):
//   K codes [blocks][kv heads][block][dim]            a token's row is contiguous
//   V codes [blocks][kv heads][block / 16][dim][16]   16 tokens of one dimension are contiguous
//   scales  [blocks][kv heads] f32, one for K and one for V; value = scale * code
// Both orders are the ones the attention's matrix operands want (attention_q8.cuh): K is contracted
// over dimensions, V over tokens, and 16 codes are one 16-byte shared-memory read of a lane.
// A code is int8 in [-127, 127] or a finite float8 e4m3 (|code| <= 448). Slot = block id * block + offset.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace drt {

enum CacheCode : int { CACHE_INT8 = 0, CACHE_E4M3 = 1 };

// ---------------------------------------------------------------- 8-bit codes
template <int kCode>
__device__ __forceinline__ float code_to_f32(uint32_t byte) {
  if constexpr (kCode == CACHE_INT8) return static_cast<float>(static_cast<int8_t>(byte));
  __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
  return __half2float(__half(h));
}
// Round to nearest even onto the codes, saturating; NaN becomes 0.
template <int kCode>
__device__ __forceinline__ uint32_t f32_to_code(float v) {
  if (v != v) v = 0.0f;
  if constexpr (kCode == CACHE_INT8)
    return static_cast<uint32_t>(__float2int_rn(fminf(127.0f, fmaxf(-127.0f, v)))) & 0xffu;
  return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
template <int kCode>
__device__ __forceinline__ constexpr float code_max() {
  return kCode == CACHE_INT8 ? 127.0f : 448.0f;
}
__device__ __forceinline__ float cache_in_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float cache_in_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T cache_out(float x);
template <>
__device__ __forceinline__ float cache_out<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half cache_out<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 cache_out<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// ---------------------------------------------------------------- block tables and slot maps
// Request r holds held[r] blocks and start[r] tokens, and gets count[r] more (-1: it has finished).
//   need_r = max(0, ceil((start + count) / block) - held)   blocks taken from the ring, in request order
//   a finished request's blocks go to the ring's end, in request order
//   row_start = exclusive sum of max(count, 0); row t of request r is position p = start + t - row_start[r]
//   slot = table[r][p / block] * block + p % block
// The ring holds `available` free ids from `head` on; ids taken now lie in [head, head + available) and
// ids given back go behind them, so the two never touch one entry. All or nothing: a call that cannot be
// served writes empty slot maps and a status and changes no table, ring or held count.
constexpr int kPlanThreads = 1024;
constexpr int kPlanSlotRows = 1024;   // rows per CTA of plan_slots_kernel
constexpr int kPlanStageRequests = 4096;  // row starts that a CTA keeps in shared memory
constexpr int kPlanInlineRows = 4096;  // up to here the first kernel writes the slots itself: one launch

struct PlanArgs {
  const int *start, *count, *held_in;
  int* held_out;
  int requests;
  int* tables;
  int64_t ld_tables;
  int width, block;
  int* ring;
  int ring_size;
  const int* ring_in;
  int* ring_out;
  int *row_start, *slots, *positions;
  int max_rows;
  int *lengths, *status;
  int fill_slots;  // 1: this launch writes the slots too
};

// Last r in [0, n) with first[r] <= t (first is ascending, first[0] <= t): the empty runs before it are passed.
__device__ __forceinline__ int plan_find(const int* first, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void plan_slot(const PlanArgs& a, const int* first, int total, int t) {
  int slot = -1, pos = -1;
  if (t < total) {
    const int r = plan_find(first, a.requests, t);
    pos = a.start[r] + (t - first[r]);
    const int b = pos / a.block;
    const int64_t id = a.tables[r * a.ld_tables + b];
    const int64_t s = id * a.block + (pos - b * a.block);
    if (id >= 0 && s <= INT32_MAX) slot = static_cast<int>(s);
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

// One CTA: checks, scans, tables and ring; also the slots of a call with few rows.
__global__ void __launch_bounds__(kPlanThreads) plan_cache_kernel(const PlanArgs a) {
  __shared__ long long tot[3][32];
  __shared__ int bad_flag, scan_w[3][32];
  __shared__ int sh_need[kPlanThreads + 1], sh_gone[kPlanThreads + 1], sh_held[kPlanThreads], sh_rows[kPlanThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad_flag = 0;
  __syncthreads();
  const int head = a.ring_in[0], available = a.ring_in[1];
  long long sum[3] = {0, 0, 0};
  int bad = 0;
  if (head < 0 || head >= a.ring_size || available < 0 || available > a.ring_size) bad = -4;
  auto read = [&](int r, int& n, int& need, int& gone, int& held) {
    const int start = a.start[r], count = a.count[r];
    held = a.held_in[r];
    n = count > 0 ? count : 0;
    need = gone = 0;
    const long long end = static_cast<long long>(start) + n;
    if (start < 0 || count < -1 || held < 0 || held > a.width) bad = -4;
    else if (count < 0) gone = held;
    else if (end > static_cast<long long>(a.width) * a.block) bad = bad == 0 ? -2 : bad;
    else need = max(0, static_cast<int>((end + a.block - 1) / a.block) - held);
  };
  for (int r = tid; r < a.requests; r += kPlanThreads) {
    int n, need, gone, held;
    read(r, n, need, gone, held);
    sum[0] += n;
    sum[1] += need;
    sum[2] += gone;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
#pragma unroll
    for (int o = 16; o; o >>= 1) sum[i] += __shfl_xor_sync(~0u, sum[i], o);
    if (lane == 0) tot[i][warp] = sum[i];
  }
  if (bad) atomicMin(&bad_flag, bad);
  __syncthreads();
  long long rows = 0, need_all = 0, gone_all = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    rows += tot[0][w];
    need_all += tot[1][w];
    gone_all += tot[2][w];
  }
  int status = bad_flag;
  if (status == 0 && rows > a.max_rows) status = -3;
  if (status == 0 && available - need_all + gone_all > a.ring_size) status = -4;
  if (status == 0 && need_all > available) status = static_cast<int>(min(need_all - available, 0x7fffffffll));
  if (status != 0) {
    for (int r = tid; r < a.requests; r += kPlanThreads) {
      a.held_out[r] = a.held_in[r];
      a.row_start[r] = 0;
      a.lengths[r] = max(0, a.start[r]);
    }
    if (tid == 0) {
      a.row_start[a.requests] = 0;
      a.ring_out[0] = head;
      a.ring_out[1] = available;
      a.status[0] = status;
    }
    // plan_slots_kernel, where it runs, writes the same
    if (a.fill_slots)
      for (int t = tid; t < a.max_rows; t += kPlanThreads) a.slots[t] = a.positions[t] = -1;
    return;
  }
  __syncthreads();  // ring_in may be ring_out, held_in held_out: everything that has to be read first is
  int base_n = 0, base_need = 0, base_gone = 0;
  for (int r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
    const int r = r0 + tid;
    int v[3] = {0, 0, 0}, held = 0, x[3];
    if (r < a.requests) read(r, v[0], v[1], v[2], held);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      x[i] = v[i];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x[i], o);
        if (lane >= o) x[i] += y;
      }
      if (lane == 31) scan_w[i][warp] = x[i];
    }
    __syncthreads();
    if (warp < 3) {
      int y = scan_w[warp][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(~0u, y, o);
        if (lane >= o) y += z;
      }
      scan_w[warp][lane] = y;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) x[i] += (warp ? scan_w[i][warp - 1] : 0) - v[i];  // exclusive within the chunk
    sh_need[tid] = x[1];
    sh_gone[tid] = x[2];
    sh_held[tid] = held;
    sh_rows[tid] = base_n + x[0];
    if (r < a.requests) {
      a.row_start[r] = base_n + x[0];
      a.lengths[r] = a.count[r] < 0 ? 0 : a.start[r] + v[0];
      a.held_out[r] = a.count[r] < 0 ? 0 : held + v[1];
    }
    const int all_n = scan_w[0][31], all_need = scan_w[1][31], all_gone = scan_w[2][31];
    __syncthreads();
    const int live = min(kPlanThreads, a.requests - r0);
    for (int e = tid; e < all_need; e += kPlanThreads) {
      const int i = plan_find(sh_need, live, e);
      a.tables[(r0 + i) * a.ld_tables + sh_held[i] + (e - sh_need[i])] =
          a.ring[(static_cast<long long>(head) + base_need + e) % a.ring_size];
    }
    for (int e = tid; e < all_gone; e += kPlanThreads) {
      const int i = plan_find(sh_gone, live, e);
      a.ring[(static_cast<long long>(head) + available + base_gone + e) % a.ring_size] =
          a.tables[(r0 + i) * a.ld_tables + (e - sh_gone[i])];
    }
    base_n += all_n;
    base_need += all_need;
    base_gone += all_gone;
    __syncthreads();
  }
  if (tid == 0) {
    a.row_start[a.requests] = base_n;
    a.ring_out[0] = static_cast<int>((static_cast<long long>(head) + base_need) % a.ring_size);
    a.ring_out[1] = available - base_need + base_gone;
    a.status[0] = 0;
  }
  if (a.fill_slots) {
    __syncthreads();
    const int* first = a.requests <= kPlanThreads ? sh_rows : a.row_start;
    for (int t = tid; t < a.max_rows; t += kPlanThreads) plan_slot(a, first, base_n, t);
  }
}

// Slots and positions of a call with many rows, after plan_cache_kernel (programmatic dependent launch).
__global__ void __launch_bounds__(256) plan_slots_kernel(const PlanArgs a) {
  __shared__ int sh[kPlanStageRequests];
  griddep_wait();
  const int total = a.row_start[a.requests];
  const int* first = a.row_start;
  const int t0 = blockIdx.x * kPlanSlotRows;
  if (a.requests <= kPlanStageRequests && t0 < total) {
    for (int r = threadIdx.x; r < a.requests; r += 256) sh[r] = a.row_start[r];
    __syncthreads();
    first = sh;
  }
  for (int t = t0 + threadIdx.x; t < min(t0 + kPlanSlotRows, a.max_rows); t += 256) plan_slot(a, first, total, t);
}

// ---------------------------------------------------------------- append
// Rows with consecutive slots inside one block are a run; one CTA takes a run of one head of K or of V:
//   amax = max |x| over the run (finite values), s = max(amax / Q, s_old if the run does not begin the block)
//   code = rn(x / s); the block's other tokens become rn(code * (s_old / s)) when s has grown
// A run that begins a block starts it anew: what the block held before is gone.
// x / s is taken as x * rn(1 / s) (two roundings of 2^-24 each before the rounding onto 8 bits, so a code
// differs from the quotient's only within 2^-22 of a tie); a scale below 2^-100 divides instead, since its
// reciprocal leaves the range.
constexpr int kAppendThreads = 256;
constexpr int kAppendSingleRows = 1024;  // up to here a CTA per row: single tokens of many requests are runs of one

struct AppendArgs {
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  const int* slots;
  int rows, heads, block;
  int group;       // rows whose run starts one CTA looks for
  int64_t blocks;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int vec;         // every row of k and v starts on a 16-byte boundary
};

template <int kCode>
__device__ __forceinline__ uint32_t append_code(float x, float s, float inv) {
  if (s == 0.0f) return 0;
  return f32_to_code<kCode>(s < 0x1p-100f ? __fdiv_rn(x, s) : x * inv);
}

template <typename T, int kDim, int kCode>
__global__ void __launch_bounds__(kAppendThreads) append_cache_kernel(const AppendArgs a) {
  __shared__ __align__(16) T sx[128 * kDim];
  __shared__ float red[kAppendThreads / 32];
  const int tid = threadIdx.x;
  const int h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const T* x = static_cast<const T*>(is_v ? a.v : a.k) + h * (is_v ? a.v_head : a.k_head);
  const int64_t ld = is_v ? a.v_row : a.k_row;
  const int64_t total = a.blocks * a.block;
  const int g0 = blockIdx.x * a.group;
  for (int t = g0; t < min(g0 + a.group, a.rows); ++t) {
    const int slot = a.slots[t];
    if (slot < 0 || slot >= total) continue;
    const int64_t b = slot / a.block;
    const int off = slot - static_cast<int>(b) * a.block;
    if (t > 0 && off > 0 && a.slots[t - 1] == slot - 1) continue;  // inside another row's run
    int m = 1;
    while (off + m < a.block && t + m < a.rows && a.slots[t + m] == slot + m) ++m;
    // the run's values into shared memory, and their largest magnitude
    float amax = 0.0f;
    auto take = [&](T v) {
      const float f = fabsf(cache_in_f32(v));
      if (f <= 3.402823466e38f) amax = fmaxf(amax, f);
    };
    if (a.vec) {
      for (int i = tid; i < m * (kDim / 8); i += kAppendThreads) {
        const int r = i / (kDim / 8), c = (i % (kDim / 8)) * 8;
        const uint4 u = *reinterpret_cast<const uint4*>(x + (t + r) * ld + c);
        *reinterpret_cast<uint4*>(sx + r * kDim + c) = u;
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < 8; ++j) take(e[j]);
      }
    } else {
      for (int i = tid; i < m * kDim; i += kAppendThreads) {
        const T v = x[(t + i / kDim) * ld + i % kDim];
        sx[i] = v;
        take(v);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
    if ((tid & 31) == 0) red[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) amax = fmaxf(amax, red[w]);
    float* scale = (is_v ? a.v_scale : a.k_scale) + b * a.heads + h;
    const float s_old = off > 0 ? *scale : 0.0f;
    const float s = fmaxf(__fdiv_rn(amax, code_max<kCode>()), s_old);
    const bool grew = off > 0 && s > s_old;
    const float ratio = grew ? __fdiv_rn(s_old, s) : 1.0f;
    const float inv = __fdiv_rn(1.0f, s);
    uint8_t* dst = (is_v ? a.v_cache : a.k_cache) + (b * a.heads + h) * (static_cast<int64_t>(a.block) * kDim);
    if (!is_v) {
      // 16 codes of a token at a time; only the run's tokens unless the scale grew
      const int first = grew ? 0 : off, last = grew ? a.block : off + m;
      for (int i = tid; i < (last - first) * (kDim / 16); i += kAppendThreads) {
        const int tok = first + i / (kDim / 16), c = (i % (kDim / 16)) * 16;
        uint4* p = reinterpret_cast<uint4*>(dst + tok * kDim + c);
        uint32_t w[4];
        if (tok >= off && tok < off + m) {
          const T* e = sx + (tok - off) * kDim + c;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) w[j] |= append_code<kCode>(cache_in_f32(e[j * 4 + q]), s, inv) << (8 * q);
          }
        } else {
          const uint4 o = *p;
          const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              w[j] |= f32_to_code<kCode>(code_to_f32<kCode>((ow[j] >> (8 * q)) & 0xff) * ratio) << (8 * q);
          }
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
      // 16 tokens of a dimension at a time; chunks that the run fills in part keep their other codes
      const int first = grew ? 0 : off / 16, last = grew ? a.block / 16 : (off + m + 15) / 16;
      for (int i = tid; i < (last - first) * kDim; i += kAppendThreads) {
        const int grp = first + i / kDim, d = i % kDim;
        uint4* p = reinterpret_cast<uint4*>(dst + (grp * kDim + d) * 16);
        const int lo = off - grp * 16, hi = lo + m;  // the run's tokens within this chunk
        uint32_t w[4];
        uint4 o = make_uint4(0, 0, 0, 0);
        if (lo > 0 || hi < 16) o = *p;
        const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int tok = j * 4 + q;
            uint32_t c = (ow[j] >> (8 * q)) & 0xff;
            if (tok >= lo && tok < hi) c = append_code<kCode>(cache_in_f32(sx[(tok - lo) * kDim + d]), s, inv);
            else if (grew) c = f32_to_code<kCode>(code_to_f32<kCode>(c) * ratio);
            w[j] |= c << (8 * q);
          }
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    __syncthreads();  // every thread has read the old scale, and sx may be filled again
    if (tid == 0) *scale = s;
  }
}

// ---------------------------------------------------------------- read back
// Values scale * code of the listed slots, rounded once to T; a slot outside the cache gives zeros.
// One CTA takes 16 list entries of one head. V's codes of one token lie 16 bytes apart, so 16 entries that
// are one aligned group are read as one 16-byte load for each dimension.
constexpr int kReadThreads = 128;
constexpr int kReadRows = 16;

struct ReadArgs {
  const int* slots;
  int rows, heads, block;
  int64_t blocks;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  void *k_out, *v_out;  // [rows][heads][dim]
};

template <typename T, int kDim, int kCode>
__global__ void __launch_bounds__(kReadThreads) read_cache_kernel(const ReadArgs a) {
  __shared__ int slot_s[kReadRows];
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * kReadRows, h = blockIdx.y;
  const int64_t total = a.blocks * a.block;
  const int n = min(kReadRows, a.rows - r0);
  if (tid < kReadRows) {
    int s = tid < n ? a.slots[r0 + tid] : -1;
    if (s >= total) s = -1;
    slot_s[tid] = s;
  }
  __syncthreads();
  const int64_t plane = static_cast<int64_t>(a.block) * kDim;
  const int s0 = slot_s[0];
  bool group = n == kReadRows && s0 >= 0 && s0 % 16 == 0;
  for (int i = 1; i < n; ++i) group = group && slot_s[i] == s0 + i;
  constexpr int kPairs = kDim / 2;            // a thread writes two dimensions of a row
  constexpr int kRowsAtOnce = kReadThreads / kPairs;
  const int d = (tid % kPairs) * 2, sub = tid / kPairs;
  T* ko = static_cast<T*>(a.k_out);
  T* vo = static_cast<T*>(a.v_out);
  uint4 c0 = make_uint4(0, 0, 0, 0), c1 = c0;
  if (group) {
    const int64_t b = s0 / a.block;
    const uint8_t* p = a.v_cache + (b * a.heads + h) * plane + ((s0 - b * a.block) / 16 * kDim + d) * 16;
    c0 = *reinterpret_cast<const uint4*>(p);
    c1 = *reinterpret_cast<const uint4*>(p + 16);
  }
  const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
  for (int j = 0; j < kReadRows / kRowsAtOnce; ++j) {
    const int i = kRowsAtOnce == 1 ? j : j * kRowsAtOnce + sub;
    if (i >= n) continue;
    const int s = slot_s[i];
    float kx = 0.0f, ky = 0.0f, vx = 0.0f, vy = 0.0f;
    if (s >= 0) {
      const int64_t b = s / a.block;
      const int off = s - static_cast<int>(b) * a.block;
      const float ks = a.k_scale[b * a.heads + h], vs = a.v_scale[b * a.heads + h];
      const uint32_t kk = *reinterpret_cast<const uint16_t*>(a.k_cache + (b * a.heads + h) * plane + off * kDim + d);
      kx = code_to_f32<kCode>(kk & 0xff) * ks;
      ky = code_to_f32<kCode>(kk >> 8) * ks;
      uint32_t v0, v1;
      if (group) {
        uint32_t u0 = w0[0], u1 = w1[0];
#pragma unroll
        for (int q = 1; q < 4; ++q)
          if ((i >> 2) == q) {
            u0 = w0[q];
            u1 = w1[q];
          }
        v0 = (u0 >> (8 * (i & 3))) & 0xff;
        v1 = (u1 >> (8 * (i & 3))) & 0xff;
      } else {
        const uint8_t* p = a.v_cache + (b * a.heads + h) * plane + (off / 16 * kDim + d) * 16 + off % 16;
        v0 = p[0];
        v1 = p[16];
      }
      vx = code_to_f32<kCode>(v0) * vs;
      vy = code_to_f32<kCode>(v1) * vs;
    }
    const int64_t at = (static_cast<int64_t>(r0 + i) * a.heads + h) * kDim + d;
    ko[at] = cache_out<T>(kx);
    ko[at + 1] = cache_out<T>(ky);
    vo[at] = cache_out<T>(vx);
    vo[at + 1] = cache_out<T>(vy);
  }
}

}  // namespace drt
