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

#include "common.cuh"

namespace drt {

enum CacheCode : int { CACHE_INT8 = 0, CACHE_E4M3 = 1 };

// ---------------------------------------------------------------- 8-bit codes
// Two f32 as e4m3 (nearest even, saturating), x in the low byte; and two e4m3 as f32.
__device__ __forceinline__ uint32_t f32_to_e4m3x2(float x, float y) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(w)));
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}
// Two values rounded to nearest even onto the codes, saturating, NaN to 0: x in the low byte.
template <int kCode>
__device__ __forceinline__ uint32_t f32_to_codes(float x, float y) {
  x = x == x ? x : 0.0f;
  y = y == y ? y : 0.0f;
  if constexpr (kCode == CACHE_INT8) {
    const int i = __float2int_rn(fminf(127.0f, fmaxf(-127.0f, x))), j = __float2int_rn(fminf(127.0f, fmaxf(-127.0f, y)));
    return (static_cast<uint32_t>(i) & 0xffu) | ((static_cast<uint32_t>(j) & 0xffu) << 8);
  }
  return f32_to_e4m3x2(x, y);
}
// Two codes (the low bytes of w) as values.
template <int kCode>
__device__ __forceinline__ float2 codes_to_f32(uint32_t w) {
  if constexpr (kCode == CACHE_INT8)
    return make_float2(static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8)));
  return e4m3x2_to_f32(w);
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
constexpr int kPlanSlotRows = 1024;   // rows per CTA of 256 threads of plan_slots_kernel
constexpr int kPlanStageRequests = 4096;  // row starts that a CTA keeps in shared memory

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

// Position p of a request whose table is `table`: its slot, -1 for an entry that is not a block.
__device__ __forceinline__ int plan_slot(const PlanArgs& a, const int* table, int p) {
  const int b = p / a.block, id = table[b];
  const int64_t s = static_cast<int64_t>(id) * a.block + (p - b * a.block);
  return id >= 0 && s <= INT32_MAX ? static_cast<int>(s) : -1;
}

// Last r in [lo, n) with first[r] <= t (first is ascending, first[lo] <= t): runs without rows are passed.
__device__ __forceinline__ int plan_find(const int* first, int lo, int n, int t) {
  for (int i = 0; i < 4; ++i) {  // rows lie close: a few steps first
    if (lo + 1 >= n || first[lo + 1] > t) return lo;
    ++lo;
  }
  int hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// store(i, k, load(i, k)) for k < size[i + 1] - size[i] of every i < n (n <= kPlanThreads, size ascending): sizes up to 2
// by a thread, up to 256 by a warp, larger ones by the CTA. Eight loads are under way before their stores: the compiler
// may not move a load over a store that might change it, and one at a time would cost a memory latency each.
template <typename L, typename S>
__device__ __forceinline__ void plan_for_each(const int* size, int n, uint32_t* big, L&& load, S&& store) {
  constexpr int kAhead = 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int at = tid < n ? size[tid] : 0, mine = tid < n ? size[tid + 1] - at : 0;
  if (mine > 0 && mine <= 2) {
    const int v0 = load(tid, 0), v1 = mine > 1 ? load(tid, 1) : 0;
    store(tid, 0, v0);
    if (mine > 1) store(tid, 1, v1);
  }
  for (uint32_t some = __ballot_sync(~0u, mine > 2 && mine <= 256); some;) {
    int i[kAhead], count[kAhead], v[kAhead], most = 0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int l = some ? __ffs(some) - 1 : 0;
      i[j] = warp * 32 + l;
      count[j] = some ? __shfl_sync(~0u, mine, l) : 0;
      most = max(most, count[j]);
      some &= some - 1;
    }
    for (int k = lane; k < most; k += 32) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = k < count[j] ? load(i[j], k) : 0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (k < count[j]) store(i[j], k, v[j]);
    }
  }
  const uint32_t large = __ballot_sync(~0u, mine > 256);
  if (lane == 0) big[warp] = large;
  if (!__syncthreads_or(mine > 256)) return;
  for (int w = 0; w < kPlanThreads / 32; ++w)
    for (uint32_t some = big[w]; some; some &= some - 1) {
      const int i = w * 32 + __ffs(some) - 1, count = size[i + 1] - size[i];
      for (int k = tid; k < count; k += kAhead * kPlanThreads) {
        int v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) v[j] = k + j * kPlanThreads < count ? load(i, k + j * kPlanThreads) : 0;
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (k + j * kPlanThreads < count) store(i, k + j * kPlanThreads, v[j]);
      }
    }
}

// One CTA: checks, scans, tables and ring; also the slots of a call with a token a request. The scans need every request,
// and what is left is a few thousand words, so one CTA and no second pass over the GPU. Bound by latency: 64 requests of
// a token 4.9 us, 1,024 of them 6.2; 509 prompts of a quarter of a million rows 21 us.
__global__ void __launch_bounds__(kPlanThreads) plan_cache_kernel(const PlanArgs a) {
  __shared__ long long tot[3][32], all_of[3];
  __shared__ uint32_t big[kPlanThreads / 32];
  __shared__ int bad_flag, scan_w[3][32];
  __shared__ int sh_need[kPlanThreads + 1], sh_gone[kPlanThreads + 1], sh_rows[kPlanThreads + 1], sh_held[kPlanThreads];
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
  if (warp < 3) {
    long long v = tot[warp][lane];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (lane == 0) all_of[warp] = v;
  }
  __syncthreads();
  const long long rows = all_of[0], need_all = all_of[1], gone_all = all_of[2];
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
    if (tid == 0) {
      sh_need[live] = all_need;
      sh_gone[live] = all_gone;
      sh_rows[live] = base_n + all_n;
    }
    __syncthreads();
    auto in_ring = [&](long long p) {  // p is below three times the ring's size
      while (p >= a.ring_size) p -= a.ring_size;
      return static_cast<int>(p);
    };
    const long long from = static_cast<long long>(head) + base_need;
    const long long to = static_cast<long long>(head) + available + base_gone;
    plan_for_each(sh_need, live, big, [&](int i, int k) { return a.ring[in_ring(from + sh_need[i] + k)]; },
                  [&](int i, int k, int id) { a.tables[(r0 + i) * a.ld_tables + sh_held[i] + k] = id; });
    if (all_gone > 0) {
      __syncthreads();  // big is free again
      plan_for_each(sh_gone, live, big, [&](int i, int k) { return a.tables[(r0 + i) * a.ld_tables + k]; },
                    [&](int i, int k, int id) { a.ring[in_ring(to + sh_gone[i] + k)] = id; });
    }
    if (a.fill_slots) {
      __syncthreads();  // and the tables are whole
      plan_for_each(sh_rows, live, big,
                    [&](int i, int k) { return plan_slot(a, a.tables + (r0 + i) * a.ld_tables, a.start[r0 + i] + k); },
                    [&](int i, int k, int slot) {
                      a.slots[sh_rows[i] + k] = slot;
                      a.positions[sh_rows[i] + k] = a.start[r0 + i] + k;
                    });
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
  if (a.fill_slots)
    for (int t = base_n + tid; t < a.max_rows; t += kPlanThreads) a.slots[t] = a.positions[t] = -1;
}

// Slots and positions of the other calls, after plan_cache_kernel (programmatic dependent launch): a CTA per 1,024 rows
// finds the request of its first row and walks on. A quarter of a million rows: 4 us.
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
  int r = 0;
  bool found = false;
  for (int t = t0 + threadIdx.x; t < min(t0 + kPlanSlotRows, a.max_rows); t += 256) {
    if (t >= total) {
      a.slots[t] = a.positions[t] = -1;
      continue;
    }
    if (!found) {  // the first search over all requests, the next ones from there on
      int hi = a.requests;
      while (hi - r > 1) {
        const int mid = (r + hi) >> 1;
        if (first[mid] <= t) r = mid;
        else hi = mid;
      }
      found = true;
    } else {
      r = plan_find(first, r, a.requests, t);
    }
    const int p = a.start[r] + (t - first[r]);
    a.slots[t] = plan_slot(a, a.tables + r * a.ld_tables, p);
    a.positions[t] = p;
  }
}

// ---------------------------------------------------------------- append
// Rows with consecutive slots inside one block are a run; one warp or CTA takes a run of one head of K or of V:
//   amax = max |x| over the run (finite values), s = max(amax / Q, s_old if the run does not begin the block)
//   code = rn(x / s); the block's other tokens become rn(code * (s_old / s)) when s has grown
// A run that begins a block starts it anew: what the block held before is gone.
// x / s is the f32 quotient, as a tie between two codes is common (amax is a number of few bits, and so is half of it):
// x * rn(1 / s) corrected by its residual (Markstein 1990), whose error before the last rounding is below 2^-46 of it. A
// plain product moved 1.6 times as many ties to the other code. Scales outside [2^-100, 2^126], whose reciprocal or
// residual would leave the range, and runs with infinities or NaN, divide.
constexpr int kAppendThreads = 256;
constexpr int kAppendGroup = 32;  // rows whose runs a CTA looks for when the call has many, a lane each
// Up to here eight rows to a CTA, a warp each if they are runs of their own, so that a step of single tokens fills the GPU:
// 256 tokens of 8 heads 8.0 us (10.3 with 32 rows to a CTA), 1,024 of them 19 (25); runs pay for it, 1,024 rows 7.2 (4.8).
// 4,096 single tokens: 65 us with eight rows to a CTA, 62 with 32; 4,096 rows in runs: 19 and 11.
constexpr int kAppendFewRows = 1024;

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

// Four finite quotients |v| <= Q (1 + 2^-23) as codes. int8: adding 1.5 2^23 rounds to an integer (ties to even) in the
// low byte, and none leaves [-127, 127].
template <int kCode>
__device__ __forceinline__ uint32_t finite_codes4(float v0, float v1, float v2, float v3) {
  if constexpr (kCode == CACHE_INT8) {
    constexpr float kRound = 12582912.0f;
    const uint32_t lo = __byte_perm(__float_as_uint(v0 + kRound), __float_as_uint(v1 + kRound), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(v2 + kRound), __float_as_uint(v3 + kRound), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
  return f32_to_e4m3x2(v0, v1) | f32_to_e4m3x2(v2, v3) << 16;
}
__device__ __forceinline__ float2 pair_f32(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ float2 pair_f32(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
// max(m, |x|) of two packed values; a NaN stays.
__device__ __forceinline__ uint32_t pair_max(uint32_t m, uint32_t x, __half) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&m), __habs2(*reinterpret_cast<const __half2*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pair_max(uint32_t m, uint32_t x, __nv_bfloat16) {
  const __nv_bfloat162 r =
      __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&m), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// x / s from inv = rn(1 / s). The signs keep a zero's own.
__device__ __forceinline__ float quotient(float x, float s, float inv) {
  const float q = __fmul_rn(x, inv);
  return __fmaf_rn(__fmaf_rn(s, q, -x), -inv, q);
}

// A run of one or two rows by one warp, as single tokens of many requests are: eight values a lane. V's codes are
// stored byte by byte, since nothing else of their groups changes unless the scale grows.
template <typename T, int kDim, int kCode>
__device__ __forceinline__ void append_few(const AppendArgs& a, const T* x, int64_t ld, bool is_v, int h, int lane, int t, int slot,
                                           int m, int shift) {
  constexpr int kLanes = kDim / 8;  // of a row
  const int off = slot & (a.block - 1), r = lane / kLanes, c = (lane % kLanes) * 8;
  const int64_t at = static_cast<int64_t>(slot >> shift) * a.heads + h;
  float* scale = (is_v ? a.v_scale : a.k_scale) + at;
  const float s_old = off > 0 ? *scale : 0.0f;
  float v[8];
  float amax = 0.0f;
  const bool mine = r < m;
  if (mine) {
    __align__(16) T e[8];
    const T* src = x + (t + r) * ld + c;
    if (a.vec) {
      *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(src));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = src[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = cache_in_f32(e[j]);
      if (fabsf(v[j]) <= 3.402823466e38f) amax = fmaxf(amax, fabsf(v[j]));
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
  const float s = fmaxf(__fdiv_rn(amax, code_max<kCode>()), s_old);
  auto quant = [&](float y) { return s > 0.0f ? __fdiv_rn(y, s) : 0.0f; };
  uint8_t* dst = (is_v ? a.v_cache : a.k_cache) + at * (static_cast<int64_t>(a.block) * kDim);
  if (off > 0 && s > s_old) {  // every code of the block under the new scale; the run's own follow
    const float ratio = __fdiv_rn(s_old, s);
    auto again4 = [&](uint32_t w) {
      const float2 p = codes_to_f32<kCode>(w & 0xffffu), q = codes_to_f32<kCode>(w >> 16);
      return f32_to_codes<kCode>(p.x * ratio, p.y * ratio) | f32_to_codes<kCode>(q.x * ratio, q.y * ratio) << 16;
    };
    uint4* p = reinterpret_cast<uint4*>(dst);
#pragma unroll 4
    for (int i = lane; i < a.block * kDim / 16; i += 32) {
      const uint4 o = p[i];
      p[i] = make_uint4(again4(o.x), again4(o.y), again4(o.z), again4(o.w));
    }
    __syncwarp();
  }
  if (mine) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = f32_to_codes<kCode>(quant(v[2 * j]), quant(v[2 * j + 1]));
    const int tok = off + r;
    if (!is_v) {
      *reinterpret_cast<uint2*>(dst + tok * kDim + c) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    } else {
      uint8_t* p = dst + ((tok / 16) * kDim + c) * 16 + tok % 16;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j * 16] = static_cast<uint8_t>(w[j / 2] >> (8 * (j & 1)));
    }
  }
  if (lane == 0) *scale = s;
}

// A longer run by the CTA. Its rows are read once, eight values a thread and turn: K's stay in registers until the scale is
// known, V's go to shared memory and are read back by columns, two dimensions of 16 tokens a thread. Runs with an infinity
// or a NaN, or with a scale outside the range above, take the checked conversions; the other ones (seven instructions a value)
// need none. Measured: two prompts of 14,500 rows together, 4 heads of 128, 45 MB read and written: 23 us (1.9 TB/s), bound
// by its instructions and the waits between reading and converting (56 % of the issue slots); 64 single tokens of 8 heads 5.
template <typename T, int kDim, int kCode>
__global__ void __launch_bounds__(kAppendThreads) append_cache_kernel(const AppendArgs a) {
  constexpr int kPitch = kDim + 8;
  constexpr int kTurns = 128 * kDim / 8 / kAppendThreads;
  __shared__ __align__(16) T sx[128 * kPitch];
  __shared__ float red[kAppendThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const T* x = static_cast<const T*>(is_v ? a.v : a.k) + h * (is_v ? a.v_head : a.k_head);
  const int64_t ld = is_v ? a.v_row : a.k_row;
  const int64_t total = a.blocks * a.block;
  const int g0 = blockIdx.x * a.group, rows = min(a.group, a.rows - g0);
  // which of the rows begin a run, and of one or two rows or of more: one lane each, in every warp
  const int shift = 31 - __clz(a.block);
  bool begins = false;
  int my_slot = -1, my_rows = 1;
  if (lane < rows) {
    const int t = g0 + lane;
    my_slot = a.slots[t];
    const int before = t > 0 ? a.slots[t - 1] : -1;
    const int next = t + 1 < a.rows ? a.slots[t + 1] : -1, third = t + 2 < a.rows ? a.slots[t + 2] : -1;
    const int off = my_slot & (a.block - 1);
    begins = my_slot >= 0 && my_slot < total && (off == 0 || before != my_slot - 1);
    if (off + 1 < a.block && next == my_slot + 1) my_rows = off + 2 < a.block && third == my_slot + 2 ? 3 : 2;
  }
  uint32_t few = __ballot_sync(~0u, begins && my_rows <= 2);
  for (int k = 0; few; ++k, few &= few - 1) {  // dealt to the warps
    if (k % (kAppendThreads / 32) != warp) continue;
    const int q = __ffs(few) - 1;
    append_few<T, kDim, kCode>(a, x, ld, is_v, h, lane, g0 + q, __shfl_sync(~0u, my_slot, q), __shfl_sync(~0u, my_rows, q), shift);
  }
  for (uint32_t runs = __ballot_sync(~0u, begins && my_rows > 2); runs; runs &= runs - 1) {
    const int q = __ffs(runs) - 1, t = g0 + q;
    const int slot = __shfl_sync(~0u, my_slot, q), off = slot & (a.block - 1);
    const int64_t b = slot >> shift;
    int m = 0;  // the run's rows: how far the slots go on by one
    const int most = min(a.block - off, a.rows - t);
    for (int i0 = 0; i0 < most; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t no = __ballot_sync(~0u, i >= most || a.slots[min(t + i, a.rows - 1)] != slot + i);
      m = i0 + (no ? __ffs(no) - 1 : 32);
      if (no) break;
    }
    float* scale = (is_v ? a.v_scale : a.k_scale) + b * a.heads + h;
    const float s_old = off > 0 ? *scale : 0.0f;
    // ---- the run's values, and their largest magnitude
    uint4 mine[kTurns];
    uint32_t packed = 0;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int i = tid + u * kAppendThreads, r = i / (kDim / 8), c = (i % (kDim / 8)) * 8;
      mine[u] = make_uint4(0, 0, 0, 0);
      if (r < m) {
        if (a.vec) {
          mine[u] = __ldg(reinterpret_cast<const uint4*>(x + (t + r) * ld + c));
        } else {
          __align__(16) T e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = x[(t + r) * ld + c + j];
          mine[u] = *reinterpret_cast<const uint4*>(e);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int i = tid + u * kAppendThreads, r = i / (kDim / 8), c = (i % (kDim / 8)) * 8;
      packed = pair_max(packed, mine[u].x, T());
      packed = pair_max(packed, mine[u].y, T());
      packed = pair_max(packed, mine[u].z, T());
      packed = pair_max(packed, mine[u].w, T());
      if (is_v && r < m) *reinterpret_cast<uint4*>(sx + r * kPitch + c) = mine[u];
    }
    auto reduce = [&](float v) {  // the CTA's maximum
#pragma unroll
      for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
      if (lane == 0) red[warp] = v;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kAppendThreads / 32; ++w) v = fmaxf(v, red[w]);
      return v;
    };
    const float2 two = pair_f32(packed, T());
    // a NaN anywhere shows as an infinity here, as an infinity does
    float amax = reduce(two.x == two.x && two.y == two.y ? fmaxf(two.x, two.y) : INFINITY);
    const bool finite = amax <= 3.402823466e38f;
    if (!finite) {
      float v = 0.0f;
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        const uint32_t w[4] = {mine[u].x, mine[u].y, mine[u].z, mine[u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = pair_f32(w[j], T());
          if (fabsf(p.x) <= 3.402823466e38f) v = fmaxf(v, fabsf(p.x));
          if (fabsf(p.y) <= 3.402823466e38f) v = fmaxf(v, fabsf(p.y));
        }
      }
      __syncthreads();  // red has been read
      amax = reduce(v);
    }
    const float s = fmaxf(__fdiv_rn(amax, code_max<kCode>()), s_old);
    const bool grew = off > 0 && s > s_old;
    const float ratio = grew ? __fdiv_rn(s_old, s) : 1.0f;
    const bool plain = finite && s >= 0x1p-100f && s <= 0x1p126f;
    const float inv = plain ? __fdiv_rn(1.0f, s) : 0.0f;
    auto fast4 = [&](float v0, float v1, float v2, float v3) {
      return finite_codes4<kCode>(quotient(v0, s, inv), quotient(v1, s, inv), quotient(v2, s, inv), quotient(v3, s, inv));
    };
    auto checked4 = [&](float v0, float v1, float v2, float v3) {  // of quotients already taken
      return f32_to_codes<kCode>(v0, v1) | f32_to_codes<kCode>(v2, v3) << 16;
    };
    auto quant = [&](float v) { return s > 0.0f ? __fdiv_rn(v, s) : 0.0f; };
    auto again4 = [&](uint32_t w) {  // four codes of the block's other tokens under the new scale
      const float2 p = codes_to_f32<kCode>(w & 0xffffu), q2 = codes_to_f32<kCode>(w >> 16);
      return checked4(p.x * ratio, p.y * ratio, q2.x * ratio, q2.y * ratio);
    };
    uint8_t* dst = (is_v ? a.v_cache : a.k_cache) + (b * a.heads + h) * (static_cast<int64_t>(a.block) * kDim);
    if (!is_v) {
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        const int i = tid + u * kAppendThreads, r = i / (kDim / 8), c = (i % (kDim / 8)) * 8;
        if (r >= m) continue;
        const float2 p0 = pair_f32(mine[u].x, T()), p1 = pair_f32(mine[u].y, T());
        const float2 p2 = pair_f32(mine[u].z, T()), p3 = pair_f32(mine[u].w, T());
        uint2 w;
        if (plain) {
          w.x = fast4(p0.x, p0.y, p1.x, p1.y);
          w.y = fast4(p2.x, p2.y, p3.x, p3.y);
        } else {
          w.x = checked4(quant(p0.x), quant(p0.y), quant(p1.x), quant(p1.y));
          w.y = checked4(quant(p2.x), quant(p2.y), quant(p3.x), quant(p3.y));
        }
        *reinterpret_cast<uint2*>(dst + (off + r) * kDim + c) = w;
      }
      if (grew)  // the block's other tokens
        for (int i = tid; i < (a.block - m) * (kDim / 16); i += kAppendThreads) {
          const int j = i / (kDim / 16), tok = j < off ? j : j + m;
          uint4* p = reinterpret_cast<uint4*>(dst + tok * kDim + (i % (kDim / 16)) * 16);
          const uint4 o = *p;
          *p = make_uint4(again4(o.x), again4(o.y), again4(o.z), again4(o.w));
        }
    } else {
      // 16 tokens of two dimensions at a time; groups that the run fills in part keep their other codes
      const int first = grew ? 0 : off / 16, last = grew ? a.block / 16 : (off + m + 15) / 16;
      for (int i = tid; i < (last - first) * (kDim / 2); i += kAppendThreads) {
        const int grp = first + i / (kDim / 2), d = (i % (kDim / 2)) * 2;
        uint4* p = reinterpret_cast<uint4*>(dst + (grp * kDim + d) * 16);
        const int lo = off - grp * 16, hi = lo + m;  // the run's tokens within this group
        uint32_t w[2][4];
        if (plain && lo <= 0 && hi >= 16) {
          const T* e = sx - lo * kPitch + d;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = pair_f32(*reinterpret_cast<const uint32_t*>(e + (j * 4 + k) * kPitch), T());
            w[0][j] = fast4(v[0].x, v[1].x, v[2].x, v[3].x);
            w[1][j] = fast4(v[0].y, v[1].y, v[2].y, v[3].y);
          }
        } else {
          const uint4 o0 = p[0], o1 = p[1];
          const uint32_t old[2][4] = {{o0.x, o0.y, o0.z, o0.w}, {o1.x, o1.y, o1.z, o1.w}};
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              w[k][j] = grew ? again4(old[k][j]) : old[k][j];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int tok = j * 4 + e;
                if (tok >= lo && tok < hi) {
                  const uint32_t c = f32_to_codes<kCode>(quant(cache_in_f32(sx[(tok - lo) * kPitch + d + k])), 0.0f) & 0xffu;
                  w[k][j] = (w[k][j] & ~(0xffu << (8 * e))) | c << (8 * e);
                }
              }
            }
        }
        p[0] = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
        p[1] = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
      }
    }
    __syncthreads();  // every thread has read the old scale and the reduction, and sx may be filled again
    if (tid == 0) *scale = s;
  }
}

// ---------------------------------------------------------------- read back
// Values scale * code of the listed slots, rounded once to T; a slot outside the cache gives zeros.
// One CTA takes 16 list entries of one head. V's codes of one token lie 16 bytes apart, so 16 entries that are one
// aligned group are read eight tokens of a dimension at a time. 14,500 rows of 4 heads of 128 (45 MB): 13 us, bound by its
// instructions and the L2.
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
  __shared__ float ks_s[kReadRows], vs_s[kReadRows];
  __shared__ int64_t plane_s[kReadRows];  // the entry's block and head in the cache, in bytes
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * kReadRows, h = blockIdx.y;
  const int64_t total = a.blocks * a.block;
  const int n = min(kReadRows, a.rows - r0);
  bool group = false;
  if (tid < 32) {
    int s = tid < n ? a.slots[r0 + tid] : -1;
    if (s >= total) s = -1;
    const int s0 = __shfl_sync(~0u, s, 0);
    const int64_t b = s >= 0 ? s / a.block : 0;
    if (tid < kReadRows) {
      slot_s[tid] = s >= 0 ? s - static_cast<int>(b) * a.block : -1;  // offset within the block
      plane_s[tid] = (b * a.heads + h) * (static_cast<int64_t>(a.block) * kDim);
      ks_s[tid] = s >= 0 ? a.k_scale[b * a.heads + h] : 0.0f;
      vs_s[tid] = s >= 0 ? a.v_scale[b * a.heads + h] : 0.0f;
    }
    group = __all_sync(~0u, tid >= kReadRows || (s0 >= 0 && s0 % 16 == 0 && s == s0 + tid));
  }
  group = __syncthreads_or(group);
  // K: 16 dimensions of an entry at a time
  for (int i = tid; i < n * (kDim / 16); i += kReadThreads) {
    const int e = i / (kDim / 16), c = (i % (kDim / 16)) * 16, off = slot_s[e];
    const float s = ks_s[e];
    uint4 u = make_uint4(0, 0, 0, 0);
    if (off >= 0) u = *reinterpret_cast<const uint4*>(a.k_cache + plane_s[e] + off * kDim + c);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    __align__(16) T o[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 p = codes_to_f32<kCode>((w[j >> 1] >> (16 * (j & 1))) & 0xffffu);
      o[2 * j] = cache_out<T>(p.x * s);
      o[2 * j + 1] = cache_out<T>(p.y * s);
    }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + (static_cast<int64_t>(r0 + e) * a.heads + h) * kDim + c);
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(T)); ++j) dst[j] = reinterpret_cast<const uint4*>(o)[j];
  }
  // V: two dimensions of a half group's eight tokens at a time
  constexpr int kPairs = kDim / 2;
  for (int i = tid; i < 2 * kPairs; i += kReadThreads) {
    const int d = (i % kPairs) * 2, half = i / kPairs;
    uint32_t w0[2] = {0, 0}, w1[2] = {0, 0};
    if (group) {
      const uint8_t* p = a.v_cache + plane_s[0] + (slot_s[0] / 16 * kDim + d) * 16 + half * 8;
      const uint2 u0 = *reinterpret_cast<const uint2*>(p), u1 = *reinterpret_cast<const uint2*>(p + 16);
      w0[0] = u0.x;
      w0[1] = u0.y;
      w1[0] = u1.x;
      w1[1] = u1.y;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = half * 8 + j;
      if (e >= n) break;
      const int off = slot_s[e];
      uint32_t pair = ((w0[j >> 2] >> (8 * (j & 3))) & 0xffu) | ((w1[j >> 2] >> (8 * (j & 3))) & 0xffu) << 8;
      if (!group && off >= 0) {
        const uint8_t* p = a.v_cache + plane_s[e] + (off / 16 * kDim + d) * 16 + off % 16;
        pair = p[0] | static_cast<uint32_t>(p[16]) << 8;
      }
      const float2 v = codes_to_f32<kCode>(pair);
      const float s = vs_s[e];
      T* dst = static_cast<T*>(a.v_out) + (static_cast<int64_t>(r0 + e) * a.heads + h) * kDim + d;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2*>(dst) = make_float2(v.x * s, v.y * s);
      } else {
        __align__(4) T o[2] = {cache_out<T>(v.x * s), cache_out<T>(v.y * s)};
        *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(o);
      }
    }
  }
}

}  // namespace drt
