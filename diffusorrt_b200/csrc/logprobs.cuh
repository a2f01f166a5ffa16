// Log probability of a given token per row of logits, with the row's entropy, the token's rank and the k
// likeliest tokens, in one pass over the logits and one small pass over their maxima.
//   c = log2(e) / T (T <= 0: log2 e), R = fl(c max x), z_j = c x_j - R (one fused operation), S = sum 2^z_j
//   logprob = ln2 (c x_t - R) - ln S      entropy = ln S - (ln2 / S) sum 2^z_j z_j
// (any R serves, as long as every term has the same; c is the same f32 number everywhere, so its rounding costs 2^-24 of
// the difference c x_t - R and no more)
//   rank    = #{x_j > x_t} + #{x_j = x_t, j < t}            (0: the row's first argmax)
//   alternatives: the k largest by (x_j, lowest j), those of probability zero left out (-1, -inf)
// The excluded token counts as x = -inf. The sums are f32 over at most a lane's share of a slice and f64
// where slices are joined.
//
// First kernel: a row is cut into segments of 4 KB (1024 f32 or 2048 16-bit logits); a warp takes a segment
// at a time (eight 16-byte loads a lane in flight), keeps a running maximum, S and the entropy sum per lane,
// and stores the segment's maximum. Second kernel, one CTA per row: joins the slices' sums, and picks the
// alternatives from the k segments with the largest maxima (equal maxima: the lowest segment). That those
// segments hold all of them: a token outside has k segments whose largest token precedes it.
//
// Measured: 1,005 rows of 152,064 bf16 logits (306 MB) with 10 alternatives 80 us, 3.8 TB/s: 61 us for the first kernel,
// bound by its instructions (69 % of the issue slots, 64 % of the exponentials' unit, 57 % of DRAM), 19 for the second,
// which reads ten segments of each row again. 32 rows of f32: 18 us, one row 10 to 11, launches and latency.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace drt {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpCtasPerSm = 4;
constexpr int kLpMaxSliceSegs = 64;  // per CTA
constexpr int kLpMaxSegs = 4096;   // segments per row: 4 million logits
constexpr int kLpCands = 512;      // candidate list of the second kernel

enum LogitType : int { LOGIT_F32 = 0, LOGIT_BF16 = 1, LOGIT_F16 = 2 };

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  const int* row_index;
  const int* tokens;
  int rows, logit_rows, vocab, top, exclude;
  float unit_log2;       // c
  int segs, slices, segs_per_slice;
  // scratch
  float4* part;          // [rows][slices] (maximum x, S, sum 2^z z, rank count as int bits)
  float* seg_max;        // [rows][segs] maximum raw logit
  // outputs
  float *logprob, *entropy;
  int* rank;
  int* top_token;
  float* top_logprob;
};

template <typename T>
__device__ __forceinline__ float lp_f32(T x) { return static_cast<float>(x); }

// 16-byte vectors of logits by type: as f32 pairs, their maximum (NaN passed over), and the bits of -inf.
template <typename T>
struct LpType;
template <>
struct LpType<float> {
  static constexpr int kVec = 4;
  static constexpr uint32_t kLow = 0xff800000u;
  static __device__ __forceinline__ float2 pair(const uint4& u, int i) {
    return i == 0 ? make_float2(__uint_as_float(u.x), __uint_as_float(u.y)) : make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ float largest(const uint4* u, int n) {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < n; ++v)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(u[v].x), __uint_as_float(u[v].y)),
                         fmaxf(__uint_as_float(u[v].z), __uint_as_float(u[v].w))));
    return m;
  }
  static __device__ __forceinline__ int above(const uint4* u, int n, float x) {  // values > x
    int c = 0;
#pragma unroll
    for (int v = 0; v < n; ++v)
      c += (__uint_as_float(u[v].x) > x) + (__uint_as_float(u[v].y) > x) + (__uint_as_float(u[v].z) > x) +
           (__uint_as_float(u[v].w) > x);
    return c;
  }
  static __device__ __forceinline__ void set_low(uint4& u, int e) {
    if (e == 0) u.x = kLow;
    if (e == 1) u.y = kLow;
    if (e == 2) u.z = kLow;
    if (e == 3) u.w = kLow;
  }
};
template <typename T, typename T2, uint32_t kLowBits>
struct LpType16 {
  static constexpr int kVec = 8;
  static constexpr uint32_t kLow = kLowBits * 0x10001u;
  static __device__ __forceinline__ float largest(const uint4* u, int n) {
    T2 m = as(kLow);
#pragma unroll
    for (int v = 0; v < n; ++v) m = __hmax2(m, __hmax2(__hmax2(as(u[v].x), as(u[v].y)), __hmax2(as(u[v].z), as(u[v].w))));
    return fmaxf(lp_f32(m.x), lp_f32(m.y));
  }
  static __device__ __forceinline__ T2 as(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
  static __device__ __forceinline__ int above(const uint4* u, int n, float x) {  // up to 32 ones a half: exact
    T2 x2, c;
    x2.x = x2.y = static_cast<T>(x);
    c.x = c.y = static_cast<T>(0.0f);
#pragma unroll
    for (int v = 0; v < n; ++v)
      c = __hadd2(c, __hadd2(__hadd2(__hgt2(as(u[v].x), x2), __hgt2(as(u[v].y), x2)),
                             __hadd2(__hgt2(as(u[v].z), x2), __hgt2(as(u[v].w), x2))));
    return static_cast<int>(lp_f32(c.x) + lp_f32(c.y));
  }
  static __device__ __forceinline__ void set_low(uint4& u, int e) {
    const uint32_t keep = e & 1 ? 0x0000ffffu : 0xffff0000u, low = kLow & ~keep;
    if (e >> 1 == 0) u.x = (u.x & keep) | low;
    if (e >> 1 == 1) u.y = (u.y & keep) | low;
    if (e >> 1 == 2) u.z = (u.z & keep) | low;
    if (e >> 1 == 3) u.w = (u.w & keep) | low;
  }
};
__device__ __forceinline__ uint32_t lp_word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }
template <>
struct LpType<__nv_bfloat16> : LpType16<__nv_bfloat16, __nv_bfloat162, 0xff80u> {
  static __device__ __forceinline__ float2 pair(const uint4& u, int i) {
    const uint32_t w = lp_word(u, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};
template <>
struct LpType<__half> : LpType16<__half, __half2, 0xfc00u> {
  static __device__ __forceinline__ float2 pair(const uint4& u, int i) { return __half22float2(as(lp_word(u, i))); }
};

// A row's geometry in 16-byte units: element i sits at position i + off of an aligned grid.
template <typename T>
__device__ __forceinline__ int lp_offset(const T* row) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// A lane's eight 16-byte vectors of segment `seg`: vector v holds the grid positions seg * kSeg + (v * 32 + lane) * kVec ..
// Positions outside the row read as -inf; the excluded token too.
template <typename T>
struct LpSeg {
  using Type = LpType<T>;
  static constexpr int kVec = Type::kVec;
  static constexpr int kSeg = 4096 / sizeof(T);
  static __device__ __forceinline__ void load(const T* row, int off, int vocab, int exclude, int seg, int lane, uint4* u) {
    const int base = seg * kSeg;
    const T* at = row - off;
    if (base >= off && base + kSeg <= off + vocab) {
#pragma unroll
      for (int v = 0; v < 8; ++v) u[v] = __ldcs(reinterpret_cast<const uint4*>(at + base + (v * 32 + lane) * kVec));
    } else {
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const int p = base + (v * 32 + lane) * kVec;
        u[v] = make_uint4(Type::kLow, Type::kLow, Type::kLow, Type::kLow);
        if (p >= off && p + kVec <= off + vocab) {
          u[v] = *reinterpret_cast<const uint4*>(at + p);
        } else if (p + kVec > off && p < off + vocab) {
          __align__(16) T e[kVec];
#pragma unroll
          for (int i = 0; i < kVec; ++i) e[i] = p + i >= off && p + i < off + vocab ? at[p + i] : static_cast<T>(-INFINITY);
          u[v] = *reinterpret_cast<const uint4*>(e);
        }
      }
    }
    const int q = exclude + off - base;  // the excluded token's place in this segment
    if (exclude >= 0 && q >= 0 && q < kSeg && (q / kVec) % 32 == lane) {
#pragma unroll
      for (int v = 0; v < 8; ++v)
        if (v == q / (32 * kVec)) Type::set_low(u[v], q % kVec);
    }
  }
};

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The next lower number of T's format (x finite or +inf, above the lowest).
template <typename T>
__device__ __forceinline__ float lp_below(float x) {
  constexpr uint32_t kUlp = std::is_same<T, __nv_bfloat16>::value ? 0x10000u : 1u;
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t h = __half_as_ushort(__float2half_rn(x));
    const uint32_t d = (h & 0x7fffu) == 0 ? 0x8001u : h & 0x8000u ? h + 1 : h - 1;
    return __half2float(__ushort_as_half(static_cast<unsigned short>(d)));
  }
  const uint32_t u = __float_as_uint(x);
  const uint32_t d = (u & 0x7fffffffu) == 0 ? 0x80000000u + kUlp : u >> 31 ? u + kUlp : u - kUlp;
  return __uint_as_float(d);
}

// R of a maximum, and R(m) - R(m2) bounded from below: by the logits where R leaves f32's range (logits near the type's
// largest magnitude), which then stands for c m itself.
__device__ __forceinline__ float lp_ref(float m, float c) { return m * c; }
__device__ __forceinline__ bool lp_huge(float r) { return fabsf(r) == INFINITY; }
__device__ __forceinline__ float lp_gap(float m, float m2, float c) {
  const float r = lp_ref(m, c), r2 = lp_ref(m2, c);
  return fmaxf(lp_huge(r) || lp_huge(r2) ? (m - m2) * c : r - r2, -1000.0f);
}

// u[v] for a v that is not known when the code is made.
__device__ __forceinline__ uint4 lp_pick(const uint4* u, int v) {
  uint4 w = u[0];
#pragma unroll
  for (int q = 1; q < 8; ++q)
    if (q == v) w = u[q];
  return w;
}

// Row r of the call and its logits: none for an index outside them.
template <typename T>
__device__ __forceinline__ const T* lp_row(const LogprobArgs& a, int r, int& vocab) {
  const int at = a.row_index ? a.row_index[r] : r;
  const bool there = at >= 0 && at < a.logit_rows;
  vocab = there ? a.vocab : 0;
  return static_cast<const T*>(a.logits) + (there ? at : 0) * a.ld;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpCtasPerSm) logprob_stats_kernel(const LogprobArgs a) {
  using Seg = LpSeg<T>;
  using Type = typename Seg::Type;
  __shared__ float4 warp_part[kLpWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  int vocab;
  const T* row = lp_row<T>(a, r, vocab);
  const int off = lp_offset(row);
  const int t = a.tokens ? a.tokens[r] : -1;
  const bool given = t >= 0 && t < vocab;
  const float xt = !given || t == a.exclude ? -INFINITY : lp_f32(row[t]);
  const float c = a.unit_log2;
  const bool low_token = xt == -INFINITY;
  const float below = low_token ? xt : lp_below<T>(xt);
  float m = -INFINITY, S = 0.0f, E = 0.0f;  // E = sum 2^z z
  int cnt = 0;
  const int seg1 = min((slice + 1) * a.segs_per_slice, a.segs);
  for (int seg = slice * a.segs_per_slice + warp; seg < seg1; seg += kLpWarps) {
    uint4 u[8];
    Seg::load(row, off, vocab, a.exclude, seg, lane, u);
    const float bm = Type::largest(u, 8);
    if (a.rank && bm >= xt) {  // else nothing of this lane's precedes the token
      const int at = seg * Seg::kSeg - off;  // token of the segment's first position
      if (low_token || (t >= at && t < at + Seg::kSeg)) {
#pragma unroll 1
        for (int v = 0; v < 8; ++v) {
          const uint4 w = lp_pick(u, v);
#pragma unroll
          for (int i = 0; i < Seg::kVec / 2; ++i) {
            const float2 x = Type::pair(w, i);
            const int tok = at + (v * 32 + lane) * Seg::kVec + 2 * i;
            cnt += (x.x > xt || (x.x == xt && tok < t)) + (x.y > xt || (x.y == xt && tok + 1 < t));
          }
        }
      } else {
        cnt += Type::above(u, 8, t < at ? xt : below);  // equal ones count before the token
      }
    }
    if (bm > m) {
      const float d = m == -INFINITY ? -1000.0f : lp_gap(m, bm, c), f = lp_ex2(d);
      E = f * __fmaf_rn(S, d, E);  // d is bounded: f is 0 there, and 0 * inf is not
      S *= f;
      m = bm;
    }
    const float R = lp_ref(m, c);
    if (m != -INFINITY && !lp_huge(R)) {
      float s0 = 0.0f, s1 = 0.0f, e0 = 0.0f, e1 = 0.0f;
#pragma unroll
      for (int v = 0; v < 8; ++v)
#pragma unroll
        for (int i = 0; i < Seg::kVec / 2; ++i) {
          const float2 x = Type::pair(u[v], i);
          const float z0 = __fmaf_rn(x.x, c, -R), z1 = __fmaf_rn(x.y, c, -R);
          const float p0 = lp_ex2(z0), p1 = lp_ex2(z1);
          s0 += p0;
          s1 += p1;
          e0 = __fmaf_rn(p0, z0, e0);
          e1 = __fmaf_rn(p1, z1, e1);
        }
      S += s0 + s1;
      float e = e0 + e1;
      if (e != e) {  // a -inf (0 * -inf: its share is 0) or a NaN (which stays)
        e = 0.0f;
#pragma unroll 1
        for (int v = 0; v < 8; ++v) {
          const uint4 w = lp_pick(u, v);
#pragma unroll
          for (int i = 0; i < Seg::kVec / 2; ++i) {
            const float2 x = Type::pair(w, i);
            const float z0 = __fmaf_rn(x.x, c, -R), z1 = __fmaf_rn(x.y, c, -R);
            e = __fmaf_rn(lp_ex2(z0), fmaxf(z0, -1000.0f), e);
            e = __fmaf_rn(lp_ex2(z1), fmaxf(z1, -1000.0f), e);
          }
        }
      }
      E += e;
    } else {
#pragma unroll 1
      for (int v = 0; v < 8; ++v) {
        const uint4 w = lp_pick(u, v);
#pragma unroll
        for (int i = 0; i < Seg::kVec / 2; ++i) {
          const float2 x = Type::pair(w, i);
          if (m == -INFINITY) {  // only -inf and NaN so far
            if (x.x != x.x || x.y != x.y) S = NAN;
          } else {
            const float z0 = (x.x - m) * c, z1 = (x.y - m) * c, p0 = lp_ex2(z0), p1 = lp_ex2(z1);
            S += p0 + p1;
            E = __fmaf_rn(p0, fmaxf(z0, -1000.0f), __fmaf_rn(p1, fmaxf(z1, -1000.0f), E));
          }
        }
      }
    }
    if (a.top > 0) {
      float sm = bm;
#pragma unroll
      for (int o = 16; o; o >>= 1) sm = fmaxf(sm, __shfl_xor_sync(~0u, sm, o));
      if (lane == 0) a.seg_max[static_cast<int64_t>(r) * a.segs + seg] = sm;
    }
  }
  auto join = [&](float m2, float S2, float E2) {
    if (m2 == -INFINITY) {
      S += S2;  // 0, or NaN
      return;
    }
    if (m == -INFINITY) {
      m = m2;
      S += S2;
      E = E2;
      return;
    }
    const float top = fmaxf(m, m2), d1 = lp_gap(m, top, c), d2 = lp_gap(m2, top, c);
    const float f1 = lp_ex2(d1), f2 = lp_ex2(d2);
    E = f1 * __fmaf_rn(S, d1, E) + f2 * __fmaf_rn(S2, d2, E2);
    S = S * f1 + S2 * f2;
    m = top;
  };
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float m2 = __shfl_xor_sync(~0u, m, o), S2 = __shfl_xor_sync(~0u, S, o), E2 = __shfl_xor_sync(~0u, E, o);
    join(m2, S2, E2);
    cnt += __shfl_xor_sync(~0u, cnt, o);
  }
  if (lane == 0) warp_part[warp] = make_float4(m, S, E, __int_as_float(cnt));
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kLpWarps; ++w) {
      const float4 p = warp_part[w];
      join(p.x, p.y, p.z);
      cnt += __float_as_int(p.w);
    }
    a.part[static_cast<int64_t>(r) * a.slices + slice] = make_float4(m, S, E, __int_as_float(cnt));
  }
  griddep_launch_dependents();
}

// Larger is earlier: by value, then by the lower token. Raw logits above -inf only.
__device__ __forceinline__ unsigned long long lp_key(float x, int tok) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(o) << 32) | static_cast<uint32_t>(~tok);
}
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// Threads per row: a batch fills the GPU with small CTAs, a few rows want their segments read at once. Both kernels, 151,936
// bf16 logits, top 8, with 512 and with 128: 1 row 9.4 and 11.1 us, 148 rows 20.9 and 21.4, 296 rows 32.0 and 33.0, 592 rows
// 52.0 and 48.9, 1,184 rows 97.7 and 87.0.
constexpr int kLpFinFewRows = 296, kLpFinMany = 128, kLpFinFew = 512;

template <typename T>
__global__ void __launch_bounds__(kLpFinFew, 2) logprob_finish_kernel(const LogprobArgs a) {
  using Seg = LpSeg<T>;
  using Type = typename Seg::Type;
  extern __shared__ __align__(16) uint8_t lp_smem[];
  unsigned long long* cand = reinterpret_cast<unsigned long long*>(lp_smem);  // [kLpCands]
  float* sm = reinterpret_cast<float*>(cand + kLpCands);                       // [segs]
  __shared__ int picked[kLpMaxTop];
  __shared__ int n_cand;
  __shared__ float cut;
  __shared__ double row_r, row_ls;
  __shared__ unsigned long long best[kLpFinFew / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads / 32;
  const int r = blockIdx.x;
  int vocab;
  const T* row = lp_row<T>(a, r, vocab);
  const int off = lp_offset(row);
  if (tid < kLpMaxTop) picked[tid] = -1;
  if (tid == 0) {
    n_cand = 0;
    cut = -INFINITY;
  }
  griddep_wait();
  if (a.top > 0)
    for (int s = tid; s < a.segs; s += threads) sm[s] = a.seg_max[static_cast<int64_t>(r) * a.segs + s];
  __syncthreads();
  if (warp == warps - 1) {
    // the row's sums in f64
    float m = -INFINITY;
    for (int s = lane; s < a.slices; s += 32) m = fmaxf(m, a.part[static_cast<int64_t>(r) * a.slices + s].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    auto ref = [&](float x) {  // what lp_ref stands for
      const float f = lp_ref(x, a.unit_log2);
      return lp_huge(f) ? static_cast<double>(x) * a.unit_log2 : static_cast<double>(f);
    };
    double S = 0.0, E = 0.0;
    int cnt = 0;
    for (int s = lane; s < a.slices; s += 32) {
      const float4 p = a.part[static_cast<int64_t>(r) * a.slices + s];
      cnt += __float_as_int(p.w);
      if (p.x == -INFINITY) {
        S += p.y;  // 0, or NaN where the slice holds only -inf and NaN
        continue;
      }
      const double d = ref(p.x) - ref(m), f = exp2(d);
      S += p.y * f;
      E += f * (p.z + p.y * fmax(d, -1e300));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      S += __shfl_xor_sync(~0u, S, o);
      E += __shfl_xor_sync(~0u, E, o);
      cnt += __shfl_xor_sync(~0u, cnt, o);
    }
    if (lane == 0) {
      const int t = a.tokens ? a.tokens[r] : -1;
      const bool given = t >= 0 && t < vocab;
      const float xt = !given || t == a.exclude ? -INFINITY : lp_f32(row[t]);
      constexpr double kLn2 = 0.69314718055994530942;
      const double ls = log(S), R = ref(m);
      const bool none = S == 0.0;  // every logit is -inf: no token can be drawn
      if (a.logprob) a.logprob[r] = none ? -INFINITY : static_cast<float>((static_cast<double>(xt) * a.unit_log2 - R) * kLn2 - ls);
      if (a.entropy) a.entropy[r] = none ? 0.0f : static_cast<float>(ls - kLn2 * E / S);
      // the off grid positions before the row read as -inf and count as earlier equals of a -inf token
      if (a.rank) a.rank[r] = given ? cnt - (xt == -INFINITY ? off : 0) : -1;
      row_r = R;
      row_ls = ls;
    }
  } else if (a.top > 0) {
    // the `top` segments of the largest maxima; the last one's maximum bounds the alternatives from below
    for (int s = tid; s < a.segs; s += threads - 32) {
      const float v = sm[s];
      if (!(v > -INFINITY)) continue;
      int before = 0;
#pragma unroll 4
      for (int q = 0; q < a.segs; ++q) before += sm[q] > v || (sm[q] == v && q < s);
      if (before < a.top) picked[before] = s;
      if (before == a.top - 1) cut = v;
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  float low = cut;
  if (low == -INFINITY) {
    // fewer segments than alternatives, and their maxima bound nothing: the `top`-th largest of the maxima of 32 / width
    // lanes' tokens does (at least two maxima for each alternative, if there are enough lanes). 1,005 rows of 32,000 bf16
    // logits with 20 alternatives: 52 us; without a bound every token was a candidate, 1,163 us.
    float* part_max = reinterpret_cast<float*>(cand);  // at most kLpMaxTop * 32
    const int n_seg = min(a.top, a.segs);
    int width = 32;                                    // lanes to a maximum
    while (width > 1 && n_seg * (32 / width) < 2 * a.top) width >>= 1;
    const int n_max = n_seg * (32 / width);
    for (int p = warp; p < n_seg; p += warps) {
      float v = -INFINITY;
      if (picked[p] >= 0) {
        uint4 u[8];
        Seg::load(row, off, vocab, a.exclude, picked[p], lane, u);
        v = Type::largest(u, 8);
      }
      for (int o = width >> 1; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
      if (lane % width == 0) part_max[p * (32 / width) + lane / width] = v;
    }
    __syncthreads();
    for (int i = tid; i < n_max; i += threads) {
      const float v = part_max[i];
      int before = 0;
      for (int q = 0; q < n_max; ++q) before += part_max[q] > v || (part_max[q] == v && q < i);
      if (before == a.top - 1) cut = v;
    }
    __syncthreads();
    low = cut;
  }
  auto offer = [&](int seg, auto&& f) {  // f(key) for this lane's tokens of `seg` that may be listed
    uint4 u[8];
    Seg::load(row, off, vocab, a.exclude, seg, lane, u);
    uint32_t hit = 0;                    // the vectors that hold one: few
#pragma unroll
    for (int v = 0; v < 8; ++v) hit |= (Type::largest(u + v, 1) >= low) << v;
    for (; hit; hit &= hit - 1) {
      const int v = __ffs(hit) - 1, tok = seg * Seg::kSeg - off + (v * 32 + lane) * Seg::kVec;
#pragma unroll 1
      for (int i = 0; i < Seg::kVec; ++i) {
        if (tok + i < 0 || tok + i >= vocab || tok + i == a.exclude) continue;
        const float x = lp_f32(row[tok + i]);
        if (x >= low && x > -INFINITY) f(lp_key(x, tok + i));
      }
    }
  };
  for (int p = warp; p < a.top; p += warps)
    if (picked[p] >= 0)
      offer(picked[p], [&](unsigned long long key) {
        const int at = atomicAdd(&n_cand, 1);
        if (at < kLpCands) cand[at] = key;
      });
  __syncthreads();
  const int n = n_cand;
  int* out_t = a.top_token + static_cast<int64_t>(r) * a.top;
  float* out_l = a.top_logprob + static_cast<int64_t>(r) * a.top;
  auto put = [&](int j, unsigned long long key) {
    out_t[j] = static_cast<int>(~static_cast<uint32_t>(key));
    out_l[j] = static_cast<float>((static_cast<double>(lp_key_value(key)) * a.unit_log2 - row_r) * 0.69314718055994530942 - row_ls);
  };
  if (n <= kLpCands) {
    for (int i = tid; i < n; i += threads) {
      const unsigned long long key = cand[i];
      int before = 0;
#pragma unroll 4
      for (int q = 0; q < n; ++q) before += cand[q] > key;
      if (before < a.top) put(before, key);
    }
  } else {
    // more equal logits than the list holds: the largest key below the last one, `top` times
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.top; ++j) {
      unsigned long long mine = 0;
      for (int p = warp; p < a.top; p += warps)
        if (picked[p] >= 0)
          offer(picked[p], [&](unsigned long long key) {
            if (key < last && key > mine) mine = key;
          });
#pragma unroll
      for (int o = 16; o; o >>= 1) mine = max(mine, __shfl_xor_sync(~0u, mine, o));
      if (lane == 0) best[warp] = mine;
      __syncthreads();
      for (int w = 0; w < warps; ++w) mine = max(mine, best[w]);
      if (tid == 0) put(j, mine);
      last = mine;
      __syncthreads();
    }
  }
  if (tid >= n && tid < a.top) {
    out_t[tid] = -1;
    out_l[tid] = -INFINITY;
  }
}

}  // namespace drt
