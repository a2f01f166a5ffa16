// Log probability of a given token per row of logits, with the row's entropy, the token's rank and the k
// likeliest tokens, in one pass over the logits and one small pass over their maxima.
//   z_j = x_j / T (T <= 0: x_j), m = max z, S = sum e^(z_j - m)
//   logprob = z_t - m - ln S      entropy = ln S - (1 / S) sum e^(z_j - m) (z_j - m)
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
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace drt {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpCtasPerSm = 4;
constexpr int kLpMaxSliceSegs = 64; // per CTA
constexpr int kLpMaxSegs = 4096;   // segments per row: 4 million logits
constexpr int kLpCands = 1024;     // candidate list of the second kernel

enum LogitType : int { LOGIT_F32 = 0, LOGIT_BF16 = 1, LOGIT_F16 = 2 };

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  const int* row_index;
  const int* tokens;
  int rows, vocab, top, exclude;
  float unit;            // 1 / T, or 1
  int segs, slices, segs_per_slice;
  // scratch
  float4* part;          // [rows][slices] (maximum z, S, entropy sum, rank count as int bits)
  float* seg_max;        // [rows][segs] maximum raw logit
  // outputs
  float *logprob, *entropy;
  int* rank;
  int* top_token;
  float* top_logprob;
};

template <typename T>
__device__ __forceinline__ float lp_f32(T x) { return static_cast<float>(x); }

// A row's geometry in 16-byte units: element i sits at position i + off of an aligned grid.
template <typename T>
__device__ __forceinline__ int lp_offset(const T* row) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// The eight 16-byte vectors of a lane of segment `seg`: x[v][e] is grid position seg * kSeg + (v * 32 + lane) * kVec + e.
// Positions outside the row read as -inf; the excluded token too.
template <typename T>
struct LpSeg {
  static constexpr int kVec = 16 / sizeof(T);
  static constexpr int kSeg = 4096 / sizeof(T);
  static constexpr int kPer = 8 * kVec;
  static __device__ __forceinline__ void load(const T* row, int off, int vocab, int exclude, int seg, int lane, float* x) {
    const int base = seg * kSeg;
    const T* at = row - off;
    const bool whole = base >= off && base + kSeg <= off + vocab;
    if (whole) {
      uint4 u[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) u[v] = __ldcs(reinterpret_cast<const uint4*>(at + base + (v * 32 + lane) * kVec));
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const T* e = reinterpret_cast<const T*>(&u[v]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[v * kVec + i] = lp_f32(e[i]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const int p = base + (v * 32 + lane) * kVec;
        if (p >= off && p + kVec <= off + vocab) {
          const uint4 u = *reinterpret_cast<const uint4*>(at + p);
          const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int i = 0; i < kVec; ++i) x[v * kVec + i] = lp_f32(e[i]);
        } else {
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            x[v * kVec + i] = p + i >= off && p + i < off + vocab ? lp_f32(at[p + i]) : -INFINITY;
        }
      }
    }
    const int q = exclude + off - base;  // the excluded token's place in this segment
    if (exclude >= 0 && q >= 0 && q < kSeg && (q / kVec) % 32 == lane) {
      const int mine = q / (32 * kVec) * kVec + q % kVec;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i == mine) x[i] = -INFINITY;
    }
  }
};

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprob_stats_kernel(const LogprobArgs a) {
  using Seg = LpSeg<T>;
  __shared__ float4 warp_part[kLpWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const T* row = static_cast<const T*>(a.logits) + static_cast<int64_t>(a.row_index ? a.row_index[r] : r) * a.ld;
  const int off = lp_offset(row);
  const int t = a.tokens ? a.tokens[r] : -1;
  const bool given = t >= 0 && t < a.vocab;
  const float xt = !given || t == a.exclude ? -INFINITY : lp_f32(row[t]);
  constexpr float kLog2e = 1.4426950408889634f;
  const float c = a.unit * kLog2e;  // e^(x unit) = 2^(x c)
  float m = -INFINITY, S = 0.0f, E = 0.0f;  // m raw; E = sum e (x - m) c, in base-2 units
  int cnt = 0;
  const int seg1 = min((slice + 1) * a.segs_per_slice, a.segs);
  for (int seg = slice * a.segs_per_slice + warp; seg < seg1; seg += kLpWarps) {
    float x[Seg::kPer];
    Seg::load(row, off, a.vocab, a.exclude, seg, lane, x);
    float bm = x[0];
#pragma unroll
    for (int i = 1; i < Seg::kPer; ++i) bm = fmaxf(bm, x[i]);
    if (a.rank) {
      const int at = seg * Seg::kSeg - off;  // token of the segment's first position
      if (t < at) {
#pragma unroll
        for (int i = 0; i < Seg::kPer; ++i) cnt += x[i] > xt;
      } else if (t >= at + Seg::kSeg) {
#pragma unroll
        for (int i = 0; i < Seg::kPer; ++i) cnt += x[i] >= xt;
      } else {
#pragma unroll
        for (int i = 0; i < Seg::kPer; ++i) {
          const int tok = at + ((i / Seg::kVec) * 32 + lane) * Seg::kVec + i % Seg::kVec;
          cnt += x[i] > xt || (x[i] == xt && tok < t);
        }
      }
    }
    if (bm > m) {
      const float d = fmaxf((m - bm) * c, -1000.0f), f = lp_ex2(d);  // bounded: f is 0 there, and 0 * inf is not
      E = f * __fmaf_rn(S, d, E);
      S *= f;
      m = bm;
    }
    if (m != -INFINITY) {
#pragma unroll
      for (int i = 0; i < Seg::kPer; ++i) {
        const float z = (x[i] - m) * c;  // exact 0 at the maximum
        const float e = lp_ex2(z);
        S += e;
        E = __fmaf_rn(e, fmaxf(z, -1000.0f), E);  // a -inf logit adds 0, a NaN one NaN through e
      }
    } else {
#pragma unroll
      for (int i = 0; i < Seg::kPer; ++i)
        if (x[i] != x[i]) S = x[i];  // only -inf and NaN so far
    }
    if (a.top > 0) {
      float sm = bm;
#pragma unroll
      for (int o = 16; o; o >>= 1) sm = fmaxf(sm, __shfl_xor_sync(~0u, sm, o));
      if (lane == 0) a.seg_max[static_cast<int64_t>(r) * a.segs + seg] = sm;
    }
  }
  auto join = [&](float m2, float S2, float E2) {
    const float top = fmaxf(m, m2);
    if (top == -INFINITY) {
      S += S2;
      return;
    }
    const float d1 = fmaxf((m - top) * c, -1000.0f), d2 = fmaxf((m2 - top) * c, -1000.0f);
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

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprob_finish_kernel(const LogprobArgs a) {
  using Seg = LpSeg<T>;
  extern __shared__ __align__(16) uint8_t lp_smem[];
  unsigned long long* cand = reinterpret_cast<unsigned long long*>(lp_smem);  // [kLpCands]
  float* sm = reinterpret_cast<float*>(cand + kLpCands);                       // [segs]
  __shared__ int picked[kLpMaxTop];
  __shared__ int n_cand;
  __shared__ float cut;
  __shared__ double row_m, row_ls;
  __shared__ unsigned long long best[kLpWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x;
  griddep_wait();
  const T* row = static_cast<const T*>(a.logits) + static_cast<int64_t>(a.row_index ? a.row_index[r] : r) * a.ld;
  const int off = lp_offset(row);
  if (tid < kLpMaxTop) picked[tid] = -1;
  if (tid == 0) {
    n_cand = 0;
    cut = -INFINITY;
  }
  if (a.top > 0)
    for (int s = tid; s < a.segs; s += kLpThreads) sm[s] = a.seg_max[static_cast<int64_t>(r) * a.segs + s];
  if (warp == 0) {
    // the row's sums in f64; a slice's maximum is raw, its entropy sum in base-2 units
    constexpr double kLn2 = 0.69314718055994530942;
    float mf = -INFINITY;
    for (int s = lane; s < a.slices; s += 32) mf = fmaxf(mf, a.part[static_cast<int64_t>(r) * a.slices + s].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) mf = fmaxf(mf, __shfl_xor_sync(~0u, mf, o));
    const double m = mf, unit = a.unit;
    double S = 0.0, E = 0.0;
    int cnt = 0;
    for (int s = lane; s < a.slices; s += 32) {
      const float4 p = a.part[static_cast<int64_t>(r) * a.slices + s];
      cnt += __float_as_int(p.w);
      if (p.x == -INFINITY) {
        S += p.y;  // 0, or NaN where the slice holds only -inf and NaN
        continue;
      }
      const double d = (static_cast<double>(p.x) - m) * unit, f = exp(d);
      S += p.y * f;
      E += f * (p.z * kLn2 + p.y * d);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      S += __shfl_xor_sync(~0u, S, o);
      E += __shfl_xor_sync(~0u, E, o);
      cnt += __shfl_xor_sync(~0u, cnt, o);
    }
    if (lane == 0) {
      const int t = a.tokens ? a.tokens[r] : -1;
      const bool given = t >= 0 && t < a.vocab;
      const float xt = !given || t == a.exclude ? -INFINITY : lp_f32(row[t]);
      const double ls = log(S);
      const bool none = S == 0.0;  // every logit is -inf: no token can be drawn
      if (a.logprob) a.logprob[r] = none ? -INFINITY : static_cast<float>((xt - m) * unit - ls);
      if (a.entropy) a.entropy[r] = none ? 0.0f : static_cast<float>(ls - E / S);
      // the off grid positions before the row read as -inf and count as earlier equals of a -inf token
      if (a.rank) a.rank[r] = given ? cnt - (xt == -INFINITY ? off : 0) : -1;
      row_m = m;
      row_ls = ls;
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  for (int s = tid; s < a.segs; s += kLpThreads) {
    const float v = sm[s];
    if (!(v > -INFINITY)) continue;
    int before = 0;
    for (int q = 0; q < a.segs; ++q) before += sm[q] > v || (sm[q] == v && q < s);
    if (before < a.top) picked[before] = s;
    if (before == a.top - 1) cut = v;
  }
  __syncthreads();
  auto offer = [&](int seg, auto&& f) {  // f(key) for this lane's tokens of `seg` that may be listed
    float x[Seg::kPer];
    Seg::load(row, off, a.vocab, a.exclude, seg, lane, x);
#pragma unroll
    for (int i = 0; i < Seg::kPer; ++i)
      if (x[i] >= cut && x[i] > -INFINITY)
        f(lp_key(x[i], seg * Seg::kSeg - off + ((i / Seg::kVec) * 32 + lane) * Seg::kVec + i % Seg::kVec));
  };
  for (int p = warp; p < a.top; p += kLpWarps)
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
    out_l[j] = static_cast<float>((lp_key_value(key) - row_m) * static_cast<double>(a.unit) - row_ls);
  };
  if (n <= kLpCands) {
    for (int i = tid; i < n; i += kLpThreads) {
      const unsigned long long key = cand[i];
      int before = 0;
      for (int q = 0; q < n; ++q) before += cand[q] > key;
      if (before < a.top) put(before, key);
    }
  } else {
    // more equal logits than the list holds: the largest key below the last one, k times
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.top; ++j) {
      unsigned long long mine = 0;
      for (int p = warp; p < a.top; p += kLpWarps)
        if (picked[p] >= 0)
          offer(picked[p], [&](unsigned long long key) {
            if (key < last && key > mine) mine = key;
          });
#pragma unroll
      for (int o = 16; o; o >>= 1) mine = max(mine, __shfl_xor_sync(~0u, mine, o));
      if (lane == 0) best[warp] = mine;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kLpWarps; ++w) mine = max(mine, best[w]);
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
