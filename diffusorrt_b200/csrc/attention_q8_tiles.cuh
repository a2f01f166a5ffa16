// Attention over the paged 8-bit cache for many rows: windows and prompt chunks (the mathematics and the shares are
// those of attention_q8.cuh). A unit is 256 rows (row = position * group + query head) of one request and kv head, two
// row tiles A and B of 128, and its key tiles have 128 keys.
//
// With this many rows the work is products, so it belongs on tcgen05 (kind::f16, f32 accumulators in TMEM), which
// wants the codes as f16 in shared memory. The roles, one CTA per SM:
//   expander (3 warps) bulk copies of the codes, 2 KB per 16-token group, and the blocks' scales; codes -> f16 in the
//                      128-byte swizzled K-major layout: K [keys x dims], V^T [dims x keys]
//   issuer   (1 warp)  S_X = Q_X K^T, O_X += W_X V for X = A, B; the two tiles share the expanded codes, and one
//                      tile's products run while the other's softmax does
//   softmax  (8 warps) a thread per row: S from TMEM, W = f16 weights back to TMEM over S (the A operand of the second
//                      product), O's rescaling, Q's conversion, the output
// Per 128 keys and two row tiles the tensor pipe needs 2048 clocks, the exponentials 2048 (16 a clock), and shared
// memory 320 KB = 2500 clocks (codes in and out 128, Q and K operands 128, V 64): W stays in TMEM for that reason.
// The references m and M of a row move only when they are off by more than 2^8 (weights then reach 256, far inside
// f16), so O is rescaled a few times per unit and not once per tile.
// Measured: two prompts of about 2,200 rows behind 5,500 tokens, 28 heads on 4, dim 128 (252 GFLOP): 352 us, 716 TFLOP/s;
// the tensor pipe is busy 35 % of the time and the exponentials' unit 37 %. What bounds it is the chain of one row tile:
// S out of TMEM, maximum, weights and W back (3.4 thousand clocks), then its products (1.8). 128 keys take 5.8 to 6.6
// thousand clocks for one row tile and hardly more for two in turn, so units of at most 128 rows pay most: 8 windows of 32
// rows x 2 heads over 600 to 4,600 tokens take 42 us.
// Slower, and not kept: a unit of one row tile whose keys are split between the two softmax groups (64 x 2,048 tokens: 186
// to 211 us against 177 to 200), codes read by plain loads ahead of the expansion (571 against 439 us), f32 sums one at a
// time instead of in pairs (381 against 358).
#pragma once
#include "attention_q8.cuh"

namespace drt {

constexpr int kQtRows = 256;
constexpr int kQtKeys = 128;
constexpr int kQtGroups = kQtKeys / 16;
constexpr int kQtThreads = 384;     // 12 warps, so that the softmax has 168 registers a thread
constexpr int kQtExpand = 96;       // threads of the expander
// Key tiles whose scales are kept. They are written four at a time, tiles j to j + 3 once K's tile j - 1 is expanded; that
// waited for the first product of tile j - 3, so the softmax is done with tile j - 4: seven tiles are in use at most.
constexpr int kQtMeta = 8;

template <int kDim>
struct QtCfg {
  static constexpr int kTile = kQtKeys * kDim * 2;  // f16 bytes of Q_X, K or V
  static constexpr int kRaw = kQtKeys * kDim;       // code bytes
  static constexpr int kStages = 2;                 // of K, of V, and of their codes together
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kStages * kTile, kCodes = kV + kStages * kTile;
  static constexpr int kEnd = kCodes + 2 * kRaw;
  static constexpr int kPrefix = (kQrMaxRequests + 1) * 8;  // the requests' places, before the tiles need the memory
  static constexpr size_t kSmem = 1024 + (kEnd > kPrefix ? kEnd : kPrefix);  // tiles on 1024-byte boundaries
};

struct __align__(16) QtMeta {
  float c[kQtGroups], lv[kQtGroups], iv[kQtGroups];  // per group ks scale log2(e), log2 vs, 1 / vs
  int live[kQtGroups];       // tokens of the group that the unit sees; 0 also for a missing block
  int full;                  // every group has 16
  float lv_low, lv_high;     // over the groups
};

// f16 x f16 -> f32, both K-major.
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// The low word of sdesc_kmajor_sw128's descriptor; the high word is kDescHigh for every tile here.
__device__ __forceinline__ uint32_t sdesc_low(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);

// One of the warp's threads, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Step kk (16 of the contracted index) of D (+)= A B^T. The descriptors are given by their low words, which a step only
// moves by a constant: two 16-byte units within a 128-byte atom, kAtom units from one atom to the next.
template <int kAtomA, int kAtomB>
__device__ __forceinline__ void umma_step_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, int kk, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_low + (kk >> 2) * kAtomA + (kk & 3) * 2), "r"(b_low + (kk >> 2) * kAtomB + (kk & 3) * 2), "r"(idesc),
      "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
// The same with the A operand in TMEM (lane = row, a 32-bit column = two consecutive k).
template <int kAtomB>
__device__ __forceinline__ void umma_step_ts(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, int kk, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_tmem + kk * 8), "r"(b_low + (kk >> 2) * kAtomB + (kk & 3) * 2), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t x, y, z;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(x) : "l"(y), "l"(z));
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(y));
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
  return d;
}
struct QtBars {
  uint64_t raw_full[2], raw_empty[2];   // codes of K, codes of V
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t q_full[2], s_full[2], w_full[2], pv_done[2];  // per row tile
  uint64_t meta_full[kQtMeta];
  uint32_t tmem;
  int failed;
};

template <typename T, int kDim, int kCode>
__global__ void __launch_bounds__(kQtThreads, 1) cache_attn_tiles_kernel(const CacheAttnArgs a) {
  using Cfg = QtCfg<kDim>;
  extern __shared__ __align__(1024) uint8_t qt_raw[];
  __shared__ QtBars bar;
  __shared__ QtMeta metas[kQtMeta];
  uint8_t* smem = align_smem_1024(qt_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.raw_full[i], 1);
      mbar_init(&bar.raw_empty[i], kQtExpand / 32);
      mbar_init(&bar.k_full[i], kQtExpand / 32);
      mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_full[i], kQtExpand / 32);
      mbar_init(&bar.v_empty[i], 1);
      mbar_init(&bar.q_full[i], 4);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.w_full[i], 4);
      mbar_init(&bar.pv_done[i], 1);
    }
    for (int i = 0; i < kQtMeta; ++i) mbar_init(&bar.meta_full[i], 1);
    bar.failed = 0;
    fence_mbar_init();
  }
  if (warp == 11) {
    tmem_alloc(&bar.tmem, 512);
    tmem_relinquish();
  }
  griddep_launch_dependents();
  int64_t* prefix = reinterpret_cast<int64_t*>(smem);
  const int64_t total = qa_prefix<kQtRows, kQtKeys, kQtThreads>(a, prefix);
  const int ctas = static_cast<int>(min(total, static_cast<int64_t>(gridDim.x)));
  const QaCut cut(total, max(ctas, 1));
  int64_t x = 0, x_end = 0;
  QaUnit cur = {};
  if (blockIdx.x < ctas) {
    x = cut.begin(blockIdx.x);
    x_end = cut.begin(blockIdx.x + 1);
    int hi = a.requests;
    while (hi - cur.r > 1) {
      const int mid = (cur.r + hi) >> 1;
      if (prefix[mid] <= x) cur.r = mid;
      else hi = mid;
    }
  }
  int64_t rem = x - prefix[cur.r];
  tc_fence_before();
  __syncthreads();           // prefix is done with: its memory becomes the tiles
  tc_fence_after();
  fence_proxy_async_smem();
  int kt = 0;
  if (x < x_end) {
    cur.q = cache_request(a, cur.r);
    qa_size<kQtRows, kQtKeys>(a, cur);
    while (rem >= static_cast<int64_t>(cur.L + kQaUnitCost) * a.heads) {
      rem -= static_cast<int64_t>(cur.L + kQaUnitCost) * a.heads;
      ++cur.t;
      qa_size<kQtRows, kQtKeys>(a, cur);
    }
    const int per = cur.L + kQaUnitCost;
    cur.h = static_cast<int>(rem / per);
    kt = static_cast<int>(rem - static_cast<int64_t>(cur.h) * per) - kQaUnitCost;
    if (kt < 0) {
      x -= kt;
      kt = 0;
    }
  }
  int4 owner = make_int4(0, 0, 0, 0);  // thread 0: the unit that this CTA begins and a later one ends
  const uint32_t tmem = bar.tmem;
  volatile int* failed = &bar.failed;
  // A bounded wait; the CTA gives up together when one runs out.
  auto wait = [&](uint64_t* b, uint32_t parity) {
    if (mbar_wait(b, parity & 1)) return true;
    *failed = 1;
    return false;
  };
  auto advance = [&](int tiles) {  // the share's next segment
    x += tiles + kQaUnitCost;
    kt = 0;
    if (x < x_end) qa_next<kQtRows, kQtKeys>(a, cur);
  };
  auto segment = [&] { return static_cast<int>(min(static_cast<int64_t>(cur.L - kt), x_end - x)); };
  const uint32_t smem_at = smem_u32(smem);

  if (warp == 11) {
    // ------------------------------------------------------------ issuer
    const uint32_t idesc_s = idesc_f16_f32(128, kQtKeys), idesc_o = idesc_f16_f32(128, kDim);
    uint32_t n = 0;                   // key tiles whose second product is issued
    uint32_t units[2] = {0, 0}, done[2] = {0, 0};
    bool ok = true;
    const uint32_t tm = __shfl_sync(~0u, tmem, 0);
    const uint32_t q_low = sdesc_low(smem_at + Cfg::kQ), k_low = sdesc_low(smem_at + Cfg::kK), v_low = sdesc_low(smem_at + Cfg::kV);
    auto issue_s = [&](int X, uint32_t tile) {  // S_X of key tile `tile` (a running number)
      const uint32_t ql = q_low + X * (Cfg::kTile / 16), kl = k_low + (tile % Cfg::kStages) * (Cfg::kTile / 16);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk) umma_step_ss<1024, 1024>(tm + X * 128, ql, kl, idesc_s, kk, kk != 0);
        umma_commit(&bar.s_full[X]);
      }
      __syncwarp();
    };
    while (x < x_end && ok) {
      const int tiles = segment();
      const int both = cur.q.n * a.group - cur.t * kQtRows > 128 ? 2 : 1;
      ok = wait(&bar.k_full[n % Cfg::kStages], n / Cfg::kStages);
      for (int X = 0; X < both && ok; ++X) {
        ok = wait(&bar.q_full[X], units[X]++);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
        issue_s(X, n);
      }
      if (ok && elect_one()) umma_commit(&bar.k_empty[n % Cfg::kStages]);
      for (int j = 0; j < tiles && ok; ++j, ++n) {
        const int st = n % Cfg::kStages;
        ok = wait(&bar.v_full[st], n / Cfg::kStages);
        for (int X = 0; X < both && ok; ++X) {
          ok = wait(&bar.w_full[X], done[X]++);
          if (!(ok = __all_sync(~0u, ok))) break;
          tc_fence_after();
          const uint32_t vl = v_low + st * (Cfg::kTile / 16);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kQtKeys / 16; ++kk)
              umma_step_ts<kDim * 8>(tm + 256 + X * 128, tm + X * 128, vl, idesc_o, kk, j > 0 || kk != 0);
            umma_commit(&bar.pv_done[X]);
          }
          __syncwarp();
          if (j + 1 < tiles) {
            if (X == 0) ok = __all_sync(~0u, wait(&bar.k_full[(n + 1) % Cfg::kStages], (n + 1) / Cfg::kStages));
            if (!ok) break;
            tc_fence_after();
            issue_s(X, n + 1);
          }
        }
        if (ok && elect_one()) {
          umma_commit(&bar.v_empty[st]);
          if (j + 1 < tiles) umma_commit(&bar.k_empty[(n + 1) % Cfg::kStages]);
        }
        ok = __all_sync(~0u, ok && !*failed);
      }
      advance(tiles);
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ expander
    const int ew = warp - 8;
    // 32 16-byte reads at a time, dealt to the three warps
    constexpr int kParts = Cfg::kRaw / 512, kTurns = (kParts + kQtExpand / 32 - 1) / (kQtExpand / 32);
    auto put2 = [](uint8_t* dst, uint32_t at0, uint32_t at1, const uint4& u) {
      uint4 lo, hi;
      codes_to_f16<kCode>(u.x, lo.x, lo.y);
      codes_to_f16<kCode>(u.y, lo.z, lo.w);
      codes_to_f16<kCode>(u.z, hi.x, hi.y);
      codes_to_f16<kCode>(u.w, hi.z, hi.w);
      *reinterpret_cast<uint4*>(dst + at0) = lo;
      *reinterpret_cast<uint4*>(dst + at1) = hi;
    };
    auto expand_k = [&](const uint8_t* raw, uint8_t* dst) {  // a token's 16 dimensions
      const int sub = lane / (kDim / 16), d = (lane % (kDim / 16)) * 16;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int part = ew + i * (kQtExpand / 32);
        if (part < kParts) {
          const int tok = part * (512 / kDim) + sub;
          put2(dst, sw128_offset(tok, d, kQtKeys), sw128_offset(tok, d + 8, kQtKeys),
               *reinterpret_cast<const uint4*>(raw + part * 512 + lane * 16));
        }
      }
    };
    auto expand_v = [&](const uint8_t* raw, uint8_t* dst, auto full, const QtMeta& m) {  // a dimension's 16 tokens
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int part = ew + i * (kQtExpand / 32);
        if (part < kParts) {
          const int grp = part / (kDim / 32), d = part % (kDim / 32) * 32 + lane;
          uint4 u = *reinterpret_cast<const uint4*>(raw + part * 512 + lane * 16);
          if constexpr (!decltype(full)::value) {
            const int live = m.live[grp];
            auto keep = [&](int w) {
              const int c = min(4, max(0, live - 4 * w));
              return c >= 4 ? ~0u : (1u << (8 * c)) - 1u;
            };
            u = make_uint4(u.x & keep(0), u.y & keep(1), u.z & keep(2), u.w & keep(3));
          }
          put2(dst, sw128_offset(d, grp * 16, kDim), sw128_offset(d, grp * 16 + 8, kDim), u);
        }
      }
    };
    const int block_shift = 31 - __clz(a.block);
    uint32_t n = 0;          // key tiles expanded
    bool ok = true;
    while (x < x_end && ok) {
      const int tiles = segment();
      // The first warp asks for K's codes and gives the softmax its scales, the second asks for V's. Table entries of four
      // key tiles at a time, lane = tile * 8 + group, and the next four's on their way.
      auto entry = [&](int tile0) {
        const int tok = (kt + tile0 + (lane >> 3)) * kQtKeys + (lane & 7) * 16;
        return tile0 + (lane >> 3) < tiles && tok < cur.lim ? a.tables[cur.r * a.ld_tables + (tok >> block_shift)] : -1;
      };
      const uint32_t n0 = n;
      int id = -1, id_next = ew < 2 ? entry(0) : -1;
      auto load = [&](int j, int is_v) -> bool {
        if ((j & 3) == 0) {
          id = id_next < a.blocks ? id_next : -1;
          id_next = entry(j + 4);
          if (!is_v) {
            const bool here = id >= 0;
            const int64_t at = static_cast<int64_t>(here ? id : 0) * a.heads + cur.h;
            const float k = here ? a.k_scale[at] : 0.0f, v = here ? a.v_scale[at] : 0.0f;
            const float lv = here ? log2f(v) : -INFINITY;
            const int live = here ? min(16, cur.lim - (kt + j + (lane >> 3)) * kQtKeys - (lane & 7) * 16) : 0;
            float low = lv, high = lv;
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) {
              low = fminf(low, __shfl_xor_sync(~0u, low, d));
              high = fmaxf(high, __shfl_xor_sync(~0u, high, d));
            }
            const uint32_t full = __ballot_sync(~0u, live == 16) >> (lane & 24) & 0xffu;
            if (j + (lane >> 3) < tiles) {
              QtMeta& m = metas[(n0 + j + (lane >> 3)) % kQtMeta];
              const int g = lane & 7;
              m.c[g] = k * a.scale_log2;
              m.lv[g] = lv;
              m.iv[g] = 1.0f / v;
              m.live[g] = live;
              if (g == 0) {
                m.full = full == 0xffu;
                m.lv_low = low;
                m.lv_high = high;
              }
            }
            __syncwarp();
            if ((lane & 7) == 0 && j + (lane >> 3) < tiles) mbar_arrive(&bar.meta_full[(n0 + j + (lane >> 3)) % kQtMeta]);
          }
        }
        const uint32_t nj = n0 + j;
        const int pg = __shfl_sync(~0u, id, (j & 3) * 8 + (lane & 7));
        const int tok = (kt + j) * kQtKeys + (lane & 7) * 16;
        const uint32_t have = __ballot_sync(~0u, pg >= 0) & 0xffu;
        const uint8_t* src = (is_v ? a.v_cache : a.k_cache) +
                             (((static_cast<int64_t>(pg) * a.heads + cur.h) << block_shift) + (tok & (a.block - 1))) * kDim;
        if (!__all_sync(~0u, wait(&bar.raw_empty[is_v], (nj & 1) ^ 1))) return false;
        if (lane == 0) mbar_expect_tx(&bar.raw_full[is_v], __popc(have) * 16 * kDim);
        __syncwarp();
        if (lane < 8 && pg >= 0)
          bulk_load(smem_at + Cfg::kCodes + is_v * Cfg::kRaw + lane * 16 * kDim, src, 16 * kDim, &bar.raw_full[is_v]);
        return true;
      };
      if (ew < 2) ok = load(0, ew);
      for (int j = 0; j < tiles && ok; ++j, ++n) {
        const int st = n % Cfg::kStages;
        const uint32_t round = n / Cfg::kStages;
        // K: a token's 16 dimensions to two 16-byte chunks of its row
        ok = wait(&bar.raw_full[0], n & 1) && wait(&bar.k_empty[st], (round & 1) ^ 1);
        if (!(ok = __all_sync(~0u, ok))) break;
        uint8_t* dst = smem + Cfg::kK + st * Cfg::kTile;
        const uint8_t* raw = smem + Cfg::kCodes;
        expand_k(raw, dst);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.k_full[st]);
          mbar_arrive(&bar.raw_empty[0]);
        }
        if (ew == 0 && j + 1 < tiles) ok = load(j + 1, 0);
        // V: a dimension's 16 tokens to two chunks of its row of V^T; tokens nobody sees become 0, since 0 times
        // whatever they hold need not be 0
        ok = ok && wait(&bar.raw_full[1], n & 1) && wait(&bar.v_empty[st], (round & 1) ^ 1);
        if (!(ok = __all_sync(~0u, ok))) break;
        dst = smem + Cfg::kV + st * Cfg::kTile;
        raw = smem + Cfg::kCodes + Cfg::kRaw;
        const QtMeta& m = metas[n % kQtMeta];
        if (m.full) expand_v(raw, dst, std::true_type(), m);
        else expand_v(raw, dst, std::false_type(), m);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.v_full[st]);
          mbar_arrive(&bar.raw_empty[1]);
        }
        if (ew == 1 && j + 1 < tiles) ok = load(j + 1, 1);
        ok = __all_sync(~0u, ok && !*failed);
      }
      advance(tiles);
    }
    if (!ok && ew < 2) mbar_wait(&bar.raw_full[ew], n & 1);  // a copy under way lands first (a bounded wait)
  } else {
    // ------------------------------------------------------------ softmax
    const int X = warp >> 2;
    const int r_tile = (warp & 3) * 32 + lane;       // row of the tile = TMEM lane
    const uint32_t lane_at = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lane_at + X * 128, o_at = tmem + lane_at + 256 + X * 128;
    uint32_t n = 0, mine = 0;                         // key tiles, and those of this row tile
    bool ok = true;
    while (x < x_end && ok) {
      const int tiles = segment();
      const int rows_all = cur.q.n * a.group, row = cur.t * kQtRows + X * 128 + r_tile;
      if (rows_all - cur.t * kQtRows <= X * 128) {    // nothing of this unit in tile B
        n += tiles;
        advance(tiles);
        continue;
      }
      const bool has = row < rows_all;
      const int i_row = min(row, rows_all - 1) / a.group;
      const int hq = cur.h * a.group + min(row, rows_all - 1) - i_row * a.group;
      const int lim = cache_limit(a, cur.q, i_row);
      // ---- Q_X: this thread's row as f16 (its last unit's products have read the old one)
      float f = a.scale_log2 == 0.0f ? 0.0f : 1.0f;   // takes a bf16 row's power of two back
      {
        const T* src = static_cast<const T*>(a.q) + (cur.q.row0 + i_row) * a.q_row + hq * a.q_head;
        uint4 u[kDim / 8];
        if (a.vec) {
#pragma unroll
          for (int c = 0; c < kDim / 8; ++c) u[c] = reinterpret_cast<const uint4*>(src)[c];
        } else {
#pragma unroll
          for (int c = 0; c < kDim / 8; ++c) {
            __align__(16) T v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = src[c * 8 + e];
            u[c] = *reinterpret_cast<const uint4*>(v);
          }
        }
        if constexpr (!std::is_same<T, __half>::value) {
          float mx = 0.0f;
#pragma unroll
          for (int c = 0; c < kDim / 8; ++c) {
            const T* v = reinterpret_cast<const T*>(&u[c]);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(cache_in_f32(v[e])));
          }
          const int e = mx > 0.0f && mx <= 3.402823466e38f ? max(-100, static_cast<int>((__float_as_uint(mx) >> 23) & 255) - 127) : 14;
          const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
          f = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
#pragma unroll
          for (int c = 0; c < kDim / 8; ++c) {
            const T* v = reinterpret_cast<const T*>(&u[c]);
            const uint4 w = make_uint4(f16_pair(cache_in_f32(v[0]) * up, cache_in_f32(v[1]) * up),
                                       f16_pair(cache_in_f32(v[2]) * up, cache_in_f32(v[3]) * up),
                                       f16_pair(cache_in_f32(v[4]) * up, cache_in_f32(v[5]) * up),
                                       f16_pair(cache_in_f32(v[6]) * up, cache_in_f32(v[7]) * up));
            u[c] = w;
          }
        }
        uint8_t* dst = smem + Cfg::kQ + X * Cfg::kTile;
#pragma unroll
        for (int c = 0; c < kDim / 8; ++c) *reinterpret_cast<uint4*>(dst + sw128_offset(r_tile, c * 8, 128)) = u[c];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.q_full[X]);

      float m = -INFINITY, M = -INFINITY, l = 0.0f;
      for (int j = 0; j < tiles && ok; ++j, ++n, ++mine) {
        ok = wait(&bar.meta_full[n % kQtMeta], n / kQtMeta) && wait(&bar.s_full[X], mine);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
        const QtMeta& meta = metas[n % kQtMeta];
        const int key0 = (kt + j) * kQtKeys;
        const bool edge = __any_sync(~0u, !meta.full || key0 + kQtKeys > lim);
        // ---- the tile's maxima, of the scores and of the scores with log2 vs
        float v[64], t = -INFINITY, u = -INFINITY;
        if (!edge) {
          // the later half first, so that the earlier one is in registers when the weights are written over its columns
          float c[kQtGroups], lv[kQtGroups];
#pragma unroll
          for (int g = 0; g < kQtGroups; ++g) {
            c[g] = meta.c[g] * f;
            lv[g] = meta.lv[g];
          }
#pragma unroll
          for (int half = 1; half >= 0; --half) {
            tmem_ld32x2(s_at + half * 64, v);
            float g_max[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float q[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                q[e] = fmaxf(fmaxf(v[g * 16 + e], v[g * 16 + 4 + e]), fmaxf(v[g * 16 + 8 + e], v[g * 16 + 12 + e]));
              g_max[g] = fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3]));
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float s = g_max[g] * c[half * 4 + g];
              t = fmaxf(t, s);
              u = fmaxf(u, s + lv[half * 4 + g]);
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            tmem_ld32(s_at + c * 32, v);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int g = c * 2 + hf, see = min(meta.live[g], lim - key0 - g * 16);
              float mx = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e) mx = e < see ? fmaxf(mx, v[hf * 16 + e]) : mx;
              if (mx > -INFINITY) {  // else all hidden (a scale of 0 is legal, and 0 * -inf is not a score)
                mx *= meta.c[g] * f;
                t = fmaxf(t, mx);
                u = fmaxf(u, mx + meta.lv[g]);
              }
            }
          }
        }
        // ---- move the references where they are too low
        const bool move = t > m + 8.0f || u > M + 8.0f;
        if (__any_sync(~0u, move)) {
          const float nm = move ? fmaxf(m, t) : m, nM = move ? fmaxf(M, u) : M;
          const float km = m == -INFINITY ? 0.0f : qa_ex2(m - nm), kM = M == -INFINITY ? 0.0f : qa_ex2(M - nM);
          l *= km;
          m = nm;
          M = nM;
          if (j > 0) {
            ok = __all_sync(~0u, wait(&bar.pv_done[X], mine - 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kDim; c += 32) {
              float o[32];
              tmem_ld32(o_at + c, o);
              uint32_t w[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(o[e] * kM);
              tmem_st16(o_at + c, w);
              tmem_st16(o_at + c + 16, w + 16);
            }
          }
        }
        const float z = m == -INFINITY ? 0.0f : m, Z = M == -INFINITY ? 0.0f : M;
        // ---- weights 2^(s - z) f_g, f_g = vs 2^(z - Z), over S's columns that have been read. Where every f_g lies within
        // 2^+-60 it joins the exponent, and a group's sum of weights over f_g is that of its probabilities.
        const bool near = meta.lv_low + (z - Z) >= -60.0f && meta.lv_high + (z - Z) <= 60.0f;
        const bool fast = __all_sync(~0u, near) && !edge;
        float p_sum = 0.0f;
        if (fast) {
          float c[kQtGroups], off[kQtGroups], iv[kQtGroups];
#pragma unroll
          for (int g = 0; g < kQtGroups; ++g) {
            c[g] = meta.c[g] * f;
            off[g] = meta.lv[g] - Z;
            iv[g] = meta.iv[g];
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half == 1) tmem_ld32x2(s_at + 64, v);
#pragma unroll
            for (int g2 = 0; g2 < 4; g2 += 2) {
              uint32_t w[16];
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const int g = g2 + hf, q = half * 4 + g;
                const float2 kk = make_float2(c[q], c[q]), dd = make_float2(off[q], off[q]);
                float2 s0 = make_float2(0.0f, 0.0f), s1 = s0;
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                  float2 y0 = fma2(make_float2(v[g * 16 + e], v[g * 16 + e + 1]), kk, dd);
                  float2 y1 = fma2(make_float2(v[g * 16 + e + 2], v[g * 16 + e + 3]), kk, dd);
                  y0 = make_float2(qa_ex2(y0.x), qa_ex2(y0.y));
                  y1 = make_float2(qa_ex2(y1.x), qa_ex2(y1.y));
                  s0 = add2(s0, y0);
                  s1 = add2(s1, y1);
                  w[hf * 8 + e / 2] = f16_pair(y0.x, y0.y);
                  w[hf * 8 + e / 2 + 1] = f16_pair(y1.x, y1.y);
                }
                s0 = add2(s0, s1);
                p_sum = __fmaf_rn(s0.x + s0.y, iv[q], p_sum);
              }
              tmem_st16(s_at + half * 32 + g2 * 8, w);
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            tmem_ld32(s_at + c * 32, v);
            uint32_t w[16];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int g = c * 2 + hf, see = edge ? min(meta.live[g], lim - key0 - g * 16) : 16;
              const float k = meta.c[g] * f, wt = qa_ex2(fminf(meta.lv[g] + (z - Z), 120.0f));
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const float p0 = e < see ? qa_ex2(__fmaf_rn(v[hf * 16 + e], k, -z)) : 0.0f;
                const float p1 = e + 1 < see ? qa_ex2(__fmaf_rn(v[hf * 16 + e + 1], k, -z)) : 0.0f;
                p_sum += p0 + p1;
                w[hf * 8 + e / 2] = f16_pair(p0 * wt, p1 * wt);
              }
            }
            tmem_st16(s_at + c * 16, w);
          }
        }
        l = fast ? __fmaf_rn(p_sum, qa_ex2(Z - z), l) : l + p_sum;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.w_full[X]);
        ok = __all_sync(~0u, !*failed);
      }
      // ---- output, or this share's part
      if (ok) ok = __all_sync(~0u, wait(&bar.pv_done[X], mine - 1));
      tc_fence_after();
      if (!ok) l = NAN;
      const bool begins = kt == 0, unit_done = kt + tiles == cur.L;
      const float inv = l == 0.0f ? 0.0f : qa_ex2(M - m) / l;
      const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + (begins ? 1 : 0)) * kQtRows + X * 128 + r_tile;
      T* dst = static_cast<T*>(a.out) + (cur.q.row0 + i_row) * a.out_row + hq * a.out_head;
#pragma unroll
      for (int c = 0; c < kDim / 32; ++c) {
        float v[32];
        tmem_ld32(o_at + c * 32, v);
        if (!has) continue;
        if (begins && unit_done) {
          if (a.out_vec) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              __align__(16) T w[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) w[q] = cache_out<T>(v[e + q] * inv);
              *reinterpret_cast<uint4*>(dst + c * 32 + e) = *reinterpret_cast<const uint4*>(w);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 2) qa_store2<T>(dst + c * 32 + e, v[e] * inv, v[e + 1] * inv);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(a.cta_part + part * kDim + c * 32 + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
      }
      if (has) {
        if (!(begins && unit_done)) a.cta_stat[part] = make_float4(m, M, l, 0.0f);
        else if (a.lse)
          a.lse[(cur.q.row0 + i_row) * static_cast<int64_t>(a.heads) * a.group + hq] = (m + log2f(l)) * 0.6931471805599453f;
      }
      if (begins && !unit_done)
        owner = make_int4(min(kQtRows, rows_all - cur.t * kQtRows) | cut.owner(x + cur.L - 1) << 9, cur.r, cur.t, cur.h);
      tc_fence_before();
      advance(tiles);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 11) tmem_dealloc(tmem, 512);
  if (tid == 0) a.desc[blockIdx.x] = owner;
}

}  // namespace drt
