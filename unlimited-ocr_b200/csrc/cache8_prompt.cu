// Attend of prompt rows (many rows per request) over the scaled 8-bit cache, on
// the 5th-generation tensor cores.
//
// Mathematics, per query head, for the rows of a tile and 128 keys at a time:
//   S = Q C^T                     f16 operands, fp32 in TMEM.  The codes C widen
//                                 to f16 exactly, and so does q times a power of
//                                 two (its largest element in [2^14, 2^15); bf16
//                                 elements under 2^-31 of that lose bits).
//   z = S * (row factor * kscale) log2 units, per 16-key group (a page's part)
//   y = z + log2 vscale
//   w = 2^(y - my + 7)            the softmax weight times the value scale, so that
//                                 both scales cost nothing per key
//   O += W D,  l += sum(w) 2^(my - log2 vscale - mz)     W rounded to f16; D the
//                                 value codes
//   out = O 2^(my - mz) / l,  lse = mz + log2(l) - 7
// mz and my are a row's own running maxima of z and y over the keys that it sees.
// They move, and l and O are rescaled, when either is passed by 8 (w stays under
// 2^15, f16's range).  So a key's product of weight and value scale keeps f16's 11
// bits down to 2^-21 of the row's largest such product, and is off by at most
// 2^-32 of that below.  Where a page's scale is 2^64 under the others it counts as
// that: w is 0 in f16 all the same, and l needs its sum.
//
// What bounds it: per 128 keys and 256 rows of 128 features, 2048 tensor cycles
// (4 * 128 * 128 * 256 flops), as many exp2 cycles, and the code conversion
// (2 * 128 * 128 elements), which is why two 128-row tiles share one CTA's keys:
// conversion and loads are paid once for 256 rows, and one tile's softmax runs
// under the other's MMAs.  Rows are (token, head of the KV head's group) pairs,
// so grouped heads share their keys' conversion too.
//
// Roles of the 13 warps: 0-3, 4-7 softmax of tile 0 / 1 (thread = row); 8-11
// read codes from the pages, widen them and write the swizzled K / V tiles
// (double buffered, the next step's codes already in registers); 12 issues the
// MMAs and owns TMEM.  TMEM, per tile: S (128 columns; W over its first 64) and O.
// (The next S overwrites W behind the product that reads it: one thread issues
// both, and its MMAs execute in order.)
//
// Measured: 8192 rows of 16 / 4 heads of 128 after 8192 tokens 1025 us, 803
// TFLOP/s, 48 % of the measured bf16 rate.  Clocks inside an earlier form of 1040
// us: a step takes 4700 cycles where its MMAs take 2048, the softmax of a tile 3300
// (its exp2 share the unit with the other tile's); the steps of the two tiles do
// not interleave fully.  One CTA an SM, 256 rows each: 28 us for 3 steps that are
// all seen in part, 38 for 6 (a window of 512), 49 / 75 / 126 for 10 / 18 / 34, so
// 20 us for the start, the end and the masked steps and 3 a step.  Ragged prompts
// with a window of 512 and 64 sinks, 10 heads: 84 us, 220 CTAs in two rounds, the
// second half full (as many equal ones: 38 and 30 us).
//
// Codes that a row does not see must not reach it: masked scores are replaced
// before use, weights of masked keys are 0, and because 0 * NaN is not, steps
// that some row sees only in part have NaN value codes replaced by 0 and marked:
// a row that does see one turns to NaN (by its mask, or with its whole tile where
// only the pair's other tile sees the step in part).

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache8_attend.cuh"
#include "tc.cuh"

namespace srswa {

constexpr int kPrThreads = 416;
constexpr int kPrConv = 8, kPrMma = 12;  // first warp of the converters, the MMA warp
constexpr int kPrKeys = 128;             // keys of a step
constexpr float kPrShift = 7.f;          // weights are kept times 2^7
constexpr float kPrRescale = 8.f;        // a row's maxima may pass mz and my by this
constexpr float kPrNoValue = -1e4f;      // log2 of a value scale of 0: adds nothing to any O in fp32
constexpr float kPrFar = -64.f;          // log2 vscale - (my - mz) from which a group's w is 0 in f16
constexpr int kPrTmem = 512;

template <int D>
struct PrSmem {
  static constexpr uint32_t kTile = 128 * D * 2;  // one f16 tile of 128 rows
  static constexpr uint32_t q(int s) { return s * kTile; }
  static constexpr uint32_t k(int st) { return (2 + st) * kTile; }
  static constexpr uint32_t v(int st) { return (4 + st) * kTile; }
  static constexpr uint32_t kBytes = 6 * kTile + 1024;
};

// idesc of kind::f16 with f16 operands and fp32 accumulators (tc.cuh's, with
// formats 0)
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int b_mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void pr_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Bounded wait that also gives up once another role has set the abort word.
__device__ __noinline__ bool pr_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  const uint64_t t0 = global_ns();
  for (;;) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (global_ns() - t0 > kWaitLimitNs) break;
  }
  atomicCAS(const_cast<int*>(abort_flag), 0, code);
  return false;
}
__device__ __forceinline__ bool pr_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  const uint32_t a = smem_u32(bar);
  for (int n = 0; n < 4096; ++n) {  // no suspension hint: a step's roles wait for microseconds at most
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return pr_wait_slow(a, parity, abort_flag, code);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&w)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]),
      "r"(w[10]), "r"(w[11]), "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
      : "memory");
}

// A CTA's rows and the steps over their keys (the same in every thread).
struct PrTile {
  int64_t req, row0;        // request, its first row of the call
  int tok0, n, tt;          // first token of tile 0, tokens of the request, tokens per tile
  int p0;                   // position of token 0
  int win, sinks, end, sink_end, main0, n_sink, n_steps;

  __device__ __forceinline__ int tokens(int s) const { return max(min(n - tok0 - s * tt, tt), 0); }
  __device__ __forceinline__ int first(int s) const { return p0 + tok0 + s * tt; }
  __device__ __forceinline__ int last(int s) const { return first(s) + tokens(s) - 1; }
  __device__ __forceinline__ int key(int i) const {
    return i < n_sink ? i * kPrKeys : main0 + (i - n_sink) * kPrKeys;
  }
  __device__ __forceinline__ int key_end(int i) const { return i < n_sink ? sink_end : end; }
  // some row of tile s sees a key of step i
  __device__ __forceinline__ bool needs(int s, int i) const {
    const int k0 = key(i);
    return tokens(s) > 0 && k0 <= last(s) && (i < n_sink || k0 + kPrKeys - 1 > first(s) - win || k0 < sinks);
  }
  // every row of tile s sees every key of step i
  __device__ __forceinline__ bool whole(int s, int i) const {
    const int k0 = key(i), k1 = k0 + kPrKeys - 1;
    return k1 <= first(s) && k1 < key_end(i) && (k0 > last(s) - win || k1 < sinks);
  }

  __device__ __forceinline__ bool set(const Attend8Args& a, int64_t tile, int G) {
    tt = 128 / G;
    int64_t lo = 0, hi = a.rows.R, nth;
    if (a.rows.cu) {  // request r's tiles begin at cu[r] / (2 tt) + r
      while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.rows.cu[mid] / (2 * tt) + mid <= tile) lo = mid;
        else hi = mid;
      }
      req = lo;
      row0 = a.rows.cu[req];
      n = a.rows.cu[req + 1] - static_cast<int>(row0);
      p0 = a.rows.prefix[req];
      nth = tile - (row0 / (2 * tt) + req);
      if (nth < 0) return false;  // ahead of the first request's rows
    } else {
      const int64_t per = (a.rows.rps + 2 * tt - 1) / (2 * tt);
      req = tile / per;
      nth = tile % per;
      n = static_cast<int>(a.rows.rps);
      row0 = req * n;
      p0 = a.rows.seq_lens[req] - n;
    }
    if (row0 < 0 || row0 + n > a.N) return false;
    tok0 = static_cast<int>(nth) * 2 * tt;
    if (tok0 >= n) return false;
    constexpr int big = 0x7ffffe00;
    win = a.window < 0 ? big : static_cast<int>(min(a.window, static_cast<int64_t>(big)));
    sinks = static_cast<int>(min(a.sinks, static_cast<int64_t>(big)));
    const int pl = p0 + min(tok0 + 2 * tt, n) - 1;  // the pair's last row (its second tile may be empty)
    end = static_cast<int>(max(min(static_cast<int64_t>(pl) + 1, min(a.W * a.BS, static_cast<int64_t>(big))),
                               static_cast<int64_t>(0)));
    const int ls = max(first(0) - win + 1, 0);
    sink_end = min(min(sinks, ls), end);
    main0 = ls & ~15;
    n_sink = (sink_end + kPrKeys - 1) / kPrKeys;
    if (sink_end >= main0) {  // one run of keys
      main0 = 0;
      n_sink = 0;
    }
    n_steps = n_sink + (end > main0 ? (end - main0 + kPrKeys - 1) / kPrKeys : 0);
    return true;
  }
};

// bits [lo, hi) of 32 (both clamped)
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = min(max(lo, 0), 32);
  hi = min(max(hi, 0), 32);
  const uint32_t below_hi = hi == 32 ? 0xffffffffu : (1u << hi) - 1u;
  const uint32_t below_lo = lo == 32 ? 0xffffffffu : (1u << lo) - 1u;
  return below_hi & ~below_lo;
}

template <int D, int KVT>
__global__ void __launch_bounds__(kPrThreads, 1) cache8_prompt_kernel(const Attend8Args a, int* status) {
  using SM = PrSmem<D>;
  constexpr uint32_t kHalf = 16384;  // 128 rows of 64 f16
  constexpr int kO = 128;            // TMEM column of O in a tile's 256
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t q_full[2], s_full[2], p_full[2], o_full[2], k_full[2], v_full[2], k_empty[2], v_empty[2];
  __shared__ uint64_t drain_bar;
  // per step, in rings that no reader can be a whole turn behind (the tiles of a
  // pair are at most 3 steps apart): kscale and log2 vscale of its 16-key groups,
  // groups that exist (bits 0-7); keys with a NaN value code, zeroed 4 steps ahead
  __shared__ __align__(16) float g_ks[8][8], g_lv[8][8];
  __shared__ uint32_t g_on[8], g_nan[16][4], g_poison[2];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = static_cast<int>(a.H / a.Hkv);
  const int64_t hk = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait();
  PrTile T;
  // the last tiles of a prompt have the most keys: they go first
  if (!T.set(a, gridDim.x - 1 - blockIdx.x, G)) return;

  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  if (warp == kPrMma) {
    tmem_alloc(&tmem_base, kPrTmem);
    tmem_relinquish();
  }
  if (tid < 64) g_nan[tid >> 2][tid & 3] = 0;
  if (tid < 2) g_poison[tid] = 0;
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 128);
      mbar_init(&s_full[s], 2);  // the MMAs, and the issuing thread's own release of what it saw
      mbar_init(&p_full[s], 128);
      mbar_init(&o_full[s], 2);  // likewise: the last step's NaN words are read behind it
      mbar_init(&k_full[s], 128);
      mbar_init(&v_full[s], 128);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(&drain_bar, 1);
    fence_mbar_init();
    abort_flag = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_p = &abort_flag;

  if (warp < kPrConv) {
    // ----------------------------------------------------------------- softmax
    const int s = warp >> 2, r = tid & 127;
    const int ntok = T.tokens(s), tok = r / G;
    const bool active = tok < ntok && r < T.tt * G;
    const int64_t row = T.row0 + T.tok0 + s * T.tt + (active ? tok : 0);
    const int64_t h = hk * G + (active ? r % G : 0);
    const int p = T.first(s) + min(tok, ntok - 1);
    float rowf;  // row factor of z: the power of two taken out of q, |sm_scale|, log2 e
    if (ntok > 0) {
      uint4 raw[D / 8];
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + row * a.s_qn + h * a.s_qh;
      float mx = 0.f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        raw[c] = active ? __ldg(reinterpret_cast<const uint4*>(qp) + c) : make_uint4(0, 0, 0, 0);
      auto unpack = [&](uint32_t w, float& x, float& y) {
        if (a.q_dtype == SRSWA_BF16) {
          x = bf16_lo(w);
          y = bf16_hi(w);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
          x = f.x;
          y = f.y;
        }
      };
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x, y;
          unpack(w[e], x, y);
          mx = fmaxf(mx, fmaxf(fabsf(x), fabsf(y)));
        }
      }
      int e2 = static_cast<int>(__float_as_uint(mx) >> 23) - 127 - 14;
      e2 = mx == 0.f ? 0 : max(min(e2, 126), -126);
      float down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23);
      rowf = __uint_as_float(static_cast<uint32_t>(127 + e2) << 23) * fabsf(a.scale_log2);
      if (a.scale_log2 < 0.f) down = -down;  // z = S * (a factor >= 0)
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x, y;
          unpack(w[e], x, y);
          o[e] = pack_half2(x * down, y * down);
        }
        const uint32_t dst = sbase + SM::q(s) + (c >> 3) * kHalf + sw128_off(r, c & 7);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                     : "memory");
      }
    }
    fence_async_smem();
    pr_arrive(&q_full[s]);

    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tm_s = tmem + s * 256 + lane_off, tm_o = tm_s + kO;
    float m = -INFINITY, dy = 0.f, l = 0.f;  // mz, my - mz
    bool poison = false, ok = true;
    int cnt = 0;
    uint32_t seen[4];   // keys that this row saw of a step seen in part, until its
    int seen_at = -1;   // NaN words are known (the value tile is ready by the next S)
    auto check_nan = [&]() {
      if (seen_at < 0) return;
#pragma unroll
      for (int c = 0; c < 4; ++c) poison = poison || (seen[c] & g_nan[seen_at][c]);
      seen_at = -1;
    };
    for (int i = 0; i < T.n_steps; ++i) {
      if (!T.needs(s, i)) continue;
      const int ri = i & 7, k0 = T.key(i);
      ok = __all_sync(0xffffffffu, pr_wait(&s_full[s], cnt & 1, abort_p, 612));
      if (!ok) break;
      tc_fence_after();
      check_nan();
      const uint32_t on = g_on[ri];
      const bool whole = T.whole(s, i) && on == 0xffu;
      // keys kb .. kb + 31 that this row sees
      auto sees = [&](int c) {
        const int kb = k0 + 32 * c, up = min(p + 1, T.key_end(i)) - kb;
        return (bit_range(max(p - T.win + 1, 0) - kb, up) | bit_range(0, min(T.sinks - kb, up))) &
               ((on >> (2 * c) & 1 ? 0xffffu : 0u) | (on >> (2 * c + 1) & 1 ? 0xffff0000u : 0u));
      };
      float tz = -INFINITY, ty = -INFINITY;  // the row's largest z and y of this step
      auto group_max = [&](const float* v, int grp) {  // 16 raw scores
        float x = max3(v[0], v[1], v[2]), y = max3(v[3], v[4], v[5]);
        x = max3(x, v[6], v[7]);
        y = max3(y, v[8], v[9]);
        x = max3(x, v[10], v[11]);
        y = max3(y, v[12], v[13]);
        x = max3(x, v[14], v[15]);
        x = fmaxf(x, y);
        return x == -INFINITY ? x : x * (g_ks[ri][grp] * rowf);
      };
      // WHOLE is compile-time: a run-time test would be turned into selects on every
      // score
      auto largest = [&](auto whole_) {
        constexpr bool WHOLE = decltype(whole_)::value;
#pragma unroll 1
        for (int c = 0; c < 4; c += 2) {
          float v[32], w[32];
          tmem_ld32(tm_s + 32 * c, v);
          tmem_ld32(tm_s + 32 * c + 32, w);
          tmem_wait_ld();
          if (!WHOLE) {
            const uint32_t va = sees(c), vb = sees(c + 1);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              v[e] = va >> e & 1 ? v[e] : -INFINITY;
              w[e] = vb >> e & 1 ? w[e] : -INFINITY;
            }
          }
          const float x0 = group_max(v, 2 * c), x1 = group_max(v + 16, 2 * c + 1);
          const float x2 = group_max(w, 2 * c + 2), x3 = group_max(w + 16, 2 * c + 3);
          tz = fmaxf(fmaxf(tz, x3), max3(x0, x1, x2));
          const float* lv = &g_lv[ri][2 * c];
          ty = fmaxf(fmaxf(ty, x3 + lv[3]), max3(x0 + lv[0], x1 + lv[1], x2 + lv[2]));
        }
      };
      if (whole) largest(std::true_type());
      else largest(std::false_type());
      const bool move = tz > m + kPrRescale || ty > m + dy + kPrRescale;
      if (__any_sync(0xffffffffu, move)) {
        const float nz = move ? fmaxf(m, tz) : m, ny = move ? fmaxf(m + dy, ty) - nz : dy;
        const float alpha = m == -INFINITY ? 0.f : ex2(m - nz), alpha_o = m == -INFINITY ? 0.f : ex2((m - nz) + (dy - ny));
        if (cnt > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float v[32];
            tmem_ld32(tm_o + 32 * c, v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= alpha_o;
            tmem_st32(tm_o + 32 * c, v);
          }
          tmem_wait_st();
        }
        l *= alpha;
        m = nz;
        dy = ny;
      }
      const float base = kPrShift - (m == -INFINITY ? 0.f : m);
      // weights of 32 keys -> f16 pairs over their scores' first 16 columns
      auto weights = [&](auto whole_, float (&v)[32], int c) {
        constexpr bool WHOLE = decltype(whole_)::value;
        const uint32_t vis = WHOLE ? 0xffffffffu : sees(c);
        uint32_t w[16];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int grp = 2 * c + g;
          // y - my = z - mz + lv; under kPrFar w is 0 and only the sum counts
          const float lv = fmaxf(g_lv[ri][grp] - dy, kPrFar);
          const float f = g_ks[ri][grp] * rowf, add = lv + base;
          const float2 f2 = make_float2(f, f), add2 = make_float2(add, add);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int k = 16 * g + 2 * e;
            float2 x = __ffma2_rn(make_float2(v[k], v[k + 1]), f2, add2);
            if (!WHOLE) {
              x.x = vis >> k & 1 ? x.x : -INFINITY;
              x.y = vis >> (k + 1) & 1 ? x.y : -INFINITY;
            }
            x = make_float2(ex2(x.x), ex2(x.y));
            sum[e & 1] = __fadd2_rn(sum[e & 1], x);
            w[8 * g + e] = pack_half2(x.x, x.y);
          }
          sum[0] = __fadd2_rn(sum[0], sum[1]);
          if (WHOLE || (vis >> (16 * g) & 0xffffu)) l = fmaf(sum[0].x + sum[0].y, ex2(-lv), l);
        }
        tmem_st16u(tm_s + 16 * c, w);
      };
      auto all_weights = [&](auto whole_) {
        float v[32], w[32];
        tmem_ld32(tm_s, v);
        tmem_wait_ld();
#pragma unroll 1
        for (int c = 0; c < 4; c += 2) {
          tmem_ld32(tm_s + 32 * c + 32, w);
          weights(whole_, v, c);
          tmem_wait_ld();
          if (c == 0) tmem_ld32(tm_s + 64, v);
          weights(whole_, w, c + 1);
          if (c == 0) tmem_wait_ld();
        }
      };
      if (whole) all_weights(std::true_type());
      else all_weights(std::false_type());
      tmem_wait_st();
      tc_fence_before();
      pr_arrive(&p_full[s]);
      if (KVT != SRSWA_I8 && !whole) {
#pragma unroll
        for (int c = 0; c < 4; ++c) seen[c] = sees(c);
        seen_at = i & 15;
      }
      ++cnt;
    }
    if (ok && ntok > 0) {
      if (cnt > 0) ok = __all_sync(0xffffffffu, pr_wait(&o_full[s], 0, abort_p, 614));
      if (ok) {
        tc_fence_after();
        check_nan();
        const bool any = l > 0.f || l != l;
        poison = poison || g_poison[s];
        // (2^(my - mz) in two halves: it may pass fp32's range where out does not)
        const float half = any ? exp2f(0.5f * dy) : 0.f, inv = poison ? NAN : any ? half / l : 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float v[32];
          if (cnt > 0) {
            tmem_ld32(tm_o + 32 * c, v);
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = cnt > 0 && (any || poison) ? v[e] * half * inv : 0.f;
          if (active) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) store8(a.out, row * a.s_on + h * a.s_oh + 32 * c + e, a.out_dtype, v + e);
          }
        }
        if (active && a.lse) a.lse[row * a.H + h] = any ? (m + log2f(l) - kPrShift) * kLn2 : -INFINITY;
      }
    }
  } else if (warp < kPrMma) {
    // -------------------------------------------------------------- converters
    constexpr int UPK = D / 16;            // 16-byte units of a key's codes
    constexpr int RPP = 128 / UPK;         // keys per pass of the 128 threads
    constexpr int NP = kPrKeys / RPP;      // passes per tile
    // unit and key of this thread in a pass.  8 lanes store 16 bytes each at once:
    // two neighbouring keys, so that the swizzle spreads them over all banks
    const int c = tid - kPrConv * 32;
    const int u = D == 128 ? (c & 3) + (c >> 1 & 4) : c % UPK;
    const int kr = D == 128 ? (c >> 2 & 1) + (c >> 3 & ~1) : c / UPK;
    const int bs = static_cast<int>(a.BS);
    struct Group {
      int page;  // of 16-key group `lane` of a step (lanes 0-7); -1: nothing to see there
      int off;   // its first key's place in the page
    };
    auto load_group = [&](int i) {
      Group g = {-1, 0};
      if (i < T.n_steps && lane < 8) {
        const int key = T.key(i) + 16 * lane;
        if (key < T.key_end(i)) {
          const int blk = key / bs, page = a.table[T.req * a.s_bt + blk];
          if (page >= 0 && page < a.P) {
            g.page = page;
            g.off = key - blk * bs;
          }
        }
      }
      return g;
    };
    // this thread's byte offsets of step i in either cache (-1: zeros)
    auto offsets = [&](const Group& g, int i, int64_t (&off)[NP]) {
      const int left = T.key_end(i) - T.key(i);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int kk = j * RPP + kr;  // key of the step
        const int page = __shfl_sync(0xffffffffu, g.page, kk >> 4), at = __shfl_sync(0xffffffffu, g.off, kk >> 4);
        off[j] = page >= 0 && kk < left ? page * a.s_page + hk * a.s_head + (at + (kk & 15)) * a.s_pos + u * 16 : -1;
      }
    };
    auto load_codes = [&](const uint8_t* cache, const int64_t (&off)[NP], uint4 (&x)[NP]) {
#pragma unroll
      for (int j = 0; j < NP; ++j)
        x[j] = off[j] >= 0 ? __ldg(reinterpret_cast<const uint4*>(cache + off[j])) : make_uint4(0, 0, 0, 0);
    };
    auto store_tile = [&](uint32_t base, const uint4 (&x)[NP]) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int kk = j * RPP + kr;
        uint32_t o[8];
        widen4<KVT>(x[j].x, o[0], o[1]);
        widen4<KVT>(x[j].y, o[2], o[3]);
        widen4<KVT>(x[j].z, o[4], o[5]);
        widen4<KVT>(x[j].w, o[6], o[7]);
        const uint32_t half = base + (u >> 2) * kHalf;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(half + sw128_off(kk, (u & 3) * 2 + e)),
                       "r"(o[4 * e]), "r"(o[4 * e + 1]), "r"(o[4 * e + 2]), "r"(o[4 * e + 3])
                       : "memory");
      }
    };
    Group g0 = load_group(0), g1 = load_group(1);
    uint4 kx[NP], vx[NP];
    int64_t off[NP];
    if (T.n_steps > 0) {
      offsets(g0, 0, off);
      load_codes(a.k, off, kx);
      load_codes(a.v, off, vx);
    }
    for (int i = 0; i < T.n_steps; ++i) {
      const int st = i & 1, ri = i & 7;
      const uint32_t par = static_cast<uint32_t>(((i >> 1) - 1) & 1);
      const Group g2 = load_group(i + 2);
      if (warp == kPrConv) {
        float ks = 0.f, lv = 0.f;
        if (g0.page >= 0) {
          ks = a.ks[g0.page * a.s_scale + hk];
          lv = log2f(a.vs[g0.page * a.s_scale + hk]);
          if (lv < kPrNoValue) lv = kPrNoValue;
        }
        const uint32_t on = __ballot_sync(0xffffffffu, g0.page >= 0) & 0xffu;
        if (lane < 8) {
          g_ks[ri][lane] = ks;
          g_lv[ri][lane] = lv;
        }
        if (lane < 4) g_nan[(i + 4) & 15][lane] = 0;
        if (lane == 0) g_on[ri] = on;
      }
      if (!__all_sync(0xffffffffu, i < 2 || pr_wait(&k_empty[st], par, abort_p, 621))) break;
      store_tile(sbase + SM::k(st), kx);
      fence_async_smem();
      pr_arrive(&k_full[st]);
      if (i + 1 < T.n_steps) {
        offsets(g1, i + 1, off);
        load_codes(a.k, off, kx);
      }
      if (KVT != SRSWA_I8) {
        const bool all0 = T.needs(0, i) && T.whole(0, i), all1 = T.needs(1, i) && T.whole(1, i);
        if ((T.needs(0, i) && !all0) || (T.needs(1, i) && !all1)) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            uint32_t* w = &vx[j].x;
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t nan = (((w[e] & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;  // bytes 0x7f / 0xff
              any = any || nan;
              w[e] &= ~(nan * 0xffu);
            }
            const int kk = j * RPP + kr;
            if (any) {
              atomicOr(&g_nan[i & 15][kk >> 5], 1u << (kk & 31));
              if (all0) g_poison[0] = 1;  // every row of that tile sees it
              if (all1) g_poison[1] = 1;
            }
          }
        }
      }
      if (!__all_sync(0xffffffffu, i < 2 || pr_wait(&v_empty[st], par, abort_p, 622))) break;
      store_tile(sbase + SM::v(st), vx);
      fence_async_smem();
      pr_arrive(&v_full[st]);
      if (i + 1 < T.n_steps) load_codes(a.v, off, vx);
      g0 = g1;
      g1 = g2;
    }
  } else if (lane == 0) {
    // --------------------------------------------------------------------- MMA
    int last[2] = {-1, -1};
    for (int s = 0; s < 2; ++s)
      for (int i = T.n_steps - 1; i >= 0 && last[s] < 0; --i)
        if (T.needs(s, i)) last[s] = i;
    bool ok = true;
    int cnt[2] = {0, 0};
    // descriptors of tile 0 / stage 0; a step in shared memory is a step >> 4 here
    // (the start address field is 14 bits: everything lies under 256 KB)
    const uint64_t q_desc = sw128_desc(sbase + SM::q(0), 16, 1024), k_desc = sw128_desc(sbase + SM::k(0), 16, 1024);
    const uint64_t v_desc = sw128_desc(sbase + SM::v(0), kHalf, 1024);
    auto issue_s = [&](int s, int i) {
      if (!T.needs(s, i)) return;
      constexpr uint32_t id = idesc_f16(128, kPrKeys, 0);
      const uint64_t qd = q_desc + (s ? SM::kTile >> 4 : 0), kd = k_desc + (i & 1 ? SM::kTile >> 4 : 0);
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const uint32_t off = ((x >> 2) * kHalf + (x & 3) * 32u) >> 4;
        mma_bf16_ss(tmem + s * 256, qd + off, kd + off, id, x > 0 ? 1u : 0u);
      }
      mma_commit(&s_full[s]);
      pr_arrive(&s_full[s]);
    };
    auto issue_o = [&](int s, int i) -> bool {
      if (!T.needs(s, i)) return true;
      if (!pr_wait(&p_full[s], cnt[s] & 1, abort_p, 632)) return false;
      tc_fence_after();
      constexpr uint32_t id = idesc_f16(128, D, 1);
      const uint64_t vd = v_desc + (i & 1 ? SM::kTile >> 4 : 0);
#pragma unroll
      for (int x = 0; x < kPrKeys / 16; ++x)
        mma_bf16_ts(tmem + s * 256 + kO, tmem + s * 256 + x * 8, vd + x * 128u, id, cnt[s] > 0 || x > 0 ? 1u : 0u);
      ++cnt[s];
      if (i == last[s]) {
        mma_commit(&o_full[s]);
        pr_arrive(&o_full[s]);
      }
      return true;
    };
    if (T.n_steps > 0) {
      ok = pr_wait(&q_full[0], 0, abort_p, 633) && pr_wait(&q_full[1], 0, abort_p, 634) &&
           pr_wait(&k_full[0], 0, abort_p, 635);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        issue_s(1, 0);
        mma_commit(&k_empty[0]);
      }
    }
    for (int i = 0; ok && i < T.n_steps; ++i) {
      const int st = i & 1, nx = i + 1;
      ok = pr_wait(&v_full[st], (i >> 1) & 1, abort_p, 636);
      for (int s = 0; ok && s < 2; ++s) {
        ok = issue_o(s, i);
        if (!ok) break;
        if (s == 1) mma_commit(&v_empty[st]);
        if (nx < T.n_steps) {
          if (s == 0) {
            ok = pr_wait(&k_full[nx & 1], (nx >> 1) & 1, abort_p, 637);
            if (!ok) break;
            tc_fence_after();
          }
          issue_s(s, nx);
          if (s == 1) mma_commit(&k_empty[nx & 1]);
        }
      }
    }
    mma_commit(&drain_bar);  // nothing of this CTA is in flight when it exits
    mbar_wait(&drain_bar, 0, 640, abort_p);
  }
  // ------------------------------------------------------------------- exit
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (tid == 0) report_status(status, abort_p);
  if (warp == kPrMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kPrTmem);
  }
}

// Ahead of the tiles: clears the status word, and writes the rows of no request
// (as in a batch padded to a fixed size): 0 and -inf.  In the tiles' kernel that
// loop costs 8 % (long dense prompts 1057 -> 1140 us) for its registers.
constexpr int kPrBeginCtas = 32;
__global__ void __launch_bounds__(256) cache8_prompt_begin_kernel(const Attend8Args a, int* status) {
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *status = 0;
  if (!a.rows.cu) return;
  const int64_t first = min(max(static_cast<int64_t>(a.rows.cu[0]), static_cast<int64_t>(0)), a.N);
  const int64_t past = min(max(static_cast<int64_t>(a.rows.cu[a.rows.R]), first), a.N);
  const int64_t units = a.D / 8, per_row = a.H * units, n = (first + a.N - past) * per_row;
  const float zero[8] = {};
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += kPrBeginCtas * 256) {
    const int64_t nth = i / per_row, row = nth < first ? nth : past + nth - first;
    const int64_t h = i / units % a.H, u = i % units;
    store8(a.out, row * a.s_on + h * a.s_oh + u * 8, a.out_dtype, zero);
    if (u == 0 && a.lse) a.lse[row * a.H + h] = -INFINITY;
  }
}

// CTAs of a KV head: pairs of tiles of 128 / G tokens each (of ragged prompts,
// the most there can be).
static int64_t tile_pairs(int64_t N, int64_t R, int64_t rows_per_req, int64_t G, bool varlen) {
  const int64_t pair = 2 * (128 / G);
  return varlen ? N / pair + R : R * ((rows_per_req + pair - 1) / pair);
}

// Rows without a selection, where the tiles take less time than the row kernel
// would, by what both cost (microseconds): the tiles 11 and 2.7 a step of 128
// keys, for each wave of CTAs; the rows 10 and 1.6 per unit of 32 keys that a
// resident warp has.  (16 / 4 heads of 128, rows and tiles: 16 rows after 4096 keys
// 33 and 98, 32 requests of them 196 and 105; 300 such ragged rows in 4 requests
// 166 and 112.  Over 585 sizes, all with tables as wide as the longest request, the
// choice takes 2 % more than the better one; the width stands for the lengths,
// which the host does not know.)
bool prompt_applies(const srswa_cache8_desc& d, bool varlen) {
  const int64_t G = d.H / d.Hkv;
  if (d.K > 0 || G > 128 || d.nsplit > 0) return false;
  const double sms = sm_count();
  const double waves = std::ceil(static_cast<double>(tile_pairs(d.N, d.R, d.rows_per_req, G, varlen)) * d.Hkv / sms);
  double keys = static_cast<double>(d.W) * d.block_size;
  if (d.window >= 0) keys = std::min(keys, static_cast<double>(d.window) + d.sinks + 2 * (128 / G));
  const RowsPlan rows = rows_plan(d, varlen);
  const double units = static_cast<double>(rows.units) * rows.ch / 2;
  return waves * (11 + 2.7 * std::ceil(keys / kPrKeys)) < 10 + 1.6 * units / (kRowsCtasPerSm * kRowsWarps * sms);
}

int prompt_launch(const Attend8Args& a, int kv_dtype, int* status, cudaStream_t st) {
  const int64_t tiles = tile_pairs(a.N, a.rows.R, a.rows.rps, a.H / a.Hkv, a.rows.cu != nullptr);
  if (tiles >= (1ll << 31)) return SRSWA_ETOOLARGE;
  const int rc = launch_pdl(cache8_prompt_begin_kernel, dim3(a.rows.cu ? kPrBeginCtas : 1), 256, 0, st, a, status);
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(a.Hkv));
  auto go = [&](auto kern, uint32_t smem, bool (&allowed)[64]) -> int {
    int dev = 0;
    SRSWA_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !allowed[dev]) {
      SRSWA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
      if (dev < 64) allowed[dev] = true;
    }
    return launch_pdl(kern, grid, kPrThreads, smem, st, a, status);
  };
  static bool allowed[4][64] = {};  // per kernel and device: the shared memory has been asked for
  if (a.D == 128) {
    if (kv_dtype == SRSWA_I8) return go(cache8_prompt_kernel<128, SRSWA_I8>, PrSmem<128>::kBytes, allowed[0]);
    return go(cache8_prompt_kernel<128, SRSWA_F8E4M3>, PrSmem<128>::kBytes, allowed[1]);
  }
  if (kv_dtype == SRSWA_I8) return go(cache8_prompt_kernel<64, SRSWA_I8>, PrSmem<64>::kBytes, allowed[2]);
  return go(cache8_prompt_kernel<64, SRSWA_F8E4M3>, PrSmem<64>::kBytes, allowed[3]);
}

}  // namespace srswa
