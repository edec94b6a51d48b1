// Attend of single rows over the scaled 8-bit cache (decode, draft tokens, and
// prompt rows that carry a block selection).
//
// Mathematics.  For a row at position p and its visible keys j (window, sinks,
// selected blocks with bias b):
//   z_j = (q . c_j) * kscale[page] * sm_scale + b_j      (c_j: the key's codes)
//   o = sum_j softmax(z)_j * vscale[page] * d_j           (d_j: the value's codes)
// online, in the log2 domain, fp32 throughout except the two MMA operands:
//   * codes widen to f16 exactly; q is scaled by a power of two so that it is
//     exact in f16 too (bf16 elements under 2^-28 of the row's largest lose
//     bits that fp32 sums would not show);
//   * softmax weights are rounded to f16 (they are <= 1: 2^-11 relative).
// Both scales are applied in fp32, outside the MMAs.
//
// What bounds it: bytes.  A key costs 2 D bytes and 4 D flops per query head,
// so even 8 heads on a key stay far under the tensor rate: mma.sync with the
// keys on the 16-row side (its columns hold up to 8 (row, head) queries that
// share the keys) is enough, and its register operands come straight from
// 16-byte shared-memory reads: the order of features inside a dot product and
// of keys inside a chunk is free, so both are chosen such that a thread's
// operands are contiguous bytes.
//
// Work split: the units (16 or 32 keys of one page and head) of all (row group,
// kv head) items are laid end to end and cut into equal parts, one per resident
// CTA, so uneven lengths leave no tail; an item cut in several parts leaves
// fp32 partials that cache8_merge_kernel joins in order.  Each warp streams its
// units through a private cp.async ring; its page ids and scales are
// prefetched a block of 32 slots ahead.

#include <cmath>
#include <type_traits>

#include "cache8_attend.cuh"
#include "tc.cuh"

namespace srswa {

constexpr int kRowsThreads = 128;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsRing = 16384;  // shared memory of a warp's ring at D = 128 (half of it at 64)
constexpr int kRowsCtasPerSm = 3;
constexpr int kCols = 8;  // queries that share a pass over the keys (columns of the MMA)

// The keys a row group can see, as slots of one page each: sinks, window,
// selected blocks, in this order.
struct Span {
  int p0, ls0, sink_end, end, n_sink, b0, n_win, units;
};

template <int CH>
__device__ __forceinline__ Span group_span(const Attend8Args& a, int64_t rg, int64_t& req) {
  int64_t p0;
  row_place(a.rows, rg * a.share, req, p0);
  Span s;
  const int64_t last = p0 + a.share - 1;
  int64_t ls = a.window < 0 ? 0 : p0 - a.window + 1;
  if (ls < 0) ls = 0;
  const int64_t end = max(min(last + 1, min(a.W * a.BS, static_cast<int64_t>(0x7fffff00))), static_cast<int64_t>(0));
  s.p0 = static_cast<int>(p0);
  s.ls0 = static_cast<int>(ls);
  s.end = static_cast<int>(end);
  s.sink_end = static_cast<int>(min(min(a.sinks, ls), end));
  const int bs = static_cast<int>(a.BS);
  s.n_sink = (s.sink_end + bs - 1) / bs;
  s.b0 = s.ls0 / bs;
  s.n_win = s.end > s.ls0 ? (s.end + bs - 1) / bs - s.b0 : 0;
  s.units = max((s.n_sink + s.n_win + static_cast<int>(a.K)) * (bs / (16 * CH)), 1);
  return s;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// Four codes -> f16 pairs (e0, e1) and (e2, e3), exactly.
template <int KVT>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (KVT == SRSWA_I8) {  // 1024 + (c + 128) as an f16 bit pattern, minus 1152
    const uint32_t x = w ^ 0x80808080u;
    const __half2 off = __floats2half2_rn(1152.f, 1152.f);
    const uint32_t a = prmt(x, 0x64646464u, 0x4140u), b = prmt(x, 0x64646464u, 0x4342u);
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// 16-byte unit c of key row r of a chunk in shared memory.  The order of units
// is such that the MMA operand reads below hit every bank once: K reads rows
// {r, r + 4} together, V reads rows 0..3 (mod 4) together.
template <int D>
__device__ __forceinline__ uint32_t k_off(int r, int c) {
  return D == 128 ? (r * 8 + (c ^ (((r >> 2) & 1) << 2))) * 16 : ((r * 4 + c) ^ (((r >> 2) & 1) << 2)) * 16;
}
template <int D>
__device__ __forceinline__ uint32_t v_off(int r, int c) {
  return D == 128 ? (r * 8 + (c ^ ((r & 3) << 1))) * 16 : ((r * 4 + c) ^ (((r >> 1) & 1) << 1)) * 16;
}

// CH: 16-key chunks of a unit, what a warp takes at a time (a divisor of a
// page's chunks; two amortise the softmax bookkeeping and keep two independent
// MMA chains going).
template <int D, int KVT, int CH>
__global__ void __launch_bounds__(kRowsThreads, kRowsCtasPerSm) cache8_rows_kernel(const Attend8Args a) {
  constexpr int CB = 16 * D;           // bytes of a chunk of K (or V)
  constexpr int SB = 2 * CH * CB;      // bytes of a stage: K of its chunks, then V
  constexpr int ST = kRowsRing * D / 128 / SB;  // stages of a warp's ring
  constexpr int UK = 16 * CH;          // keys of a unit
  constexpr int KS = D / 16;           // MMA steps of a dot product, and feature tiles of the output
  constexpr int RPI = 512 / D;         // key rows per warp copy instruction
  extern __shared__ __align__(128) uint8_t smem[];
  int* sel_blk = reinterpret_cast<int*>(smem + kRowsWarps * ST * SB);
  float* sel_b2 = reinterpret_cast<float*>(sel_blk + a.K);
  __shared__ float w_m[kRowsWarps][kCols], w_l[kRowsWarps][kCols];
  __shared__ int64_t f_part[kRowsWarps], f_off;
  __shared__ int f_rg;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = lane & 3, g = lane >> 2;
  const int bs = static_cast<int>(a.BS), upp = bs / UK;  // units per page
  const int G = static_cast<int>(a.H / a.Hkv), K = static_cast<int>(a.K), share = static_cast<int>(a.share);
  const int sinks = static_cast<int>(min(a.sinks, static_cast<int64_t>(0x7fffff00)));
  const int win = a.window < 0 ? 0x7fffff00 : static_cast<int>(min(a.window, static_cast<int64_t>(0x7fffff00)));
  const uint32_t ring = smem_u32(smem) + warp * ST * SB;
  const int krow = (g >> 1) + 4 * (g & 1);  // the key of MMA row g (and + 8 of row g + 8)
  const int cr = lane / (D / 16), cc = lane % (D / 16);  // key row and 16-byte unit of this lane's copies
  pdl_launch_dependents();                  // the merge kernel waits for this grid before it reads

  // One (row group, kv head, column group), units [c0, c1) of its `s.units`;
  // slot < 0: the whole item, results written out; else partial `slot`.
  auto process = [&](int64_t rg, int64_t req, const Span& s, int64_t hk, int grp, int c0, int c1, int64_t slot) {
    const int64_t n0 = rg * a.share;
    __syncthreads();  // the previous item's epilogue and list are done with
    if (K) {
      const int64_t ib = hk * a.s_ti_h + n0 * a.s_ti_n;
      for (int i = tid; i < K; i += kRowsThreads) {
        const int64_t b = load_index(a.sel, ib + i, a.idx_is64);
        sel_blk[i] = b >= 0 && b < a.W ? static_cast<int>(b) : -1;
        sel_b2[i] = a.bias ? a.bias[hk * a.s_b_h + n0 * a.s_b_n + i] * kLog2e : 0.f;
      }
      __syncthreads();
      uint32_t again = 0;  // repeats of an earlier slot (K <= 4 * threads)
      for (int i = tid, u = 0; i < K; i += kRowsThreads, ++u)
        if (sel_blk[i] >= 0)
          for (int j = 0; j < i; ++j) again |= static_cast<uint32_t>(sel_blk[j] == sel_blk[i]) << u;
      __syncthreads();
      for (int i = tid, u = 0; i < K; i += kRowsThreads, ++u)
        if (again >> u & 1) sel_blk[i] = -1;
      __syncthreads();
    }

    // ---- slots: lane l of (cur, nxt) holds slot base + l, base + 32 + l ----
    const int n_fix = s.n_sink + s.n_win, nslots = n_fix + K;
    struct Pages {
      int blk, page;  // page < 0: nothing to see there
      float ks, vs;
    };
    auto load_pages = [&](int i) {
      Pages r = {0, -1, 0.f, 0.f};
      if (i < nslots) {
        r.blk = i < s.n_sink ? i : i < n_fix ? s.b0 + i - s.n_sink : sel_blk[i - n_fix];
        if (r.blk >= 0) {
          const int page = a.table[req * a.s_bt + r.blk];
          if (page >= 0 && page < a.P) {
            r.page = page;
            r.ks = a.ks[page * a.s_scale + hk];
            r.vs = a.vs[page * a.s_scale + hk];
          }
        }
      }
      return r;
    };
    int base = (c0 / upp) & ~31;
    Pages cur = load_pages(base + lane), nxt = load_pages(base + 32 + lane);
    auto limits = [&](int si, int blk, int& lo, int& hi) {
      lo = si < s.n_sink ? 0 : si < n_fix ? s.ls0 : max(blk * bs, sinks);
      hi = si < s.n_sink ? s.sink_end : si < n_fix ? s.end : min(min((blk + 1) * bs, s.ls0), s.end);
    };

    // units c0 + warp, + 4, + 8 ...: the producer runs ST - 1 of them ahead
    const int mine = (c1 - c0 - warp + kRowsWarps - 1) / kRowsWarps;
    int p_si = (c0 + warp) / upp, p_u = (c0 + warp) % upp, p_i = 0, p_stage = 0;
    auto issue = [&]() {
      if (p_i < mine) {
        const int rel = p_si - base;
        const int page = rel < 32 ? __shfl_sync(0xffffffffu, cur.page, rel) : __shfl_sync(0xffffffffu, nxt.page, rel - 32);
        const int blk = rel < 32 ? __shfl_sync(0xffffffffu, cur.blk, rel) : __shfl_sync(0xffffffffu, nxt.blk, rel - 32);
        int lo, hi;
        limits(p_si, blk, lo, hi);
        const int k0 = blk * bs + p_u * UK;
        if (page >= 0 && k0 < hi && k0 + UK > lo) {
          const uint32_t dst = ring + p_stage * SB;
          const int64_t off = page * a.s_page + hk * a.s_head + (p_u * UK + cr) * a.s_pos + cc * 16;
          const uint8_t *kp = a.k + off, *vp = a.v + off;
          if (k0 >= lo && k0 + UK <= hi) {
#pragma unroll
            for (int j = 0; j < UK / RPI; ++j) {
              const int r = (j * RPI) % 16 + cr, c = (j * RPI) / 16;
              cp_async16(dst + c * CB + k_off<D>(r, cc), kp + j * RPI * a.s_pos);
              cp_async16(dst + (CH + c) * CB + v_off<D>(r, cc), vp + j * RPI * a.s_pos);
            }
          } else {
#pragma unroll
            for (int j = 0; j < UK / RPI; ++j) {
              const int r = (j * RPI) % 16 + cr, c = (j * RPI) / 16, key = k0 + j * RPI + cr;
              const bool in = key >= lo && key < hi;
              cp_async16_zfill(dst + c * CB + k_off<D>(r, cc), in ? kp + j * RPI * a.s_pos : a.k, in);
              cp_async16_zfill(dst + (CH + c) * CB + v_off<D>(r, cc), in ? vp + j * RPI * a.s_pos : a.v, in);
            }
          }
        }
        p_u += kRowsWarps;
        while (p_u >= upp) { p_u -= upp; ++p_si; }
        ++p_i;
        p_stage = p_stage + 1 == ST ? 0 : p_stage + 1;
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) issue();

    // ---- this thread's part of query column g, as f16 MMA operands ----
    uint32_t qf[KS][2];
    float qexp;  // the power of two taken out of it
    {
      const int col = grp * kCols + g;
      const bool on = col < share * G;
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (n0 + (on ? col / G : 0)) * a.s_qn +
                           (hk * G + (on ? col % G : 0)) * a.s_qh + t * 16;
      float f[KS * 4];
#pragma unroll
      for (int hseg = 0; hseg < D / 64; ++hseg) {
        load8(qp, hseg * 64, a.q_dtype, f + hseg * 16);
        load8(qp, hseg * 64 + 8, a.q_dtype, f + hseg * 16 + 8);
      }
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < KS * 4; ++e) {
        f[e] = on ? f[e] : 0.f;
        mx = fmaxf(mx, fabsf(f[e]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // largest element into [2^14, 2^15)
      int e = static_cast<int>(__float_as_uint(mx) >> 23) - 127 - 14;
      e = mx == 0.f ? 0 : max(min(e, 126), -126);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      qexp = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        qf[i][0] = pack_half2(f[4 * i] * down, f[4 * i + 1] * down);
        qf[i][1] = pack_half2(f[4 * i + 2] * down, f[4 * i + 3] * down);
      }
    }
    const float z0 = __shfl_sync(0xffffffffu, qexp, (2 * t) * 4) * a.scale_log2;
    const float z1 = __shfl_sync(0xffffffffu, qexp, (2 * t + 1) * 4) * a.scale_log2;
    const int row0 = (grp * kCols + 2 * t) / G, row1 = (grp * kCols + 2 * t + 1) / G;  // rows of this thread's columns

    float o[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    // P.V of the unit in `src`: this thread's keys (t, t + 4, t + 8, t + 12 of
    // each chunk), each word four features of one key
    auto load_v = [&](uint32_t src, uint32_t (&w)[CH][4][D / 32]) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = t + 4 * i;
          if constexpr (D == 128) {
            const uint4 x = lds128(src + c * CB + v_off<D>(r, g));
            w[c][i][0] = x.x; w[c][i][1] = x.y; w[c][i][2] = x.z; w[c][i][3] = x.w;
          } else {
            const uint2 x = lds64(src + c * CB + v_off<D>(r, g >> 1) + (g & 1) * 8);
            w[c][i][0] = x.x; w[c][i][1] = x.y;
          }
        }
    };
    auto pv_tile = [&](const uint32_t (&w)[CH][4][D / 32], int e, const uint32_t (&pb)[CH][2], float (&acc)[2][4]) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        // (key, key + 4) pairs of features 4e .. 4e + 3
        uint32_t a01[4], a23[4];
        widen4<KVT>(prmt(w[c][0][e], w[c][1][e], 0x5140u), a01[0], a01[1]);
        widen4<KVT>(prmt(w[c][0][e], w[c][1][e], 0x7362u), a01[2], a01[3]);
        widen4<KVT>(prmt(w[c][2][e], w[c][3][e], 0x5140u), a23[0], a23[1]);
        widen4<KVT>(prmt(w[c][2][e], w[c][3][e], 0x7362u), a23[2], a23[3]);
        mma16816(acc[0], a01[0], a01[1], a23[0], a23[1], pb[c][0], pb[c][1]);
        mma16816(acc[1], a01[2], a01[3], a23[2], a23[3], pb[c][0], pb[c][1]);
      }
    };

    int c_si = (c0 + warp) / upp, c_u = (c0 + warp) % upp, c_stage = 0;
    for (int i = 0; i < mine; ++i) {
      if (c_si - base >= 32) {
        base += 32;
        cur = nxt;
        nxt = load_pages(base + 32 + lane);
      }
      cp_async_wait<ST - 2>();
      __syncwarp();  // every lane's copies have landed, and every lane is done with the stage issued next
      issue();
      const int rel = c_si - base, si = c_si;
      const int page = __shfl_sync(0xffffffffu, cur.page, rel), blk = __shfl_sync(0xffffffffu, cur.blk, rel);
      const float ks = __shfl_sync(0xffffffffu, cur.ks, rel), vs = __shfl_sync(0xffffffffu, cur.vs, rel);
      int lo, hi;
      limits(si, blk, lo, hi);
      const int k0 = blk * bs + c_u * UK;
      const uint32_t src = ring + c_stage * SB;
      c_u += kRowsWarps;
      while (c_u >= upp) { c_u -= upp; ++c_si; }
      c_stage = c_stage + 1 == ST ? 0 : c_stage + 1;
      if (page < 0 || k0 >= hi || k0 + UK <= lo) continue;

      float x[CH][4];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[c][e] = 0.f;
#pragma unroll
      for (int hseg = 0; hseg < D / 64; ++hseg)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const uint4 xr = lds128(src + c * CB + k_off<D>(krow, hseg * 4 + t));
          const uint4 yr = lds128(src + c * CB + k_off<D>(krow + 8, hseg * 4 + t));
          const uint32_t xa[4] = {xr.x, xr.y, xr.z, xr.w}, ya[4] = {yr.x, yr.y, yr.z, yr.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a0, a1, a2, a3;
            widen4<KVT>(xa[e], a0, a2);
            widen4<KVT>(ya[e], a1, a3);
            mma16816(x[c], a0, a1, a2, a3, qf[hseg * 4 + e][0], qf[hseg * 4 + e][1]);
          }
        }
      const float b2 = si >= n_fix ? sel_b2[si - n_fix] : 0.f, f0 = z0 * ks, f1 = z1 * ks;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        x[c][0] = fmaf(x[c][0], f0, b2);
        x[c][1] = fmaf(x[c][1], f1, b2);
        x[c][2] = fmaf(x[c][2], f0, b2);
        x[c][3] = fmaf(x[c][3], f1, b2);
      }
      // whole: every column sees every key of the unit.  Else a key counts if
      // it lies in [lo, hi) and, in a group of several rows, the column's own
      // row (at p0 + r) sees it.
      bool whole = k0 >= lo && k0 + UK <= hi;
      if (share > 1) whole = whole && k0 + UK - 1 <= s.p0 && (k0 > s.p0 + share - 1 - win || k0 + UK - 1 < sinks);
      auto sees = [&](int j, int r) { return j <= s.p0 + r && (j > s.p0 + r - win || j < sinks); };
      if (!whole) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const int j = k0 + c * 16 + krow + 8 * hh;
            const bool in = j >= lo && j < hi;
            if (!(in && (share == 1 || sees(j, row0)))) x[c][2 * hh] = -INFINITY;
            if (!(in && (share == 1 || sees(j, row1)))) x[c][2 * hh + 1] = -INFINITY;
          }
      }
      float c0m = -INFINITY, c1m = -INFINITY;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        c0m = fmaxf(c0m, fmaxf(x[c][0], x[c][2]));
        c1m = fmaxf(c1m, fmaxf(x[c][1], x[c][3]));
      }
#pragma unroll
      for (int msk = 4; msk < 32; msk <<= 1) {
        c0m = fmaxf(c0m, __shfl_xor_sync(0xffffffffu, c0m, msk));
        c1m = fmaxf(c1m, __shfl_xor_sync(0xffffffffu, c1m, msk));
      }
      const float n0m = fmaxf(m0, c0m), n1m = fmaxf(m1, c1m);
      const float u0 = n0m == -INFINITY ? 0.f : n0m, u1 = n1m == -INFINITY ? 0.f : n1m;
      if (__any_sync(0xffffffffu, n0m != m0 || n1m != m1)) {
        const float al0 = exp2f(m0 - u0), al1 = exp2f(m1 - u1);
        l0 *= al0;
        l1 *= al1;
#pragma unroll
        for (int e = 0; e < KS; ++e) {
          o[e][0] *= al0; o[e][1] *= al1; o[e][2] *= al0; o[e][3] *= al1;
        }
        m0 = n0m;
        m1 = n1m;
      }
      uint32_t pb[CH][2];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float p0 = exp2f(x[c][0] - u0), p1 = exp2f(x[c][1] - u1), p2 = exp2f(x[c][2] - u0), p3 = exp2f(x[c][3] - u1);
        l0 += p0 + p2;
        l1 += p1 + p3;
        pb[c][0] = transpose8x8(pack_half2(p0, p1));
        pb[c][1] = transpose8x8(pack_half2(p2, p3));
      }
      uint32_t w[CH][4][D / 32];
      load_v(src + CH * CB, w);
      if (whole || share == 1) {  // masked keys were filled with zeros
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          float acc[2][4] = {};
          pv_tile(w, e, pb, acc);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int y = 0; y < 4; ++y) o[2 * e + u][y] = fmaf(vs, acc[u][y], o[2 * e + u][y]);
        }
      } else {
        // rows of the group see different keys: each takes the unit with the
        // keys that it does not see zeroed (their codes may be NaN), or not at
        // all (the page's scale may be)
        for (int r = 0; r < share; ++r) {
          uint32_t wr[CH][4][D / 32];
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2)
#pragma unroll
              for (int e = 0; e < D / 32; ++e) wr[c][i2][e] = sees(k0 + c * 16 + t + 4 * i2, r) ? w[c][i2][e] : 0;
          const bool take0 = row0 == r && c0m != -INFINITY, take1 = row1 == r && c1m != -INFINITY;
#pragma unroll
          for (int e = 0; e < D / 32; ++e) {
            float acc[2][4] = {};
            pv_tile(wr, e, pb, acc);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float* oo = o[2 * e + u];
              oo[0] = take0 ? fmaf(vs, acc[u][0], oo[0]) : oo[0];
              oo[1] = take1 ? fmaf(vs, acc[u][1], oo[1]) : oo[1];
              oo[2] = take0 ? fmaf(vs, acc[u][2], oo[2]) : oo[2];
              oo[3] = take1 ? fmaf(vs, acc[u][3], oo[3]) : oo[3];
            }
          }
        }
      }
    }
    cp_async_wait<0>();

    // ---- join the warps ----
#pragma unroll
    for (int msk = 4; msk < 32; msk <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, msk);
      l1 += __shfl_xor_sync(0xffffffffu, l1, msk);
    }
    __syncthreads();  // the rings become the warps' outputs
    float* wo = reinterpret_cast<float*>(smem);
    const int ncol = min(share * G - grp * kCols, kCols);
    if (g == 0) {
      w_m[warp][2 * t] = m0; w_l[warp][2 * t] = l0;
      w_m[warp][2 * t + 1] = m1; w_l[warp][2 * t + 1] = l1;
    }
#pragma unroll
    for (int e = 0; e < KS; ++e) {
      const int d = g * 2 * KS + 2 * e;  // MMA rows g and g + 8 of tile e: see add_pv
      float* x = wo + (warp * kCols + 2 * t) * D + d;
      if (2 * t < ncol) { x[0] = o[e][0]; x[1] = o[e][2]; }
      if (2 * t + 1 < ncol) { x[D] = o[e][1]; x[D + 1] = o[e][3]; }
    }
    __syncthreads();
    for (int i = tid; i < ncol * D; i += kRowsThreads) {
      const int c = i / D, d = i % D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) M = fmaxf(M, w_m[w][c]);
      const float Mu = M == -INFINITY ? 0.f : M;
      float L = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        const float f = exp2f(w_m[w][c] - Mu);
        L += w_l[w][c] * f;
        acc += wo[(w * kCols + c) * D + d] * f;
      }
      if (slot < 0) {
        const int gc = grp * kCols + c;
        const int64_t n = n0 + gc / G, h = hk * G + gc % G;
        store_elem(a.out, n * a.s_on + h * a.s_oh + d, a.out_dtype, L > 0.f || L != L ? acc / L : 0.f);
        if (d == 0 && a.lse) a.lse[n * a.H + h] = L > 0.f || L != L ? (M + log2f(L)) * kLn2 : -INFINITY;
      } else {
        a.part_o[(slot * kCols + c) * D + d] = acc;
        if (d == 0) {
          a.part_ml[(slot * kCols + c) * 2] = M;
          a.part_ml[(slot * kCols + c) * 2 + 1] = L;
        }
      }
    }
  };

  const int64_t per_group = a.Hkv * a.ngrp;  // items of a row group
  int64_t req, pos, stop;
  if (!a.balanced) {  // one CTA per item
    pos = 0;
    stop = 1;
    f_rg = static_cast<int>(blockIdx.x / per_group);
  } else {  // this CTA's equal part of all units
    const int64_t groups = a.N / a.share;
    const int64_t per = (groups + kRowsThreads - 1) / kRowsThreads;
    const int64_t g_lo = min(tid * per, groups), g_hi = min(g_lo + per, groups);
    int64_t sum = 0;
    for (int64_t i = g_lo; i < g_hi; ++i) sum += group_span<CH>(a, i, req).units;
    sum *= per_group;
    int64_t x = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) f_part[warp] = x;
    __syncthreads();
    int64_t before = x - sum, total = 0;
    for (int w = 0; w < kRowsWarps; ++w) {
      if (w < warp) before += f_part[w];
      total += f_part[w];
    }
    pos = total * blockIdx.x / gridDim.x;
    stop = total * (blockIdx.x + 1) / gridDim.x;
    if (pos >= before && pos < before + sum) {
      int64_t off = pos - before, i = g_lo;
      for (;; ++i) {
        const int64_t n = group_span<CH>(a, i, req).units * per_group;
        if (off < n) break;
        off -= n;
      }
      f_rg = static_cast<int>(i);
      f_off = off;
    }
  }
  __syncthreads();
  int head_item_rg = -1, head_item = 0, tail_item_rg = -1, tail_item = 0;
  if (pos < stop) {
    int64_t rg = f_rg;
    Span s = group_span<CH>(a, rg, req);
    int64_t off = a.balanced ? f_off : (blockIdx.x % per_group) * s.units;
    if (!a.balanced) stop = s.units;
    while (pos < stop) {
      const int64_t it = off / s.units;
      const int c0 = static_cast<int>(off % s.units);
      const int c1 = static_cast<int>(min(static_cast<int64_t>(s.units), c0 + stop - pos));
      int64_t slot = -1;
      if (c0 > 0) {
        slot = 2 * static_cast<int64_t>(blockIdx.x);
        head_item_rg = static_cast<int>(rg);
        head_item = static_cast<int>(it);
      } else if (c1 < s.units) {
        slot = 2 * static_cast<int64_t>(blockIdx.x) + 1;
        tail_item_rg = static_cast<int>(rg);
        tail_item = static_cast<int>(it);
      }
      process(rg, req, s, it / a.ngrp, static_cast<int>(it % a.ngrp), c0, c1, slot);
      pos += c1 - c0;
      off += c1 - c0;
      if (off == s.units * per_group && pos < stop) {
        off = 0;
        s = group_span<CH>(a, ++rg, req);
      }
    }
  } else if (tid == 0) {
    head_item_rg = -2;  // an empty part: the item goes on behind it
  }
  if (tid == 0 && a.balanced) {
    int* meta = a.part_meta + 4 * static_cast<int64_t>(blockIdx.x);
    meta[0] = head_item_rg; meta[1] = head_item; meta[2] = tail_item_rg; meta[3] = tail_item;
  }
}

// Joins the parts of the item that CTA blockIdx.x began and did not finish, in
// the order of the parts.
template <int D>
__global__ void __launch_bounds__(256) cache8_merge_kernel(const Attend8Args a, int ncta) {
  pdl_wait();
  const int c = blockIdx.x;
  const int rg = a.part_meta[4 * c + 2], it = a.part_meta[4 * c + 3];
  if (rg < 0) return;
  int last = c;  // last part of the item
  for (int j = c + 1; j < ncta; ++j) {
    const int r = a.part_meta[4 * j], i = a.part_meta[4 * j + 1];
    if (r == -2) continue;
    if (r != rg || i != it) break;
    last = j;
    if (a.part_meta[4 * j + 2] >= 0) break;  // this CTA went on to another item
  }
  const int64_t hk = it / a.ngrp;
  const int grp = static_cast<int>(it % a.ngrp), G = static_cast<int>(a.H / a.Hkv);
  const int ncol = min(static_cast<int>(a.share) * G - grp * kCols, kCols);
  for (int i = threadIdx.x; i < ncol * D; i += blockDim.x) {
    const int col = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int j = c; j <= last; ++j) {
      if (j > c && a.part_meta[4 * j] == -2) continue;
      const int64_t slot = (j == c ? 2 * static_cast<int64_t>(j) + 1 : 2 * static_cast<int64_t>(j)) * kCols + col;
      const float m = a.part_ml[slot * 2], l = a.part_ml[slot * 2 + 1];
      const float mn = fmaxf(M, m), mu = mn == -INFINITY ? 0.f : mn;
      const float fo = exp2f(M - mu), fn = exp2f(m - mu);
      L = L * fo + l * fn;
      acc = acc * fo + a.part_o[slot * D + d] * fn;
      M = mn;
    }
    const int gc = grp * kCols + col;
    const int64_t n = static_cast<int64_t>(rg) * a.share + gc / G, h = hk * G + gc % G;
    store_elem(a.out, n * a.s_on + h * a.s_oh + d, a.out_dtype, L > 0.f || L != L ? acc / L : 0.f);
    if (d == 0 && a.lse) a.lse[n * a.H + h] = L > 0.f || L != L ? (M + log2f(L)) * kLn2 : -INFINITY;
  }
}

static int sm_count() {
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (sms[dev] == 0) {
    int v = 0;
    sms[dev] = cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0 ? v : 148;
  }
  return sms[dev];
}

RowsPlan rows_plan(const srswa_cache8_desc& d, bool varlen) {
  RowsPlan p = {};
  const int64_t G = d.H / d.Hkv;
  // rows of one request share a pass over its keys unless each has its own selection
  p.share = varlen || d.K > 0 ? 1 : d.rows_per_req;
  p.ngrp = (p.share * G + kCols - 1) / kCols;
  const int64_t groups = d.N / p.share;
  p.items = groups * d.Hkv * p.ngrp;
  // the most units an item can have
  p.ch = d.block_size % 32 == 0 ? 2 : 1;
  const int64_t upp = d.block_size / (16 * p.ch);
  int64_t blocks = d.W;
  if (d.window >= 0) {
    const int64_t win = (d.window + p.share - 1 + d.block_size - 1) / d.block_size + 1;
    const int64_t snk = (d.sinks + d.block_size - 1) / d.block_size;
    blocks = win < d.W && snk < d.W && win + snk < d.W ? win + snk : d.W;
  }
  const int64_t most = (blocks + d.K) * upp;
  const int64_t slots = static_cast<int64_t>(sm_count()) * kRowsCtasPerSm;
  if (d.nsplit > 0) {
    p.balanced = d.nsplit > 1;
    p.ctas = d.nsplit * p.items;
  } else if (most <= 4 * kRowsWarps || groups > 2048 || p.items > 16 * slots) {
    // short items (a join would cost more than it saves), or so many that their
    // uneven ends do not show: one CTA each
    p.balanced = false;
    p.ctas = p.items;
  } else {
    p.balanced = true;
    const int64_t enough = (p.items * most + kRowsWarps - 1) / kRowsWarps;
    p.ctas = enough < slots ? enough : slots;
  }
  if (p.balanced) {
    const int64_t f = p.ctas * 2 * kCols;
    p.o_floats = f * d.D;
    p.bytes = static_cast<size_t>(p.o_floats + f * 2 + p.ctas * 4) * 4;
  }
  return p;
}

int rows_launch(Attend8Args a, const RowsPlan& p, int kv_dtype, void* workspace, cudaStream_t st) {
  if (a.K > 4 * kRowsThreads || p.ctas >= (1ll << 30)) return SRSWA_ETOOLARGE;
  a.share = p.share;
  a.ngrp = p.ngrp;
  a.balanced = p.balanced ? 1 : 0;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + p.o_floats;
  a.part_meta = reinterpret_cast<int*>(a.part_ml + p.ctas * 2 * kCols * 2);
  const int ring = kRowsWarps * kRowsRing * static_cast<int>(a.D) / 128;
  auto go = [&](auto kern) -> int {
    static_assert(kCols * 128 * 4 <= kRowsRing, "a warp's outputs fit its ring");
    SRSWA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        ring + 4 * kRowsThreads * 8));
    kern<<<static_cast<unsigned>(p.ctas), kRowsThreads, ring + static_cast<int>(a.K) * 8, st>>>(a);
    return srswa_last_launch_status();
  };
  auto by_type = [&](auto d_, auto ch_) -> int {
    constexpr int D = decltype(d_)::value, CH = decltype(ch_)::value;
    return kv_dtype == SRSWA_I8 ? go(cache8_rows_kernel<D, SRSWA_I8, CH>) : go(cache8_rows_kernel<D, SRSWA_F8E4M3, CH>);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  const int rc = a.D == 128 ? (p.ch == 2 ? by_type(D128(), Two()) : by_type(D128(), One()))
                            : (p.ch == 2 ? by_type(D64(), Two()) : by_type(D64(), One()));
  if (rc || !p.balanced) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.ctas), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = a.D == 128 ? cudaLaunchKernelEx(&cfg, cache8_merge_kernel<128>, a, static_cast<int>(p.ctas))
                                   : cudaLaunchKernelEx(&cfg, cache8_merge_kernel<64>, a, static_cast<int>(p.ctas));
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}

}  // namespace srswa
