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
// Work split: the chunks (16 keys of one page and head) of all (row group, kv
// head) items are laid end to end and cut into equal parts, one per resident
// CTA, so uneven lengths leave no tail; an item cut in several parts leaves
// fp32 partials that cache8_merge_kernel joins in order.  Each warp streams its
// chunks through a private cp.async ring; its page ids and scales are
// prefetched a block of 32 slots ahead.

#include <cmath>

#include "cache8_attend.cuh"
#include "tc.cuh"

namespace srswa {

constexpr int kRowsThreads = 128;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsStages = 4;
constexpr int kRowsCtasPerSm = 3;
constexpr int kCols = 8;  // queries that share a pass over the keys (columns of the MMA)

// The keys a row group can see, as slots of one page each: sinks, window,
// selected blocks, in this order.
struct Span {
  int p0, ls0, sink_end, end, n_sink, b0, n_win, chunks;
};

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
  s.chunks = max((s.n_sink + s.n_win + static_cast<int>(a.K)) * (bs / 16), 1);
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
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
    lo = static_cast<uint32_t>(a.x) | (static_cast<uint32_t>(a.y) << 16);
    hi = static_cast<uint32_t>(b.x) | (static_cast<uint32_t>(b.y) << 16);
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

template <int D, int KVT>
__global__ void __launch_bounds__(kRowsThreads, kRowsCtasPerSm) cache8_rows_kernel(const Attend8Args a) {
  constexpr int CB = 16 * D;           // bytes of a chunk of K (or V)
  constexpr int KS = D / 16;           // MMA steps of a dot product, and feature tiles of the output
  constexpr int RPI = 512 / D;         // key rows per warp copy instruction
  extern __shared__ __align__(128) uint8_t smem[];
  int* sel_blk = reinterpret_cast<int*>(smem + kRowsWarps * kRowsStages * 2 * CB);
  float* sel_b2 = reinterpret_cast<float*>(sel_blk + a.K);
  __shared__ float w_m[kRowsWarps][kCols], w_l[kRowsWarps][kCols];
  __shared__ int64_t f_part[kRowsWarps], f_off;
  __shared__ int f_rg;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = lane & 3, g = lane >> 2;
  const int bs = static_cast<int>(a.BS), cpb = bs / 16;
  const int G = static_cast<int>(a.H / a.Hkv);
  const uint32_t ring = smem_u32(smem) + warp * kRowsStages * 2 * CB;
  const int krow = (g >> 1) + 4 * (g & 1);  // the key of MMA row g (and + 8 of row g + 8)
  pdl_launch_dependents();                  // the merge kernel waits for this grid before it reads

  // One (row group, kv head, column group), chunks [c0, c1) of its `s.chunks`;
  // slot < 0: the whole item, results written out; else partial `slot`.
  auto process = [&](int64_t rg, int64_t req, const Span& s, int64_t hk, int grp, int c0, int c1, int64_t slot) {
    const int K = static_cast<int>(a.K);
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
      int again[4];  // repeats of an earlier slot (K <= 4 * threads)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = tid + u * kRowsThreads;
        again[u] = 0;
        if (i < K && sel_blk[i] >= 0)
          for (int j = 0; j < i; ++j) again[u] |= sel_blk[j] == sel_blk[i];
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (again[u]) sel_blk[tid + u * kRowsThreads] = -1;
      __syncthreads();
    }

    // ---- this thread's part of query column g, as f16 MMA operands ----
    uint32_t qf[KS][2];
    float qexp;  // the power of two taken out of it
    {
      const int col = grp * kCols + g;
      const bool on = col < a.share * G;
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

    // ---- slots: lane l of (cur, nxt) holds slot base + l, base + 32 + l ----
    const int nslots = s.n_sink + s.n_win + K;
    struct Pages {
      int blk, page;
      float ks, vs;
    };
    auto load_pages = [&](int i) {
      Pages r = {0, -1, 0.f, 0.f};
      if (i < nslots) {
        r.blk = i < s.n_sink ? i : i < s.n_sink + s.n_win ? s.b0 + i - s.n_sink : sel_blk[i - s.n_sink - s.n_win];
        if (r.blk >= 0) {
          const int64_t page = a.table[req * a.s_bt + r.blk];
          if (page >= 0 && page < a.P) {
            r.page = static_cast<int>(page);
            r.ks = a.ks[page * a.s_scale + hk];
            r.vs = a.vs[page * a.s_scale + hk];
          }
        }
      }
      return r;
    };
    int base = (c0 / cpb) & ~31;
    Pages cur = load_pages(base + lane), nxt = load_pages(base + 32 + lane);
    auto limits = [&](int slot_i, int blk, int& lo, int& hi) {
      if (slot_i < s.n_sink) { lo = 0; hi = s.sink_end; }
      else if (slot_i < s.n_sink + s.n_win) { lo = s.ls0; hi = s.end; }
      else {
        lo = static_cast<int>(max(static_cast<int64_t>(blk) * bs, min(a.sinks, static_cast<int64_t>(0x7fffff00))));
        hi = min(min((blk + 1) * bs, s.ls0), s.end);
      }
    };

    const int mine = (c1 - c0 - warp + kRowsWarps - 1) / kRowsWarps;  // chunks of this warp (may be <= 0)
    auto issue = [&](int i) {
      if (i < mine) {
        const int ch = c0 + warp + i * kRowsWarps, si = ch / cpb, sub = ch % cpb, rel = si - base;
        const int page = rel < 32 ? __shfl_sync(0xffffffffu, cur.page, rel) : __shfl_sync(0xffffffffu, nxt.page, rel - 32);
        const int blk = rel < 32 ? __shfl_sync(0xffffffffu, cur.blk, rel) : __shfl_sync(0xffffffffu, nxt.blk, rel - 32);
        int lo, hi;
        limits(si, blk, lo, hi);
        const int k0 = blk * bs + sub * 16;
        if (page >= 0 && k0 < hi && k0 + 16 > lo) {
          const uint32_t dst = ring + (i % kRowsStages) * 2 * CB;
          const int c = lane % (D / 16);
          const int64_t off = page * a.s_page + hk * a.s_head + c * 16;
#pragma unroll
          for (int j = 0; j < 16 / RPI; ++j) {
            const int r = j * RPI + lane / (D / 16);
            const bool in = k0 + r >= lo && k0 + r < hi;
            const int64_t o = off + (sub * 16 + (in ? r : 0)) * a.s_pos;
            cp_async16_zfill(dst + k_off<D>(r, c), a.k + o, in);
            cp_async16_zfill(dst + CB + v_off<D>(r, c), a.v + o, in);
          }
        }
      }
      cp_async_commit();
    };

    float o[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    // P.V of the chunk in `src`, added to the columns that take it; keep: the
    // thread's four keys (t, t + 4, t + 8, t + 12) that count
    auto add_pv = [&](uint32_t src, uint32_t b0, uint32_t b1, float vs, bool take0, bool take1, uint32_t keep) {
      uint32_t w[4][D / 32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = t + 4 * i;
        if constexpr (D == 128) {
          const uint4 x = lds128(src + v_off<D>(r, g));
          w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
        } else {
          const uint2 x = lds64(src + v_off<D>(r, g >> 1) + (g & 1) * 8);
          w[i][0] = x.x; w[i][1] = x.y;
        }
        if (!(keep >> i & 1)) {
#pragma unroll
          for (int e = 0; e < D / 32; ++e) w[i][e] = 0;
        }
      }
#pragma unroll
      for (int e = 0; e < D / 32; ++e) {
        // (key, key + 4) pairs of features 4e .. 4e + 3
        uint32_t a01[4], a23[4];
        widen4<KVT>(prmt(w[0][e], w[1][e], 0x5140u), a01[0], a01[1]);
        widen4<KVT>(prmt(w[0][e], w[1][e], 0x7362u), a01[2], a01[3]);
        widen4<KVT>(prmt(w[2][e], w[3][e], 0x5140u), a23[0], a23[1]);
        widen4<KVT>(prmt(w[2][e], w[3][e], 0x7362u), a23[2], a23[3]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(acc, a01[2 * u], a01[2 * u + 1], a23[2 * u], a23[2 * u + 1], b0, b1);
          float* oo = o[2 * e + u];
          oo[0] = take0 ? fmaf(vs, acc[0], oo[0]) : oo[0];
          oo[1] = take1 ? fmaf(vs, acc[1], oo[1]) : oo[1];
          oo[2] = take0 ? fmaf(vs, acc[2], oo[2]) : oo[2];
          oo[3] = take1 ? fmaf(vs, acc[3], oo[3]) : oo[3];
        }
      }
    };

#pragma unroll
    for (int i = 0; i < kRowsStages - 1; ++i) issue(i);
    for (int i = 0; i < mine; ++i) {
      const int ch = c0 + warp + i * kRowsWarps, si = ch / cpb, sub = ch % cpb;
      if (si - base >= 32) {
        base += 32;
        cur = nxt;
        nxt = load_pages(base + 32 + lane);
      }
      cp_async_wait<kRowsStages - 2>();
      __syncwarp();  // every lane's copies have landed, and every lane is done with the stage issued next
      issue(i + kRowsStages - 1);
      const int rel = si - base;
      const int page = __shfl_sync(0xffffffffu, cur.page, rel), blk = __shfl_sync(0xffffffffu, cur.blk, rel);
      const float ks = __shfl_sync(0xffffffffu, cur.ks, rel), vs = __shfl_sync(0xffffffffu, cur.vs, rel);
      int lo, hi;
      limits(si, blk, lo, hi);
      const int k0 = blk * bs + sub * 16;
      if (page < 0 || k0 >= hi || k0 + 16 <= lo) continue;
      const uint32_t src = ring + (i % kRowsStages) * 2 * CB;

      float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int hseg = 0; hseg < D / 64; ++hseg) {
        const uint4 x = lds128(src + k_off<D>(krow, hseg * 4 + t));
        const uint4 y = lds128(src + k_off<D>(krow + 8, hseg * 4 + t));
        const uint32_t xa[4] = {x.x, x.y, x.z, x.w}, ya[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t a0, a1, a2, a3;
          widen4<KVT>(xa[e], a0, a2);
          widen4<KVT>(ya[e], a1, a3);
          mma16816(sc, a0, a1, a2, a3, qf[hseg * 4 + e][0], qf[hseg * 4 + e][1]);
        }
      }
      const float b2 = si >= s.n_sink + s.n_win ? sel_b2[si - s.n_sink - s.n_win] : 0.f;
      float x0 = fmaf(sc[0], z0 * ks, b2), x1 = fmaf(sc[1], z1 * ks, b2);
      float x2 = fmaf(sc[2], z0 * ks, b2), x3 = fmaf(sc[3], z1 * ks, b2);
      // whole: every column sees all 16 keys
      bool whole = k0 >= lo && k0 + 16 <= hi;
      const int share = static_cast<int>(a.share);
      int w = 0;
      if (share > 1) {
        w = a.window < 0 ? 0x7fffffff : static_cast<int>(min(a.window, static_cast<int64_t>(0x7fffff00)));
        const int lsl = a.window < 0 ? 0 : s.p0 + share - w;  // the last row's window start
        whole = whole && k0 + 15 <= s.p0 && (k0 >= lsl || k0 + 15 < a.sinks);
      }
      auto sees = [&](int j, int r) {  // row p0 + r of a shared group
        const int p = s.p0 + r;
        return j <= p && (a.window < 0 || j > p - w || j < a.sinks);
      };
      if (!whole) {
        const int ja = k0 + krow, jb = ja + 8;
        const bool ina = ja >= lo && ja < hi, inb = jb >= lo && jb < hi;
        if (!(ina && (share == 1 || sees(ja, row0)))) x0 = -INFINITY;
        if (!(ina && (share == 1 || sees(ja, row1)))) x1 = -INFINITY;
        if (!(inb && (share == 1 || sees(jb, row0)))) x2 = -INFINITY;
        if (!(inb && (share == 1 || sees(jb, row1)))) x3 = -INFINITY;
      }
      float c0m = fmaxf(x0, x2), c1m = fmaxf(x1, x3);
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
      const float p0 = exp2f(x0 - u0), p1 = exp2f(x1 - u1), p2 = exp2f(x2 - u0), p3 = exp2f(x3 - u1);
      l0 += p0 + p2;
      l1 += p1 + p3;
      const uint32_t b0 = transpose8x8(pack_half2(p0, p1)), b1 = transpose8x8(pack_half2(p2, p3));
      if (whole || share == 1) {
        // a column whose keys are all masked here takes nothing (0 times a NaN scale)
        add_pv(src + CB, b0, b1, vs, whole || c0m != -INFINITY, whole || c1m != -INFINITY, 15u);
      } else {
        // rows of the group see different keys: each with the others' keys zeroed
        for (int r = 0; r < share; ++r) {
          uint32_t keep = 0;
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) keep |= static_cast<uint32_t>(sees(k0 + t + 4 * i2, r)) << i2;
          add_pv(src + CB, b0, b1, vs, row0 == r && c0m != -INFINITY, row1 == r && c1m != -INFINITY, keep);
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
    const int ncol = min(static_cast<int>(a.share) * G - grp * kCols, kCols);
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
  } else {  // this CTA's equal part of all chunks
    const int64_t groups = a.N / a.share;
    const int64_t per = (groups + kRowsThreads - 1) / kRowsThreads;
    const int64_t g_lo = min(tid * per, groups), g_hi = min(g_lo + per, groups);
    int64_t sum = 0;
    for (int64_t i = g_lo; i < g_hi; ++i) sum += group_span(a, i, req).chunks;
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
        const int64_t n = group_span(a, i, req).chunks * per_group;
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
    Span s = group_span(a, rg, req);
    int64_t off = a.balanced ? f_off : (blockIdx.x % per_group) * s.chunks;
    if (!a.balanced) stop = s.chunks;
    while (pos < stop) {
      const int64_t it = off / s.chunks;
      const int c0 = static_cast<int>(off % s.chunks);
      const int c1 = static_cast<int>(min(static_cast<int64_t>(s.chunks), c0 + stop - pos));
      int64_t slot = -1;
      if (c0 > 0) {
        slot = 2 * static_cast<int64_t>(blockIdx.x);
        head_item_rg = static_cast<int>(rg);
        head_item = static_cast<int>(it);
      } else if (c1 < s.chunks) {
        slot = 2 * static_cast<int64_t>(blockIdx.x) + 1;
        tail_item_rg = static_cast<int>(rg);
        tail_item = static_cast<int>(it);
      }
      process(rg, req, s, it / a.ngrp, static_cast<int>(it % a.ngrp), c0, c1, slot);
      pos += c1 - c0;
      off += c1 - c0;
      if (off == s.chunks * per_group && pos < stop) {
        off = 0;
        s = group_span(a, ++rg, req);
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
  // the most chunks an item can have
  const int64_t cpb = d.block_size / 16;
  int64_t blocks = d.W;
  if (d.window >= 0) {
    const int64_t win = (d.window + p.share - 1 + d.block_size - 1) / d.block_size + 1;
    const int64_t snk = (d.sinks + d.block_size - 1) / d.block_size;
    blocks = win < d.W && snk < d.W && win + snk < d.W ? win + snk : d.W;
  }
  const int64_t most = (blocks + d.K) * cpb;
  const int64_t slots = static_cast<int64_t>(sm_count()) * kRowsCtasPerSm;
  if (d.nsplit > 0) {
    p.balanced = d.nsplit > 1;
    p.ctas = d.nsplit * p.items;
  } else if (most <= 8 * kRowsWarps || groups > 2048 || p.items > 16 * slots) {
    // short items (a join would cost more than it saves), or so many that their
    // uneven ends do not show: one CTA each
    p.balanced = false;
    p.ctas = p.items;
  } else {
    p.balanced = true;
    const int64_t enough = (p.items * most + 2 * kRowsWarps - 1) / (2 * kRowsWarps);
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
  const int smem = kRowsWarps * kRowsStages * 2 * 16 * static_cast<int>(a.D) + static_cast<int>(a.K) * 8;
  auto go = [&](auto kern) -> int {
    static_assert(kRowsWarps * kCols * 128 * 4 <= kRowsWarps * kRowsStages * 2 * 16 * 128, "outputs fit the rings");
    SRSWA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kRowsWarps * kRowsStages * 2 * 16 * 128 + 4 * kRowsThreads * 8));
    kern<<<static_cast<unsigned>(p.ctas), kRowsThreads, smem, st>>>(a);
    return srswa_last_launch_status();
  };
  int rc;
  if (a.D == 128) rc = kv_dtype == SRSWA_I8 ? go(cache8_rows_kernel<128, SRSWA_I8>) : go(cache8_rows_kernel<128, SRSWA_F8E4M3>);
  else rc = kv_dtype == SRSWA_I8 ? go(cache8_rows_kernel<64, SRSWA_I8>) : go(cache8_rows_kernel<64, SRSWA_F8E4M3>);
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
