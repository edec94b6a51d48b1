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
//   * softmax weights are rounded to f16 times 2^15 and relative to the largest of
//     their own unit (16 or 32 keys of one page): 2^-11 relative down to 2^-29 of
//     that, where f16 runs out of exponents, whatever the page's value scale.
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
// warp, so uneven lengths leave no tail and warps never wait for one another;
// an item cut in several parts leaves fp32 partials that cache8_merge_kernel
// joins in order.  Where the items are few and short the join would cost more
// than the balance gives: there the warps of a CTA share an item, and where they
// are many and short each warp has an item of its own (rows_plan).  A warp
// streams its units through a private cp.async ring; page ids, scales and biases
// are prefetched a block of 32 slots ahead.
//
// Measured: six requests of 30k to 131k keys, 32 / 8 heads of 128 (750 MB) 134
// us, 87 % of the copy rate; 256 requests with a window of 512 and 8 selected
// pages (672 MB) 126 us, 82 %.  A unit of 32 keys takes a warp about 1.3 us from
// one dependent step to the next, so few short items are bound by that chain:
// 16 requests of 1024 keys 12.2 us.

#include <cmath>
#include <type_traits>

#include "cache8_attend.cuh"
#include "tc.cuh"

namespace srswa {

constexpr float kRowsShift = 15.f;  // weights, their sums and the outputs are kept times 2^15 (of their unit, or row)
// Warps of a CTA whose warps share an item: where an SM has one such CTA, and two
// (of 128 features four warps with room for three units in flight take 18.0 us
// where six with two take 19.0: 64 requests of 16 / 4 heads, 1024 keys; of 64
// features six are faster, 14.5 and 15.3 us for 128 requests of 14 / 2 heads).
constexpr int alone_warps(int D) { return D == 128 ? 8 : 12; }
constexpr int pair_warps(int D) { return D == 128 ? 4 : 6; }
// Shared memory of a warp's ring, D = 128: three units of 32 keys; 64: two (four
// are no faster, and eight warps an SM with 24 KB each beat twelve with 16 KB
// at D = 128: 134.5 and 139 us for the 750 MB of six requests of 30k to 131k keys).
constexpr int ring_bytes(int D) { return D == 128 ? 24576 : 8192; }
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
template <int D, int KVT, int CH, bool MULTI, int NW>
__global__ void __launch_bounds__(32 * NW, NW == alone_warps(D) ? 1 : 2) cache8_rows_kernel(const Attend8Args a) {
  constexpr int CB = 16 * D;           // bytes of a chunk of K (or V)
  constexpr int SB = 2 * CH * CB;      // bytes of a stage: K of its chunks, then V
  constexpr int ST = ring_bytes(D) / SB;  // stages of a warp's ring
  constexpr int UK = 16 * CH;          // keys of a unit
  constexpr int KS = D / 16;           // MMA steps of a dot product, and feature tiles of the output
  constexpr int RPI = 512 / D;         // key rows per warp copy instruction
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t f_sum[(32 * NW) + 1];
  __shared__ float w_ml[NW][2 * kCols];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t = lane & 3, g = lane >> 2;
  const int bs = static_cast<int>(a.BS), upp = bs / UK;  // units per page
  const int G = static_cast<int>(a.H / a.Hkv), K = static_cast<int>(a.K);
  const int share = MULTI ? static_cast<int>(a.share) : 1;
  const int sinks = static_cast<int>(min(a.sinks, static_cast<int64_t>(0x7fffff00)));
  const int win = a.window < 0 ? 0x7fffff00 : static_cast<int>(min(a.window, static_cast<int64_t>(0x7fffff00)));
  const uint32_t ring = smem_u32(smem) + warp * ST * SB;
  const int krow = (g >> 1) + 4 * (g & 1);  // the key of MMA row g (and + 8 of row g + 8)
  const int cr = lane / (D / 16), cc = lane % (D / 16);  // key row and 16-byte unit of this lane's copies
  pdl_launch_dependents();
  pdl_wait();

  // One (row group, kv head, column group), units [c0, c1) of its `s.units`.
  // po == nullptr: the whole item, results written out; else a part: its
  // unnormalised outputs to po [8 columns][D], maxima and sums to pml [8][2].
  auto process = [&](int64_t rg, int64_t req, const Span& s, int64_t hk, int grp, int c0, int c1, float* po,
                     float* pml) {
    const int64_t n0 = rg * share;
    // ---- slots: lane l of (cur, nxt) holds slot base + l, base + 32 + l ----
    const int n_fix = s.n_sink + s.n_win, nslots = n_fix + K;
    struct Pages {
      int blk, page;  // page < 0: nothing to see there
      float ks, vs, b2;
    };
    auto load_pages = [&](int first) {
      const int i = first + lane, si = i - n_fix;
      Pages r = {i < s.n_sink ? i : s.b0 + i - s.n_sink, -1, 0.f, 0.f, 0.f};
      bool on = i < n_fix;
      if (first + 31 >= n_fix && first < nslots) {  // selected blocks: ids in the table, each once
        const int64_t ib = hk * a.s_ti_h + n0 * a.s_ti_n;
        int64_t b = -1;
        if (si >= 0 && si < K) {
          b = load_index(a.sel, ib + si, a.idx_is64);
          if (a.bias) {  // (the ends of fp32 stay finite: such a mask is not -inf)
            const float b0 = a.bias[hk * a.s_b_h + n0 * a.s_b_n + si];
            r.b2 = fabsf(b0) < INFINITY ? fminf(fmaxf(b0 * kLog2e, -3.402823466e38f), 3.402823466e38f) : b0;
          }
        }
        bool once = b >= 0 && b < a.W;
        const int upto = min(first + 31 - n_fix, K - 1);  // the last selected slot of this block
        for (int j0 = 0; j0 <= upto; j0 += 32) {
          const int64_t other = j0 + lane < K ? load_index(a.sel, ib + j0 + lane, a.idx_is64) : -1;
          for (int j = 0; j < min(32, upto - j0); ++j)
            if (__shfl_sync(0xffffffffu, other, j) == b && j0 + j < si) once = false;
        }
        if (si >= 0) r.blk = once ? static_cast<int>(b) : 0;
        on = on || (si >= 0 && once);
      }
      if (on) {
        const int page = a.table[req * a.s_bt + r.blk];
        if (page >= 0 && page < a.P) {
          r.page = page;
          r.ks = a.ks[page * a.s_scale + hk];
          r.vs = a.vs[page * a.s_scale + hk];
        }
      }
      return r;
    };
    int base = (c0 / upp) & ~31;
    Pages cur = load_pages(base), nxt = load_pages(base + 32);
    auto limits = [&](int si, int blk, int& lo, int& hi) {
      lo = si < s.n_sink ? 0 : si < n_fix ? s.ls0 : max(blk * bs, sinks);
      hi = si < s.n_sink ? s.sink_end : si < n_fix ? s.end : min(min((blk + 1) * bs, s.ls0), s.end);
    };

    // the producer runs ST - 1 units ahead
    int p_si = c0 / upp, p_u = c0 % upp, p_i = c0, p_stage = 0;
    auto issue = [&]() {
      if (p_i < c1) {
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
        if (++p_u == upp) { p_u = 0; ++p_si; }
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

    int c_si = c0 / upp, c_u = c0 % upp, c_stage = 0;
    for (int i = c0; i < c1; ++i) {
      if (c_si - base >= 32) {
        base += 32;
        cur = nxt;
        nxt = load_pages(base + 32);
      }
      cp_async_wait<ST - 2>();
      __syncwarp();  // every lane's copies have landed, and every lane is done with the stage issued next
      issue();
      const int rel = c_si - base, si = c_si;
      const int page = __shfl_sync(0xffffffffu, cur.page, rel), blk = __shfl_sync(0xffffffffu, cur.blk, rel);
      const float ks = __shfl_sync(0xffffffffu, cur.ks, rel), vs = __shfl_sync(0xffffffffu, cur.vs, rel);
      const float b2 = __shfl_sync(0xffffffffu, cur.b2, rel);
      int lo, hi;
      limits(si, blk, lo, hi);
      const int k0 = blk * bs + c_u * UK;
      const uint32_t src = ring + c_stage * SB;
      if (++c_u == upp) { c_u = 0; ++c_si; }
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
      const float f0 = z0 * ks, f1 = z1 * ks;
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
      if (MULTI) whole = whole && k0 + UK - 1 <= s.p0 && (k0 > s.p0 + share - 1 - win || k0 + UK - 1 < sinks);
      auto sees = [&](int j, int r) { return j <= s.p0 + r && (j > s.p0 + r - win || j < sinks); };
      if (!whole) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const int j = k0 + c * 16 + krow + 8 * hh;
            const bool in = j >= lo && j < hi;
            if (!(in && (!MULTI || sees(j, row0)))) x[c][2 * hh] = -INFINITY;
            if (!(in && (!MULTI || sees(j, row1)))) x[c][2 * hh + 1] = -INFINITY;
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
        const float al0 = ex2(m0 - u0), al1 = ex2(m1 - u1);
        l0 *= al0;
        l1 *= al1;
#pragma unroll
        for (int e = 0; e < KS; ++e) {
          o[e][0] *= al0; o[e][1] *= al1; o[e][2] *= al0; o[e][3] *= al1;
        }
        m0 = n0m;
        m1 = n1m;
      }
      // weights relative to the unit's largest; what that is to the row's comes in
      // fp32, with the value scale
      const float a0 = ex2(c0m - u0), a1 = ex2(c1m - u1);
      const float e0 = (c0m == -INFINITY ? 0.f : c0m) - kRowsShift, e1 = (c1m == -INFINITY ? 0.f : c1m) - kRowsShift;
      float s0 = 0.f, s1 = 0.f;
      uint32_t pb[CH][2];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float p0 = ex2(x[c][0] - e0), p1 = ex2(x[c][1] - e1), p2 = ex2(x[c][2] - e0), p3 = ex2(x[c][3] - e1);
        s0 += p0 + p2;
        s1 += p1 + p3;
        pb[c][0] = transpose8x8(pack_half2(p0, p1));
        pb[c][1] = transpose8x8(pack_half2(p2, p3));
      }
      l0 = fmaf(s0, a0, l0);
      l1 = fmaf(s1, a1, l1);
      const float vs0 = vs * a0, vs1 = vs * a1;
      uint32_t w[CH][4][D / 32];
      load_v(src + CH * CB, w);
      if (!MULTI || whole) {  // masked keys were filled with zeros
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          float acc[2][4] = {};
          pv_tile(w, e, pb, acc);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int y = 0; y < 4; ++y) o[2 * e + u][y] = fmaf(y & 1 ? vs1 : vs0, acc[u][y], o[2 * e + u][y]);
        }
      } else {
        // rows of the group see different keys: each takes the unit with the
        // keys that it does not see zeroed (their codes may be NaN), or not at
        // all (the page's scale may be)
        for (int r = grp * kCols / G; r <= min((grp * kCols + kCols - 1) / G, share - 1); ++r) {
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
              oo[0] = take0 ? fmaf(vs0, acc[u][0], oo[0]) : oo[0];
              oo[1] = take1 ? fmaf(vs1, acc[u][1], oo[1]) : oo[1];
              oo[2] = take0 ? fmaf(vs0, acc[u][2], oo[2]) : oo[2];
              oo[3] = take1 ? fmaf(vs1, acc[u][3], oo[3]) : oo[3];
            }
          }
        }
      }
    }
    cp_async_wait<0>();

    __syncwarp();  // the ring is free for the next item

#pragma unroll
    for (int msk = 4; msk < 32; msk <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, msk);
      l1 += __shfl_xor_sync(0xffffffffu, l1, msk);
    }
    // this thread: columns 2 t, 2 t + 1, features g * 2 KS .. + 2 KS - 1 (MMA
    // rows g and g + 8 of tile e hold 2 e and 2 e + 1 of them)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int col = 2 * t + u, gc = grp * kCols + col;
      if (gc >= share * G) continue;
      const float m = u ? m1 : m0, l = u ? l1 : l0;
      float x[2 * KS];
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        x[2 * e] = o[e][u];
        x[2 * e + 1] = o[e][2 + u];
      }
      if (!po) {
        const int64_t n = n0 + gc / G, h = hk * G + gc % G;
        const bool any = l > 0.f || l != l;
#pragma unroll
        for (int e = 0; e < 2 * KS; ++e) x[e] = any ? x[e] / l : 0.f;
#pragma unroll
        for (int e = 0; e < 2 * KS; e += 8) store8(a.out, n * a.s_on + h * a.s_oh + g * 2 * KS + e, a.out_dtype, x + e);
        if (g == 0 && a.lse) a.lse[n * a.H + h] = any ? (m - kRowsShift + log2f(l)) * kLn2 : -INFINITY;
      } else {
        float4* p = reinterpret_cast<float4*>(po + col * D + g * 2 * KS);
#pragma unroll
        for (int e = 0; e < 2 * KS; e += 4) p[e / 4] = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        if (g == 0) {
          pml[col * 2] = m;
          pml[col * 2 + 1] = l;
        }
      }
    }
  };

  const int64_t per_group = a.Hkv * a.ngrp;  // items of a row group
  const int64_t me = static_cast<int64_t>(blockIdx.x) * NW + warp;  // this warp's part
  const int64_t groups = a.N / share;
  int64_t req, pos, stop, rg, off;
  Span s;
  if (a.split == kSplitCta) {  // a part of the CTA's item
    rg = blockIdx.x / per_group;
    s = group_span<CH>(a, rg, req);
    pos = s.units * warp / NW;
    stop = s.units * (warp + 1) / NW;
    off = (blockIdx.x % per_group) * s.units + pos;
  } else if (a.split == kSplitNone) {  // one warp per item
    rg = me / per_group;
    if (rg >= groups) return;
    s = group_span<CH>(a, rg, req);
    pos = 0;
    stop = s.units;
    off = (me % per_group) * s.units;
  } else {  // an equal part of all units
    const int64_t per = (groups + (32 * NW) - 1) / (32 * NW);
    const int64_t g_lo = min(tid * per, groups), g_hi = min(g_lo + per, groups);
    int64_t sum = 0;
    for (int64_t i = g_lo; i < g_hi; ++i) sum += group_span<CH>(a, i, req).units;
    f_sum[tid + 1] = sum;
    if (tid == 0) f_sum[0] = 0;
    __syncthreads();
    if (warp == 0) {  // prefix sums of the threads' shares
      int64_t run = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        int64_t x = f_sum[w * 32 + lane + 1];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
          if (lane >= d) x += y;
        }
        f_sum[w * 32 + lane + 1] = run + x;
        run += __shfl_sync(0xffffffffu, x, 31);
      }
    }
    __syncthreads();
    const int64_t total = f_sum[(32 * NW)] * per_group, parts = static_cast<int64_t>(gridDim.x) * NW;
    pos = total * me / parts;
    stop = total * (me + 1) / parts;
    // the share, then the row group, that holds unit `pos`
    int lo = 0, hi = (32 * NW);
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (f_sum[mid] * per_group <= pos) lo = mid;
      else hi = mid;
    }
    off = pos - f_sum[lo] * per_group;
    rg = lo * per;
    if (pos < stop) {
      for (;; ++rg) {
        s = group_span<CH>(a, rg, req);
        if (off < s.units * per_group) break;
        off -= s.units * per_group;
      }
    }
  }
  int head_rg = pos < stop ? -1 : -2;  // -2, an empty part: an item may go on behind it
  int head_item = 0, tail_rg = -1, tail_item = 0;
  bool once = a.split == kSplitCta;  // its part, an empty one too, goes to shared memory
  while (pos < stop || once) {
    const int64_t it = off / s.units;
    const int c0 = static_cast<int>(off % s.units);
    const int c1 = static_cast<int>(min(static_cast<int64_t>(s.units), c0 + stop - pos));
    float *po = nullptr, *pml = nullptr;
    if (once) {
      po = reinterpret_cast<float*>(smem + warp * ST * SB);  // this warp's ring, when it is done with it
      pml = w_ml[warp];
      once = false;
    } else if (c0 > 0 || c1 < s.units) {
      const int64_t slot = c0 > 0 ? 2 * me : 2 * me + 1;
      (c0 > 0 ? head_rg : tail_rg) = static_cast<int>(rg);
      (c0 > 0 ? head_item : tail_item) = static_cast<int>(it);
      po = a.part_o + slot * kCols * D;
      pml = a.part_ml + slot * kCols * 2;
    }
    process(rg, req, s, it / a.ngrp, static_cast<int>(it % a.ngrp), c0, c1, po, pml);
    pos += c1 - c0;
    off += c1 - c0;
    if (off == s.units * per_group && pos < stop) {
      off = 0;
      s = group_span<CH>(a, ++rg, req);
    }
  }
  if (a.split == kSplitEqual) {
    if (lane == 0) reinterpret_cast<int4*>(a.part_meta)[me] = make_int4(head_rg, head_item, tail_rg, tail_item);
  } else if (a.split == kSplitCta) {  // join the warps' parts
    __syncthreads();
    const int64_t it = blockIdx.x % per_group, hk = it / a.ngrp, row0 = blockIdx.x / per_group * share;
    const int first = static_cast<int>(it % a.ngrp) * kCols, ncol = min(share * G - first, kCols);
    for (int i = tid; i < ncol * D; i += (32 * NW)) {
      const int col = i / D, d = i % D, gc = first + col;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, w_ml[w][2 * col]);
      const float Mu = M == -INFINITY ? 0.f : M;
      float L = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = exp2f(w_ml[w][2 * col] - Mu);
        L += w_ml[w][2 * col + 1] * f;
        x += reinterpret_cast<const float*>(smem + w * ST * SB)[col * D + d] * f;
      }
      const bool any = L > 0.f || L != L;
      const int64_t n = row0 + gc / G, h = hk * G + gc % G;
      store_elem(a.out, n * a.s_on + h * a.s_oh + d, a.out_dtype, any ? x / L : 0.f);
      if (d == 0 && a.lse) a.lse[n * a.H + h] = any ? (M - kRowsShift + log2f(L)) * kLn2 : -INFINITY;
    }
  }
}

// Joins the parts of one column (blockIdx.y) of the item that part blockIdx.x
// began and did not finish, in their order: the weights first, then the four
// warps add every fourth part's features, then the four sums are added.
template <int D>
__global__ void __launch_bounds__(128) cache8_merge_kernel(const Attend8Args a, int parts) {
  constexpr int V = D / 32;  // features of a lane
  __shared__ float wt[128], red[4][D], top[4];
  // (no early launch of what follows: beside these CTAs a next attend would not get
  // all its CTAs at once, and its equal parts want to start together: 171 us for 130)
  pdl_wait();
  const int c = blockIdx.x, col = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4* meta = reinterpret_cast<const int4*>(a.part_meta);
  const int rg = meta[c].z, it = meta[c].w;
  if (rg < 0) return;
  const int64_t hk = it / a.ngrp;
  const int grp = static_cast<int>(it % a.ngrp), G = static_cast<int>(a.H / a.Hkv), gc = grp * kCols + col;
  if (gc >= a.share * G) return;
  // the parts behind it that go on with the item: a run, with empty parts in it
  int end = c + 1;
  for (;; end += 32) {
    const int j = end + lane;
    const int4 x = j < parts ? meta[j] : make_int4(-1, 0, 0, 0);
    const unsigned stop = __ballot_sync(0xffffffffu, !(x.x == -2 || (x.x == rg && x.y == it)));
    if (stop) {
      end += __ffs(stop) - 1;
      break;
    }
  }
  float M = -INFINITY, L = 0.f, acc[V] = {};
  for (int j0 = c; j0 < end; j0 += 128) {
    const int j = j0 + tid;
    const bool on = j < end && (j == c || meta[j].x != -2);
    const int64_t at = (j == c ? 2 * static_cast<int64_t>(j) + 1 : 2 * static_cast<int64_t>(j)) * kCols + col;
    const float m = on ? a.part_ml[at * 2] : -INFINITY, l = on ? a.part_ml[at * 2 + 1] : 0.f;
    const float wm = warp_max(m);
    __syncthreads();  // the previous round's weights are used up
    if (lane == 0) top[warp] = wm;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), M), mu = mn == -INFINITY ? 0.f : mn;
    const float old = exp2f(M - mu), f = on ? exp2f(m - mu) : -1.f;  // -1: nothing was written there
    wt[tid] = f;
    __syncthreads();
    L = L * old + warp_sum(on ? l * f : 0.f);  // this warp's 32 parts of each round
    M = mn;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= old;
    const int n = min(128, end - j0);
#pragma unroll 4
    for (int i = warp; i < n; i += 4) {
      const float w = wt[i];
      if (w >= 0.f || w != w) {
        const int64_t part = j0 + i;
        const float* x = a.part_o + ((part == c ? 2 * part + 1 : 2 * part) * kCols + col) * D + lane * V;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(w, x[e], acc[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) red[warp][lane * V + e] = acc[e];
  __syncthreads();
  if (lane == 0) top[warp] = L;
  __syncthreads();
  L = (top[0] + top[1]) + (top[2] + top[3]);
  const int64_t n = static_cast<int64_t>(rg) * a.share + gc / G, h = hk * G + gc % G;
  const bool any = L > 0.f || L != L;
  if (tid < D) {
    const float x = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
    store_elem(a.out, n * a.s_on + h * a.s_oh + tid, a.out_dtype, any ? x / L : 0.f);
  }
  if (tid == 0 && a.lse) a.lse[n * a.H + h] = any ? (M - kRowsShift + log2f(L)) * kLn2 : -INFINITY;
}

int sm_count() {
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
  // units of 32 keys where a page holds whole ones (16: 2 to 14 % slower on the
  // same pages from 512 keys up, as 215 for 196 us for 512 requests of 2048)
  p.ch = d.block_size % 32 == 0 ? 2 : 1;
  const int64_t upp = d.block_size / (16 * p.ch);
  int64_t blocks = d.W;
  if (d.window >= 0) {
    const int64_t win = (d.window + p.share - 1 + d.block_size - 1) / d.block_size + 1;
    const int64_t snk = (d.sinks + d.block_size - 1) / d.block_size;
    blocks = win < d.W && snk < d.W && win + snk < d.W ? win + snk : d.W;
  }
  const int64_t most = (blocks + d.K) * upp;
  const int64_t slots = static_cast<int64_t>(sm_count()) * kRowsCtasPerSm * kRowsWarps;
  int64_t parts = p.items;
  p.warps = kRowsWarps;
  p.split = kSplitNone;
  p.units = p.items * most;
  const int64_t wave = slots / kRowsWarps;  // CTAs of four warps at a time
  if (d.nsplit > 0) {
    const int64_t n = d.nsplit < most ? d.nsplit : most > 1 ? most : 1;  // a unit each at least
    if (n > 1) p.split = kSplitEqual;
    parts = n * p.items;
  } else {
    // The three ways, in us for n requests of 16 / 4 heads of 128 and L keys (4 n
    // items of L / 32 units; one warp each, a CTA each, equal parts):
    //     n   L=128               256                  512                  1024                 2048
    //     1  10.6   7.9  12.8   14.5   7.6  12.9   22.2   8.8  12.8   37.7  11.8  12.9   68.4  17.4  13.8
    //    16  10.9   7.1  11.8   14.9   7.6  12.7   22.7   9.2  13.1   38.3  12.2  14.9   69.4  17.7  19.2
    //    64  11.4   8.0  14.2   16.1   9.5  14.8   23.9  12.3  20.2   41.8  17.8  24.4   81.8  31.3  38.0
    //   128  12.1  14.5  15.3   17.2  17.3  20.8   27.9  23.0  25.0   50.7  38.0  38.4   91.6  59.0  59.4
    //   256  12.6  26.8  23.7   18.2  32.5  29.4   31.9  50.2  41.9   53.2  71.8  63.0   95.6 108.2 101.3
    //  1024  54.3 104.2  71.2   77.1 129.0  96.8  114.6 168.9 131.5  192.6 241.0 196.1  347.6 390.3 349.4
    // (pages in L2 up to 128 MB).  Over 13 x 8 sizes of 16 / 4 and 10 / 10 heads,
    // with tables as wide as the longest request, the rules below take 1.5 % more
    // than the best of the three.  The host knows a table's width, not the lengths: a
    // short request in a wide table takes equal parts (n = 1, L = 256: 12.9 for 7.6).
    // A join of parts costs about 6 us; a warp or a CTA per item leaves the long
    // items' ends alone on the GPU, so neither takes items of many units.
    const bool many = p.items > wave && most * slots <= 20 * p.items;  // one warp each while the others have items too
    const int64_t cap = 12 * p.items / slots > 16 ? 12 * p.items / slots : 16;
    const int64_t warps = p.items <= sm_count() ? alone_warps(static_cast<int>(d.D))
                          : p.items <= 2 * sm_count() ? pair_warps(static_cast<int>(d.D)) : kRowsWarps;
    if (groups > 2048 || (many && most <= cap)) {
      // (over 2048 groups each warp's search for its equal part costs more than
      // the balance gives: 2500 requests of 1024 keys 439, equal parts 454)
    } else if (2 * p.items <= 3 * wave && most <= (p.items <= wave ? 64 : 16) &&
               5 * most * slots <= warps * (20 * slots + 6 * p.units)) {
      p.split = kSplitCta;  // a warp's units, most / warps, at most 4 + 1.2 times an equal part
      p.warps = static_cast<int>(warps);
      parts = p.items * p.warps;
    } else {
      p.split = kSplitEqual;
      const int64_t enough = (p.units + 1) / 2;  // two units each at least
      parts = enough < slots ? enough : slots;
    }
  }
  p.ctas = (parts + p.warps - 1) / p.warps;
  if (p.split == kSplitEqual) {
    parts = p.ctas * kRowsWarps;
    const int64_t f = parts * 2 * kCols;
    p.o_floats = f * d.D;
    p.bytes = static_cast<size_t>(p.o_floats + f * 2 + parts * 4) * 4;
  }
  return p;
}

template <int D, int KVT, int CH, bool MULTI, int NW>
static int rows_start(const Attend8Args& a, unsigned ctas, cudaStream_t st) {
  auto kern = cache8_rows_kernel<D, KVT, CH, MULTI, NW>;
  const int ring = NW * ring_bytes(D);
  static bool allowed[64] = {};  // per device: the shared memory has been asked for
  int dev = 0;
  SRSWA_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !allowed[dev]) {
    SRSWA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ring));
    if (dev < 64) allowed[dev] = true;
  }
  return launch_pdl(kern, dim3(ctas), 32 * NW, ring, st, a);
}

int rows_launch(Attend8Args a, const RowsPlan& p, int kv_dtype, void* workspace, cudaStream_t st) {
  if (p.ctas >= (1ll << 28)) return SRSWA_ETOOLARGE;
  a.share = p.share;
  a.ngrp = p.ngrp;
  a.split = p.split;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + p.o_floats;
  const int64_t parts = p.ctas * kRowsWarps;
  a.part_meta = reinterpret_cast<int*>(a.part_ml + parts * 2 * kCols * 2);
  const unsigned ctas = static_cast<unsigned>(p.ctas);
  auto by_warps = [&](auto d_, auto ch_, auto type_, auto multi_) -> int {
    constexpr int D = decltype(d_)::value, CH = decltype(ch_)::value, KVT = decltype(type_)::value;
    constexpr bool MULTI = decltype(multi_)::value;
    return p.warps == kRowsWarps      ? rows_start<D, KVT, CH, MULTI, kRowsWarps>(a, ctas, st)
           : p.warps == pair_warps(D) ? rows_start<D, KVT, CH, MULTI, pair_warps(D)>(a, ctas, st)
                                      : rows_start<D, KVT, CH, MULTI, alone_warps(D)>(a, ctas, st);
  };
  auto by_type = [&](auto d_, auto ch_) -> int {
    using I8 = std::integral_constant<int, SRSWA_I8>;
    using E4 = std::integral_constant<int, SRSWA_F8E4M3>;
    if (p.share > 1)
      return kv_dtype == SRSWA_I8 ? by_warps(d_, ch_, I8(), std::true_type()) : by_warps(d_, ch_, E4(), std::true_type());
    return kv_dtype == SRSWA_I8 ? by_warps(d_, ch_, I8(), std::false_type()) : by_warps(d_, ch_, E4(), std::false_type());
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  const int rc = a.D == 128 ? (p.ch == 2 ? by_type(D128(), Two()) : by_type(D128(), One()))
                            : (p.ch == 2 ? by_type(D64(), Two()) : by_type(D64(), One()));
  if (rc || p.split != kSplitEqual) return rc;
  const int64_t cols = p.share * (a.H / a.Hkv);
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(cols < kCols ? cols : kCols));
  return a.D == 128 ? launch_pdl(cache8_merge_kernel<128>, grid, 128, 0, st, a, static_cast<int>(parts))
                    : launch_pdl(cache8_merge_kernel<64>, grid, 128, 0, st, a, static_cast<int>(parts));
}

}  // namespace srswa
