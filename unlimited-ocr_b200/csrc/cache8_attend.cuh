// Arguments of the scaled 8-bit cache's attend kernels.
#pragma once

#include "cache8.cuh"

namespace srswa {

// One warp per item; the warps of a CTA per item; equal parts of all units per warp.
enum { kSplitNone = 0, kSplitCta = 1, kSplitEqual = 2 };

struct Attend8Args {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  RowMap rows;
  const int32_t* table;
  const void* sel;
  const float* bias;
  void* out;
  float* lse;
  int64_t s_bt, W, P, BS, N, H, Hkv, D, K;
  int64_t window, sinks;
  int64_t s_qn, s_qh, s_on, s_oh, s_page, s_pos, s_head, s_scale;
  int64_t s_ti_h, s_ti_n, s_b_h, s_b_n;
  float scale_log2;
  int q_dtype, out_dtype, idx_is64;
  // single rows
  int64_t share, ngrp;  // rows that share a pass over the keys; column groups of an item
  int split;            // how the items are shared out (below)
  float* part_o;        // [2 per part][8 columns][D] unnormalised partial outputs
  float* part_ml;       // [..][8][2] their maxima (log2) and sums
  int* part_meta;       // [part][4] the items its two partials belong to (row group, item, twice)
};

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

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^x to 2 ulp, subnormal results as 0 (a softmax weight under 2^-126 is one).
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
struct RowsPlan {
  int64_t share, ngrp, items, ctas, o_floats;
  int64_t units;  // of all items, at most
  size_t bytes;  // workspace
  int split;
  int ch;     // 16-key chunks of a unit
  int warps;  // of a CTA
};
constexpr int kRowsWarps = 4;  // of a CTA of the row kernel (plan.warps may be more), and CTAs an SM holds
constexpr int kRowsCtasPerSm = 2;
constexpr int kMaxSelected = 512;  // selected blocks of a row
int sm_count();
RowsPlan rows_plan(const srswa_cache8_desc& d, bool varlen);
int rows_launch(Attend8Args a, const RowsPlan& p, int kv_dtype, void* workspace, cudaStream_t st);

// Whether the tensor-core tiles take the call, and its launch (status: the
// call's status word).
bool prompt_applies(const srswa_cache8_desc& d, bool varlen);
int prompt_launch(const Attend8Args& a, int kv_dtype, int* status, cudaStream_t st);

}  // namespace srswa
