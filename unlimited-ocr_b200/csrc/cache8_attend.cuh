// Arguments of the scaled 8-bit cache's attend kernels.
#pragma once

#include "cache8.cuh"

namespace srswa {

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
  int balanced;         // 1: equal parts of all units per warp, 0: one warp per item
  float* part_o;        // [2 per part][8 columns][D] unnormalised partial outputs
  float* part_ml;       // [..][8][2] their maxima (log2) and sums
  int* part_meta;       // [part][4] the items its two partials belong to (row group, item, twice)
};

struct RowsPlan {
  int64_t share, ngrp, items, ctas, o_floats;
  size_t bytes;  // workspace
  bool balanced;
  int ch;  // 16-key chunks of a unit
};
RowsPlan rows_plan(const srswa_cache8_desc& d, bool varlen);
int rows_launch(Attend8Args a, const RowsPlan& p, int kv_dtype, void* workspace, cudaStream_t st);

}  // namespace srswa
