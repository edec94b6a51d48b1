// Scaled 8-bit paged cache: what the append and attend kernels share.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace srswa {

// Which request a row belongs to and where it sits (the two row forms of
// srswa_cache8_desc).
struct RowMap {
  const int32_t* seq_lens;
  const int32_t* cu;
  const int32_t* prefix;
  int64_t R, rps;
};

__device__ __forceinline__ void row_place(const RowMap& m, int64_t n, int64_t& req, int64_t& pos) {
  if (m.cu) {
    int64_t lo = 0, hi = m.R;  // the last request whose first row is <= n (empty requests come before it)
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (m.cu[mid] <= n) lo = mid;
      else hi = mid;
    }
    req = lo;
    // a row of no request is ahead of every key
    pos = n >= m.cu[lo] && n < m.cu[lo + 1] ? static_cast<int64_t>(m.prefix[lo]) + n - m.cu[lo] : -1;
  } else {
    req = n / m.rps;
    pos = static_cast<int64_t>(m.seq_lens[req]) - m.rps + n % m.rps;
  }
}

__device__ __forceinline__ float code_to_float(uint8_t c, int kv_dtype) {
  if (kv_dtype == SRSWA_I8) return static_cast<float>(static_cast<int8_t>(c));
  __nv_fp8_e4m3 v;
  v.__x = c;
  return static_cast<float>(v);
}

static inline bool kv_code_ok(int t) { return t == SRSWA_F8E4M3 || t == SRSWA_I8; }

}  // namespace srswa
