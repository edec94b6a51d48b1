// Scaled 8-bit paged cache: the append (quantise new tokens into their pages)
// and the C entries of the append and the attend.
//
// Append.  Per (page, head), for K and V apart:
//   s_new = 2^ceil(log2(max|x| / qmax)) over the new elements of the page,
//   s = s_new, or max(s_old, s_new) when the page holds earlier tokens,
//   earlier codes c <- round(c * s_old / s) if s > s_old, new codes round(x / s).
// A power of two makes x / s exact (the one rounding is the code's) and costs
// e4m3 no precision (a shift of the exponent); a page whose scale grows shifts
// its e4m3 codes exactly until they reach the smallest exponents, and an int8
// code is off by less than one step after any number of growths (each adds half
// a step, and halves what was there).

#include <cmath>

#include "cache8_attend.cuh"

namespace srswa {

struct AppendArgs {
  const void* x[2];  // new k, v
  uint8_t* cache[2];
  float* scale[2];
  int64_t s_xn[2], s_xh[2];
  RowMap rows;
  const int32_t* table;
  int64_t s_bt, W, P, BS, N, Hkv;
  int64_t s_page, s_pos, s_head, s_scale;
  int x_dtype;
};

template <int KVT>
__device__ __forceinline__ uint8_t to_code(float y) {
  if (KVT == SRSWA_I8) {
    if (y != y) return 0;
    return static_cast<uint8_t>(static_cast<int8_t>(static_cast<int>(rintf(fminf(fmaxf(y, -127.f), 127.f)))));
  }
  return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

// The smallest power of two s with amax <= qmax * s, at least 2^-64 (its
// inverse is then a normal number too).  qmax is 1.75 * 2^8 or 1.984375 * 2^6.
template <int KVT>
__device__ __forceinline__ float pow2_scale(float amax) {
  constexpr int shift = KVT == SRSWA_I8 ? 6 : 8;
  constexpr uint32_t top = KVT == SRSWA_I8 ? 0x7e0000u : 0x600000u;  // mantissa of qmax
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - 127 - shift + ((u & 0x7fffffu) > top ? 1 : 0);
  e = e < -64 ? -64 : e;  // subnormal amax too: its exponent field is 0
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

constexpr int kAppendThreads = 128;

// One CTA per (page a request's new tokens touch, head, K or V).
template <int D, int KVT>
__global__ void __launch_bounds__(kAppendThreads) cache8_append_kernel(const AppendArgs a) {
  constexpr int LPT = D / 8;                     // lanes per token, 8 elements each
  constexpr int TPP = kAppendThreads / LPT;      // tokens per pass
  __shared__ float red[kAppendThreads / 32];
  const int tid = threadIdx.x;
  const int64_t head = blockIdx.y;
  const int which = blockIdx.z;

  // the slot's request and page: request r has at most (n + BS - 2) / BS + 1
  // touched pages, so its slots begin at cu[r] / BS + 2 r (varlen)
  int64_t req, start, n, row0, nth;
  if (a.rows.cu) {
    const int64_t i = blockIdx.x;
    int64_t lo = 0, hi = a.rows.R;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.rows.cu[mid] / a.BS + 2 * mid <= i) lo = mid;
      else hi = mid;
    }
    req = lo;
    row0 = a.rows.cu[req];
    nth = i - (row0 / a.BS + 2 * req);
    n = a.rows.cu[req + 1] - row0;
    start = a.rows.prefix[req];
  } else {
    const int64_t per = (a.rows.rps + a.BS - 2) / a.BS + 1;
    req = blockIdx.x / per;
    nth = blockIdx.x % per;
    n = a.rows.rps;
    row0 = req * n;
    start = static_cast<int64_t>(a.rows.seq_lens[req]) - n;
  }
  if (n <= 0 || start < 0 || row0 < 0 || row0 + n > a.N) return;
  const int64_t blk = start / a.BS + nth;
  const int64_t lo = max(start, blk * a.BS), hi = min(start + n, (blk + 1) * a.BS);  // positions written here
  if (lo >= hi || blk >= a.W) return;
  const int64_t page = a.table[req * a.s_bt + blk];
  if (page < 0 || page >= a.P) return;

  const void* x = a.x[which];
  const int64_t xoff = head * a.s_xh[which];
  const int64_t s_xn = a.s_xn[which];
  uint8_t* dst = a.cache[which] + page * a.s_page + head * a.s_head;
  float* scale = a.scale[which] + page * a.s_scale + head;
  const int g = tid / LPT, u = tid % LPT;

  float amax = 0.f;
  for (int64_t p = lo + g; p < hi; p += TPP) {
    float f[8];
    load8(x, (row0 + p - start) * s_xn + xoff + u * 8, a.x_dtype, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = fabsf(f[e]);
      if (v <= 3.402823466e38f) amax = fmaxf(amax, v);  // finite elements only
    }
  }
  amax = warp_max(amax);
  if ((tid & 31) == 0) red[tid >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) amax = fmaxf(amax, red[w]);

  float s = pow2_scale<KVT>(amax);
  const int64_t held = lo - blk * a.BS;  // earlier tokens of the page
  if (held > 0) {
    const float old = *scale;
    __syncthreads();  // every thread has read it
    if (s > old) {
      const float r = old / s;
      for (int64_t p = g; p < held; p += TPP) {
        uint2* c = reinterpret_cast<uint2*>(dst + p * a.s_pos + u * 8);
        uint2 w = *c;
        uint8_t* b = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = to_code<KVT>(code_to_float(b[e], KVT) * r);
        *c = w;
      }
    } else {
      s = old;
    }
  }
  if (tid == 0) *scale = s;
  for (int64_t p = lo + g; p < hi; p += TPP) {
    float f[8];
    load8(x, (row0 + p - start) * s_xn + xoff + u * 8, a.x_dtype, f);
    uint2 w;
    uint8_t* b = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = to_code<KVT>(f[e] / s);
    *reinterpret_cast<uint2*>(dst + (p - blk * a.BS) * a.s_pos + u * 8) = w;
  }
}

}  // namespace srswa

using namespace srswa;

static bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// What both calls ask of the shape, the row form and the cache.
static int check_common(const srswa_cache8_desc* d, const int32_t* seq_lens, const int32_t* cu_rows,
                        const int32_t* prefix_lens) {
  SRSWA_CHECK_ARG(d->N >= 0 && d->R >= 0 && d->Hkv > 0 && d->P >= 0 && d->W >= 0 && d->block_size > 0, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(kv_code_ok(d->kv_dtype) && (d->D == 64 || d->D == 128), SRSWA_EUNSUPPORTED);
  SRSWA_CHECK_ARG(d->block_size % 16 == 0, SRSWA_EUNSUPPORTED);
  SRSWA_CHECK_ARG(d->block_size <= 1024 && d->Hkv <= 65535, SRSWA_ETOOLARGE);
  SRSWA_CHECK_ARG(((d->s_page | d->s_pos | d->s_head) & 15) == 0, SRSWA_EALIGN);
  if (cu_rows) {
    SRSWA_CHECK_ARG(prefix_lens, SRSWA_EINVAL);
  } else {
    SRSWA_CHECK_ARG(seq_lens || d->N == 0, SRSWA_EINVAL);
    SRSWA_CHECK_ARG(d->rows_per_req > 0 && d->N == d->R * d->rows_per_req, SRSWA_EINVAL);
  }
  SRSWA_CHECK_ARG(d->N == 0 || d->R > 0, SRSWA_EINVAL);
  return SRSWA_OK;
}

static RowMap row_map(const srswa_cache8_desc* d, const int32_t* seq_lens, const int32_t* cu_rows,
                      const int32_t* prefix_lens) {
  return RowMap{seq_lens, cu_rows, prefix_lens, d->R, d->rows_per_req};
}

extern "C" int srswa_cache8_append(const srswa_cache8_desc* d, const void* k, const void* v, void* k_cache,
                                   void* v_cache, float* k_scale, float* v_scale, const int32_t* block_table,
                                   const int32_t* seq_lens, const int32_t* cu_rows, const int32_t* prefix_lens,
                                   srswa_stream_t stream) {
  SRSWA_CHECK_ARG(d, SRSWA_EINVAL);
  const int rc = check_common(d, seq_lens, cu_rows, prefix_lens);
  if (rc) return rc;
  SRSWA_CHECK_ARG(d->q_dtype == SRSWA_F32 || d->q_dtype == SRSWA_BF16 || d->q_dtype == SRSWA_F16, SRSWA_EUNSUPPORTED);
  if (d->N == 0) return SRSWA_OK;
  SRSWA_CHECK_ARG(k && v && k_cache && v_cache && k_scale && v_scale && block_table, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(aligned(k, 16) && aligned(v, 16) && aligned(k_cache, 16) && aligned(v_cache, 16), SRSWA_EALIGN);
  const int64_t m = d->q_dtype == SRSWA_F32 ? 3 : 7;
  SRSWA_CHECK_ARG(((d->s_qn | d->s_qh | d->s_on | d->s_oh) & m) == 0, SRSWA_EALIGN);
  const int64_t slots = cu_rows ? d->N / d->block_size + 2 * d->R
                                : d->R * ((d->rows_per_req + d->block_size - 2) / d->block_size + 1);
  SRSWA_CHECK_ARG(slots < (1ll << 31), SRSWA_ETOOLARGE);
  AppendArgs a = {};
  a.x[0] = k; a.x[1] = v;
  a.cache[0] = static_cast<uint8_t*>(k_cache); a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale; a.scale[1] = v_scale;
  a.s_xn[0] = d->s_qn; a.s_xh[0] = d->s_qh; a.s_xn[1] = d->s_on; a.s_xh[1] = d->s_oh;
  a.rows = row_map(d, seq_lens, cu_rows, prefix_lens);
  a.table = block_table; a.s_bt = d->s_bt; a.W = d->W; a.P = d->P; a.BS = d->block_size; a.N = d->N; a.Hkv = d->Hkv;
  a.s_page = d->s_page; a.s_pos = d->s_pos; a.s_head = d->s_head; a.s_scale = d->s_scale;
  a.x_dtype = d->q_dtype;
  const dim3 grid(static_cast<unsigned>(slots), static_cast<unsigned>(d->Hkv), 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (d->D == 128) {
    if (d->kv_dtype == SRSWA_I8) cache8_append_kernel<128, SRSWA_I8><<<grid, kAppendThreads, 0, st>>>(a);
    else cache8_append_kernel<128, SRSWA_F8E4M3><<<grid, kAppendThreads, 0, st>>>(a);
  } else {
    if (d->kv_dtype == SRSWA_I8) cache8_append_kernel<64, SRSWA_I8><<<grid, kAppendThreads, 0, st>>>(a);
    else cache8_append_kernel<64, SRSWA_F8E4M3><<<grid, kAppendThreads, 0, st>>>(a);
  }
  return srswa_last_launch_status();
}

extern "C" size_t srswa_cache8_attend_workspace_size(const srswa_cache8_desc* d, int varlen) {
  if (!d || d->N <= 0 || d->Hkv <= 0 || d->H <= 0 || d->H % d->Hkv || d->block_size <= 0 || d->rows_per_req <= 0) return 0;
  if (prompt_applies(*d, varlen != 0)) return 16;  // the status word
  return rows_plan(*d, varlen != 0).bytes;
}

extern "C" int srswa_cache8_attend(const srswa_cache8_desc* d, const void* q, const void* k_cache,
                                   const void* v_cache, const float* k_scale, const float* v_scale,
                                   const int32_t* block_table, const int32_t* seq_lens, const int32_t* cu_rows,
                                   const int32_t* prefix_lens, const void* topk_idx, const float* bias, void* out,
                                   float* lse_out, void* workspace, size_t workspace_bytes, srswa_stream_t stream) {
  SRSWA_CHECK_ARG(d, SRSWA_EINVAL);
  const int rc = check_common(d, seq_lens, cu_rows, prefix_lens);
  if (rc) return rc;
  SRSWA_CHECK_ARG(d->H > 0 && d->H % d->Hkv == 0 && d->K >= 0 && d->sinks >= 0, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(d->q_dtype == SRSWA_BF16 || d->q_dtype == SRSWA_F16, SRSWA_EUNSUPPORTED);
  SRSWA_CHECK_ARG(d->out_dtype == d->q_dtype || d->out_dtype == SRSWA_F32, SRSWA_EUNSUPPORTED);
  SRSWA_CHECK_ARG(d->H <= 65535 && d->N < (1ll << 31), SRSWA_ETOOLARGE);
  if (d->N == 0) return SRSWA_OK;
  SRSWA_CHECK_ARG(q && k_cache && v_cache && k_scale && v_scale && block_table && out, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(d->K == 0 || topk_idx, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16), SRSWA_EALIGN);
  SRSWA_CHECK_ARG(((d->s_qn | d->s_qh | d->s_on | d->s_oh) & 7) == 0, SRSWA_EALIGN);
  Attend8Args a = {};
  a.q = q; a.k = static_cast<const uint8_t*>(k_cache); a.v = static_cast<const uint8_t*>(v_cache);
  a.ks = k_scale; a.vs = v_scale;
  a.rows = row_map(d, seq_lens, cu_rows, prefix_lens);
  a.table = block_table; a.sel = topk_idx; a.bias = bias; a.out = out; a.lse = lse_out;
  a.s_bt = d->s_bt; a.W = d->W; a.P = d->P; a.BS = d->block_size; a.N = d->N; a.H = d->H; a.Hkv = d->Hkv; a.D = d->D;
  a.K = d->K; a.window = d->window; a.sinks = d->sinks;
  a.s_qn = d->s_qn; a.s_qh = d->s_qh; a.s_on = d->s_on; a.s_oh = d->s_oh;
  a.s_page = d->s_page; a.s_pos = d->s_pos; a.s_head = d->s_head; a.s_scale = d->s_scale;
  a.s_ti_h = d->s_ti_h; a.s_ti_n = d->s_ti_n; a.s_b_h = d->s_b_h; a.s_b_n = d->s_b_n;
  a.scale_log2 = d->sm_scale * kLog2e;
  a.q_dtype = d->q_dtype; a.out_dtype = d->out_dtype; a.idx_is64 = d->idx_is64;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (prompt_applies(*d, cu_rows != nullptr)) {
    SRSWA_CHECK_ARG(workspace && workspace_bytes >= 16, SRSWA_EWORKSPACE);
    SRSWA_CHECK_ARG(aligned(workspace, 16), SRSWA_EALIGN);
    return prompt_launch(a, d->kv_dtype, static_cast<int*>(workspace), st);
  }
  const RowsPlan p = rows_plan(*d, cu_rows != nullptr);
  SRSWA_CHECK_ARG(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes), SRSWA_EWORKSPACE);
  SRSWA_CHECK_ARG(aligned(workspace, 16), SRSWA_EALIGN);
  return rows_launch(a, p, d->kv_dtype, workspace, st);
}
