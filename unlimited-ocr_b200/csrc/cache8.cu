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

// Two elements -> two codes (the first in the low byte).
template <int KVT>
__device__ __forceinline__ uint32_t to_code2(float x, float y) {
  if (KVT == SRSWA_I8) {
    const int a = x != x ? 0 : __float2int_rn(fminf(fmaxf(x, -127.f), 127.f));
    const int b = y != y ? 0 : __float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
    return (static_cast<uint32_t>(a) & 0xffu) | ((static_cast<uint32_t>(b) & 0xffu) << 8);
  }
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}

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

// 1 / s of a power of two is exact, and so is x times it; another writer's scale
// is divided by.
struct Scaler {
  float s, inv;
  bool pow2;
  __device__ __forceinline__ explicit Scaler(float scale) : s(scale), inv(1.f / scale) {
    const uint32_t u = __float_as_uint(scale);
    pow2 = (u & 0x7fffffu) == 0 && u >= 0x00800000u && u < 0x7f000000u;
  }
  template <int KVT>
  __device__ __forceinline__ uint8_t code(float x) const { return to_code<KVT>(pow2 ? x * inv : x / s); }
};

__device__ __forceinline__ float finite_abs(float x) {
  const float v = fabsf(x);
  return v <= 3.402823466e38f ? v : 0.f;
}

// Earlier tokens [0, held) of a page, rounded from scale `old` to `s`: thread
// `i` of `n`, 8 codes at a time.
template <int D, int KVT>
__device__ __forceinline__ void regrow(uint8_t* tile, int64_t s_pos, int held, float old, float s, int i, int n) {
  const float r = old / s;
  for (int w = i; w < held * (D / 8); w += n) {
    uint2* c = reinterpret_cast<uint2*>(tile + (w / (D / 8)) * s_pos + (w % (D / 8)) * 8);
    uint2 x = *c;
    uint8_t* b = reinterpret_cast<uint8_t*>(&x);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = to_code<KVT>(code_to_float(b[e], KVT) * r);
    *c = x;
  }
}

// One CTA per (page a request's new tokens touch, head, K or V).  Bound by
// memory: the new elements of a page stay in registers between the maximum and
// the rounding (pages of up to 8 passes of the CTA; longer ones are read twice,
// the second time from L2), so each is read once and its code written once.
// 132 MB of bf16 and e4m3 (nine ragged prompts of up to 7001 tokens, 10 heads of
// 128): 29 us, 71 % of the copy rate; with 5 / 8 / 10 CTAs an SM for six 33 / 35 / 39.
template <int D, int KVT>
__global__ void __launch_bounds__(kAppendThreads, 6) cache8_append_kernel(const AppendArgs a) {
  constexpr int LPT = D / 8;                     // lanes per token, 8 elements each
  constexpr int TPP = kAppendThreads / LPT;      // tokens per pass
  constexpr int NP = 8;                          // passes held in registers
  __shared__ float red[kAppendThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const int64_t head = blockIdx.y;
  const int which = blockIdx.z;

  // the slot's request and page: request r has at most (n + BS - 2) / BS + 1
  // touched pages, so its slots begin at cu[r] / BS + 2 r (varlen)
  int64_t req, start, n, row0, nth;
  if (a.rows.cu) {
    const int64_t i = blockIdx.x;
    int64_t before = 0;  // requests that begin at or before this slot
    for (int64_t r0 = 0; r0 < a.rows.R; r0 += kAppendThreads) {
      const int64_t r = r0 + tid;
      const int here = __syncthreads_count(r < a.rows.R && a.rows.cu[r] / a.BS + 2 * r <= i);
      before += here;
      if (here < kAppendThreads) break;
    }
    if (before == 0) return;  // rows ahead of the first request's
    req = before - 1;
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
    if (start < 0) {  // a request shorter than its rows: the first of them have no position
      row0 -= start;
      n += start;
      start = 0;
    }
  }
  if (n <= 0 || start < 0 || row0 < 0 || row0 + n > a.N) return;
  const int64_t blk = start / a.BS + nth;
  const int64_t lo = max(start, blk * a.BS), hi = min(start + n, (blk + 1) * a.BS);  // positions written here
  if (lo >= hi || blk >= a.W) return;
  const int count = static_cast<int>(hi - lo), held = static_cast<int>(lo - blk * a.BS);  // new, earlier tokens

  const void* x = a.x[which];
  const int g = tid / LPT, u = tid % LPT;
  const int64_t x0 = (row0 + lo - start) * a.s_xn[which] + head * a.s_xh[which] + u * 8;
  const int64_t s_xn = a.s_xn[which];
  const bool fits = count <= NP * TPP && a.x_dtype != SRSWA_F32;  // uniform
  uint4 raw[NP];
  float amax = 0.f;
  if (fits) {
#pragma unroll
    for (int j = 0; j < NP; ++j)
      raw[j] = j * TPP + g < count ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + x0 + (j * TPP + g) * s_xn))
                                   : make_uint4(0, 0, 0, 0);
  }
  const int64_t page = a.table[req * a.s_bt + blk];
  if (page < 0 || page >= a.P) return;
  uint8_t* dst = a.cache[which] + page * a.s_page + head * a.s_head;
  float* scale = a.scale[which] + page * a.s_scale + head;
  const float old = held > 0 ? *scale : 0.f;

  auto unpack = [&](uint32_t w) {
    if (a.x_dtype == SRSWA_BF16) return make_float2(bf16_lo(w), bf16_hi(w));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  };
  float f[8];
  if (fits) {
    // the largest magnitude in the elements' own type, two at a time (its maximum
    // skips NaN); an infinity among them is rare and sends us over them again
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t v = w[e] & 0x7fff7fffu;
        if (a.x_dtype == SRSWA_BF16) {
          const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&top),
                                           *reinterpret_cast<const __nv_bfloat162*>(&v));
          top = *reinterpret_cast<const uint32_t*>(&r);
        } else {
          const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&top), *reinterpret_cast<const __half2*>(&v));
          top = *reinterpret_cast<const uint32_t*>(&r);
        }
      }
    }
    const float2 t2 = unpack(top);
    amax = fmaxf(t2.x, t2.y);
    if (!(amax <= 3.402823466e38f)) {
      amax = 0.f;
#pragma unroll 1
      for (int t = g; t < count; t += TPP) {
        load8(x, x0 + t * s_xn, a.x_dtype, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(f[e]));
      }
    }
  } else {
    for (int t = g; t < count; t += TPP) {
      load8(x, x0 + t * s_xn, a.x_dtype, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(f[e]));
    }
  }
  amax = warp_max(amax);
  if ((tid & 31) == 0) red[tid >> 5] = amax;
  __syncthreads();  // and every thread has read the old scale
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) amax = fmaxf(amax, red[w]);

  float s = pow2_scale<KVT>(amax);
  if (held > 0) {
    if (s > old) regrow<D, KVT>(dst, a.s_pos, held, old, s, tid, kAppendThreads);
    else s = old;
  }
  if (tid == 0) *scale = s;
  const Scaler sc(s);
  uint8_t* out = dst + held * a.s_pos + u * 8;
  if (fits && sc.pow2) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
      uint32_t c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = unpack(w[e]);
        c[e] = to_code2<KVT>(v.x * sc.inv, v.y * sc.inv);
      }
      if (j * TPP + g < count)
        *reinterpret_cast<uint2*>(out + (j * TPP + g) * a.s_pos) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
    }
  } else {
#pragma unroll 1
    for (int t = g; t < count; t += TPP) {
      load8(x, x0 + t * s_xn, a.x_dtype, f);
      uint2 w;
      uint8_t* b = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = sc.code<KVT>(f[e]);
      *reinterpret_cast<uint2*>(out + t * a.s_pos) = w;
    }
  }
}

// One new token per request (decode): one warp per (request, head, K or V), a
// lane holds D / 32 features.  Bound by the latency of its dependent reads (length,
// page, scale; the elements come beside them): 256 requests of 10 heads 4.6 us a
// call, 12.2 with the kernel above.
template <int D, int KVT>
__global__ void __launch_bounds__(kAppendThreads) cache8_append_one_kernel(const AppendArgs a) {
  constexpr int E = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int which = static_cast<int>(item % 2);
  const int64_t head = item / 2 % a.Hkv, req = item / 2 / a.Hkv;
  if (req >= a.rows.R) return;
  const int64_t pos = static_cast<int64_t>(a.rows.seq_lens[req]) - 1;
  float f[E], amax = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    f[e] = load_elem(a.x[which], req * a.s_xn[which] + head * a.s_xh[which] + lane * E + e, a.x_dtype);
    amax = fmaxf(amax, finite_abs(f[e]));
  }
  if (pos < 0 || pos >= a.W * a.BS) return;
  const int64_t blk = pos / a.BS, page = a.table[req * a.s_bt + blk];
  if (page < 0 || page >= a.P) return;
  const int held = static_cast<int>(pos - blk * a.BS);
  uint8_t* dst = a.cache[which] + page * a.s_page + head * a.s_head;
  float* scale = a.scale[which] + page * a.s_scale + head;
  float s = pow2_scale<KVT>(warp_max(amax));
  if (held > 0) {
    const float old = *scale;
    if (s > old) regrow<D, KVT>(dst, a.s_pos, held, old, s, lane, 32);
    else s = old;
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale = s;
  const Scaler sc(s);
  uint8_t b[E];
#pragma unroll
  for (int e = 0; e < E; ++e) b[e] = sc.code<KVT>(f[e]);
  uint8_t* p = dst + held * a.s_pos + lane * E;
  if constexpr (E == 4) *reinterpret_cast<uchar4*>(p) = make_uchar4(b[0], b[1], b[2], b[3]);
  else *reinterpret_cast<uchar2*>(p) = make_uchar2(b[0], b[1]);
}

template <int D, int KVT>
static int append_start(const AppendArgs& a, int64_t slots, cudaStream_t st) {
  if (!a.rows.cu && a.rows.rps == 1) {
    const int64_t ctas = (2 * a.rows.R * a.Hkv + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
    return launch_pdl(cache8_append_one_kernel<D, KVT>, dim3(static_cast<unsigned>(ctas)), kAppendThreads, 0, st, a);
  }
  const dim3 grid(static_cast<unsigned>(slots), static_cast<unsigned>(a.Hkv), 2);
  return launch_pdl(cache8_append_kernel<D, KVT>, grid, kAppendThreads, 0, st, a);
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
  SRSWA_CHECK_ARG(d->block_size <= 1024 && d->Hkv <= 65535 && d->W < (1ll << 31) && d->P < (1ll << 31), SRSWA_ETOOLARGE);
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

// A pool of no pages and a table of no blocks have no addresses.
static bool there(const srswa_cache8_desc* d, const void* k, const void* v, const void* ks, const void* vs,
                  const void* table) {
  return (d->P == 0 || (k && v && ks && vs)) && (d->W == 0 || table);
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
  SRSWA_CHECK_ARG(k && v && there(d, k_cache, v_cache, k_scale, v_scale, block_table), SRSWA_EINVAL);
  SRSWA_CHECK_ARG(aligned(k, 16) && aligned(v, 16) && aligned(k_cache, 16) && aligned(v_cache, 16), SRSWA_EALIGN);
  const int64_t m = d->q_dtype == SRSWA_F32 ? 3 : 7;
  SRSWA_CHECK_ARG(((d->s_qn | d->s_qh | d->s_on | d->s_oh) & m) == 0, SRSWA_EALIGN);
  const int64_t slots = cu_rows ? d->N / d->block_size + 2 * d->R
                                : d->R * ((d->rows_per_req + d->block_size - 2) / d->block_size + 1);
  SRSWA_CHECK_ARG(slots < (1ll << 31) && d->R * d->Hkv < (1ll << 31), SRSWA_ETOOLARGE);
  AppendArgs a = {};
  a.x[0] = k; a.x[1] = v;
  a.cache[0] = static_cast<uint8_t*>(k_cache); a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale; a.scale[1] = v_scale;
  a.s_xn[0] = d->s_qn; a.s_xh[0] = d->s_qh; a.s_xn[1] = d->s_on; a.s_xh[1] = d->s_oh;
  a.rows = row_map(d, seq_lens, cu_rows, prefix_lens);
  a.table = block_table; a.s_bt = d->s_bt; a.W = d->W; a.P = d->P; a.BS = d->block_size; a.N = d->N; a.Hkv = d->Hkv;
  a.s_page = d->s_page; a.s_pos = d->s_pos; a.s_head = d->s_head; a.s_scale = d->s_scale;
  a.x_dtype = d->q_dtype;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (d->D == 128)
    return d->kv_dtype == SRSWA_I8 ? append_start<128, SRSWA_I8>(a, slots, st) : append_start<128, SRSWA_F8E4M3>(a, slots, st);
  return d->kv_dtype == SRSWA_I8 ? append_start<64, SRSWA_I8>(a, slots, st) : append_start<64, SRSWA_F8E4M3>(a, slots, st);
}

// Positions are 32-bit: a window or sinks past them are all there is.
static srswa_cache8_desc within_positions(const srswa_cache8_desc* d) {
  constexpr int64_t all = 0x7ffffe00;
  srswa_cache8_desc c = *d;
  if (c.window > all) c.window = all;
  if (c.sinks > all) c.sinks = all;
  return c;
}

extern "C" size_t srswa_cache8_attend_workspace_size(const srswa_cache8_desc* desc, int varlen) {
  if (!desc) return 0;
  const srswa_cache8_desc bounded = within_positions(desc), *d = &bounded;
  if (d->N <= 0 || d->Hkv <= 0 || d->H <= 0 || d->H % d->Hkv || d->block_size <= 0) return 0;
  if (!varlen && d->rows_per_req <= 0) return 0;
  if (prompt_applies(*d, varlen != 0)) return 16;  // the status word
  return rows_plan(*d, varlen != 0).bytes;
}

extern "C" int srswa_cache8_attend(const srswa_cache8_desc* desc, const void* q, const void* k_cache,
                                   const void* v_cache, const float* k_scale, const float* v_scale,
                                   const int32_t* block_table, const int32_t* seq_lens, const int32_t* cu_rows,
                                   const int32_t* prefix_lens, const void* topk_idx, const float* bias, void* out,
                                   float* lse_out, void* workspace, size_t workspace_bytes, srswa_stream_t stream) {
  SRSWA_CHECK_ARG(desc, SRSWA_EINVAL);
  const srswa_cache8_desc bounded = within_positions(desc), *d = &bounded;
  const int rc = check_common(d, seq_lens, cu_rows, prefix_lens);
  if (rc) return rc;
  SRSWA_CHECK_ARG(d->H > 0 && d->H % d->Hkv == 0 && d->K >= 0 && d->sinks >= 0, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(d->q_dtype == SRSWA_BF16 || d->q_dtype == SRSWA_F16, SRSWA_EUNSUPPORTED);
  SRSWA_CHECK_ARG(d->out_dtype == d->q_dtype || d->out_dtype == SRSWA_F32, SRSWA_EUNSUPPORTED);
  SRSWA_CHECK_ARG(d->H <= 65535 && d->N < (1ll << 31) && d->K <= kMaxSelected, SRSWA_ETOOLARGE);
  if (d->N == 0) return SRSWA_OK;
  SRSWA_CHECK_ARG(q && there(d, k_cache, v_cache, k_scale, v_scale, block_table) && out, SRSWA_EINVAL);
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
