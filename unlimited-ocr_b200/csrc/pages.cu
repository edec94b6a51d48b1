// Pages of a cache: free, extend, fork and compact over block tables with
// reference counts.
//
// Every choice of a page is by order (the lowest free page to the first item
// that needs one), so the tables do not depend on how the GPU schedules the
// work: one CTA plans (block-wide prefix sums over the items and the free
// pages), a second kernel applies the plan and moves the pages' data.

#include "cache8.cuh"

namespace srswa {

constexpr int kPlanThreads = 1024;
constexpr int kChunkBytes = 16384;  // page data moved by one CTA of the fork / compact kernels

struct PageTensors {
  int n;
  int chunks;  // chunks of one page over all tensors
  struct {
    char* base;
    int64_t bytes, stride;
    int first;  // index of its first chunk
    int align;  // 16, 4 or 1: the widest access that base, bytes and stride allow
  } t[SRSWA_MAX_PAGE_TENSORS];
};

// One chunk of page src to page dst, by the whole CTA (256 threads).
__device__ __forceinline__ void copy_chunk(const PageTensors& pt, int chunk, int64_t src, int64_t dst) {
  int i = 0;
  while (i + 1 < pt.n && pt.t[i + 1].first <= chunk) ++i;
  const int64_t off = static_cast<int64_t>(chunk - pt.t[i].first) * kChunkBytes;
  const int64_t n = min(pt.t[i].bytes - off, static_cast<int64_t>(kChunkBytes));
  const char* s = pt.t[i].base + src * pt.t[i].stride + off;
  char* d = pt.t[i].base + dst * pt.t[i].stride + off;
  if (pt.t[i].align == 16) {
    const uint4* s4 = reinterpret_cast<const uint4*>(s);
    uint4* d4 = reinterpret_cast<uint4*>(d);
    // all of a thread's loads before its first store
    constexpr int kEach = kChunkBytes / 16 / 256;
    const int n4 = static_cast<int>(n / 16);
    uint4 v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (static_cast<int>(threadIdx.x) + 256 * i < n4) v[i] = s4[threadIdx.x + 256 * i];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (static_cast<int>(threadIdx.x) + 256 * i < n4) d4[threadIdx.x + 256 * i] = v[i];
  } else if (pt.t[i].align == 4) {
    const uint32_t* s4 = reinterpret_cast<const uint32_t*>(s);
    uint32_t* d4 = reinterpret_cast<uint32_t*>(d);
    for (int64_t e = threadIdx.x; e < n / 4; e += blockDim.x) d4[e] = s4[e];
  } else {
    for (int64_t e = threadIdx.x; e < n; e += blockDim.x) d[e] = s[e];
  }
}

// Exclusive prefix sum over the CTA (kPlanThreads threads); total to all.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& total) {
  __shared__ int64_t part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) part[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t y = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    part[lane] = y;
  }
  __syncthreads();
  const int64_t before = warp ? part[warp - 1] : 0;
  total = part[31];
  __syncthreads();
  return before + x - v;
}

__global__ void __launch_bounds__(256) pages_free_kernel(const int32_t* rows, int32_t* table, int64_t s_bt,
                                                         int64_t R, int64_t W, int32_t* seq_lens, int32_t* refs,
                                                         int64_t P, int64_t BS) {
  __shared__ int len;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = rows[blockIdx.x];
  if (row < 0 || row >= R) return;
  // a row named twice: whoever takes its length first does the work
  if (threadIdx.x == 0) len = atomicExch(&seq_lens[row], 0);
  __syncthreads();
  const int64_t n = min((static_cast<int64_t>(len) + BS - 1) / BS, W);
  for (int64_t b = threadIdx.x; b < n; b += blockDim.x) {
    const int64_t page = table[row * s_bt + b];
    table[row * s_bt + b] = -1;
    if (page >= 0 && page < P) atomicSub(&refs[page], 1);
  }
}

// One item as the apply kernels take it: everything they need in one read.
struct __align__(16) PlanItem {
  int32_t made, row, len, have;     // carried out; row that changes; its new length; pages it has
  int32_t first, parent, src, dst;  // rank of its first free page; fork: parent row, part-filled page, its copy (-1)
};

struct PlanArgs {
  const int32_t* rows;     // fork: children; extend: rows
  const int32_t* parents;  // fork
  const int32_t* lens;     // extend: new lengths
  int64_t n;
  int32_t* table;
  int64_t s_bt, R, W, P, BS;
  int32_t* seq_lens;
  int32_t* refs;
  int32_t* short_out;
  // workspace
  PlanItem* items;  // [n]
  int32_t* claim;   // [R] the first item that names a row (kept on chip for up to kClaimRows rows)
  int32_t* pages;   // [P] free pages, lowest first
};
constexpr int kClaimRows = 8192;

__device__ __forceinline__ int64_t pages_for(int64_t tokens, int64_t BS) { return (tokens + BS - 1) / BS; }

// Whether item i would be carried out, apart from repeats; its row, the new pages
// it needs, the new length, and the pages that the row has.
__device__ __forceinline__ bool plan_item(const PlanArgs& a, int64_t i, int64_t& row, int64_t& need, int64_t& len,
                                          int64_t& have) {
  row = a.rows[i];
  const int64_t par = a.parents ? a.parents[i] : 0;
  const int64_t want = a.lens ? a.lens[i] : 0;
  if (row < 0 || row >= a.R || par < 0 || par >= a.R) return false;
  const int64_t now = a.seq_lens[row];
  len = a.parents ? a.seq_lens[par] : want;
  have = pages_for(now, a.BS);
  if (now < 0 || pages_for(len, a.BS) > a.W) return false;
  if (a.parents) {
    need = len % a.BS ? 1 : 0;
    return now == 0 && len > 0;
  }
  need = pages_for(len, a.BS) - have;
  return len >= now;
}

__global__ void __launch_bounds__(kPlanThreads) pages_plan_kernel(const PlanArgs a) {
  __shared__ int32_t near_claim[kClaimRows];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  int32_t* claim = a.R <= kClaimRows ? near_claim : a.claim;
  // more items than threads: they are looked at again in each pass
  int64_t row = 0, need = 0, len = 0, have = 0;
  bool ok = false;
  const bool once = a.n <= kPlanThreads;
  auto look = [&](int64_t i) { ok = i < a.n && plan_item(a, i, row, need, len, have); };
  for (int64_t i = tid; i < a.n; i += kPlanThreads) {
    look(i);
    if (ok) claim[row] = 0x7fffffff;
  }
  __syncthreads();
  for (int64_t i = tid; i < a.n; i += kPlanThreads) {
    if (!once) look(i);
    if (ok) atomicMin(&claim[row], static_cast<int>(i));
  }
  __syncthreads();
  int64_t all = 0;  // pages the items need together
  for (int64_t i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int64_t i = i0 + tid;
    if (!once) look(i);
    const bool mine = ok && claim[row] == i;
    int64_t sum;
    const int64_t at = all + block_scan(mine ? need : 0, sum);
    if (i < a.n) {
      PlanItem x = {mine ? 1 : 0, static_cast<int32_t>(row), static_cast<int32_t>(len), static_cast<int32_t>(have),
                    static_cast<int32_t>(min(at, static_cast<int64_t>(0x7ffffffe))), 0, -1, -1};
      if (mine && a.parents) {
        x.parent = a.parents[i];
        if (need) x.src = a.table[x.parent * a.s_bt + len / a.BS];
      }
      a.items[i] = x;
    }
    all += sum;
  }
  // the lowest free pages, as many as are needed
  int64_t found = 0;
  for (int64_t p0 = 0; p0 < a.P && found < all; p0 += kPlanThreads) {
    const int64_t p = p0 + tid;
    int64_t sum;
    const bool free = p < a.P && a.refs[p] == 0;
    const int64_t at = found + block_scan(free, sum);
    if (free && at < all) a.pages[at] = static_cast<int32_t>(p);
    found += sum;
  }
  __syncthreads();
  int64_t miss = 0;
  for (int64_t i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int64_t i = i0 + tid;
    bool none = false;
    if (i < a.n) {
      PlanItem x = a.items[i];
      if (x.made) {
        const int64_t needs = a.parents ? (x.len % a.BS ? 1 : 0) : pages_for(x.len, a.BS) - x.have;
        none = needs > 0 && x.first + needs > found;
        if (none) a.items[i].made = 0;
        else if (a.parents && needs) a.items[i].dst = a.pages[x.first];
      }
    }
    miss += __syncthreads_count(none);
  }
  if (tid == 0) *a.short_out = static_cast<int32_t>(miss);
}

__global__ void __launch_bounds__(256) pages_extend_kernel(const PlanArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const PlanItem x = a.items[blockIdx.x];
  if (!x.made) return;
  const int64_t want = pages_for(x.len, a.BS);
  for (int64_t b = x.have + threadIdx.x; b < want; b += blockDim.x) {
    const int64_t page = a.pages[x.first + b - x.have];
    a.table[x.row * a.s_bt + b] = static_cast<int32_t>(page);
    a.refs[page] = 1;
  }
  if (threadIdx.x == 0) a.seq_lens[x.row] = x.len;
}

// grid (1 + chunks of a page, items): part 0 makes the child's row, the others
// copy the part-filled page.
__global__ void __launch_bounds__(256) pages_fork_kernel(const PlanArgs a, const PageTensors pt) {
  pdl_launch_dependents();
  pdl_wait();
  const PlanItem x = a.items[blockIdx.y];
  if (!x.made) return;
  if (blockIdx.x > 0) {
    if (x.dst >= 0 && x.src >= 0 && x.src < a.P) copy_chunk(pt, blockIdx.x - 1, x.src, x.dst);
    return;
  }
  const int64_t full = x.len / a.BS;
  const int32_t* from = a.table + x.parent * a.s_bt;  // (a parent is never a child of the same call: it holds tokens)
  int32_t* to = a.table + x.row * a.s_bt;
  for (int64_t b = threadIdx.x; b < full; b += blockDim.x) {
    const int32_t p = from[b];
    to[b] = p;
    if (p >= 0 && p < a.P) atomicAdd(&a.refs[p], 1);
  }
  if (threadIdx.x == 0) {
    if (x.dst >= 0) {
      to[full] = x.dst;
      a.refs[x.dst] = 1;
    }
    a.seq_lens[x.row] = x.len;
  }
}

struct CompactArgs {
  const int32_t* table;
  const int32_t* refs;
  int32_t* out_table;
  int32_t* out_refs;
  int32_t* live_out;
  int64_t s_bt, s_out, R, W, P;
  // workspace
  int32_t* moves;  // [1] pages that move
  int32_t* src;    // [P]
  int32_t* dst;    // [P]
  int32_t* to;     // [P] where a page is afterwards
};

__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const CompactArgs a) {
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  // a thread's pages are neighbours, so two prefix sums do for any number of pages
  const int64_t per = (a.P + kPlanThreads - 1) / kPlanThreads, lo = min(tid * per, a.P), hi = min(lo + per, a.P);
  int64_t mine = 0, live, sum;
  for (int64_t p = lo; p < hi; ++p) mine += a.refs[p] > 0;
  block_scan(mine, live);
  // pages in use at or past `live` (low half), free ones below it (high half)
  const int64_t used_past = hi <= live ? 0 : lo >= live ? mine : -1, below = min(max(live - lo, static_cast<int64_t>(0)), hi - lo);
  int64_t ns = used_past, nd;
  if (ns < 0) {
    ns = 0;
    for (int64_t p = live; p < hi; ++p) ns += a.refs[p] > 0;
  }
  nd = below - (mine - ns);
  int64_t at = block_scan(ns | (nd << 32), sum);
  int32_t *src = a.src + (at & 0xffffffff), *dst = a.dst + (at >> 32);
  for (int64_t p = lo; p < hi; ++p) {
    const bool used = a.refs[p] > 0;
    if (used && p >= live) *src++ = static_cast<int32_t>(p);
    if (!used && p < live) *dst++ = static_cast<int32_t>(p);
    a.to[p] = static_cast<int32_t>(p);
  }
  ns = sum & 0xffffffff;
  __syncthreads();
  if (a.out_refs != a.refs) {
    for (int64_t p = tid; p < a.P; p += kPlanThreads) a.out_refs[p] = a.refs[p];
    __syncthreads();
  }
  for (int64_t i = tid; i < ns; i += kPlanThreads) {
    const int32_t s = a.src[i], d = a.dst[i];
    a.to[s] = d;
    a.out_refs[d] = a.refs[s];
    a.out_refs[s] = 0;
  }
  if (tid == 0) {
    *a.moves = static_cast<int32_t>(ns);
    *a.live_out = static_cast<int32_t>(live);
  }
}

__global__ void __launch_bounds__(256) pages_compact_kernel(const CompactArgs a, const PageTensors pt) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t work = static_cast<int64_t>(*a.moves) * pt.chunks;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int64_t i = w / pt.chunks;
    copy_chunk(pt, static_cast<int>(w % pt.chunks), a.src[i], a.dst[i]);
  }
  const int64_t entries = a.R * a.W;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < entries;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = e / a.W, b = e % a.W;
    const int32_t p = a.table[r * a.s_bt + b];
    a.out_table[r * a.s_out + b] = p >= 0 && p < a.P ? a.to[p] : p;
  }
}

}  // namespace srswa

using namespace srswa;

static int page_tensors(const srswa_page_tensor* t, int64_t n, PageTensors& out) {
  SRSWA_CHECK_ARG(n >= 0 && (n == 0 || t), SRSWA_EINVAL);
  SRSWA_CHECK_ARG(n <= SRSWA_MAX_PAGE_TENSORS, SRSWA_ETOOLARGE);
  out.n = static_cast<int>(n);
  int64_t chunks = 0;
  for (int64_t i = 0; i < n; ++i) {
    SRSWA_CHECK_ARG(t[i].base && t[i].page_bytes > 0 && t[i].stride_bytes >= t[i].page_bytes, SRSWA_EINVAL);
    const int64_t bits = reinterpret_cast<intptr_t>(t[i].base) | t[i].page_bytes | t[i].stride_bytes;
    out.t[i].base = static_cast<char*>(t[i].base);
    out.t[i].bytes = t[i].page_bytes;
    out.t[i].stride = t[i].stride_bytes;
    out.t[i].first = static_cast<int>(chunks);
    out.t[i].align = (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1;
    chunks += (t[i].page_bytes + kChunkBytes - 1) / kChunkBytes;
    SRSWA_CHECK_ARG(chunks < (1 << 24), SRSWA_ETOOLARGE);
  }
  out.chunks = static_cast<int>(chunks);
  return SRSWA_OK;
}

static int check_pool(const int32_t* table, int64_t s_bt, int64_t R, int64_t W, const int32_t* refs, int64_t P) {
  SRSWA_CHECK_ARG(table && refs && R > 0 && W > 0 && P > 0 && s_bt >= W, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(P < (1ll << 31) && R < (1ll << 31), SRSWA_ETOOLARGE);
  return SRSWA_OK;
}

extern "C" size_t srswa_pages_workspace_size(int64_t n, int64_t R, int64_t P) {
  return static_cast<size_t>(n > 0 ? n : 0) * sizeof(PlanItem) + static_cast<size_t>((R > 0 ? R : 0) + (P > 0 ? P : 0)) * 4;
}

static int make_plan(PlanArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  SRSWA_CHECK_ARG(workspace && workspace_bytes >= srswa_pages_workspace_size(a.n, a.R, a.P), SRSWA_EWORKSPACE);
  SRSWA_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, SRSWA_EALIGN);
  a.items = static_cast<PlanItem*>(workspace);
  a.claim = reinterpret_cast<int32_t*>(a.items + a.n);
  a.pages = a.claim + a.R;
  return launch_pdl(pages_plan_kernel, dim3(1), kPlanThreads, 0, st, a);
}

extern "C" int srswa_pages_free(const int32_t* rows, int64_t n, int32_t* block_table, int64_t s_bt, int64_t R,
                                int64_t W, int32_t* seq_lens, int32_t* refs, int64_t P, int64_t block_size,
                                srswa_stream_t stream) {
  const int rc = check_pool(block_table, s_bt, R, W, refs, P);
  if (rc) return rc;
  SRSWA_CHECK_ARG(n >= 0 && block_size > 0 && seq_lens && (n == 0 || rows), SRSWA_EINVAL);
  SRSWA_CHECK_ARG(n < (1ll << 31) && block_size < (1ll << 31), SRSWA_ETOOLARGE);
  if (n == 0) return SRSWA_OK;
  return launch_pdl(pages_free_kernel, dim3(static_cast<unsigned>(n)), 256, 0, reinterpret_cast<cudaStream_t>(stream),
                    rows, block_table, s_bt, R, W, seq_lens, refs, P, block_size);
}

extern "C" int srswa_pages_extend(const int32_t* rows, const int32_t* new_lens, int64_t n, int32_t* block_table,
                                  int64_t s_bt, int64_t R, int64_t W, int32_t* seq_lens, int32_t* refs, int64_t P,
                                  int64_t block_size, int32_t* short_out, void* workspace, size_t workspace_bytes,
                                  srswa_stream_t stream) {
  int rc = check_pool(block_table, s_bt, R, W, refs, P);
  if (rc) return rc;
  SRSWA_CHECK_ARG(n >= 0 && block_size > 0 && seq_lens && short_out && (n == 0 || (rows && new_lens)), SRSWA_EINVAL);
  SRSWA_CHECK_ARG(n <= 65535 && block_size < (1ll << 31), SRSWA_ETOOLARGE);
  PlanArgs a = {rows, nullptr, new_lens, n, block_table, s_bt, R, W, P, block_size, seq_lens, refs, short_out};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = make_plan(a, workspace, workspace_bytes, st);
  if (rc || n == 0) return rc;
  return launch_pdl(pages_extend_kernel, dim3(static_cast<unsigned>(n)), 256, 0, st, a);
}

extern "C" int srswa_pages_fork(const int32_t* parents, const int32_t* children, int64_t n, int32_t* block_table,
                                int64_t s_bt, int64_t R, int64_t W, int32_t* seq_lens, int32_t* refs, int64_t P,
                                int64_t block_size, const srswa_page_tensor* tensors, int64_t ntensors,
                                int32_t* short_out, void* workspace, size_t workspace_bytes, srswa_stream_t stream) {
  int rc = check_pool(block_table, s_bt, R, W, refs, P);
  if (rc) return rc;
  SRSWA_CHECK_ARG(n >= 0 && block_size > 0 && seq_lens && short_out && (n == 0 || (parents && children)), SRSWA_EINVAL);
  SRSWA_CHECK_ARG(n <= 65535 && block_size < (1ll << 31), SRSWA_ETOOLARGE);
  PageTensors pt = {};
  rc = page_tensors(tensors, ntensors, pt);
  if (rc) return rc;
  PlanArgs a = {children, parents, nullptr, n, block_table, s_bt, R, W, P, block_size, seq_lens, refs, short_out};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = make_plan(a, workspace, workspace_bytes, st);
  if (rc || n == 0) return rc;
  return launch_pdl(pages_fork_kernel, dim3(static_cast<unsigned>(1 + pt.chunks), static_cast<unsigned>(n)), 256, 0, st,
                    a, pt);
}

extern "C" size_t srswa_pages_compact_workspace_size(int64_t P) {
  return static_cast<size_t>(3 * (P > 0 ? P : 0) + 1) * 4;
}

extern "C" int srswa_pages_compact(const int32_t* block_table, int64_t s_bt, int64_t R, int64_t W,
                                   const int32_t* refs, int64_t P, const srswa_page_tensor* tensors,
                                   int64_t ntensors, int32_t* out_table, int64_t s_out, int32_t* out_refs,
                                   int32_t* live_out, void* workspace, size_t workspace_bytes,
                                   srswa_stream_t stream) {
  int rc = check_pool(block_table, s_bt, R, W, refs, P);
  if (rc) return rc;
  SRSWA_CHECK_ARG(out_table && out_refs && live_out && s_out >= W, SRSWA_EINVAL);
  SRSWA_CHECK_ARG(workspace && workspace_bytes >= srswa_pages_compact_workspace_size(P), SRSWA_EWORKSPACE);
  SRSWA_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 3) == 0, SRSWA_EALIGN);
  PageTensors pt = {};
  rc = page_tensors(tensors, ntensors, pt);
  if (rc) return rc;
  CompactArgs a = {block_table, refs, out_table, out_refs, live_out, s_bt, s_out, R, W, P};
  a.moves = static_cast<int32_t*>(workspace);
  a.src = a.moves + 1;
  a.dst = a.src + P;
  a.to = a.dst + P;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = launch_pdl(pages_compact_plan_kernel, dim3(1), kPlanThreads, 0, st, a);
  if (rc) return rc;
  return launch_pdl(pages_compact_kernel, dim3(148 * 8), 256, 0, st, a, pt);
}
