// Pages of the key/value cache: reserve, fork, copy, free, compact.
//
// The page tables, lengths and reference counts are device arrays, and every
// decision is made on the device, so a captured decode step can let its
// sequences grow over a page's end, and no call waits for the host.  A page with
// reference count 0 is free; pages are handed out lowest id first, to the
// requests in list order, so the state after a call is a function of the
// state before it.
//
// One block makes the plan (it needs global order: prefix sums over the requests
// and over the free pages; 16 reference counts a thread and step, and the scan stops at the last page
// that is needed), then a grid moves page contents.  Contents are what costs:
// 2 x the moved bytes (204 pages of 1 MB: 70 us, 6.1 TB/s; a reservation for 48 rows takes 4 us, a fork's plan 10 us).
#include <algorithm>

#include "attn_common.cuh"

namespace klc {
namespace attn {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = kCopyThreads * 16 * 4;  // per block and step

// workspace of a plan, all int32
struct KvWork {
  int* count;  // [1] page moves (+ 3 spare words)
  int* ids;    // [pages] free pages found
  int* src;    // [pages] moves
  int* dst;    // [pages]
  int* to;     // [pages] new id of a page (compact)
  int* first;  // [rows] first listed child of a row
  int* need;   // [rows] pages a request needs; -1: refused
};

struct KvParams {
  klc_kv_cache c;
  KvWork w;
  DeviceStatus* status;
};

// exclusive prefix sum over the block; *total gets the sum
__device__ int block_scan(int v, int* total) {
  __shared__ int sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const int s = sums[lane];
    int t = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    sums[lane] = t;
  }
  __syncthreads();
  const int base = warp > 0 ? sums[warp - 1] : 0;
  *total = sums[31];
  __syncthreads();
  return base + incl - v;
}

// 16 reference counts of pages from..from+15 (pages past the end read as taken)
__device__ __forceinline__ void load_refs(const KvParams& p, int64_t from, int (&r)[16]) {
  const bool whole = from + 16 <= p.c.pages;
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    if (whole) {
      const int4 v = *reinterpret_cast<const int4*>(p.c.refs + from + j);
      r[j] = v.x;
      r[j + 1] = v.y;
      r[j + 2] = v.z;
      r[j + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[j + e] = from + j + e < p.c.pages ? p.c.refs[from + j + e] : 1;
    }
  }
}

// the lowest `want` free page ids into ids, ascending; returns how many there are (at most want)
__device__ int collect_free(const KvParams& p, int want) {
  int found = 0;
  for (int64_t base = 0; base < p.c.pages && found < want; base += kPlanThreads * 16) {
    const int64_t from = base + threadIdx.x * 16;
    int r[16], n = 0, total;
    if (from < p.c.pages) {
      load_refs(p, from, r);
#pragma unroll
      for (int j = 0; j < 16; ++j) n += r[j] <= 0;
    }
    int at = found + block_scan(n, &total);
    if (n > 0) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (r[j] <= 0) {
          if (at < want) p.w.ids[at] = int(from + j);
          ++at;
        }
    }
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

__device__ __forceinline__ int pages_of(int len, int ps) { return (len + ps - 1) / ps; }

__device__ __forceinline__ bool len_ok(const KvParams& p, int len) {
  return len >= 0 && int64_t(len) <= p.c.table_width * p.c.page_size;
}

// New pages for rows that grow by add[row] keys.
__global__ void __launch_bounds__(kPlanThreads) kv_reserve_kernel(const KvParams p, const int32_t* add) {
  pdl_trigger();
  pdl_wait();
  const int ps = p.c.page_size;
  int demand = 0;
  for (int64_t base = 0; base < p.c.rows; base += kPlanThreads) {
    const int64_t r = base + threadIdx.x;
    int need = 0;
    if (r < p.c.rows) {
      const int len = p.c.lens[r], a = add[r];
      if (!len_ok(p, len) || a < 0 || int64_t(len) + a > p.c.table_width * ps) {
        record_fault(p.status, KLC_ERR_DEVICE_FAULT, 530, int(r));
        p.w.need[r] = -1;
      } else {
        need = pages_of(len + a, ps) - pages_of(len, ps);
        p.w.need[r] = need;
      }
    }
    int total;
    block_scan(need, &total);
    demand += total;
  }
  const int have = demand > 0 ? collect_free(p, demand) : 0;
  int at = 0;
  for (int64_t base = 0; base < p.c.rows; base += kPlanThreads) {
    const int64_t r = base + threadIdx.x;
    const int need = r < p.c.rows ? p.w.need[r] : 0;
    int total;
    const int mine = at + block_scan(max(need, 0), &total);
    at += total;
    if (r >= p.c.rows || need < 0) continue;
    if (need > 0 && mine + need > have) {
      record_fault(p.status, KLC_ERR_DEVICE_FAULT, 531, int(r));  // out of pages: the row stays as it is
      continue;
    }
    const int len = p.c.lens[r], slot = pages_of(len, ps);
    for (int j = 0; j < need; ++j) {
      const int page = p.w.ids[mine + j];
      p.c.block_table[r * p.c.table_stride + slot + j] = page;
      p.c.refs[page] = 1;
    }
    p.c.lens[r] = len + add[r];
  }
}

// Children take over their parents' pages: shared, the last partial one copied; or (copy) copies of all.
__global__ void __launch_bounds__(kPlanThreads)
kv_fork_kernel(const KvParams p, const int32_t* parents, const int32_t* children, int n, int copy) {
  pdl_trigger();
  pdl_wait();
  const int ps = p.c.page_size;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int c = children[i];
    if (c >= 0 && c < p.c.rows) p.w.first[c] = 0x7fffffff;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int c = children[i];
    if (c >= 0 && c < p.c.rows) atomicMin(&p.w.first[c], i);
  }
  __syncthreads();
  int demand = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int par = parents[i], c = children[i];
      const bool ok = par >= 0 && par < p.c.rows && c >= 0 && c < p.c.rows && p.w.first[c] == i && p.c.lens[c] == 0 &&
                      len_ok(p, p.c.lens[par]);
      if (ok) {
        const int len = p.c.lens[par];
        need = copy ? pages_of(len, ps) : (len % ps != 0);
        p.w.need[i] = need;
      } else {
        record_fault(p.status, KLC_ERR_DEVICE_FAULT, 532, i);
        p.w.need[i] = -1;
      }
    }
    int total;
    block_scan(need, &total);
    demand += total;
  }
  const int have = demand > 0 ? collect_free(p, demand) : 0;
  __shared__ int moves;
  if (threadIdx.x == 0) moves = demand;
  __syncthreads();
  // lengths are still the old ones: a child that is a parent too passes on what it had (nothing)
  int at = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    const int need = i < n ? p.w.need[i] : 0;
    int total;
    const int mine = at + block_scan(max(need, 0), &total);
    at += total;
    if (i < n && need > 0 && mine + need > have) {
      record_fault(p.status, KLC_ERR_DEVICE_FAULT, 533, i);  // out of pages: the child stays empty
      p.w.need[i] = -1;
      atomicMin(&moves, mine);  // so do all later ones that need pages: the moves end here
    }
    if (i < n && need > 0) p.w.first[children[i]] = mine;  // the child's first new page (its index in ids)
  }
  __syncthreads();
  // tables: one warp per child
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < n; i += kPlanThreads / 32) {
    if (p.w.need[i] < 0) continue;
    const int par = parents[i], c = children[i];
    const int len = p.c.lens[par], held = pages_of(len, ps), shared = copy ? 0 : len / ps;
    const int mine = p.w.need[i] > 0 ? p.w.first[c] : 0;
    for (int j = lane; j < held; j += 32) {
      const int src = p.c.block_table[int64_t(par) * p.c.table_stride + j];
      int page = src;
      if (src < 0 || src >= p.c.pages) {
        record_fault(p.status, KLC_ERR_DEVICE_FAULT, 534, src);
        page = -1;
      } else if (j < shared) {
        atomicAdd(&p.c.refs[src], 1);
      }
      if (j >= shared) {
        const int e = mine + j - shared;
        const int fresh = p.w.ids[e];
        p.w.src[e] = page;  // -1: nothing to copy
        p.w.dst[e] = fresh;
        p.c.refs[fresh] = 1;
        page = fresh;
      }
      p.c.block_table[int64_t(c) * p.c.table_stride + j] = page;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if (p.w.need[i] >= 0) p.w.need[i] = p.c.lens[parents[i]];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if (p.w.need[i] >= 0) p.c.lens[children[i]] = p.w.need[i];
  if (threadIdx.x == 0) *p.w.count = moves;
}

// Rows give their pages back; one block per listed row.  Who lists a row twice finds it empty the second time.
__global__ void __launch_bounds__(kCopyThreads) kv_free_kernel(const KvParams p, const int32_t* rows) {
  pdl_trigger();
  pdl_wait();
  __shared__ int len_s;
  const int r = rows[blockIdx.x];
  if (r < 0 || r >= p.c.rows) {
    if (threadIdx.x == 0) record_fault(p.status, KLC_ERR_DEVICE_FAULT, 535, r);
    return;
  }
  if (threadIdx.x == 0) len_s = atomicExch(&p.c.lens[r], 0);
  __syncthreads();
  const int len = len_s;
  if (!len_ok(p, len)) {
    if (threadIdx.x == 0) {
      p.c.lens[r] = len;  // the row stays as it was
      record_fault(p.status, KLC_ERR_DEVICE_FAULT, 536, r);
    }
    return;
  }
  const int held = pages_of(len, p.c.page_size);
  for (int j = threadIdx.x; j < held; j += kCopyThreads) {
    int32_t* entry = &p.c.block_table[int64_t(r) * p.c.table_stride + j];
    const int page = *entry;
    *entry = -1;
    if (page < 0 || page >= p.c.pages) {
      record_fault(p.status, KLC_ERR_DEVICE_FAULT, 534, page);
    } else if (atomicSub(&p.c.refs[page], 1) <= 0) {
      atomicAdd(&p.c.refs[page], 1);
      record_fault(p.status, KLC_ERR_DEVICE_FAULT, 537, page);  // the page was free already
    }
  }
}

// Live pages with the highest ids move into the lowest free ones, so that the live pages are 0 .. n_live - 1.
__global__ void __launch_bounds__(kPlanThreads) kv_compact_kernel(const KvParams p, int32_t* n_live) {
  pdl_trigger();
  pdl_wait();
  int live = 0;
  for (int64_t base = 0; base < p.c.pages; base += kPlanThreads * 16) {
    const int64_t from = base + threadIdx.x * 16;
    int r[16], n = 0, total;
    if (from < p.c.pages) {
      load_refs(p, from, r);
#pragma unroll
      for (int j = 0; j < 16; ++j) n += from + j < p.c.pages && r[j] > 0;
    }
    block_scan(n, &total);
    live += total;
  }
  int holes = 0, movers = 0;  // the same number in the end
  for (int64_t base = 0; base < p.c.pages; base += kPlanThreads * 16) {
    const int64_t from = base + threadIdx.x * 16;
    int r[16], nh = 0, nm = 0, th, tm;
    if (from < p.c.pages) {
      load_refs(p, from, r);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        nh += from + j < live && r[j] <= 0;
        nm += from + j >= live && from + j < p.c.pages && r[j] > 0;
      }
    }
    int h = holes + block_scan(nh, &th), m = movers + block_scan(nm, &tm);
    if (from < p.c.pages) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int64_t id = from + j;
        if (id < live && r[j] <= 0) p.w.dst[h++] = int(id);
        if (id >= live && id < p.c.pages && r[j] > 0) p.w.src[m++] = int(id);
      }
    }
    holes += th;
    movers += tm;
  }
  __syncthreads();
  for (int64_t id = live + int64_t(threadIdx.x); id < p.c.pages; id += kPlanThreads) p.w.to[id] = int(id);
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kPlanThreads) {
    const int s = p.w.src[i], d = p.w.dst[i];
    p.w.to[s] = d;
    p.c.refs[d] = p.c.refs[s];
    p.c.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    *p.w.count = movers;
    p.w.count[1] = live;
    if (n_live != nullptr) *n_live = live;
  }
}

// Page contents of the planned moves; with `remap` the tables follow.
__global__ void __launch_bounds__(kCopyThreads) kv_move_kernel(const KvParams p, int remap) {
  pdl_trigger();
  pdl_wait();
  const int count = *p.w.count;
  const int64_t chunks = (p.c.page_bytes + kCopyBytes - 1) / kCopyBytes, per_move = chunks * p.c.planes;
  for (int64_t u = blockIdx.x; u < count * per_move; u += gridDim.x) {
    const int64_t mv = u / per_move, rest = u - mv * per_move, plane = rest / chunks, ch = rest - plane * chunks;
    const int s = p.w.src[mv], d = p.w.dst[mv];
    if (s < 0 || d < 0) continue;
    unsigned char* base = reinterpret_cast<unsigned char*>(p.c.pool) + plane * p.c.plane_stride;
    const unsigned char* from = base + int64_t(s) * p.c.page_bytes;
    unsigned char* to = base + int64_t(d) * p.c.page_bytes;
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t off = ch * kCopyBytes + (j * kCopyThreads + threadIdx.x) * 16;
      if (off < p.c.page_bytes) v[j] = ldg_nc_v4(from + off);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t off = ch * kCopyBytes + (j * kCopyThreads + threadIdx.x) * 16;
      if (off < p.c.page_bytes) *reinterpret_cast<uint4*>(to + off) = v[j];
    }
  }
  if (remap) {
    const int live = p.w.count[1];
    const int64_t n = p.c.rows * p.c.table_width;
    for (int64_t e = int64_t(blockIdx.x) * kCopyThreads + threadIdx.x; e < n; e += int64_t(gridDim.x) * kCopyThreads) {
      const int64_t r = e / p.c.table_width, j = e - r * p.c.table_width;
      if (j * p.c.page_size >= p.c.lens[r]) continue;
      int32_t* entry = &p.c.block_table[r * p.c.table_stride + j];
      if (*entry >= live && *entry < p.c.pages) *entry = p.w.to[*entry];
    }
  }
}

size_t work_layout(const klc_kv_cache& c, unsigned char* ws, KvWork* w) {
  size_t off = 0;
  auto take = [&](size_t n) {
    int* at = reinterpret_cast<int*>(ws + off);
    off = align_up(off + n * 4, 256);
    return at;
  };
  KvWork l{};
  l.count = take(4);
  l.ids = take(size_t(c.pages));
  l.src = take(size_t(c.pages));
  l.dst = take(size_t(c.pages));
  l.to = take(size_t(c.pages));
  l.first = take(size_t(c.rows));
  l.need = take(size_t(c.rows));
  if (w != nullptr) *w = l;
  return off;
}

int check_cache(const klc_kv_cache* c, const std::string& w) {
  KLC_CHECK_ARG(c != nullptr, w + ": null cache");
  KLC_CHECK_ARG(c->pages >= 1 && c->pages < (1 << 30), w + ": pages must be between 1 and 2^30");
  KLC_CHECK_ARG(c->rows >= 0 && c->rows < (1 << 24), w + ": rows must be between 0 and 2^24");
  KLC_CHECK_ARG(page_size_ok(c->page_size), w + ": page_size must be 16, 32, 64 or 128");
  KLC_CHECK_ARG(c->table_width >= 0 && c->table_width < (int64_t(1) << 31) && c->table_stride >= c->table_width && c->table_width * c->page_size < (int64_t(1) << 31),
                w + ": bad block table width or stride");
  KLC_CHECK_ARG(c->rows * c->table_width < (int64_t(1) << 31), w + ": the block table is too large");  // pages asked for at once
  KLC_CHECK_ARG(c->planes >= 0 && c->page_bytes > 0 && c->page_bytes % 16 == 0 && c->plane_stride % 16 == 0,
                w + ": page_bytes and plane_stride must be multiples of 16");
  KLC_CHECK_ARG(c->planes <= 1 || c->plane_stride >= c->pages * c->page_bytes, w + ": plane_stride must hold all pages");
  KLC_CHECK_ARG(c->refs != nullptr && (c->rows == 0 || (c->lens != nullptr && (c->block_table != nullptr || c->table_width == 0))),
                w + ": null pointer");
  KLC_CHECK_ARG(aligned16(c->refs), w + ": refs must be 16-byte aligned");
  KLC_CHECK_ARG(c->planes == 0 || (c->pool != nullptr && aligned16(c->pool)), w + ": the pool must be 16-byte aligned");
  return KLC_OK;
}

int bind(const klc_kv_cache* c, const std::string& w, void* workspace, size_t bytes, KvParams* p) {
  const size_t need = work_layout(*c, nullptr, nullptr);
  KLC_CHECK_ARG(workspace != nullptr && aligned16(workspace), w + ": the workspace must be 16-byte aligned");
  if (bytes < need) return fail(KLC_ERR_WORKSPACE, w + ": workspace of " + std::to_string(bytes) + " bytes, need " + std::to_string(need));
  work_layout(*c, reinterpret_cast<unsigned char*>(workspace), &p->w);
  p->c = *c;
  p->status = reinterpret_cast<DeviceStatus*>(c->status);
  return KLC_OK;
}

int launch_moves(const KvParams& p, int64_t max_moves, int remap, cudaStream_t s) {
  const int64_t chunks = (p.c.page_bytes + kCopyBytes - 1) / kCopyBytes * p.c.planes;
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(int64_t(sm_count()) * 8, max_moves * chunks));
  KLC_CUDA(launch_chain(kv_move_kernel, dim3(unsigned(grid)), dim3(kCopyThreads), 0, s, 0, p, remap));
  KLC_LAUNCH_CHECK("kv_move");
  return KLC_OK;
}

}  // namespace
}  // namespace attn
}  // namespace klc

extern "C" int klc_kv_workspace_size(const klc_kv_cache* cache, size_t* out_bytes) {
  using namespace klc;
  using namespace klc::attn;
  KLC_CHECK_ARG(cache != nullptr && out_bytes != nullptr, "klc_kv_workspace_size: null pointer");
  KLC_CHECK_ARG(cache->pages >= 1 && cache->pages < (1 << 30) && cache->rows >= 0 && cache->rows < (1 << 24),
                "klc_kv_workspace_size: bad sizes");
  *out_bytes = work_layout(*cache, nullptr, nullptr);
  return KLC_OK;
}

extern "C" int klc_kv_reserve(const klc_kv_cache* cache, const int32_t* add, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace klc;
  using namespace klc::attn;
  int st = check_cache(cache, "klc_kv_reserve");
  if (st != KLC_OK) return st;
  if (cache->rows == 0) return KLC_OK;
  KLC_CHECK_ARG(add != nullptr, "klc_kv_reserve: null add");
  KvParams p{};
  if ((st = bind(cache, "klc_kv_reserve", workspace, workspace_bytes, &p)) != KLC_OK) return st;
  KLC_CUDA(launch_chain(kv_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), 0, p, add));
  KLC_LAUNCH_CHECK("kv_reserve");
  return KLC_OK;
}

extern "C" int klc_kv_fork(const klc_kv_cache* cache, const int32_t* parents, const int32_t* children, int64_t n, int copy,
                           void* workspace, size_t workspace_bytes, void* stream) {
  using namespace klc;
  using namespace klc::attn;
  int st = check_cache(cache, "klc_kv_fork");
  if (st != KLC_OK) return st;
  KLC_CHECK_ARG(n >= 0 && n <= cache->rows, "klc_kv_fork: n must be between 0 and the number of rows");
  if (n == 0) return KLC_OK;
  KLC_CHECK_ARG(parents != nullptr && children != nullptr, "klc_kv_fork: null list");
  KvParams p{};
  if ((st = bind(cache, "klc_kv_fork", workspace, workspace_bytes, &p)) != KLC_OK) return st;
  KLC_CUDA(launch_chain(kv_fork_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), 0, p, parents, children, int(n), copy));
  KLC_LAUNCH_CHECK("kv_fork");
  return launch_moves(p, copy ? std::min(cache->pages, n * cache->table_width) : n, 0, as_stream(stream));
}

extern "C" int klc_kv_free(const klc_kv_cache* cache, const int32_t* rows, int64_t n, void* stream) {
  using namespace klc;
  using namespace klc::attn;
  int st = check_cache(cache, "klc_kv_free");
  if (st != KLC_OK) return st;
  KLC_CHECK_ARG(n >= 0 && n < (1 << 24), "klc_kv_free: bad number of rows");
  if (n == 0) return KLC_OK;
  KLC_CHECK_ARG(rows != nullptr, "klc_kv_free: null list");
  KvParams p{};
  p.c = *cache;
  p.status = reinterpret_cast<DeviceStatus*>(cache->status);
  KLC_CUDA(launch_chain(kv_free_kernel, dim3(unsigned(n)), dim3(kCopyThreads), 0, as_stream(stream), 0, p, rows));
  KLC_LAUNCH_CHECK("kv_free");
  return KLC_OK;
}

extern "C" int klc_kv_compact(const klc_kv_cache* cache, int32_t* n_live, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace klc;
  using namespace klc::attn;
  int st = check_cache(cache, "klc_kv_compact");
  if (st != KLC_OK) return st;
  KvParams p{};
  if ((st = bind(cache, "klc_kv_compact", workspace, workspace_bytes, &p)) != KLC_OK) return st;
  KLC_CUDA(launch_chain(kv_compact_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), 0, p, n_live));
  KLC_LAUNCH_CHECK("kv_compact");
  return launch_moves(p, cache->pages / 2 + 1, 1, as_stream(stream));
}
