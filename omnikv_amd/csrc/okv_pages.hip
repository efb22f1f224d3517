// Page operations of a pool (okv_pages_*): plans made by one workgroup, data moved by many.
//
// A page is free when no table row names it (refs 0).  Free pages are handed out lowest first and entries are served
// in their order, so a call's result depends on its inputs alone, whatever the timing.
#include "okv_internal.h"

namespace okv {

constexpr int kBuffersPerLaunch = 128;
constexpr int kPlanThreads = 1024;

struct BufferList {
  okv_page_buffer_t b[kBuffersPerLaunch];
};

__device__ __forceinline__ int pages_of(int64_t tokens, int page_size) {
  return (int)((tokens + page_size - 1) / page_size);
}

// inclusive prefix sum over the 1024 threads of a plan; total: of all
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int s_wave[kPlanThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last scan's sums have been read
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += s_wave[w];
    all += s_wave[w];
  }
  *total = all;
  return x + before;
}

// Scratch of a plan, shared through the second-level cache: every cell is written and read with device-scope
// accesses, since atomics pass the first level by.
__device__ __forceinline__ int get(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void put(int32_t* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct PagesWs {
  int32_t* first;  // [num_seqs] lowest entry that names the sequence
  int32_t* fresh;  // [num_pages] free pages, ascending (compact: the new number of every page)
  int32_t* count;  // [4] 0: moves of a compaction
  int32_t* a;      // [n] fork: shared pages of the pair; extend: pages held
  int32_t* b;      // [n] fork: page to copy or -1;       extend: pages after
  int32_t* c;      // [n] fork: page to copy it to;       extend: place of its first page in `fresh`
  int32_t *src, *dst;  // compact: [num_pages] moves
};
static size_t pages_ws_bytes(const okv_page_pool_t* p, int64_t n) {
  return 4 * ((size_t)p->num_seqs + 3 * (size_t)p->num_pages + 16 + 3 * (size_t)n) + 256;
}
static PagesWs carve(const okv_page_pool_t* p, int64_t n, void* ws) {
  int32_t* x = (int32_t*)(((size_t)ws + 255) & ~(size_t)255);
  PagesWs w;
  w.first = x; x += p->num_seqs;
  w.fresh = x; x += p->num_pages;
  w.src = x; x += p->num_pages;
  w.dst = x; x += p->num_pages;
  w.count = x; x += 16;
  w.a = x; x += n;
  w.b = x; x += n;
  w.c = x;
  return w;
}

__global__ __launch_bounds__(256) void pages_free_kernel(okv_page_pool_t p, const int32_t* seqs, int n, int32_t* status) {
  __shared__ int s_pages, s_bad;
  const int s = seqs[blockIdx.x];
  const bool ok = (uint32_t)s < (uint32_t)p.num_seqs;
  if (threadIdx.x == 0) {
    s_bad = 0;
    // whoever takes the length gives the pages back: a sequence named twice is freed once
    const int len = ok ? atomicExch(&p.lens[s], 0) : 0;
    s_pages = len > 0 ? min(pages_of(len, p.page_size), p.max_pages) : 0;
  }
  __syncthreads();
  const int np = s_pages;
  for (int i = threadIdx.x; i < np; i += 256) {
    int32_t* e = p.table + (int64_t)s * p.table_stride + i;
    const int id = *e;
    *e = -1;
    if ((uint32_t)id < (uint32_t)p.num_pages) atomicSub(&p.refs[id], 1);
  }
  if (status && blockIdx.x == 0) {
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += 256) bad += (uint32_t)seqs[i] >= (uint32_t)p.num_seqs;
    if (bad) atomicAdd(&s_bad, bad);
    __syncthreads();
    if (threadIdx.x == 0) {
      status[0] = 0;
      status[1] = s_bad;
    }
  }
}

// first[s] = the lowest entry that names sequence s; every thread of the plan calls it
__device__ void claim(const okv_page_pool_t& p, const int32_t* seqs, int n, int32_t* first) {
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if ((uint32_t)seqs[i] < (uint32_t)p.num_seqs) put(&first[seqs[i]], 0x7fffffff);
  __threadfence();
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if ((uint32_t)seqs[i] < (uint32_t)p.num_seqs) atomicMin(&first[seqs[i]], i);
  __threadfence();
  __syncthreads();
}

// The `want` lowest free pages into fresh[]; returns how many there are (at most want).
__device__ int find_free(const okv_page_pool_t& p, int want, int32_t* fresh) {
  int have = 0;
  for (int base = 0; base < p.num_pages && have < want; base += kPlanThreads) {
    const int id = base + (int)threadIdx.x;
    const int is_free = id < p.num_pages && p.refs[id] <= 0;
    int total;
    const int at = have + block_scan(is_free, &total) - is_free;
    if (is_free && at < want) put(&fresh[at], id);
    have += total;
  }
  __threadfence();
  __syncthreads();
  return have < want ? have : want;
}

__global__ __launch_bounds__(kPlanThreads) void pages_fork_plan(okv_page_pool_t p, const int32_t* parents,
                                                               const int32_t* children, int n, int32_t* status, PagesWs w) {
  claim(p, children, n, w.first);
  int want = 0, bad = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + (int)threadIdx.x;
    int need = 0, refuse = 0;
    if (i < n) {
      const int from = parents[i], to = children[i];
      bool ok = (uint32_t)from < (uint32_t)p.num_seqs && (uint32_t)to < (uint32_t)p.num_seqs && from != to;
      ok = ok && get(&w.first[to]) == i && p.lens[to] <= 0;
      const int len = ok ? p.lens[from] : 0;
      const int full = len > 0 ? len / p.page_size : 0;
      const int part = len > 0 && len % p.page_size && full < p.max_pages;
      const int old = part ? p.table[(int64_t)from * p.table_stride + full] : -1;
      refuse = !ok;
      need = part;
      w.a[i] = ok ? min(full, p.max_pages) : -1;
      w.b[i] = (uint32_t)old < (uint32_t)p.num_pages ? old : -1;
    }
    int total;
    const int at = want + block_scan(need, &total) - need;
    if (i < n) w.c[i] = need ? at : -1;
    want += total;
    block_scan(refuse, &total);
    bad += total;
  }
  const int have = find_free(p, want, w.fresh);
  const bool enough = have == want;
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {  // each thread its own entries of a, b, c
    const int full = w.a[i];
    if (!enough || full < 0) {
      w.a[i] = -1;
      w.c[i] = -1;
      continue;
    }
    const int at = w.c[i];
    if (at >= 0) {
      const int page = get(&w.fresh[at]);
      w.c[i] = page;
      p.refs[page] = 1;
    }
  }
  __syncthreads();  // every length has been read
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    // a parent that is itself a child of this call was empty before it
    const int from = parents[i];
    if (w.a[i] > 0 || w.c[i] >= 0) p.lens[children[i]] = p.lens[from];
  }
  if (status && threadIdx.x == 0) {
    status[0] = want - have;
    status[1] = bad;
  }
}

// one page of one buffer, by a workgroup of 256 threads
__device__ __forceinline__ void copy_page(const okv_page_buffer_t& buf, int src, int dst) {
  const char* s = (const char*)buf.base + (int64_t)src * buf.page_bytes;
  char* d = (char*)buf.base + (int64_t)dst * buf.page_bytes;
  if ((((uintptr_t)buf.base | (uintptr_t)buf.page_bytes) & 15) == 0) {
    for (int64_t o = 16 * threadIdx.x; o < buf.page_bytes; o += 16 * 256)
      *reinterpret_cast<uint4*>(d + o) = *reinterpret_cast<const uint4*>(s + o);
  } else {
    for (int64_t o = 4 * threadIdx.x; o < buf.page_bytes; o += 4 * 256)
      *reinterpret_cast<uint32_t*>(d + o) = *reinterpret_cast<const uint32_t*>(s + o);
  }
}

// grid (n, 1 + buffers): y = 0 names the pages in the child's row, the others copy the partly filled page
__global__ __launch_bounds__(256) void pages_fork_apply(okv_page_pool_t p, const int32_t* parents, const int32_t* children,
                                                        PagesWs w, BufferList bufs, int rows) {
  const int i = blockIdx.x, full = w.a[i], fresh = w.c[i];
  if (full < 0) return;
  if (rows && blockIdx.y == 0) {
    const int32_t* from = p.table + (int64_t)parents[i] * p.table_stride;
    int32_t* to = p.table + (int64_t)children[i] * p.table_stride;
    for (int k = threadIdx.x; k < full; k += 256) {
      const int id = from[k];
      to[k] = id;
      if ((uint32_t)id < (uint32_t)p.num_pages) atomicAdd(&p.refs[id], 1);
    }
    if (fresh >= 0 && threadIdx.x == 0) to[full] = fresh;
    return;
  }
  const int old = w.b[i];
  if (fresh >= 0 && old >= 0) copy_page(bufs.b[blockIdx.y - rows], old, fresh);
}

__global__ __launch_bounds__(kPlanThreads) void pages_extend_plan(okv_page_pool_t p, const int32_t* seqs, const int32_t* more,
                                                                 int n, int32_t* status, PagesWs w) {
  claim(p, seqs, n, w.first);
  int want = 0, bad = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + (int)threadIdx.x;
    int need = 0, refuse = 0;
    if (i < n) {
      const int s = seqs[i];
      bool ok = (uint32_t)s < (uint32_t)p.num_seqs && get(&w.first[s]) == i;
      const int64_t len = ok ? max(p.lens[s], 0) : 0, to = len + max(more[i], 0);
      ok = ok && to <= 0x7fffffff && to <= (int64_t)p.max_pages * p.page_size;
      refuse = !ok;
      w.a[i] = ok ? pages_of(len, p.page_size) : -1;
      w.b[i] = ok ? pages_of(to, p.page_size) : -1;
      need = ok ? w.b[i] - w.a[i] : 0;
    }
    int total;
    const int at = want + block_scan(need, &total) - need;
    if (i < n) w.c[i] = at;
    want += total;
    block_scan(refuse, &total);
    bad += total;
  }
  const int have = find_free(p, want, w.fresh);
  if (have == want) {
    for (int i = 0; i < n; ++i) {
      const int from = w.a[i], to = w.b[i], at = w.c[i], s = seqs[i];
      if (from < 0) continue;
      for (int k = from + (int)threadIdx.x; k < to; k += kPlanThreads) {
        const int page = get(&w.fresh[at + k - from]);
        p.table[(int64_t)s * p.table_stride + k] = page;
        p.refs[page] = 1;
      }
      if (threadIdx.x == 0) p.lens[s] = max(p.lens[s], 0) + max(more[i], 0);
    }
  }
  if (status && threadIdx.x == 0) {
    status[0] = want - have;
    status[1] = bad;
  }
}

__global__ __launch_bounds__(256) void pages_copy_kernel(BufferList bufs, int num_buffers, int num_pages, const int32_t* src,
                                                         const int32_t* dst, const int32_t* count, int n) {
  int m = count ? *count : n;
  m = m > n ? n : m;
  for (int64_t u = blockIdx.x; u < (int64_t)m * num_buffers; u += gridDim.x) {
    const int i = (int)(u / num_buffers), j = (int)(u % num_buffers);
    const int s = src[i], d = dst[i];
    if ((uint32_t)s < (uint32_t)num_pages && (uint32_t)d < (uint32_t)num_pages && s != d) copy_page(bufs.b[j], s, d);
  }
}

__global__ __launch_bounds__(kPlanThreads) void pages_compact_plan(okv_page_pool_t p, int32_t* refs_out, int32_t* used_out,
                                                                  PagesWs w) {
  int used = 0;
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {
    const int id = base + (int)threadIdx.x;
    int total;
    block_scan(id < p.num_pages && p.refs[id] > 0, &total);
    used += total;
  }
  int nf = 0, nu = 0;
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {
    const int id = base + (int)threadIdx.x;
    const bool in = id < p.num_pages, busy = in && p.refs[id] > 0;
    const int hole = in && !busy && id < used, high = busy && id >= used;
    int total;
    const int af = nf + block_scan(hole, &total) - hole;
    nf += total;
    const int au = nu + block_scan(high, &total) - high;
    nu += total;
    if (hole) put(&w.dst[af], id);
    if (high) put(&w.src[au], id);
    if (in && !high) put(&w.fresh[id], id);  // keeps its number
  }
  __threadfence();
  __syncthreads();
  // as many holes below `used` as pages in use at or above it
  for (int i = threadIdx.x; i < nu; i += kPlanThreads) put(&w.fresh[get(&w.src[i])], get(&w.dst[i]));
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {  // the pages that stay; refs_out may be refs
    const int id = base + (int)threadIdx.x;
    if (id < p.num_pages && id < used && p.refs[id] > 0) refs_out[id] = p.refs[id];
  }
  for (int i = threadIdx.x; i < nu; i += kPlanThreads) {
    const int s = get(&w.src[i]), v = p.refs[s];
    refs_out[get(&w.dst[i])] = v;
  }
  __syncthreads();
  for (int id = used + (int)threadIdx.x; id < p.num_pages; id += kPlanThreads) refs_out[id] = 0;
  if (threadIdx.x == 0) {
    w.count[0] = nu;
    if (used_out) *used_out = used;
  }
}

// grid (blocks, num_seqs): every entry gets its page's new number
__global__ __launch_bounds__(256) void pages_compact_table(okv_page_pool_t p, int32_t* out, int64_t out_stride, PagesWs w) {
  const int s = blockIdx.y, k = blockIdx.x * 256 + threadIdx.x;
  if (k >= p.max_pages) return;
  const int id = p.table[(int64_t)s * p.table_stride + k];
  out[(int64_t)s * out_stride + k] = (uint32_t)id < (uint32_t)p.num_pages ? w.fresh[id] : id;
}

static int check_pool(const okv_page_pool_t* p, const char* what, bool lens) {
  OKV_REQUIRE(p != nullptr, OKV_ERR_INVALID, "%s: pool is NULL", what);
  OKV_REQUIRE(p->table && p->refs && (p->lens || !lens), OKV_ERR_INVALID, "%s: NULL table, lens or refs", what);
  OKV_REQUIRE(p->num_seqs >= 1 && p->max_pages >= 1 && p->num_pages >= 1 && p->page_size >= 1, OKV_ERR_INVALID,
              "%s: num_seqs %d, max_pages %d, num_pages %d, page_size %d", what, p->num_seqs, p->max_pages, p->num_pages,
              p->page_size);
  OKV_REQUIRE(p->table_stride >= p->max_pages, OKV_ERR_INVALID, "%s: table_stride < max_pages", what);
  return OKV_OK;
}
static int check_buffers(const okv_page_buffer_t* b, int n, const char* what) {
  OKV_REQUIRE(n >= 0 && (n == 0 || b), OKV_ERR_INVALID, "%s: buffers are NULL", what);
  for (int i = 0; i < n; ++i)
    OKV_REQUIRE(b[i].base && b[i].page_bytes > 0 && (((uintptr_t)b[i].base | (uintptr_t)b[i].page_bytes) & 3) == 0,
                OKV_ERR_INVALID, "%s: buffer %d: base and page_bytes must be multiples of 4", what, i);
  return OKV_OK;
}
static int check_ws(const okv_page_pool_t* p, int64_t n, void* ws, size_t ws_bytes) {
  const size_t need = pages_ws_bytes(p, n);
  OKV_REQUIRE(ws != nullptr, OKV_ERR_INVALID, "workspace pointer is NULL");
  OKV_REQUIRE(ws_bytes >= need, OKV_ERR_WORKSPACE, "workspace too small: have %zu, need %zu", ws_bytes, need);
  return OKV_OK;
}
static BufferList take(const okv_page_buffer_t* b, int n) {
  BufferList l{};
  for (int i = 0; i < n; ++i) l.b[i] = b[i];
  return l;
}

}  // namespace okv

using namespace okv;

extern "C" {

int okv_pages_workspace_bytes(const okv_page_pool_t* pool, int32_t n, size_t* out_bytes) {
  OKV_REQUIRE(pool != nullptr && out_bytes != nullptr && n >= 0 && pool->num_seqs >= 1 && pool->num_pages >= 1, OKV_ERR_INVALID,
              "bad argument");
  *out_bytes = pages_ws_bytes(pool, n);
  return OKV_OK;
}

int okv_pages_free(const okv_page_pool_t* pool, const int32_t* seqs, int32_t n, int32_t* status, okv_stream_t stream) {
  int rc = check_pool(pool, "okv_pages_free", true);
  if (rc) return rc;
  OKV_REQUIRE(n >= 1 && seqs, OKV_ERR_INVALID, "okv_pages_free: n >= 1 entries");
  hipLaunchKernelGGL(pages_free_kernel, dim3(n), dim3(256), 0, (hipStream_t)stream, *pool, seqs, n, status);
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_pages_fork(const okv_page_pool_t* pool, const int32_t* parents, const int32_t* children, int32_t n,
                   const okv_page_buffer_t* host_buffers, int32_t num_buffers, int32_t* status, void* ws, size_t ws_bytes,
                   okv_stream_t stream) {
  int rc = check_pool(pool, "okv_pages_fork", true);
  if (!rc) rc = check_buffers(host_buffers, num_buffers, "okv_pages_fork");
  if (rc) return rc;
  OKV_REQUIRE(n >= 1 && parents && children, OKV_ERR_INVALID, "okv_pages_fork: n >= 1 pairs");
  rc = check_ws(pool, n, ws, ws_bytes);
  if (rc) return rc;
  const PagesWs w = carve(pool, n, ws);
  hipLaunchKernelGGL(pages_fork_plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, *pool, parents, children, n, status, w);
  for (int lo = 0; lo == 0 || lo < num_buffers; lo += kBuffersPerLaunch) {
    const int m = num_buffers - lo < kBuffersPerLaunch ? num_buffers - lo : kBuffersPerLaunch, rows = lo == 0;
    hipLaunchKernelGGL(pages_fork_apply, dim3(n, m + rows), dim3(256), 0, (hipStream_t)stream, *pool, parents, children, w,
                       take(host_buffers + lo, m), rows);
  }
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_pages_extend(const okv_page_pool_t* pool, const int32_t* seqs, const int32_t* more, int32_t n, int32_t* status,
                     void* ws, size_t ws_bytes, okv_stream_t stream) {
  int rc = check_pool(pool, "okv_pages_extend", true);
  if (rc) return rc;
  OKV_REQUIRE(n >= 1 && seqs && more, OKV_ERR_INVALID, "okv_pages_extend: n >= 1 entries");
  OKV_REQUIRE((int64_t)n * pool->max_pages < (1ll << 30), OKV_ERR_UNSUPPORTED,
              "okv_pages_extend: %d entries of up to %d pages in one call", n, pool->max_pages);
  rc = check_ws(pool, n, ws, ws_bytes);
  if (rc) return rc;
  hipLaunchKernelGGL(pages_extend_plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, *pool, seqs, more, n, status,
                     carve(pool, n, ws));
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_pages_copy(const okv_page_buffer_t* host_buffers, int32_t num_buffers, int32_t num_pages, const int32_t* src,
                   const int32_t* dst, const int32_t* count, int32_t n, okv_stream_t stream) {
  int rc = check_buffers(host_buffers, num_buffers, "okv_pages_copy");
  if (rc) return rc;
  OKV_REQUIRE(n >= 0 && num_pages >= 1 && (n == 0 || (src && dst)), OKV_ERR_INVALID, "okv_pages_copy: bad lists");
  if (n == 0) return OKV_OK;
  for (int lo = 0; lo < num_buffers; lo += kBuffersPerLaunch) {
    const int m = num_buffers - lo < kBuffersPerLaunch ? num_buffers - lo : kBuffersPerLaunch;
    const int64_t units = (int64_t)n * m;
    hipLaunchKernelGGL(pages_copy_kernel, dim3((uint32_t)(units < 4096 ? units : 4096)), dim3(256), 0, (hipStream_t)stream,
                       take(host_buffers + lo, m), m, num_pages, src, dst, count, n);
  }
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_pages_compact(const okv_page_pool_t* pool, int32_t* table_out, int64_t table_out_stride, int32_t* refs_out,
                      int32_t* used_out, const okv_page_buffer_t* host_buffers, int32_t num_buffers, void* ws,
                      size_t ws_bytes, okv_stream_t stream) {
  int rc = check_pool(pool, "okv_pages_compact", false);
  if (!rc) rc = check_buffers(host_buffers, num_buffers, "okv_pages_compact");
  if (rc) return rc;
  OKV_REQUIRE(table_out && refs_out && table_out_stride >= pool->max_pages, OKV_ERR_INVALID, "okv_pages_compact: bad outputs");
  OKV_REQUIRE(pool->num_seqs <= 65535, OKV_ERR_UNSUPPORTED, "okv_pages_compact: %d sequences", pool->num_seqs);
  rc = check_ws(pool, 0, ws, ws_bytes);
  if (rc) return rc;
  const PagesWs w = carve(pool, 0, ws);
  hipLaunchKernelGGL(pages_compact_plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, *pool, refs_out, used_out, w);
  hipLaunchKernelGGL(pages_compact_table, dim3((pool->max_pages + 255) / 256, pool->num_seqs), dim3(256), 0,
                     (hipStream_t)stream, *pool, table_out, table_out_stride, w);
  OKV_HIP_CHECK(hipGetLastError());
  if (num_buffers == 0) return OKV_OK;
  return okv_pages_copy(host_buffers, num_buffers, pool->num_pages, w.src, w.dst, w.count, pool->num_pages / 2, stream);
}

}  // extern "C"
