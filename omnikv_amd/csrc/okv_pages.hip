// Page operations of a pool (okv_pages_*): plans made by one workgroup, data moved by many.
//
// A page is free when no table row names it (refs 0).  Free pages are handed out lowest first and entries are served
// in their order, so a call's result depends on its inputs alone, whatever the timing.
//
// A plan is one workgroup, because "lowest free first" is one prefix sum over the counts and because a scan over workgroups
// would need device-wide fences, which cost more than the scan (a plan with them took 16 us, without 3.6).  Its threads meet in LDS; what it
// decides is read by the next launch.  It is bound by its chain of round trips to memory: 3.6 to 4.9 us for 64 forks, 4.9 to
// compact 4096 pages, 5.3 for 64 sequences to grow (it writes the table's entries itself; 7.9 with a second trip through the counts).  The pages' bytes are moved by the
// launch after it, all buffers at once.
#include "okv_internal.h"

namespace okv {

constexpr int kBuffersPerLaunch = 128;
constexpr int kPlanThreads = 1024;
constexpr int kMaxEntries = kPlanThreads;  // entries of a call: one per thread of the plan
constexpr int kPerThread = 4;              // pages of a plan's trip through the counts, per thread
constexpr int kTrip = kPlanThreads * kPerThread;
constexpr int kMost = 1 << 30;  // pages, sequences, pages of a sequence, entries: what is counted runs a step past the last, in 32 bits

struct BufferList {
  okv_page_buffer_t b[kBuffersPerLaunch];
};

__device__ __forceinline__ int pages_of(int64_t tokens, int page_size) {
  return (int)((tokens + page_size - 1) / page_size);
}

__device__ __forceinline__ int wave_scan(int x) {  // inclusive prefix sum over the wave
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 of a row to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
  return x;
}

// Exclusive prefix sum over the threads of a plan, and the sum of all.  `turn` counts the calls: two sets of cells in
// turn, so that one barrier per call is enough.
__device__ __forceinline__ int block_scan(int v, int* total, int& turn) {
  constexpr int W = kPlanThreads / 64;
  __shared__ int s_wave[2][W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  int* cells = s_wave[turn & 1];
  ++turn;
  if (lane == 63) cells[wave] = x;
  __syncthreads();
  const int sums = wave_scan(lane < W ? cells[lane] : 0);  // the waves' sums, by every wave
  *total = __builtin_amdgcn_readlane(sums, W - 1);
  return x - v + (wave ? __builtin_amdgcn_readlane(sums, __builtin_amdgcn_readfirstlane(wave) - 1) : 0);
}

// The counts of a trip's pages, four per thread in order; 1 behind the last page (in use).
__device__ __forceinline__ int4 load_refs(const okv_page_pool_t& p, int base) {
  const int id = base + kPerThread * (int)threadIdx.x;
  if (id + 3 < p.num_pages && ((uintptr_t)p.refs & 15) == 0) return *reinterpret_cast<const int4*>(p.refs + id);
  int4 r = make_int4(1, 1, 1, 1);
  if (id < p.num_pages) r.x = p.refs[id];
  if (id + 1 < p.num_pages) r.y = p.refs[id + 1];
  if (id + 2 < p.num_pages) r.z = p.refs[id + 2];
  if (id + 3 < p.num_pages) r.w = p.refs[id + 3];
  return r;
}

// Which entry names a sequence first: an open-addressed table in LDS, cleared by its first barrier's other side.
constexpr int kCells = 2 * kMaxEntries;
__device__ __forceinline__ bool first_to_name(int seq, bool valid) {
  __shared__ int s_key[kCells], s_first[kCells];
  for (int i = threadIdx.x; i < kCells; i += kPlanThreads) {
    s_key[i] = -1;
    s_first[i] = kMaxEntries;
  }
  __syncthreads();
  int cell = 0;
  if (valid) {
    cell = (int)(((uint32_t)seq * 2654435761u) >> 21) & (kCells - 1);
    while (true) {  // at most kMaxEntries keys in twice as many cells: an empty one is always found
      const int seen = atomicCAS(&s_key[cell], -1, seq);
      if (seen == -1 || seen == seq) break;
      cell = (cell + 1) & (kCells - 1);
    }
    atomicMin(&s_first[cell], (int)threadIdx.x);
  }
  __syncthreads();
  return valid && s_first[cell] == (int)threadIdx.x;
}

struct PagesWs {
  int32_t* count;  // [16] 0: moves of a compaction
  int32_t* full;   // [n] fork: shared pages of the pair, -1: nothing to do
  int32_t *src, *dst;  // fork [n], compact [num_pages / 2]: pages to copy and where to; -1: none
  int32_t* to;     // compact: [num_pages] the page's new number
  int32_t *from_seq, *to_seq;  // fork [n]: sequences of the pairs that are served, -1: none
};
static size_t pages_ws_bytes(const okv_page_pool_t* p, int64_t n) {
  return 4 * (2 * (size_t)p->num_pages + 16 + 5 * (size_t)n) + 256;
}
static PagesWs carve(const okv_page_pool_t* p, int64_t n, void* ws) {
  int32_t* x = (int32_t*)(((size_t)ws + 255) & ~(size_t)255);
  PagesWs w;
  w.count = x; x += 16;
  w.full = x; x += n;
  const int64_t m = n > 0 ? n : p->num_pages / 2;
  w.src = x; x += m;
  w.dst = x; x += m;
  w.from_seq = x; x += n;
  w.to_seq = x; x += n;
  w.to = x;
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

// One thread per pair.  A chain of three round trips to memory (the pair, the lengths, the last page's number), with
// the counts of the first 4096 pages on their way meanwhile.
__global__ __launch_bounds__(kPlanThreads) void pages_fork_plan(okv_page_pool_t p, const int32_t* parents,
                                                               const int32_t* children, int n, int32_t* status, PagesWs w) {
  __shared__ int s_fresh[kMaxEntries];
  const int i = threadIdx.x;
  int turn = 0;
  int4 refs = load_refs(p, 0);
  const int from = i < n ? parents[i] : -1, to = i < n ? children[i] : -1;
  const bool from_in = (uint32_t)from < (uint32_t)p.num_seqs, to_in = (uint32_t)to < (uint32_t)p.num_seqs;
  int len = from_in ? p.lens[from] : 0;
  const int held = to_in ? p.lens[to] : 0;
  const bool named_first = first_to_name(to, to_in);
  const bool ok = named_first && from_in && from != to && held <= 0;
  if (!ok || len < 0) len = 0;
  const int full = min(len / p.page_size, p.max_pages);
  const bool part = len % p.page_size != 0 && full < p.max_pages;
  const int old = part ? p.table[(int64_t)from * p.table_stride + full] : -1;
  int want, bad;
  const int at = block_scan(part, &want, turn);
  block_scan(i < n && !ok, &bad, turn);
  int have = 0;
  for (int base = 0; base < p.num_pages && have < want; base += kTrip) {
    if (base) refs = load_refs(p, base);
    const int f[4] = {refs.x <= 0, refs.y <= 0, refs.z <= 0, refs.w <= 0};
    int total;
    int k = have + block_scan(f[0] + f[1] + f[2] + f[3], &total, turn);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (f[x] && k < want) s_fresh[k] = base + kPerThread * i + x;
      k += f[x];
    }
    have = min(have + total, want);
  }
  __syncthreads();  // fresh pages known; every length has been read
  const bool act = have == want && ok && len > 0;
  const int fresh = act && part ? s_fresh[at] : -1;
  if (i < n) {
    w.full[i] = act ? full : -1;
    w.src[i] = fresh >= 0 ? old : -1;
    w.dst[i] = fresh;
    w.from_seq[i] = act ? from : -1;
    w.to_seq[i] = act ? to : -1;
  }
  // a parent that is itself a child of this call was empty before it: its length is not one that is written here
  if (act) p.lens[to] = len;
  if (fresh >= 0) p.refs[fresh] = 1;
  if (status && i == 0) {
    status[0] = want - have;
    status[1] = bad;
  }
}

// Pages of one buffer, by a workgroup of 256 threads: moves [first, first + per), `per` pages of a small buffer side
// by side, a page of a large one with four loads of a thread in flight.
// Bound by the bytes: 64 forks over 64 arrays (61 pages of 16 tokens, 64 MB read and written) 15 us = 4.3 TB/s, 906 pages of 64 tokens over
// 64 arrays (3.8 GB) 736 us = 5.2; one load in flight and cached stores 268 us where this takes 183 (1.08 GB).
template <typename V>
__device__ __forceinline__ void copy_pages(const okv_page_buffer_t& buf, const int32_t* src, const int32_t* dst, int first, int per,
                                           int m, int num_pages) {
  const uint32_t unit = (uint32_t)(buf.page_bytes / (int64_t)sizeof(V));
  V* base = reinterpret_cast<V*>(buf.base);
  if (per > 1) {
    const uint32_t k = threadIdx.x / unit, o = threadIdx.x % unit;
    const int i = first + (int)k;
    if ((int)k >= per || i >= m) return;
    const int s = src[i], d = dst[i];
    if ((uint32_t)s < (uint32_t)num_pages && (uint32_t)d < (uint32_t)num_pages) base[(int64_t)d * unit + o] = base[(int64_t)s * unit + o];
    return;
  }
  if (first >= m) return;
  const int s = src[first], d = dst[first];
  if ((uint32_t)s >= (uint32_t)num_pages || (uint32_t)d >= (uint32_t)num_pages || s == d) return;
  const int64_t pu = buf.page_bytes / (int64_t)sizeof(V);
  const V* from = base + (int64_t)s * pu;
  V* to = base + (int64_t)d * pu;
  int64_t o = threadIdx.x;
  for (; o + 768 < pu; o += 1024) {
    const V x0 = __builtin_nontemporal_load(from + o), x1 = __builtin_nontemporal_load(from + o + 256),
            x2 = __builtin_nontemporal_load(from + o + 512), x3 = __builtin_nontemporal_load(from + o + 768);
    __builtin_nontemporal_store(x0, to + o);
    __builtin_nontemporal_store(x1, to + o + 256);
    __builtin_nontemporal_store(x2, to + o + 512);
    __builtin_nontemporal_store(x3, to + o + 768);
  }
  for (; o < pu; o += 256) to[o] = from[o];
}
typedef __attribute__((ext_vector_type(4))) uint32_t page_vec;
// moves blockIdx.x, + gridDim.x, ... of `m` (in steps of as many pages as a workgroup takes at once)
__device__ __forceinline__ void copy_moves(const okv_page_buffer_t& buf, const int32_t* src, const int32_t* dst, int m, int num_pages,
                                           int block, int blocks) {
  const bool wide = (((uintptr_t)buf.base | (uintptr_t)buf.page_bytes) & 15) == 0;
  const int64_t unit = buf.page_bytes / (wide ? 16 : 4);
  const int per = unit <= 128 ? 256 / (int)unit : 1;
  for (int64_t first = (int64_t)block * per; first < m; first += (int64_t)blocks * per) {
    if (wide) copy_pages<page_vec>(buf, src, dst, (int)first, per, m, num_pages);
    else copy_pages<uint32_t>(buf, src, dst, (int)first, per, m, num_pages);
  }
}

// grid (n, 1 + buffers): y = 0 names the pages in the child's row, the others copy the partly filled pages, and from buffer
// `first_row` on the sequences' rows
__global__ __launch_bounds__(256) void pages_fork_apply(okv_page_pool_t p, const int32_t* parents, const int32_t* children,
                                                        int n, PagesWs w, BufferList bufs, int first_row, int rows) {
  if (!rows || blockIdx.y > 0) {
    const int j = (int)blockIdx.y - rows;
    if (j < first_row) copy_moves(bufs.b[j], w.src, w.dst, n, p.num_pages, blockIdx.x, gridDim.x);
    else copy_moves(bufs.b[j], w.from_seq, w.to_seq, n, p.num_seqs, blockIdx.x, gridDim.x);
    return;
  }
  const int i = blockIdx.x, full = w.full[i], fresh = w.dst[i];
  if (full < 0) return;
  const int32_t* from = p.table + (int64_t)parents[i] * p.table_stride;
  int32_t* to = p.table + (int64_t)children[i] * p.table_stride;
  for (int k = threadIdx.x; k < full; k += 256) {
    const int id = from[k];
    to[k] = id;
    if ((uint32_t)id < (uint32_t)p.num_pages) atomicAdd(&p.refs[id], 1);
  }
  if (fresh >= 0 && threadIdx.x == 0) to[full] = fresh;
}

// One thread per entry.  A trip through the counts finds the free pages, the first kFresh of them are kept in LDS, and if
// there are enough a thread per page writes it into the table; a call that takes more pages goes through the counts again.
constexpr int kFresh = 4096;
__global__ __launch_bounds__(kPlanThreads) void pages_extend_plan(okv_page_pool_t p, const int32_t* seqs, const int32_t* more,
                                                                 int n, int32_t* status) {
  __shared__ int s_at[kMaxEntries + 1], s_seq[kMaxEntries], s_from[kMaxEntries], s_fresh[kFresh];
  const int i = threadIdx.x;
  int turn = 0;
  int4 refs = load_refs(p, 0);
  const int s = i < n ? seqs[i] : -1;
  const int64_t grow = i < n ? max(more[i], 0) : 0;
  const bool in = (uint32_t)s < (uint32_t)p.num_seqs;
  const int64_t len = in ? max(p.lens[s], 0) : 0, to = len + grow;
  const bool ok = first_to_name(s, in) && to <= 0x7fffffff && to <= (int64_t)p.max_pages * p.page_size;
  const int from = ok ? pages_of(len, p.page_size) : 0, need = ok ? pages_of(to, p.page_size) - from : 0;
  int want, bad, have = 0, total;
  s_at[i] = block_scan(need, &want, turn);
  s_seq[i] = s;
  s_from[i] = from;
  block_scan(i < n && !ok, &bad, turn);
  // the k-th page taken goes to the last entry whose pages start at or before the k-th
  auto give = [&](int k, int page) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_at[mid] <= k) lo = mid;
      else hi = mid - 1;
    }
    p.table[(int64_t)s_seq[lo] * p.table_stride + s_from[lo] + (k - s_at[lo])] = page;
    p.refs[page] = 1;
  };
  auto trip = [&](int base, const int4& r, int k0, auto take) {  // the number of free pages of a trip; take(k, page) of each
    const int f[4] = {r.x <= 0, r.y <= 0, r.z <= 0, r.w <= 0};
    int k = k0 + block_scan(f[0] + f[1] + f[2] + f[3], &total, turn);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (f[x] && k < want) take(k, base + kPerThread * i + x);
      k += f[x];
    }
    return total;
  };
  for (int base = 0; base < p.num_pages && have < want; base += kTrip)
    have = min(have + trip(base, base ? load_refs(p, base) : refs, have,
                           [&](int k, int page) { if (k < kFresh) s_fresh[k] = page; }), want);
  __syncthreads();
  if (have == want) {
    if (ok) p.lens[s] = (int)to;
    if (want <= kFresh)
      for (int k = i; k < want; k += kPlanThreads) give(k, s_fresh[k]);
    else
      for (int base = 0, k0 = 0; base < p.num_pages && k0 < want; base += kTrip)
        k0 += trip(base, base ? load_refs(p, base) : refs, k0, give);
  }
  if (status && i == 0) {
    status[0] = want - have;
    status[1] = bad;
  }
}

// grid (blocks, buffers)
__global__ __launch_bounds__(256) void pages_copy_kernel(BufferList bufs, int num_pages, const int32_t* src, const int32_t* dst,
                                                         const int32_t* count, int n) {
  const int m = count ? min(*count, n) : n;
  copy_moves(bufs.b[blockIdx.y], src, dst, m, num_pages, blockIdx.x, gridDim.x);
}

// Pages at or above `used` that are in use, in order, go to the free ones below it, in order: equally many of both.
__global__ __launch_bounds__(kPlanThreads) void pages_compact_plan(okv_page_pool_t p, int32_t* refs_out, int32_t* used_out,
                                                                  PagesWs w) {
  const int i = threadIdx.x;
  int turn = 0, used = 0, total;
  const int4 first = load_refs(p, 0);
  auto busy = [&](int base, const int4& r, int x) {
    const int v = x == 0 ? r.x : x == 1 ? r.y : x == 2 ? r.z : r.w;
    return v > 0 && base + kPerThread * i + x < p.num_pages;
  };
  for (int base = 0; base < p.num_pages; base += kTrip) {
    const int4 r = base ? load_refs(p, base) : first;
    block_scan(busy(base, r, 0) + busy(base, r, 1) + busy(base, r, 2) + busy(base, r, 3), &total, turn);
    used += total;
  }
  int holes = 0, highs = 0;
  for (int base = 0; base < p.num_pages; base += kTrip) {
    const int4 r = base ? load_refs(p, base) : first;
    int hole[4], high[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int id = base + kPerThread * i + x;
      const bool b = busy(base, r, x);
      hole[x] = id < p.num_pages && id < used && !b;
      high[x] = b && id >= used;
      if (id < p.num_pages && !high[x]) w.to[id] = id;
    }
    int h = holes + block_scan(hole[0] + hole[1] + hole[2] + hole[3], &total, turn);
    holes += total;
    int u = highs + block_scan(high[0] + high[1] + high[2] + high[3], &total, turn);
    highs += total;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int id = base + kPerThread * i + x;
      if (hole[x]) w.dst[h] = id;
      if (high[x]) w.src[u] = id;
      h += hole[x];
      u += high[x];
    }
  }
  __syncthreads();
  for (int k = i; k < highs; k += kPlanThreads) {
    const int s = w.src[k], d = w.dst[k];
    w.to[s] = d;
    refs_out[d] = p.refs[s];  // page s is not below `used`: nothing here has written its count
  }
  if (refs_out != p.refs)
    for (int base = 0; base < used; base += kTrip) {
      const int4 r = base ? load_refs(p, base) : first;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int id = base + kPerThread * i + x;
        if (id < used && busy(base, r, x)) refs_out[id] = x == 0 ? r.x : x == 1 ? r.y : x == 2 ? r.z : r.w;
      }
    }
  __syncthreads();  // the moved pages' counts have been read
  for (int id = used + i; id < p.num_pages; id += kPlanThreads) refs_out[id] = 0;
  if (i == 0) {
    w.count[0] = highs;
    if (used_out) *used_out = used;
  }
}

// grid (blocks, table rows' blocks + buffers): the table's entries get their pages' new numbers, the others move the pages
__global__ __launch_bounds__(256) void pages_compact_apply(okv_page_pool_t p, int32_t* out, int64_t out_stride, PagesWs w,
                                                           BufferList bufs, int table) {
  if (!table || blockIdx.y > 0) {
    copy_moves(bufs.b[blockIdx.y - table], w.src, w.dst, w.count[0], p.num_pages, blockIdx.x, gridDim.x);
    return;
  }
  for (int s = blockIdx.x; s < p.num_seqs; s += gridDim.x)
    for (int k = threadIdx.x; k < p.max_pages; k += 256) {
      const int id = p.table[(int64_t)s * p.table_stride + k];
      out[(int64_t)s * out_stride + k] = (uint32_t)id < (uint32_t)p.num_pages ? w.to[id] : id;
    }
}

// Workgroups along x for `moves` moves of each of `buffers` buffers: some thousands in all, which fill the chip.
static uint32_t copy_blocks(int64_t moves, int buffers) {
  const int64_t most = buffers > 0 ? (4096 + buffers - 1) / buffers : 4096;
  return (uint32_t)(moves < 1 ? 1 : moves < most ? moves : most);
}

static int check_pool(const okv_page_pool_t* p, const char* what, bool lens) {
  OKV_REQUIRE(p != nullptr, OKV_ERR_INVALID, "%s: pool is NULL", what);
  OKV_REQUIRE(p->table && p->refs && (p->lens || !lens), OKV_ERR_INVALID, "%s: NULL table, lens or refs", what);
  OKV_REQUIRE(p->num_seqs >= 1 && p->max_pages >= 1 && p->num_pages >= 1 && p->page_size >= 1, OKV_ERR_INVALID,
              "%s: num_seqs %d, max_pages %d, num_pages %d, page_size %d", what, p->num_seqs, p->max_pages, p->num_pages,
              p->page_size);
  OKV_REQUIRE(p->table_stride >= p->max_pages, OKV_ERR_INVALID, "%s: table_stride < max_pages", what);
  OKV_REQUIRE(p->num_seqs <= kMost && p->max_pages <= kMost && p->num_pages <= kMost, OKV_ERR_UNSUPPORTED,
              "%s: num_seqs %d, max_pages %d, num_pages %d (at most 2^30 each)", what, p->num_seqs, p->max_pages, p->num_pages);
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
// `n` buffers from number `lo` on, of the list `b` of `nb` and the list `c` behind it
static BufferList take(const okv_page_buffer_t* b, int lo, int n, int nb = 1 << 30, const okv_page_buffer_t* c = nullptr) {
  BufferList l{};
  for (int i = 0; i < n; ++i) l.b[i] = lo + i < nb ? b[lo + i] : c[lo + i - nb];
  return l;
}

}  // namespace okv

using namespace okv;

extern "C" {

int okv_pages_workspace_bytes(const okv_page_pool_t* pool, int32_t n, size_t* out_bytes) {
  OKV_REQUIRE(pool != nullptr && out_bytes != nullptr && n >= 0 && pool->num_seqs >= 1 && pool->num_pages >= 1, OKV_ERR_INVALID,
              "bad argument");
  OKV_REQUIRE(pool->num_seqs <= kMost && pool->num_pages <= kMost && n <= kMost, OKV_ERR_UNSUPPORTED,
              "okv_pages_workspace_bytes: %d sequences, %d pages, %d entries (at most 2^30 each)", pool->num_seqs, pool->num_pages, n);
  *out_bytes = pages_ws_bytes(pool, n);
  return OKV_OK;
}

int okv_pages_free(const okv_page_pool_t* pool, const int32_t* seqs, int32_t n, int32_t* status, okv_stream_t stream) {
  int rc = check_pool(pool, "okv_pages_free", true);
  if (rc) return rc;
  OKV_REQUIRE(n >= 1 && seqs, OKV_ERR_INVALID, "okv_pages_free: n >= 1 entries");
  OKV_REQUIRE(n <= kMost, OKV_ERR_UNSUPPORTED, "okv_pages_free: %d entries in one call (at most 2^30)", n);
  hipLaunchKernelGGL(pages_free_kernel, dim3(n), dim3(256), 0, (hipStream_t)stream, *pool, seqs, n, status);
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_pages_fork(const okv_page_pool_t* pool, const int32_t* parents, const int32_t* children, int32_t n,
                   const okv_page_buffer_t* host_buffers, int32_t num_buffers, const okv_page_buffer_t* host_rows,
                   int32_t num_rows, int32_t* status, void* ws, size_t ws_bytes, okv_stream_t stream) {
  int rc = check_pool(pool, "okv_pages_fork", true);
  if (!rc) rc = check_buffers(host_buffers, num_buffers, "okv_pages_fork");
  if (!rc) rc = check_buffers(host_rows, num_rows, "okv_pages_fork, rows");
  if (rc) return rc;
  OKV_REQUIRE(n >= 1 && parents && children, OKV_ERR_INVALID, "okv_pages_fork: n >= 1 pairs");
  OKV_REQUIRE(n <= kMaxEntries, OKV_ERR_UNSUPPORTED, "okv_pages_fork: %d pairs in one call (at most %d)", n, kMaxEntries);
  rc = check_ws(pool, n, ws, ws_bytes);
  if (rc) return rc;
  const PagesWs w = carve(pool, n, ws);
  hipLaunchKernelGGL(pages_fork_plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, *pool, parents, children, n, status, w);
  const int all = num_buffers + num_rows;
  for (int lo = 0; lo == 0 || lo < all; lo += kBuffersPerLaunch) {
    const int m = all - lo < kBuffersPerLaunch ? all - lo : kBuffersPerLaunch, table = lo == 0;
    hipLaunchKernelGGL(pages_fork_apply, dim3(n, m + table), dim3(256), 0, (hipStream_t)stream, *pool, parents, children, n, w,
                       take(host_buffers, lo, m, num_buffers, host_rows), num_buffers - lo, table);
  }
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_pages_extend(const okv_page_pool_t* pool, const int32_t* seqs, const int32_t* more, int32_t n, int32_t* status,
                     okv_stream_t stream) {
  int rc = check_pool(pool, "okv_pages_extend", true);
  if (rc) return rc;
  OKV_REQUIRE(n >= 1 && seqs && more, OKV_ERR_INVALID, "okv_pages_extend: n >= 1 entries");
  OKV_REQUIRE(n <= kMaxEntries, OKV_ERR_UNSUPPORTED, "okv_pages_extend: %d entries in one call (at most %d)", n, kMaxEntries);
  OKV_REQUIRE((int64_t)n * pool->max_pages < (1ll << 30), OKV_ERR_UNSUPPORTED,
              "okv_pages_extend: %d entries of up to %d pages in one call", n, pool->max_pages);
  hipLaunchKernelGGL(pages_extend_plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, *pool, seqs, more, n, status);
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_pages_copy(const okv_page_buffer_t* host_buffers, int32_t num_buffers, int32_t num_pages, const int32_t* src,
                   const int32_t* dst, const int32_t* count, int32_t n, okv_stream_t stream) {
  int rc = check_buffers(host_buffers, num_buffers, "okv_pages_copy");
  if (rc) return rc;
  OKV_REQUIRE(n >= 0 && num_pages >= 1 && (n == 0 || (src && dst)), OKV_ERR_INVALID, "okv_pages_copy: bad lists");
  OKV_REQUIRE(n <= kMost && num_pages <= kMost, OKV_ERR_UNSUPPORTED, "okv_pages_copy: %d entries, %d pages (at most 2^30 each)", n,
              num_pages);
  if (n == 0) return OKV_OK;
  for (int lo = 0; lo < num_buffers; lo += kBuffersPerLaunch) {
    const int m = num_buffers - lo < kBuffersPerLaunch ? num_buffers - lo : kBuffersPerLaunch;
    hipLaunchKernelGGL(pages_copy_kernel, dim3(copy_blocks(n, m), m), dim3(256), 0, (hipStream_t)stream, take(host_buffers, lo, m),
                       num_pages, src, dst, count, n);
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
  rc = check_ws(pool, 0, ws, ws_bytes);
  if (rc) return rc;
  const PagesWs w = carve(pool, 0, ws);
  hipLaunchKernelGGL(pages_compact_plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, *pool, refs_out, used_out, w);
  for (int lo = 0; lo == 0 || lo < num_buffers; lo += kBuffersPerLaunch) {
    const int m = num_buffers - lo < kBuffersPerLaunch ? num_buffers - lo : kBuffersPerLaunch, table = lo == 0;
    const uint32_t blocks = copy_blocks(pool->num_pages / 2 > pool->num_seqs ? pool->num_pages / 2 : pool->num_seqs, m + table);
    hipLaunchKernelGGL(pages_compact_apply, dim3(blocks, m + table), dim3(256), 0, (hipStream_t)stream, *pool, table_out,
                       table_out_stride, w, take(host_buffers, lo, m), table);
  }
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

}  // extern "C"
