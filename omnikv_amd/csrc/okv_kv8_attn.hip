// Decode attention over the 8-bit K/V cache: okv_kv8_dense_attn, okv_kv8_sparse_attn.
//
// out = sum_t p_t v_t, p_t = exp(s q.k_t - m) / sum exp(...), with k_t and v_t codes times a scale per block: the K scale
// multiplies the logit, the V scale the probability, and the codes themselves go through the matrix cores as they are
// (every code of either format is exact in 16 bits).
//
// A launch of splits (each workgroup a share of one request's rows for one kv head or two: running maximum,
// sum and output of a softmax over its rows), then one launch that joins the shares and finishes the
// filter layer's scores.  Short requests take one launch (kv8_plan).
#include <math.h>
#include <string.h>

#include <algorithm>

#include "okv_kv8.h"

namespace okv {

constexpr int kMaxGroup = 8;
constexpr int kMaxHeads = 256;
constexpr int kGatherResident = 3;  // workgroups of the gather mode that a CU holds (160 VGPRs; capped for four it spills: 19.4 against 13.2 us at 8781 rows)

struct Kv8Attn {
  okv_kv8_cache_t c;
  const void* q;
  int32_t hq, group;
  float scale;
  // rows: dense [0, lens[b]), sparse idx[b][0 .. lens[b]) then the tail
  const int32_t* lens;
  int32_t max_len;
  int32_t sparse, slots;
  const int32_t* idx;
  int64_t idx_stride;
  const void* late[2];  // 16-bit rows behind the codes: the tail, or the open buffers
  int64_t late_token_stride, late_head_stride, late_batch_stride;
  const int32_t* tail_lens;
  int32_t max_tail_len;
  const int32_t* score_lens;
  int32_t max_score_len;
  // partial results
  float* part_o;    // [shares][Hq][128]
  float* part_lse;  // [shares][Hq], log2 domain; -inf: no row took part
  float* logits;    // [batch][logit_heads][logits_stride], natural units
  int64_t logits_stride;
  int32_t batch;
  float inv_target, inv_fine;  // 1 / full shares that fit next to the requests' last, short ones (half a share each)
  int32_t most_rows;  // of a share (its logits are staged in LDS)
  int32_t items;      // shares the grid and the partial results have room for
  int32_t least_rows;
  int32_t pair;       // two kv heads to a wave (NH 2)
  int32_t fine;       // shares of a batch longer than this are cut in three; 0: not
  int32_t direct;     // waves per workgroup where one share per request writes the output itself, without a second launch; 0: not
  int32_t fold;         // raw scores: the q heads of a kv head are folded by the split (1 max, 2 sum): one logits row per kv head
  int32_t logit_heads;  // rows of `logits` per request
  int32_t lds_scales;   // floats before the scale staging of the gather mode
  int32_t page_shift, block_shift;  // log2; page_shift -1: the page size is no power of two
  // outputs
  void* out;
  float* scores;
  int64_t score_stride;
  int32_t head_reduce, normalise;
};

__device__ __forceinline__ int clamp_len(const int32_t* lens, int b, int most) {
  const int n = lens ? lens[b] : most;
  return n < 0 ? 0 : n > most ? most : n;
}
__device__ __forceinline__ int kv8_score_len(const Kv8Attn& a, int b, int len) {
  const int s = a.max_score_len ? clamp_len(a.score_lens, b, a.max_score_len) : 0;
  return s < len ? s : len;
}

// ---------------------------------------------------------------- shares
// The rows of all requests are cut into shares of equal length, worked out on the device from the lengths as they are: a
// ragged batch, or a length far below its bound, leaves no workgroup idle.  Every wave that needs the
// cut works it out by itself (a lane per request), so nothing waits for it.
struct Share {
  int b;       // request
  int L, A;    // its rows, and how many of them are scored
  int main_len;
  int rows;    // rows of a share
  int index;   // this share among the request's
  int first;   // the request's first share among all
  int count;   // shares of the request
};


// inclusive prefix sum over the wave
__device__ __forceinline__ int lane_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 of a row to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
  return x;
}
__device__ __forceinline__ int share_rows(int total, const Kv8Attn& a) {
  // (less than one off where it is not cut to most_rows anyway: at or above total / target)
  uint32_t r = ((uint32_t)((float)total * a.inv_target) + 64) & ~63u;
  if (a.fine && r > (uint32_t)a.fine) r = max(((uint32_t)((float)total * a.inv_fine) + 64) & ~63u, (uint32_t)a.fine);
  return r < (uint32_t)a.least_rows ? a.least_rows : r > (uint32_t)a.most_rows ? a.most_rows : (int)r;
}
// x / rows, rounded up: quotients below 2^16 from a product with the reciprocal, put right by one step
__device__ __forceinline__ int shares_up(int x, int rows) {
  if (x <= 0) return 0;
  int q = (int)((float)(x - 1) * __builtin_amdgcn_rcpf((float)rows));
  const int r = x - 1 - q * rows;
  q += r >= rows ? 1 : r < 0 ? -1 : 0;
  return q + 1;
}
// The scored rows [0, A) and the rest [A, L) are cut separately: no share holds both.
__device__ __forceinline__ int shares_of(int rows, int A, int L) { return shares_up(A, rows) + shares_up(L - A, rows); }

__device__ __forceinline__ void request_lens(const Kv8Attn& a, int b, int* main_len, int* L, int* A) {
  *main_len = clamp_len(a.lens, b, a.max_len);
  *L = *main_len + (a.max_tail_len ? clamp_len(a.tail_lens, b, a.max_tail_len) : 0);
  *A = kv8_score_len(a, b, *main_len);
}

// The share `item` (false: there is none), or with item < 0 the shares of request `request`.
template <bool DIRECT>
__device__ __forceinline__ bool find_share(const Kv8Attn& a, int item, int request, Share* s) {
  const int lane = threadIdx.x & 63;
  if (DIRECT) {
    const int b = item;
    if (b >= a.batch) return false;
    request_lens(a, b, &s->main_len, &s->L, &s->A);
    s->main_len = __builtin_amdgcn_readfirstlane(s->main_len);
    s->L = __builtin_amdgcn_readfirstlane(s->L);
    s->b = b;
    s->index = s->first = 0;
    s->rows = max(s->L, 1);
    return true;
  }
  if (a.batch == 1) {
    request_lens(a, 0, &s->main_len, &s->L, &s->A);
    s->main_len = __builtin_amdgcn_readfirstlane(s->main_len);
    s->L = __builtin_amdgcn_readfirstlane(s->L);
    s->A = __builtin_amdgcn_readfirstlane(s->A);
    s->rows = __builtin_amdgcn_readfirstlane(share_rows(s->L, a));
    s->b = 0;
    s->first = 0;
    s->index = item;
    s->count = shares_of(s->rows, s->A, s->L);
    return item < s->count;
  }
  int main_len = 0, L = 0, A = 0, total = 0;
  for (int base = 0; base < a.batch; base += 64) {
    main_len = L = A = 0;
    if (base + lane < a.batch) request_lens(a, base + lane, &main_len, &L, &A);
    total += __builtin_amdgcn_readlane(lane_scan(L), 63);
  }
  s->rows = __builtin_amdgcn_readfirstlane(share_rows(total, a));
  int before = 0;
  for (int base = 0; base < a.batch; base += 64) {
    if (a.batch > 64) {
      main_len = L = A = 0;
      if (base + lane < a.batch) request_lens(a, base + lane, &main_len, &L, &A);
    }
    const int n = shares_of(s->rows, A, L);
    const int x = lane_scan(n);
    const uint64_t hit = __ballot(item >= 0 ? before + x > item : base + lane == request);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      s->b = base + at;
      s->main_len = __builtin_amdgcn_readlane(main_len, at);
      s->L = __builtin_amdgcn_readlane(L, at);
      s->A = __builtin_amdgcn_readlane(A, at);
      s->count = __builtin_amdgcn_readlane(n, at);
      s->first = before + __builtin_amdgcn_readlane(x, at) - s->count;
      s->index = item - s->first;
      return true;
    }
    before += __builtin_amdgcn_readlane(x, 63);
  }
  return false;
}

// ---------------------------------------------------------------- matrix-core pieces
__device__ __forceinline__ f32x2_t unpack_pair(const BF16*, uint32_t x) {
  return f32x2_t{__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)};
}
__device__ __forceinline__ f32x2_t unpack_pair(const F16*, uint32_t x) {
  const f16x2_t h = __builtin_bit_cast(f16x2_t, x);
  return f32x2_t{(float)h.x, (float)h.y};
}

// bytes 2H and 2H+1 of x -> a dword of two 16-bit elements; every code is exact in both types
template <int H>
__device__ __forceinline__ uint32_t decode_pair(E4M3, const BF16*, uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, H != 0));
}
template <int H>
__device__ __forceinline__ uint32_t decode_pair(E4M3, const F16*, uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, H != 0));
}
template <int H, typename T>
__device__ __forceinline__ uint32_t decode_pair(I8, const T*, uint32_t x) {
  return pack_pair((const T*)nullptr, (float)(int8_t)(x >> (16 * H)), (float)(int8_t)(x >> (16 * H + 8)));
}

typedef __attribute__((ext_vector_type(4))) short s16x4_t;
// D(16x16 fp32) += A(16 x 16) . B(16 x 16) in bf16: four elements of the contraction per lane
__device__ __forceinline__ f32x4_t mfma16k16(uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, make_uint2(a0, a1)),
                                                   __builtin_bit_cast(s16x4_t, make_uint2(b0, b1)), c, 0, 0, 0);
}

// Four 16-bit elements of V as the B operand next to probabilities in bf16: bfloat16's as they are, float16's in two parts,
// the nearest bf16 and the rest, exact together (11 bits = 8 + 3; bf16 has the range).  (Probabilities in float16, whose
// smallest step is 2^-24, lose what is below 2^-25 of the largest.)
template <typename T> constexpr bool kTwoParts = false;
template <> constexpr bool kTwoParts<F16> = true;
__device__ __forceinline__ uint4 bf16_rows(const BF16*, uint32_t a, uint32_t b) { return make_uint4(a, b, 0, 0); }
__device__ __forceinline__ uint4 bf16_rows(const F16* f, uint32_t a, uint32_t b) {
  const BF16* bf = nullptr;
  const f32x2_t va = unpack_pair(f, a), vb = unpack_pair(f, b);
  const uint32_t ha = pack_pair(bf, va.x, va.y), hb = pack_pair(bf, vb.x, vb.y);
  const f32x2_t ua = unpack_pair(bf, ha), ub = unpack_pair(bf, hb);
  return make_uint4(ha, hb, pack_pair(bf, va.x - ua.x, va.y - ua.y), pack_pair(bf, vb.x - ub.x, vb.y - ub.y));
}

// lanes 8..15 (MASK 0xC) or 0..7 (MASK 0x3) of every 16-lane row take `from` of the lane eight away, the others keep `own`
template <int MASK>
__device__ __forceinline__ uint32_t take8(uint32_t own, uint32_t from) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)own, (int)from, 0x128, 0xf, MASK, false);
}
// value of lane H of the caller's 16-lane row
template <int H>
__device__ __forceinline__ float row_lane(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x150 + H, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp_f(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
// over the four lane rows (lanes l, l^16, l^32, l^48), left in all of them
__device__ __forceinline__ float rows_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// `bytes` bytes at p as a buffer: what lies beyond them reads as zero and is not fetched, and the loads take a lane's 32-bit
// offset as it is, so that the loop computes no addresses per lane.  (A lane's address registers, taken from those of loads
// under way, would make the next tile's loads wait for this one's.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t as_buffer(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x27000);
}
__device__ __forceinline__ uint4 buffer16(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
  const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 2);  // 2: non-temporal
  return make_uint4(v.x, v.y, v.z, v.w);
}

// What is read at the same address by the whole wave and written by nobody meanwhile, as a scalar load: among the vector
// loads, which come back in order, it would have to wait for the rows asked for before it (sixteen requests of 8K..32K tokens
// in a pool, with scores: 154.6 -> 143.5 us; 131073 tokens with scores 57.7 -> 57.3).
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

enum { kContiguous = 0, kPaged = 1, kGather = 2 };

// A wave's 32 rows as lane l = 16j + m holds them: load i has K row 8i + (m & 7), chunk j + 4(m >> 3) of sixteen bytes, and
// V row 16(i / 2) + 4j + 2(i % 2) + (m >> 3), chunk m & 7; every load covers eight whole 128-byte rows.
struct Kv8Tile {
  uint4 k[4], v[4];
  float ks[2], vs[2];  // dense: scales of rows 0-15 and 16-31; gather: ks[0] alone, see load()
  uint32_t ok;   // dense: bit s = page of rows 16s.. lies in the pool; gather: this lane's own row (l % 32) takes part
};
struct Kv8Rows {
  int page[2];         // paged
  int k[4], v[4], s;   // gather: index entries
};

// A workgroup per share and kv head (or pair of them), W waves that take 32-row tiles in turn.
//
// Bound by the codes' bytes: every row is read once, in whole 128-byte lines, a tile in flight while the one before is
// consumed.  One launch, eight kv heads: 450001 tokens of int8 (922 MB) 143 us = 6.4 TB/s, 131073 of e4m3 (269 MB) 44 us = 6.1,
// with scores 52 (16.8 MB of logits are written besides), sixteen requests of 8K..32K tokens in a pool of 16-token pages (608 MB) 114 us =
// 5.3.  With the arithmetic replaced by xors the same loads take as long (142, 51 with scores, 118).  Through an index, a
// wave has one or two tiles and the round trips (length, index, rows, write) bound it: 8781 rows of 131072 11.1 us, 9.6 for the
// loads alone; 19854 rows of sixteen requests 17.8.  Row loads are non-temporal: 149 against 167 us at 450001 tokens, and as
// much better through an index (23.2 against 24.5) unless the rows lie in the last-level cache already.
//
// q.K^T: the tile's codes become 16-bit elements (exact) and are the A operand of v_mfma_f32_16x16x32: lane 16j + m
// holds row m, elements 16j .. +16 and 64 + 16j .. +16.  Loading that directly would touch 16 rows x 64 bytes per
// instruction; the loads take whole 128-byte rows instead, and lanes m and m^8 exchange halves (one DPP move per dword).
// The kv head's q heads are columns 0..7 of B (padded by repeating the last) and AGAIN columns 8..15.
// P.V: the logits come out as lane (column m, rows 4j .. +4), which is the A operand's layout of P.  Columns 0..7
// carry bf16(p), columns 8..15 the rest p - bf16(p): the spare half of the matrix instruction gives P 16 bits.  The V
// scale of a row is folded into its p; V's codes, exact in bf16, are the B operand: a lane's eight rows x
// eight elements, turned by byte permutes as they are decoded.
// Scales of K are applied to the fp32 logits.  One running maximum per q head and wave; the waves meet in LDS.
//
// NH 2 (paged, an even number of kv heads, a token's heads next to each other): a wave takes sixteen rows of two neighbouring
// heads instead of 32 rows of one; what is said of the upper sixteen rows then holds for the second head.
// 128-byte pieces a token's row apart reach memory less well than 256-byte ones: 288000 tokens of one request
// 122.3 -> 113.2 us, sixteen of 18000 each 121.1 -> 117.6; one descriptor for both heads 119.5 -> 117.9
// (sixteen of 8K..32K).  Through an index it made no difference (22.1, 22.6).
template <typename T, typename F, int MODE, bool LOGITS, int NH, bool DIRECT, int W>
__global__ __launch_bounds__(64 * W, MODE == kGather && W == 4 ? kGatherResident : 2) void kv8_split(Kv8Attn a) {
  extern __shared__ float lds[];
  constexpr int TR = 32 / NH, kStep = W * TR;  // rows of a tile, and between a wave's tiles
  const okv_kv8_cache_t& c = a.c;
  if constexpr (MODE != kPaged) {  // one batch of scalar loads instead of a round trip before each first use (the paged mode's
    // page descriptors leave too few scalar registers for that: 131 against 121 us)
    fetch_now(c.k_codes); fetch_now(c.v_codes); fetch_now(c.k_scale); fetch_now(c.v_scale); fetch_now(c.token_stride);
    fetch_now(c.head_stride); fetch_now(c.batch_stride); fetch_now(c.scale_block_stride); fetch_now(c.scale_head_stride);
    fetch_now(c.scale_batch_stride); fetch_now(a.q); fetch_now(a.lens); fetch_now(a.idx); fetch_now(a.idx_stride);
    fetch_now(a.batch); fetch_now(a.inv_target); fetch_now(a.max_len); fetch_now(a.max_tail_len); fetch_now(a.tail_lens);
    fetch_now(a.late[0]); fetch_now(a.late[1]); fetch_now(a.late_token_stride); fetch_now(a.late_head_stride);
    fetch_now(a.late_batch_stride);
  }
  const int G = a.group;
  // workgroups go to the XCDs round-robin: the kv heads of a share run on one XCD, one after the other, so that rows
  // stored head by head next to each other (pools) are fetched together
  const int turn = blockIdx.x >> 3, groups = c.num_kv_heads / NH, g = turn % groups * NH;
  Share sh;
  if (!find_share<DIRECT>(a, (int)((turn / groups) * 8 + (blockIdx.x & 7)), 0, &sh)) return;
  const int b = sh.b, main_len = sh.main_len, L = sh.L, A = LOGITS ? sh.A : 0;
  int begin, end;
  {
    const int nA = LOGITS ? shares_up(A, sh.rows) : 0;
    begin = sh.index < nA ? sh.index * sh.rows : A + (sh.index - nA) * sh.rows;
    end = min(begin + sh.rows, sh.index < nA ? A : L);
  }
  if (begin >= end && !DIRECT) return;  // (a request without rows gets its zeros below)
  // rows [0, closed) are codes, the rest 16-bit rows: the open block, or the tail
  const int closed = a.sparse || !c.open_k ? main_len : main_len >> a.block_shift << a.block_shift;
  const int main_end = min(end, closed);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, j = lane >> 4, m8 = m16 & 7, hi8 = m16 >> 3;

  uint4 qf[NH][4];
#pragma unroll
  for (int s = 0; s < NH; ++s) {
    const int h = m8 < G ? m8 : G - 1;
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(b * a.hq + (g + s) * G + h) * kD + 16 * j;
    qf[s][0] = *reinterpret_cast<const uint4*>(qp);
    qf[s][1] = *reinterpret_cast<const uint4*>(qp + 8);
    qf[s][2] = *reinterpret_cast<const uint4*>(qp + 64);
    qf[s][3] = *reinterpret_cast<const uint4*>(qp + 72);
  }

  const uint32_t ts = (uint32_t)c.token_stride;
  const int64_t head = (int64_t)g * c.head_stride + (MODE == kPaged || c.page_table ? 0 : (int64_t)b * c.batch_stride);
  const int64_t shead = (int64_t)g * c.scale_head_stride + (MODE == kPaged || c.page_table ? 0 : (int64_t)b * c.scale_batch_stride);
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(c.k_codes) + head;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(c.v_codes) + head;
  const float* ksb = c.k_scale + shead;
  const float* vsb = c.v_scale + shead;
  const uint32_t kcol = 16 * (j + 4 * hi8), vcol = 16 * m8;
  uint32_t koff[4], voff[4];  // of the lane's rows in a tile
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t second = NH == 2 && i >= 2 ? (uint32_t)c.head_stride : 0;  // the pair's other head
    koff[i] = (uint32_t)(8 * (MODE == kPaged ? i & 1 : i) + m8) * ts + kcol + second;
    voff[i] = (uint32_t)((MODE == kPaged ? 0 : 16 * (i >> 1)) + 4 * j + 2 * (i & 1) + hi8) * ts + vcol + second;
  }
  const int last = main_end - 1;
  const int32_t* table = c.page_table + (int64_t)b * c.page_table_stride;
  const int32_t* idx = a.idx + (int64_t)b * a.idx_stride;
  const uint32_t room = MODE != kGather ? 0 : a.slots ? (uint32_t)(c.num_pages * c.page_size) : (uint32_t)kv8_room(c);

  auto page_of = [&](int t) -> int { return a.page_shift >= 0 ? t >> a.page_shift : t / c.page_size; };
  auto slot_of = [&](int t) -> int { return a.page_shift >= 0 ? t & (c.page_size - 1) : t % c.page_size; };
  // ---- what has to be known of a tile's rows before they can be addressed
  auto rows_of = [&](int t, Kv8Rows& r) {
    if (MODE == kPaged) {
#pragma unroll
      for (int s = 0; s < 2 / NH; ++s) r.page[s] = scalar_load(table + page_of(min(t + 16 * s, last)));
    } else if (MODE == kGather) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        r.k[x] = idx[min(t + 8 * x + m8, last)];
        r.v[x] = idx[min(t + 16 * (x >> 1) + 4 * j + 2 * (x & 1) + hi8, last)];
      }
      r.s = idx[min(t + (lane & 31), last)];
    }
  };
  auto load = [&](int t, const Kv8Rows& r, Kv8Tile& x) {
    if (MODE == kContiguous) {
      const int n = min(32, main_end - t);  // rows of the tile; none: past the last tile
      const uint32_t bytes = n > 0 ? (uint32_t)(n - 1) * ts + kD : 0;
      const __amdgpu_buffer_rsrc_t kr = as_buffer(kb + (int64_t)t * ts, bytes), vr = as_buffer(vb + (int64_t)t * ts, bytes);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.k[i] = buffer16(kr, koff[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = buffer16(vr, voff[i]);
#pragma unroll
      for (int s = 0; s < 2; ++s) {  // the same four bytes for every lane; behind the end the last row's, unused
        const int64_t so = (int64_t)(min(t + 16 * s, last) >> a.block_shift) * c.scale_block_stride;
        x.ks[s] = scalar_load(ksb + so);
        x.vs[s] = scalar_load(vsb + so);
      }
      x.ok = 3;
    } else if (MODE == kPaged) {
      // sixteen rows lie in one page: those behind the end are in it too, and a scale is always there to be read
      x.ok = 0;
#pragma unroll
      for (int s = 0; s < 2 / NH; ++s) {
        const int u = t + 16 * s, n = min(16, main_end - u), page = r.page[s];
        const bool in = (uint32_t)page < (uint32_t)c.num_pages;
        const int64_t p = in ? page : 0;
        const int slot = slot_of(u);
        const int64_t base = p * c.page_stride + (int64_t)slot * ts;
        const uint32_t bytes = in && n > 0 ? (uint32_t)(n - 1) * ts + kD + (NH == 2 ? (uint32_t)c.head_stride : 0) : 0;
        const __amdgpu_buffer_rsrc_t kr = as_buffer(kb + base, bytes), vr = as_buffer(vb + base, bytes);
#pragma unroll
        for (int i = 2 * s; i < 2 * s + 2 * NH; ++i) x.k[i] = buffer16(kr, koff[i]);
#pragma unroll
        for (int i = 2 * s; i < 2 * s + 2 * NH; ++i) x.v[i] = buffer16(vr, voff[i]);
        const int64_t so = p * c.scale_page_stride + (int64_t)(slot >> a.block_shift) * c.scale_block_stride;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          x.ks[s + h] = scalar_load(ksb + so + h * c.scale_head_stride);
          x.vs[s + h] = scalar_load(vsb + so + h * c.scale_head_stride);
          x.ok |= in ? 1u << (s + h) : 0u;
        }
      }
    } else {
      // an entry outside the request's room is read as row 0 and takes no part
      auto at = [&](int t_, int64_t* row, int64_t* scale) -> bool {
        bool in = (uint32_t)t_ < room;
        const int tt = in ? t_ : 0;
        if (c.page_table && !a.slots) {
          const int pg = table[page_of(tt)], slot = slot_of(tt);
          in = in && (uint32_t)pg < (uint32_t)c.num_pages;
          const int64_t p = (uint32_t)pg < (uint32_t)c.num_pages ? pg : 0;
          *row = p * c.page_stride + (int64_t)slot * ts;
          *scale = p * c.scale_page_stride + (int64_t)(slot >> a.block_shift) * c.scale_block_stride;
        } else {
          *row = (int64_t)tt * ts;
          *scale = (int64_t)(tt >> a.block_shift) * c.scale_block_stride;
        }
        return in;
      };
      int64_t row, scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at(r.k[i], &row, &scale);
        x.k[i] = load_stream16(kb + row + kcol);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at(r.v[i], &row, &scale);
        x.v[i] = load_stream16(vb + row + vcol);
      }
      x.ok = at(r.s, &row, &scale);  // lanes 0..31: the K scales of rows l, 32..63: the V scales of rows l - 32
      x.ks[0] = (lane < 32 ? ksb : vsb)[scale];
    }
  };

  float m[NH];          // running maximum of q head m8's logits, times log2(e), over the wave's rows
  float l[NH];          // sum of exponentials over the rows of lane row j, relative to m
  f32x4_t acc[NH][8];   // acc[.][e][i]: element 16 m8 + 8 hi8 + e of q head (4j + i) % 8; j < 2: from bf16(p), else the rest
#pragma unroll
  for (int s = 0; s < NH; ++s) {
    m[s] = -INFINITY;
    l[s] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[s][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const bool scored = LOGITS && begin < A;
  float* slog = lds;  // [NH][G, or 1 when the heads are folded][rows]: handed over at the end

  auto raise_max = [&](int n, float top) {  // n: of the wave's kv heads
    if (__ballot(top > m[n]) == 0ull) return;
    const float mn = rows_max(fmaxf(top, m[n]));
    const float al = __builtin_amdgcn_exp2f(m[n] - (mn == -INFINITY ? 0.f : mn));
    l[n] *= al;
    m[n] = mn;
    const float lo[4] = {row_lane<0>(al), row_lane<1>(al), row_lane<2>(al), row_lane<3>(al)};
    const float hi[4] = {row_lane<4>(al), row_lane<5>(al), row_lane<6>(al), row_lane<7>(al)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = (j & 1) ? hi[i] : lo[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[n][e][i] *= f;
    }
  };
  auto stage_logits = [&](int n, int row, const float (&v)[4]) {  // natural units, rows row .. +4
    float o[4] = {v[0], v[1], v[2], v[3]};
    if (a.fold) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = a.fold == 2 && m8 >= G ? 0.f : o[i];
        const float x1 = dpp_f<0xB1>(x);  // lane ^ 1
        x = a.fold == 1 ? fmaxf(x, x1) : x + x1;
        const float x2 = dpp_f<0x4E>(x);  // lane ^ 2
        x = a.fold == 1 ? fmaxf(x, x2) : x + x2;
        const float x4 = dpp_f<0x141>(x);  // lane 7 - m8: the other quad, each uniform by now
        o[i] = a.fold == 1 ? fmaxf(x, x4) : x + x4;
      }
    }
    if (m16 < (a.fold ? 1 : G))
      *reinterpret_cast<float4*>(slog + (n * (a.fold ? 1 : G) + m16) * sh.rows + (row - begin)) = make_float4(o[0], o[1], o[2], o[3]);
  };
  // a probability in two bf16 parts: this lane's part of four of them
  auto split_p = [&](const float (&p)[4], uint32_t* out) {
    const BF16* ty = nullptr;
    const uint32_t h0 = pack_pair(ty, p[0], p[1]), h1 = pack_pair(ty, p[2], p[3]);
    const f32x2_t u0 = unpack_pair(ty, h0), u1 = unpack_pair(ty, h1);
    out[0] = hi8 ? pack_pair(ty, p[0] - u0.x, p[1] - u0.y) : h0;
    out[1] = hi8 ? pack_pair(ty, p[2] - u1.x, p[3] - u1.y) : h1;
  };

  auto compute = [&](int t, Kv8Tile& x, float* sstage) {
    float ks[2][4], vs[2][4];
    bool whole = t >= begin && t + TR <= main_end;
    if (MODE == kGather) {
      // every lane has the scale of one row: the wave's 256 bytes of LDS hand the rows' four to their lane row
      const bool okl = x.ok != 0;
      sstage[lane] = okl ? x.ks[0] : 0.f;
      const uint64_t oks = __ballot(okl);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float4 kk = *reinterpret_cast<const float4*>(sstage + 16 * s + 4 * j);
        const float4 vv = *reinterpret_cast<const float4*>(sstage + 32 + 16 * s + 4 * j);
        ks[s][0] = kk.x; ks[s][1] = kk.y; ks[s][2] = kk.z; ks[s][3] = kk.w;
        vs[s][0] = vv.x; vs[s][1] = vv.y; vs[s][2] = vv.z; vs[s][3] = vv.w;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (oks != ~0ull) {  // wave-uniform: some entry is padding
        whole = false;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!((oks >> (16 * (i >> 1) + 4 * j + 2 * (i & 1) + hi8)) & 1)) x.v[i] = make_uint4(0, 0, 0, 0);
        x.ok = (uint32_t)oks;
      } else {
        x.ok = 0xffffffffu;
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ks[s][i] = x.ks[s];
          vs[s][i] = x.vs[s];
        }
      }
      if (MODE == kPaged && x.ok != 3) {
        whole = false;
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (!((x.ok >> s) & 1)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[s][i] = 0.f;  // (its codes have come as zeros)
          }
      }
    }
    float p[2][4];
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4_t S = {0.f, 0.f, 0.f, 0.f};
      const uint4 k0 = x.k[2 * s], k1 = x.k[2 * s + 1];
      const uint32_t lo[4] = {take8<0xC>(k0.x, k1.x), take8<0xC>(k0.y, k1.y), take8<0xC>(k0.z, k1.z), take8<0xC>(k0.w, k1.w)};
      const uint32_t up[4] = {take8<0x3>(k1.x, k0.x), take8<0x3>(k1.y, k0.y), take8<0x3>(k1.z, k0.z), take8<0x3>(k1.w, k0.w)};
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const uint4 x0 = make_uint4(decode_pair<0>(F{}, (const T*)nullptr, lo[2 * f]), decode_pair<1>(F{}, (const T*)nullptr, lo[2 * f]),
                                    decode_pair<0>(F{}, (const T*)nullptr, lo[2 * f + 1]), decode_pair<1>(F{}, (const T*)nullptr, lo[2 * f + 1]));
        S = mfma16((const T*)nullptr, x0, qf[NH == 1 ? 0 : s][f], S);
      }
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const uint4 x1 = make_uint4(decode_pair<0>(F{}, (const T*)nullptr, up[2 * f]), decode_pair<1>(F{}, (const T*)nullptr, up[2 * f]),
                                    decode_pair<0>(F{}, (const T*)nullptr, up[2 * f + 1]), decode_pair<1>(F{}, (const T*)nullptr, up[2 * f + 1]));
        S = mfma16((const T*)nullptr, x1, qf[NH == 1 ? 0 : s][2 + f], S);
      }
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = S[i] * (ks[s][i] * a.scale);
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = t + (NH == 1 ? 16 * s : 0) + 4 * j + i;
          const bool in = r >= begin && r < main_end &&
                          (MODE == kContiguous || ((x.ok >> (MODE == kPaged ? s : 16 * s + 4 * j + i)) & 1));
          v[i] = in ? v[i] : -INFINITY;
          vs[s][i] = in ? vs[s][i] : 0.f;
        }
      }
      const int row0 = t + (NH == 1 ? 16 * s : 0);
      if (scored && row0 < main_end) stage_logits(NH == 1 ? 0 : s, row0 + 4 * j, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[s][i] = v[i] * kLog2e;
        top[s] = fmaxf(top[s], p[s][i]);
      }
    }
    if (NH == 1) {
      raise_max(0, fmaxf(top[0], top[1]));
    } else {
#pragma unroll
      for (int s = 0; s < NH; ++s) raise_max(s, top[s]);
    }
    uint32_t pa[4];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int n = NH == 1 ? 0 : s;
      const float neg = m[n] == -INFINITY ? 0.f : -m[n];
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(p[s][i] + neg);
        l[n] += e;
        w[i] = e * vs[s][i];
      }
      split_p(w, pa + 2 * s);
    }
    const uint4 pf = make_uint4(pa[0], pa[1], pa[2], pa[3]);
    // lane m keeps eight elements of its lane row's four rows of either sixteen
    uint32_t lo[4][2], up[4][2];  // [row 4j + i][dword] of the lower and the upper sixteen
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lo[2 * i][0] = take8<0xC>(x.v[i].x, x.v[i].z);
      lo[2 * i][1] = take8<0xC>(x.v[i].y, x.v[i].w);
      lo[2 * i + 1][0] = take8<0x3>(x.v[i].z, x.v[i].x);
      lo[2 * i + 1][1] = take8<0x3>(x.v[i].w, x.v[i].y);
      up[2 * i][0] = take8<0xC>(x.v[2 + i].x, x.v[2 + i].z);
      up[2 * i][1] = take8<0xC>(x.v[2 + i].y, x.v[2 + i].w);
      up[2 * i + 1][0] = take8<0x3>(x.v[2 + i].z, x.v[2 + i].x);
      up[2 * i + 1][1] = take8<0x3>(x.v[2 + i].w, x.v[2 + i].y);
    }
#pragma unroll
    for (int d = 0; d < 2; ++d) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // elements 4d + 2h, 4d + 2h + 1
        const uint32_t sel = h ? 0x07030602u : 0x05010400u;
        const uint32_t l01 = __builtin_amdgcn_perm(lo[1][d], lo[0][d], sel), l23 = __builtin_amdgcn_perm(lo[3][d], lo[2][d], sel);
        const uint32_t u01 = __builtin_amdgcn_perm(up[1][d], up[0][d], sel), u23 = __builtin_amdgcn_perm(up[3][d], up[2][d], sel);
        const BF16* bf = nullptr;
        const uint4 e0 = make_uint4(decode_pair<0>(F{}, bf, l01), decode_pair<0>(F{}, bf, l23), decode_pair<0>(F{}, bf, u01),
                                    decode_pair<0>(F{}, bf, u23));
        const uint4 e1 = make_uint4(decode_pair<1>(F{}, bf, l01), decode_pair<1>(F{}, bf, l23), decode_pair<1>(F{}, bf, u01),
                                    decode_pair<1>(F{}, bf, u23));
        const int e = 4 * d + 2 * h;
        if (NH == 1) {
          acc[0][e] = mfma16(bf, pf, e0, acc[0][e]);
          acc[0][e + 1] = mfma16(bf, pf, e1, acc[0][e + 1]);
        } else {
          acc[0][e] = mfma16k16(pf.x, pf.y, e0.x, e0.y, acc[0][e]);
          acc[0][e + 1] = mfma16k16(pf.x, pf.y, e1.x, e1.y, acc[0][e + 1]);
          acc[NH - 1][e] = mfma16k16(pf.z, pf.w, e0.z, e0.w, acc[NH - 1][e]);
          acc[NH - 1][e + 1] = mfma16k16(pf.z, pf.w, e1.z, e1.w, acc[NH - 1][e + 1]);
        }
      }
    }
  };

  float* sstage = lds + a.lds_scales + 64 * wave;
  {
    int t = (begin & ~(TR - 1)) + TR * wave;
    if (t < main_end) {
      const int t_last = t + (last - t) / kStep * kStep;
      Kv8Rows r0, r1;
      Kv8Tile x0, x1;
      rows_of(t, r0);
      if (MODE == kGather) {
        for (; t <= t_last; t += kStep) {
          load(t, r0, x0);
          rows_of(min(t + kStep, t_last), r0);
          compute(t, x0, sstage);
        }
      } else if (t == t_last) {
        load(t, r0, x0);
        compute(t, x0, sstage);
      } else {
        rows_of(t + kStep, r1);
        load(t, r0, x0);
        while (true) {  // tile t + kStep in flight while t is consumed; past the last one nothing is fetched.  The loads stay
          __builtin_amdgcn_sched_barrier(0);  // where they are: among the arithmetic they would wait for its data.
          load(t + kStep, r1, x1);
          rows_of(t + 2 * kStep, r0);
          __builtin_amdgcn_sched_barrier(0);
          compute(t, x0, sstage);
          t += kStep;
          if (t > t_last) break;
          __builtin_amdgcn_sched_barrier(0);
          load(t + kStep, r0, x0);
          rows_of(t + 2 * kStep, r1);
          __builtin_amdgcn_sched_barrier(0);
          compute(t, x1, sstage);
          t += kStep;
          if (t > t_last) break;
        }
      }
    }
  }

  // ---- 16-bit rows: sixteen per tile, K straight in the A operand's layout
  if (end > closed) {
    const int lo = max(begin, closed);
    const int64_t lts = a.late_token_stride;
    const int64_t lbase = (int64_t)b * a.late_batch_stride + (int64_t)g * a.late_head_stride;
    const T* ty = nullptr;
    const BF16* bf = nullptr;
    for (int t = lo + 16 * wave; t < end; t += 16 * W) {
      const int top_row = end - 1 - closed;  // rows counted from the first late one
#pragma unroll
      for (int n = 0; n < NH; ++n) {
      const T* lk = reinterpret_cast<const T*>(a.late[0]) + lbase + n * a.late_head_stride;
      const T* lv = reinterpret_cast<const T*>(a.late[1]) + lbase + n * a.late_head_stride;
      const T* kp = lk + (int64_t)min(t - closed + m16, top_row) * lts + 16 * j;
      const uint4 kf[4] = {*reinterpret_cast<const uint4*>(kp), *reinterpret_cast<const uint4*>(kp + 8),
                           *reinterpret_cast<const uint4*>(kp + 64), *reinterpret_cast<const uint4*>(kp + 72)};
      uint4 vf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vf[i] = *reinterpret_cast<const uint4*>(lv + (int64_t)min(t - closed + 4 * j + i, top_row) * lts + 16 * m8 + 8 * hi8);
      f32x4_t S = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < 4; ++f) S = mfma16(ty, kf[f], qf[n][f], S);
      float v[4], p[4], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = t + 4 * j + i < end ? S[i] * a.scale : -INFINITY;
      if (scored) stage_logits(n, t + 4 * j, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = v[i] * kLog2e;
        top = fmaxf(top, p[i]);
      }
      raise_max(n, top);
      const float neg = m[n] == -INFINITY ? 0.f : -m[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = __builtin_amdgcn_exp2f(p[i] + neg);
        l[n] += p[i];
      }
      uint32_t pa[2];
      split_p(p, pa);
      // the contraction's upper four rows are the same ones again, with what bf16 leaves of float16's V (bf16's: nothing)
      const uint4 pf = kTwoParts<T> ? make_uint4(pa[0], pa[1], pa[0], pa[1]) : make_uint4(pa[0], pa[1], 0, 0);
      const uint32_t r0[4] = {vf[0].x, vf[0].y, vf[0].z, vf[0].w}, r1[4] = {vf[1].x, vf[1].y, vf[1].z, vf[1].w};
      const uint32_t r2[4] = {vf[2].x, vf[2].y, vf[2].z, vf[2].w}, r3[4] = {vf[3].x, vf[3].y, vf[3].z, vf[3].w};
#pragma unroll
      for (int d = 0; d < 4; ++d) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t sel = h ? 0x07060302u : 0x05040100u;
          const uint4 e = bf16_rows(ty, __builtin_amdgcn_perm(r1[d], r0[d], sel), __builtin_amdgcn_perm(r3[d], r2[d], sel));
          acc[n][2 * d + h] = mfma16(bf, pf, e, acc[n][2 * d + h]);
        }
      }
      }
    }
  }

  // ---- a scored split hands its logits over, then LDS changes hands
  if (scored) {
    __syncthreads();
    const int nh = a.fold ? 1 : G;
    for (int h = 0; h < NH * nh; ++h) {
      float* dst = a.logits + (int64_t)(b * a.logit_heads + g * nh + h) * a.logits_stride + begin;
      const float* src = slog + h * sh.rows;
      for (int r = 4 * threadIdx.x; r < end - begin; r += 256 * W) {
        const float4 v = *reinterpret_cast<const float4*>(src + r);
        if (begin + r + 3 < end) {
          *reinterpret_cast<float4*>(dst + r) = v;
        } else {
          dst[r] = v.x;
          if (begin + r + 1 < end) dst[r + 1] = v.y;
          if (begin + r + 2 < end) dst[r + 2] = v.z;
        }
      }
    }
    __syncthreads();
  }

  // ---- the W waves meet
  constexpr int kCell = NH * kMaxGroup;
  float* sm = lds;                  // [W][NH][8] running maximum
  float* sl = lds + W * kCell;      // [W][NH][8] sum of exponentials
  float* so = lds + 2 * W * kCell;  // [W][NH G][128]
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    l[n] = rows_sum(l[n]);
    if (lane < kMaxGroup) {
      sm[wave * kCell + n * kMaxGroup + lane] = m[n];
      sl[wave * kCell + n * kMaxGroup + lane] = l[n];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[n][e][i]), __float_as_uint(acc[n][e][i]), false, false);
        acc[n][e][i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = 4 * j + i;
      if (j < 2 && h < G) {
        float4* dst = reinterpret_cast<float4*>(so + ((wave * NH + n) * G + h) * kD + 16 * m8 + 8 * hi8);
        dst[0] = make_float4(acc[n][0][i], acc[n][1][i], acc[n][2][i], acc[n][3][i]);
        dst[1] = make_float4(acc[n][4][i], acc[n][5][i], acc[n][6][i], acc[n][7][i]);
      }
    }
  }
  __syncthreads();
  for (int o = threadIdx.x; o < NH * G * kD; o += 64 * W) {
    const int h = o / kD, d = o % kD;  // q head of the workgroup's NH G
    const int cell = NH == 1 ? h : h < G ? h : kMaxGroup + h - G;
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < W; ++x) M = fmaxf(M, sm[x * kCell + cell]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float den = 0.f, num = 0.f;
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float f = __builtin_amdgcn_exp2f(sm[x * kCell + cell] - Ms);
      den = fmaf(sl[x * kCell + cell], f, den);
      num = fmaf(so[(x * NH * G + h) * kD + d], f, num);
    }
    // den 0: no row took part (a NaN among the logits leaves NaN)
    if (DIRECT) {
      store1(reinterpret_cast<T*>(a.out) + (int64_t)(b * a.hq + g * G + h) * kD + d, den == 0.f ? 0.f : num / den);
      continue;
    }
    const int64_t ph = (int64_t)(sh.first + sh.index) * a.hq + g * G + h;
    a.part_o[ph * kD + d] = den == 0.f ? 0.f : num / den;
    if (d == 0) a.part_lse[ph] = den == 0.f ? -INFINITY : Ms + log2f(den);
  }
}

// out = sum_s 2^(lse_s - m) out_s / sum_s 2^(lse_s - m) over the shares s of a request.  Blocks [0, Hq) of a request do that for
// one q head: 32 float4 columns x 8 share lanes, eight shares of a lane in flight (one column per thread and one share at a
// time took 26 us; sixteen in flight -0.15 us for one request, +0.85 for sixteen).  The other blocks
// finish 256 TPT scores each and work out the heads' normalisers themselves from the shares' partial
// log-sum-exps (a few KB), so that no block waits for another.  Bound by the launch and two round trips: 64 shares of 32 heads
// 4.4 us, with 131072 scores of 32 logits each (16.8 MB) 6.0.  Two scores to a thread where blocks of 512 are few enough to be on
// the chip at once, else four.
template <typename T, int TPT>
__global__ __launch_bounds__(256) void kv8_join(Kv8Attn a) {
  const int b = blockIdx.y, tid = threadIdx.x;
  Share sh;
  find_share<false>(a, -1, b, &sh);
  const int A = sh.A;
  constexpr int U = 8;
  if ((int)blockIdx.x < a.hq) {
    __shared__ float4 s_num[8][32];
    __shared__ float s_m[8], s_den[8];
    const int h = blockIdx.x, dq = tid & 31, sl = tid >> 5, ns = sh.count;
    const float* lse = a.part_lse + (int64_t)sh.first * a.hq + h;
    const float4* po = reinterpret_cast<const float4*>(a.part_o + ((int64_t)sh.first * a.hq + h) * kD) + dq;
    float m = -INFINITY, den = 0.f;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = sl; s0 < ns; s0 += 8 * U) {
      float x[U];
      float4 o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + 8 * u;
        x[u] = s < ns ? lse[(int64_t)s * a.hq] : -INFINITY;
        o[u] = s < ns ? po[(int64_t)s * a.hq * (kD / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, x[u]);
      const float ref = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - ref);
      den *= al;
      num = make_float4(num.x * al, num.y * al, num.z * al, num.w * al);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float f = __builtin_amdgcn_exp2f(x[u] - ref);
        den += f;
        num.x = fmaf(f, o[u].x, num.x);
        num.y = fmaf(f, o[u].y, num.y);
        num.z = fmaf(f, o[u].z, num.z);
        num.w = fmaf(f, o[u].w, num.w);
      }
      m = mn;
    }
    s_num[sl][dq] = num;
    if (dq == 0) {
      s_m[sl] = m;
      s_den[sl] = den;
    }
    __syncthreads();
    if (tid < kD) {
      float M = -INFINITY;
#pragma unroll
      for (int x = 0; x < 8; ++x) M = fmaxf(M, s_m[x]);
      const float ref = M == -INFINITY ? 0.f : M;
      const float* sn = reinterpret_cast<const float*>(&s_num[0][0]);
      float n = 0.f, d = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float f = __builtin_amdgcn_exp2f(s_m[x] - ref);
        n = fmaf(sn[x * kD + tid], f, n);
        d = fmaf(s_den[x], f, d);
      }
      store1(reinterpret_cast<T*>(a.out) + (int64_t)(b * a.hq + h) * kD + tid, d == 0.f ? 0.f : n / d);
    }
    return;
  }
  __shared__ float s_lse[kMaxHeads];
  const int t0 = ((blockIdx.x - a.hq) * 256 + tid) * TPT;
  if ((int)(blockIdx.x - a.hq) * 256 * TPT >= A) return;
  const bool soft = a.normalise == OKV_NORM_SOFTMAX, is_max = a.head_reduce == OKV_REDUCE_MAX;
  if (soft) {  // eight threads per head
    const int nA = shares_up(A, sh.rows), sub = tid & 7;
    for (int h0 = 0; h0 < a.hq; h0 += 32) {
      const int h = h0 + (tid >> 3);
      float m = -INFINITY, den = 0.f;
      if (h < a.hq) {
        const float* lse = a.part_lse + (int64_t)sh.first * a.hq + h;
        for (int s0 = sub; s0 < nA; s0 += 8 * U) {
          float x[U], mn = m;
#pragma unroll
          for (int u = 0; u < U; ++u) x[u] = s0 + 8 * u < nA ? lse[(int64_t)(s0 + 8 * u) * a.hq] : -INFINITY;
#pragma unroll
          for (int u = 0; u < U; ++u) mn = fmaxf(mn, x[u]);
          const float ref = mn == -INFINITY ? 0.f : mn;
          den *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
          for (int u = 0; u < U; ++u) den += __builtin_amdgcn_exp2f(x[u] - ref);
          m = mn;
        }
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const float m2 = __shfl_xor(m, o), d2 = __shfl_xor(den, o), mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
        den = den * __builtin_amdgcn_exp2f(m - ref) + d2 * __builtin_amdgcn_exp2f(m2 - ref);
        m = mn;
      }
      if (h < a.hq && sub == 0) s_lse[h] = m == -INFINITY ? 0.f : m + log2f(den);
    }
    __syncthreads();
  }
  if (t0 >= A) return;
  float acc[TPT];
#pragma unroll
  for (int i = 0; i < TPT; ++i) acc[i] = is_max ? -INFINITY : 0.f;
  const float* lg = a.logits + (int64_t)b * a.logit_heads * a.logits_stride + t0;
#pragma unroll 16
  for (int h = 0; h < a.logit_heads; ++h) {
    float v[TPT];  // the row ends at a multiple of 64: reading past A stays inside it
    if constexpr (TPT == 4) {
      const float4 x = *reinterpret_cast<const float4*>(lg + (int64_t)h * a.logits_stride);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(lg + (int64_t)h * a.logits_stride);
      v[0] = x.x; v[1] = x.y;
    }
    const float lse = soft ? s_lse[h] : 0.f;
#pragma unroll
    for (int i = 0; i < TPT; ++i) {
      const float x = soft ? __builtin_amdgcn_exp2f(fmaf(v[i], kLog2e, -lse)) : v[i];
      acc[i] = is_max ? fmaxf(acc[i], x) : acc[i] + x;
    }
  }
  float* sp = a.scores + (int64_t)b * a.score_stride + t0;
#pragma unroll
  for (int i = 0; i < TPT; ++i)
    if (t0 + i < A) sp[i] = acc[i];
}

// ---------------------------------------------------------------- host side
static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// How a call is run, from its sizes and layout alone.
struct Kv8Plan {
  int direct;  // waves of a workgroup, or 0
  bool pair;
  int target, most, least, items;
  bool fine;
};

// direct: a share per request, and no second launch: where requests are short, and longer ones where there are many, the
// rows a wave then takes one after the other cost less than the join and the round trip through memory.  Eight waves to a
// workgroup as long as every workgroup has a CU of its own, else four.  Measured (bf16, int8, eight kv heads; one launch against
// two, us): contiguous 1 x 333 rows 6.5 / 7.4, 1 x 512 7.7 / 7.2, 4 x 512 7.8 / 8.3, 4 x 768 9.5 / 8.3, 16 x 1024 11.8 / 15.0,
// 64 x 1536 32.4 / 44.2; through an index 1 x 333 6.9 / 7.9, 1 x 512 8.2 / 8.1, 8 x 512 8.9 / 9.3, 8 x 768 11.9 / 10.9,
// 16 x 768 13.0 / 14.0, 16 x 1536 20.2 / 19.4, 64 x 1536 38.0 / 44.3.  Four waves: 1 x 333 7.1; eight at 64 x 512 16.5 for 12.6.
// Requests of unequal lengths gain less, since the longest decides: hence no more than 2048.
//
// Else one round of workgroups, of which the chip holds two per CU (their registers allow two waves per SIMD), three of
// the gather mode.  In a batch every request ends in a share cut short, so long shares are cut in three (sixteen
// requests of 8K..32K tokens: 136 us in one round, 124 / 121 / 122 / 127 / 136 in 2 / 3 / 4 / 6 / 8); short ones are not: a
// workgroup's first microseconds move nothing.  A scored share stages its logits in LDS, up to 32 KB.
static Kv8Plan kv8_plan(const okv_kv8_cache_t& c, bool gather, int batch, int group, int64_t rows, int max_score, bool folded) {
  Kv8Plan p{};
  const int hkv = c.num_kv_heads;
  const int64_t wgs = (int64_t)batch * hkv, all = std::max<int64_t>(rows, 1) * batch;
  if (max_score == 0 && rows <= std::min<int64_t>(2048, std::max<int64_t>(512, (gather ? 6 : 8) * wgs)))
    p.direct = wgs <= 256 ? 8 : 4;
  // (a token's heads in order within its row: rows behind the end then lie behind the second head's last one)
  p.pair = c.page_table && !gather && hkv % 2 == 0 && !p.direct && c.head_stride >= kD && c.head_stride + kD <= c.token_stride;
  const int nh = p.pair ? 2 : 1;
  p.least = 128 / nh;  // one tile per wave
  p.target = std::max(1, 256 * (gather ? kGatherResident : 2) * nh / hkv);  // shares of one round
  p.most = max_score > 0 ? 32768 / 4 / (nh * (folded ? 1 : group)) / 64 * 64 : 8192;
  p.fine = !gather && batch > 1;
  const int64_t n = std::min((all + p.least - 1) / p.least, std::max<int64_t>((p.fine ? 3 : 1) * (int64_t)p.target + 1, (all + p.most - 1) / p.most));
  p.items = p.direct ? batch : (int)std::min<int64_t>(n + (int64_t)batch * (max_score > 0 ? 2 : 1), 1 << 30);
  return p;
}

// Carves the partial results; the bytes they take.  `folded` saves logits, never adds.
static size_t kv8_workspace(const Kv8Plan& p, int batch, int hq, int hkv, int max_score, bool folded, Kv8Attn* a, char* ws) {
  if (a) {
    a->batch = batch;
    a->direct = p.direct;
    a->pair = p.pair;
    a->fine = p.fine ? 1024 / (p.pair ? 2 : 1) : 0;
    a->items = p.items;
    a->most_rows = p.most;
    a->least_rows = p.least;
    a->inv_target = 1.f / (float)std::max(p.target - batch / 2, (p.target + 1) / 2);
    a->inv_fine = 1.f / (float)std::max(3 * p.target - batch / 2, p.target);
  }
  if (p.direct) return 0;
  const size_t o = align256((size_t)p.items * hq * kD * 4), l = align256((size_t)p.items * hq * 4);
  const size_t stride = ((size_t)max_score + 63) / 64 * 64;
  const int heads = folded ? hkv : hq;
  const size_t g = max_score > 0 ? align256((size_t)batch * heads * stride * 4) : 0;
  if (a) {
    ws = (char*)align256((size_t)ws);
    a->part_o = (float*)ws;
    a->part_lse = (float*)(ws + o);
    a->logits = max_score > 0 ? (float*)(ws + o + l) : nullptr;
    a->logits_stride = (int64_t)stride;
    a->logit_heads = heads;
  }
  return o + l + g + 256;
}

template <typename T, typename F, int MODE, bool LOGITS, int NH, bool DIRECT = false, int W = 4>
static int launch_split(Kv8Attn& a, int batch, hipStream_t stream) {
  size_t floats = NH * (2 * W * kMaxGroup + (size_t)W * a.group * kD);
  if (LOGITS) floats = std::max(floats, (size_t)NH * (a.fold ? 1 : a.group) * a.most_rows);
  a.lds_scales = (int)floats;
  if (MODE == kGather) floats += 64 * W;
  hipLaunchKernelGGL((kv8_split<T, F, MODE, LOGITS, NH, DIRECT, W>), dim3((a.items + 7) / 8 * 8 * (a.c.num_kv_heads / NH)), dim3(64 * W), floats * 4, stream, a);
  return OKV_OK;
}

template <typename T, typename F, int W>
static void launch_direct(Kv8Attn& a, int batch, hipStream_t stream) {
  if (a.idx) launch_split<T, F, kGather, false, 1, true, W>(a, batch, stream);
  else if (a.c.page_table) launch_split<T, F, kPaged, false, 1, true, W>(a, batch, stream);
  else launch_split<T, F, kContiguous, false, 1, true, W>(a, batch, stream);
}

template <typename T, typename F>
static int launch_kv8(Kv8Attn& a, int batch, hipStream_t stream) {
  const bool paged = a.c.page_table != nullptr, scored = a.max_score_len > 0;
  if (a.direct) {
    if (a.direct == 8) launch_direct<T, F, 8>(a, batch, stream);
    else launch_direct<T, F, 4>(a, batch, stream);
    OKV_HIP_CHECK(hipGetLastError());
    return OKV_OK;
  }
  if (a.idx) launch_split<T, F, kGather, false, 1>(a, batch, stream);
  else if (paged && scored && a.pair) launch_split<T, F, kPaged, true, 2>(a, batch, stream);
  else if (paged && scored) launch_split<T, F, kPaged, true, 1>(a, batch, stream);
  else if (paged && a.pair) launch_split<T, F, kPaged, false, 2>(a, batch, stream);
  else if (paged) launch_split<T, F, kPaged, false, 1>(a, batch, stream);
  else if (scored) launch_split<T, F, kContiguous, true, 1>(a, batch, stream);
  else launch_split<T, F, kContiguous, false, 1>(a, batch, stream);
  const int64_t shares = a.items / a.batch;
  const int tokens = shares * ((a.max_score_len + 511) / 512) <= 65536 ? 512 : 1024;
  const dim3 grid(a.hq + (a.max_score_len + tokens - 1) / tokens, batch);
  if (tokens == 512) hipLaunchKernelGGL((kv8_join<T, 2>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((kv8_join<T, 4>), grid, dim3(256), 0, stream, a);
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

// What a plan is made for: without these bounds its divisions mean nothing (a group above 128 leaves a scored share no rows).
static int check_sizes(int hq, int hkv, int64_t rows, int batch) {
  OKV_REQUIRE(hq >= hkv && hq % hkv == 0, OKV_ERR_INVALID, "bad head counts q=%d kv=%d", hq, hkv);
  OKV_REQUIRE(hq / hkv <= kMaxGroup, OKV_ERR_UNSUPPORTED, "GQA group size %d not supported (1 to %d)", hq / hkv, kMaxGroup);
  OKV_REQUIRE(hq <= kMaxHeads, OKV_ERR_UNSUPPORTED, "%d q heads not supported (at most %d)", hq, kMaxHeads);
  OKV_REQUIRE(batch <= 65535, OKV_ERR_UNSUPPORTED, "batch %d not supported", batch);
  // (row numbers run past the last row by up to two steps of a workgroup, and stay in 32 bits)
  OKV_REQUIRE(rows * batch <= (1ll << 31) - 65536, OKV_ERR_UNSUPPORTED, "%lld rows not supported", (long long)rows * batch);
  return OKV_OK;
}

static int kv8_attend(Kv8Attn& a, int64_t rows, int batch, void* ws, size_t ws_bytes, hipStream_t stream) {
  const int hkv = a.c.num_kv_heads;
  OKV_REQUIRE(a.q && a.out, OKV_ERR_INVALID, "q or out is NULL");
  OKV_REQUIRE(((uintptr_t)a.q & 15) == 0, OKV_ERR_INVALID, "q must be 16-byte aligned");
  if (int rc = check_sizes(a.hq, hkv, rows, batch)) return rc;
  a.group = a.hq / hkv;
  a.block_shift = __builtin_ctz(a.c.block_tokens);
  a.page_shift = a.c.page_table && (a.c.page_size & (a.c.page_size - 1)) == 0 ? __builtin_ctz(a.c.page_size) : -1;
  const bool folded = a.max_score_len > 0 && a.normalise == OKV_NORM_RAW;
  if (folded) a.fold = a.head_reduce == OKV_REDUCE_MAX ? 1 : 2;
  const Kv8Plan p = kv8_plan(a.c, a.idx != nullptr, batch, a.group, rows, a.max_score_len, folded);
  const size_t need = kv8_workspace(p, batch, a.hq, hkv, a.max_score_len, folded, &a, (char*)ws);
  OKV_REQUIRE(ws != nullptr || need == 0, OKV_ERR_INVALID, "workspace pointer is NULL");
  OKV_REQUIRE(ws_bytes >= need, OKV_ERR_WORKSPACE, "workspace too small: have %zu, need %zu", ws_bytes, need);
  OKV_REQUIRE((int64_t)(a.items + 7) * hkv < (1ll << 31), OKV_ERR_UNSUPPORTED, "%d requests of up to %lld rows", batch, (long long)rows);
  if (a.c.dtype == OKV_BF16)
    return a.c.format == OKV_E4M3 ? launch_kv8<BF16, E4M3>(a, batch, stream) : launch_kv8<BF16, I8>(a, batch, stream);
  return a.c.format == OKV_E4M3 ? launch_kv8<F16, E4M3>(a, batch, stream) : launch_kv8<F16, I8>(a, batch, stream);
}

}  // namespace okv

using namespace okv;

extern "C" {

int okv_kv8_workspace_bytes(const okv_kv8_cache_t* cache, int32_t num_q_heads, int32_t batch, int32_t max_rows,
                            int32_t max_score_len, int32_t indexed, size_t* out_bytes) {
  OKV_REQUIRE(cache != nullptr && out_bytes != nullptr, OKV_ERR_INVALID, "NULL argument");
  const int hkv = cache->num_kv_heads;
  OKV_REQUIRE(batch >= 1 && hkv >= 1 && num_q_heads >= hkv && max_rows >= 0 && max_score_len >= 0, OKV_ERR_INVALID,
              "bad batch, head counts or lengths");
  if (int rc = check_sizes(num_q_heads, hkv, max_rows, batch)) return rc;
  // an index without entries may come as NULL: a call planned as one without an index
  size_t bytes = 0;
  for (int gather = 0; gather <= (indexed != 0); ++gather) {
    const Kv8Plan p = kv8_plan(*cache, gather != 0, batch, num_q_heads / hkv, max_rows, max_score_len, false);
    bytes = std::max(bytes, kv8_workspace(p, batch, num_q_heads, hkv, max_score_len, false, nullptr, nullptr));
  }
  *out_bytes = bytes;
  return OKV_OK;
}

int okv_kv8_dense_attn(const void* q, int32_t num_q_heads, const okv_kv8_cache_t* cache, const int32_t* seq_lens,
                       int32_t max_seq_len, int32_t batch, float scale, void* out, const int32_t* score_lens,
                       int32_t max_score_len, int32_t head_reduce, int32_t normalise, float* scores,
                       int64_t score_stride, void* ws, size_t ws_bytes, okv_stream_t stream) {
  int rc = kv8_validate(cache, "okv_kv8_dense_attn");
  if (rc) return rc;
  OKV_REQUIRE(batch >= 1 && max_seq_len >= 1, OKV_ERR_INVALID, "bad batch or length");
  OKV_REQUIRE(max_seq_len <= kv8_room(*cache), OKV_ERR_INVALID, "max_seq_len %d exceeds the cache's %lld tokens", max_seq_len,
              (long long)kv8_room(*cache));
  Kv8Attn a;
  memset(&a, 0, sizeof a);
  a.c = *cache;
  a.q = q;
  a.hq = num_q_heads;
  a.scale = scale;
  a.lens = seq_lens;
  a.max_len = max_seq_len;
  a.late[0] = cache->open_k;
  a.late[1] = cache->open_v;
  a.late_token_stride = cache->open_token_stride;
  a.late_head_stride = cache->open_head_stride;
  a.late_batch_stride = cache->open_batch_stride;
  a.out = out;
  if (scores) {
    OKV_REQUIRE(max_score_len >= 0 && max_score_len <= max_seq_len, OKV_ERR_INVALID, "max_score_len out of range");
    OKV_REQUIRE(score_stride >= max_score_len, OKV_ERR_INVALID, "score_stride < max_score_len");
    OKV_REQUIRE(head_reduce == OKV_REDUCE_MAX || head_reduce == OKV_REDUCE_SUM, OKV_ERR_INVALID, "bad head_reduce %d",
                head_reduce);
    OKV_REQUIRE(normalise == OKV_NORM_RAW || normalise == OKV_NORM_SOFTMAX, OKV_ERR_INVALID, "bad normalise %d", normalise);
    a.score_lens = score_lens;
    a.max_score_len = max_score_len;
    a.scores = scores;
    a.score_stride = score_stride;
    a.head_reduce = head_reduce;
    a.normalise = normalise;
  }
  return kv8_attend(a, max_seq_len, batch, ws, ws_bytes, (hipStream_t)stream);
}

int okv_kv8_sparse_attn(const void* q, int32_t num_q_heads, const okv_kv8_cache_t* cache, const int32_t* idx,
                        int64_t idx_stride, int32_t slots, const int32_t* sel_lens, int32_t max_sel_len,
                        const void* tail_k, const void* tail_v, int64_t tail_token_stride, int64_t tail_head_stride,
                        int64_t tail_batch_stride, const int32_t* tail_lens, int32_t max_tail_len, int32_t batch,
                        float scale, void* out, void* ws, size_t ws_bytes, okv_stream_t stream) {
  int rc = kv8_validate(cache, "okv_kv8_sparse_attn");
  if (rc) return rc;
  OKV_REQUIRE(batch >= 1 && max_sel_len >= 0 && max_tail_len >= 0, OKV_ERR_INVALID, "bad batch or length");
  OKV_REQUIRE((int64_t)max_sel_len + max_tail_len >= 1, OKV_ERR_INVALID, "no rows to attend to");
  if (idx) OKV_REQUIRE(idx_stride >= max_sel_len, OKV_ERR_INVALID, "idx_stride < max_sel_len");
  else OKV_REQUIRE(max_sel_len <= kv8_room(*cache), OKV_ERR_INVALID, "max_sel_len %d exceeds the cache's %lld tokens",
                   max_sel_len, (long long)kv8_room(*cache));
  if (slots)
    OKV_REQUIRE((idx || max_sel_len == 0) && cache->page_table && cache->page_stride == cache->page_size * cache->token_stride &&
                    cache->scale_page_stride == cache->page_size / cache->block_tokens * cache->scale_block_stride,
                OKV_ERR_INVALID, "slots need an index and a pool whose pages lie back to back");
  if (max_tail_len > 0)
    OKV_REQUIRE(tail_k && tail_v && ((uintptr_t)tail_k & 15) == 0 && ((uintptr_t)tail_v & 15) == 0 &&
                    tail_token_stride % 8 == 0 && tail_head_stride % 8 == 0 && tail_batch_stride % 8 == 0,
                OKV_ERR_INVALID, "tail: not NULL, 16-byte aligned, strides multiples of 8 elements");
  Kv8Attn a;
  memset(&a, 0, sizeof a);
  a.c = *cache;
  a.q = q;
  a.hq = num_q_heads;
  a.scale = scale;
  a.sparse = 1;
  a.slots = slots ? 1 : 0;
  a.lens = sel_lens;
  a.max_len = max_sel_len;
  a.idx = idx;
  a.idx_stride = idx_stride;
  a.late[0] = tail_k;
  a.late[1] = tail_v;
  a.late_token_stride = tail_token_stride;
  a.late_head_stride = tail_head_stride;
  a.late_batch_stride = tail_batch_stride;
  a.tail_lens = tail_lens;
  a.max_tail_len = max_tail_len;
  a.out = out;
  return kv8_attend(a, (int64_t)max_sel_len + max_tail_len, batch, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
