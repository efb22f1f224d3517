// Writing (okv_kv8_append) and reading back (okv_kv8_read) rows of the 8-bit K/V cache.
#include <math.h>

#include "okv_kv8.h"

namespace okv {

int kv8_validate(const okv_kv8_cache_t* c, const char* what) {
  OKV_REQUIRE(c != nullptr, OKV_ERR_INVALID, "%s: cache is NULL", what);
  OKV_REQUIRE(c->k_codes && c->v_codes && c->k_scale && c->v_scale, OKV_ERR_INVALID, "%s: NULL codes or scales", what);
  OKV_REQUIRE(c->format == OKV_E4M3 || c->format == OKV_I8, OKV_ERR_UNSUPPORTED,
              "%s: code format %d (OKV_E4M3 and OKV_I8 are)", what, c->format);
  OKV_REQUIRE(c->dtype == OKV_BF16 || c->dtype == OKV_F16, OKV_ERR_UNSUPPORTED,
              "%s: dtype %d next to an 8-bit cache (OKV_BF16 and OKV_F16 are)", what, c->dtype);
  OKV_REQUIRE(c->head_dim == kD, OKV_ERR_UNSUPPORTED, "%s: head_dim %d not supported (kernels are built for 128)", what,
              c->head_dim);
  OKV_REQUIRE(c->num_kv_heads >= 1, OKV_ERR_INVALID, "%s: num_kv_heads %d", what, c->num_kv_heads);
  const int bt = c->block_tokens;
  OKV_REQUIRE(bt == 16 || bt == 32 || bt == 64 || bt == 128, OKV_ERR_UNSUPPORTED, "%s: block_tokens %d (16, 32, 64, 128)",
              what, bt);
  OKV_REQUIRE(((uintptr_t)c->k_codes & 15) == 0 && ((uintptr_t)c->v_codes & 15) == 0, OKV_ERR_INVALID,
              "%s: code pointers must be 16-byte aligned", what);
  OKV_REQUIRE(((uintptr_t)c->k_scale & 3) == 0 && ((uintptr_t)c->v_scale & 3) == 0, OKV_ERR_INVALID,
              "%s: scale pointers must be 4-byte aligned", what);
  OKV_REQUIRE(c->token_stride % 16 == 0 && c->head_stride % 16 == 0 && c->batch_stride % 16 == 0 && c->page_stride % 16 == 0,
              OKV_ERR_INVALID, "%s: code strides must be multiples of 16 bytes", what);
  OKV_REQUIRE(c->token_stride >= 0 && c->token_stride < (1ll << 26), OKV_ERR_UNSUPPORTED, "%s: token stride %lld", what,
              (long long)c->token_stride);
  if (c->page_table) {
    OKV_REQUIRE(c->page_size >= bt && c->page_size % bt == 0, OKV_ERR_INVALID,
                "%s: page_size %d is not a multiple of block_tokens %d", what, c->page_size, bt);
    OKV_REQUIRE((int64_t)c->num_pages * c->page_size < (1ll << 31) && (int64_t)c->page_table_stride * c->page_size < (1ll << 31),
                OKV_ERR_UNSUPPORTED, "%s: 2^31 token slots or more", what);
    OKV_REQUIRE(c->page_table_stride >= 1 && c->num_pages >= 1, OKV_ERR_INVALID, "%s: page_table_stride %d, num_pages %d",
                what, c->page_table_stride, c->num_pages);
  } else {
    OKV_REQUIRE(c->capacity >= bt && c->capacity % bt == 0, OKV_ERR_INVALID,
                "%s: capacity %d is not a multiple of block_tokens %d", what, c->capacity, bt);
  }
  OKV_REQUIRE((c->open_k == nullptr) == (c->open_v == nullptr), OKV_ERR_INVALID, "%s: one of open_k / open_v is NULL", what);
  if (c->open_k)
    OKV_REQUIRE(((uintptr_t)c->open_k & 15) == 0 && ((uintptr_t)c->open_v & 15) == 0 && c->open_token_stride % 8 == 0 &&
                    c->open_head_stride % 8 == 0 && c->open_batch_stride % 8 == 0,
                OKV_ERR_INVALID, "%s: open buffers: 16-byte aligned, strides multiples of 8 elements", what);
  return OKV_OK;
}

struct AppendArgs {
  okv_kv8_cache_t c;
  const void* rows[2];  // new K, new V
  int64_t token_stride[2], head_stride[2], batch_stride[2];
  const int32_t* starts;
  const int32_t* new_lens;
  int32_t start, max_new, close;
};

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
template <typename T> constexpr uint32_t kInfBits = 0x7f80;  // of bfloat16
template <> constexpr uint32_t kInfBits<F16> = 0x7c00;
__device__ __forceinline__ float magnitude(const BF16*, uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ float magnitude(const F16*, uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// scale = max(amax / qmax, 2^-126), code = nearest(x * fl32(1 / scale)).  One workgroup per (touched block, kv head, request, K
// or V): 16 lanes hold a row (eight elements each), sixteen rows per trip, the whole block in registers between
// the two passes (maximum, then codes), so that each element is read once and written once.  Bound by that: 131073 tokens of
// eight heads, bf16 to e4m3 in blocks of 64 (805 MB), 134 us = 6.0 TB/s; one token for each of sixteen requests a
// launch.  Rows come in and codes go out non-temporal (147 us without, 145 and 138 with one of the two); 152 before
// the maximum was taken over bit patterns and the rows a block does not have were left out.
// The workgroup of the first touched block also moves the rows of the block that stays open: it has read the old
// open rows by then, and nobody else touches the request's open buffer.
template <typename T, typename F>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs a) {
  __shared__ uint32_t s_max[4];
  const okv_kv8_cache_t& c = a.c;
  const int B = c.block_tokens;
  const int g = blockIdx.y, b = blockIdx.z >> 1, is_v = blockIdx.z & 1;
  const int start = a.starts ? a.starts[b] : a.start;
  int n = a.new_lens ? a.new_lens[b] : a.max_new;
  n = n < 0 ? 0 : n > a.max_new ? a.max_new : n;
  if (n == 0 || start < 0 || (int64_t)start + n > kv8_room(c)) return;
  const int end = start + n;
  const int first = start / B, blk = first + blockIdx.x;
  if (blk > (end - 1) / B) return;  // (blk * B may pass 2^31 behind the last block)
  const T* src = reinterpret_cast<const T*>(a.rows[is_v]) + (int64_t)b * a.batch_stride[is_v] + (int64_t)g * a.head_stride[is_v];
  const int64_t row_stride = a.token_stride[is_v];
  T* open = reinterpret_cast<T*>(is_v ? c.open_v : c.open_k);
  if (open) open += (int64_t)b * c.open_batch_stride + (int64_t)g * c.open_head_stride;
  const int tid = threadIdx.x, col = tid & 15, row = tid >> 4;
  const bool whole = (blk + 1) * B <= end || a.close;  // this block becomes codes
  if (whole) {
    constexpr int P = kMaxBlockTokens / 16;
    uint4 x[P];
    // magnitudes order as the 16-bit patterns without the sign, infinities and NaNs above all numbers: the maximum needs
    // no conversion and no test of each element
    u16x2_t top = {0, 0};
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (16 * p >= B) break;
      const int r = 16 * p + row, t = blk * B + r;
      x[p] = make_uint4(0, 0, 0, 0);
      if (t < end) {
        const T* q = t >= start ? src + (int64_t)(t - start) * row_stride : open + (int64_t)r * c.open_token_stride;
        x[p] = load_stream16(q + 8 * col);
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (16 * p >= B) break;
      for (const uint32_t w : {x[p].x, x[p].y, x[p].z, x[p].w})
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu));
    }
    uint32_t m = top.x > top.y ? top.x : top.y;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    if ((tid & 63) == 0) s_max[tid >> 6] = m;
    __syncthreads();
    m = __builtin_amdgcn_readfirstlane(max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3])));
    const bool poison = m >= kInfBits<T>;
    const float amax = magnitude((const T*)nullptr, m);
    const float scale = poison ? NAN : fmaxf(amax / qmax_of(F{}), kMinScale);
    const float inv = 1.f / scale;
    int64_t ro, so;
    if (kv8_locate(c, b, blk * B, &ro, &so)) {
      uint8_t* dst = reinterpret_cast<uint8_t*>(is_v ? c.v_codes : c.k_codes) + ro + (int64_t)g * c.head_stride;
      if (tid == 0) (is_v ? c.v_scale : c.k_scale)[so + (int64_t)g * c.scale_head_stride] = scale;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (16 * p >= B) break;
        const int r = 16 * p + row;
        if (blk * B + r >= end) continue;
        uint2 codes = make_uint2(0, 0);
        if (!poison) {
          float v[8];
          cvt8((const T*)nullptr, x[p], v);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_fmed3f(v[i] * inv, -qmax_of(F{}), qmax_of(F{}));
          codes = make_uint2(encode4(F{}, v), encode4(F{}, v + 4));
        }
        __builtin_nontemporal_store(u32x2_t{codes.x, codes.y}, reinterpret_cast<u32x2_t*>(dst + (int64_t)r * c.token_stride + 8 * col));
      }
    }
  }
  if (blockIdx.x != 0 || a.close || end % B == 0) return;
  // rows of the last block, which stays open; the old open rows have been read
  __syncthreads();
  const int lo = max(start, end / B * B);
  for (int t = lo + row; t < end; t += 16)
    *reinterpret_cast<uint4*>(open + (int64_t)(t % B) * c.open_token_stride + 8 * col) =
        *reinterpret_cast<const uint4*>(src + (int64_t)(t - start) * row_stride + 8 * col);
}

// value = code * scale, rounded once to 16 bits; 16 lanes per row.  Bound by the bytes: 131073 tokens of eight heads (268 MB
// read, 537 MB written) 178 us = 4.5 TB/s, 8001 tokens 10.9 us.  Stores of eight elements that do not stay in the caches: 201 and 13.1
// with element-wise ones, 180 and 14.5 where the loads are non-temporal instead.  Four or eight rows of a thread in flight: no
// difference.
struct ReadArgs {
  okv_kv8_cache_t c;
  const int32_t* idx;
  int64_t idx_stride;
  const int32_t* seq_lens;
  int32_t max_seq_len, max_rows;
  void* out[2];
  int64_t token_stride, head_stride, batch_stride;
};

template <typename T, typename F>
__global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a) {
  const okv_kv8_cache_t& c = a.c;
  const int g = blockIdx.y, b = blockIdx.z >> 1, is_v = blockIdx.z & 1;
  const int col = threadIdx.x & 15, j = blockIdx.x * 16 + (threadIdx.x >> 4);
  if (j >= a.max_rows) return;
  const int64_t room = kv8_room(c);
  int64_t len = a.seq_lens ? a.seq_lens[b] : a.max_seq_len;
  len = len < 0 ? 0 : len > a.max_seq_len ? a.max_seq_len : len;
  const int64_t closed = c.open_k ? len / c.block_tokens * c.block_tokens : len;
  const int t = a.idx ? a.idx[(int64_t)b * a.idx_stride + j] : j;
  T* dst = reinterpret_cast<T*>(a.out[is_v]) + (int64_t)b * a.batch_stride + (int64_t)j * a.token_stride +
           (int64_t)g * a.head_stride + 8 * col;
  if (t >= closed && t < len) {
    const T* open = reinterpret_cast<const T*>(is_v ? c.open_v : c.open_k) + (int64_t)b * c.open_batch_stride +
                    (int64_t)g * c.open_head_stride + (int64_t)(t % c.block_tokens) * c.open_token_stride;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(open + 8 * col);
    return;
  }
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int64_t ro, so;
  if (t >= 0 && t < len && t < room && kv8_locate(c, b, t, &ro, &so)) {
    const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(is_v ? c.v_codes : c.k_codes) + ro +
                                                    (int64_t)g * c.head_stride + 8 * col);
    const float s = (is_v ? c.v_scale : c.k_scale)[so + (int64_t)g * c.scale_head_stride];
    decode4(F{}, x.x, v);
    decode4(F{}, x.y, v + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
  }
  const T* ty = nullptr;
  __builtin_nontemporal_store(u32x4_t{pack_pair(ty, v[0], v[1]), pack_pair(ty, v[2], v[3]), pack_pair(ty, v[4], v[5]), pack_pair(ty, v[6], v[7])},
                              reinterpret_cast<u32x4_t*>(dst));
}

}  // namespace okv

using namespace okv;

#define OKV_KV8_DISPATCH(c, KERNEL, grid, args)                                                               \
  do {                                                                                                        \
    if ((c)->dtype == OKV_BF16) {                                                                             \
      if ((c)->format == OKV_E4M3) hipLaunchKernelGGL((KERNEL<BF16, E4M3>), grid, dim3(256), 0, (hipStream_t)stream, args); \
      else hipLaunchKernelGGL((KERNEL<BF16, I8>), grid, dim3(256), 0, (hipStream_t)stream, args);             \
    } else {                                                                                                  \
      if ((c)->format == OKV_E4M3) hipLaunchKernelGGL((KERNEL<F16, E4M3>), grid, dim3(256), 0, (hipStream_t)stream, args); \
      else hipLaunchKernelGGL((KERNEL<F16, I8>), grid, dim3(256), 0, (hipStream_t)stream, args);              \
    }                                                                                                         \
  } while (0)

extern "C" {

int okv_kv8_append(const okv_kv8_cache_t* cache, const void* new_k, int64_t k_token_stride, int64_t k_head_stride,
                   int64_t k_batch_stride, const void* new_v, int64_t v_token_stride, int64_t v_head_stride,
                   int64_t v_batch_stride, const int32_t* starts, int32_t start,
                   const int32_t* new_lens, int32_t max_new, int32_t close, int32_t batch, okv_stream_t stream) {
  int rc = kv8_validate(cache, "okv_kv8_append");
  if (rc) return rc;
  const int B = cache->block_tokens;
  OKV_REQUIRE((new_k && new_v) || max_new == 0, OKV_ERR_INVALID, "new_k or new_v is NULL");
  OKV_REQUIRE(batch >= 1 && max_new >= 0, OKV_ERR_INVALID, "bad batch or length");
  const AppendArgs a{*cache, {new_k, new_v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride},
                     {k_batch_stride, v_batch_stride}, starts, new_lens, start, max_new, close ? 1 : 0};
  OKV_REQUIRE(((uintptr_t)new_k & 15) == 0 && ((uintptr_t)new_v & 15) == 0 &&
                  ((k_token_stride | k_head_stride | k_batch_stride | v_token_stride | v_head_stride | v_batch_stride) & 7) == 0,
              OKV_ERR_INVALID,
              "new rows: 16-byte aligned, strides multiples of 8 elements");
  if (!starts)
    OKV_REQUIRE(start >= 0 && (new_lens || (int64_t)start + max_new <= kv8_room(*cache)), OKV_ERR_INVALID,
                "rows [%d, %lld) do not fit the cache's %lld tokens", start, (long long)start + max_new,
                (long long)kv8_room(*cache));
  if (close || !cache->open_k)
    OKV_REQUIRE(!starts && start % B == 0, OKV_ERR_INVALID,
                "closing the last block, and a cache without open buffers, need a start at a block's border, known to the host");
  if (!cache->open_k && !close)
    OKV_REQUIRE(!new_lens && max_new % B == 0, OKV_ERR_INVALID,
                "without open buffers an append ends at a block's border or closes the last block");
  if (max_new == 0) return OKV_OK;
  // a start the device knows may lie anywhere in its block
  const int64_t blocks = starts ? ((int64_t)max_new + 2 * B - 2) / B : ((int64_t)start % B + max_new + B - 1) / B;
  OKV_REQUIRE(cache->num_kv_heads <= 65535 && batch <= 32767, OKV_ERR_UNSUPPORTED, "too many heads or requests");
  OKV_KV8_DISPATCH(cache, kv8_append_kernel, dim3((uint32_t)blocks, cache->num_kv_heads, 2 * batch), a);
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

int okv_kv8_read(const okv_kv8_cache_t* cache, const int32_t* idx, int64_t idx_stride, int32_t max_rows,
                 const int32_t* seq_lens, int32_t max_seq_len, int32_t batch, void* k_out, void* v_out,
                 int64_t out_token_stride, int64_t out_head_stride, int64_t out_batch_stride, okv_stream_t stream) {
  int rc = kv8_validate(cache, "okv_kv8_read");
  if (rc) return rc;
  OKV_REQUIRE((k_out && v_out) || max_rows == 0, OKV_ERR_INVALID, "k_out or v_out is NULL");
  OKV_REQUIRE(batch >= 1 && max_rows >= 0 && max_seq_len >= 0 && max_seq_len <= kv8_room(*cache), OKV_ERR_INVALID,
              "bad batch or length");
  if (idx) OKV_REQUIRE(idx_stride >= max_rows, OKV_ERR_INVALID, "idx_stride < max_rows");
  ReadArgs a{*cache, idx, idx_stride, seq_lens, max_seq_len, max_rows, {k_out, v_out}, out_token_stride, out_head_stride,
             out_batch_stride};
  OKV_REQUIRE(((uintptr_t)k_out & 15) == 0 && ((uintptr_t)v_out & 15) == 0 &&
                  ((out_token_stride | out_head_stride | out_batch_stride) & 7) == 0, OKV_ERR_INVALID,
              "outputs: 16-byte aligned, strides multiples of 8 elements");
  if (max_rows == 0) return OKV_OK;
  OKV_REQUIRE(cache->num_kv_heads <= 65535 && batch <= 32767, OKV_ERR_UNSUPPORTED, "too many heads or requests");
  OKV_KV8_DISPATCH(cache, kv8_read_kernel, dim3((max_rows + 15) / 16, cache->num_kv_heads, 2 * batch), a);
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

}  // extern "C"
