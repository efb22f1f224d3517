// The 8-bit K/V cache as its kernels see it (okv_kv8_cache_t in include/omnikv_hip.h has the format).
#pragma once

#include "okv_device.h"
#include "okv_internal.h"

namespace okv {

struct E4M3 {};
struct I8 {};

constexpr int kMaxBlockTokens = 128;
constexpr float kMinScale = 1.17549435082228750797e-38f;  // 2^-126: its reciprocal is finite

// tokens a request has room for
__host__ __device__ __forceinline__ int64_t kv8_room(const okv_kv8_cache_t& c) {
  return c.page_table ? (int64_t)c.page_table_stride * c.page_size : c.capacity;
}

// Where token t of request b lies: byte offset of its row (kv head 0) and float offset of its scale.
// false for a page number outside the pool: the offsets are then those of page 0, safe to read.
__device__ __forceinline__ bool kv8_locate(const okv_kv8_cache_t& c, int b, int t, int64_t* row, int64_t* scale) {
  if (!c.page_table) {
    *row = (int64_t)b * c.batch_stride + (int64_t)t * c.token_stride;
    *scale = (int64_t)b * c.scale_batch_stride + (int64_t)(t / c.block_tokens) * c.scale_block_stride;
    return true;
  }
  const int slot = t % c.page_size;
  const int page = c.page_table[(int64_t)b * c.page_table_stride + t / c.page_size];
  const bool ok = (uint32_t)page < (uint32_t)c.num_pages;
  const int64_t p = ok ? page : 0;
  *row = p * c.page_stride + (int64_t)slot * c.token_stride;
  *scale = p * c.scale_page_stride + (int64_t)(slot / c.block_tokens) * c.scale_block_stride;
  return ok;
}

// ---- codes -> fp32
__device__ __forceinline__ void decode4(E4M3, uint32_t x, float* o) {
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}
__device__ __forceinline__ void decode4(I8, uint32_t x, float* o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (float)(int8_t)(x >> (8 * i));
}
// two fp32 -> one dword of two 16-bit elements, the first in the low half
__device__ __forceinline__ uint32_t pack_pair(const BF16*, float a, float b) {
  const f32x2_t x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2_t));
}
__device__ __forceinline__ uint32_t pack_pair(const F16*, float a, float b) {
  const f32x2_t x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2_t));
}
// ---- fp32 within the format's range -> code, ties to even
__device__ __forceinline__ uint32_t encode4(E4M3, const float* v) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true);
}
__device__ __forceinline__ uint32_t encode4(I8, const float* v) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= ((uint32_t)(int)rintf(v[i]) & 0xffu) << (8 * i);
  return r;
}
__device__ __forceinline__ constexpr float qmax_of(E4M3) { return 448.f; }
__device__ __forceinline__ constexpr float qmax_of(I8) { return 127.f; }

int kv8_validate(const okv_kv8_cache_t* c, const char* what);

}  // namespace okv
