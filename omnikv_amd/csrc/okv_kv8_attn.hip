// Decode attention over the 8-bit K/V cache: okv_kv8_dense_attn, okv_kv8_sparse_attn.
//
// A launch of splits (each workgroup a range of one request's rows for one kv head: running maximum,
// sum and output of a softmax over its rows), then one launch that joins the splits and finishes the
// filter layer's scores.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "okv_kv8.h"

namespace okv {

constexpr int kMaxGroup = 8;
constexpr int kMaxHeads = 256;

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
  const void* tail[2];
  int64_t tail_token_stride, tail_head_stride, tail_batch_stride;
  const int32_t* tail_lens;
  int32_t max_tail_len;
  const int32_t* score_lens;
  int32_t max_score_len;
  // partial results
  float* part_o;    // [batch][Hq][splits][128]
  float* part_lse;  // [batch][Hq][splits], log2 domain; -inf: no row took part
  float* logits;    // [batch][Hq][logits_stride], natural units
  int64_t logits_stride;
  int32_t splits, split_rows;
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

// grid (Hkv, splits, batch): eight lanes hold a row, 16 elements each.
template <typename T, typename F>
__global__ __launch_bounds__(256) void kv8_split(Kv8Attn a) {
  __shared__ float s_q[kMaxGroup][kD];
  __shared__ float s_m[32][kMaxGroup], s_l[32][kMaxGroup];
  __shared__ float s_o[4][kMaxGroup][kD];
  const okv_kv8_cache_t& c = a.c;
  const int g = blockIdx.x, split = blockIdx.y, b = blockIdx.z, G = a.group;
  const int main_len = clamp_len(a.lens, b, a.max_len);
  const int tail_len = a.max_tail_len ? clamp_len(a.tail_lens, b, a.max_tail_len) : 0;
  const int L = main_len + tail_len, A = kv8_score_len(a, b, main_len);
  int begin, end;
  rl_split_range(split, a.split_rows, A, L, &begin, &end);
  if (begin >= end) return;
  const int closed = a.sparse || !c.open_k ? main_len : main_len / c.block_tokens * c.block_tokens;
  for (int i = threadIdx.x; i < G * kD; i += 256) {
    const T x = reinterpret_cast<const T*>(a.q)[(int64_t)(b * a.hq + g * G) * kD + i];
    float v;
    if constexpr (sizeof(T) == 2) {
      uint4 u = make_uint4(x.v, 0, 0, 0);
      float o[8];
      cvt8((const T*)nullptr, u, o);
      v = o[0];
    }
    s_q[i / kD][i % kD] = v;
  }
  __syncthreads();
  const int lane8 = threadIdx.x & 7, slot = threadIdx.x >> 3, e0 = 16 * lane8;
  const int64_t room = a.slots ? (int64_t)c.num_pages * c.page_size : kv8_room(c);
  float m[kMaxGroup], l[kMaxGroup], o[kMaxGroup][16];
#pragma unroll
  for (int h = 0; h < kMaxGroup; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[h][i] = 0.f;
  }
  for (int r0 = begin; r0 < end; r0 += 32) {
    const int r = r0 + slot;
    bool ok = r < end;
    float kv[2][16];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) kv[x][i] = 0.f;
    if (ok && r >= closed) {
      const bool tail = r >= main_len;
      const int t = tail ? r - main_len : r % c.block_tokens;
      for (int x = 0; x < 2; ++x) {
        const T* p = reinterpret_cast<const T*>(tail ? a.tail[x] : x ? c.open_v : c.open_k);
        p += tail ? (int64_t)b * a.tail_batch_stride + (int64_t)t * a.tail_token_stride + (int64_t)g * a.tail_head_stride
                  : (int64_t)b * c.open_batch_stride + (int64_t)t * c.open_token_stride + (int64_t)g * c.open_head_stride;
        load8(p + e0, kv[x]);
        load8(p + e0 + 8, kv[x] + 8);
      }
    } else if (ok) {
      const int t = a.idx ? a.idx[(int64_t)b * a.idx_stride + r] : r;
      ok = t >= 0 && t < room;
      if (ok) {
        int64_t ro, so;
        if (a.slots) {
          ro = (int64_t)t * c.token_stride;
          so = (int64_t)(t / c.block_tokens) * c.scale_block_stride;
        } else {
          ok = kv8_locate(c, b, t, &ro, &so);
        }
        for (int x = 0; x < 2; ++x) {
          const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(x ? c.v_codes : c.k_codes) + ro +
                                                          (int64_t)g * c.head_stride + e0);
          const float s = (x ? c.v_scale : c.k_scale)[so + (int64_t)g * c.scale_head_stride];
          decode4(F{}, u.x, kv[x]);
          decode4(F{}, u.y, kv[x] + 4);
          decode4(F{}, u.z, kv[x] + 8);
          decode4(F{}, u.w, kv[x] + 12);
#pragma unroll
          for (int i = 0; i < 16; ++i) kv[x][i] *= s;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kMaxGroup; ++h) {
      if (h >= G) break;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s = fmaf(s_q[h][e0 + i], kv[0][i], s);
      s += __shfl_xor(s, 1);
      s += __shfl_xor(s, 2);
      s += __shfl_xor(s, 4);
      s = ok ? s * a.scale : -INFINITY;
      if (a.logits && r < end && r < A && lane8 == 0) a.logits[(int64_t)(b * a.hq + g * G + h) * a.logits_stride + r] = s;
      if (!ok) continue;
      const float x = s * kLog2e, mn = fmaxf(m[h], x);
      const float al = exp2f(m[h] - mn), p = exp2f(x - mn);
      l[h] = fmaf(l[h], al, p);
#pragma unroll
      for (int i = 0; i < 16; ++i) o[h][i] = fmaf(o[h][i], al, p * kv[1][i]);
      m[h] = mn;
    }
  }
  // the 32 row slots of the workgroup meet: maxima and sums in LDS, outputs over the wave's slots first
#pragma unroll
  for (int h = 0; h < kMaxGroup; ++h)
    if (lane8 == 0) {
      s_m[slot][h] = m[h];
      s_l[slot][h] = l[h];
    }
  __syncthreads();
  float M[kMaxGroup];
#pragma unroll
  for (int h = 0; h < kMaxGroup; ++h) {
    if (h >= G) break;
    M[h] = -INFINITY;
    for (int x = 0; x < 32; ++x) M[h] = fmaxf(M[h], s_m[x][h]);
    const float f = m[h] == -INFINITY ? 0.f : exp2f(m[h] - M[h]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = o[h][i] * f;
      v += __shfl_xor(v, 8);
      v += __shfl_xor(v, 16);
      v += __shfl_xor(v, 32);
      if ((threadIdx.x & 63) < 8) s_o[threadIdx.x >> 6][h][e0 + i] = v;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * kD; i += 256) {
    const int h = i / kD, d = i % kD;
    float Mh = -INFINITY, den = 0.f;
    for (int x = 0; x < 32; ++x) Mh = fmaxf(Mh, s_m[x][h]);
    for (int x = 0; x < 32; ++x) den += s_m[x][h] == -INFINITY ? 0.f : s_l[x][h] * exp2f(s_m[x][h] - Mh);
    const float num = s_o[0][h][d] + s_o[1][h][d] + s_o[2][h][d] + s_o[3][h][d];
    const int64_t ph = (int64_t)(b * a.hq + g * G + h) * a.splits + split;
    a.part_o[ph * kD + d] = Mh == -INFINITY ? 0.f : num / den;
    if (d == 0) a.part_lse[ph] = Mh == -INFINITY ? -INFINITY : Mh + log2f(den);
  }
}

// Blocks [0, Hq) of a request join the splits of one q head; the others finish 1024 scores each, working out
// the heads' normalisers themselves from the splits' partial log-sum-exps.
template <typename T>
__global__ __launch_bounds__(256) void kv8_join(Kv8Attn a) {
  __shared__ float s_lse[kMaxHeads];
  const int b = blockIdx.y;
  const int main_len = clamp_len(a.lens, b, a.max_len);
  const int L = main_len + (a.max_tail_len ? clamp_len(a.tail_lens, b, a.max_tail_len) : 0);
  const int A = kv8_score_len(a, b, main_len);
  if ((int)blockIdx.x < a.hq) {
    const int h = blockIdx.x, d = threadIdx.x & (kD - 1), ns = rl_num_splits(a.split_rows, A, L);
    const float* lse = a.part_lse + (int64_t)(b * a.hq + h) * a.splits;
    const float* po = a.part_o + (int64_t)(b * a.hq + h) * a.splits * kD + d;
    float M = -INFINITY, den = 0.f, num = 0.f;
    for (int s = 0; s < ns; ++s) {
      const float x = lse[s];
      if (x == -INFINITY) continue;
      const float mn = fmaxf(M, x), f = exp2f(M - mn), e = exp2f(x - mn);
      den = fmaf(den, f, e);
      num = fmaf(num, f, e * po[(int64_t)s * kD]);
      M = mn;
    }
    if (threadIdx.x < kD) store1(reinterpret_cast<T*>(a.out) + (int64_t)(b * a.hq + h) * kD + d, den == 0.f ? 0.f : num / den);
    return;
  }
  const int t0 = (blockIdx.x - a.hq) * 1024;
  if (t0 >= A) return;
  const bool soft = a.normalise == OKV_NORM_SOFTMAX, is_max = a.head_reduce == OKV_REDUCE_MAX;
  if (soft) {
    const int nA = (A + a.split_rows - 1) / a.split_rows;
    for (int h = threadIdx.x; h < a.hq; h += 256) {
      const float* lse = a.part_lse + (int64_t)(b * a.hq + h) * a.splits;
      float M = -INFINITY, den = 0.f;
      for (int s = 0; s < nA; ++s) M = fmaxf(M, lse[s]);
      for (int s = 0; s < nA; ++s) den += lse[s] == -INFINITY ? 0.f : exp2f(lse[s] - M);
      s_lse[h] = M == -INFINITY ? 0.f : M + log2f(den);
    }
    __syncthreads();
  }
  for (int t = t0 + threadIdx.x; t < min(t0 + 1024, A); t += 256) {
    float acc = is_max ? -INFINITY : 0.f;
    for (int h = 0; h < a.hq; ++h) {
      const float v = a.logits[(int64_t)(b * a.hq + h) * a.logits_stride + t];
      const float x = soft ? exp2f(fmaf(v, kLog2e, -s_lse[h])) : v;
      acc = is_max ? fmaxf(acc, x) : acc + x;
    }
    a.scores[(int64_t)b * a.score_stride + t] = acc;
  }
}

// ---------------------------------------------------------------- host side
static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

static int kv8_plan(int batch, int hkv, int64_t rows, int max_score, int* split_rows) {
  const int64_t work = std::max<int64_t>(rows, 1) * hkv * batch;
  int64_t per = (work + 511) / 512;
  per = std::max<int64_t>(64, (per + 63) / 64 * 64);
  *split_rows = (int)std::min<int64_t>(per, 8192);
  return (int)((rows + *split_rows - 1) / *split_rows) + (max_score > 0 ? 1 : 0);
}

static size_t kv8_workspace(int batch, int hq, int hkv, int64_t rows, int max_score, Kv8Attn* a, char* p) {
  int C = 0;
  const int S = std::max(1, kv8_plan(batch, hkv, rows, max_score, &C));
  const size_t o = align256((size_t)batch * hq * S * kD * 4), l = align256((size_t)batch * hq * S * 4);
  const size_t stride = ((size_t)max_score + 63) / 64 * 64;
  const size_t g = max_score > 0 ? align256((size_t)batch * hq * stride * 4) : 0;
  if (a) {
    p = (char*)align256((size_t)p);
    a->splits = S;
    a->split_rows = C;
    a->part_o = (float*)p;
    a->part_lse = (float*)(p + o);
    a->logits = max_score > 0 ? (float*)(p + o + l) : nullptr;
    a->logits_stride = (int64_t)stride;
  }
  return o + l + g + 256;
}

template <typename T, typename F>
static int launch_kv8(const Kv8Attn& a, int batch, hipStream_t stream) {
  hipLaunchKernelGGL((kv8_split<T, F>), dim3(a.c.num_kv_heads, a.splits, batch), dim3(256), 0, stream, a);
  hipLaunchKernelGGL(kv8_join<T>, dim3(a.hq + (a.max_score_len + 1023) / 1024, batch), dim3(256), 0, stream, a);
  OKV_HIP_CHECK(hipGetLastError());
  return OKV_OK;
}

static int kv8_attend(Kv8Attn& a, int64_t rows, int batch, void* ws, size_t ws_bytes, hipStream_t stream) {
  const int hkv = a.c.num_kv_heads;
  OKV_REQUIRE(a.q && a.out, OKV_ERR_INVALID, "q or out is NULL");
  OKV_REQUIRE(((uintptr_t)a.q & 15) == 0, OKV_ERR_INVALID, "q must be 16-byte aligned");
  OKV_REQUIRE(a.hq >= hkv && a.hq % hkv == 0, OKV_ERR_INVALID, "bad head counts q=%d kv=%d", a.hq, hkv);
  a.group = a.hq / hkv;
  OKV_REQUIRE(a.group <= kMaxGroup, OKV_ERR_UNSUPPORTED, "GQA group size %d not supported (1 to %d)", a.group, kMaxGroup);
  OKV_REQUIRE(a.hq <= kMaxHeads, OKV_ERR_UNSUPPORTED, "%d q heads not supported (at most %d)", a.hq, kMaxHeads);
  OKV_REQUIRE(batch <= 65535, OKV_ERR_UNSUPPORTED, "batch %d not supported", batch);
  OKV_REQUIRE(rows < (1ll << 31), OKV_ERR_UNSUPPORTED, "%lld rows not supported", (long long)rows);
  OKV_REQUIRE(ws != nullptr, OKV_ERR_INVALID, "workspace pointer is NULL");
  const size_t need = kv8_workspace(batch, a.hq, hkv, rows, a.max_score_len, &a, (char*)ws);
  OKV_REQUIRE(ws_bytes >= need, OKV_ERR_WORKSPACE, "workspace too small: have %zu, need %zu", ws_bytes, need);
  OKV_REQUIRE(a.splits <= 65535, OKV_ERR_UNSUPPORTED, "%d splits", a.splits);
  if (a.c.dtype == OKV_BF16)
    return a.c.format == OKV_E4M3 ? launch_kv8<BF16, E4M3>(a, batch, stream) : launch_kv8<BF16, I8>(a, batch, stream);
  return a.c.format == OKV_E4M3 ? launch_kv8<F16, E4M3>(a, batch, stream) : launch_kv8<F16, I8>(a, batch, stream);
}

}  // namespace okv

using namespace okv;

extern "C" {

int okv_kv8_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t max_rows,
                            int32_t max_score_len, size_t* out_bytes) {
  OKV_REQUIRE(out_bytes != nullptr, OKV_ERR_INVALID, "NULL argument");
  OKV_REQUIRE(batch >= 1 && num_kv_heads >= 1 && num_q_heads >= num_kv_heads && max_rows >= 0 && max_score_len >= 0,
              OKV_ERR_INVALID, "bad batch, head counts or lengths");
  *out_bytes = kv8_workspace(batch, num_q_heads, num_kv_heads, max_rows, max_score_len, nullptr, nullptr);
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
    OKV_REQUIRE(idx && cache->page_table && cache->page_stride == cache->page_size * cache->token_stride &&
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
  a.tail[0] = tail_k;
  a.tail[1] = tail_v;
  a.tail_token_stride = tail_token_stride;
  a.tail_head_stride = tail_head_stride;
  a.tail_batch_stride = tail_batch_stride;
  a.tail_lens = tail_lens;
  a.max_tail_len = max_tail_len;
  a.out = out;
  return kv8_attend(a, (int64_t)max_sel_len + max_tail_len, batch, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
