// attn.cuh - what the paged attention kernels share: arguments, tensor maps, key ranges.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "ftb_common.cuh"

namespace ftb {

constexpr uint32_t kAttnBadPage = 1, kAttnBadRows = 2, kAttnTimeout = 4;  // status word bits
constexpr int kAttnCounters = FTB_ATTN_ZERO_BYTES / 4 - 4;  // after the status word (16 bytes)

struct AttnParams {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  const int32_t* block_table;
  const int32_t* kv_len;
  const int32_t* cu_q;
  uint32_t* status;
  int32_t* counters;
  float* partial;
  int64_t q_st, q_sh;
  int64_t total_q, table_stride, num_pages;
  int batch, max_q, table_width, page_log2;
  int Hq, Hkv, G, D;
  int causal, window, keys_max;  // keys_max = table_width * page
  float scale_log2;              // scale * log2(e): scores are kept as base-2 logarithms
};

// Tensor maps of the caches. A box is `r` = min(page, tile keys) key rows of one kv head by 64
// elements (128 bytes, 128-byte swizzle): dims (element, row in page, kv head, page, half), the
// last with both 64-element halves of a 128-element head, so one copy can bring r x 128 elements
// as [half][r][64]. Where D is no multiple of 64 a copy takes one half, whose elements past D are
// filled with zeros. Any page id is safe: a box outside the tensor reads zeros.
struct AttnMaps {
  CUtensorMap k, v, q;
};

int attn_cache_map(CUtensorMap* m, const void* base, const ftb_attn_args& a,
                   const int64_t (&strides)[3], uint32_t box_rows, uint32_t halves);
// Query rows of one kv head: boxes of `tokens` tokens x `group` heads x 64 elements.
int attn_q_map(CUtensorMap* m, const ftb_attn_args& a, uint32_t group, uint32_t tokens);

int launch_attn_stream(const ftb_attn_args& a, AttnParams P, cudaStream_t stream);
size_t attn_stream_partial_bytes(int64_t rows_max, int D);
bool attn_chunk_fits(const ftb_attn_args& a);  // its plan's batch and piece counts
int launch_attn_chunk(const ftb_attn_args& a, AttnParams P, cudaStream_t stream);
size_t attn_chunk_workspace_bytes(int64_t total_q, int batch, int Hkv, int G, int D);

__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap* map, int x, int row,
                                       int head, int page, int half, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(head), "r"(page), "r"(half),
      "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two fp32 values rounded to a packed pair.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The two numbers of pack2().
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// One sequence as the kernels see it: clamped, so that no length or offset a caller passes can
// reach outside the tensors.
struct AttnSeq {
  int q0;   // first row of q
  int n;    // new tokens
  int len;  // keys
  bool bad_len, bad_rows;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams& P, int b) {
  AttnSeq s;
  int64_t q0 = b, q1 = b + 1;
  if (P.cu_q) q0 = P.cu_q[b], q1 = P.cu_q[b + 1];
  const int len = P.kv_len[b];
  s.bad_rows = q0 < 0 || q1 < q0 || q1 > P.total_q || q1 - q0 > P.max_q;
  if (q0 < 0) q0 = 0;
  if (q1 > P.total_q) q1 = P.total_q;
  int64_t n = q1 - q0;
  if (n < 0) n = 0;
  if (n > P.max_q) n = P.max_q;
  s.q0 = (int)q0;
  s.n = (int)n;
  s.bad_len = len < 0 || len > P.keys_max;
  s.len = len < 0 ? 0 : len > P.keys_max ? P.keys_max : len;
  return s;
}

// Keys [lo, hi) that tokens i0..i1 of a sequence see between them.
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange attn_range(const AttnParams& P, const AttnSeq& s, int i0,
                                               int i1) {
  KeyRange r{0, s.len};
  // position + 1 of a token, as far as it limits it
  const int64_t first = (int64_t)s.len - s.n + i0, last = (int64_t)s.len - s.n + i1;
  if (P.causal && last + 1 < r.hi) r.hi = last + 1 < 0 ? 0 : (int)(last + 1);
  if (P.window > 0 && first - P.window + 1 > 0) r.lo = (int)(first - P.window + 1);
  return r;
}

}  // namespace ftb
