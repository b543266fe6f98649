// rope.cuh - what the kernels that turn queries and keys by their positions share: the arguments,
// their checks, and the loads and stores of a head's elements.
#pragma once

#include <string.h>

#include "ftb_common.cuh"

namespace ftb {

constexpr int kMaxPairs = 128;  // rot <= 256

struct RopeParams {
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_dst, *v_dst;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;      // token and head strides, elements
  int64_t kc_page, kc_tok, kc_head;                // cache strides (k_out: kc_tok, kc_head)
  int64_t vc_page, vc_tok, vc_head;
  const void* positions;  // [axes, tokens], axis stride pos_stride
  int64_t pos_stride;
  const float* table;
  int64_t table_rows;
  const void* slots;  // NULL: k_dst holds a row per token
  int64_t tokens, n_slots;
  int pos64, slot64, page, Hq, Hkv, D, rot, adjacent, axes;
  uint32_t axis[kMaxPairs / 16];  // 2 bits per frequency
};

template <int VEC>
struct Chunk;
template <>
struct Chunk<8> { using type = uint4; };
template <>
struct Chunk<4> { using type = uint2; };
template <>
struct Chunk<1> { using type = uint16_t; };

template <typename T>
__device__ __forceinline__ float elem_f32(uint16_t b);
template <>
__device__ __forceinline__ float elem_f32<__nv_bfloat16>(uint16_t b) { return bf16_bits_to_f32(b); }
template <>
__device__ __forceinline__ float elem_f32<__half>(uint16_t b) { return __half2float(__ushort_as_half(b)); }
template <typename T>
__device__ __forceinline__ uint16_t elem_bits(float f);
template <>
__device__ __forceinline__ uint16_t elem_bits<__nv_bfloat16>(float f) { return f32_to_bf16_bits(f); }
template <>
__device__ __forceinline__ uint16_t elem_bits<__half>(float f) { return __half_as_ushort(__float2half_rn(f)); }

template <int VEC>
__device__ __forceinline__ void load_bits(const uint16_t* p, uint16_t (&v)[VEC]) {
  // a plain load: q_out may be q itself
  const typename Chunk<VEC>::type w = *reinterpret_cast<const typename Chunk<VEC>::type*>(p);
  memcpy(v, &w, sizeof(w));
}
template <int VEC>
__device__ __forceinline__ void store_bits(uint16_t* p, const uint16_t (&v)[VEC]) {
  typename Chunk<VEC>::type w;
  memcpy(&w, v, sizeof(w));
  *reinterpret_cast<typename Chunk<VEC>::type*>(p) = w;
}

// Checks the arguments and fills the kernels' (host).
inline int rope_params(const ftb_rope_args* a, RopeParams& P) {
  if (!a) return FTB_ERR_ARG;
  if (a->tokens < 0 || a->tokens > 0x7fffffff || a->Hq < 1 || a->Hkv < 1 || a->D < 2 ||
      a->D > 512 || a->D % 2 || a->rot < 2 || a->rot % 2 || a->rot > a->D ||
      a->rot > 2 * kMaxPairs || a->axes < 1 || a->axes > 4 || a->table_rows < 1)
    return FTB_ERR_SHAPE;
  if (a->type != FTB_TYPE_BF16 && a->type != FTB_TYPE_F16) return FTB_ERR_ARG;
  if (a->pairs != FTB_PAIRS_HALF && a->pairs != FTB_PAIRS_ADJACENT) return FTB_ERR_ARG;
  if (a->order != FTB_AXES_BLOCKS && a->order != FTB_AXES_CYCLIC) return FTB_ERR_ARG;
  const int half = a->rot / 2;
  P = RopeParams{};
  int sum = 0;
  for (int x = 0; x < a->axes; ++x) {
    if (a->sections[x] < 0) return FTB_ERR_SHAPE;
    sum += a->sections[x];
  }
  if (sum != half) return FTB_ERR_SHAPE;
  for (int i = 0, x = 0, used = 0; i < half; ++i) {
    int axis;
    if (a->order == FTB_AXES_BLOCKS) {
      while (used == a->sections[x]) ++x, used = 0;
      ++used;
      axis = x;
    } else {  // the axes in turn while an axis has frequencies left, axis 0 for the rest
      axis = i % a->axes;
      if (i / a->axes >= a->sections[axis]) axis = 0;
    }
    P.axis[i >> 4] |= (uint32_t)axis << (2 * (i & 15));
  }
  if (a->tokens == 0) return FTB_OK;  // (nothing else is looked at)
  if (!a->q || !a->k || !a->q_out || !a->k_dst || !a->positions || !a->table) return FTB_ERR_ARG;
  if (a->slots ? (!a->v || !a->v_dst || a->page < 1) : (a->v_dst != nullptr)) return FTB_ERR_ARG;
  P.q = a->q, P.k = a->k, P.v = a->v, P.q_out = a->q_out, P.k_dst = a->k_dst, P.v_dst = a->v_dst;
  P.q_st = a->q_strides[0], P.q_sh = a->q_strides[1];
  P.k_st = a->k_strides[0], P.k_sh = a->k_strides[1];
  P.v_st = a->v_strides[0], P.v_sh = a->v_strides[1];
  P.kc_page = a->k_dst_strides[0], P.kc_tok = a->k_dst_strides[1], P.kc_head = a->k_dst_strides[2];
  P.vc_page = a->v_dst_strides[0], P.vc_tok = a->v_dst_strides[1], P.vc_head = a->v_dst_strides[2];
  P.positions = a->positions, P.pos_stride = a->pos_stride, P.table = a->table;
  P.table_rows = a->table_rows, P.slots = a->slots, P.tokens = a->tokens;
  P.n_slots = a->n_slots, P.pos64 = a->pos64, P.slot64 = a->slot64, P.page = a->page;
  P.Hq = a->Hq, P.Hkv = a->Hkv, P.D = a->D, P.rot = a->rot;
  P.adjacent = a->pairs == FTB_PAIRS_ADJACENT, P.axes = a->axes;
  return FTB_OK;
}

}  // namespace ftb
