// rope.cu - rotary positions on one or several axes, with the write of the new tokens' keys and
// values into the paged cache.
//
// Frequency i of a head turns the pair (a, b) = (x[i], x[i + rot/2]) ("half" pairs) or
// (x[2i], x[2i+1]) ("adjacent") by the angle of position[axis(i)]:
//   a' = a cos - b sin,  b' = b cos + a sin            (fp32, rounded once)
// cos and sin come from a table [positions, rot] (cos in its first rot/2 columns); elements past
// rot are copied. q goes to q_out, k (rotated) and v (copied) to the cache row of the token's
// slot, or to k_out without a cache.
//
// Bound: DRAM, 2 * (Hq + 2 Hkv) * D * 2 bytes per token. A thread owns one column of VEC pairs in
// every head it visits, so it takes the token's cos and sin once into registers.
#include "ftb_common.cuh"

namespace ftb {
namespace {

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

// Block (cols, heads per sweep), one per token: column threadIdx.x of 2 VEC elements of heads
// threadIdx.y, + blockDim.y, ... The first heads are loaded before the token's cos and sin (which
// every head shares) have come through shared memory, so the two latencies overlap; beyond that,
// many resident warps hide more than loads ahead, which cost registers (8190 tokens of 32 + 8 + 8
// heads of 128 with 1 / 2 / 4 heads ahead, us: 38.4 / 38.2 / 48.6, 5.4 TB/s; with random positions
// 39.4 / 43.1 / 55.4). Eight blocks leave 32 registers: the widest variant spills (56 bytes stored, 88
// loaded per thread in bf16; 28 and 52 in f16).
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 8) k_rope(const __grid_constant__ RopeParams P) {
  __shared__ float table[2 * kMaxPairs];  // cos, then sin
  pdl_launch_dependents();
  const int col = threadIdx.x;
  const int half = P.rot / 2, rot_cols = half / VEC;
  const bool turns = col < rot_cols;
  // element offsets of this column's two chunks in a rotated head and in a copied one
  int e0, e1;
  if (!turns) {
    e0 = P.rot + (col - rot_cols) * 2 * VEC;
    e1 = e0 + VEC;
  } else if (P.adjacent) {
    e0 = col * 2 * VEC;
    e1 = e0 + VEC;
  } else {
    e0 = col * VEC;
    e1 = e0 + half;
  }
  const int c0 = col * 2 * VEC;
  const int64_t tok = blockIdx.x;
  const int heads = P.Hq + 2 * P.Hkv;
  uint16_t a[VEC], b[VEC];
  auto load = [&](int hh) {
    const bool is_v = hh >= P.Hq + P.Hkv;
    if (hh >= heads || (is_v && !P.v_dst)) return;
    const uint16_t* src = hh < P.Hq ? P.q + tok * P.q_st + hh * P.q_sh
                          : is_v    ? P.v + tok * P.v_st + (hh - P.Hq - P.Hkv) * P.v_sh
                                    : P.k + tok * P.k_st + (hh - P.Hq) * P.k_sh;
    load_bits<VEC>(src + (is_v ? c0 : e0), a);
    load_bits<VEC>(src + (is_v ? c0 + VEC : e1), b);
  };
  pdl_wait();
  load(threadIdx.y);
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < P.rot; i += blockDim.x * blockDim.y) {
    const int f = i < half ? i : i - half;
    const int64_t at = (P.axis[f >> 4] >> (2 * (f & 15)) & 3) * P.pos_stride + tok;
    const int64_t p = P.pos64 ? static_cast<const int64_t*>(P.positions)[at]
                              : static_cast<const int32_t*>(P.positions)[at];
    // a position outside the table has no angle: the outputs are NaN, not another position's
    table[i] = p >= 0 && p < P.table_rows ? __ldg(P.table + p * P.rot + i)
                                          : __int_as_float(0x7fffffff);
  }
  int64_t slot = tok, page = 0;
  bool keep = true;
  if (P.slots) {
    slot = P.slot64 ? static_cast<const int64_t*>(P.slots)[tok]
                    : static_cast<const int32_t*>(P.slots)[tok];
    keep = slot >= 0 && slot < P.n_slots;  // -1: a padded token, not stored
    page = slot / P.page;
    slot -= page * P.page;
  }
  __syncthreads();
  float cs[VEC], sn[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    cs[j] = turns ? table[col * VEC + j] : 1.f;
    sn[j] = turns ? table[half + col * VEC + j] : 0.f;
  }
  for (int hh = threadIdx.y; hh < heads; hh += blockDim.y) {
    if (hh != threadIdx.y) load(hh);
    const bool is_q = hh < P.Hq, is_v = hh >= P.Hq + P.Hkv;
    if (!is_q && (!keep || (is_v && !P.v_dst))) continue;
    uint16_t* dst =
        is_q ? P.q_out + (tok * P.Hq + hh) * P.D
        : is_v ? P.v_dst + page * P.vc_page + slot * P.vc_tok + (hh - P.Hq - P.Hkv) * P.vc_head
               : P.k_dst + page * P.kc_page + slot * P.kc_tok + (hh - P.Hq) * P.kc_head;
    if (turns && !is_v) {
      if (P.adjacent) {
        uint16_t w[2 * VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = a[j], w[VEC + j] = b[j];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u = elem_f32<T>(w[2 * j]), v = elem_f32<T>(w[2 * j + 1]);
          w[2 * j] = elem_bits<T>(u * cs[j] - v * sn[j]);
          w[2 * j + 1] = elem_bits<T>(v * cs[j] + u * sn[j]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] = w[j], b[j] = w[VEC + j];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u = elem_f32<T>(a[j]), v = elem_f32<T>(b[j]);
          a[j] = elem_bits<T>(u * cs[j] - v * sn[j]);
          b[j] = elem_bits<T>(v * cs[j] + u * sn[j]);
        }
      }
    }
    store_bits<VEC>(dst + (is_v ? c0 : e0), a);
    store_bits<VEC>(dst + (is_v ? c0 + VEC : e1), b);
  }
}

template <typename T, int VEC>
int launch_rope(const RopeParams& P, cudaStream_t stream) {
  const int cols = P.D / (2 * VEC), heads = P.Hq + 2 * P.Hkv;
  const int most = 256 / cols < 1 ? 1 : 256 / cols;
  const int sweeps = (heads + most - 1) / most;
  const dim3 block(cols, (heads + sweeps - 1) / sweeps);
  return cuda_status(launch_pdl(k_rope<T, VEC>, dim3((unsigned)P.tokens), block, 0, stream, P));
}

template <typename T>
int pick_rope(const RopeParams& P, int vec, cudaStream_t stream) {
  return vec == 8   ? launch_rope<T, 8>(P, stream)
         : vec == 4 ? launch_rope<T, 4>(P, stream)
                    : launch_rope<T, 1>(P, stream);
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" int ftb_rope(const ftb_rope_args* a, ftb_stream_t stream) {
  if (!a) return FTB_ERR_ARG;
  if (a->tokens < 0 || a->tokens > 0x7fffffff || a->Hq < 1 || a->Hkv < 1 || a->D < 2 ||
      a->D > 512 || a->D % 2 || a->rot < 2 || a->rot % 2 || a->rot > a->D ||
      a->rot > 2 * kMaxPairs || a->axes < 1 || a->axes > 4 || a->table_rows < 1)
    return FTB_ERR_SHAPE;
  if (a->type != FTB_TYPE_BF16 && a->type != FTB_TYPE_F16) return FTB_ERR_ARG;
  if (a->pairs != FTB_PAIRS_HALF && a->pairs != FTB_PAIRS_ADJACENT) return FTB_ERR_ARG;
  if (a->order != FTB_AXES_BLOCKS && a->order != FTB_AXES_CYCLIC) return FTB_ERR_ARG;
  const int half = a->rot / 2;
  RopeParams P{};
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
  if (a->tokens == 0) return FTB_OK;
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
  // the widest chunk that divides the rotated and the copied part, and that every head of every
  // operand starts aligned to
  auto fits = [&](int n) {
    if (half % n || (a->D - a->rot) % (2 * n) || a->D % (2 * n)) return false;
    uint64_t m = 0;
    const void* ptrs[] = {a->q, a->k, a->q_out, a->k_dst, a->v_dst ? a->v : nullptr, a->v_dst};
    for (const void* p : ptrs) m |= reinterpret_cast<uintptr_t>(p);
    int64_t st = 0;
    for (int i = 0; i < 2; ++i) st |= a->q_strides[i] | a->k_strides[i];
    for (int i = 0; i < 3; ++i) st |= a->k_dst_strides[i];
    if (a->v_dst) {
      for (int i = 0; i < 2; ++i) st |= a->v_strides[i];
      for (int i = 0; i < 3; ++i) st |= a->v_dst_strides[i];
    }
    return (m | (uint64_t)(st * 2)) % (2 * n) == 0;
  };
  const int vec = fits(8) ? 8 : fits(4) ? 4 : 1;
  return a->type == FTB_TYPE_BF16 ? pick_rope<__nv_bfloat16>(P, vec, (cudaStream_t)stream)
                                  : pick_rope<__half>(P, vec, (cudaStream_t)stream);
}
