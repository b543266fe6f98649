// block_norm.cu - the norms before and after a block, fused with its gate and residual scale.
//
//   n = post ? y * rsqrt(mean(y^2) + eps) * post : y        (norm after the block)
//   r = x + scale * act(gate) * n                           (gated, scaled residual)
//   h = r * rsqrt(mean(r^2) + eps) * pre                    (norm before the next block)
//
// One pass: a row of x and y is read once into registers, both sums of squares are block
// reductions over those registers, and r and h are written once. All arithmetic is fp32; h is
// computed from r before r is rounded to its stored type, so each output is rounded once.
//
// Bound: DRAM, rows * H * (2 s_y + 2 s_x) bytes (+ the gate). A row is held by TPR threads,
// VPT vectors of VEC elements each; TPR is the smallest power of two that covers the row, so a
// block holds several short rows or one long one.
#include "ftb_common.cuh"

namespace ftb {
namespace {

struct NormParams {
  const void* x;     // residual stream [rows, H], TR
  const void* y;     // block output [rows, H], TY, or NULL (r = x)
  const void* gate;  // NULL, or [H] / [rows] / [rows, H]
  const void* post;  // [H] or NULL
  const void* pre;   // [H] or NULL (h not computed)
  void* r;           // [rows, H] TR, or NULL (not stored)
  void* h;           // [rows, H] TY
  int64_t rows, x_stride, y_stride, gate_stride;
  int H, gate_kind, gate_act, w_f32, tpr_log2;
  float scale, eps, inv_h;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// VEC consecutive elements as fp32; VEC == 8 takes 16-byte accesses (the pointer is aligned).
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  constexpr int kBytes = VEC * sizeof(T);
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int b = 0; b < kBytes / 16; ++b) {
      const uint4 w = reinterpret_cast<const uint4*>(p)[b];  // plain: r may be x, h may be y
      T t[16 / sizeof(T)];
      memcpy(t, &w, 16);
#pragma unroll
      for (int i = 0; i < (int)(16 / sizeof(T)); ++i) v[b * (16 / sizeof(T)) + i] = to_f32(t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(p[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  constexpr int kBytes = VEC * sizeof(T);
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int b = 0; b < kBytes / 16; ++b) {
      T t[16 / sizeof(T)];
#pragma unroll
      for (int i = 0; i < (int)(16 / sizeof(T)); ++i)
        t[i] = from_f32<T>(v[b * (16 / sizeof(T)) + i]);
      uint4 w;
      memcpy(&w, t, 16);
      reinterpret_cast<uint4*>(p)[b] = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = from_f32<T>(v[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const void* p, bool f32, int c, float (&v)[VEC]) {
  if (f32)
    load_vec<float, VEC>(static_cast<const float*>(p) + c, v);
  else
    load_vec<T, VEC>(static_cast<const T*>(p) + c, v);
}

// Sum over the tpr (a power of two, 32..1024) threads of this thread's row. `red` has one slot
// per warp of the block and is reused: a barrier precedes each write after the first use.
__device__ __forceinline__ float row_sum(float v, int tpr_log2, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr_log2 <= 5) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = 1 << (tpr_log2 - 5);  // warps per row, <= 32
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < per ? red[(warp & ~(per - 1)) + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename TR, typename TY, int VEC, int VPT>
__global__ void __launch_bounds__(1024) k_block_norm(NormParams P) {
  __shared__ float red[2][32];
  pdl_launch_dependents();
  const int tpr = 1 << P.tpr_log2;
  const int t = threadIdx.x & (tpr - 1);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> P.tpr_log2) + (threadIdx.x >> P.tpr_log2);
  const bool live = row < P.rows;
  float y[VPT][VEC], x[VPT][VEC];
  pdl_wait();
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * tpr) * VEC;
    const bool in = live && c < P.H;
    if (in) {
      load_vec<TR, VEC>(static_cast<const TR*>(P.x) + row * P.x_stride + c, x[i]);
      if (P.y) load_vec<TY, VEC>(static_cast<const TY*>(P.y) + row * P.y_stride + c, y[i]);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (!in) x[i][j] = 0.f;
      if (!in || !P.y) y[i][j] = 0.f;
    }
  }
  if (P.y) {
    float a = P.scale;
    if (P.gate_kind == FTB_GATE_TOKEN && live) {
      float g;
      if (P.w_f32)
        g = static_cast<const float*>(P.gate)[row * P.gate_stride];
      else
        g = to_f32(static_cast<const TY*>(P.gate)[row * P.gate_stride]);
      a *= P.gate_act == FTB_GATE_SIGMOID ? sigmoid_f32<false>(g) : g;
    }
    if (P.post) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss += y[i][j] * y[i][j];
      a *= rsqrtf(row_sum(ss, P.tpr_log2, red[0]) * P.inv_h + P.eps);
    }
    const bool vec_gate = P.gate_kind == FTB_GATE_CHANNEL || P.gate_kind == FTB_GATE_FULL;
    const int64_t g0 = P.gate_kind == FTB_GATE_FULL ? row * P.gate_stride : 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * tpr) * VEC;
      if (live && c < P.H) {
        float w[VEC];
        if (P.post) {
          load_weight<TY, VEC>(P.post, P.w_f32, c, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[i][j] *= w[j];
        }
        if (vec_gate) {
          const char* gp = static_cast<const char*>(P.gate) +
                           g0 * (P.w_f32 ? (int64_t)sizeof(float) : (int64_t)sizeof(TY));
          load_weight<TY, VEC>(gp, P.w_f32, c, w);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            y[i][j] *= P.gate_act == FTB_GATE_SIGMOID ? sigmoid_f32<false>(w[j]) : w[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i][j] = fmaf(a, y[i][j], x[i][j]);
        if (P.r) store_vec<TR, VEC>(static_cast<TR*>(P.r) + row * P.H + c, x[i]);
      }
    }
  }
  if (!P.pre) return;
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) ss += x[i][j] * x[i][j];
  const float s = rsqrtf(row_sum(ss, P.tpr_log2, red[1]) * P.inv_h + P.eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * tpr) * VEC;
    if (live && c < P.H) {
      float w[VEC];
      load_weight<TY, VEC>(P.pre, P.w_f32, c, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] *= x[i][j] * s;
      store_vec<TY, VEC>(static_cast<TY*>(P.h) + row * P.H + c, w);
    }
  }
}

template <typename TR, typename TY, int VEC, int VPT>
int launch_norm(NormParams P, cudaStream_t stream) {
  const int64_t need = ceil_div(ceil_div(P.H, VEC), VPT);
  int lg = 5;
  while ((1 << lg) < need) ++lg;
  P.tpr_log2 = lg;
  const int threads = lg < 8 ? 256 : 1 << lg;
  const int64_t grid = ceil_div(P.rows, threads >> lg);
  if (grid > 0x7fffffff) return FTB_ERR_SHAPE;
  return cuda_status(launch_pdl(k_block_norm<TR, TY, VEC, VPT>, dim3((unsigned)grid),
                                dim3(threads), 0, stream, P));
}

template <typename TR, typename TY>
int pick_norm(const NormParams& P, bool vec, cudaStream_t stream) {
  if (vec) {
    if (P.H <= 8 * 1024) return launch_norm<TR, TY, 8, 1>(P, stream);
    return launch_norm<TR, TY, 8, 2>(P, stream);
  }
  if (P.H <= 4 * 1024) return launch_norm<TR, TY, 1, 4>(P, stream);
  return launch_norm<TR, TY, 1, 16>(P, stream);
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" int ftb_block_norm(const ftb_norm_args* a, ftb_stream_t stream) {
  if (!a) return FTB_ERR_ARG;
  if (a->rows < 0 || a->H < 1 || a->H > 16384) return FTB_ERR_SHAPE;
  if (a->type != FTB_TYPE_BF16 && a->type != FTB_TYPE_F16) return FTB_ERR_ARG;
  if (a->residual_type != a->type && a->residual_type != FTB_TYPE_F32) return FTB_ERR_ARG;
  if (a->gate_kind < FTB_GATE_NONE || a->gate_kind > FTB_GATE_FULL) return FTB_ERR_ARG;
  if (a->gate_act != FTB_GATE_LINEAR && a->gate_act != FTB_GATE_SIGMOID) return FTB_ERR_ARG;
  if (a->rows == 0) return FTB_OK;
  if (!a->x || (a->y && !a->r) || (!a->y && !a->pre) || (a->pre && !a->h)) return FTB_ERR_ARG;
  if ((a->gate_kind != FTB_GATE_NONE) != (a->gate != nullptr)) return FTB_ERR_ARG;
  if (!a->y && (a->gate || a->post || a->r)) return FTB_ERR_ARG;
  NormParams P{a->x, a->y, a->gate, a->post, a->pre, a->r, a->h, a->rows, a->x_stride, a->y_stride,
               a->gate_stride, a->H, a->gate_kind, a->gate_act, a->weights_f32, 0, a->scale,
               a->eps, 1.0f / (float)a->H};
  // 16-byte accesses where every row of every operand starts on a 16-byte boundary
  auto rows16 = [&](const void* p, int64_t stride, int size) {
    return aligned16(p) && stride * size % 16 == 0;
  };
  const int rs = a->residual_type == FTB_TYPE_F32 ? 4 : 2, ws = a->weights_f32 ? 4 : 2;
  const bool vec = a->H % 8 == 0 && rows16(a->x, a->x_stride, rs) &&
                   rows16(a->y, a->y ? a->y_stride : 0, 2) && aligned16(a->post) &&
                   aligned16(a->pre) && aligned16(a->r) && aligned16(a->h) &&
                   (a->gate_kind != FTB_GATE_CHANNEL || aligned16(a->gate)) &&
                   (a->gate_kind != FTB_GATE_FULL || rows16(a->gate, a->gate_stride, ws));
  cudaStream_t st = (cudaStream_t)stream;
  const bool f32 = a->residual_type == FTB_TYPE_F32;
  if (a->type == FTB_TYPE_BF16)
    return f32 ? pick_norm<float, __nv_bfloat16>(P, vec, st)
               : pick_norm<__nv_bfloat16, __nv_bfloat16>(P, vec, st);
  return f32 ? pick_norm<float, __half>(P, vec, st) : pick_norm<__half, __half>(P, vec, st);
}
