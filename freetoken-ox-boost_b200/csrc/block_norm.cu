// block_norm.cu - the norms before and after a block, fused with its gate and residual scale.
//
//   n = post ? y * rsqrt(mean(y^2) + eps) * post : y        (norm after the block)
//   r = x + scale * act(gate) * n                           (gated, scaled residual)
//   h = r * rsqrt(mean(r^2) + eps) * pre                    (norm before the next block)
//
// One pass: a row of x, y and the gate is read once into registers, both sums of squares are
// block reductions over those registers, and r and h are written once. All arithmetic is fp32; h
// is computed from r before r is rounded to its stored type, so each output is rounded once.
//
// Bound: DRAM, rows * H * (2 s_y + 2 s_x) bytes (+ the gate). A row is held by TPR threads (a
// multiple of 32), VPT vectors of VEC elements each, and all of it is loaded before the first
// reduction (the weights come from the L1 cache at their use); the memory is kept busy by many
// small blocks. Few threads with several
// vectors beat many with one: fewer warps per barrier, and as many bytes in flight.
#include <algorithm>
#include <type_traits>

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
  int H, gate_kind, gate_act, w_f32, tpr, per_block;
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

// VEC consecutive elements as loaded (16-byte accesses where VEC == 8: the pointer is aligned
// then), and as fp32. Plain loads: r may be x, h may be y.
template <typename T, int VEC>
struct Raw {
  static constexpr int kWords = VEC * (int)sizeof(T) / 16, kPer = 16 / (int)sizeof(T);
  uint4 w[kWords > 0 ? kWords : 1];
  T e[kWords > 0 ? 1 : VEC];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int b = 0; b < kWords; ++b) w[b] = reinterpret_cast<const uint4*>(p)[b];
#pragma unroll
    for (int i = 0; kWords == 0 && i < VEC; ++i) e[i] = p[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int b = 0; b < kWords; ++b) w[b] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; kWords == 0 && i < VEC; ++i) e[i] = from_f32<T>(0.f);
  }
  // the elements c.. of a row of H that lie inside it, zeros for the others
  __device__ __forceinline__ void load_part(const T* row, int c, int H) {
    T v[VEC];  // loads of a clamped index, not branches around loads: all in flight together
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = row[min(max(c + i, 0), H - 1)];
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (c + i < 0 || c + i >= H) v[i] = from_f32<T>(0.f);
    if constexpr (kWords > 0)
      memcpy(w, v, sizeof(v));
    else
      memcpy(e, v, sizeof(v));
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
#pragma unroll
    for (int b = 0; b < kWords; ++b) {
      T t[kPer];
      memcpy(t, &w[b], 16);
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[b * kPer + i] = to_f32(t[i]);
    }
#pragma unroll
    for (int i = 0; kWords == 0 && i < VEC; ++i) v[i] = to_f32(e[i]);
  }
};
// Elements c..c+7 of an aligned vector of H, where c + s is a multiple of 8 (0 <= s < 8): the two
// aligned vectors that hold them, moved down by 8 - s elements.
template <typename T>
__device__ __forceinline__ void load_shifted(const T* p, int c, int s, int H, Raw<T, 8>& out) {
  Raw<T, 8> a, b;
  a.zero();
  const int lo = c + s - 8, k = 8 - s;
  if (lo >= 0 && lo + 8 <= H)
    a.load(p + lo);
  else if (lo >= 0)
    a.load_part(p, lo, H);
  if (lo + 16 <= H)
    b.load(p + lo + 8);
  else
    b.load_part(p, lo + 8, H);
  constexpr int n = Raw<T, 8>::kWords * 4;  // 32-bit words of 8 elements
  uint32_t w[2 * n];
  memcpy(w, a.w, n * 4);
  memcpy(w + n, b.w, n * 4);
  constexpr int per = sizeof(T) == 2 ? 2 : 1;  // elements per word
  if (k & 8) {
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = w[i + n];
  }
  if (k & 4) {
#pragma unroll
    for (int i = 0; i < 2 * n - 4 / per; ++i) w[i] = w[i + 4 / per];
  }
  if (k & 2) {
#pragma unroll
    for (int i = 0; i < 2 * n - 6 / per; ++i) w[i] = w[i + 2 / per];
  }
  if (k & 1) {
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = per == 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i + 1];
  }
  memcpy(out.w, w, n * 4);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  constexpr int kWords = VEC * (int)sizeof(T) / 16, kPer = 16 / (int)sizeof(T);
#pragma unroll
  for (int b = 0; b < kWords; ++b) {
    T t[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) t[i] = from_f32<T>(v[b * kPer + i]);
    uint4 w;
    memcpy(&w, t, 16);
    reinterpret_cast<uint4*>(p)[b] = w;
  }
#pragma unroll
  for (int i = 0; kWords == 0 && i < VEC; ++i) p[i] = from_f32<T>(v[i]);
}

// Sum over this thread's row: the TPR threads (32, 64, or all of the block's, a multiple of 32)
// that hold it. `red` has one slot per warp of the block and is used once.
__device__ __forceinline__ float row_sum(float v, int tpr, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr <= 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = tpr >> 5, first = per == 2 ? warp & ~1 : 0;  // this row's warps
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < per ? red[first + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// TW: type of gate and weights. MIN_BLOCKS blocks of THREADS threads fit an SM.
// MODE: what the call has besides x, so that a row without a gate of its own spends no registers.
enum { kVector = 0, kFlat = 1, kScalar = 2 };  // how rows are accessed
enum { kNormOnly = 0, kBlock = 1, kBlockGate = 2 };  // kBlockGate: a channel or full gate
// FLAT: rows of a width that is no multiple of 8 follow one another in every operand. A thread then
// owns 8 elements that are aligned in memory, so they start up to 7 before a multiple of 8 of the
// row: all row accesses are vectors but those at a row's two ends.
template <typename TR, typename TY, typename TW, int MODE, bool FLAT, int VEC, int VPT,
          int THREADS, int MIN_BLOCKS>
__global__ void __launch_bounds__(THREADS, MIN_BLOCKS)
    k_block_norm(const __grid_constant__ NormParams P) {
  __shared__ float red[2][32];
  pdl_launch_dependents();
  const int tpr = P.tpr;
  const int mine = tpr == 32 ? threadIdx.x >> 5 : tpr == 64 ? threadIdx.x >> 6 : 0;
  const int t = threadIdx.x - mine * tpr;
  const int64_t row = (int64_t)blockIdx.x * P.per_block + mine;
  const bool live = row < P.rows;
  const bool full = P.gate_kind == FTB_GATE_FULL;
  const bool token = P.gate_kind == FTB_GATE_TOKEN, sig = P.gate_act == FTB_GATE_SIGMOID;
  const int c0 = FLAT ? t * VEC - (int)(row * P.H & 7) : t * VEC;
  Raw<TR, VEC> x[VPT];
  Raw<TY, VEC> y[VPT];
  Raw<TW, VEC> g[VPT];
  auto inside = [&](int c) { return live && c < P.H && (!FLAT || c > -VEC); };
  auto whole = [&](int c) { return !FLAT || (c >= 0 && c + VEC <= P.H); };
  // elements c.. of the row at p; with FLAT also what lies beyond its ends, as long as that is
  // inside the tensor (get() drops it): only the tensor's last vector is taken element by element
  auto load = [&](auto& v, const auto* p, int c) {
    if (!FLAT || row * P.H + c + VEC <= P.rows * P.H)
      v.load(p + c);
    else
      v.load_part(p, c, P.H);
  };
  auto get = [&](const auto& raw, int c, float(&v)[VEC]) {
    raw.get(v);
    if (!whole(c)) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j < 0 || c + j >= P.H) v[j] = 0.f;
    }
  };
  auto load_weight = [&](Raw<TW, VEC>& w, const void* p, int c) {  // elements c.. of [H]
    if constexpr (FLAT)
      load_shifted(static_cast<const TW*>(p), c, (int)(row * P.H & 7), P.H, w);
    else
      w.load(static_cast<const TW*>(p) + c);
  };
  // weights: with FLAT loaded with the row (their ends take element accesses, which are not to
  // wait one after another), else at their use
  Raw<TW, VEC> post[FLAT ? VPT : 1], pre[FLAT ? VPT : 1];
  auto weight = [&](const Raw<TW, VEC>* ready, const void* p, int i, int c, float(&v)[VEC]) {
    if constexpr (FLAT) {
      ready[i].get(v);
    } else {
      Raw<TW, VEC> w;
      load_weight(w, p, c);
      w.get(v);
    }
  };
  auto store = [&](auto* p, int c, const float(&v)[VEC]) {
    if (whole(c)) {
      store_vec(p + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j >= 0 && c + j < P.H) p[c + j] = from_f32<std::decay_t<decltype(*p)>>(v[j]);
    }
  };
  float a = P.scale;
  pdl_wait();
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = c0 + i * tpr * VEC;
    if (!inside(c)) continue;
    if (MODE != kNormOnly) load(y[i], static_cast<const TY*>(P.y) + row * P.y_stride, c);
    load(x[i], static_cast<const TR*>(P.x) + row * P.x_stride, c);
    if (MODE == kBlockGate) {
      if (full)
        load(g[i], static_cast<const TW*>(P.gate) + row * P.gate_stride, c);
      else
        load_weight(g[i], P.gate, c);
    }
  }
  if constexpr (FLAT) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = c0 + i * tpr * VEC;
      if (!inside(c)) continue;
      if (MODE != kNormOnly && P.post) load_weight(post[i], P.post, c);
      if (P.pre) load_weight(pre[i], P.pre, c);
    }
  }
  if (token && live) {
    const float v = to_f32(static_cast<const TW*>(P.gate)[row * P.gate_stride]);
    a *= sig ? sigmoid_f32<false>(v) : v;
  }
  if (MODE != kNormOnly && P.post) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = c0 + i * tpr * VEC;
      if (!inside(c)) continue;
      float v[VEC];
      get(y[i], c, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss += v[j] * v[j];
    }
    a *= rsqrtf(row_sum(ss, P.tpr, red[0]) * P.inv_h + P.eps);
  }
  float r[VPT][VEC], ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = c0 + i * tpr * VEC;
    if (!inside(c)) continue;
    get(x[i], c, r[i]);
    if (MODE != kNormOnly) {
      float n[VEC], w[VEC];
      get(y[i], c, n);
      if (P.post) {
        weight(post, P.post, i, c, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) n[j] *= w[j];
      }
      if (MODE == kBlockGate) {
        get(g[i], c, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) n[j] *= sig ? sigmoid_f32<false>(w[j]) : w[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[i][j] = fmaf(a, n[j], r[i][j]);
      store(static_cast<TR*>(P.r) + row * P.H, c, r[i]);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) ss += r[i][j] * r[i][j];
  }
  if (!P.pre) return;
  const float k = rsqrtf(row_sum(ss, P.tpr, red[1]) * P.inv_h + P.eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = c0 + i * tpr * VEC;
    if (!inside(c)) continue;
    float w[VEC];
    weight(pre, P.pre, i, c, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[j] *= r[i][j] * k;
    store(static_cast<TY*>(P.h) + row * P.H, c, w);
  }
}

template <typename TR, typename TY, typename TW, int MODE, bool FLAT, int VEC, int VPT,
          int THREADS, int MIN_BLOCKS>
int launch_norm(NormParams P, cudaStream_t stream) {
  const int64_t need = ceil_div(ceil_div(P.H + (FLAT ? 7 : 0), VEC), VPT);
  P.tpr = need <= 32 ? 32 : need <= 64 ? 64 : (int)ceil_div(need, 32) * 32;
  const int threads = P.tpr <= 64 ? 128 : P.tpr;
  P.per_block = P.tpr <= 64 ? threads / P.tpr : 1;
  const int64_t grid = ceil_div(P.rows, P.per_block);
  if (threads > THREADS || grid > 0x7fffffff) return FTB_ERR_SHAPE;
  return cuda_status(launch_pdl(k_block_norm<TR, TY, TW, MODE, FLAT, VEC, VPT, THREADS, MIN_BLOCKS>,
                                dim3((unsigned)grid), dim3(threads), 0, stream, P));
}

// Few rows (they all run at once): a thread per vector, for the shortest row (one row of 4096: 2.3 us,
// 3.7 with four vectors per thread). Many rows: several vectors per thread and few threads per row,
// so that each row's two barriers join few warps (4096 rows of 4096, us: bf16 residual 26.0 with
// 4 x 128 threads against 30.9 with 1 x 512, which is 5.2 TB/s; fp32 residual 34.7 with 2 x 256
// against 39.9 with 1 x 512, 5.8 TB/s, 0.89 of the measured copy rate).
// Rows at an odd width as vectors (FLAT): 4096 rows of 4095 52.6 us, 66 element by element.
template <typename TR, typename TY, typename TW, int MODE>
int pick_norm(const NormParams& P, int kind, cudaStream_t stream) {
  if (kind == kScalar) {
    if (P.H <= 2048) return launch_norm<TR, TY, TW, MODE, false, 1, 8, 256, 4>(P, stream);
    if (P.H <= 4096) return launch_norm<TR, TY, TW, MODE, false, 1, 8, 512, 2>(P, stream);
    return launch_norm<TR, TY, TW, MODE, false, 1, 16, 1024, 1>(P, stream);
  }
  if (kind == kFlat) {
    // (a row may touch one more vector than it would from an aligned start)
    if (P.H <= 2048) return launch_norm<TR, TY, TW, MODE, true, 8, 2, 160, 5>(P, stream);
    if (P.H <= 4096) return launch_norm<TR, TY, TW, MODE, true, 8, 2, 288, 3>(P, stream);
    if (P.H <= 8192) return launch_norm<TR, TY, TW, MODE, true, 8, 2, 544, 1>(P, stream);
    return launch_norm<TR, TY, TW, MODE, true, 8, 4, 544, 1>(P, stream);
  }
  const bool few = P.rows <= 2 * sm_count();
  if (P.H <= (few ? 2048 : 256)) return launch_norm<TR, TY, TW, MODE, false, 8, 1, 256, 4>(P, stream);
  if (P.H <= 4096 && few) return launch_norm<TR, TY, TW, MODE, false, 8, 1, 512, 2>(P, stream);
  if (P.H <= 2048) return launch_norm<TR, TY, TW, MODE, false, 8, 2, 128, 8>(P, stream);
  if (P.H <= 4096) {
    if constexpr (sizeof(TR) == 2)
      return launch_norm<TR, TY, TW, MODE, false, 8, 4, 128, MODE == kBlockGate ? 6 : 8>(P, stream);
    else
      return launch_norm<TR, TY, TW, MODE, false, 8, 2, 256, 4>(P, stream);
  }
  if (P.H <= 8192) return launch_norm<TR, TY, TW, MODE, false, 8, 2, 512, 2>(P, stream);
  return launch_norm<TR, TY, TW, MODE, false, 8, 2, 1024, 1>(P, stream);
}

template <typename TR, typename TY, typename TW>
int pick_mode(const NormParams& P, int kind, cudaStream_t stream) {
  if (!P.y) return pick_norm<TR, TY, TW, kNormOnly>(P, kind, stream);
  const bool gate = P.gate_kind == FTB_GATE_CHANNEL || P.gate_kind == FTB_GATE_FULL;
  return gate ? pick_norm<TR, TY, TW, kBlockGate>(P, kind, stream)
              : pick_norm<TR, TY, TW, kBlock>(P, kind, stream);
}

template <typename TR, typename TY>
int pick_weights(const NormParams& P, int kind, cudaStream_t stream) {
  return P.w_f32 ? pick_mode<TR, TY, float>(P, kind, stream) : pick_mode<TR, TY, TY>(P, kind, stream);
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
  NormParams P{};
  P.x = a->x, P.y = a->y, P.gate = a->gate, P.post = a->post, P.pre = a->pre, P.r = a->r, P.h = a->h;
  P.rows = a->rows, P.x_stride = a->x_stride, P.y_stride = a->y_stride;
  P.gate_stride = a->gate_stride, P.H = a->H, P.gate_kind = a->gate_kind;
  P.gate_act = a->gate_act, P.w_f32 = a->weights_f32;
  P.scale = a->scale, P.eps = a->eps, P.inv_h = 1.0f / (float)a->H;
  // Row accesses are 16-byte vectors where every row starts on a 16-byte boundary, or where the rows
  // follow one another from one; else element by element.
  const int rs = a->residual_type == FTB_TYPE_F32 ? 4 : 2, ws = a->weights_f32 ? 4 : 2;
  const bool full = a->gate_kind == FTB_GATE_FULL;
  bool rows16 = a->H % 8 == 0, flat = true, starts16 = aligned16(a->r) && aligned16(a->h);
  auto look = [&](const void* p, int64_t stride, int size) {
    if (!p) return;
    starts16 &= aligned16(p);
    rows16 &= stride * size % 16 == 0;
    flat &= stride == a->H;
  };
  look(a->x, a->x_stride, rs);
  look(a->y, a->y_stride, 2);
  if (full) look(a->gate, a->gate_stride, ws);
  const bool weights16 = aligned16(a->post) && aligned16(a->pre) &&
                         (a->gate_kind != FTB_GATE_CHANNEL || aligned16(a->gate));
  const int kind = !starts16 || !weights16 ? kScalar : rows16 ? kVector : flat ? kFlat : kScalar;
  cudaStream_t st = (cudaStream_t)stream;
  const bool f32 = a->residual_type == FTB_TYPE_F32;
  if (a->type == FTB_TYPE_BF16)
    return f32 ? pick_weights<float, __nv_bfloat16>(P, kind, st)
               : pick_weights<__nv_bfloat16, __nv_bfloat16>(P, kind, st);
  return f32 ? pick_weights<float, __half>(P, kind, st) : pick_weights<__half, __half>(P, kind, st);
}
