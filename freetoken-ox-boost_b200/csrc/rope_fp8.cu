// rope_fp8.cu - rotary positions, with the write of the new tokens' keys and values into a cache
// held in e4m3 with one scale for each block of S tokens and kv head.
//
// A call writes rows W of a block (its tokens whose slots lie there). With A the largest |x| that it
// writes for a head (x the turned key or the value, fp32), 2^e the smallest power of two with
// A <= 448 * 2^e, -40 <= e <= 40, and s the scale so far (rounded up to a power of two):
//   s' = 2^e where W has the block's first row (what was there belongs to no sequence any more) or s
//        is no positive finite number, else max(s, 2^e)
//   rows of W:                           c = e4m3(x / s')
//   the others below the last row of W:  c = e4m3(c * s / s')   where s' != s
// Scales are powers of two, so both divisions are exact and a row that is rounded again loses nothing
// but what falls below the new scale's smallest steps. x is rounded once, from fp32; it is computed
// without fused multiply-adds, so that it is the same number wherever it is computed.
//
// The rows of a block are spread over the call's tokens in any order, so a block has one owner: the
// token with its lowest written row. Its thread block collects W, takes the maximum over W and writes
// all of W. In calls of up to kTogether tokens, which have few blocks or few rows in each, the written
// tokens of a block share its heads instead. A call of few tokens finds W by a scan of all slots (kScan);
// a larger one by a table of the token at each slot, written by a small launch before. Entries of the table are checked against the
// slots, so what it held before does not matter; of two tokens with one slot one is kept.
//
// Bound: DRAM, (2 Hq + 2 Hkv) D 2 + 2 Hkv D bytes per token. The blocks are bound by latencies (the
// table, the slots, the tokens, then the second pass over them, which comes from L1), so they come first
// in the grid and the tokens' q, a plain stream, fills the SMs beside them: registers are kept low for
// both. With four items a thread kept in fp32 (171 registers, one block per SM) and q in a launch of its
// own, 19106 tokens of 32 + 8 + 8 heads of 128 took 243 us; they take 104, 4.2 TB/s, 0.66 of the measured
// copy rate; 64 tokens of 64 sequences 6.7 us.
#include "rope.cuh"

namespace ftb {
namespace {

constexpr int kThreads = 256;
constexpr int kPerSm = 4;        // thread blocks per SM
constexpr int kKept = 1;         // items of a thread that stay in registers
constexpr int kItems = 8;        // items of a thread that a thread block is made for
constexpr int kMaxBlock = 128;   // tokens per scale
constexpr int kMaxHeads = 256;   // of a thread block
// Tokens up to which the slots are scanned (one prompt of 1280 tokens 19.8 us, by the table 21.6, of 2048
// 24.3 and 26.5; as many sequences of one token lose: 1280 59 against 55, 2048 90 against 79), and up to
// which a block's tokens share its heads (us, shared / by owners: a prompt of 600 tokens 12.2 / 17.3, 1024
// 18.0 / 19.8, 1280 21.8 / 19.8, 2048 36 / 24; as many sequences of one token 600 18 / 29, 1024 28 / 43,
// 1280 35 / 59).
constexpr int kScan = 2048, kTogether = 1024;
static_assert(kTogether <= kScan, "what is shared is scanned for");
constexpr int kMaxRange = 64;    // tokens per thread block beyond that, at most
constexpr int kManyTokens = 4096;  // from here on a thread block turns q of eight tokens (30.2 us, one: 35.4)
constexpr float kMaxScale = 0x1p40f, kMinScale = 0x1p-40f;

struct AppendParams {
  RopeParams r;
  uint8_t* dst[2];       // caches: k, v
  int64_t st[2][3];      // their {page, row, head} strides
  float* scale[2];
  int64_t scale_st[2][3];  // {page, block, head}
  int32_t* token_at;     // the table; NULL: scan
  int block_log2;
  int splits, per_split;  // thread blocks per token range: K or V, per_split heads each
  int together;
  int append_blocks;
  int range, q_tokens;  // tokens per thread block: of keys and values, of q
};

__device__ __forceinline__ int64_t slot_of(const RopeParams& P, int64_t t) {
  const int64_t s = P.slot64 ? static_cast<const int64_t*>(P.slots)[t]
                             : static_cast<const int32_t*>(P.slots)[t];
  return s >= 0 && s < P.n_slots ? s : -1;
}

// The smallest power of two 2^e with a <= 448 * 2^e, within the limits. 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float a) {
  const uint32_t b = __float_as_uint(a);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);
  e = min(max(e, -40), 40);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// s rounded up to a power of two within the limits; 0 where it is no positive finite number.
__device__ __forceinline__ float scale_so_far(float s) {
  if (!(s > 0.f && s < INFINITY)) return 0.f;
  s = fminf(fmaxf(s, kMinScale), kMaxScale);
  const uint32_t b = __float_as_uint(s);
  return __uint_as_float((b + 0x7fffffu) & 0x7f800000u);
}

__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int VEC>
struct Bytes;
template <>
struct Bytes<8> { using type = uint2; };
template <>
struct Bytes<4> { using type = uint32_t; };
template <>
struct Bytes<1> { using type = uint8_t; };

// VEC numbers times `by`, rounded to e4m3.
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* v, float by) {
  uint8_t w[VEC < 2 ? 2 : VEC];
  if constexpr (VEC == 1) {
    const uint16_t c = to_e4m3x2(v[0] * by, 0.f);
    memcpy(w, &c, 2);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const uint16_t c = to_e4m3x2(v[j] * by, v[j + 1] * by);
      memcpy(w + j, &c, 2);
    }
  }
  typename Bytes<VEC>::type all;
  memcpy(&all, w, VEC);
  *reinterpret_cast<typename Bytes<VEC>::type*>(p) = all;
}

// A thread's column of 2 VEC elements of a head: where its two chunks are, and its turn.
template <typename T, int VEC>
struct Column {
  int col, e0, e1, f0;  // f0: its first frequency
  bool turns;
  __device__ __forceinline__ Column(const RopeParams& P, int c) : col(c) {
    const int half = P.rot / 2, rot_cols = half / VEC;
    turns = col < rot_cols;
    f0 = col * VEC;
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
  }
  struct Raw {
    typename Chunk<VEC>::type a, b;
  };
  __device__ __forceinline__ Raw load(const uint16_t* head) const {
    return Raw{*reinterpret_cast<const typename Chunk<VEC>::type*>(head + e0),
               *reinterpret_cast<const typename Chunk<VEC>::type*>(head + e1)};
  }
  __device__ __forceinline__ void unpack(const Raw& r, float (&x)[2 * VEC]) const {
    uint16_t a[VEC], b[VEC];
    memcpy(a, &r.a, sizeof(a));
    memcpy(b, &r.b, sizeof(b));
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = elem_f32<T>(a[j]), x[VEC + j] = elem_f32<T>(b[j]);
  }
  __device__ __forceinline__ Raw pack(const float (&x)[2 * VEC]) const {
    uint16_t a[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[j] = elem_bits<T>(x[j]), b[j] = elem_bits<T>(x[VEC + j]);
    Raw r;
    memcpy(&r.a, a, sizeof(a));
    memcpy(&r.b, b, sizeof(b));
    return r;
  }
  // cos and sin of token t at this column's frequencies
  __device__ __forceinline__ void angles(const RopeParams& P, int64_t t, float (&cs)[VEC],
                                         float (&sn)[VEC]) const {
    const int half = P.rot / 2;
    auto row = [&](int axis) {
      const int64_t at = axis * P.pos_stride + t;
      const int64_t p = P.pos64 ? static_cast<const int64_t*>(P.positions)[at]
                                : static_cast<const int32_t*>(P.positions)[at];
      return p >= 0 && p < P.table_rows ? p : -1;
    };
    if (P.axes == 1) {
      const int64_t p = row(0);
      if (p >= 0) {
        const float* c = P.table + p * P.rot + f0;
        if constexpr (VEC >= 4) {
#pragma unroll
          for (int j = 0; j < VEC; j += 4) {
            *reinterpret_cast<float4*>(cs + j) = __ldg(reinterpret_cast<const float4*>(c + j));
            *reinterpret_cast<float4*>(sn + j) = __ldg(reinterpret_cast<const float4*>(c + half + j));
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) cs[j] = __ldg(c + j), sn[j] = __ldg(c + half + j);
        }
        return;
      }
    }
    // a position outside the table has no angle: NaN, not another position's
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int f = f0 + j;
      const int64_t p = row(P.axis[f >> 4] >> (2 * (f & 15)) & 3);
      cs[j] = p >= 0 ? __ldg(P.table + p * P.rot + f) : __int_as_float(0x7fffffff);
      sn[j] = p >= 0 ? __ldg(P.table + p * P.rot + half + f) : __int_as_float(0x7fffffff);
    }
  }
  __device__ __forceinline__ void turn(const RopeParams& P, const float (&cs)[VEC],
                                       const float (&sn)[VEC], float (&x)[2 * VEC]) const {
    auto pair = [&](int j, float& u, float& v) {
      const float a = u, b = v;
      u = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
      v = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
    };
    if (P.adjacent) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) pair(j, x[2 * j], x[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) pair(j, x[j], x[VEC + j]);
    }
  }
};

// q of tokens [t0, t1), by all threads of a block. A thread has a column of several heads of one token,
// whose angles it takes once, and asks for the elements of the next head before it turns one.
template <typename T, int VEC>
__device__ __forceinline__ void turn_q(const RopeParams& P, int64_t t0, int64_t t1) {
  const int cols = P.D / (2 * VEC), slots = kThreads / cols;
  const int count = (int)(t1 - t0);
  const int per = slots < count ? 1 : slots / count, tokens = slots / per;  // slots of a token; tokens at once
  const int slot = threadIdx.x / cols;
  if (slot >= per * tokens) return;
  const Column<T, VEC> c(P, threadIdx.x % cols);
  using Raw = typename Column<T, VEC>::Raw;
  for (int64_t t = t0 + slot / per; t < t1; t += tokens) {
    int h = slot % per;
    if (h >= P.Hq) return;
    const uint16_t* src = P.q + t * P.q_st;
    Raw next = c.load(src + h * P.q_sh);
    float cs[VEC], sn[VEC];
    if (c.turns) c.angles(P, t, cs, sn);
    while (h < P.Hq) {
      Raw r = next;
      uint16_t* dst = P.q_out + (t * P.Hq + h) * P.D;
      h += per;
      if (h < P.Hq) next = c.load(src + h * P.q_sh);
      if (c.turns) {
        float x[2 * VEC];
        c.unpack(r, x);
        c.turn(P, cs, sn, x);
        r = c.pack(x);
      }
      *reinterpret_cast<typename Chunk<VEC>::type*>(dst + c.e0) = r.a;
      *reinterpret_cast<typename Chunk<VEC>::type*>(dst + c.e1) = r.b;
    }
  }
}

struct AppendShared {
  int token[kMaxBlock];  // by row of the block: the call's token there, -1: none
  int row[kMaxBlock], tok[kMaxBlock];  // the written rows, ascending
  int n, last, rank;
  uint32_t candidates[kMaxRange / 32];
  uint32_t top[kMaxHeads];  // by head: largest |x|, as bits
  float by[kMaxHeads];      // 1 / scale
  float again[kMaxHeads];   // old scale / scale where they differ, else 0
};

// The block with token t's slot, if t is its owner: heads [h0, h0 + nh) of K (kind 0) or V.
template <typename T, int VEC>
__device__ void append_block(const AppendParams& A, AppendShared& sh, int64_t t, int64_t slot,
                             int kind, int h0, int nh) {
  const RopeParams& P = A.r;
  const int tid = threadIdx.x, lane = tid & 31;
  const int size = 1 << A.block_log2;
  const int64_t block0 = slot >> A.block_log2 << A.block_log2;  // slot of its first row
  const int64_t page = block0 / P.page;
  const int row0 = (int)(block0 - page * P.page);
  for (int r = tid; r < size; r += kThreads) {
    int at = -1;
    if (A.token_at) {
      const int w = A.token_at[block0 + r];
      if (w >= 0 && w < P.tokens && slot_of(P, w) == block0 + r) at = w;
    }
    sh.token[r] = at;
  }
  __syncthreads();
  if (!A.token_at) {
    for (int64_t i = tid; i < P.tokens; i += kThreads) {
      const int64_t s = slot_of(P, i) - block0;
      if (s >= 0 && s < size) atomicMax(&sh.token[s], (int)i);
    }
    __syncthreads();
  }
  if (tid == 0) sh.rank = -1;
  if (tid < 32) {
    int n = 0, last = 0;
    for (int r0 = 0; r0 < size; r0 += 32) {
      const int r = r0 + lane, w = r < size ? sh.token[r] : -1;
      const uint32_t set = __ballot_sync(0xffffffffu, w >= 0);
      const int at = n + __popc(set & ((1u << lane) - 1u));
      if (w >= 0) sh.row[at] = r, sh.tok[at] = w;
      n += __popc(set);
      if (set) last = r0 + 31 - __clz(set);
    }
    if (lane == 0) sh.n = n, sh.last = last;
  }
  for (int h = tid; h < nh; h += kThreads) sh.top[h] = 0;
  __syncthreads();
  const int n = sh.n;
  // The owner's thread block has all heads; or token r of the n written has heads r, r + n, ...
  int h_step = 1;
  if (A.together) {
    if (tid < n && sh.tok[tid] == t) sh.rank = tid;
    __syncthreads();
    const int rank = sh.rank;
    if (rank < 0 || rank >= nh) return;  // (below 0: another token of this slot is kept)
    h0 += rank, h_step = n, nh = (nh - rank + n - 1) / n;
  } else if (n == 0 || sh.tok[0] != t) {
    return;
  }
  const bool fresh = sh.row[0] == 0;
  // old scales, asked for early
  float* scale = A.scale[kind] + page * A.scale_st[kind][0] +
                 (int64_t)(row0 >> A.block_log2) * A.scale_st[kind][1];
  float old = 0.f;
  if (tid < nh && !fresh) old = scale[(h0 + tid * h_step) * A.scale_st[kind][2]];

  // A thread has a column of some heads of some rows: slot / across is its first row, slot % across its
  // first head. Where there are many rows it has all heads of a row, whose angles it takes once a pass;
  // where there are few, the heads lie side by side.
  const int cols = P.D / (2 * VEC), step = kThreads / cols;
  const int slot_in = tid / cols;
  const int across = n >= step ? 1 : min(nh, step / n), down = step / across;
  const bool works = slot_in < across * down;
  const int heads_each = (nh + across - 1) / across, items = (n + down - 1) / down * heads_each;
  const Column<T, VEC> c(P, tid % cols);
  const bool turns = kind == 0 && c.turns;
  const uint16_t* src = kind ? P.v : P.k;
  const int64_t src_st = kind ? P.v_st : P.k_st, src_sh = kind ? P.v_sh : P.k_sh;
  using Raw = typename Column<T, VEC>::Raw;
  struct Item {
    int w, h;
    bool in;
  };
  auto item_at = [&](int i) {  // heads first
    const int k = heads_each == 1 ? i : i / heads_each;
    Item it{slot_in / across + k * down, slot_in % across + (i - k * heads_each) * across, false};
    it.in = works && it.w < n && it.h < nh;
    return it;
  };
  auto get = [&](const Item& it) {
    return c.load(src + sh.tok[it.w] * src_st + (h0 + it.h * h_step) * src_sh);
  };
  float cs[VEC], sn[VEC];
  int angles_of = -1;
  auto number = [&](const Item& it, const Raw& r, float (&x)[2 * VEC]) {
    c.unpack(r, x);
    if (turns) {
      if (it.w != angles_of) c.angles(P, sh.tok[it.w], cs, sn);
      angles_of = it.w;
      c.turn(P, cs, sn, x);
    }
  };
  // (all threads of a warp together: its lanes mostly have one head)
  auto highest = [&](const Item& it, const Raw& r) {
    float m = 0.f;  // (fmaxf passes over NaN)
    if (it.in) {
      float x[2 * VEC];
      number(it, r, x);
#pragma unroll
      for (int j = 0; j < 2 * VEC; ++j) m = fmaxf(m, fabsf(x[j]));
    }
    const uint32_t bits = __float_as_uint(m);
    const int h = min(it.h, nh - 1);
    if (__all_sync(0xffffffffu, h == __shfl_sync(0xffffffffu, h, 0))) {
      const uint32_t most = __reduce_max_sync(0xffffffffu, bits);
      if (lane == 0) atomicMax(&sh.top[h], most);
    } else if (it.in) {
      atomicMax(&sh.top[h], bits);
    }
  };
  Raw kept[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (item_at(i).in) kept[i] = get(item_at(i));
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (i < items) highest(item_at(i), kept[i]);
#pragma unroll 2
  for (int i = kKept; i < items; ++i) {
    const Item it = item_at(i);
    Raw r{};
    if (it.in) r = get(it);
    highest(it, r);
  }
  __syncthreads();
  for (int h = tid; h < nh; h += kThreads) {
    if (h != tid && !fresh) old = scale[(h0 + h * h_step) * A.scale_st[kind][2]];
    const float so_far = fresh ? 0.f : scale_so_far(old);
    const float now = fmaxf(so_far, scale_for(__uint_as_float(sh.top[h])));
    scale[(h0 + h * h_step) * A.scale_st[kind][2]] = now;
    sh.by[h] = 1.f / now;
    sh.again[h] = so_far > 0.f && now != old ? old / now : 0.f;
  }
  __syncthreads();
  uint8_t* dst = A.dst[kind] + page * A.st[kind][0] + (int64_t)row0 * A.st[kind][1];
  const int64_t st_row = A.st[kind][1], st_head = A.st[kind][2];
  auto put = [&](const Item& it, const Raw& r) {
    float x[2 * VEC];
    number(it, r, x);
    uint8_t* to = dst + sh.row[it.w] * st_row + (h0 + it.h * h_step) * st_head;
    store_e4m3<VEC>(to + c.e0, x, sh.by[it.h]);
    store_e4m3<VEC>(to + c.e1, x + VEC, sh.by[it.h]);
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (item_at(i).in) put(item_at(i), kept[i]);
#pragma unroll 2
  for (int i = kKept; i < items; ++i) {
    const Item it = item_at(i);
    if (it.in) put(it, get(it));
  }
  // older rows of heads whose scale moved
  if (!fresh) {
    const int rows = sh.last;
    for (int item = slot_in; slot_in < step && item < nh * rows; item += step) {
      const int h = item / rows, r = item - h * rows;
      const float f = sh.again[h];
      if (f == 0.f || sh.token[r] >= 0) continue;
      uint8_t* at = dst + r * st_row + (h0 + h * h_step) * st_head;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint8_t* p = at + (k ? c.e1 : c.e0);
        typename Bytes<VEC>::type w = *reinterpret_cast<typename Bytes<VEC>::type*>(p);
        uint8_t b[VEC < 2 ? 2 : VEC] = {};
        memcpy(b, &w, VEC);
        float x[VEC < 2 ? 2 : VEC];
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          uint16_t two;
          memcpy(&two, b + j, 2);
          const uint32_t h2 = e4m3x2_to_f16x2(two);
          const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&h2));
          x[j] = u.x, x[j + 1] = u.y;
        }
        store_e4m3<VEC>(p, x, f);
      }
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, kPerSm)
    k_rope_append_fp8(const __grid_constant__ AppendParams A) {
  __shared__ AppendShared sh;
  const RopeParams& P = A.r;
  pdl_launch_dependents();
  pdl_wait();
  if ((int)blockIdx.x >= A.append_blocks) {
    const int64_t t = ((int64_t)blockIdx.x - A.append_blocks) * A.q_tokens;
    turn_q<T, VEC>(P, t, t + A.q_tokens < P.tokens ? t + A.q_tokens : P.tokens);
    return;
  }
  const int split = blockIdx.x % A.splits;
  const int kind = split & 1, h0 = (split >> 1) * A.per_split;
  const int nh = min(A.per_split, P.Hkv - h0);
  const int64_t chunk = blockIdx.x / A.splits;
  // tokens with no written row right below theirs, as far as that is seen at once
  const int64_t t0 = chunk * A.range;
  if (threadIdx.x < kMaxRange) {  // (two warps)
    const int64_t t = t0 + threadIdx.x;
    bool can = false;
    if ((int)threadIdx.x < A.range && t < P.tokens) {
      const int64_t s = slot_of(P, t);
      const bool first = (s & ((1 << A.block_log2) - 1)) == 0;
      if (s >= 0 && A.together) {
        can = true;
      } else if (s >= 0 && !A.token_at) {
        can = first || t == 0 || slot_of(P, t - 1) != s - 1;
      } else if (s >= 0 && A.token_at[s] == t) {
        const int w = first ? -1 : A.token_at[s - 1];
        can = !(w >= 0 && w < P.tokens && slot_of(P, w) == s - 1);
      }
    }
    const uint32_t set = __ballot_sync(0xffffffffu, can);
    if ((threadIdx.x & 31) == 0) sh.candidates[threadIdx.x >> 5] = set;
  }
  __syncthreads();
  for (uint64_t set = sh.candidates[0] | (uint64_t)sh.candidates[1] << 32; set; set &= set - 1) {
    const int64_t t = t0 + __ffsll(set) - 1;
    append_block<T, VEC>(A, sh, t, slot_of(P, t), kind, h0, nh);
    __syncthreads();
  }
}

// The table of the tokens at each slot.
__global__ void __launch_bounds__(kThreads) k_slot_table(const __grid_constant__ AppendParams A) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (t >= A.r.tokens) return;
  const int64_t s = slot_of(A.r, t);
  if (s >= 0) A.token_at[s] = (int32_t)t;
}

template <typename T, int VEC>
int run_append(AppendParams A, cudaStream_t stream) {
  const RopeParams& P = A.r;
  const int64_t T0 = P.tokens;
  const int step = kThreads / (P.D / (2 * VEC));
  // heads per thread block: as many as its registers hold of a full block of tokens
  const int rows = (int)(T0 < (1 << A.block_log2) ? T0 : (1 << A.block_log2));
  int per = step * kItems / rows;
  per = per < 1 ? 1 : per;
  A.together = T0 <= kTogether;
  // (shared, more heads where the blocks would not all be on the SMs at once)
  while (A.together && per < P.Hkv && T0 * 2 * ceil_div(P.Hkv, per) > kPerSm * sm_count()) per *= 2;
  per = per > kMaxHeads ? kMaxHeads : per;
  per = per < 1 ? 1 : per > P.Hkv ? P.Hkv : per;
  A.per_split = per;
  A.splits = 2 * (int)ceil_div(P.Hkv, per);
  // Tokens of a thread block: a block of the cache, so that neighbours have one owner among them; fewer
  // where that would not fill the SMs twice.
  A.range = 1;
  while (!A.together && A.range < kMaxRange && A.range < (1 << A.block_log2) &&
         T0 * A.splits >= (int64_t)A.range * 2 * 2 * kPerSm * sm_count())
    A.range *= 2;
  int64_t blocks = ceil_div(T0, A.range) * A.splits;
  if (blocks + T0 > 0x7fffffff) return FTB_ERR_SHAPE;
  A.append_blocks = (int)blocks;
  if (A.token_at) {
    cudaError_t err = launch_pdl(k_slot_table, dim3((unsigned)ceil_div(T0, kThreads)), dim3(kThreads), 0,
                                 stream, A);
    if (err != cudaSuccess) return cuda_status(err);
  }
  A.q_tokens = T0 >= kManyTokens ? 8 : 1;
  blocks += ceil_div(T0, A.q_tokens);
  return cuda_status(launch_pdl(k_rope_append_fp8<T, VEC>, dim3((unsigned)blocks), dim3(kThreads), 0,
                                stream, A));
}

template <typename T>
int pick_append(const AppendParams& A, int vec, cudaStream_t stream) {
  return vec == 8   ? run_append<T, 8>(A, stream)
         : vec == 4 ? run_append<T, 4>(A, stream)
                    : run_append<T, 1>(A, stream);
}

}  // namespace
}  // namespace ftb

using namespace ftb;

extern "C" {

size_t ftb_rope_fp8_workspace_bytes(int64_t tokens, int64_t n_slots) {
  if (tokens < 0 || n_slots < 0) return 0;
  return FTB_ATTN_ZERO_BYTES + (tokens > kScan ? (size_t)n_slots * 4 : 0);
}

int ftb_rope_fp8(const ftb_rope_fp8_args* args, ftb_stream_t stream) {
  if (!args) return FTB_ERR_ARG;
  const ftb_rope_args* a = &args->rope;
  AppendParams A{};
  const int st = rope_params(a, A.r);
  if (st != FTB_OK) return st;
  const int size = args->scale_block;
  if (size < 16 || size > kMaxBlock || (size & (size - 1)) || a->page < size || a->page % size)
    return FTB_ERR_SHAPE;
  if (a->tokens == 0) return FTB_OK;
  if (!a->slots || !args->k_scale || !args->v_scale) return FTB_ERR_ARG;
  if (a->n_slots < 0 || a->n_slots % a->page) return FTB_ERR_SHAPE;
  if (a->Hkv > 1024) return FTB_ERR_SHAPE;
  while ((1 << A.block_log2) < size) ++A.block_log2;
  A.dst[0] = reinterpret_cast<uint8_t*>(a->k_dst), A.dst[1] = reinterpret_cast<uint8_t*>(a->v_dst);
  A.scale[0] = args->k_scale, A.scale[1] = args->v_scale;
  for (int i = 0; i < 3; ++i) {
    A.st[0][i] = a->k_dst_strides[i], A.st[1][i] = a->v_dst_strides[i];
    A.scale_st[0][i] = args->k_scale_strides[i], A.scale_st[1][i] = args->v_scale_strides[i];
  }
  if (a->tokens > kScan) {
    if (!args->workspace ||
        args->workspace_bytes < ftb_rope_fp8_workspace_bytes(a->tokens, a->n_slots))
      return FTB_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(args->workspace) & 3u) return FTB_ERR_ALIGN;
    A.token_at = reinterpret_cast<int32_t*>(static_cast<char*>(args->workspace) + FTB_ATTN_ZERO_BYTES);
  }
  if ((reinterpret_cast<uintptr_t>(args->k_scale) | reinterpret_cast<uintptr_t>(args->v_scale)) & 3u)
    return FTB_ERR_ALIGN;
  // every element and scale has an address of its own: thread blocks write them side by side
  if (a->k_dst == a->v_dst || args->k_scale == args->v_scale) return FTB_ERR_ARG;
  for (int i = 0; i < 2; ++i) {
    const int64_t pages = a->n_slots / a->page;
    if ((pages > 1 && (A.st[i][0] == 0 || A.scale_st[i][0] == 0)) || A.st[i][1] == 0 ||
        (a->page > size && A.scale_st[i][1] == 0) ||
        (a->Hkv > 1 && (A.st[i][2] == 0 || A.scale_st[i][2] == 0)))
      return FTB_ERR_SHAPE;
  }
  // the widest chunk that divides the turned and the copied part, and that every head of every
  // operand starts aligned to (16-bit tensors, bytes, and the table's floats)
  const int half = a->rot / 2;
  auto fits = [&](int n) {
    if (half % n || (a->D - a->rot) % (2 * n) || a->D % (2 * n)) return false;
    uint64_t wide = 0, bytes = 0;
    for (const void* p : {(const void*)a->q, (const void*)a->k, (const void*)a->v, (const void*)a->q_out})
      wide |= reinterpret_cast<uintptr_t>(p);
    for (int i = 0; i < 2; ++i) wide |= 2 * (uint64_t)(a->q_strides[i] | a->k_strides[i] | a->v_strides[i]);
    bytes |= reinterpret_cast<uintptr_t>(a->k_dst) | reinterpret_cast<uintptr_t>(a->v_dst);
    for (int i = 0; i < 3; ++i) bytes |= (uint64_t)(a->k_dst_strides[i] | a->v_dst_strides[i]);
    return wide % (2 * n) == 0 && bytes % n == 0 &&
           (n < 4 || reinterpret_cast<uintptr_t>(a->table) % 16 == 0);
  };
  const int vec = fits(8) ? 8 : fits(4) ? 4 : 1;
  return a->type == FTB_TYPE_BF16 ? pick_append<__nv_bfloat16>(A, vec, (cudaStream_t)stream)
                                  : pick_append<__half>(A, vec, (cudaStream_t)stream);
}

}  // extern "C"
