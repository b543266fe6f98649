// attn_stream.cu - paged attention for few query rows per kv head (single-token decode).
//
// For one sequence and kv head the rows are its new tokens x the G query heads that share the kv
// head; 16 of them (row tile blockIdx.y) are the M of mma.sync.m16n8k16. Every key and value row
// is read once from DRAM and used by all rows:
//   S = Q K^T (fp32),  m, l = running maximum and sum per row,  O = O 2^(m_old - m) + P V.
// Bound: DRAM, 2 * D * 2 bytes per key and kv head. On one B200, bf16, 32 heads of 128 over 8: 61
// tokens at up to 8192 keys (850 MB) 151 us, 5.6 TB/s, 0.86 of the measured copy rate; 3 at up to
// 131072 keys (754 MB) 128 us, 5.9 TB/s; one at 777 keys 10.8 us, latency of the chain of loads,
// join and launch. DRAM traffic is 1.04 of the algorithmic bytes; what is left is mostly the spread
// between SMs (241K cycles on average, 276K the slowest: equal shares, unequal distances to the
// memory). Four shares taken in turn per block instead of one cost more in restarts and joins than
// they evened out (146 -> 157 us, 128 -> 194, before P was two operands).
//
// P is two operands, its rounding to the tensors' type and what that left, each with its own MMAs: the
// output's error is then its own rounding alone, where P rounded once adds as much again (few
// outputs, as a single token has, may show more than that on average). It costs little beside the
// loads: 147 -> 151 us, 10.6 -> 10.8 and nothing on the longest.
//
// Split: the work of all (sequence, kv head) pairs, in tiles of 64 keys, is one line cut into
// gridDim.x equal shares, whatever the lengths; a block finds its share by a scan over the batch
// and walks it from pair to pair. A pair that several blocks share leaves (m, l, O) of each part
// in the workspace, and the last block to finish joins the parts in their order in the sequence
// (so the result does not depend on the order of arrival).
//
// A block is one producer warp and four consumer warps. The producer copies a tile's K and V
// pages with TMA into a ring (mbarriers, bounded waits); warp w takes keys 16w..16w+15 of each
// tile with its own m, l and O, and the four are joined in shared memory at the end of a pair.
//
// The consumers share barriers without a limit, so a warp whose wait gives up passes them all the
// same: it takes no more tiles, makes its rows' sums NaN, and walks on through its share's joins
// and counts. Every block so ends, and the counters return to zero.
#include "attn.cuh"

namespace ftb {
namespace {

constexpr int kTile = 64;  // keys per stage
constexpr int kConsumers = 4, kThreads = (kConsumers + 1) * kWarp;
constexpr int kRows = 16;
constexpr int kMergeCols = 32, kMergePitch = kMergeCols + 8;  // pitch: 8 rows hit 32 banks
constexpr int kCtasPerSm = 2;

constexpr int stream_stages(int DP) { return DP == 128 ? 3 : 6; }
template <int DP>
struct StreamSmem {
  static constexpr int kStages = stream_stages(DP);
  alignas(1024) uint8_t ring[kStages][2][kTile * DP * 2];
  alignas(16) float merge[kConsumers][kRows][kMergePitch];
  float ml[kConsumers][kRows][2];
  float fac[kConsumers][kRows];  // weight of each warp's part of a row
  float row_m[kRows], row_l[kRows];
  uint64_t full[kStages], empty[kStages];
  int64_t scan[kThreads / kWarp];
  int64_t start_item;  // line position of the start pair's first tile
  int64_t total;
  int start_seq;
  int flag;
  int abort;
};

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    mma_16816_f16(d, a[0], a[1], a[2], a[3], b0, b1);
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
// Key tiles of a pair of sequence b in this row tile.
struct PairTiles {
  int lo, hi;  // keys
  int t0, t1;  // tiles
};
__device__ __forceinline__ PairTiles pair_tiles(const AttnParams& P, const AttnSeq& s, int row0) {
  PairTiles t{0, 0, 0, 0};
  const int64_t rows = (int64_t)s.n * P.G;
  if (row0 >= rows) return t;
  const int last = (int)(rows < row0 + kRows ? rows : row0 + kRows) - 1;
  const KeyRange k = attn_range(P, s, row0 / P.G, last / P.G);
  if (k.lo >= k.hi) return t;
  t.lo = k.lo, t.hi = k.hi, t.t0 = k.lo / kTile, t.t1 = (k.hi + kTile - 1) / kTile;
  return t;
}

// The walk over a block's share of the line; producer and consumers take the same steps.
struct Walk {
  int seq, head, tile;  // next tile of pair (seq, head)
  int64_t item;         // line position of the pair's first tile
  int64_t left;         // tiles of the share still to do
  AttnSeq s;
  PairTiles t;
  __device__ void start(const AttnParams& P, int row0, int seq0, int64_t seq_at, int64_t at,
                        int64_t count) {
    seq = seq0;
    s = attn_seq(P, seq);
    t = pair_tiles(P, s, row0);
    const int64_t off = at - seq_at;  // into the sequence's Hkv pairs
    const int n = t.t1 - t.t0;
    head = (int)(off / n);
    item = seq_at + (int64_t)head * n;
    tile = t.t0 + (int)(at - item);
    left = count;
  }
  // tiles of the current pair in this share
  __device__ int take() const {
    const int n = t.t1 - tile;
    return left < n ? (int)left : n;
  }
  __device__ void next(const AttnParams& P, int row0, int done) {
    left -= done;
    tile += done;
    if (left <= 0) return;
    item += t.t1 - t.t0;  // left > 0: the pair is done
    if (++head == P.Hkv) {
      head = 0;
      do {
        ++seq;  // left > 0: a later sequence has tiles
        s = attn_seq(P, seq);
        t = pair_tiles(P, s, row0);
      } while (t.t1 == t.t0);
    }
    tile = t.t0;
  }
};

template <int DP>
struct StreamSync {
  StreamSmem<DP>* sh;
  uint32_t* status;
  __device__ bool wait(uint64_t* bar, uint32_t parity) const {
    if (mbar_try_wait(bar, parity)) return true;
    volatile int* ab = &sh->abort;
    for (uint32_t i = 0; i < kSpinLimit; ++i) {
      if (*ab) return false;
      if (mbar_try_wait(bar, parity)) return true;
      if (i > 1024) __nanosleep(64);
    }
    *ab = 1;
    atomicOr(status, kAttnTimeout);
    return false;
  }
};

// One warp. Copies the tiles of the share into the ring.
template <int DP>
__device__ void stream_producer(const AttnParams& P, const AttnMaps& M, StreamSmem<DP>* sh,
                                Walk w, int row0) {
  constexpr int kStages = StreamSmem<DP>::kStages;
  const int lane = threadIdx.x & 31;
  const StreamSync<DP> sy{sh, P.status};
  const int page = 1 << P.page_log2;
  const int r = page < kTile ? page : kTile;  // keys per box
  const int boxes = kTile / r;                // <= 8
  const bool whole = P.D == DP;               // a box holds every half
  const uint32_t box_bytes = (uint32_t)r * DP * 2;
  int stage = 0;
  uint32_t parity = 1, issued = 0;
  bool ok = true;
  while (w.left > 0 && ok) {
    const int n = w.take();
    for (int j = 0; j < n && ok; ++j) {
      const int key0 = (w.tile + j) * kTile;
      // boxes with a key in [lo, hi)
      const int b0 = w.t.lo > key0 ? (w.t.lo - key0) / r : 0;
      int b1 = (w.t.hi - key0 + r - 1) / r;
      if (b1 > boxes) b1 = boxes;
      int id = 0, row = 0;
      const bool mine = lane >= b0 && lane < b1;
      if (mine) {
        const int key = key0 + lane * r;
        id = P.block_table[(int64_t)w.seq * P.table_stride + (key >> P.page_log2)];
        row = key & (page - 1);
        if (id < 0 || id >= P.num_pages) {
          atomicOr(P.status, kAttnBadPage);
          id = (int)P.num_pages;  // outside the tensor: reads zeros
        }
      }
      ok = __all_sync(0xffffffffu, sy.wait(&sh->empty[stage], parity));
      if (!ok) break;
      ++issued;
      if (lane == 0)
        mbar_arrive_expect_tx(&sh->full[stage], 2u * (uint32_t)(b1 - b0) * box_bytes);
      __syncwarp();
      if (mine) {
        const uint32_t dk = smem_u32(sh->ring[stage][0]) + lane * box_bytes;
        const uint32_t dv = smem_u32(sh->ring[stage][1]) + lane * box_bytes;
        if (whole) {
          tma_5d(dk, &M.k, 0, row, w.head, id, 0, &sh->full[stage]);
          tma_5d(dv, &M.v, 0, row, w.head, id, 0, &sh->full[stage]);
        } else {
#pragma unroll
          for (int h = 0; h < DP / 64; ++h) {
            tma_5d(dk + h * r * 128, &M.k, h * 64, row, w.head, id, 0, &sh->full[stage]);
            tma_5d(dv + h * r * 128, &M.v, h * 64, row, w.head, id, 0, &sh->full[stage]);
          }
        }
      }
      if (++stage == kStages) stage = 0, parity ^= 1u;
    }
    w.next(P, row0, n);
  }
  // Stay until the last copies have landed, again with a limit: a consumer that gave up leaves
  // without them.
  for (uint32_t u = issued > kStages ? issued - kStages : 0; u < issued; ++u)
    for (uint32_t i = 0; i < kSpinLimit; ++i)
      if (mbar_try_wait(&sh->full[u % kStages], (u / kStages) & 1u)) break;
}

template <typename T, int DP>
__device__ void stream_consumer(const AttnParams& P, StreamSmem<DP>* sh, Walk w, int row0,
                                int64_t share) {
  constexpr int kStages = StreamSmem<DP>::kStages;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  const StreamSync<DP> sy{sh, P.status};
  const int page = 1 << P.page_log2;
  const int r = page < kTile ? page : kTile;
  const int half_bytes = r * 128, box_bytes = half_bytes * (DP / 64);
  // ldmatrix addresses of this lane: its key row's offset in the tile, and the row's swizzle
  const int mi = lane >> 3;
  const int kk = warp * 16 + (mi >> 1) * 8 + (lane & 7);  // K: matrices (keys 0-7, 8-15) x 2 chunks
  const int kv = warp * 16 + (mi & 1) * 8 + (lane & 7);   // V: 2 key groups x 2 chunks
  const int k_off = (kk / r) * box_bytes + (kk % r) * 128, k_sw = (kk % r) & 7;
  const int v_off = (kv / r) * box_bytes + (kv % r) * 128, v_sw = (kv % r) & 7;
  const int kc = mi & 1, vc = mi >> 1;
  int stage = 0;
  uint32_t parity = 0;  // + kGaveUp once a wait did (one register for both)
  constexpr uint32_t kGaveUp = 2;
  while (w.left > 0) {
    const int n = w.take();
    const AttnSeq s = w.s;
    const int rows_all = s.n * P.G - row0;
    const int rows = rows_all < kRows ? rows_all : kRows;
    // this lane's rows: limits on their keys, and Q fragments
    uint32_t qa[DP / 16][4];
    int kmin[2], kmax[2];  // keys kmin <= j < kmax
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = row0 + g + 8 * e;
      const int i = row / P.G, hq = w.head * P.G + row % P.G;
      const bool in = g + 8 * e < rows;
      kmin[e] = kmax[e] = 0;
      if (in) {
        const KeyRange k = attn_range(P, s, i, i);
        kmin[e] = k.lo, kmax[e] = k.hi;
      }
      const uint16_t* qp = P.q + (int64_t)(s.q0 + i) * P.q_st + (int64_t)hq * P.q_sh;
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const int d = c * 16 + t2;
        qa[c][e] = in && d < P.D ? *reinterpret_cast<const uint32_t*>(qp + d) : 0u;
        qa[c][2 + e] = in && d + 8 < P.D ? *reinterpret_cast<const uint32_t*>(qp + d + 8) : 0u;
      }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    for (int j = 0; j < n && parity < kGaveUp; ++j) {
      const int key0 = (w.tile + j) * kTile + warp * 16;
      if (!__all_sync(0xffffffffu, sy.wait(&sh->full[stage], parity))) {
        parity = kGaveUp;
        break;
      }
      const uint32_t kb = smem_u32(sh->ring[stage][0]), vb = smem_u32(sh->ring[stage][1]);
      float sc[2][4] = {};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        uint32_t b[4];
        const int chunk = (2 * c + kc) & 7;
        ldsm4(kb + k_off + (c >> 2) * half_bytes + ((chunk ^ k_sw) << 4), b);
        mma16816<T>(sc[0], qa[c], b[0], b[1]);
        mma16816<T>(sc[1], qa[c], b[2], b[3]);
      }
      // a warp's 16 keys, all seen by all of the tile's rows, need no mask
      const bool clean = key0 >= w.t.lo && key0 + 16 <= w.t.hi && (!P.causal || s.n == 1) &&
                         (P.window <= 0 || s.n == 1);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + h * 8 + t2 + (i & 1);
          const bool seen = clean || (key >= kmin[i >> 1] && key < kmax[i >> 1]);
          sc[h][i] = seen ? sc[h][i] * P.scale_log2 : -INFINITY;
        }
      uint32_t pa[4], pr[4];  // P rounded to the operand's type, and what the rounding left
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(fmaxf(sc[0][2 * e], sc[0][2 * e + 1]), fmaxf(sc[1][2 * e], sc[1][2 * e + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[e], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(m[e] - ref);
        m[e] = mn;
        float p0 = ex2(sc[0][2 * e] - ref), p1 = ex2(sc[0][2 * e + 1] - ref);
        float p2 = ex2(sc[1][2 * e] - ref), p3 = ex2(sc[1][2 * e + 1] - ref);
        l[e] = l[e] * f + ((p0 + p1) + (p2 + p3));
        pa[e] = pack2<T>(p0, p1);
        pa[2 + e] = pack2<T>(p2, p3);
        const float2 a = unpack2<T>(pa[e]), b = unpack2<T>(pa[2 + e]);
        pr[e] = pack2<T>(p0 - a.x, p1 - a.y);
        pr[2 + e] = pack2<T>(p2 - b.x, p3 - b.y);
        if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
          for (int jj = 0; jj < DP / 8; ++jj) o[jj][2 * e] *= f, o[jj][2 * e + 1] *= f;
        }
      }
      // V rows outside [lo, hi) have weight 0 but may hold NaN or infinity: made zero
      const bool inside = key0 >= w.t.lo && key0 + 16 <= w.t.hi;
      uint32_t mk[2] = {0xffffffffu, 0xffffffffu};
      if (!inside) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key0 + h * 8 + t2;
          mk[h] = (key >= w.t.lo && key < w.t.hi ? 0xffffu : 0u) |
                  (key + 1 >= w.t.lo && key + 1 < w.t.hi ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        uint32_t b[4];
        const int chunk = (2 * c + vc) & 7;
        ldsm4_t(vb + v_off + (c >> 2) * half_bytes + ((chunk ^ v_sw) << 4), b);
        if (!inside) b[0] &= mk[0], b[1] &= mk[1], b[2] &= mk[0], b[3] &= mk[1];
        mma16816<T>(o[2 * c], pa, b[0], b[1]);
        mma16816<T>(o[2 * c + 1], pa, b[2], b[3]);
        mma16816<T>(o[2 * c], pr, b[0], b[1]);
        mma16816<T>(o[2 * c + 1], pr, b[2], b[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->empty[stage]);
      if (++stage == kStages) stage = 0, parity ^= 1u;
    }
    if (parity >= kGaveUp) l[0] = l[1] = NAN;
    // join the four warps' parts of the rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if ((lane & 3) == 0) {
        sh->ml[warp][g + 8 * e][0] = m[e];
        sh->ml[warp][g + 8 * e][1] = l[e];
      }
    }
    named_bar(1, kConsumers * kWarp);
    if (threadIdx.x < kRows) {
      const int row = threadIdx.x;
      float mm = sh->ml[0][row][0];
      for (int i = 1; i < kConsumers; ++i) mm = fmaxf(mm, sh->ml[i][row][0]);
      const float ref = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      for (int i = 0; i < kConsumers; ++i) {
        const float f = ex2(sh->ml[i][row][0] - ref);
        sh->fac[i][row] = f;
        ll += f * sh->ml[i][row][1];
      }
      sh->row_m[row] = mm;
      sh->row_l[row] = ll;
    }
    named_bar(1, kConsumers * kWarp);
    const bool begins = w.tile == w.t.t0, ends = w.tile + n == w.t.t1;
    const bool whole = begins && ends;
    // part slots: 2 per block; 0 for a pair this block did not begin, 1 for one it did
    const int64_t blk = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    constexpr int kSlot = kRows * DP + 2 * kRows;
    float* slot = P.partial + (2 * blk + (begins ? 1 : 0)) * kSlot;
    const float f0 = sh->fac[warp][g], f1 = sh->fac[warp][g + 8];
    const int orow = threadIdx.x >> 3, oc = (threadIdx.x & 7) * 4;  // 16 rows x 8 threads x 4
#pragma unroll
    for (int c = 0; c < DP / kMergeCols; ++c) {
#pragma unroll
      for (int jj = 0; jj < kMergeCols / 8; ++jj) {
        const float(&v)[4] = o[c * (kMergeCols / 8) + jj];
        *reinterpret_cast<float2*>(&sh->merge[warp][g][jj * 8 + t2]) = make_float2(v[0] * f0, v[1] * f0);
        *reinterpret_cast<float2*>(&sh->merge[warp][g + 8][jj * 8 + t2]) = make_float2(v[2] * f1, v[3] * f1);
      }
      named_bar(1, kConsumers * kWarp);
      float4 a = *reinterpret_cast<float4*>(&sh->merge[0][orow][oc]);
#pragma unroll
      for (int i = 1; i < kConsumers; ++i) {
        const float4 b = *reinterpret_cast<float4*>(&sh->merge[i][orow][oc]);
        a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
      }
      const int d = c * kMergeCols + oc;
      if (orow < rows) {
        if (!whole) {
          *reinterpret_cast<float4*>(slot + orow * DP + d) = a;
        } else if (d < P.D) {
          const float inv = sh->row_l[orow] > 0.f || sh->row_l[orow] != sh->row_l[orow]
                                ? 1.f / sh->row_l[orow] : 0.f;
          const int row = row0 + orow;
          uint16_t* op = P.out + ((int64_t)(s.q0 + row / P.G) * P.Hq + w.head * P.G + row % P.G) * P.D + d;
          *reinterpret_cast<uint2*>(op) =
              make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
        }
      }
      named_bar(1, kConsumers * kWarp);
    }
    if (whole) {
      if (P.lse && threadIdx.x < rows) {
        const int row = row0 + threadIdx.x;
        P.lse[(int64_t)(s.q0 + row / P.G) * P.Hq + w.head * P.G + row % P.G] =
            sh->row_l[threadIdx.x] == 0.f
                ? -INFINITY
                : (sh->row_m[threadIdx.x] + log2f(sh->row_l[threadIdx.x])) * 0.69314718055994531f;
      }
    } else {
      if (threadIdx.x < rows) {
        slot[kRows * DP + threadIdx.x] = sh->row_m[threadIdx.x];
        slot[kRows * DP + kRows + threadIdx.x] = sh->row_l[threadIdx.x];
      }
      // blocks c0..c1 hold the pair's parts: the last one to get here joins them
      const int64_t c0 = w.item / share, c1 = (w.item + (w.t.t1 - w.t.t0) - 1) / share;
      const int64_t blk0 = (int64_t)blockIdx.y * gridDim.x + c0;
      const int parts = (int)(c1 - c0) + 1;
      __threadfence();
      named_bar(1, kConsumers * kWarp);
      if (threadIdx.x == 0) {
        const bool last = atomicAdd(&P.counters[blk0], 1) == parts - 1;
        if (last) P.counters[blk0] = 0;
        sh->flag = last;
        __threadfence();
      }
      named_bar(1, kConsumers * kWarp);
      if (sh->flag) {
        // part 0 is slot 1 of its block (it began the pair), the others slot 0 of theirs
        const float* p0 = P.partial + (2 * blk0 + 1) * kSlot;
        const float* p1 = P.partial + 2 * (blk0 + 1) * kSlot;
        // Where there are few rows, the threads of the others take their share of the parts: part i
        // goes to way i % ways of its row (one token at 777 keys 11.2 -> 10.6 us, at 4096 16.0 -> 14.9).
        const int lg = rows > 1 ? 32 - __clz(rows - 1) : 0, ways = kRows >> lg;
        const int jrow = orow & ((1 << lg) - 1), way = orow >> lg;
        const bool mine = jrow < rows;
        float mm = -INFINITY, ll = 0.f;
        float4 acc[DP / kMergeCols];
#pragma unroll
        for (int c = 0; c < DP / kMergeCols; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float f, const float4& b, int c) {
          acc[c].x += f * b.x, acc[c].y += f * b.y, acc[c].z += f * b.z, acc[c].w += f * b.w;
        };
        if (mine) {
          for (int i = way; i < parts; i += ways) {
            const float* p = i == 0 ? p0 : p1 + (int64_t)(i - 1) * 2 * kSlot;
            mm = fmaxf(mm, __ldcg(p + kRows * DP + jrow));
          }
          const float ref = mm == -INFINITY ? 0.f : mm;
          for (int i = way; i < parts; i += ways) {
            const float* p = i == 0 ? p0 : p1 + (int64_t)(i - 1) * 2 * kSlot;
            const float f = ex2(__ldcg(p + kRows * DP + jrow) - ref);
            ll += f * __ldcg(p + kRows * DP + kRows + jrow);
#pragma unroll
            for (int c = 0; c < DP / kMergeCols; ++c)
              add(f, __ldcg(reinterpret_cast<const float4*>(p + jrow * DP + c * kMergeCols + oc)), c);
          }
        }
        if (ways > 1) {
          static_assert(kConsumers * kMergePitch >= DP, "the ways' sums fit the merge buffer");
          float* all = &sh->merge[0][0][0];
#pragma unroll
          for (int c = 0; c < DP / kMergeCols; ++c)
            *reinterpret_cast<float4*>(all + orow * DP + c * kMergeCols + oc) = acc[c];
          if (oc == 0) sh->ml[0][orow][0] = mm, sh->ml[0][orow][1] = ll;
          named_bar(1, kConsumers * kWarp);
          if (mine && way == 0) {
            for (int i = 1; i < ways; ++i) mm = fmaxf(mm, sh->ml[0][jrow + (i << lg)][0]);
            const float ref = mm == -INFINITY ? 0.f : mm;
            ll = 0.f;
#pragma unroll
            for (int c = 0; c < DP / kMergeCols; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < ways; ++i) {
              const int at = jrow + (i << lg);
              const float f = ex2(sh->ml[0][at][0] - ref);
              ll += f * sh->ml[0][at][1];
#pragma unroll
              for (int c = 0; c < DP / kMergeCols; ++c)
                add(f, *reinterpret_cast<const float4*>(all + at * DP + c * kMergeCols + oc), c);
            }
          }
          named_bar(1, kConsumers * kWarp);  // (the next pair writes the merge buffer)
        }
        if (mine && way == 0) {
          const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
          const int row = row0 + jrow;
          const int64_t at = (int64_t)(s.q0 + row / P.G) * P.Hq + w.head * P.G + row % P.G;
#pragma unroll
          for (int c = 0; c < DP / kMergeCols; ++c) {
            const int d = c * kMergeCols + oc;
            if (d < P.D)
              *reinterpret_cast<uint2*>(P.out + at * P.D + d) = make_uint2(
                  pack2<T>(acc[c].x * inv, acc[c].y * inv), pack2<T>(acc[c].z * inv, acc[c].w * inv));
          }
          if (P.lse && oc == 0)
            P.lse[at] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
        }
      }
    }
    w.next(P, row0, n);
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    k_attn_stream(const __grid_constant__ AttnMaps M, const __grid_constant__ AttnParams P) {
  extern __shared__ uint8_t smem_raw[];
  StreamSmem<DP>* sh = reinterpret_cast<StreamSmem<DP>*>(
      smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.y * kRows;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < StreamSmem<DP>::kStages; ++i) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->empty[i], kConsumers);
    }
    sh->abort = 0;
    fence_mbar_init();
    prefetch_map(&M.k);
    prefetch_map(&M.v);
  }
  pdl_wait();
  // scan over the batch: thread i has sequences [i * per, (i + 1) * per)
  const int per = (P.batch + kThreads - 1) / kThreads;
  const int b0 = threadIdx.x * per, b1 = b0 + per < P.batch ? b0 + per : P.batch;
  int64_t mine = 0;
  bool empty = false;
  for (int b = b0; b < b1; ++b) {
    const AttnSeq s = attn_seq(P, b);
    const PairTiles t = pair_tiles(P, s, row0);
    mine += (int64_t)(t.t1 - t.t0) * P.Hkv;
    if (blockIdx.x == 0 && blockIdx.y == 0 && (s.bad_len || s.bad_rows))
      atomicOr(P.status, (s.bad_len ? kAttnBadPage : 0u) | (s.bad_rows ? kAttnBadRows : 0u));
    empty |= t.t1 == t.t0 && (int64_t)s.n * P.G > row0;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh->scan[warp] = incl;
  const bool any_empty = __syncthreads_or(empty);
  int64_t before = 0, total = 0;
  for (int i = 0; i < kThreads / kWarp; ++i) {
    if (i < warp) before += sh->scan[i];
    total += sh->scan[i];
  }
  const int64_t excl = before + incl - mine;
  const int64_t share = total > 0 ? (total + gridDim.x - 1) / gridDim.x : 1;
  const int64_t at = share * blockIdx.x;
  if (at >= excl && at < excl + mine) {
    int64_t pos = excl;
    for (int b = b0; b < b1; ++b) {
      const PairTiles t = pair_tiles(P, attn_seq(P, b), row0);
      const int64_t n = (int64_t)(t.t1 - t.t0) * P.Hkv;
      if (at < pos + n) {
        sh->start_seq = b;
        sh->start_item = pos;
        break;
      }
      pos += n;
    }
  }
  __syncthreads();
  // rows without any key: out 0, lse -inf
  if (any_empty) {
    for (int b = blockIdx.x; b < P.batch; b += gridDim.x) {
      const AttnSeq s = attn_seq(P, b);
      const PairTiles t = pair_tiles(P, s, row0);
      const int64_t all = (int64_t)s.n * P.G - row0;
      if (t.t1 != t.t0 || all <= 0) continue;
      const int rows = all < kRows ? (int)all : kRows;
      for (int i = threadIdx.x; i < rows * P.Hkv; i += kThreads) {
        const int row = row0 + i % rows, head = i / rows;
        const int64_t to = (int64_t)(s.q0 + row / P.G) * P.Hq + head * P.G + row % P.G;
        for (int d = 0; d < P.D; d += 8)
          *reinterpret_cast<uint4*>(P.out + to * P.D + d) = make_uint4(0, 0, 0, 0);
        if (P.lse) P.lse[to] = -INFINITY;
      }
    }
  }
  if (at >= total) return;
  const int64_t count = total - at < share ? total - at : share;
  Walk w;
  w.start(P, row0, sh->start_seq, sh->start_item, at, count);
  if (warp == kConsumers)
    stream_producer<DP>(P, M, sh, w, row0);
  else
    stream_consumer<T, DP>(P, sh, w, row0, share);
}

template <typename T, int DP>
int run_stream(const AttnMaps& M, const AttnParams& P, dim3 grid, cudaStream_t stream) {
  constexpr size_t smem = sizeof(StreamSmem<DP>) + 1024;
  static_assert(smem <= 113 * 1024, "two blocks per SM");
  static std::atomic<uint64_t> done{0};
  cudaError_t err = allow_smem(k_attn_stream<T, DP>, smem, done);
  if (err != cudaSuccess) return cuda_status(err);
  return cuda_status(launch_pdl(k_attn_stream<T, DP>, grid, dim3(kThreads), smem, stream, M, P));
}

// Blocks per row tile: two per SM over all row tiles, at least one.
int stream_blocks(int64_t row_tiles) {
  int64_t w = (int64_t)kCtasPerSm * sm_count() / row_tiles;
  if (w < 1) w = 1;
  return (int)w;
}

}  // namespace

size_t attn_stream_partial_bytes(int64_t rows_max, int D) {
  const int64_t tiles = ceil_div(rows_max < 1 ? 1 : rows_max, kRows);
  const int dp = D <= 64 ? 64 : 128;
  const int64_t w = stream_blocks(tiles);
  if (w == 1) return 0;  // nothing is split
  return (size_t)(tiles * w) * 2 * (kRows * dp + 2 * kRows) * sizeof(float);
}

int launch_attn_stream(const ftb_attn_args& a, AttnParams P, cudaStream_t stream) {
  AttnMaps M;
  const uint32_t r = a.page < kTile ? a.page : kTile;
  const int dp = a.D <= 64 ? 64 : 128;
  const uint32_t halves = a.D == dp ? dp / 64 : 1;
  int st = attn_cache_map(&M.k, a.k_cache, a, a.k_strides, r, halves);
  if (!st) st = attn_cache_map(&M.v, a.v_cache, a, a.v_strides, r, halves);
  if (st) return st;
  M.q = M.k;  // unused
  const int64_t tiles = ceil_div((int64_t)a.max_q * P.G, kRows);
  const int64_t w = stream_blocks(tiles);
  if (tiles > 65535 || (w > 1 && tiles * w > kAttnCounters)) return FTB_ERR_SHAPE;
  const dim3 grid((unsigned)w, (unsigned)tiles);
  if (a.type == FTB_TYPE_BF16)
    return dp == 64 ? run_stream<__nv_bfloat16, 64>(M, P, grid, stream)
                    : run_stream<__nv_bfloat16, 128>(M, P, grid, stream);
  return dp == 64 ? run_stream<__half, 64>(M, P, grid, stream)
                  : run_stream<__half, 128>(M, P, grid, stream);
}

}  // namespace ftb
