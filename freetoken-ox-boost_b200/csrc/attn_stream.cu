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
// A cache of bytes (C8, attn.cuh has the arithmetic of its scales) is read by the same walk and ring: codes
// become f16 in registers, and a stage's scales come by plain loads beside its copies. Up to 8 rows have
// a form of their own (stream_consumer8), by one or two kv heads a block. On one B200, 32 heads of 128
// over 8: 61 tokens at up to 8192 keys (418 MB) 89 us, 4.7 TB/s, 0.73 of the measured copy rate; 3 at up
// to 131072 keys (719 MB) 131 us, 5.5 TB/s, 0.86; one at 901 keys 13.3 us. P is f16, whose numbers the codes
// are, and the rest of that rounding here too, whatever the tensors' type: with P alone 87, 131 and 13.2 us in
// bf16, where 7 to 10 outputs of 100 were rounded otherwise than the exact ones (now 1 to 2 of 1000).
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

constexpr int stream_stages(int DP, bool C8) { return DP == 128 && !C8 ? 3 : 6; }
// C8: the cache is one of bytes. Its rows take 128 bytes whatever D is.
template <int DP, bool C8>
struct StreamSmem {
  static constexpr int kStages = stream_stages(DP, C8);
  alignas(1024) uint8_t ring[kStages][2][kTile * (C8 ? 128 : DP * 2)];
  BlockScale scale[C8 ? kStages : 1][kConsumers];  // of each 16 keys of a tile
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

// The form for up to 8 rows over a cache of bytes. A stage is 64 rows of 128 bytes of K and of V: 64
// keys of a head, or (HP = 2, an even number of kv heads) 32 keys of two heads that lie side by side. Pairs
// because memory is read faster in 256 bytes than in 128: copies alone, without any products, took 83 us
// for 61 tokens at up to 8192 keys one head at a time and 74 us by pairs.
constexpr int kRows8 = 8;
template <int DP, int HP>
struct StreamSmem8 {
  static constexpr int kStages = 6;
  alignas(1024) uint8_t ring[kStages][2][64 * 128];  // [box][head][row][128]
  alignas(16) float merge[kConsumers][kRows8][DP / 2 + 4];  // half of the columns
  BlockScale scale[kStages][kConsumers];  // of each warp's keys
  float ml[kConsumers][kRows8][2];
  float fac[kConsumers][kRows8];
  float row_m[HP][kRows8], row_l[HP][kRows8];
  uint64_t full[kStages], empty[kStages];
  int64_t scan[kThreads / kWarp];
  int64_t start_item;
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
template <int R, int KT>  // rows of a row tile, keys of a stage
__device__ __forceinline__ PairTiles pair_tiles(const AttnParams& P, const AttnSeq& s, int row0) {
  PairTiles t{0, 0, 0, 0};
  const int64_t rows = (int64_t)s.n * P.G;
  if (row0 >= rows) return t;
  const int last = (int)(rows < row0 + R ? rows : row0 + R) - 1;
  const KeyRange k = attn_range(P, s, row0 / P.G, last / P.G);
  if (k.lo >= k.hi) return t;
  t.lo = k.lo, t.hi = k.hi, t.t0 = k.lo / KT, t.t1 = (k.hi + KT - 1) / KT;
  return t;
}

// The walk over a block's share of the line; producer and consumers take the same steps.
// (heads: the kv heads, or pairs of them, that the line has one after another)
template <int R, int KT>
struct Walk {
  int seq, head, tile;  // next tile of pair (seq, head)
  int heads;
  int64_t item;         // line position of the pair's first tile
  int64_t left;         // tiles of the share still to do
  AttnSeq s;
  PairTiles t;
  __device__ void start(const AttnParams& P, int row0, int seq0, int64_t seq_at, int64_t at,
                        int64_t count, int n_heads) {
    seq = seq0;
    heads = n_heads;
    s = attn_seq(P, seq);
    t = pair_tiles<R, KT>(P, s, row0);
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
    if (++head == heads) {
      head = 0;
      do {
        ++seq;  // left > 0: a later sequence has tiles
        s = attn_seq(P, seq);
        t = pair_tiles<R, KT>(P, s, row0);
      } while (t.t1 == t.t0);
    }
    tile = t.t0;
  }
};

template <class Smem>
struct StreamSync {
  Smem* sh;
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
__device__ void stream_producer(const AttnParams& P, const AttnMaps& M, StreamSmem<DP, false>* sh,
                                Walk<kRows, kTile> w, int row0) {
  constexpr int kStages = StreamSmem<DP, false>::kStages;
  const int lane = threadIdx.x & 31;
  const StreamSync<StreamSmem<DP, false>> sy{sh, P.status};
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

// A load that keeps its place among volatile statements: asked for before the waits that hide it. (Coherent:
// the kernel before this one, which writes the scales, may run beside this one's start.)
__device__ __forceinline__ int ldg_now(const int32_t* p) {
  int r;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ float ldg_now(const float* p) {
  float r;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(r) : "l"(p));
  return r;
}

// The same for a cache of bytes, whose scales come by plain loads: four groups of 16 keys per tile (a
// block of tokens is 16 keys or more). A tile takes half as long as one of 16 bits, no longer than a
// page id and the scales behind it take to come, so the lanes look after eight tiles at once, lane l after
// 16 keys of one head of tile l / 4, and ask for the scales of the next eight and the ids of those after them
// before they turn to these.
template <int HP, class Smem, int R, int KT>
__device__ void stream_producer8(const AttnParams& P, const AttnMaps& M, Smem* sh, Walk<R, KT> w,
                                 int row0) {
  constexpr int kStages = Smem::kStages;
  // a lane's group of keys, of kGroups per tile, and its head: four lanes per tile
  constexpr int kGroups = KT / 16, kLanes = kGroups * HP, kAhead = kWarp / kLanes;
  const int lane = threadIdx.x & 31;
  const StreamSync<Smem> sy{sh, P.status};
  const int page = 1 << P.page_log2;
  const int r = page < KT ? page : KT;  // keys per box, >= 16
  const int boxes = KT / r;             // <= kGroups
  const int my_key = (lane & (kGroups - 1)) * 16, my_box = my_key / r;
  const int my_head = (lane & (kLanes - 1)) / kGroups;
  int stage = 0;
  uint32_t parity = 1, issued = 0;
  bool ok = true;
  while (w.left > 0 && ok) {
    const int n = w.take();
    const int32_t* table = P.block_table + (int64_t)w.seq * P.table_stride;
    const float* ks_of = P.k_scale + (w.head * HP + my_head) * P.ks_st[2];
    const float* vs_of = P.v_scale + (w.head * HP + my_head) * P.vs_st[2];
    // boxes [b0, b1) of a tile have a key in [lo, hi)
    auto box0 = [&](int key0) { return w.t.lo > key0 ? (w.t.lo - key0) / r : 0; };
    auto box1 = [&](int key0) { return min(boxes, (w.t.hi - key0 + r - 1) / r); };
    // the first key of this lane's group of the tiles from j0 on; whether anybody reads it
    auto key_at = [&](int j0) { return (w.tile + j0 + lane / kLanes) * KT + my_key; };
    auto wanted = [&](int j0) {
      const int key0 = (w.tile + j0 + lane / kLanes) * KT;
      return j0 + lane / kLanes < n && my_box >= box0(key0) && my_box < box1(key0);
    };
    auto load_id = [&](int j0) {  // -1: not wanted
      return wanted(j0) ? ldg_now(table + (key_at(j0) >> P.page_log2)) : -1;
    };
    auto load_scales = [&](int j0, int id, float& ks, float& vs) {
      ks = vs = 1.f;
      if (id >= 0 && id < P.num_pages) {
        const int block = (key_at(j0) & (page - 1)) >> P.block_log2;
        ks = ldg_now(ks_of + id * P.ks_st[0] + block * P.ks_st[1]);
        vs = ldg_now(vs_of + id * P.vs_st[0] + block * P.vs_st[1]);
      }
    };
    int id = load_id(0), id_next = load_id(kAhead);
    float ks, vs;
    load_scales(0, id, ks, vs);
    for (int j0 = 0; j0 < n && ok; j0 += kAhead) {
      float ks_next, vs_next;
      load_scales(j0 + kAhead, id_next, ks_next, vs_next);
      const int id_after = load_id(j0 + 2 * kAhead);
      if (wanted(j0) && (id < 0 || id >= P.num_pages)) {
        atomicOr(P.status, kAttnBadPage);
        id = (int)P.num_pages;  // outside the tensor: reads zeros
      }
      const int count = min(kAhead, n - j0);
      for (int j = 0; j < count; ++j) {
        const int key0 = (w.tile + j0 + j) * KT;
        const int b0 = box0(key0), b1 = box1(key0);
        // (a box's groups are of one page)
        const int box_id = __shfl_sync(0xffffffffu, id, j * kLanes + ((lane * r >> 4) & (kGroups - 1)));
        ok = __all_sync(0xffffffffu, sy.wait(&sh->empty[stage], parity));
        if (!ok) break;
        ++issued;
        if (lane >= b0 && lane < b1) {
          const uint32_t at = lane * r * 128 * HP;
          const int row = (key0 + lane * r) & (page - 1);
          tma_5d(smem_u32(sh->ring[stage][0]) + at, &M.k, 0, row, w.head * HP, box_id, 0, &sh->full[stage]);
          tma_5d(smem_u32(sh->ring[stage][1]) + at, &M.v, 0, row, w.head * HP, box_id, 0, &sh->full[stage]);
        }
        if (lane / kLanes == j) sh->scale[stage][lane & (kLanes - 1)] = block_scale(ks, vs);
        __syncwarp();
        // (the phase stays open for this arrival, whatever has landed by now)
        if (lane == 0)
          mbar_arrive_expect_tx(&sh->full[stage], 2u * HP * (uint32_t)(b1 - b0) * (uint32_t)r * 128u);
        __syncwarp();
        if (++stage == kStages) stage = 0, parity ^= 1u;
      }
      id = id_next, id_next = id_after, ks = ks_next, vs = vs_next;
    }
    w.next(P, row0, n);
  }
  for (uint32_t u = issued > kStages ? issued - kStages : 0; u < issued; ++u)  // as above
    for (uint32_t i = 0; i < kSpinLimit; ++i)
      if (mbar_try_wait(&sh->full[u % kStages], (u / kStages) & 1u)) break;
}

// The key of column n of an 8-key group, by which rows of 128 swizzled bytes are read without bank
// conflicts: K's 16-byte chunks 4 to a row (columns 2i and 2i + 1 in opposite halves of the banks) and
// V's chunks 2 to a row (columns 0, 2, 4, 6, and 1, 3, 5, 7, in different quarters).
__device__ __forceinline__ int key_of(int n) { return n & 1 ? (n - 1) ^ 5 : n; }

// One row's part of a query head as A fragments of f16: this lane's elements are 16 (lane % 4) .. + 15
// of each 64, as K's bytes lie in a lane. bf16 rows whose largest element f16 would not hold with all
// its bits are taken times a power of two (returned: its inverse).
template <typename T, int DP>
__device__ __forceinline__ float load_q8(const uint16_t* qp, bool in, int D,
                                         uint32_t (&lo)[DP / 16], uint32_t (&hi)[DP / 16]) {
  const int tig = threadIdx.x & 3;
  uint4 w[DP / 64][2];
#pragma unroll
  for (int h = 0; h < DP / 64; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = h * 64 + tig * 16 + i * 8;
      w[h][i] = in && d < D ? *reinterpret_cast<const uint4*>(qp + d) : make_uint4(0, 0, 0, 0);
    }
  float back = 1.f, by = 1.f;
  if constexpr (!std::is_same<T, __half>::value) {
    uint32_t top = 0;  // largest |x| as bf16 bits, in the upper half
#pragma unroll
    for (int h = 0; h < DP / 64; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t v[4] = {w[h][i].x, w[h][i].y, w[h][i].z, w[h][i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          top = max(top, max(v[k] << 16 & 0x7fff0000u, v[k] & 0x7fff0000u));
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = (int)(top >> 23) - 127;
    if (top && ex < 128 && (ex < -4 || ex > 14)) {  // (infinite and NaN rows stay so)
      const int x = ex > 14 ? ex - 14 : max(ex, -126);  // (both factors are normal numbers)
      by = __uint_as_float((uint32_t)(127 - x) << 23);
      back = __uint_as_float((uint32_t)(127 + x) << 23);
    }
  }
#pragma unroll
  for (int h = 0; h < DP / 64; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t v[4] = {w[h][i].x, w[h][i].y, w[h][i].z, w[h][i].w};
      if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack2<T>(v[k]);
          v[k] = pack2<__half>(f.x * by, f.y * by);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        const int c = h * 4 + i * 2 + (k >> 1);
        lo[c] = v[k], hi[c] = v[k + 1];
      }
    }
  return back;
}

// An 8 x 8 matrix of 16-bit elements, a row's pair per lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Up to 8 rows over a cache of bytes. The rows are the N of the products, so that none of their 16 M is
// wasted on rows that are not there:
//   S^T = K Q^T    M = 16 keys of the warp, K = 16 elements
//   O^T = V^T P^T  M = 16 columns of V, K = 16 keys; P goes from the accumulators of S^T to the operand by
//                  a transposition of 8 x 8 (movmatrix)
// Half the products, exponentials and registers of the form above, whose chain of instructions bound it (61
// tokens at up to 8192 keys 130 us). Each warp has 16 keys of one head of a stage.
// A row's reference moves to a tile's maximum where that exceeds it by more than 2^kLazy (P reaches
// 2^kLazy, f16 holds it), so the warp's maxima are rarely brought together: one vote per tile.
template <typename T, int DP, int HP>
__device__ void stream_consumer8(const AttnParams& P, StreamSmem8<DP, HP>* sh, Walk<kRows8, 64 / HP> w,
                                 int row0, int64_t share) {
  using Smem = StreamSmem8<DP, HP>;
  constexpr int kWarps = kConsumers / HP, KT = 64 / HP;  // warps of a head, keys of a stage
  constexpr int kStages = Smem::kStages, VB = DP / 8;
  constexpr float kLazy = 10.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t2 = (lane & 3) * 2;  // key (or columns) of the lane; its rows t2, t2 + 1
  const StreamSync<Smem> sy{sh, P.status};
  const int wh = warp / kWarps, wk = warp % kWarps * 16;  // the warp's head and first key of a stage
  const int page = 1 << P.page_log2, r = page < KT ? page : KT;  // keys per box
  const int base = (wk / r * HP + wh) * r * 128 + wk % r * 128;  // its rows
  // K: keys kr, kr + 8 of the warp's, chunk lane % 4 of each 64 elements; V: keys kv0, kv1, + 8, VB bytes
  const int kr = key_of(g), kv0 = key_of(t2), kv1 = key_of(t2 + 1);
  auto v_at = [&](int key) {
    const int byte = g * VB;
    return key * 128 + (((byte >> 4) ^ (key & 7)) << 4) + (byte & 15);
  };
  int stage = 0;
  uint32_t parity = 0;  // + kGaveUp once a wait did
  constexpr uint32_t kGaveUp = 2;
  while (w.left > 0) {
    const int n = w.take();
    const AttnSeq s = w.s;
    const int rows_all = s.n * P.G - row0;
    const int rows = rows_all < kRows8 ? rows_all : kRows8;
    int kmin[2], kmax[2];  // keys of rows t2, t2 + 1
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      kmin[e] = kmax[e] = 0;
      if (t2 + e < rows) {
        const int i = (row0 + t2 + e) / P.G;
        const KeyRange k = attn_range(P, s, i, i);
        kmin[e] = k.lo, kmax[e] = k.hi;
      }
    }
    uint32_t q_lo[DP / 16], q_hi[DP / 16];  // row g
    float factor[2];                        // of the codes' scores, rows t2, t2 + 1
    {
      const int row = row0 + g;
      const uint16_t* qp =
          P.q + (int64_t)(s.q0 + row / P.G) * P.q_st + (int64_t)((w.head * HP + wh) * P.G + row % P.G) * P.q_sh;
      const float back = load_q8<T, DP>(qp, g < rows, P.D, q_lo, q_hi) * P.scale_log2;
      factor[0] = __shfl_sync(0xffffffffu, back, t2 * 4);
      factor[1] = __shfl_sync(0xffffffffu, back, t2 * 4 + 4);
    }
    float ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[VB / 2][4];  // columns VB g + 2 j, + 1 of rows t2, t2 + 1
#pragma unroll
    for (int j = 0; j < VB / 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    for (int j = 0; j < n && parity < kGaveUp; ++j) {
      const int key0 = (w.tile + j) * KT + wk;
      if (!__all_sync(0xffffffffu, sy.wait(&sh->full[stage], parity))) {
        parity = kGaveUp;
        break;
      }
      const uint8_t *kb = sh->ring[stage][0] + base, *vb = sh->ring[stage][1] + base;
      const BlockScale bs = sh->scale[stage][warp];
      float sc[4] = {}, sd[4] = {};
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        uint4 b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          b[h] = *reinterpret_cast<const uint4*>(kb + (kr + 8 * h) * 128 +
                                                 (((4 * c + (lane & 3)) ^ (kr & 7)) << 4));
        const uint32_t v[2][4] = {{b[0].x, b[0].y, b[0].z, b[0].w}, {b[1].x, b[1].y, b[1].z, b[1].w}};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a[4] = {e4m3x2_to_f16x2((uint16_t)(v[0][k] & 0xffffu)),
                                 e4m3x2_to_f16x2((uint16_t)(v[1][k] & 0xffffu)),
                                 e4m3x2_to_f16x2((uint16_t)(v[0][k] >> 16)),
                                 e4m3x2_to_f16x2((uint16_t)(v[1][k] >> 16))};
          mma16816<__half>(k & 1 ? sd : sc, a, q_lo[4 * c + k], q_hi[4 * c + k]);
        }
      }
      // V's bytes, asked for before the exponentials; rows outside [lo, hi) may hold NaN: made zero
      const bool inside = key0 >= w.t.lo && key0 + 16 <= w.t.hi;
      uint32_t v[2][2][VB / 4];  // [key group][key's parity][bytes]
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = (e ? kv1 : kv0) + 8 * h;
          if constexpr (VB == 16) {
            const uint4 b = *reinterpret_cast<const uint4*>(vb + v_at(row));
            v[h][e][0] = b.x, v[h][e][1] = b.y, v[h][e][2] = b.z, v[h][e][3] = b.w;
          } else {
            const uint2 b = *reinterpret_cast<const uint2*>(vb + v_at(row));
            v[h][e][0] = b.x, v[h][e][1] = b.y;
          }
          const int key = key0 + row;
          if (!inside && (key < w.t.lo || key >= w.t.hi)) {
#pragma unroll
            for (int k = 0; k < VB / 4; ++k) v[h][e][k] = 0u;
          }
        }
      const bool clean = inside && (!P.causal || s.n == 1) && (P.window <= 0 || s.n == 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + (i >> 1) * 8 + kr;
        const bool seen = clean || (key >= kmin[i & 1] && key < kmax[i & 1]);
        sc[i] = seen ? fmaf(sc[i] + sd[i], bs.k * factor[i & 1], bs.v_log2) : -INFINITY;
      }
      if (__any_sync(0xffffffffu, fmaxf(sc[0], sc[2]) > ref[0] + kLazy || fmaxf(sc[1], sc[3]) > ref[1] + kLazy)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(sc[e], sc[2 + e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          if (mx > ref[e] + kLazy) {  // (the same for all lanes of the row)
            const float f = ex2(ref[e] - mx);
            ref[e] = mx;
            l[e] *= f;
#pragma unroll
            for (int jj = 0; jj < VB / 2; ++jj) o[jj][e] *= f, o[jj][2 + e] *= f;
          }
        }
      }
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = ex2(sc[i] - (ref[i & 1] == -INFINITY ? 0.f : ref[i & 1]));
#pragma unroll
      for (int e = 0; e < 2; ++e) l[e] = fmaf(p[e] + p[2 + e], bs.v_inv, l[e]);
      uint32_t pb[2], rb[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pb[h] = pack2<__half>(p[2 * h], p[2 * h + 1]);
        const float2 a = unpack2<__half>(pb[h]);
        rb[h] = transpose8(pack2<__half>(p[2 * h] - a.x, p[2 * h + 1] - a.y));
        pb[h] = transpose8(pb[h]);
      }
#pragma unroll
      for (int k = 0; k < VB / 4; ++k) {
        // bytes of two keys side by side, two columns to a word
        uint32_t x[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x[h][0] = __byte_perm(v[h][0][k], v[h][1][k], 0x5140);
          x[h][1] = __byte_perm(v[h][0][k], v[h][1][k], 0x7362);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t a[4] = {e4m3x2_to_f16x2((uint16_t)(x[0][c] & 0xffffu)),
                                 e4m3x2_to_f16x2((uint16_t)(x[0][c] >> 16)),
                                 e4m3x2_to_f16x2((uint16_t)(x[1][c] & 0xffffu)),
                                 e4m3x2_to_f16x2((uint16_t)(x[1][c] >> 16))};
          mma16816<__half>(o[2 * k + c], a, pb[0], pb[1]);
          mma16816<__half>(o[2 * k + c], a, rb[0], rb[1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->empty[stage]);
      if (++stage == kStages) stage = 0, parity ^= 1u;
    }
    if (parity >= kGaveUp) l[0] = l[1] = NAN;
    // join the four warps' parts of the rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
      if (g == 0) {
        sh->ml[warp][t2 + e][0] = ref[e];
        sh->ml[warp][t2 + e][1] = l[e];
      }
    }
    named_bar(1, kConsumers * kWarp);
    if (threadIdx.x < HP * kRows8) {
      const int row = threadIdx.x % kRows8, hh = threadIdx.x / kRows8, w0 = hh * kWarps;
      float mm = sh->ml[w0][row][0];
      for (int i = 1; i < kWarps; ++i) mm = fmaxf(mm, sh->ml[w0 + i][row][0]);
      const float top = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      for (int i = 0; i < kWarps; ++i) {
        const float f = ex2(sh->ml[w0 + i][row][0] - top);
        sh->fac[w0 + i][row] = f;
        ll += f * sh->ml[w0 + i][row][1];
      }
      sh->row_m[hh][row] = mm;
      sh->row_l[hh][row] = ll;
    }
    named_bar(1, kConsumers * kWarp);
    const bool begins = w.tile == w.t.t0, ends = w.tile + n == w.t.t1;
    const bool whole = begins && ends;
    const int64_t blk = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    constexpr int kPart = kRows8 * DP + 2 * kRows8, kSlot = HP * kPart;  // of a head; of all
    auto out_row = [&](int row, int hh) {  // of the outputs
      return (int64_t)(s.q0 + row / P.G) * P.Hq + (w.head * HP + hh) * P.G + row % P.G;
    };
    float* slot = P.partial + (2 * blk + (begins ? 1 : 0)) * kSlot;  // (as above)
    const float f0 = sh->fac[warp][t2], f1 = sh->fac[warp][t2 + 1];
    constexpr int kHalf = DP / 2, kPer = kHalf / 4;  // columns of a pass, threads of a row
    const int orow = threadIdx.x / kPer, oc = threadIdx.x % kPer * 4;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (g >> 2 == c) {
#pragma unroll
        for (int i = 0; i < VB / 4; ++i) {
          const float(&a)[4] = o[2 * i], (&b)[4] = o[2 * i + 1];
          const int at = (g & 3) * VB + 4 * i;
          *reinterpret_cast<float4*>(&sh->merge[warp][t2][at]) =
              make_float4(a[0] * f0, a[2] * f0, b[0] * f0, b[2] * f0);
          *reinterpret_cast<float4*>(&sh->merge[warp][t2 + 1][at]) =
              make_float4(a[1] * f1, a[3] * f1, b[1] * f1, b[3] * f1);
        }
      }
      named_bar(1, kConsumers * kWarp);
      const int d = c * kHalf + oc;
#pragma unroll
      for (int hh = 0; hh < HP; ++hh) {
        if (orow >= rows) continue;
        float4 a = *reinterpret_cast<float4*>(&sh->merge[hh * kWarps][orow][oc]);
#pragma unroll
        for (int i = 1; i < kWarps; ++i) {
          const float4 b = *reinterpret_cast<float4*>(&sh->merge[hh * kWarps + i][orow][oc]);
          a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
        }
        if (!whole) {
          *reinterpret_cast<float4*>(slot + hh * kPart + orow * DP + d) = a;
        } else if (d < P.D) {
          const float ll = sh->row_l[hh][orow], inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
          *reinterpret_cast<uint2*>(P.out + out_row(row0 + orow, hh) * P.D + d) =
              make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
        }
      }
      named_bar(1, kConsumers * kWarp);
    }
    if (whole) {
      const int row = threadIdx.x % kRows8, hh = threadIdx.x / kRows8;
      if (P.lse && hh < HP && row < rows) {
        const float ll = sh->row_l[hh][row];
        P.lse[out_row(row0 + row, hh)] =
            ll == 0.f ? -INFINITY : (sh->row_m[hh][row] + log2f(ll)) * 0.69314718055994531f;
      }
    } else {
      const int row = threadIdx.x % kRows8, hh = threadIdx.x / kRows8;
      if (hh < HP && row < rows) {
        slot[hh * kPart + kRows8 * DP + row] = sh->row_m[hh][row];
        slot[hh * kPart + kRows8 * DP + kRows8 + row] = sh->row_l[hh][row];
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
        const float* p0 = P.partial + (2 * blk0 + 1) * kSlot;
        const float* p1 = P.partial + 2 * (blk0 + 1) * kSlot;
        // All heads' rows at once, 16 / HP threads a row, kCols x 4 columns each; the threads of rows that
        // are not there take their share of the parts: part i goes to way i % ways of its row.
        constexpr int kRowThreads = 16 / HP, kStep = kRowThreads * 4, kCols = DP / kStep;
        const int jc = threadIdx.x % kRowThreads * 4, any = threadIdx.x / kRowThreads;
        const int hh = any / kRows8, trow = any % kRows8;
        const int lg = rows > 1 ? 32 - __clz(rows - 1) : 0, ways = kRows8 >> lg;
        const int jrow = trow & ((1 << lg) - 1), way = trow >> lg;
        const bool mine = jrow < rows;
        float mm = -INFINITY, ll = 0.f;
        float4 acc[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float f, const float4& b, int c) {
          acc[c].x += f * b.x, acc[c].y += f * b.y, acc[c].z += f * b.z, acc[c].w += f * b.w;
        };
        if (mine) {
          auto part = [&](int i) { return (i == 0 ? p0 : p1 + (int64_t)(i - 1) * 2 * kSlot) + hh * kPart; };
          // (so many parts' loads in flight: one at a time, a single sequence's 37 or 74 parts took as long
          // as its keys)
          constexpr int kAtOnce = 4;
          for (int i = way; i < parts; i += ways * kAtOnce) {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
              if (i + u * ways < parts) mm = fmaxf(mm, __ldcg(part(i + u * ways) + kRows8 * DP + jrow));
          }
          const float top = mm == -INFINITY ? 0.f : mm;
          for (int i = way; i < parts; i += ways * kAtOnce) {
            float m[kAtOnce], l1[kAtOnce];
            float4 v[kAtOnce][kCols];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
              const float* q = part(min(i + u * ways, parts - 1));
              m[u] = __ldcg(q + kRows8 * DP + jrow);
              l1[u] = __ldcg(q + kRows8 * DP + kRows8 + jrow);
#pragma unroll
              for (int c = 0; c < kCols; ++c)
                v[u][c] = __ldcg(reinterpret_cast<const float4*>(q + jrow * DP + c * kStep + jc));
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
              if (i + u * ways >= parts) continue;
              const float f = ex2(m[u] - top);
              ll += f * l1[u];
#pragma unroll
              for (int c = 0; c < kCols; ++c) add(f, v[u][c], c);
            }
          }
        }
        if (ways > 1) {
          static_assert(sizeof(sh->merge) >= HP * kRows8 * DP * sizeof(float) &&
                            HP * kRows8 <= kConsumers * kRows8, "the ways' sums fit");
          float* all = &sh->merge[0][0][0];
          float(*sums)[2] = &sh->ml[0][0];  // [head and row][2]
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            *reinterpret_cast<float4*>(all + any * DP + c * kStep + jc) = acc[c];
          if (jc == 0) sums[any][0] = mm, sums[any][1] = ll;
          named_bar(1, kConsumers * kWarp);
          if (mine && way == 0) {
            for (int i = 1; i < ways; ++i) mm = fmaxf(mm, sums[any + (i << lg)][0]);
            const float top = mm == -INFINITY ? 0.f : mm;
            ll = 0.f;
#pragma unroll
            for (int c = 0; c < kCols; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < ways; ++i) {
              const int at = any + (i << lg);
              const float f = ex2(sums[at][0] - top);
              ll += f * sums[at][1];
#pragma unroll
              for (int c = 0; c < kCols; ++c)
                add(f, *reinterpret_cast<const float4*>(all + at * DP + c * kStep + jc), c);
            }
          }
          named_bar(1, kConsumers * kWarp);  // (the next pair writes the merge buffer)
        }
        if (mine && way == 0) {
          const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
          const int64_t at = out_row(row0 + jrow, hh);
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            if (c * kStep + jc < P.D)
              *reinterpret_cast<uint2*>(P.out + at * P.D + c * kStep + jc) = make_uint2(
                  pack2<T>(acc[c].x * inv, acc[c].y * inv), pack2<T>(acc[c].z * inv, acc[c].w * inv));
          if (P.lse && jc == 0)
            P.lse[at] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
        }
      }
    }
    w.next(P, row0, n);
  }
}

template <typename T, int DP, bool C8>
__device__ void stream_consumer(const AttnParams& P, StreamSmem<DP, C8>* sh, Walk<kRows, kTile> w, int row0,
                                int64_t share) {
  constexpr int kStages = StreamSmem<DP, C8>::kStages;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  const StreamSync<StreamSmem<DP, C8>> sy{sh, P.status};
  // P's type: the tensors', or f16 beside V's codes, which are f16 numbers
  using TP = typename std::conditional<C8, __half, T>::type;
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
    float q_back[2] = {1.f, 1.f};  // C8: what q was taken times, the inverse
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
      if constexpr (C8) {
        uint32_t lo[DP / 16], hi[DP / 16];
        q_back[e] = load_q8<T, DP>(qp, in, P.D, lo, hi);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) qa[c][e] = lo[c], qa[c][2 + e] = hi[c];
      } else {
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          const int d = c * 16 + t2;
          qa[c][e] = in && d < P.D ? *reinterpret_cast<const uint32_t*>(qp + d) : 0u;
          qa[c][2 + e] = in && d + 8 < P.D ? *reinterpret_cast<const uint32_t*>(qp + d + 8) : 0u;
        }
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
      BlockScale bs{1.f, 0.f, 1.f};
      if constexpr (C8) {
        bs = sh->scale[stage][warp];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int kr = warp * 16 + h * 8 + key_of(g);
#pragma unroll
          for (int c = 0; c < DP / 64; ++c) {
            const uint4 b = *reinterpret_cast<const uint4*>(
                sh->ring[stage][0] + kr * 128 + (((4 * c + (lane & 3)) ^ (kr & 7)) << 4));
            const uint32_t v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma16816<__half>(sc[h], qa[4 * c + k], e4m3x2_to_f16x2((uint16_t)(v[k] & 0xffffu)),
                               e4m3x2_to_f16x2((uint16_t)(v[k] >> 16)));
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          uint32_t b[4];
          const int chunk = (2 * c + kc) & 7;
          ldsm4(kb + k_off + (c >> 2) * half_bytes + ((chunk ^ k_sw) << 4), b);
          mma16816<T>(sc[0], qa[c], b[0], b[1]);
          mma16816<T>(sc[1], qa[c], b[2], b[3]);
        }
      }
      // a warp's 16 keys, all seen by all of the tile's rows, need no mask
      const bool clean = key0 >= w.t.lo && key0 + 16 <= w.t.hi && (!P.causal || s.n == 1) &&
                         (P.window <= 0 || s.n == 1);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + h * 8 + (C8 ? key_of(t2 + (i & 1)) : t2 + (i & 1));
          const bool seen = clean || (key >= kmin[i >> 1] && key < kmax[i >> 1]);
          const float score =
              C8 ? fmaf(sc[h][i], bs.k * (P.scale_log2 * q_back[i >> 1]), bs.v_log2)
                 : sc[h][i] * P.scale_log2;
          sc[h][i] = seen ? score : -INFINITY;
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
        l[e] = C8 ? fmaf((p0 + p1) + (p2 + p3), bs.v_inv, l[e] * f)
                  : l[e] * f + ((p0 + p1) + (p2 + p3));
        pa[e] = pack2<TP>(p0, p1);
        pa[2 + e] = pack2<TP>(p2, p3);
        const float2 a = unpack2<TP>(pa[e]), b = unpack2<TP>(pa[2 + e]);
        pr[e] = pack2<TP>(p0 - a.x, p1 - a.y);
        pr[2 + e] = pack2<TP>(p2 - b.x, p3 - b.y);
        if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
          for (int jj = 0; jj < DP / 8; ++jj) o[jj][2 * e] *= f, o[jj][2 * e + 1] *= f;
        }
      }
      // V rows outside [lo, hi) have weight 0 but may hold NaN or infinity: made zero
      const bool inside = key0 >= w.t.lo && key0 + 16 <= w.t.hi;
      if constexpr (C8) {
        constexpr int VB = DP / 8;  // columns of O: VB (lane / 4) .. of V, VB n .. of the result
        uint32_t v[2][2][VB / 4];   // [key group][column's parity][bytes]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int kr = warp * 16 + h * 8 + key_of(t2 + e);
            const int byte = g * VB;
            const uint8_t* at = sh->ring[stage][1] + kr * 128 + (((byte >> 4) ^ (kr & 7)) << 4) + (byte & 15);
            if constexpr (VB == 16) {
              const uint4 b = *reinterpret_cast<const uint4*>(at);
              v[h][e][0] = b.x, v[h][e][1] = b.y, v[h][e][2] = b.z, v[h][e][3] = b.w;
            } else {
              const uint2 b = *reinterpret_cast<const uint2*>(at);
              v[h][e][0] = b.x, v[h][e][1] = b.y;
            }
            const int key = key0 - warp * 16 + kr;
            if (!inside && (key < w.t.lo || key >= w.t.hi)) {
#pragma unroll
              for (int k = 0; k < VB / 4; ++k) v[h][e][k] = 0u;
            }
          }
#pragma unroll
        for (int k = 0; k < VB / 4; ++k) {
          // bytes of two keys side by side, two columns to a word
          uint32_t x[2][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            x[h][0] = __byte_perm(v[h][0][k], v[h][1][k], 0x5140);
            x[h][1] = __byte_perm(v[h][0][k], v[h][1][k], 0x7362);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t b[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
              b[h] = e4m3x2_to_f16x2((uint16_t)(c & 1 ? x[h][c >> 1] >> 16 : x[h][c >> 1] & 0xffffu));
            mma16816<TP>(o[4 * k + c], pa, b[0], b[1]);
            mma16816<TP>(o[4 * k + c], pr, b[0], b[1]);
          }
        }
      } else {
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
    // column of chunk c of 32 that this thread joins: C8's lanes hold DP / 8 columns in a row
    auto col_of = [&](int c) { return C8 ? (int)(threadIdx.x & 7) * (DP / 8) + 4 * c : c * kMergeCols + oc; };
#pragma unroll
    for (int c = 0; c < DP / kMergeCols; ++c) {
      if constexpr (C8) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float(&v0)[4] = o[4 * c], (&v1)[4] = o[4 * c + 1], (&v2)[4] = o[4 * c + 2],
                     (&v3)[4] = o[4 * c + 3];
          *reinterpret_cast<float4*>(&sh->merge[warp][g][t2 * 4 + e * 4]) =
              make_float4(v0[e] * f0, v1[e] * f0, v2[e] * f0, v3[e] * f0);
          *reinterpret_cast<float4*>(&sh->merge[warp][g + 8][t2 * 4 + e * 4]) =
              make_float4(v0[2 + e] * f1, v1[2 + e] * f1, v2[2 + e] * f1, v3[2 + e] * f1);
        }
      } else {
#pragma unroll
        for (int jj = 0; jj < kMergeCols / 8; ++jj) {
          const float(&v)[4] = o[c * (kMergeCols / 8) + jj];
          *reinterpret_cast<float2*>(&sh->merge[warp][g][jj * 8 + t2]) = make_float2(v[0] * f0, v[1] * f0);
          *reinterpret_cast<float2*>(&sh->merge[warp][g + 8][jj * 8 + t2]) = make_float2(v[2] * f1, v[3] * f1);
        }
      }
      named_bar(1, kConsumers * kWarp);
      float4 a = *reinterpret_cast<float4*>(&sh->merge[0][orow][oc]);
#pragma unroll
      for (int i = 1; i < kConsumers; ++i) {
        const float4 b = *reinterpret_cast<float4*>(&sh->merge[i][orow][oc]);
        a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
      }
      const int d = col_of(c);
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
              add(f, __ldcg(reinterpret_cast<const float4*>(p + jrow * DP + col_of(c))), c);
          }
        }
        if (ways > 1) {
          static_assert(kConsumers * kMergePitch >= DP, "the ways' sums fit the merge buffer");
          float* all = &sh->merge[0][0][0];
#pragma unroll
          for (int c = 0; c < DP / kMergeCols; ++c)
            *reinterpret_cast<float4*>(all + orow * DP + col_of(c)) = acc[c];
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
                add(f, *reinterpret_cast<const float4*>(all + at * DP + col_of(c)), c);
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
            const int d = col_of(c);
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

// HP: the form for few rows over a cache of bytes, by so many heads; 0: the other.
template <typename T, int DP, bool C8, int HP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    k_attn_stream(const __grid_constant__ AttnMaps M, const __grid_constant__ AttnParams P) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int R = HP ? kRows8 : kRows, KT = HP ? 64 / (HP ? HP : 1) : kTile;
  using Smem = typename std::conditional<HP != 0, StreamSmem8<DP, HP ? HP : 1>, StreamSmem<DP, C8>>::type;
  const int heads = HP == 2 ? P.Hkv / 2 : P.Hkv;
  Smem* sh = reinterpret_cast<Smem*>(
      smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.y * R;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < Smem::kStages; ++i) {
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
    const PairTiles t = pair_tiles<R, KT>(P, s, row0);
    mine += (int64_t)(t.t1 - t.t0) * heads;
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
  int64_t share = total > 0 ? (total + gridDim.x - 1) / gridDim.x : 1;
  if (HP == 2 && share < 2) share = 2;  // (64 keys, as in the other forms)
  const int64_t at = share * blockIdx.x;
  if (at >= excl && at < excl + mine) {
    int64_t pos = excl;
    for (int b = b0; b < b1; ++b) {
      const PairTiles t = pair_tiles<R, KT>(P, attn_seq(P, b), row0);
      const int64_t n = (int64_t)(t.t1 - t.t0) * heads;
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
      const PairTiles t = pair_tiles<R, KT>(P, s, row0);
      const int64_t all = (int64_t)s.n * P.G - row0;
      if (t.t1 != t.t0 || all <= 0) continue;
      const int rows = all < R ? (int)all : R;
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
  Walk<R, KT> w;
  w.start(P, row0, sh->start_seq, sh->start_item, at, count, heads);
  if (warp == kConsumers) {
    if constexpr (C8)
      stream_producer8<HP ? HP : 1>(P, M, sh, w, row0);
    else
      stream_producer<DP>(P, M, sh, w, row0);
  } else if constexpr (HP != 0) {
    stream_consumer8<T, DP, HP>(P, sh, w, row0, share);
  } else {
    stream_consumer<T, DP, C8>(P, sh, w, row0, share);
  }
}

template <typename T, int DP, bool C8, int HP>
int run_stream(const AttnMaps& M, const AttnParams& P, dim3 grid, cudaStream_t stream) {
  constexpr size_t smem =
      (HP ? sizeof(StreamSmem8<DP, HP ? HP : 1>) : sizeof(StreamSmem<DP, C8>)) + 1024;
  static_assert(smem <= 113 * 1024, "two blocks per SM");
  static std::atomic<uint64_t> done{0};
  cudaError_t err = allow_smem(k_attn_stream<T, DP, C8, HP>, smem, done);
  if (err != cudaSuccess) return cuda_status(err);
  return cuda_status(launch_pdl(k_attn_stream<T, DP, C8, HP>, grid, dim3(kThreads), smem, stream, M, P));
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

template <bool C8, int HP>
int pick_stream(const ftb_attn_args& a, const AttnMaps& M, const AttnParams& P, int dp, dim3 grid,
                cudaStream_t stream) {
  if (a.type == FTB_TYPE_BF16)
    return dp == 64 ? run_stream<__nv_bfloat16, 64, C8, HP>(M, P, grid, stream)
                    : run_stream<__nv_bfloat16, 128, C8, HP>(M, P, grid, stream);
  return dp == 64 ? run_stream<__half, 64, C8, HP>(M, P, grid, stream)
                  : run_stream<__half, 128, C8, HP>(M, P, grid, stream);
}

// Whether the form for few rows takes kv heads by pairs. That reads memory faster, but cuts half as many
// pairs of sequence and heads into twice as many parts each, whose join is the end of a block's chain. By
// what the host knows of the keys: where a block has at least 1.5 times as many tiles as a pair has parts.
// On one B200, us (one head / pairs), 32 heads of 128 over 8: 1 token at 8192 keys 18.8 / 29.8, at 131072
// 75.7 / 86.8; 2 at 32768 47.8 / 54.4, at 131072 123 / 114; 16 at 500 12.6 / 13.3; 64 at 300 23.1 / 21.2;
// 61 at up to 8192 97 / 89; 3 at up to 131072 150 / 130.
bool pair_heads(const ftb_attn_args& a) {
  if (a.Hkv % 2) return false;
  const double blocks = stream_blocks(1), pairs = 0.5 * a.batch * a.Hkv;
  const double tiles = (double)a.batch * a.Hkv * (double)ceil_div((int64_t)a.table_width * a.page, kTile);
  return tiles * pairs >= 1.5 * blocks * blocks;
}

int launch_attn_stream(const ftb_attn_args& a, AttnParams P, bool fp8, cudaStream_t stream) {
  AttnMaps M;
  const int dp = a.D <= 64 ? 64 : 128;
  const uint32_t halves = a.D == dp ? dp / 64 : 1;
  const int hp = !fp8 || (int64_t)a.max_q * P.G > kRows8 ? 0 : pair_heads(a) ? 2 : 1;
  const uint32_t keys = hp == 2 ? kTile / 2 : kTile, r = a.page < (int)keys ? a.page : keys;
  int st = fp8 ? attn_cache_map8(&M.k, a.k_cache, a, a.k_strides, r, hp == 2 ? 2 : 1)
               : attn_cache_map(&M.k, a.k_cache, a, a.k_strides, r, halves);
  if (!st)
    st = fp8 ? attn_cache_map8(&M.v, a.v_cache, a, a.v_strides, r, hp == 2 ? 2 : 1)
             : attn_cache_map(&M.v, a.v_cache, a, a.v_strides, r, halves);
  if (st) return st;
  M.q = M.k;  // unused
  if (hp) {
    // (parts of 2 x 8 rows are no larger than those of 16 that the workspace is for)
    const dim3 grid((unsigned)stream_blocks(1));
    if ((int)grid.x > kAttnCounters) return FTB_ERR_SHAPE;
    return hp == 2 ? pick_stream<true, 2>(a, M, P, dp, grid, stream)
                   : pick_stream<true, 1>(a, M, P, dp, grid, stream);
  }
  const int64_t tiles = ceil_div((int64_t)a.max_q * P.G, kRows);
  const int64_t w = stream_blocks(tiles);
  if (tiles > 65535 || (w > 1 && tiles * w > kAttnCounters)) return FTB_ERR_SHAPE;
  const dim3 grid((unsigned)w, (unsigned)tiles);
  return fp8 ? pick_stream<true, 0>(a, M, P, dp, grid, stream)
             : pick_stream<false, 0>(a, M, P, dp, grid, stream);
}

}  // namespace ftb
