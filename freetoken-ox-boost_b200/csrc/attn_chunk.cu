// attn_chunk.cu - paged attention for many query rows per kv head (prompts, chunks of a prefill)
// on the 5th-generation tensor cores.
//
// The rows of a sequence and kv head are its new tokens x the G query heads that share the kv
// head. An item is two tiles A and B of up to 128 rows (whole tokens, floor(128 / G) each), one
// kv head and a range of 128-key tiles, computed by one persistent block:
//   S = Q K^T   tcgen05.mma M = 128, N = 128 keys, Q and K from shared memory, S in tensor memory
//   P = 2^(s - ref), l += sum P     one thread per row, all 128 scores in registers
//   O += P V    tcgen05.mma M = 128, N = D, P from tensor memory (it takes S's place), V from
//               shared memory (its rows are keys: the MN-major operand layout)
// ref is the row's reference. It starts at 0 and moves to a tile's maximum only where that exceeds
// it by more than 2^8, or falls short of it with nothing summed yet (by more than 2^8 in bf16, at
// all in f16), so O, in tensor memory, is rescaled rarely. The sums are fp32. P is rounded to the
// tensors' type: in bf16, with fp32's exponents, to 2^-8 of itself wherever ref lies; in f16, where
// ref is never above the row's maximum, to 2^-11 of itself down to weights of 2^-14 of the largest,
// and to at most 2^-25 of the largest below that. The rest of the rounding is dropped by choice: as
// a second operand, which the streaming kernel can afford, it would make half as many MMAs again,
// and they are the bound here. It adds about as much error as the output's own rounding (1.4 times
// in all).
//
// Bound: the tensor cores, 4 D per visible (row, key), with the exponentials next: a 128 x 128
// tile costs 1024 cycles of MMA at D = 128 and as many of the special-function unit. Two tiles
// are in flight so that A's softmax runs beside B's MMAs; a third would not fit tensor memory
// (S and O of a tile take 256 of its 512 columns). A pair of tiles takes about 3100 cycles where
// MMAs and exponentials alone would take 2048 each: with two in flight, a tile's chain (S, its
// softmax of about 2000 cycles, P V) is not covered entirely.
//
// On one B200, bf16, 32 query heads of 128 over 8: 4093 new tokens at 32771 keys 1.94 ms, 1.06
// PFLOP/s, 64 % of a large matrix product's rate (at the 1000 W power limit, where the clock is
// 1.5 to 1.75 GHz); 8 causal prompts of up to 2048 tokens (62 GFLOP) 108 us, most of the rest in
// half-masked tiles and the starts and ends of short items; 12 ragged chunks of up to 300 tokens,
// 24 heads of 64 over 8, window 1000 (4.1 GFLOP) 38 us, of which the plan about 5.
// A chunk of 2048 tokens at 16384 keys keeps the tensor pipe and the special-function pipe each
// active 60 % of the time, and reads 85 MB from DRAM (87 % of the loads hit L2).
//
// Warps: 0-3 softmax and output of tile A, 4-7 of tile B (one thread per row: no exchange of
// maxima or sums; two threads per row spilt registers), 8 issues the MMAs of both tiles in turn,
// 9 the TMA copies, 10 clears V rows that no token of the item may see (their weight is 0, but
// 0 x NaN is not). K and V tiles share a ring in the order of their use: K0 V0 K1 V1 ...
//
// A cache of bytes (C8, attn.cuh has the arithmetic of its scales): tiles land as bytes, and warps 10 and
// 11 turn them into 16-bit operands in place; P is f16, its reference a base-2 logarithm that starts at
// the lowest scale of V in the first tile and may lag by 2^14; the scales come by plain loads of the
// copying warp. The chunk above takes 2.25 ms so (0.57 of a large product's rate; the 16-bit kernel 1.92 on
// the same GPU), 8 causal prompts of 53.8 GFLOP 129 us, 12 ragged chunks in f16 of 3.3 GFLOP 50 us: per
// operation 0.85, 0.75 and 0.63 of the 16-bit kernel. Of a chunk of 2048 tokens at 16384 keys (636 us) the
// tensor pipe is active 42 %, and 58 MB come from DRAM.
//
// k_attn_plan lists the pieces of a call (an item, or a part of its keys where items are too few
// or too long to fill the SMs evenly), largest first; parts leave (ref, l, O) in the workspace and
// k_attn_join puts them together in their order in the sequence.
#include "attn.cuh"

namespace ftb {
namespace {

constexpr int kTileK = 128;   // keys per tile
constexpr int kTileM = 128;   // rows per tile
constexpr int kThreadsC = 384;
constexpr int kWarpMma = 8, kWarpLoad = 9, kWarpFix = 10;
// C8 (a cache of bytes): warps 10 and 11 turn the tiles, each with so many 16-byte loads at once. More
// disturb the MMAs' reads of shared memory (1, 2, 4, 8: 2.50, 2.24, 2.55, 2.72 ms for 4093 tokens at 32771
// keys), and four such warps, which leave the softmax 200 registers, are no faster (2.36 ms).
constexpr int kTurners = 2, kInFlight = 2;
// registers: softmax 2 x 128 threads x 216 + 128 x 72 = 64512 = 384 x 168 at launch
constexpr int kRegsLaunch = 168, kRegsSoftmax = 216, kRegsOther = 72;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsOther <= kThreadsC * kRegsLaunch, "registers");
constexpr int kTmemS = 0, kTmemO = 256;  // + 128 for tile B
constexpr float kLazy = 8.f;             // log2 of what a score may exceed the reference by
// The same for a cache of bytes, whose P is always f16: as far as f16 goes. The scales' logarithms are
// terms of the exponents and widen their range, and a row that moves costs its warp a second pass (with 8
// in place of 14, 4093 tokens at 32771 keys whose scales differ by 4 took 4.1 ms).
constexpr float kLazyBytes = 14.f;
// log2 of what a row's maximum may fall short of it. f16 has no exponents to spare: 2^8 above the
// maximum, weights of 2^-17 of the largest would be rounded away, and many of those can hold much
// of the sum.
template <typename T>
constexpr float kShort = std::is_same<T, __half>::value ? 0.f : kLazy;

// ---- plan --------------------------------------------------------------------------------------

struct alignas(16) Piece {
  int q_tok;    // row of q of the first token
  int n_tok;    // tokens
  int seq, head;
  int pos;      // position of the first token
  int len;      // keys of the sequence
  int lo, hi;   // keys that the item's tokens see between them
  int t0, t1;   // key tiles of this piece
  int slot;     // part number in the workspace, -1: the whole item
  int pad;
};
static_assert(sizeof(Piece) == 48, "three 16-byte loads");

struct alignas(16) Join {
  int q_tok, n_tok, head, slot, parts;
  int pad[3];
};
static_assert(sizeof(Join) == 32, "two 16-byte loads");

// A sequence's tokens of two row tiles, as the plan keeps it.
struct PlanGroup {
  int seq, q_tok, n_tok, pos, len, lo, hi;  // as in Piece
  int t0, tiles;
  int place, part0;  // among its size class, and of its first part
};

struct Plan {
  int* head;        // kPlan* counts
  Piece* pieces;
  Join* joins;
  int* scratch;     // a PlanGroup per group, where they do not fit the plan block's shared memory
  int max_pieces, max_parts, max_joins, max_groups;
};
enum { kPlanPieces = 0, kPlanJoins = 1, kPlanNext = 2, kPlanInts = 64 };
constexpr int kClasses = 4;
constexpr int kPlanThreads = 512;
constexpr int kPartsPerSm = 8;
constexpr int kPlanSmem = 200 * 1024, kMaxBatch = kPlanSmem / 8;

// Parts of split items: their number, not the sizes of the call, bounds the workspace.
int plan_parts() { return kPartsPerSm * sm_count(); }

Plan carve_plan(char* base, int64_t groups, int Hkv, size_t* bytes) {
  size_t off = 0;
  auto take = [&](size_t n) {
    char* p = base ? base + off : nullptr;
    off += (n + 255) / 256 * 256;
    return p;
  };
  Plan p;
  p.max_parts = plan_parts();
  p.max_joins = p.max_parts / 2;
  p.max_groups = (int)groups;
  p.max_pieces = (int)(groups * Hkv + p.max_parts);
  p.head = reinterpret_cast<int*>(take(kPlanInts * 4));
  p.pieces = reinterpret_cast<Piece*>(take((size_t)p.max_pieces * sizeof(Piece)));
  p.joins = reinterpret_cast<Join*>(take((size_t)p.max_joins * sizeof(Join)));
  p.scratch = reinterpret_cast<int*>(take((size_t)groups * sizeof(PlanGroup)));
  *bytes = off;
  return p;
}

// Inclusive sums of N counts over the block; total[] gets the block's sums.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*red)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int u = __shfl_up_sync(0xffffffffu, v[k], o);
      if (lane >= o) v[k] += u;
    }
  __syncthreads();
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < N; ++k) red[k][warp] = v[k];
  __syncthreads();
  int w[N];
#pragma unroll
  for (int k = 0; k < N; ++k) w[k] = lane < kPlanThreads / 32 ? red[k][lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int u = __shfl_up_sync(0xffffffffu, w[k], o);
      if (lane >= o) w[k] += u;
    }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    total[k] = __shfl_sync(0xffffffffu, w[k], 31);
    const int before = __shfl_sync(0xffffffffu, w[k], (warp + 31) & 31);
    v[k] += warp ? before : 0;
  }
}

// How a group of `tiles` key tiles is cut: into `parts` pieces of at most `size` tiles.
struct Cut {
  int parts, size;
};
__device__ __forceinline__ Cut cut_group(int tiles, int most) {
  Cut c{1, tiles};
  if (tiles > most) {
    c.parts = (tiles + most - 1) / most;
    c.size = (tiles + c.parts - 1) / c.parts;
    c.parts = (tiles + c.size - 1) / c.size;
  }
  return c;
}

// One block. tok = tokens per group (two row tiles); blocks = blocks that will take the pieces.
__global__ void __launch_bounds__(kPlanThreads)
    k_attn_plan(const __grid_constant__ AttnParams P, const __grid_constant__ Plan plan, int tok,
                int blocks) {
  extern __shared__ int dyn[];
  __shared__ int red[kClasses + 1][32];
  __shared__ unsigned long long sum_tiles, cheapest;
  __shared__ int biggest, n_joins, most_best, tail_best, fine_best, parts_of[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* first_group = dyn;  // [batch + 1]
  pdl_launch_dependents();
  if (tid == 0) sum_tiles = 0, cheapest = ~0ull, biggest = 0, n_joins = 0;
  if (tid < 32) parts_of[tid] = 0;
  pdl_wait();
  int groups = 0;
  for (int b0 = 0; b0 < P.batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n[1] = {0}, total[1];
    if (b < P.batch) {
      const AttnSeq s = attn_seq(P, b);
      if (s.bad_len || s.bad_rows)
        atomicOr(P.status, (s.bad_len ? kAttnBadPage : 0u) | (s.bad_rows ? kAttnBadRows : 0u));
      n[0] = (s.n + tok - 1) / tok;
    }
    const int mine = n[0];
    block_scan<1>(n, total, red);
    if (b < P.batch) first_group[b] = groups + n[0] - mine;
    groups += total[0];
  }
  // (sequences that overlap, status bit 1, could make more groups than the rows allow)
  groups = min(groups, plan.max_groups);
  if (tid == 0) first_group[P.batch] = groups;
  __syncthreads();
  PlanGroup* group = reinterpret_cast<PlanGroup*>(dyn + P.batch + 1);
  if ((size_t)(P.batch + 1) * 4 + (size_t)groups * sizeof(PlanGroup) > (size_t)kPlanSmem)
    group = reinterpret_cast<PlanGroup*>(plan.scratch);
  int tiles_mine = 0, big = 0;
  for (int g = tid; g < groups; g += kPlanThreads) {
    int a = 0, z = P.batch;  // the sequence with first_group[a] <= g < first_group[a + 1]
    while (z - a > 1) {
      const int mid = (a + z) >> 1;
      if (first_group[mid] <= g)
        a = mid;
      else
        z = mid;
    }
    const AttnSeq s = attn_seq(P, a);
    const int i0 = (g - first_group[a]) * tok, n = min(tok, s.n - i0);
    const KeyRange r = attn_range(P, s, i0, i0 + n - 1);
    const bool any = r.lo < r.hi;
    const int t0 = any ? r.lo / kTileK : 0, t1 = any ? (r.hi + kTileK - 1) / kTileK : 0;
    group[g] = PlanGroup{a, s.q0 + i0, n, s.len - s.n + i0, s.len, r.lo, r.hi, t0, t1 - t0, 0, 0};
    tiles_mine += t1 - t0;
    big = max(big, t1 - t0);
  }
  tiles_mine = __reduce_add_sync(0xffffffffu, tiles_mine);
  big = __reduce_max_sync(0xffffffffu, big);
  if (lane == 0 && big > 0) {
    atomicAdd(&sum_tiles, (unsigned long long)tiles_mine);
    atomicMax(&biggest, big);
  }
  __syncthreads();
  // The longest piece: the longest item cut into 1, 2, ... parts (lane by lane). These fill some
  // whole rounds of the blocks; what is left for the last one may be cut 1..8 times finer (warp by
  // warp), so that all blocks share it. Whichever ends first by an estimate: pieces of the mean
  // size (less is lost to whole rounds where sizes differ: the small ones, last, fill the gaps),
  // kPieceTiles for the start and end of a piece, kJoinTiles more for a part that has to be joined
  // (133 KB at D = 128, both row tiles, written and read again). Against equal cuts of every item: 2048
  // tokens at 16384 keys, 256 items, 505 -> 465 us; 700 tokens of 64 heads over one, 175 items, 187
  // -> 137 us; 512 tokens at 65536 keys, 64 long items, 504 -> 510 us.
  constexpr int kPieceTiles = 2, kJoinTiles = 3, kFewest = 2, kFiner = 8;
  const int top = max(biggest, 1);
  const int ways = lane < 16 ? lane + 1 : (lane - 13) * (lane - 13) / 2 + 12;  // 1..16, 16.., 174
  const int most = max((top + ways - 1) / ways, kFewest);
  int n_mine = 0;
  for (int g = warp; g < groups; g += kPlanThreads / 32)
    n_mine += cut_group(group[g].tiles, most).parts;
  if (n_mine) atomicAdd(&parts_of[lane], n_mine);
  __syncthreads();
  if (warp < kFiner) {
    const float n = (float)parts_of[lane] * P.Hkv, items = (float)groups * P.Hkv;
    const float k = (float)(warp + 1), per_block = 1.f / (float)blocks;
    const float tiles = (float)sum_tiles * P.Hkv, mean = n > 0.f ? tiles / n : 0.f;
    const float rounds = floorf((n + 0.5f) * per_block), left = n - rounds * (float)blocks;
    const float last = ceilf((left * k - 0.5f) * per_block);  // rounds of the finer pieces
    const float even = tiles * per_block, gap = mean * (rounds + last / k) - even;
    const float alike = fmaxf(0.f, 2.f * mean / (float)most - 1.f);  // 1: all of the longest's size
    const float joined = n > items ? n + left * (k - 1.f) : warp ? left * k : 0.f;
    float cost = fmaxf((float)most, even + gap * alike) + kPieceTiles * (rounds + last) +
                 kJoinTiles * joined * per_block;
    // (parts <= 2 (pieces - items): in whole numbers, since past 2^24 pieces the difference of two
    // floats is off by more than the workspace allows. The finer cut is counted again below.)
    const long long more = (long long)(parts_of[lane] - groups) * P.Hkv;
    if ((warp && mean < k * kFewest) || more > plan.max_parts / 2 ||
        n - items + left * (k - 1.f) > (float)(plan.max_parts / 2))
      cost = INFINITY;
    const unsigned long long key = (unsigned long long)__float_as_uint(cost) << 32 |
                                   (uint32_t)(warp << 5 | lane);  // (costs are not negative)
    atomicMin(&cheapest, key);
  }
  __syncthreads();
  if (tid == (int)(cheapest & 0xffffffffu)) {
    most_best = most;
    const float n = (float)parts_of[lane];
    const int left = (int)((long long)parts_of[lane] * P.Hkv % blocks);
    tail_best = warp ? (int)ceilf((float)left * (float)groups / (n * P.Hkv)) : 0;
    fine_best = (most + warp) / (warp + 1);
  }
  __syncthreads();
  const int limit = min(most_best, top), fine = min(fine_best, limit);
  int tail = min(tail_best, groups);  // groups 0..tail-1 are cut finer
  // places: largest pieces first, by class
  int run[kClasses + 1];
  for (;;) {
#pragma unroll
    for (int i = 0; i <= kClasses; ++i) run[i] = 0;
    for (int g0 = 0; g0 < groups; g0 += kPlanThreads) {
      const int g = g0 + tid;
      int v[kClasses + 1] = {}, total[kClasses + 1];
      int k = 0, parts = 0;
      if (g < groups) {
        const Cut c = cut_group(group[g].tiles, g < tail ? fine : limit);
        k = min(kClasses - 1, (limit - c.size) * kClasses / limit);
        parts = c.parts;
#pragma unroll
        for (int i = 0; i < kClasses; ++i) v[i] = i == k ? parts : 0;
        v[kClasses] = parts > 1 ? parts : 0;
      }
      block_scan<kClasses + 1>(v, total, red);
      if (g < groups) {
        int at = 0;
#pragma unroll
        for (int i = 0; i < kClasses; ++i)
          if (i == k) at = run[i] + v[i] - parts;
        group[g].place = at;
        group[g].part0 = run[kClasses] + v[kClasses] - (parts > 1 ? parts : 0);
      }
#pragma unroll
      for (int i = 0; i <= kClasses; ++i) run[i] += total[i];
    }
    // (the estimate counts pieces of the mean size: where the finer cut makes more parts than there
    // is room for, it is left out)
    if (tail == 0 || run[kClasses] * P.Hkv <= plan.max_parts) break;
    tail = 0;
  }
  __syncthreads();
  // emission: a warp per group, a lane per piece; in a class one kv head after another, so that
  // blocks that run at the same time share keys
  for (int g = warp; g < groups; g += kPlanThreads / 32) {
    const PlanGroup u = group[g];
    const Cut c = cut_group(u.tiles, g < tail ? fine : limit);
    const int k = min(kClasses - 1, (limit - c.size) * kClasses / limit);
    int start = 0, per_head = 0;
#pragma unroll
    for (int i = 0; i < kClasses; ++i) {
      if (i < k) start += run[i] * P.Hkv;
      if (i == k) per_head = run[i];
    }
    for (int i = lane; i < c.parts * P.Hkv; i += 32) {
      const int head = i / c.parts, part = i - head * c.parts, t0 = u.t0 + part * c.size;
      Piece p{u.q_tok, u.n_tok, u.seq, head, u.pos, u.len, u.lo, u.hi, t0,
              min(t0 + c.size, u.t0 + u.tiles), c.parts > 1 ? u.part0 * P.Hkv + i : -1, 0};
      int4* to = reinterpret_cast<int4*>(plan.pieces + start + head * per_head + u.place + part);
      to[0] = make_int4(p.q_tok, p.n_tok, p.seq, p.head);
      to[1] = make_int4(p.pos, p.len, p.lo, p.hi);
      to[2] = make_int4(p.t0, p.t1, p.slot, 0);
      if (c.parts > 1 && part == 0) {
        Join o{};
        o.q_tok = p.q_tok, o.n_tok = p.n_tok, o.head = head, o.slot = p.slot, o.parts = c.parts;
        plan.joins[atomicAdd(&n_joins, 1)] = o;
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kClasses; ++i) n += run[i] * P.Hkv;
    plan.head[kPlanPieces] = n;
    plan.head[kPlanJoins] = n_joins;
    plan.head[kPlanNext] = blocks;
  }
}

// ---- tensor-core helpers -----------------------------------------------------------------------

// Shared-memory operand descriptors, 128-byte swizzle, 8-row atoms 1024 bytes apart. K-major (Q,
// K): rows of 64 elements. MN-major (V): a row is a key; blocks of 64 of the D columns are
// kTileK * 128 bytes apart.
// The high word is the same for all: the helpers below take the low one.
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo) {
  return ((saddr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16);
}
// Instruction descriptor, kind::f16: fp32 D, A and B bf16 or f16, M = 128, B K-major or MN-major.
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_mn) {
  const uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileM >> 4) << 24);
}
// Issued by one elected lane of the converged warp.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 y, {%2, %5};\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_commit1(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tc_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// 32 columns of this warp's 32 lanes (no wait).
__device__ __forceinline__ void tm_ld32(uint32_t t, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t)
      : "memory");
}
// 16 columns of this warp's 32 lanes (no wait).
__device__ __forceinline__ void tm_ld16(uint32_t t, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(t),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tm_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int x, int g, int head,
                                       int tok, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(g), "r"(head), "r"(tok), "r"(smem_u32(bar))
      : "memory");
}
// Two fp32 values as one operand of the packed instructions.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
// Packed and special-function instructions as volatile statements, which keep their order.
__device__ __forceinline__ uint64_t fma2v(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2v(uint64_t a, uint64_t b) {
  uint64_t r;
  asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2v(float x) {
  float r;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2v(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float max3v(float a, float b, float c) {
  float r;
  asm volatile("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ---- the kernel --------------------------------------------------------------------------------

constexpr int kPieceRing = 4, kPieceReaders = 8 + 2;  // softmax warps, MMA, fixer (C8: kTurners)
// Three Q buffers for the two tiles: the next item's A comes in while this one is still in use.
constexpr int kQBufs = 3;
constexpr int chunk_stages(int DP) { return DP == 128 ? 4 : 8; }
// C8: the cache is one of bytes. A tile's rows of 128 bytes land in the last 16 KB of its stage and are
// turned into f16 in place.
// Key tiles whose scales are kept. A tile's scales come when its K stage is free, that is after S of the
// tile kStages / 2 before it, which followed P of the one before that: so many tiles and one more may
// still be read, and a tile further back is not.
constexpr int scale_ring(int DP) { return DP == 128 ? 4 : 8; }
constexpr int kGroup = 16;      // keys that share their scales for certain
template <int DP, bool C8>
struct ChunkSmem {
  static constexpr int kStages = chunk_stages(DP);
  static constexpr int kTileBytes = kTileK * DP * 2;
  static constexpr int kScaleRing = scale_ring(DP);
  static_assert(kScaleRing > kStages / 2, "no scales are written over that are still read");
  alignas(1024) uint8_t q[kQBufs][kTileBytes];      // [half][row][64]
  alignas(1024) uint8_t ring[kStages][kTileBytes];  // [half][key][64]
  // of each kGroup keys: the scale of K, log2 and reciprocal of V's, and (in the first) the lowest log2
  float4 scale[C8 ? kScaleRing : 1][kTileK / kGroup];
  uint64_t full[kStages], empty[kStages];
  uint64_t land[kStages];  // a V tile that the fixer completes has landed (C8: any tile)
  uint64_t q_full[kQBufs], q_empty[kQBufs];
  uint64_t scale_full[C8 ? kScaleRing : 1];
  uint64_t s_full[2], p_ready[2][2], o_full[2];  // p_ready: by halves of the keys
  Piece piece[kPieceRing];
  uint64_t piece_full[kPieceRing], piece_empty[kPieceRing];
  uint64_t drain;
  uint32_t tmem;
  int abort;
};

template <int DP, bool C8>
struct ChunkSync {
  ChunkSmem<DP, C8>* sh;
  uint32_t* status;
  __device__ bool wait(uint64_t* bar, uint32_t parity) const {
    if (mbar_try_wait(bar, parity)) return true;
    volatile int* ab = &sh->abort;
    for (uint32_t i = 0; i < kSpinLimit; ++i) {
      if (*ab) return false;
      if (mbar_try_wait(bar, parity)) return true;
      if (i > (1u << 16)) __nanosleep(64);
    }
    *ab = 1;
    atomicOr(status, kAttnTimeout);
    return false;
  }
  __device__ bool wait_warp(uint64_t* bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, wait(bar, parity));
  }
};

// Blocks take pieces from the list as they come free: block x starts with piece x, the next ones
// go by a counter. The copying warp fetches them and passes them on through a ring.
__device__ __forceinline__ Piece load_piece(const Piece* p) {
  Piece r;
  const int4* s = reinterpret_cast<const int4*>(p);
  int4* d = reinterpret_cast<int4*>(&r);
  d[0] = __ldcg(s), d[1] = __ldcg(s + 1), d[2] = __ldcg(s + 2);
  return r;
}
template <int DP, bool C8>
struct PieceReader {
  int at = 0;
  uint32_t parity = 0;
  // the next piece; false at the end of the list or after a timeout
  __device__ bool next(const ChunkSync<DP, C8>& sy, Piece& p) {
    if (!sy.wait_warp(&sy.sh->piece_full[at], parity)) return false;
    p = sy.sh->piece[at];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sy.sh->piece_empty[at]);
    if (++at == kPieceRing) at = 0, parity ^= 1u;
    return p.seq >= 0;
  }
};
// Rows and key tiles of tile X of a piece: its first and last token, tiles [t0, t0 + n).
struct RowTile {
  int tok0, toks, n;
};
__device__ __forceinline__ RowTile row_tile(const AttnParams& P, const Piece& p, int x, int tok1) {
  RowTile r;
  r.tok0 = x * tok1;
  r.toks = min(tok1, p.n_tok - r.tok0);
  r.n = 0;
  if (r.toks <= 0) {
    r.toks = 0;
    return r;
  }
  int hi = p.hi;
  if (P.causal) hi = min(hi, p.pos + r.tok0 + r.toks);
  const int t1 = min(p.t1, (hi + kTileK - 1) / kTileK);  // hi may be <= 0
  r.n = max(0, t1 - p.t0);
  return r;
}

template <int DP>
__device__ void chunk_load(const AttnParams& P, const AttnMaps& M, const Plan& plan, int tok1,
                           ChunkSmem<DP, false>* sh) {
  constexpr int kStages = ChunkSmem<DP, false>::kStages, kH = DP / 64;
  const int lane = threadIdx.x & 31;
  const ChunkSync<DP, false> sy{sh, P.status};
  const int page = 1 << P.page_log2;
  const int r = page < kTileK ? page : kTileK;
  const int boxes = kTileK / r;  // <= 16
  const uint32_t box_bytes = (uint32_t)r * 128 * kH;
  const uint32_t q_bytes = (uint32_t)(tok1 * P.G) * 128 * kH;
  int stage = 0;
  int qb = 0;  // next Q buffer
  uint32_t parity = 1, q_par = 1;
  // for the exit: stages whose last copy signals land[], a bit each
  uint32_t on_land = 0, land_par = 0;  // parity of a stage's next phase on land[]
  bool ok = true, first_round = true;
  // (the first piece is loaded before the length of the list is known: there is one at least)
  Piece p = load_piece(plan.pieces + blockIdx.x);
  const int n_pieces = __ldcg(plan.head + kPlanPieces);
  if ((int)blockIdx.x >= n_pieces) p.seq = -1;
  int slot = 0;
  uint32_t slot_parity = 1;
  for (;;) {
    ok = sy.wait_warp(&sh->piece_empty[slot], slot_parity);
    if (!ok) break;
    if (lane == 0) {
      sh->piece[slot] = p;
      mbar_arrive(&sh->piece_full[slot]);
    }
    if (++slot == kPieceRing) slot = 0, slot_parity ^= 1u;
    if (p.seq < 0) break;
    const RowTile ra = row_tile(P, p, 0, tok1), rb = row_tile(P, p, 1, tok1);
    const int n = max(ra.n, rb.n);
    const int32_t* table = P.block_table + (int64_t)p.seq * P.table_stride;
    auto load_q = [&](const RowTile& rt) {
      if (!sy.wait_warp(&sh->q_empty[qb], q_par)) return false;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh->q_full[qb], q_bytes);
#pragma unroll
        for (int h = 0; h < kH; ++h)
          tma_4d(smem_u32(sh->q[qb]) + h * kTileM * 128, &M.q, h * 64, 0, p.head,
                 p.q_tok + rt.tok0, &sh->q_full[qb]);
      }
      __syncwarp();
      if (++qb == kQBufs) qb = 0, q_par ^= 1u;
      return true;
    };
    // Q of A, K0, Q of B (whose buffer comes free last), V0, K1, V1, ...
    if (ra.n > 0) ok = load_q(ra);
    for (int j = 0; j < 2 * n && ok; ++j) {
      const bool v = j & 1;
      const int key0 = (p.t0 + (j >> 1)) * kTileK;
      const int b0 = p.lo > key0 ? (p.lo - key0) / r : 0;
      const int b1 = min(boxes, (p.hi - key0 + r - 1) / r);
      const bool mine = lane >= b0 && lane < b1;
      int id = 0, row = 0;
      if (mine) {
        const int key = key0 + lane * r;
        id = table[key >> P.page_log2];
        row = key & (page - 1);
        if (id < 0 || id >= P.num_pages) {
          atomicOr(P.status, kAttnBadPage);
          id = (int)P.num_pages;  // outside the tensor: reads zeros
        }
      }
      ok = sy.wait_warp(&sh->empty[stage], parity);
      if (!ok) break;
      const bool fix = v && (key0 < p.lo || key0 + kTileK > p.hi);
      uint64_t* bar = fix ? &sh->land[stage] : &sh->full[stage];
      on_land = fix ? on_land | 1u << stage : on_land & ~(1u << stage);
      land_par ^= (uint32_t)fix << stage;
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(b1 - b0) * box_bytes);
      __syncwarp();
      if (mine) {
        const uint32_t dst = smem_u32(sh->ring[stage]) + lane * r * 128;
#pragma unroll
        for (int h = 0; h < kH; ++h)
          tma_5d(dst + h * kTileK * 128, v ? &M.v : &M.k, h * 64, row, p.head, id, 0, bar);
      }
      if (++stage == kStages) stage = 0, parity ^= 1u, first_round = false;
      if (j == 0 && rb.n > 0) ok = load_q(rb);
    }
    if (!ok) break;
    // (taken only now: a block that took its next piece early could hold it while others idle)
    int next = 0;
    if (lane == 0) next = atomicAdd(plan.head + kPlanNext, 1);
    next = __shfl_sync(0xffffffffu, next, 0);
    if (next < n_pieces)
      p = load_piece(plan.pieces + next);
    else
      p.seq = -1;
  }
  // Stay until the last copies have landed, again with a limit: a warp that gave up leaves without
  // them.
  for (int i = 0; i < kStages; ++i) {
    // the last use of stage i: this round of the ring before `stage`, the one before after it
    const bool land = on_land >> i & 1u;
    const uint32_t par = land ? (land_par >> i & 1u) ^ 1u : i < stage ? parity ^ 1u : parity;
    if (!land && i >= stage && first_round) continue;  // never used
    for (uint32_t k = 0; k < kSpinLimit; ++k)
      if (mbar_try_wait(land ? &sh->land[i] : &sh->full[i], par)) break;
  }
  for (int i = 0; i < kQBufs; ++i)  // (before a buffer's first copy: passes at once)
    for (uint32_t k = 0; k < kSpinLimit; ++k)
      if (mbar_try_wait(&sh->q_full[i], i < qb ? q_par ^ 1u : q_par)) break;
}

// Clears the rows of V tiles that no token of the piece's item sees.
template <int DP>
__device__ void chunk_fix(const AttnParams& P, int tok1, ChunkSmem<DP, false>* sh) {
  constexpr int kStages = ChunkSmem<DP, false>::kStages, kH = DP / 64;
  const int lane = threadIdx.x & 31;
  const ChunkSync<DP, false> sy{sh, P.status};
  int stage = 0;
  uint32_t land_par = 0;  // a bit per stage
  PieceReader<DP, false> pieces;
  for (Piece p; pieces.next(sy, p);) {
    const RowTile ra = row_tile(P, p, 0, tok1), rb = row_tile(P, p, 1, tok1);
    const int n = max(ra.n, rb.n);
    for (int j = 0; j < n; ++j) {
      if (++stage == kStages) stage = 0;  // past K
      const int key0 = (p.t0 + j) * kTileK;
      if (key0 < p.lo || key0 + kTileK > p.hi) {
        if (!sy.wait_warp(&sh->land[stage], (land_par >> stage) & 1u)) return;
        land_par ^= 1u << stage;
        const int below = max(0, p.lo - key0), above = min(kTileK, p.hi - key0);
        const int rows = below + kTileK - above;
        for (int i = lane; i < rows * 8 * kH; i += 32) {
          const int c = i & 7, k = (i >> 3) % rows, h = (i >> 3) / rows;
          const int key = k < below ? k : above + k - below;
          *reinterpret_cast<uint4*>(sh->ring[stage] + h * kTileK * 128 + key * 128 + c * 16) =
              make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->full[stage]);
      }
      if (++stage == kStages) stage = 0;  // past V
    }
  }
}

// Where in its stage a tile of bytes lands.
constexpr int raw_at(int tile_bytes) { return tile_bytes - kTileK * 128; }

// chunk_load for a cache of bytes. All tiles signal land[]; lanes 0..7 bring the scales of the tile's
// groups of keys.
template <int DP>
__device__ void chunk_load8(const AttnParams& P, const AttnMaps& M, const Plan& plan, int tok1,
                            ChunkSmem<DP, true>* sh) {
  using Smem = ChunkSmem<DP, true>;
  constexpr int kStages = Smem::kStages, kH = DP / 64, kGroups = kTileK / kGroup;
  const int lane = threadIdx.x & 31;
  const ChunkSync<DP, true> sy{sh, P.status};
  const int page = 1 << P.page_log2;
  const int r = page < kTileK ? page : kTileK;  // >= kGroup
  const int boxes = kTileK / r;                 // <= 8
  const uint32_t q_bytes = (uint32_t)(tok1 * P.G) * 128 * kH;
  int stage = 0, qb = 0, sc = 0;
  uint32_t parity = 1, q_par = 1;
  uint32_t land_next = 0;  // parity of a stage's next phase on land[], a bit each
  uint32_t used = 0;       // stages that had a copy
  bool ok = true;
  Piece p = load_piece(plan.pieces + blockIdx.x);
  const int n_pieces = __ldcg(plan.head + kPlanPieces);
  if ((int)blockIdx.x >= n_pieces) p.seq = -1;
  int slot = 0;
  uint32_t slot_parity = 1;
  for (;;) {
    ok = sy.wait_warp(&sh->piece_empty[slot], slot_parity);
    if (!ok) break;
    if (lane == 0) {
      sh->piece[slot] = p;
      mbar_arrive(&sh->piece_full[slot]);
    }
    if (++slot == kPieceRing) slot = 0, slot_parity ^= 1u;
    if (p.seq < 0) break;
    const RowTile ra = row_tile(P, p, 0, tok1), rb = row_tile(P, p, 1, tok1);
    const int n = max(ra.n, rb.n);
    const int32_t* table = P.block_table + (int64_t)p.seq * P.table_stride;
    auto load_q = [&](const RowTile& rt) {
      if (!sy.wait_warp(&sh->q_empty[qb], q_par)) return false;
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh->q_full[qb], q_bytes);
#pragma unroll
        for (int h = 0; h < kH; ++h)
          tma_4d(smem_u32(sh->q[qb]) + h * kTileM * 128, &M.q, h * 64, 0, p.head,
                 p.q_tok + rt.tok0, &sh->q_full[qb]);
      }
      __syncwarp();
      if (++qb == kQBufs) qb = 0, q_par ^= 1u;
      return true;
    };
    if (ra.n > 0) ok = load_q(ra);
    for (int j = 0; j < n && ok; ++j) {
      const int key0 = (p.t0 + j) * kTileK;
      const int b0 = p.lo > key0 ? (p.lo - key0) / r : 0;
      const int b1 = min(boxes, (p.hi - key0 + r - 1) / r);
      // page of this lane's group of keys, and its scales
      const int key = key0 + lane * kGroup, box_of = lane * kGroup / r;
      const bool has = lane < kGroups && box_of >= b0 && box_of < b1;
      int id = 0;
      if (has) {
        id = table[key >> P.page_log2];
        if (id < 0 || id >= P.num_pages) {
          atomicOr(P.status, kAttnBadPage);
          id = (int)P.num_pages;  // outside the tensor: reads zeros
        }
      }
      // (a block of the same page that no token sees may have any scale: it takes no part in the lowest)
      const bool seen = has && key < p.hi && key + kGroup > p.lo;
      float ks = 1.f, vs = seen ? 1.f : kMaxScale;
      if (seen && id < P.num_pages) {
        const int block = (key & (page - 1)) >> P.block_log2;
        ks = P.k_scale[id * P.ks_st[0] + block * P.ks_st[1] + p.head * P.ks_st[2]];
        vs = P.v_scale[id * P.vs_st[0] + block * P.vs_st[1] + p.head * P.vs_st[2]];
      }
      const int box_id = __shfl_sync(0xffffffffu, id, (lane * r / kGroup) & (kGroups - 1));
      const bool mine = lane >= b0 && lane < b1;
      for (int v = 0; v < 2 && ok; ++v) {
        ok = sy.wait_warp(&sh->empty[stage], parity);
        if (!ok) break;
        uint64_t* bar = &sh->land[stage];
        used |= 1u << stage;
        land_next ^= 1u << stage;
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(b1 - b0) * (uint32_t)r * 128u);
        __syncwarp();
        if (mine)
          tma_5d(smem_u32(sh->ring[stage]) + raw_at(Smem::kTileBytes) + lane * r * 128, v ? &M.v : &M.k, 0,
                 (key0 + lane * r) & (page - 1), p.head, box_id, 0, bar);
        if (++stage == kStages) stage = 0, parity ^= 1u;
        if (v == 0) {
          const BlockScale b = block_scale(ks, vs);
          float low = b.v_log2;
#pragma unroll
          for (int o = 1; o < kGroups; o <<= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
          if (lane < kGroups) sh->scale[sc][lane] = make_float4(b.k, b.v_log2, b.v_inv, low);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->scale_full[sc]);
          if (++sc == Smem::kScaleRing) sc = 0;
          if (j == 0 && rb.n > 0) ok = load_q(rb);
        }
      }
    }
    if (!ok) break;
    int next = 0;
    if (lane == 0) next = atomicAdd(plan.head + kPlanNext, 1);
    next = __shfl_sync(0xffffffffu, next, 0);
    if (next < n_pieces)
      p = load_piece(plan.pieces + next);
    else
      p.seq = -1;
  }
  // Stay until the last copies have landed, as above.
  for (int i = 0; i < kStages; ++i) {
    if (!(used >> i & 1u)) continue;
    for (uint32_t k = 0; k < kSpinLimit; ++k)
      if (mbar_try_wait(&sh->land[i], (land_next >> i & 1u) ^ 1u)) break;
  }
  for (int i = 0; i < kQBufs; ++i)
    for (uint32_t k = 0; k < kSpinLimit; ++k)
      if (mbar_try_wait(&sh->q_full[i], i < qb ? q_par ^ 1u : q_par)) break;
}

// 16 codes as numbers of T (exact, NaN among them).
template <typename T>
__device__ __forceinline__ void codes16(const uint4& x, uint32_t (&f)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = e4m3x2_to_f16x2((uint16_t)(w[i] & 0xffffu));
    f[2 * i + 1] = e4m3x2_to_f16x2((uint16_t)(w[i] >> 16));
  }
  if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = unpack2<__half>(f[i]);
      f[i] = pack2<T>(v.x, v.y);
    }
  }
}

// kTurners warps (`part` of the rows each) turn what lands into 16-bit operands, in place: K into q's type
// T, since both operands of a product have one, V into f16, like P. (Turning bf16 queries into f16
// instead kept the start of an item waiting: 8 prompts 144 us against 129.) A row's bytes
// become (DP = 128) a row of the first 64 elements in the lower half of the stage and one of the others
// where the bytes were, so no row waits for another. V rows that no token sees become zeros.
template <typename T, int DP>
__device__ void chunk_turn(const AttnParams& P, int tok1, int part, ChunkSmem<DP, true>* sh) {
  using Smem = ChunkSmem<DP, true>;
  constexpr int kStages = Smem::kStages;
  const int lane = threadIdx.x & 31;
  const ChunkSync<DP, true> sy{sh, P.status};
  constexpr int kLanes = DP / 16;        // lanes of a row, 16 bytes each
  constexpr int kRows = 32 / kLanes;     // rows of an access of the warp
  constexpr int kAccesses = kTileK / kTurners / kRows;
  const int c = lane % kLanes;           // elements 16 c ..: two 16-byte chunks of half h
  const int h = c >> 2, o = 2 * (c & 3);
  // The rows that eight lanes meet together. DP = 128: the second half of the row beside the one whose
  // first half the others turn, which the swizzle puts into the other eight chunks' banks. DP = 64: rows
  // 4 apart, for the same reason.
  const int row0 = part * (kTileK / kTurners) +
                   (DP == 64 ? (lane / kLanes >> 1) + 4 * (lane / kLanes & 1) : lane / kLanes ^ h);
  int stage = 0;
  uint32_t land_par = 0;  // a bit per stage
  PieceReader<DP, true> pieces;
  for (Piece p; pieces.next(sy, p);) {
    const int n = max(row_tile(P, p, 0, tok1).n, row_tile(P, p, 1, tok1).n);
    for (int j = 0; j < 2 * n; ++j) {
      const int key0 = (p.t0 + (j >> 1)) * kTileK;
      if (!sy.wait_warp(&sh->land[stage], (land_par >> stage) & 1u)) return;
      land_par ^= 1u << stage;
      uint8_t* tile = sh->ring[stage];
      constexpr int kAtOnce = kAccesses < kInFlight ? kAccesses : kInFlight;
      auto turn = [&](auto type, bool cut) {
#pragma unroll 1
        for (int u0 = 0; u0 < kAccesses; u0 += kAtOnce) {
          uint4 x[kAtOnce];
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int row = row0 + (u0 + u) * kRows;
            x[u] = *reinterpret_cast<const uint4*>(tile + raw_at(Smem::kTileBytes) + row * 128 +
                                                   ((c ^ (row & 7)) << 4));
            if (cut && (key0 + row < p.lo || key0 + row >= p.hi)) x[u] = make_uint4(0, 0, 0, 0);
          }
          __syncwarp();  // a row's bytes have been read before they are written over
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int row = row0 + (u0 + u) * kRows;
            uint32_t f[8];
            codes16<decltype(type)>(x[u], f);
            uint8_t* to = tile + h * kTileK * 128 + row * 128;
            *reinterpret_cast<uint4*>(to + ((o ^ (row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<uint4*>(to + ((o + 1 ^ (row & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
          }
        }
      };
      if (j & 1)
        turn(__half(), key0 < p.lo || key0 + kTileK > p.hi);
      else
        turn(T(), false);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->full[stage]);
      if (++stage == kStages) stage = 0;
    }
  }
}

// T: q's type.
template <typename T, int DP, bool C8>
__device__ void chunk_mma(const AttnParams& P, int tok1, ChunkSmem<DP, C8>* sh) {
  constexpr int kStages = ChunkSmem<DP, C8>::kStages;
  constexpr int kTileBytes = ChunkSmem<DP, C8>::kTileBytes;
  const ChunkSync<DP, C8> sy{sh, P.status};
  const uint32_t tb = sh->tmem;
  const uint32_t qd = desc_low(smem_u32(sh->q[0]), 16);
  const uint32_t kd = desc_low(smem_u32(sh->ring[0]), 16);
  const uint32_t vd = desc_low(smem_u32(sh->ring[0]), kTileK * 128);
  using TP = typename std::conditional<C8, __half, T>::type;  // P's and V's type
  constexpr uint32_t kIdS = idesc<T>(kTileK, false), kIdO = idesc<TP>(DP, true);
  int stage = 0;
  int qb = 0, q_of[2] = {0, 0};  // next Q buffer; the tiles' buffers
  uint32_t parity = 0, q_par = 0, p_par[2] = {0, 0};
  // tile x's P V of the last step: not issued yet; whether it adds to O, ends its row tile
  bool pend[2] = {false, false}, acc[2] = {false, false}, last[2] = {false, false};
  int v_stage = -1;
  uint32_t v_par = 0;
  bool v_there = false, ok = true, issued = false;

  auto pv = [&](int x) {
    ok = sy.wait_warp(&sh->p_ready[x][0], p_par[x]);
    if (!ok) return;
    if (!v_there) {
      ok = sy.wait_warp(&sh->full[v_stage], v_par);
      if (!ok) return;
      v_there = true;
    }
    tc_after();
    const uint32_t d = tb + kTmemO + x * 128, a = tb + kTmemS + x * 128;
    const uint32_t b = vd + (uint32_t)((v_stage * kTileBytes) >> 4);
#pragma unroll
    for (int k = 0; k < kTileK / 16; ++k) {
      if (k == kTileK / 32) {
        ok = sy.wait_warp(&sh->p_ready[x][1], p_par[x]);
        if (!ok) return;
        tc_after();
      }
      mma_ts(d, a + k * 8, b + (uint32_t)((k * 16 * 128) >> 4), kIdO, (k > 0 || acc[x]) ? 1u : 0u);
    }
    p_par[x] ^= 1u;
    if (last[x]) mma_commit1(&sh->o_full[x]);
    pend[x] = false;
  };

  PieceReader<DP, C8> pieces;
  for (Piece p; ok && pieces.next(sy, p);) {
    const int nx[2] = {row_tile(P, p, 0, tok1).n, row_tile(P, p, 1, tok1).n};
    const int n = max(nx[0], nx[1]);
    // An item without keys brings no step to issue the last P V of the one before in. The softmax warps
    // wait for that before they take another item, so a ring full of such items would never move on.
    if (n == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (ok && pend[x]) pv(x);
    }
    for (int j = 0; j < n && ok; ++j) {
      ok = sy.wait_warp(&sh->full[stage], parity);
      if (!ok) break;
      issued = true;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (pend[x]) pv(x);
        if (!ok) break;
        if (j >= nx[x]) continue;
        if (j == 0) {
          ok = sy.wait_warp(&sh->q_full[qb], q_par);
          if (!ok) break;
          q_of[x] = qb;
          if (++qb == kQBufs) qb = 0, q_par ^= 1u;
        }
        tc_after();
        const uint32_t a = qd + (uint32_t)((q_of[x] * kTileBytes) >> 4);
        const uint32_t b = kd + (uint32_t)((stage * kTileBytes) >> 4);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t o = (uint32_t)(((k >> 2) * kTileK * 128 + (k & 3) * 32) >> 4);
          mma_ss(tb + kTmemS + x * 128, a + o, b + o, kIdS, k > 0 ? 1u : 0u);
        }
        mma_commit1(&sh->s_full[x]);
        pend[x] = true, acc[x] = j > 0, last[x] = j == nx[x] - 1;
      }
      if (!ok) break;
      if (v_stage >= 0) mma_commit1(&sh->empty[v_stage]);
      mma_commit1(&sh->empty[stage]);
      if (++stage == kStages) stage = 0, parity ^= 1u;
      v_stage = stage, v_par = parity, v_there = false;
      if (++stage == kStages) stage = 0, parity ^= 1u;
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (ok && pend[x]) pv(x);
  if (issued) {  // every MMA has finished once the drain barrier completes
    mma_commit1(&sh->drain);
    for (uint32_t k = 0; k < kSpinLimit; ++k)
      if (mbar_try_wait(&sh->drain, 0)) break;
  }
}

// 32 bytes, one sector.
__device__ __forceinline__ void st_sector(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

template <typename T, int DP, bool C8>
__device__ void chunk_softmax(const AttnParams& P, int tok1, int x, ChunkSmem<DP, C8>* sh) {
  using TP = typename std::conditional<C8, __half, T>::type;  // P's type
  const ChunkSync<DP, C8> sy{sh, P.status};
  const int row = threadIdx.x & 127, lane = threadIdx.x & 31;
  const uint32_t lanes = (uint32_t)(row & ~31) << 16;
  const uint32_t ts = sh->tmem + kTmemS + x * 128 + lanes, to = sh->tmem + kTmemO + x * 128 + lanes;
  const int tok = row / P.G, g = row % P.G;
  // scores are multiplied by |scale|; a negative scale flips their sign first. A scale of 0
  // becomes one that is small enough to be flat and keeps a masked -inf at -inf.
  const bool flip = P.scale_log2 < 0.f;
  const float sc = fmaxf(fabsf(P.scale_log2), 1e-30f);
  int q_next = 0;
  uint32_t tile_at = 0;  // C8: key tiles of the pieces before
  uint32_t s_par = 0, o_par = 0;
  constexpr int kSlot = 2 * kTileM * (DP + 2);
  PieceReader<DP, C8> pieces;
  for (Piece p; pieces.next(sy, p);) {
    const RowTile rt = row_tile(P, p, x, tok1);
    // Q buffers are taken in order: A's, B's, the next item's A's, ...
    const int n_other = row_tile(P, p, x ^ 1, tok1).n;
    int q_mine = q_next;
    if (rt.n > 0 && x == 1 && n_other > 0) q_mine = q_mine + 1 == kQBufs ? 0 : q_mine + 1;
    q_next += (rt.n > 0) + (n_other > 0);
    if (q_next >= kQBufs) q_next -= kQBufs;
    const uint32_t tile0 = tile_at;
    if constexpr (C8) tile_at += max(rt.n, n_other);
    if (rt.toks == 0) continue;
    const bool live = tok < rt.toks;
    // keys this row sees: [kmin, kmax); the tile's rows all see [tile_min, tile_max)
    const int pos0 = p.pos + rt.tok0;
    const int kmax = !live ? 0 : P.causal ? min(p.len, pos0 + tok + 1) : p.len;
    const int kmin = P.window > 0 ? max(0, pos0 + tok - P.window + 1) : 0;
    const int all_max = P.causal ? min(p.len, pos0 + 1) : p.len;
    const int all_min = P.window > 0 ? max(0, pos0 + rt.toks - 1 - P.window + 1) : 0;
    float ref = -INFINITY, l = 0.f;
    for (int j = 0; j < rt.n; ++j) {
      if (!sy.wait_warp(&sh->s_full[x], s_par)) return;
      s_par ^= 1u;
      tc_after();
      const float4* scales = nullptr;
      if constexpr (C8) {
        constexpr uint32_t kScaleRing = ChunkSmem<DP, C8>::kScaleRing;
        const uint32_t at = tile0 + j;
        if (!sy.wait_warp(&sh->scale_full[at % kScaleRing], at / kScaleRing & 1u)) return;
        scales = sh->scale[at % kScaleRing];
      }
      float s[kTileK];
      const int key0 = (p.t0 + j) * kTileK;
      const bool masked = key0 < all_min || key0 + kTileK > all_max;
      auto load = [&] {
#pragma unroll
        for (int c = 0; c < kTileK; c += 32) tm_ld32(ts + c, s + c);
        tm_ld_wait();
        if (flip) {
#pragma unroll
          for (int c = 0; c < kTileK; ++c) s[c] = -s[c];
        }
        if (masked) {  // a bit per key: one test and one select per score
#pragma unroll
          for (int c0 = 0; c0 < kTileK; c0 += 32) {
            const int a = kmin - key0 - c0, b = kmax - key0 - c0;
            const uint32_t below = a <= 0 ? 0u : a >= 32 ? ~0u : (1u << a) - 1u;
            const uint32_t seen = b <= 0 ? 0u : (b >= 32 ? ~0u : (1u << b) - 1u) & ~below;
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c0 + c] = seen & (1u << c) ? s[c0 + c] : -INFINITY;
          }
        }
      };
      auto highest = [&] {
        float m0 = -INFINITY, m1 = m0, m2 = m0, m3 = m0;
#pragma unroll
        for (int c = 0; c < kTileK; c += 8) {
          m0 = max3v(m0, s[c], s[c + 1]), m1 = max3v(m1, s[c + 2], s[c + 3]);
          m2 = max3v(m2, s[c + 4], s[c + 5]), m3 = max3v(m3, s[c + 6], s[c + 7]);
        }
        return fmaxf(max3v(m0, m1, m2), m3);
      };
      // A row is off where a score exceeds the reference by more than 2^kLazy, or all fall short of
      // it by more than 2^kShort with nothing summed yet (`high` in powers of two above it).
      auto is_off = [&](float high) {
        return high > (C8 ? kLazyBytes : kLazy) || (l == 0.f && high < -kShort<TP> && high != -INFINITY);
      };
      // Makes this tile's maximum the reference of the rows that are off, and moves what was summed
      // with the old one. (C8: the first pass has found which rows are off; theirs are exponents by
      // then, base-2 logarithms like the reference.)
      bool off_row = false;
      auto move = [&] {
        const float mx = highest(), by = C8 ? 1.f : sc;
        const bool off = C8 ? off_row : is_off((mx - ref) * by);
        const float f = off && l > 0.f ? ex2((ref - mx) * by) : 1.f;  // (nothing summed: O is 0)
        if (off) ref = mx;
        l *= f;
        if (j == 0) return;
        // (P V of the tiles before has finished: S of this one came after it)
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {  // 16 at a time: the scores stay in registers
          float o[16];
          tm_ld16(to + c, o);
          tm_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= f;
          tm_st16(to + c, reinterpret_cast<uint32_t*>(o));
        }
      };
      // The reference starts at 0, where normalised queries and keys leave it, and the maximum is
      // rarely news after the first tile. So it is taken beside the exponentials with the
      // reference so far, and looked at before any of P is announced; where a row of the warp is
      // off, the tile is begun again.
      // (C8: at the lowest scale of V among the tile's keys, a term of their exponents)
      if (j == 0) ref = C8 ? scales[0].w : 0.f;
      bool moved = false;
      // The instructions of other pairs are laid between the two exponentials of a pair, which keep
      // the special-function unit busy for 16 cycles: the products of pairs to come (all of them,
      // and so the maximum, within the first half), rounding and summing of one kAhead before. In
      // program order (volatile): left to itself the compiler does all of a kind in a row, and the
      // unit waits. P goes out in two halves: the MMAs of the first run beside the exponentials of
      // the second.
      constexpr int kPairs = kTileK / 2, kAhead = 4;
      // C8: a factor of scores is not 0, so that a masked -inf stays -inf
      constexpr float kLeast = 1e-35f;
      uint64_t l0, l1;
      for (;;) {
        load();
        if (C8 && moved) {
          // Exponents first, each rounded by itself: the largest is then no higher than the reference
          // that it gives, however large it is. (Rows that are not off stay as in the first pass:
          // no row's result goes by the others of its warp.)
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const float4 u = scales[i / (kGroup / 2)];
            const float a = off_row ? fmaxf(u.x * sc, kLeast) : 1.f, b = off_row ? u.y : 0.f;
            unpair(fma2v(pair(s[2 * i], s[2 * i + 1]), pair(a, a), pair(b, b)), s[2 * i], s[2 * i + 1]);
          }
        }
        if (moved) move();
        const float off = -ref * sc;
        uint64_t sc2 = pair(sc, sc), off2 = pair(off, off), inv2 = 0;
        float4 ahead;  // C8: scales of the next group of keys
        if constexpr (C8) ahead = scales[0];
        uint32_t pk[kPairs / 2];
        float m0 = -INFINITY, m1 = -INFINITY;
        l0 = l1 = 0;
        constexpr int kGroupPairs = kGroup / 2;
        auto scaled = [&](int i, float& m) {
          if constexpr (C8) {
            if (i % kGroupPairs == 0) {
              const float a = off_row ? 1.f : fmaxf(ahead.x * sc, kLeast);
              const float b = off_row ? -ref : ahead.y - ref;
              sc2 = pair(a, a), off2 = pair(b, b);
            } else if (i % kGroupPairs == 1 && i + kGroupPairs < kPairs) {
              ahead = scales[i / kGroupPairs + 1];
            }
          }
          unpair(fma2v(pair(s[2 * i], s[2 * i + 1]), sc2, off2), s[2 * i], s[2 * i + 1]);
          // (two pairs behind: a warp issues in order, and would wait for the product)
          if (i >= 2) m = max3v(m, s[2 * i - 4], s[2 * i - 3]);
        };
        auto done = [&](int d) {
          pk[d % (kPairs / 2)] = pack2v<TP>(s[2 * d], s[2 * d + 1]);
          uint64_t& sum = d & 1 ? l1 : l0;
          if constexpr (C8) {
            if (d % kGroupPairs == 0) {
              const float inv = scales[d / kGroupPairs].z;
              inv2 = pair(inv, inv);
            }
            sum = fma2v(pair(s[2 * d], s[2 * d + 1]), inv2, sum);
          } else {
            sum = add2v(sum, pair(s[2 * d], s[2 * d + 1]));
          }
        };
        auto announce = [&](int half) {
          tm_st16(ts + half * 32, pk);
          tm_st16(ts + half * 32 + 16, pk + 16);
          tm_st_wait();
          tc_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->p_ready[x][half]);
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) scaled(i, i & 1 ? m1 : m0);
#pragma unroll
        for (int i = 0; i < kPairs / 2; ++i) {
          s[2 * i] = ex2v(s[2 * i]);
          if (kAhead + 2 * i < kPairs) scaled(kAhead + 2 * i, m0);
          s[2 * i + 1] = ex2v(s[2 * i + 1]);
          if (kAhead + 2 * i + 1 < kPairs) scaled(kAhead + 2 * i + 1, m1);
          if (kAhead + 2 * i == kPairs) {  // the last two pairs, before they are exponentials
            m0 = max3v(m0, s[kTileK - 4], s[kTileK - 3]);
            m1 = max3v(m1, s[kTileK - 2], s[kTileK - 1]);
          }
          if (i >= kAhead) done(i - kAhead);
        }
        if (!moved && __any_sync(0xffffffffu, is_off(fmaxf(m0, m1)))) {
          if constexpr (C8) off_row = is_off(fmaxf(m0, m1));
          moved = true;
          continue;
        }
#pragma unroll
        for (int i = kPairs / 2; i < kPairs + kAhead; ++i) {
          if (i < kPairs) s[2 * i] = ex2v(s[2 * i]);
          done(i - kAhead);
          if (i < kPairs) s[2 * i + 1] = ex2v(s[2 * i + 1]);
          if (i - kAhead == kPairs / 2 - 1) announce(0);
        }
        announce(1);
        break;
      }
      float la, lb;
      unpair(add2v(l0, l1), la, lb);
      l += la + lb;
    }
    // output of the row tile
    const float ref_log2 = C8 ? ref : ref * sc;
    if (rt.n > 0) {
      if (!sy.wait_warp(&sh->o_full[x], o_par)) return;
      o_par ^= 1u;
      tc_after();
    }
    if (p.slot >= 0) {
      float* part = P.partial + (int64_t)p.slot * kSlot + (int64_t)x * kTileM * (DP + 2);
      if (live) {
        // (a row that summed nothing here has no reference: the one it started from, 0, may lie so
        // far above those of the other parts that the join would weigh them as nothing)
        part[kTileM * DP + row] = l == 0.f ? -INFINITY : ref_log2;
        part[kTileM * DP + kTileM + row] = l;
      }
#pragma unroll 1
      for (int c = 0; c < DP && rt.n > 0; c += 16) {
        float o[16];
        tm_ld16(to + c, o);
        tm_ld_wait();
        if (live) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(part + ((c + i) / 4 * kTileM + row) * 4) =
                make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
    } else {
      // Through the tile's Q buffer (its last S is done), each warp its own rows, so that the
      // stores are whole lines: a lane's row would take a line per 32 bytes. 16-byte units are
      // placed at unit ^ (row % 8), which spreads both the columns and the rows over the banks.
      constexpr int kUnits = DP / 8;  // 16-byte units of a row
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      uint8_t* stage = sh->q[q_mine] + (row & ~31) * DP * 2;
      // (short loops: code that runs once per item is fetched as it runs)
      if (rt.n > 0) {
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {
          float o[16];
          tm_ld16(to + c, o);
          tm_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack2<T>(o[i + 2 * k] * inv, o[i + 2 * k + 1] * inv);
            // (inv is 0 for a row without keys, whose O is 0 too)
            *reinterpret_cast<uint4*>(stage + lane * DP * 2 + (((c + i) / 8 ^ (lane & 7)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
      }
      constexpr int kRowsAt = 32 / kUnits;  // rows per store of the warp
      const int unit = lane % kUnits;
      uint16_t* out0 = P.out + ((int64_t)(p.q_tok + rt.tok0) * P.Hq + p.head * P.G) * P.D + unit * 8;
      const int to_row = live ? tok * P.Hq + g : -1;
#pragma unroll 2
      for (int r = lane / kUnits; r < 32; r += kRowsAt) {
        const int dst = __shfl_sync(0xffffffffu, to_row, r);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (rt.n > 0) v = *reinterpret_cast<const uint4*>(stage + r * DP * 2 + ((unit ^ (r & 7)) << 4));
        if (dst >= 0 && unit * 8 < P.D) *reinterpret_cast<uint4*>(out0 + (int64_t)dst * P.D) = v;
      }
      if (live && P.lse)
        P.lse[(int64_t)(p.q_tok + rt.tok0 + tok) * P.Hq + p.head * P.G + g] =
            l == 0.f ? -INFINITY : (ref_log2 + log2f(l)) * 0.69314718055994531f;
    }
    if (rt.n > 0) {  // the Q buffer goes back to the copies
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->q_empty[q_mine]);
    }
    tc_before();  // O has been read before the next item's P is announced
  }
}

template <typename T, int DP, bool C8>
__global__ void __launch_bounds__(kThreadsC, 1)
    k_attn_chunk(const __grid_constant__ AttnMaps M, const __grid_constant__ AttnParams P,
                 const __grid_constant__ Plan plan, int tok1) {
  extern __shared__ uint8_t smem_raw[];
  ChunkSmem<DP, C8>* sh = reinterpret_cast<ChunkSmem<DP, C8>*>(
      smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
  const int warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < ChunkSmem<DP, C8>::kStages; ++i) {
      mbar_init(&sh->full[i], C8 ? kTurners : 1);
      mbar_init(&sh->empty[i], 1);
      mbar_init(&sh->land[i], 1);
    }
    for (int i = 0; i < kQBufs; ++i) {
      mbar_init(&sh->q_full[i], 1);
      mbar_init(&sh->q_empty[i], 4);  // the tile's softmax warps
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sh->s_full[x], 1);
      mbar_init(&sh->p_ready[x][0], 4);
      mbar_init(&sh->p_ready[x][1], 4);
      mbar_init(&sh->o_full[x], 1);
    }
    for (int i = 0; i < kPieceRing; ++i) {
      mbar_init(&sh->piece_full[i], 1);
      mbar_init(&sh->piece_empty[i], kPieceReaders + (C8 ? kTurners - 1 : 0));
    }
    for (int i = 0; C8 && i < ChunkSmem<DP, C8>::kScaleRing; ++i) mbar_init(&sh->scale_full[i], 1);
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_mbar_init();
    prefetch_map(&M.k);
    prefetch_map(&M.v);
    prefetch_map(&M.q);
  }
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&sh->tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  pdl_wait();
  if (warp < kWarpMma) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    chunk_softmax<T, DP, C8>(P, tok1, warp >> 2, sh);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kWarpMma) {
      chunk_mma<T, DP, C8>(P, tok1, sh);
    } else if constexpr (C8) {
      if (warp == kWarpLoad)
        chunk_load8<DP>(P, M, plan, tok1, sh);
      else
        chunk_turn<T, DP>(P, tok1, warp - kWarpFix, sh);
    } else {
      if (warp == kWarpLoad)
        chunk_load<DP>(P, M, plan, tok1, sh);
      else if (warp == kWarpFix)
        chunk_fix<DP>(P, tok1, sh);
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh->tmem));
}

// Joins the parts of split items. A part's O is [D / 4][row][4]: a warp takes 32 rows (a lane
// each) and 16 columns, so that it reads whole lines and writes whole sectors.
template <typename T, int DP>
__global__ void __launch_bounds__(256) k_attn_join(const __grid_constant__ AttnParams P,
                                                   const __grid_constant__ Plan plan, int tok1) {
  pdl_launch_dependents();
  pdl_wait();
  const int joins = __ldcg(plan.head + kPlanJoins);
  const int lane = threadIdx.x & 31;
  constexpr int64_t kSlot = 2 * kTileM * (DP + 2);
  constexpr int kCols = 16, kUnits = 2 * (kTileM / 32) * (DP / kCols);  // per join
  const bool sectors = P.D % 16 == 0 && (reinterpret_cast<uintptr_t>(P.out) & 31) == 0;
  const int64_t warps = (int64_t)gridDim.x * 8;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < (int64_t)joins * kUnits;
       i += warps) {
    const Join* jn = plan.joins + i / kUnits;
    const int4 j0 = __ldcg(reinterpret_cast<const int4*>(jn));
    const int parts = __ldcg(&jn->parts);
    const int q_tok = j0.x, n_tok = j0.y, head = j0.z, slot = j0.w;
    const int u = (int)(i % kUnits), c0 = u % (DP / kCols) * kCols, r = u / (DP / kCols) * 32 + lane;
    const int x = r / kTileM, row = r % kTileM, tok = row / P.G;
    const bool live = tok < tok1 && x * tok1 + tok < n_tok;
    if (!__any_sync(0xffffffffu, live) || c0 >= P.D) continue;
    const float* base = P.partial + slot * kSlot + (int64_t)x * kTileM * (DP + 2);
    float m = -INFINITY, l = 0.f, o[kCols] = {};
    constexpr int kTogether = 4;  // parts whose loads are in flight together
    for (int k0 = 0; k0 < parts; k0 += kTogether) {
      float mk[kTogether], lk[kTogether];
      float4 v[kTogether][kCols / 4];
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const float* b = base + (k0 + k) * kSlot;
        const bool in = live && k0 + k < parts;
        mk[k] = in ? __ldcg(b + kTileM * DP + row) : -INFINITY;
        lk[k] = in ? __ldcg(b + kTileM * DP + kTileM + row) : 0.f;
#pragma unroll
        for (int q = 0; q < kCols / 4; ++q)
          if (in) v[k][q] = __ldcg(reinterpret_cast<const float4*>(b) + (c0 / 4 + q) * kTileM + row);
      }
      float mx = m;
#pragma unroll
      for (int k = 0; k < kTogether; ++k) mx = fmaxf(mx, mk[k]);
      if (mx == -INFINITY) continue;
      const float keep = ex2(m - mx);  // of the parts before
      m = mx;
      l *= keep;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[c] *= keep;
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        if (mk[k] == -INFINITY) continue;  // a part that summed nothing of this row left no O
        const float f = ex2(mk[k] - mx);
        l += f * lk[k];
#pragma unroll
        for (int q = 0; q < kCols / 4; ++q) {
          o[4 * q] += f * v[k][q].x, o[4 * q + 1] += f * v[k][q].y;
          o[4 * q + 2] += f * v[k][q].z, o[4 * q + 3] += f * v[k][q].w;
        }
      }
    }
    if (!live) continue;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const int64_t out_row = (int64_t)(q_tok + x * tok1 + tok) * P.Hq + head * P.G + row % P.G;
    uint16_t* op = P.out + out_row * P.D + c0;
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = pack2<T>(o[2 * k] * inv, o[2 * k + 1] * inv);
    if (sectors) {
      st_sector(op, w);
    } else {
      *reinterpret_cast<uint4*>(op) = make_uint4(w[0], w[1], w[2], w[3]);
      if (c0 + 8 < P.D) *reinterpret_cast<uint4*>(op + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    }
    if (c0 == 0 && P.lse)
      P.lse[out_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
  }
}

int64_t chunk_groups(int64_t total_q, int batch, int G) {
  return total_q / (2 * (kTileM / G)) + batch;
}

template <typename T, int DP, bool C8>
int run_chunk(const AttnMaps& M, const AttnParams& P, const Plan& plan, int tok1, int64_t groups,
              cudaStream_t stream) {
  constexpr size_t smem = sizeof(ChunkSmem<DP, C8>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory");
  // the warpgroups' shares must add up to what a block is launched with
  static const bool fits = [] {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, k_attn_chunk<T, DP, C8>) == cudaSuccess &&
           at.numRegs >= kRegsLaunch;
  }();
  if (!fits) return FTB_ERR_NOT_BUILT;
  static std::atomic<uint64_t> done{0}, plan_done{0};
  cudaError_t err = allow_smem(k_attn_chunk<T, DP, C8>, smem, done);
  if (err == cudaSuccess) err = allow_smem(k_attn_plan, kPlanSmem, plan_done);
  if (err != cudaSuccess) return cuda_status(err);
  const int sms = sm_count();
  // the plan's arrays by sequence and by group, the latter in the workspace where they are too many
  size_t plan_smem = ((size_t)P.batch + 1) * sizeof(int) + (size_t)groups * sizeof(PlanGroup);
  if (plan_smem > (size_t)kPlanSmem) plan_smem = kPlanSmem;
  err = launch_pdl(k_attn_plan, dim3(1), dim3(kPlanThreads), plan_smem, stream, P, plan, 2 * tok1,
                   sms);
  if (err != cudaSuccess) return cuda_status(err);
  err = launch_pdl(k_attn_chunk<T, DP, C8>, dim3((unsigned)sms), dim3(kThreadsC), smem, stream, M, P,
                   plan, tok1);
  if (err != cudaSuccess) return cuda_status(err);
  return cuda_status(launch_pdl(k_attn_join<T, DP>, dim3((unsigned)sms * 8), dim3(256), 0, stream,
                                P, plan, tok1));
}

template <bool C8>
int pick_chunk(const ftb_attn_args& a, const AttnMaps& M, const AttnParams& P, const Plan& plan,
               int tok1, int64_t groups, cudaStream_t stream) {
  if (a.type == FTB_TYPE_BF16)
    return a.D <= 64 ? run_chunk<__nv_bfloat16, 64, C8>(M, P, plan, tok1, groups, stream)
                     : run_chunk<__nv_bfloat16, 128, C8>(M, P, plan, tok1, groups, stream);
  return a.D <= 64 ? run_chunk<__half, 64, C8>(M, P, plan, tok1, groups, stream)
                   : run_chunk<__half, 128, C8>(M, P, plan, tok1, groups, stream);
}

}  // namespace

size_t attn_chunk_workspace_bytes(int64_t total_q, int batch, int Hkv, int G, int D) {
  size_t bytes;
  const int64_t groups = chunk_groups(total_q, batch, G);
  carve_plan(nullptr, groups, Hkv, &bytes);
  const int dp = D <= 64 ? 64 : 128;
  return bytes + (size_t)plan_parts() * 2 * kTileM * (dp + 2) * sizeof(float);
}

bool attn_chunk_fits(const ftb_attn_args& a) {
  return a.batch <= kMaxBatch &&
         chunk_groups(a.total_q, a.batch, a.Hq / a.Hkv) * a.Hkv <= 0x3fffffff;
}

int launch_attn_chunk(const ftb_attn_args& a, AttnParams P, bool fp8, cudaStream_t stream) {
  if (!attn_chunk_fits(a)) return FTB_ERR_SHAPE;
  const int tok1 = kTileM / P.G;
  const int64_t groups = chunk_groups(a.total_q, a.batch, P.G);
  AttnMaps M;
  const uint32_t r = a.page < kTileK ? a.page : kTileK;
  int st = fp8 ? attn_cache_map8(&M.k, a.k_cache, a, a.k_strides, r)
               : attn_cache_map(&M.k, a.k_cache, a, a.k_strides, r, 1);
  if (!st)
    st = fp8 ? attn_cache_map8(&M.v, a.v_cache, a, a.v_strides, r)
             : attn_cache_map(&M.v, a.v_cache, a, a.v_strides, r, 1);
  if (!st) st = attn_q_map(&M.q, a, (uint32_t)P.G, (uint32_t)tok1);
  if (st) return st;
  size_t bytes;
  const Plan plan = carve_plan(reinterpret_cast<char*>(P.partial), groups, a.Hkv, &bytes);
  P.partial = reinterpret_cast<float*>(reinterpret_cast<char*>(P.partial) + bytes);
  return fp8 ? pick_chunk<true>(a, M, P, plan, tok1, groups, stream)
             : pick_chunk<false>(a, M, P, plan, tok1, groups, stream);
}

}  // namespace ftb
