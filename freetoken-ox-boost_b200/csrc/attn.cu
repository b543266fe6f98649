// attn.cu - entry point of the paged attention (ftb_attention): argument checks, tensor maps,
// and the choice between the kernels.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "attn.cuh"

namespace ftb {

PFN_cuTensorMapEncodeTiled encode_fn();  // moe_decode_tma.cu

namespace {
CUtensorMapDataType attn_dtype(int type) {
  return type == FTB_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Which kernel: the streaming one for up to 16 query rows per kv head (one mma.sync row tile, bound
// by DRAM), and for small work, where the tensor-core kernel's plan and join cost more than its
// rate gives: at most 1.1 GFLOP by the bound that the host knows (every token against the whole
// table, or its window). On one B200, us (streaming / tensor cores), 32 heads over 8 of 128: prompts
// of 64 tokens 7.6 / 18.0, 256 (1.1 GFLOP) 19.3 / 20.2, 300 35.2 / 21.6, 384 37.7 / 22.8, 512 53.7 /
// 22.5; 16 tokens at 2048 keys (0.5 GFLOP) 17.4 / 20.6, 64 32.0 / 24.3. Its row tiles are a grid's
// rows, so that many at most.
constexpr int kStreamRows = 16;
constexpr double kStreamFlops = 1.1e9;
// Of the two, a batch beyond the tensor-core kernel's plan goes to the streaming one.
bool streams(const ftb_attn_args& a, int64_t keys) {
  const int64_t rows = (int64_t)a.max_q * (a.Hq / a.Hkv);
  return rows <= kStreamRows ||
         (rows <= (int64_t)kStreamRows * 65535 &&
          (4.0 * a.D * a.Hq * (double)a.total_q * (double)keys <= kStreamFlops ||
           !attn_chunk_fits(a)));
}
int64_t keys_bound(const ftb_attn_args& a) {
  const int64_t all = (int64_t)a.table_width * a.page;
  return a.window > 0 ? std::min<int64_t>(all, a.window) : all;
}
}  // namespace

int attn_cache_map(CUtensorMap* m, const void* base, const ftb_attn_args& a,
                   const int64_t (&strides)[3], uint32_t box_rows, uint32_t halves) {
  PFN_cuTensorMapEncodeTiled fn = encode_fn();
  if (!fn) return FTB_ERR_CUDA;
  const bool split = halves > 1;  // the halves of a head as a dimension of their own
  const cuuint64_t dims[5] = {split ? 64u : (cuuint64_t)a.D, (cuuint64_t)a.page,
                              (cuuint64_t)a.Hkv, (cuuint64_t)a.num_pages, halves};
  const cuuint64_t st[4] = {(cuuint64_t)strides[1] * 2, (cuuint64_t)strides[2] * 2,
                            (cuuint64_t)strides[0] * 2, 128};
  const cuuint32_t box[5] = {64, box_rows, 1, 1, halves};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(m, attn_dtype(a.type), 5, const_cast<void*>(base), dims, st, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FTB_OK : FTB_ERR_CUDA;
}

int attn_q_map(CUtensorMap* m, const ftb_attn_args& a, uint32_t group, uint32_t tokens) {
  PFN_cuTensorMapEncodeTiled fn = encode_fn();
  if (!fn) return FTB_ERR_CUDA;
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, group, (cuuint64_t)a.Hkv, (cuuint64_t)a.total_q};
  const cuuint64_t st[3] = {(cuuint64_t)a.q_strides[1] * 2, (cuuint64_t)a.q_strides[1] * 2 * group,
                            (cuuint64_t)a.q_strides[0] * 2};
  const cuuint32_t box[4] = {64, group, 1, tokens};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, attn_dtype(a.type), 4, const_cast<uint16_t*>(a.q), dims, st, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FTB_OK : FTB_ERR_CUDA;
}

}  // namespace ftb

using namespace ftb;

extern "C" {

size_t ftb_attention_workspace_bytes(int64_t total_q, int batch, int max_q, int Hq, int Hkv, int D) {
  if (total_q < 0 || batch < 0 || max_q < 0 || Hkv < 1 || Hq < Hkv || D < 8) return 0;
  const int G = Hq / Hkv;
  if (G > 128) return 0;
  const int64_t rows = std::min<int64_t>(max_q, total_q) * G;
  const size_t stream = attn_stream_partial_bytes(rows, D);
  if (rows <= kStreamRows) return FTB_ATTN_ZERO_BYTES + stream;
  // (more rows: either kernel, by the lengths)
  return FTB_ATTN_ZERO_BYTES +
         std::max(stream, attn_chunk_workspace_bytes(total_q, batch, Hkv, G, D));
}

int ftb_attention(const ftb_attn_args* args, ftb_stream_t stream) {
  if (!args) return FTB_ERR_ARG;
  ftb_attn_args call = *args;
  // (a caller's bound may be its model's; no sequence has more than all rows)
  if (call.total_q >= 0) call.max_q = (int)std::min<int64_t>(call.max_q, call.total_q);
  // (nor does a window that reaches every key hide any: j > p - window for all j and p < keys. As no
  // window it also stays out of the kernels' 32-bit differences)
  if (call.window >= (int64_t)call.table_width * call.page) call.window = std::min(call.window, 0);
  const ftb_attn_args* a = &call;
  if (a->type != FTB_TYPE_BF16 && a->type != FTB_TYPE_F16) return FTB_ERR_ARG;
  if (a->total_q < 0 || a->total_q > 0x7fffffff || a->batch < 0 || a->max_q < 0 || a->Hkv < 1 ||
      a->Hq < 1 || a->Hq % a->Hkv || a->Hq / a->Hkv > 128 || a->D < 8 || a->D > 128 || a->D % 8 ||
      a->page < 8 || (a->page & (a->page - 1)) || a->num_pages < 1 ||
      a->num_pages > 0x7fffffff - 1 || a->table_width < 0 || a->window < 0 ||
      (int64_t)a->table_width * a->page > 0x7fffff00)
    return FTB_ERR_SHAPE;
  if (a->total_q == 0 || a->batch == 0 || a->max_q == 0) return FTB_OK;
  if (!a->q || !a->k_cache || !a->v_cache || (!a->block_table && a->table_width > 0) || !a->kv_len ||
      !a->out)  // (a table without a column has no address: no sequence has a key)
    return FTB_ERR_ARG;
  if (!a->cu_q && a->total_q != a->batch) return FTB_ERR_SHAPE;
  if (!std::isfinite(a->scale)) return FTB_ERR_ARG;
  if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->out))
    return FTB_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if (a->k_strides[i] % 8 || a->v_strides[i] % 8 || a->k_strides[i] < 0 || a->v_strides[i] < 0)
      return FTB_ERR_ALIGN;
  for (int i = 0; i < 2; ++i)
    if (a->q_strides[i] % 8 || a->q_strides[i] < 0) return FTB_ERR_ALIGN;
  if (!a->workspace ||
      a->workspace_bytes < ftb_attention_workspace_bytes(a->total_q, a->batch, a->max_q, a->Hq,
                                                         a->Hkv, a->D))
    return FTB_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 255u) return FTB_ERR_ALIGN;
  AttnParams P{};
  P.q = a->q, P.out = a->out, P.lse = a->lse;
  P.block_table = a->block_table, P.kv_len = a->kv_len, P.cu_q = a->cu_q;
  char* ws = static_cast<char*>(a->workspace);
  P.status = reinterpret_cast<uint32_t*>(ws);
  P.counters = reinterpret_cast<int32_t*>(ws + 16);
  P.partial = reinterpret_cast<float*>(ws + FTB_ATTN_ZERO_BYTES);
  P.q_st = a->q_strides[0], P.q_sh = a->q_strides[1];
  P.total_q = a->total_q, P.table_stride = a->table_stride, P.num_pages = a->num_pages;
  P.batch = a->batch, P.max_q = a->max_q, P.table_width = a->table_width;
  int lg = 0;
  while ((1 << lg) < a->page) ++lg;
  P.page_log2 = lg;
  P.Hq = a->Hq, P.Hkv = a->Hkv, P.G = a->Hq / a->Hkv, P.D = a->D;
  P.causal = a->causal != 0, P.window = a->window;
  P.keys_max = a->table_width * a->page;
  P.scale_log2 = a->scale * 1.44269504088896341f;
  return streams(*a, keys_bound(*a))
             ? launch_attn_stream(*a, P, (cudaStream_t)stream)
             : launch_attn_chunk(*a, P, (cudaStream_t)stream);
}

}  // extern "C"
