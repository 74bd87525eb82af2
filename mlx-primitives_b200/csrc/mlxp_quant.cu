// mlxp_quant.cu — host side of attention over an 8-bit paged cache: argument checks, the choice
// of a kernel and the launches.

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/mlxp_attn.h"
#include "host_common.h"
#include "quant_attn_rows.cuh"

namespace mlxp {

MLXP_INTERNAL int qa_rows_launch(int64_t dtype, int64_t D, bool int8, const QaParams& p, unsigned grid,
                                 cudaStream_t s);  // mlxp_quant_rows.cu

namespace {

// Query rows a pool head from which the many-row kernel (tcgen05, 256 rows a unit) is taken.  It
// reads and converts the codes once for all of a unit's rows, the other once for every 16.
// Measured at 8 heads of 128, e4m3, four contexts of 8 K / 64 of 2 K / one of 1000 tokens:
//   48 rows   65 us against  82 / 290 against 220 / 19 against 21
//   64        65 against  93     / 281 to 294 against 276 / 19 against 21
//  128        72 against 148     / 290 to 300 against 503 / 21 against 26
//  256        90 against 254     / 315 to 325 against 956 / 27 against 37
constexpr int kRowsFrom = 64;

struct QaPlan {
  bool many;         // the many-row kernel
  int nt;            // 8-row query tiles a warp
  int per_sm;        // CTAs an SM holds
  long long grid;
  size_t o_bytes, ml_bytes, info_bytes;
  size_t bytes() const { return o_bytes + ml_bytes + info_bytes; }
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// CTAs an SM holds (the launch bounds below are the same numbers).  Three rather than the four
// that 128 registers a thread allow: four contexts of 128 K tokens 180 us against 190, 48 ragged
// ones at head_dim 64 35 against 40, at two 239 and 43.  With two row tiles at head_dim 128 (9 to 63
// rows a pool head) the 168 registers of three spill (up to 148 bytes a thread stored, 272 loaded),
// those of two do not; 32 heads over 8 of 128, e4m3, three against two: four contexts of 128 K tokens
// 259 us against 263 at 16 rows and 657 against 720 at 48, eight of 4 K 52 against 43 and 80 against
// 76.
template <int D, int NT, bool SPLIT>
constexpr int qa_min_ctas() {
  return SPLIT && D == 128 ? 2 : 3;
}

int qa_ctas(int64_t dtype, int64_t D, int nt) {
  const bool split = dtype == MLXP_DTYPE_FP32;
  if (D == 128) return split ? qa_min_ctas<128, 1, true>()
                             : nt == 2 ? qa_min_ctas<128, 2, false>() : qa_min_ctas<128, 1, false>();
  return split ? qa_min_ctas<64, 1, true>()
               : nt == 2 ? qa_min_ctas<64, 2, false>() : qa_min_ctas<64, 1, false>();
}

int qa_check(const mlxp_quant_paged_attn_args* a) {
  if (!a || a->size != sizeof(*a)) return fail(MLXP_ERR_INVALID, "argument struct of another size");
  if (a->dtype < 0 || a->dtype > 2) return fail(MLXP_ERR_INVALID, "unknown dtype %lld", (long long)a->dtype);
  if (a->cache_dtype != MLXP_DTYPE_E4M3 && a->cache_dtype != MLXP_DTYPE_INT8)
    return fail(MLXP_ERR_INVALID, "the cache must be e4m3 or int8, got dtype %lld", (long long)a->cache_dtype);
  if (a->B < 0 || a->Sq < 0 || a->H < 1 || a->kv_heads < 1 || a->num_blocks < 0 || a->block_size < 1 ||
      a->max_blocks < 0)
    return fail(MLXP_ERR_INVALID, "invalid paged shape B=%lld H=%lld Sq=%lld kv_heads=%lld num_blocks=%lld "
                "block_size=%lld max_blocks=%lld", (long long)a->B, (long long)a->H, (long long)a->Sq,
                (long long)a->kv_heads, (long long)a->num_blocks, (long long)a->block_size,
                (long long)a->max_blocks);
  if (a->H % a->kv_heads)
    return fail(MLXP_ERR_INVALID, "num_heads (%lld) must be divisible by the pool's heads (%lld)",
                (long long)a->H, (long long)a->kv_heads);
  if (a->D != 32 && a->D != 64 && a->D != 128)
    return fail(MLXP_ERR_UNSUPPORTED, "paged attention supports head_dim 32, 64 and 128, got %lld",
                (long long)a->D);
  if (a->num_blocks > INT32_MAX || a->block_size > INT32_MAX || a->max_blocks > INT32_MAX ||
      a->max_blocks * a->block_size > kMaxCacheIndex || a->B > INT32_MAX || a->Sq > INT32_MAX ||
      a->H > INT32_MAX || a->B * a->Sq > INT32_MAX || a->B * a->Sq * a->H > kMaxCacheIndex)
    return fail(MLXP_ERR_INVALID, "paged shape too large");
  if (a->window < -1) return fail(MLXP_ERR_INVALID, "window must be >= 0, or -1 for none");
  return MLXP_OK;
}

// What qa_check lets through with B, Sq > 0.
QaPlan qa_plan(const mlxp_quant_paged_attn_args* a, int sms, QaParams& p) {
  QaPlan n{};
  p.B = (int)a->B;
  p.H = (int)a->H;
  p.Hk = (int)a->kv_heads;
  p.G = (int)(a->H / a->kv_heads);
  p.Sq = (int)a->Sq;
  p.R = (int)(p.G * a->Sq);
  n.many = p.R >= kRowsFrom && a->dtype != MLXP_DTYPE_FP32 && a->D >= 64 && a->block_size % kQaTile == 0 &&
           !a->alibi_slopes;
  const long long cap = a->max_blocks * a->block_size;
  if (n.many) {
    p.rows = std::min(p.R, kQrRows);
    p.RT = (p.R + kQrRows - 1) / kQrRows;
    p.HP = 1;
    p.HG = p.Hk;
    n.per_sm = 1;
  } else {
    // 16 rows a warp where there are more than 8 (the codes are then converted once for both
    // halves); the split operands of fp32 leave registers for 8
    n.nt = p.R > 8 && a->dtype != MLXP_DTYPE_FP32 ? 2 : 1;
    n.per_sm = qa_ctas(a->dtype, a->D, n.nt);
    p.rows = std::min(p.R, 8 * n.nt);
    p.RT = (p.R + 8 * n.nt - 1) / (8 * n.nt);
    p.HP = p.Hk % 4 == 0 ? 4 : p.Hk % 2 == 0 ? 2 : 1;
    p.HG = p.Hk / p.HP;
  }
  const int chunk = n.many ? kQrKeys : kQaChunk;
  const long long chunks = std::max<long long>(1, (cap + chunk - 1) / chunk + 1);
  n.grid = std::min<long long>((long long)sms * n.per_sm, (long long)p.B * p.RT * p.HG * chunks);
  const size_t rows = (size_t)n.grid * 2 * p.HP * p.rows;
  n.o_bytes = up256(rows * a->D * 4);
  n.ml_bytes = up256(rows * 2 * 4);
  n.info_bytes = up256((size_t)n.grid * sizeof(QaPartInfo));
  return n;
}

// Tensor maps of the pools, {D, heads, block_size, blocks} with boxes of one head's 16 rows.
struct QaMaps {
  CUtensorMap k, v;
  bool use;  // a tile of 16 keys lies in one block, and the pools suit TMA
};

int qa_maps(const mlxp_quant_paged_attn_args* a, QaMaps& m) {
  m.use = false;
  if (a->block_size % kQaTile || a->num_blocks < 1) return MLXP_OK;
  int64_t sb = a->pool_strides[0], st = a->pool_strides[1], sh = a->pool_strides[2];
  if (a->kv_heads == 1) sh = a->D;                 // strides that no coordinate uses
  if (a->num_blocks == 1) sb = st * a->block_size;
  for (const int64_t x : {sb, st, sh})
    if (x <= 0 || x % 16 || x >= (int64_t(1) << 40)) return MLXP_OK;
  PFN_cuTensorMapEncodeTiled_v12000 encode;
  if (int rc = tensor_map_encoder(&encode)) return rc;
  const cuuint64_t dims[4] = {(cuuint64_t)a->D, (cuuint64_t)a->kv_heads, (cuuint64_t)a->block_size,
                              (cuuint64_t)a->num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)sh, (cuuint64_t)st, (cuuint64_t)sb};
  const cuuint32_t box[4] = {(cuuint32_t)a->D, 1, (cuuint32_t)kQaTile, 1}, ones[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle swizzle = a->D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : a->D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  for (int i = 0; i < 2; ++i)
    if (encode(i ? &m.v : &m.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(i ? a->v_pool : a->k_pool),
               dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return MLXP_OK;
  m.use = true;
  return MLXP_OK;
}

template <typename T, int D>
int qa_merge(const QaParams& p, long long grid, cudaStream_t s) {
  if (grid == 1) return MLXP_OK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(grid - 1), (unsigned)std::min(p.HP * p.rows, 16));
  cfg.blockDim = dim3(32 * kQaMergeWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, quant_attn_merge_kernel<T, D>, p);
  return e == cudaSuccess ? MLXP_OK : cuda_fail(e, "quantized paged attention merge launch");
}

template <typename T, int D, int NT, bool INT8, bool BS16>
int qa_launch(const QaMaps& maps, const QaParams& p, const QaPlan& n, cudaStream_t s) {
  auto kernel = quant_attn_kernel<T, D, NT, INT8, BS16, qa_min_ctas<D, NT, sizeof(T) == 4>()>;
  constexpr int smem = qa_smem_bytes<D, NT, BS16>();
  static std::atomic<unsigned long long> attr_done{0};  // one bit per device
  int dev;
  if (int rc = current_device(dev)) return rc;
  cudaError_t e;
  if (!(attr_done.load() >> dev & 1ull)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(quantized paged attention)");
    attr_done.fetch_or(1ull << dev);
  }
  kernel<<<(unsigned)n.grid, 32 * kQaWarps, smem, s>>>(maps.k, maps.v, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "quantized paged attention launch");
  return qa_merge<T, D>(p, n.grid, s);
}

template <typename T, int D, int NT>
int qa_launch_n(const QaMaps& m, const QaParams& p, const QaPlan& n, bool int8, cudaStream_t s) {
  if (int8) return m.use ? qa_launch<T, D, NT, true, true>(m, p, n, s) : qa_launch<T, D, NT, true, false>(m, p, n, s);
  return m.use ? qa_launch<T, D, NT, false, true>(m, p, n, s) : qa_launch<T, D, NT, false, false>(m, p, n, s);
}

template <typename T, int D>
int qa_launch_d(const QaMaps& m, const QaParams& p, const QaPlan& n, bool int8, cudaStream_t s) {
  if (n.many) {
    if (int rc = qa_rows_launch(std::is_same<T, __nv_bfloat16>::value ? MLXP_DTYPE_BF16 : MLXP_DTYPE_FP16, D, int8,
                                p, (unsigned)n.grid, s))
      return rc;
    return qa_merge<T, D>(p, n.grid, s);
  }
  if constexpr (sizeof(T) == 2)
    if (n.nt == 2) return qa_launch_n<T, D, 2>(m, p, n, int8, s);
  return qa_launch_n<T, D, 1>(m, p, n, int8, s);
}

template <typename T>
int qa_launch_t(int64_t D, const QaMaps& m, const QaParams& p, const QaPlan& n, bool int8, cudaStream_t s) {
  if (D == 128) return qa_launch_d<T, 128>(m, p, n, int8, s);
  if (D == 64) return qa_launch_d<T, 64>(m, p, n, int8, s);
  return qa_launch_d<T, 32>(m, p, n, int8, s);
}

}  // namespace
}  // namespace mlxp

using namespace mlxp;

extern "C" {

size_t mlxp_quant_paged_attn_workspace_size(const mlxp_quant_paged_attn_args* a) {
  if (qa_check(a) != MLXP_OK || a->B == 0 || a->Sq == 0) return 0;
  int sms;
  if (device_info(nullptr, &sms) != MLXP_OK) return 0;
  QaParams p{};
  return qa_plan(a, sms, p).bytes();
}

int mlxp_quant_paged_attn(const mlxp_quant_paged_attn_args* a) {
  if (int rc = qa_check(a)) return rc;
  if (!(a->scale > 0) || !std::isfinite((float)a->scale))
    return fail(MLXP_ERR_INVALID, "scale must be positive and finite");
  if (a->B == 0 || a->Sq == 0) return MLXP_OK;
  if (!a->q || !a->o || !a->context_lens) return fail(MLXP_ERR_INVALID, "q, o and context_lens must be non-null");
  if (a->max_blocks > 0 &&
      (!a->block_tables || (a->num_blocks > 0 && (!a->k_pool || !a->v_pool || !a->k_scales || !a->v_scales))))
    return fail(MLXP_ERR_INVALID, "the pools, their scales and block_tables must be non-null");
  if (a->max_blocks > 0 && a->B > 1 && a->bt_stride < a->max_blocks)
    return fail(MLXP_ERR_INVALID, "block-table row stride (%lld) is below max_blocks (%lld)",
                (long long)a->bt_stride, (long long)a->max_blocks);
  const int es = a->dtype == MLXP_DTYPE_FP32 ? 4 : 2;
  for (const void* ptr : {a->q, (const void*)a->o, a->k_pool, a->v_pool})
    if (reinterpret_cast<uintptr_t>(ptr) % 16)
      return fail(MLXP_ERR_INVALID, "q, o and the pools must be 16-byte aligned");
  for (int d = 0; d < 3; ++d) {
    if ((a->q_strides[d] * es) % 16 || (a->o_strides[d] * es) % 16)
      return fail(MLXP_ERR_INVALID, "q and o rows must start on 16 bytes");
    if (a->pool_strides[d] % 16) return fail(MLXP_ERR_INVALID, "pool strides must be multiples of 16");
  }
  int sms, *status;
  if (int rc = device_info(&status, &sms)) return rc;
  QaMaps maps{};
  if (int rc = qa_maps(a, maps)) return rc;
  QaParams p{};
  p.status = status;
  p.timeout_ns = wait_timeout_ns();
  const QaPlan n = qa_plan(a, sms, p);
  if (!a->workspace || a->ws_bytes < n.bytes())
    return fail(MLXP_ERR_WORKSPACE, "quantized paged attention needs %zu bytes of workspace, got %llu",
                n.bytes(), (unsigned long long)a->ws_bytes);
  if (reinterpret_cast<uintptr_t>(a->workspace) % 256)
    return fail(MLXP_ERR_INVALID, "workspace must be 256-byte aligned");
  char* w = static_cast<char*>(a->workspace);
  p.o_part = reinterpret_cast<float*>(w);
  p.ml_part = reinterpret_cast<float*>(w + n.o_bytes);
  p.info = reinterpret_cast<QaPartInfo*>(w + n.o_bytes + n.ml_bytes);
  p.q = a->q;
  p.o = a->o;
  p.k_pool = static_cast<const unsigned char*>(a->k_pool);
  p.v_pool = static_cast<const unsigned char*>(a->v_pool);
  p.k_scales = a->k_scales;
  p.v_scales = a->v_scales;
  p.block_tables = a->block_tables;
  p.context_lens = a->context_lens;
  p.query_lens = a->query_lens;
  p.alibi = a->alibi_slopes;
  p.q_sb = a->q_strides[0];
  p.q_sh = a->q_strides[1];
  p.q_ss = a->q_strides[2];
  p.o_sb = a->o_strides[0];
  p.o_sh = a->o_strides[1];
  p.o_ss = a->o_strides[2];
  p.p_sb = a->pool_strides[0];
  p.p_st = a->pool_strides[1];
  p.p_sh = a->pool_strides[2];
  p.sc_sb = a->scale_strides[0];
  p.sc_sh = a->scale_strides[1];
  p.bt_stride = a->bt_stride;
  p.num_blocks = (int)a->num_blocks;
  p.block_size = (int)a->block_size;
  p.max_blocks = (int)a->max_blocks;
  p.p_scale = n.many ? 1.f : kQaPScale;
  p.causal = a->causal ? 1 : 0;
  p.bs_pow2 = (p.block_size & (p.block_size - 1)) == 0;
  p.window = std::min<long long>(a->window, 1LL << 40);  // positions are below 2^32: room to add
  p.scale_log2 = (float)(a->scale * 1.4426950408889634);
  const bool int8 = a->cache_dtype == MLXP_DTYPE_INT8;
  const cudaStream_t s = (cudaStream_t)a->stream;
  if (a->dtype == MLXP_DTYPE_BF16) return qa_launch_t<__nv_bfloat16>(a->D, maps, p, n, int8, s);
  if (a->dtype == MLXP_DTYPE_FP16) return qa_launch_t<__half>(a->D, maps, p, n, int8, s);
  return qa_launch_t<float>(a->D, maps, p, n, int8, s);
}

}  // extern "C"
