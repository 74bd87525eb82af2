// mlxp_cache.cu — host side of the query/key norm + rotation and of appending to a paged cache:
// argument checks, the choice of a row layout and the launches.

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/mlxp_attn.h"
#include "cache_append.cuh"
#include "host_common.h"
#include "norm_rope.cuh"

namespace mlxp {
namespace {

constexpr int kMaxGridSms = 256;   // workspace bound; devices have fewer SMs

int check_dtype(int64_t dt, const char* what) {
  if (dt < 0 || dt > 2) return fail(MLXP_ERR_INVALID, "%s: unknown dtype %lld", what, (long long)dt);
  return MLXP_OK;
}

int check_dim(int64_t D) {
  if (D < 2 || D % 2) return fail(MLXP_ERR_INVALID, "head_dim must be even, got %lld", (long long)D);
  if (D > 256) return fail(MLXP_ERR_UNSUPPORTED, "head_dim must be at most 256, got %lld", (long long)D);
  return MLXP_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Whether rows at these element strides start on 16 bytes.
bool rows16(const void* p, const int64_t st[3], int es) {
  if (!aligned16(p)) return false;
  for (int i = 0; i < 3; ++i)
    if ((st[i] * es) % 16) return false;
  return true;
}

void copy3(long long (&to)[3], const int64_t from[3]) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

// Calls f with the RowShape for (dtype, half, wide): 16-byte pieces, as few lanes a row as hold
// them (so that a warp holds as many rows as it can), or single elements where an address or
// head_dim does not allow 16 bytes.
template <typename T, typename F>
int with_row_shape_t(int half, bool wide, F&& f) {
  constexpr int V = 16 / (int)sizeof(T);
  if (!wide) return f(RowShape<T, 1, 32, 4>{});
  const int pieces = half / V;
  if (pieces <= 4) return f(RowShape<T, V, 4, 1>{});
  if (pieces <= 8) return f(RowShape<T, V, 8, 1>{});
  if (sizeof(T) == 2 || pieces <= 16) return f(RowShape<T, V, 16, 1>{});
  if constexpr (sizeof(T) == 4) return f(RowShape<T, V, 32, 1>{});
  return MLXP_ERR_UNSUPPORTED;  // not reached: half <= 128
}

template <typename F>
int with_row_shape(int64_t dtype, int half, bool wide, F&& f) {
  wide = wide && half % (dtype == MLXP_DTYPE_FP32 ? 4 : 8) == 0;
  if (dtype == MLXP_DTYPE_FP32) return with_row_shape_t<float>(half, wide, f);
  if (dtype == MLXP_DTYPE_BF16) return with_row_shape_t<__nv_bfloat16>(half, wide, f);
  return with_row_shape_t<__half>(half, wide, f);
}

// Row steps loaded at a time and the CTAs of 256 threads an SM holds (the registers' limit).
// Measured on 2 x 16384 x 64 rows of 128 bf16, units of U steps: forward 199 us at (2, 3), 220 at
// (4, 2), 266 at (2, 2); backward 335 at (2, 2), 443 at (2, 1), 362 at (4, 1).  Units of whole
// tokens, at (2, 3) and (2, 2): 184 us (5.8 TB/s) and 280 us (5.8 TB/s).
constexpr int kFwdCtas = 3, kBwdCtas = 2;
template <typename R>
constexpr int fwd_steps() { return 2; }
template <typename R>
constexpr int bwd_steps() { return R::kWide ? 2 : 1; }

// From this many query units an SM, appends to 8-bit pools take two launches: the query rows run
// at three CTAs an SM in a kernel of their own, at two beside the block units, whose registers
// they share (8 ragged prompts, 17.6 K tokens of 32 + 2 x 8 heads of 128: 131 us in two launches,
// 173 in one; below it the second launch costs more than it gives).
constexpr long long kSplitUnits = 64;

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MLXP_OK : cuda_fail(e, what);
}

template <typename R, int U, bool INT8>
int append_quant_launch(const AppendParams& p, unsigned grid, cudaStream_t s) {
  constexpr int smem = 8 * kAppendSteps * R::NP * 32 * (int)sizeof(float4);
  static std::atomic<unsigned long long> attr_done{0};  // one bit per device
  int dev;
  if (int rc = current_device(dev)) return rc;
  if (!(attr_done.load() >> dev & 1ull)) {
    const cudaError_t e = cudaFuncSetAttribute(append_quant_kernel<R, U, INT8>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_append)");
    attr_done.fetch_or(1ull << dev);
  }
  append_quant_kernel<R, U, INT8><<<grid, 256, smem, s>>>(p);
  return launched("paged_append launch");
}

int norm_rope_check(const mlxp_qk_norm_rope_args* a, bool bwd) {
  if (!a || a->size != sizeof(*a)) return fail(MLXP_ERR_INVALID, "argument struct of another size");
  if (int rc = check_dtype(a->dtype, "q, k")) return rc;
  if (int rc = check_dim(a->D)) return rc;
  if (a->B < 0 || a->Sq < 0 || a->Sk < 0 || a->Hq < 0 || a->Hk < 0)
    return fail(MLXP_ERR_INVALID, "negative sizes");
  if (!a->cos_cache != !a->sin_cache) return fail(MLXP_ERR_INVALID, "cos and sin go together");
  if (!a->q_weight != !a->k_weight) return fail(MLXP_ERR_INVALID, "q_weight and k_weight go together");
  if (a->q_weight) {
    if (int rc = check_dtype(a->q_weight_dtype, "q_weight")) return rc;
    if (int rc = check_dtype(a->k_weight_dtype, "k_weight")) return rc;
  }
  if (!(a->eps >= 0) || !std::isfinite(a->eps)) return fail(MLXP_ERR_INVALID, "eps must be finite and >= 0");
  if (a->cos_cache && a->n_pos < 1) return fail(MLXP_ERR_INVALID, "the cos/sin tables are empty");
  if (a->positions) {
    if (a->Sq != a->Sk)
      return fail(MLXP_ERR_INVALID, "positions need q and k of one length, got %lld and %lld",
                  (long long)a->Sq, (long long)a->Sk);
  } else if (a->cos_cache) {
    const int64_t off[2] = {a->q_offset, a->k_offset}, len[2] = {a->Sq, a->Sk};
    for (int i = 0; i < 2; ++i)
      if (off[i] < 0 || off[i] > a->n_pos - len[i])
        return fail(MLXP_ERR_INVALID, "positions [%lld, %lld) exceed the cos/sin cache of %lld positions",
                    (long long)off[i], (long long)(off[i] + len[i]), (long long)a->n_pos);
  }
  const bool some[2] = {a->B * a->Sq * a->Hq > 0, a->B * a->Sk * a->Hk > 0};
  if ((some[0] && (!a->q || (!a->q_out && (!bwd || a->gq)))) ||
      (some[1] && (!a->k || (!a->k_out && (!bwd || a->gk)))))
    return fail(MLXP_ERR_INVALID, "q, k and their outputs must be non-null");
  if (bwd && ((a->dq_weight && !a->q_weight) || (a->dk_weight && !a->k_weight)))
    return fail(MLXP_ERR_INVALID, "a weight's gradient needs the weight");
  // units are counted in 32 bits; a unit has at least one row
  for (const int64_t n : {a->B * a->Sq, a->B * a->Sk})
    if (n > INT32_MAX || n * std::max(a->Hq, a->Hk) > INT32_MAX)
      return fail(MLXP_ERR_INVALID, "too many rows");
  return MLXP_OK;
}

// Fills the kernel's parameters; `wide`: 16-byte pieces are possible.
NormRopeParams norm_rope_params(const mlxp_qk_norm_rope_args* a, bool bwd, bool& wide) {
  NormRopeParams p{};
  const int es = a->dtype == MLXP_DTYPE_FP32 ? 4 : 2;
  wide = aligned16(a->cos_cache) && aligned16(a->sin_cache) && aligned16(a->q_weight) &&
         aligned16(a->k_weight);
  const void* x[2] = {a->q, a->k};
  void* y[2] = {a->q_out, a->k_out};
  const void* g[2] = {a->gq, a->gk};
  const void* w[2] = {a->q_weight, a->k_weight};
  const int64_t* xs[2] = {a->q_strides, a->k_strides};
  const int64_t* ys[2] = {a->q_out_strides, a->k_out_strides};
  const int64_t* gs[2] = {a->gq_strides, a->gk_strides};
  const int64_t H[2] = {a->Hq, a->Hk}, S[2] = {a->Sq, a->Sk}, off[2] = {a->q_offset, a->k_offset};
  const int64_t wd[2] = {a->q_weight_dtype, a->k_weight_dtype};
  for (int i = 0; i < 2; ++i) {
    NormRopeTensor& t = p.t[i];
    t.x = x[i];
    t.y = y[i];
    t.gy = g[i];
    copy3(t.xs, xs[i]);
    copy3(t.ys, ys[i]);
    copy3(t.gs, gs[i]);
    t.H = (int)H[i];
    t.S = (int)S[i];
    t.offset = off[i];
    t.norm = NormSpec{w[i], (int)wd[i], (float)a->eps, 1.f / (float)a->D};
    if (H[i] * S[i] * a->B == 0 || (bwd && !g[i])) t.H = 0;  // nothing to do for this tensor
    if (t.H == 0) continue;
    wide = wide && rows16(x[i], xs[i], es) && rows16(y[i], ys[i], es) &&
           (!bwd || rows16(g[i], gs[i], es));
  }
  p.half = (int)(a->D / 2);
  p.cosc = a->cos_cache;
  p.sinc = a->sin_cache;
  p.n_pos = a->n_pos;
  p.positions = a->positions;
  p.pos_sb = a->pos_strides[0];
  p.pos_ss = a->pos_strides[1];
  return p;
}

// Row steps a unit (one warp's work at a time) takes of a token's `all`: all of them where the
// tokens alone fill the SMs' warps, else the kernel's U.
int unit_steps(long long tokens, int all, int U, int sms) {
  return tokens >= 24LL * sms ? std::max(all, 1) : U;
}

// Units of both tensors for rpw rows a step.
void count_units(NormRopeParams& p, int64_t B, int rpw, int U, int sms) {
  for (NormRopeTensor& t : p.t) {
    const int all = (t.H + rpw - 1) / rpw;
    t.steps = unit_steps(B * t.S, all, U, sms);
    t.groups = std::max(1, (all + t.steps - 1) / t.steps);
    t.units = t.H ? B * t.S * (long long)t.groups : 0;
  }
}

}  // namespace
}  // namespace mlxp

using namespace mlxp;

extern "C" {

int mlxp_qk_norm_rope(const mlxp_qk_norm_rope_args* a) {
  if (int rc = norm_rope_check(a, false)) return rc;
  bool wide;
  NormRopeParams p = norm_rope_params(a, false, wide);
  if (p.t[0].H == 0 && p.t[1].H == 0) return MLXP_OK;
  int sms;
  if (int rc = device_info(nullptr, &sms)) return rc;
  return with_row_shape(a->dtype, p.half, wide, [&](auto shape) {
    using R = decltype(shape);
    constexpr int U = fwd_steps<R>();
    count_units(p, a->B, R::RPW, U, sms);
    const long long units = p.t[0].units + p.t[1].units;
    // few units: one warp a block, so that they spread over the SMs
    const int warps = units >= 8LL * sms ? 8 : 1;
    const long long grid = std::min<long long>((units + warps - 1) / warps, 64LL * sms);
    norm_rope_kernel<R, U, kFwdCtas><<<(unsigned)grid, 32 * warps, 0, (cudaStream_t)a->stream>>>(p);
    return launched("qk_norm_rope launch");
  });
}

size_t mlxp_qk_norm_rope_bwd_workspace_size(int64_t D) {
  if (D < 2 || D > 256) return 0;
  return (size_t)kMaxGridSms * kBwdCtas * 2 * D * sizeof(float);
}

int mlxp_qk_norm_rope_bwd(const mlxp_qk_norm_rope_args* a) {
  if (int rc = norm_rope_check(a, true)) return rc;
  bool wide;
  NormRopeParams p = norm_rope_params(a, true, wide);
  const bool dw = a->dq_weight || a->dk_weight;
  if (dw && (!a->workspace || a->ws_bytes < mlxp_qk_norm_rope_bwd_workspace_size(a->D)))
    return fail(MLXP_ERR_WORKSPACE, "qk_norm_rope_bwd needs %zu bytes of workspace, got %llu",
                mlxp_qk_norm_rope_bwd_workspace_size(a->D), (unsigned long long)a->ws_bytes);
  if (dw && !aligned16(a->workspace)) return fail(MLXP_ERR_INVALID, "workspace must be 16-byte aligned");
  if (p.t[0].H == 0 && p.t[1].H == 0 && !dw) return MLXP_OK;
  int sms;
  if (int rc = device_info(nullptr, &sms)) return rc;
  sms = std::min(sms, kMaxGridSms);
  const cudaStream_t s = (cudaStream_t)a->stream;
  return with_row_shape(a->dtype, p.half, wide, [&](auto shape) {
    using R = decltype(shape);
    constexpr int U = bwd_steps<R>();
    count_units(p, a->B, R::RPW, U, sms);
    const long long most = std::max(p.t[0].units, p.t[1].units);
    const long long grid =
        std::max<long long>(1, std::min<long long>((most + 7) / 8, (long long)kBwdCtas * sms));
    float* part = static_cast<float*>(a->workspace);
    p.t[0].dw_part = a->dq_weight ? part : nullptr;
    p.t[1].dw_part = a->dk_weight ? part + grid * a->D : nullptr;
    norm_rope_bwd_kernel<R, U, kBwdCtas><<<(unsigned)grid, 256, 8 * a->D * sizeof(float), s>>>(p);
    if (int rc = launched("qk_norm_rope backward launch")) return rc;
    if (!dw) return (int)MLXP_OK;
    NormRopeDw d{{p.t[0].dw_part, p.t[1].dw_part},
                 {a->dq_weight, a->dk_weight},
                 {(int)a->q_weight_dtype, (int)a->k_weight_dtype},
                 (int)grid,
                 (int)a->D};
    norm_rope_dw_kernel<<<dim3((unsigned)(a->D + 31) / 32, 2), dim3(32, 32), 0, s>>>(d);
    return launched("qk_norm_rope weight gradient launch");
  });
}

int mlxp_paged_append(const mlxp_paged_append_args* a) {
  if (!a || a->size != sizeof(*a)) return fail(MLXP_ERR_INVALID, "argument struct of another size");
  if (int rc = check_dtype(a->dtype, "k, v")) return rc;
  if (int rc = check_dim(a->D)) return rc;
  const bool quant = a->cache_dtype == MLXP_DTYPE_E4M3 || a->cache_dtype == MLXP_DTYPE_INT8;
  if (!quant && a->cache_dtype != a->dtype)
    return fail(MLXP_ERR_INVALID, "the pools' dtype must be the inputs', or an 8-bit one");
  if (a->B < 0 || a->S < 0 || a->Hk < 1 || a->num_blocks < 0 || a->block_size < 1 || a->max_blocks < 0 ||
      (a->q && a->Hq < 1))
    return fail(MLXP_ERR_INVALID, "invalid shape B=%lld S=%lld Hq=%lld Hk=%lld num_blocks=%lld "
                "block_size=%lld max_blocks=%lld", (long long)a->B, (long long)a->S, (long long)a->Hq,
                (long long)a->Hk, (long long)a->num_blocks, (long long)a->block_size, (long long)a->max_blocks);
  if (!a->cos_cache != !a->sin_cache) return fail(MLXP_ERR_INVALID, "cos and sin go together");
  if (a->q_weight)
    if (int rc = check_dtype(a->q_weight_dtype, "q_weight")) return rc;
  if (a->k_weight)
    if (int rc = check_dtype(a->k_weight_dtype, "k_weight")) return rc;
  if (!(a->eps >= 0) || !std::isfinite(a->eps)) return fail(MLXP_ERR_INVALID, "eps must be finite and >= 0");
  if (a->num_blocks > INT32_MAX || a->block_size > INT32_MAX || a->max_blocks > INT32_MAX ||
      a->max_blocks * a->block_size > kMaxCacheIndex || a->B > INT32_MAX || a->S > INT32_MAX ||
      a->B * a->S > INT32_MAX || a->B * a->S * std::max(a->q ? a->Hq : 1, a->Hk) > INT32_MAX)
    return fail(MLXP_ERR_INVALID, "paged shape too large");
  if (a->B == 0 || a->S == 0) return MLXP_OK;
  if (a->cos_cache && (a->n_pos < 1 || a->n_pos < a->max_blocks * a->block_size))
    return fail(MLXP_ERR_INVALID, "the cos/sin tables have %lld positions, the block tables %lld",
                (long long)a->n_pos, (long long)(a->max_blocks * a->block_size));
  if (!a->k || !a->v || !a->context_lens || (a->q && !a->q_out))
    return fail(MLXP_ERR_INVALID, "k, v, context_lens and q's output must be non-null");
  if (a->max_blocks > 0 && (!a->block_tables || (a->num_blocks > 0 && (!a->k_pool || !a->v_pool))))
    return fail(MLXP_ERR_INVALID, "the pools and block_tables must be non-null");
  if (a->max_blocks > 0 && a->B > 1 && a->bt_stride < a->max_blocks)
    return fail(MLXP_ERR_INVALID, "block-table row stride (%lld) is below max_blocks (%lld)",
                (long long)a->bt_stride, (long long)a->max_blocks);
  if (quant && a->num_blocks > 0 && (!a->k_scales || !a->v_scales))
    return fail(MLXP_ERR_INVALID, "8-bit pools need their scales");
  if (a->num_blocks > 0 && (a->k_pool == a->v_pool || (quant && a->k_scales == a->v_scales)))
    return fail(MLXP_ERR_INVALID, "keys and values must go to different pools and scales");

  AppendParams p{};
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.q_out = a->q_out;
  p.k_pool = a->k_pool;
  p.v_pool = a->v_pool;
  p.k_scales = a->k_scales;
  p.v_scales = a->v_scales;
  p.block_tables = a->block_tables;
  p.context_lens = a->context_lens;
  p.new_lens = a->new_lens;
  copy3(p.q_s, a->q_strides);
  copy3(p.k_s, a->k_strides);
  copy3(p.v_s, a->v_strides);
  copy3(p.qo_s, a->q_out_strides);
  p.p_sb = a->pool_strides[0];
  p.p_st = a->pool_strides[1];
  p.p_sh = a->pool_strides[2];
  p.sc_sb = a->scale_strides[0];
  p.sc_sh = a->scale_strides[1];
  p.bt_stride = a->bt_stride;
  p.B = (int)a->B;
  p.S = (int)a->S;
  p.Hq = a->q ? (int)a->Hq : 0;
  p.Hk = (int)a->Hk;
  p.half = (int)(a->D / 2);
  // without blocks every id is out of range: nothing is written
  p.num_blocks = (int)a->num_blocks;
  p.block_size = (int)a->block_size;
  p.max_blocks = (int)a->max_blocks;
  const float inv_d = 1.f / (float)a->D;
  p.q_norm = NormSpec{a->q_weight, (int)a->q_weight_dtype, (float)a->eps, inv_d};
  p.k_norm = NormSpec{a->k_weight, (int)a->k_weight_dtype, (float)a->eps, inv_d};
  p.cosc = a->cos_cache;
  p.sinc = a->sin_cache;
  p.n_pos = a->n_pos;

  const int es = a->dtype == MLXP_DTYPE_FP32 ? 4 : 2;
  bool wide = aligned16(a->cos_cache) && aligned16(a->sin_cache) && aligned16(a->q_weight) &&
              aligned16(a->k_weight) && rows16(a->k, a->k_strides, es) && rows16(a->v, a->v_strides, es);
  if (a->q) wide = wide && rows16(a->q, a->q_strides, es) && rows16(a->q_out, a->q_out_strides, es);
  if (quant) {  // pieces of 8 or 4 codes
    for (const void* pool : {a->k_pool, a->v_pool}) wide = wide && reinterpret_cast<uintptr_t>(pool) % 8 == 0;
    for (int i = 0; i < 3; ++i) wide = wide && a->pool_strides[i] % 8 == 0;
  } else {
    wide = wide && rows16(a->k_pool, a->pool_strides, es) && aligned16(a->v_pool);
  }
  int sms;
  if (int rc = device_info(nullptr, &sms)) return rc;
  const cudaStream_t s = (cudaStream_t)a->stream;
  return with_row_shape(a->dtype, p.half, wide, [&](auto shape) {
    using R = decltype(shape);
    constexpr int U = bwd_steps<R>();
    const int heads = R::RPW * U;
    const long long tokens = a->B * a->S;
    const int all = (p.Hq + R::RPW - 1) / R::RPW;
    p.q_steps = unit_steps(tokens, all, U, sms);
    p.q_groups = std::max(1, (all + p.q_steps - 1) / p.q_steps);
    p.k_groups = (p.Hk + heads - 1) / heads;
    p.q_units = p.Hq ? tokens * p.q_groups : 0;
    p.kv_units = tokens * p.k_groups;
    if (!quant) {
      const long long units = p.q_units + 2 * p.kv_units;
      const int warps = units >= 8LL * sms ? 8 : 1;
      const long long grid = std::min<long long>((units + warps - 1) / warps, 64LL * sms);
      append_kernel<R, U><<<(unsigned)grid, 32 * warps, 0, s>>>(p);
      return launched("paged_append launch");
    }
    // warps a unit: as many as hold the rows it can have, at most all eight
    constexpr int ROWS = kAppendSteps * R::RPW;
    const long long rows = std::min<long long>(a->block_size, a->S);
    p.wpu = 1;
    while (p.wpu < 8 && p.wpu * ROWS < rows) p.wpu *= 2;
    p.touch = (int)((a->S + a->block_size - 2) / a->block_size + 1);
    p.block_units = a->B * p.touch * 2 * a->Hk;
    if (p.block_units > INT32_MAX) return fail(MLXP_ERR_INVALID, "paged shape too large");
    const int upc = 8 / p.wpu;
    if (p.q_units >= kSplitUnits * sms) {  // many query rows: a launch of their own, see there
      append_q_kernel<R, U><<<(unsigned)std::min<long long>((p.q_units + 7) / 8, 64LL * sms), 256, 0, s>>>(p);
      if (int rc = launched("paged_append launch (queries)")) return rc;
      p.q_units = 0;
    }
    p.q_ctas = (int)std::min<long long>((p.q_units + 7) / 8, 16LL * sms);
    const long long ctas = std::min<long long>((p.block_units + upc - 1) / upc, 64LL * sms);
    const unsigned grid = (unsigned)(p.q_ctas + ctas);
    return a->cache_dtype == MLXP_DTYPE_INT8 ? append_quant_launch<R, U, true>(p, grid, s)
                                             : append_quant_launch<R, U, false>(p, grid, s);
  });
}

}  // extern "C"
