// cache_append.cuh — new keys and values into a paged K/V pool, the keys (and the queries beside
// them) normed and rotated on the way, in one launch (long prompts into 8-bit pools: two).
//
// Token i of sequence b (i < new_lens[b]) has position pos = context_lens[b] + i and goes to row
// pos % block_size of pool block block_tables[b][pos / block_size].  A position below 0 or past
// the table, and a table entry outside [0, num_blocks), drop the token; nothing else is written.
// Queries of padding tokens and of positions outside the table become zeros (one whose block is
// missing is computed: it may attend to what is there).
//
// 16/32-bit pools: the rows are written as computed, rounded once (row units as in norm_rope.cuh,
// which also describes the norm and the rotation).
//
// 8-bit pools hold codes and one fp32 scale a (block, head); the value is code * scale.  Over the
// new tokens of a block, least = the least power of two 2^k >= 2^-126 with amax <= qmax * 2^k
// (qmax 448 for e4m3, 127 for int8; amax over the finite values).  A block whose row 0 is among
// the new tokens takes that scale; one that already holds tokens keeps its own, or grows to
// `least` where that is larger, and its old codes are then rescaled.  Powers of two because a
// block filled token by token may grow its scale several times: rescaling by 2^-n leaves e4m3
// codes exact down to their subnormals, and a scale grows at most once an octave.
// A code is x / scale rounded to nearest even, clamped to +-qmax; NaN stays NaN in e4m3 and is 0
// in int8.
//
// One unit is (sequence, touched block, head, K or V), taken by WPU warps: they read the block's
// new rows once and keep them (16 bf16 rows of 128 a warp: blocks of 16 need no other warp), in
// registers as loaded and in shared memory as computed, until amax is known, on which they agree
// through shared memory where they are several.  A block of more rows than eight warps hold is
// read a second time (from L2).
//
// What bounds it: latency for single tokens (8 of them 3 us into 16-bit pools, 4.4 into e4m3: table
// entry, scale, rows, maximum, old codes, one after the other); for prompts HBM on the query side
// (32 heads of 128, 17.6 K ragged tokens: 75 us, 5.4 TB/s) and issue on the block side (2 x 8
// heads of the same tokens: 56 us, 27.8 M warp instructions; 17 by its bytes).
#pragma once

#include <cuda_fp8.h>

#include "norm_rope.cuh"

namespace mlxp {

struct AppendParams {
  const void *q, *k, *v;                  // q nullable
  void* q_out;
  void *k_pool, *v_pool;
  float *k_scales, *v_scales;             // 8-bit pools: [num_blocks][Hk], strides sc_sb, sc_sh
  const int* block_tables;
  const int* context_lens;
  const int* new_lens;                    // nullable: S for every sequence
  long long q_s[3], k_s[3], v_s[3], qo_s[3];  // element strides of (batch, head, seq)
  long long p_sb, p_st, p_sh;             // pool element strides (block, token, head)
  long long sc_sb, sc_sh;
  long long bt_stride;
  int B, S, Hq, Hk, half;
  int num_blocks, block_size, max_blocks;
  NormSpec q_norm, k_norm;
  const float *cosc, *sinc;
  long long n_pos;
  int q_steps, q_groups;                  // row steps a unit of q, units a token
  int k_groups;                           // units a token of each of k and v
  long long q_units, kv_units;            // row units (kv: 16/32-bit pools)
  int q_ctas;                             // 8-bit pools: CTAs [0, q_ctas) take the q units
  int touch;                              // 8-bit pools: blocks a sequence may touch
  int wpu;                                // 8-bit pools: warps a unit
  long long block_units;
};

// New tokens of sequence b and its length before.
__device__ __forceinline__ int append_count(const AppendParams& p, int b) {
  if (!p.new_lens) return p.S;
  const int n = __ldg(p.new_lens + b);
  return n < 0 ? 0 : min(n, p.S);
}

__device__ __forceinline__ int pool_block(const AppendParams& p, int b, long long slot) {
  if (slot < 0 || slot >= p.max_blocks) return -1;
  const int id = __ldg(p.block_tables + b * p.bt_stride + slot);
  return id < p.num_blocks ? id : -1;
}

// Query rows of unit u, normed and rotated into q_out.
template <typename R, int U>
__device__ __forceinline__ void append_q_unit(const AppendParams& p, unsigned u, int j, int g) {
  using T = typename R::T;
  const unsigned tok = u / (unsigned)p.q_groups;
  const int first = (int)(u - tok * (unsigned)p.q_groups) * p.q_steps * R::RPW;
  const int last = min(p.Hq, first + p.q_steps * R::RPW);
  const int b = (int)(tok / (unsigned)p.S), i = (int)(tok - (unsigned)b * (unsigned)p.S);
  const T* x = static_cast<const T*>(p.q) + b * p.q_s[0] + i * p.q_s[2];
  T* y = static_cast<T*>(p.q_out) + b * p.qo_s[0] + i * p.qo_s[2];
  // padding rows of a ragged batch are not read: their number is looked up first
  const bool within = i < append_count(p, b);
  RowData<R> d[U];
  auto load = [&](int h0) {
#pragma unroll
    for (int r = 0; r < U; ++r) {
      const int h = h0 + r * R::RPW + g;
      row_load<R>(x + h * p.q_s[1], p.half, j, within && h < last, d[r]);
    }
  };
  load(first);
  RowCoef<R> k;
  coef_weights<R>(p.q_norm, p.half, j, k);
  const long long pos = (long long)__ldg(p.context_lens + b) + i;
  const bool live = within && pos >= 0 && pos < (long long)p.max_blocks * p.block_size;
  coef_tables<R>(p.cosc, p.sinc, live ? pos : 0, p.half, j, k);
  for (int h0 = first;;) {
#pragma unroll
    for (int r = 0; r < U; ++r) {
      const int h = h0 + r * R::RPW + g;
      float2 y1[R::NP], y2[R::NP];
      row_norm_rope<R>(d[r], p.q_norm, p.cosc != nullptr, k, y1, y2);
      if (!live) fill2<R::NP>(0.f, y1, y2);
      if (h < last) row_store<R>(y + h * p.qo_s[1], p.half, j, y1, y2);
    }
    h0 += U * R::RPW;
    if (h0 >= last) return;
    load(h0);
  }
}

// Query units alone (many of them, beside an 8-bit pool's block units in another launch).
template <typename R, int U>
__global__ void __launch_bounds__(256, 3) append_q_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 31, j = lane % R::LPR, g = lane / R::LPR;
  for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < p.q_units; u += 8LL * gridDim.x)
    append_q_unit<R, U>(p, (unsigned)u, j, g);
}

// Pools of the inputs' type: units [0, q_units) are queries, then keys, then values.
template <typename R, int U>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  using T = typename R::T;
  const int lane = threadIdx.x & 31, j = lane % R::LPR, g = lane / R::LPR;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  const long long total = p.q_units + 2 * p.kv_units;
  for (long long u = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < total;
       u += warps) {
    if (u < p.q_units) {
      append_q_unit<R, U>(p, (unsigned)u, j, g);
      continue;
    }
    const bool is_v = u >= p.q_units + p.kv_units;
    const unsigned w = (unsigned)(u - p.q_units - (is_v ? p.kv_units : 0));
    const unsigned tok = w / (unsigned)p.k_groups;
    const int h0 = (int)(w - tok * (unsigned)p.k_groups) * (R::RPW * U) + g;
    const int b = (int)(tok / (unsigned)p.S), i = (int)(tok - (unsigned)b * (unsigned)p.S);
    const long long* st = is_v ? p.v_s : p.k_s;
    const T* x = static_cast<const T*>(is_v ? p.v : p.k) + b * st[0] + i * st[2];
    RowData<R> d[U];
#pragma unroll
    for (int r = 0; r < U; ++r) {
      const int h = h0 + r * R::RPW;
      row_load<R>(x + h * st[1], p.half, j, h < p.Hk, d[r]);
    }
    RowCoef<R> k;
    if (!is_v) coef_weights<R>(p.k_norm, p.half, j, k);
    const long long pos = (long long)__ldg(p.context_lens + b) + i;
    int id = -1;
    if (i < append_count(p, b) && pos >= 0) id = pool_block(p, b, pos / p.block_size);
    if (id < 0) continue;  // the same for the whole warp
    T* y = static_cast<T*>(is_v ? p.v_pool : p.k_pool) + id * p.p_sb + (pos % p.block_size) * p.p_st;
    if (!is_v) coef_tables<R>(p.cosc, p.sinc, pos, p.half, j, k);
#pragma unroll
    for (int r = 0; r < U; ++r) {
      const int h = h0 + r * R::RPW;
      float2 y1[R::NP], y2[R::NP];
      if (is_v) {
        row_to_f<R>(d[r].x1, y1);
        row_to_f<R>(d[r].x2, y2);
      } else {
        row_norm_rope<R>(d[r], p.k_norm, p.cosc != nullptr, k, y1, y2);
      }
      if (h < p.Hk) row_store<R>(y + h * p.p_sh, p.half, j, y1, y2);
    }
  }
}

// Exponent k of the least 2^k >= 2^-126 with amax <= qmax * 2^k, as the fp32 scale.  qmax =
// (1 + QM / 2^23) * 2^QE.
template <bool INT8>
__device__ __forceinline__ float least_scale(float amax) {
  constexpr unsigned QM = INT8 ? 0x7e0000u : 0x600000u;  // 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
  constexpr int QE = INT8 ? 6 : 8;
  const unsigned u = __float_as_uint(amax);
  int k = (int)(u >> 23) - 127 - QE + ((u & 0x7fffffu) > QM);
  k = max(k, -126);
  return __uint_as_float((unsigned)(k + 127) << 23);
}

template <bool INT8>
__device__ __forceinline__ unsigned to_code(float x) {
  if constexpr (INT8) {
    return (unsigned)__float2int_rn(fminf(fmaxf(x != x ? 0.f : x, -127.f), 127.f)) & 0xffu;
  } else {
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  }
}

template <bool INT8>
__device__ __forceinline__ float from_code(unsigned c) {
  if constexpr (INT8) return (float)(signed char)c;
  const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
  return __half2float(__half(h));
}

// Codes of one half-row piece: VEC bytes.
template <bool INT8, int VEC>
__device__ __forceinline__ void store_codes(unsigned char* y, const float* x) {
  if constexpr (VEC == 1) {
    *y = (unsigned char)to_code<INT8>(x[0]);
  } else {
    unsigned w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      if constexpr (INT8) {
        w[i] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[i] |= to_code<INT8>(x[4 * i + e]) << (8 * e);
      } else {
        const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
        w[i] = lo | hi << 16;
      }
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(y) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<unsigned*>(y) = w[0];
  }
}

constexpr int kAppendSteps = 4;           // row steps of a block that a warp keeps

template <typename R, int U, bool INT8>
__global__ void __launch_bounds__(256, 2) append_quant_kernel(const AppendParams p) {
  using T = typename R::T;
  constexpr int ROWS = kAppendSteps * R::RPW;  // rows a warp keeps
  __shared__ float s_amax[8];
  extern __shared__ float4 s_keep[];      // [8 warps][kAppendSteps][NP][32 lanes]
  const int lane = threadIdx.x & 31, j = lane % R::LPR, g = lane / R::LPR;
  const int warp = threadIdx.x >> 5;
  if ((int)blockIdx.x < p.q_ctas) {
    for (long long u = (long long)blockIdx.x * 8 + warp; u < p.q_units; u += 8LL * p.q_ctas)
      append_q_unit<R, U>(p, (unsigned)u, j, g);
    return;
  }
  const int upc = 8 / p.wpu;              // units a CTA at a time
  const int part = warp % p.wpu;          // this warp's share of its unit's rows
  const long long ctas = gridDim.x - p.q_ctas;
  for (long long u0 = (long long)(blockIdx.x - p.q_ctas) * upc; u0 < p.block_units; u0 += ctas * upc) {
    const long long u = u0 + warp / p.wpu;
    // unit = ((sequence * touch + slot) * 2 + is_v) * Hk + head
    const bool there = u < p.block_units;
    const unsigned uu = (unsigned)(there ? u : 0);
    const int h = (int)(uu % (unsigned)p.Hk);
    const unsigned rest = uu / (unsigned)p.Hk;
    const bool is_v = rest & 1;
    const unsigned bs = rest >> 1;
    const int b = (int)(bs / (unsigned)p.touch);
    const int slot_i = (int)(bs - (unsigned)b * (unsigned)p.touch);
    const long long ctx = __ldg(p.context_lens + b);
    const long long lo = ctx < 0 ? 0 : ctx, hi = ctx + append_count(p, b);  // new positions
    const long long slot = lo / p.block_size + slot_i, base = slot * p.block_size;
    const int r0 = (int)max(lo - base, 0LL);                        // new rows of the block
    // none where the block is past the table: so are its positions, which the cos/sin tables need
    // not cover
    const int r1 = there && hi > lo && slot < p.max_blocks
                       ? (int)max(min(hi - base, (long long)p.block_size), (long long)r0)
                       : r0;
    const int stride = ROWS * p.wpu;      // rows the unit's warps hold at a time
    // slabs of `stride` rows that hold new ones: [first, first + n) of the block's
    const int first = r0 / stride, n = r1 > r0 ? (r1 - 1) / stride - first + 1 : 0;
    if (p.wpu == 1 && n == 0) continue;   // the same for the whole warp, which syncs with none
    const long long* st = is_v ? p.v_s : p.k_s;
    const T* x = static_cast<const T*>(is_v ? p.v : p.k) + b * st[0] + h * st[1];
    // The rows are on their way before the block is known.
    RowData<R> d[kAppendSteps];
    auto load = [&](int sl) {
      const int row0 = (first + sl) * stride + part * ROWS + g;
#pragma unroll
      for (int i = 0; i < kAppendSteps; ++i) {
        const int r = row0 + i * R::RPW;
        row_load<R>(x + (base + r - ctx) * st[2], p.half, j, r >= r0 && r < r1, d[i]);
      }
    };
    if (n > 0) load(0);
    const int id = n > 0 ? pool_block(p, b, slot) : -1;
    const bool on = id >= 0;
    unsigned char* pool = static_cast<unsigned char*>(is_v ? p.v_pool : p.k_pool) +
                          (on ? id : 0) * p.p_sb + h * p.p_sh;
    float* scale = (is_v ? p.v_scales : p.k_scales) + (on ? id : 0) * p.sc_sb + h * p.sc_sh;
    const float s_old = on && r0 > 0 ? *scale : 0.f;
    RowCoef<R> kw;
    if (!is_v) coef_weights<R>(p.k_norm, p.half, j, kw);
    float s_new = 1.f;
    // The rows' values wait in shared memory for the block's scale, every lane's own, so without a
    // barrier: in registers they would take twice the rows' room.
    float4* mine = s_keep + warp * kAppendSteps * R::NP * 32 + lane;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      float amax = 0.f;
      const bool divide = pass == 1 && (__float_as_uint(s_new) & 0x7fffffu) != 0;
      const float inv = pass == 1 && !divide ? __fdiv_rn(1.f, s_new) : 1.f;
#pragma unroll 1
      for (int sl = 0; sl < n; ++sl) {
        if (n > 1 && (pass == 1 || sl > 0)) load(sl);
        const int row0 = (first + sl) * stride + part * ROWS + g;
        if (pass == 0 || n > 1) {
#pragma unroll
          for (int i = 0; i < kAppendSteps; ++i) {
            const int r = row0 + i * R::RPW;
            const bool live = r >= r0 && r < r1;
            if (!__any_sync(0xffffffffu, live)) continue;
            float2 y1[R::NP], y2[R::NP];
            if (is_v) {
              row_to_f<R>(d[i].x1, y1);
              row_to_f<R>(d[i].x2, y2);
            } else {
              coef_tables<R>(p.cosc, p.sinc, live ? base + r : 0, p.half, j, kw);
              row_norm_rope<R>(d[i], p.k_norm, p.cosc != nullptr, kw, y1, y2);
            }
            float4* keep = mine + i * R::NP * 32;
            float big = 0.f;
#pragma unroll
            for (int e = 0; e < R::NP; ++e) {
              keep[32 * e] = make_float4(y1[e].x, y1[e].y, y2[e].x, y2[e].y);
              big = fmaxf(fmaxf(big, fmaxf(fabsf(y1[e].x), fabsf(y1[e].y))),
                          fmaxf(fabsf(y2[e].x), fabsf(y2[e].y)));
            }
            if (big > 3.402823466e38f) {  // infinities: the finite ones one by one
              big = 0.f;
#pragma unroll 1
              for (int e = 0; e < R::NP; ++e) {
                const float4 z = keep[32 * e];
                for (const float v : {z.x, z.y, z.z, z.w})
                  if (fabsf(v) <= 3.402823466e38f) big = fmaxf(big, fabsf(v));
              }
            }
            if (live) amax = fmaxf(amax, big);  // fmaxf passes NaN over
          }
        }
        if (pass == 0 || !on) continue;
#pragma unroll 1
        for (int i = 0; i < kAppendSteps; ++i) {
          const int r = row0 + i * R::RPW;
          if (r < r0 || r >= r1) continue;
          const float4* keep = mine + i * R::NP * 32;
          float v1[R::NE], v2[R::NE];
#pragma unroll
          for (int e = 0; e < R::NP; ++e) {
            const float4 z = keep[32 * e];
            v1[2 * e] = z.x;
            v1[2 * e + 1] = z.y;
            v2[2 * e] = z.z;
            v2[2 * e + 1] = z.w;
          }
          if (divide) {
#pragma unroll 1
            for (int e = 0; e < R::NP; ++e) {
              float4* z = mine + (i * R::NP + e) * 32;
              *z = make_float4(__fdiv_rn(z->x, s_new), __fdiv_rn(z->y, s_new), __fdiv_rn(z->z, s_new), __fdiv_rn(z->w, s_new));
            }
#pragma unroll
            for (int e = 0; e < R::NP; ++e) {
              const float4 z = keep[32 * e];
              v1[2 * e] = z.x;
              v1[2 * e + 1] = z.y;
              v2[2 * e] = z.z;
              v2[2 * e + 1] = z.w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < R::NE; ++e) {
              v1[e] *= inv;
              v2[e] *= inv;
            }
          }
#pragma unroll
          for (int c = 0; c < R::NC; ++c) {
            const int at = piece_at<R>(c, j);
            if (at >= p.half) continue;
            unsigned char* y = pool + r * p.p_st + at;
            store_codes<INT8, R::VEC>(y, v1 + c * R::VEC);
            store_codes<INT8, R::VEC>(y + p.half, v2 + c * R::VEC);
          }
        }
      }
      if (pass == 1) break;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      if (p.wpu > 1) {
        if (lane == 0) s_amax[warp] = amax;
        __syncthreads();
        for (int w = 0; w < p.wpu; ++w) amax = fmaxf(amax, s_amax[warp / p.wpu * p.wpu + w]);
        __syncthreads();  // also: every warp has read the old scale
      }
      const float least = least_scale<INT8>(amax);
      s_new = r0 > 0 && !(s_old < least) ? s_old : least;
      if (!on) continue;
      if (part == 0 && lane == 0) *scale = s_new;
      if (r0 > 0 && s_new != s_old) {     // the block's earlier rows, in the new scale
        const float ratio = __fdiv_rn(s_old, s_new);
        for (int r = part * R::RPW + g; r < r0; r += R::RPW * p.wpu) {
#pragma unroll
          for (int c = 0; c < R::NC; ++c) {
            const int at = piece_at<R>(c, j);
            if (at >= p.half) continue;
#pragma unroll 1
            for (int hf = 0; hf < 2; ++hf) {
              unsigned char* y = pool + r * p.p_st + hf * p.half + at;
              float f[R::VEC];
#pragma unroll
              for (int e = 0; e < R::VEC; ++e) f[e] = from_code<INT8>(y[e]) * ratio;
              store_codes<INT8, R::VEC>(y, f);
            }
          }
        }
      }
    }
  }
}

}  // namespace mlxp
