// norm_rope.cuh — RMS norm of each query/key head row followed by the half-split rotation, the
// forward and the backward, in one pass over the rows.
//
// With h = D / 2, x1 = x[:h], x2 = x[h:], r = (mean(x^2) + eps)^-1/2 and (c, s) the table row of
// the token's position,
//   y = x * r * w,   out1 = y1 c - y2 s,   out2 = y1 s + y2 c,
// and for a gradient g_out: g1 = g_out1 c + g_out2 s, g2 = g_out2 c - g_out1 s (the rotation's
// transpose), dw = sum over rows of g x r, dx = r (g w - x r^2 mean(g w x)).  Sums, norms and the
// rotation are fp32; outputs are rounded once to the element type.  A negative position marks a
// padding row: its output and gradient are zero and it adds nothing to dw.  A position past the
// tables gives a row of NaN.
//
// Layout of the work.  A row is held by LPR lanes, each with one 16-byte piece of either half, so
// that the pairs of the rotation meet in one lane; 32 / LPR rows (heads of one token) make a
// step and U steps a unit, whose loads are all issued before the first is used.  The heads of a
// unit share a position, so its table rows are loaded once for U * 32 / LPR heads: they would
// otherwise cost twice the bytes of the data itself in L1.  Both kernels are bound by HBM: the
// forward reads and writes each element once, the backward reads x and g_out and writes dx.
#pragma once

#include "rope.cuh"

namespace mlxp {

// A lane's elements of one row: NC pieces of VEC elements of either half.  VEC elements are
// 16 bytes (NC = 1), or one element (LPR = 32, NC = 4: any even head_dim to 256, any alignment).
template <typename T_, int VEC_, int LPR_, int NC_>
struct RowShape {
  using T = T_;
  static constexpr int VEC = VEC_, LPR = LPR_, NC = NC_;
  static constexpr int NE = VEC * NC;  // elements of either half in a lane
  static constexpr int RPW = 32 / LPR; // rows a warp holds at a time
  static constexpr bool kWide = VEC * sizeof(T) == 16;
};

// Element index (within a half) of piece c of the lane with row index j.
template <typename R>
__device__ __forceinline__ int piece_at(int c, int j) {
  return (c * R::LPR + j) * R::VEC;
}

template <typename R>
struct RowData {  // as loaded: both halves
  alignas(16) typename R::T x1[R::NE];
  alignas(16) typename R::T x2[R::NE];
};

template <typename R>
__device__ __forceinline__ void row_load(const typename R::T* x, int half, int j, bool on,
                                         RowData<R>& d) {
  using T = typename R::T;
#pragma unroll
  for (int c = 0; c < R::NC; ++c) {
    const int at = piece_at<R>(c, j);
    const bool ok = on && at < half;
    if constexpr (R::kWide) {
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (ok) {
        a = *reinterpret_cast<const uint4*>(x + at);
        b = *reinterpret_cast<const uint4*>(x + half + at);
      }
      *reinterpret_cast<uint4*>(d.x1 + c * R::VEC) = a;
      *reinterpret_cast<uint4*>(d.x2 + c * R::VEC) = b;
    } else {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) {
        d.x1[c * R::VEC + e] = ok ? x[at + e] : from_f<T>(0.f);
        d.x2[c * R::VEC + e] = ok ? x[half + at + e] : from_f<T>(0.f);
      }
    }
  }
}

template <typename R>
__device__ __forceinline__ void row_store(typename R::T* y, int half, int j,
                                          const float (&a)[R::NE], const float (&b)[R::NE]) {
  using T = typename R::T;
#pragma unroll
  for (int c = 0; c < R::NC; ++c) {
    const int at = piece_at<R>(c, j);
    if (at >= half) continue;
    alignas(16) T o1[R::VEC], o2[R::VEC];
#pragma unroll
    for (int e = 0; e < R::VEC; ++e) {
      o1[e] = from_f<T>(a[c * R::VEC + e]);
      o2[e] = from_f<T>(b[c * R::VEC + e]);
    }
    if constexpr (R::kWide) {
      *reinterpret_cast<uint4*>(y + at) = *reinterpret_cast<const uint4*>(o1);
      *reinterpret_cast<uint4*>(y + half + at) = *reinterpret_cast<const uint4*>(o2);
    } else {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) {
        y[at + e] = o1[e];
        y[half + at + e] = o2[e];
      }
    }
  }
}

// VEC consecutive values of an fp32/bf16/fp16 array (dtype as the C ABI codes it) as floats.
// 16-byte aligned where VEC > 1.
template <int VEC>
__device__ __forceinline__ void load_f(const void* p, int dtype, long long at, float* out) {
  if (dtype == 0) {
    const float* f = static_cast<const float*>(p) + at;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(f) + i);
        out[4 * i] = v.x;
        out[4 * i + 1] = v.y;
        out[4 * i + 2] = v.z;
        out[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = __ldg(f + i);
    }
    return;
  }
  const unsigned short* u = static_cast<const unsigned short*>(p) + at;
  alignas(16) unsigned short s[VEC];
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint4*>(s) = __ldg(reinterpret_cast<const uint4*>(u));
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<uint2*>(s) = __ldg(reinterpret_cast<const uint2*>(u));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[i] = __ldg(u + i);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    out[i] = dtype == 1 ? __uint_as_float((unsigned)s[i] << 16) : __half2float(__ushort_as_half(s[i]));
}

// The lane's part of a table or weight row of `half` values (zeros past the end).
template <typename R>
__device__ __forceinline__ void half_load(const void* p, int dtype, long long base, int half, int j,
                                          float (&out)[R::NE]) {
#pragma unroll
  for (int c = 0; c < R::NC; ++c) {
    const int at = piece_at<R>(c, j);
    if (at < half) {
      load_f<R::VEC>(p, dtype, base + at, out + c * R::VEC);
    } else {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) out[c * R::VEC + e] = 0.f;
    }
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// What a token's rows share: its table row (identity without tables) and its weights.
template <typename R>
struct RowCoef {
  float c[R::NE], s[R::NE], w1[R::NE], w2[R::NE];
};

struct NormSpec {
  const void* w;     // nullable: no norm
  int w_dtype;
  float eps, inv_d;
};

template <typename R>
__device__ __forceinline__ void coef_weights(const NormSpec& n, int half, int j, RowCoef<R>& k) {
  if (!n.w) return;
  half_load<R>(n.w, n.w_dtype, 0, half, j, k.w1);
  half_load<R>(n.w, n.w_dtype, half, half, j, k.w2);
}

template <typename R>
__device__ __forceinline__ void coef_tables(const float* cosc, const float* sinc, long long pos,
                                            int half, int j, RowCoef<R>& k) {
  if (!cosc) return;
  half_load<R>(cosc, 0, pos * half, half, j, k.c);
  half_load<R>(sinc, 0, pos * half, half, j, k.s);
}

// Normed and rotated row, fp32.  Every lane of the warp takes part.
template <typename R>
__device__ __forceinline__ void row_norm_rope(const RowData<R>& d, const NormSpec& n, bool rotate,
                                              const RowCoef<R>& k, float (&y1)[R::NE],
                                              float (&y2)[R::NE]) {
  using T = typename R::T;
#pragma unroll
  for (int e = 0; e < R::NE; ++e) {
    y1[e] = to_f<T>(d.x1[e]);
    y2[e] = to_f<T>(d.x2[e]);
  }
  if (n.w) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < R::NE; ++e) ss = fmaf(y1[e], y1[e], fmaf(y2[e], y2[e], ss));
    const float r = rsqrtf(fmaf(row_sum<R::LPR>(ss), n.inv_d, n.eps));
#pragma unroll
    for (int e = 0; e < R::NE; ++e) {
      y1[e] = y1[e] * r * k.w1[e];
      y2[e] = y2[e] * r * k.w2[e];
    }
  }
  if (rotate) {
#pragma unroll
    for (int e = 0; e < R::NE; ++e) {
      float a, b;
      rope_pair(y1[e], y2[e], k.c[e], k.s[e], a, b);
      y1[e] = a;
      y2[e] = b;
    }
  }
}

template <int NE>
__device__ __forceinline__ void fill2(float v, float (&a)[NE], float (&b)[NE]) {
#pragma unroll
  for (int e = 0; e < NE; ++e) a[e] = b[e] = v;
}

struct NormRopeTensor {
  const void* x;
  const void* gy;                         // backward only
  void* y;                                // output (forward) or dx (backward)
  long long xs[3], gs[3], ys[3];          // element strides of (batch, head, seq)
  int H, S;
  int groups;                             // units a token: ceil(H / heads per unit)
  long long units;                        // tokens * groups
  long long offset;                       // position of sequence index 0 without `positions`
  NormSpec norm;
  float* dw_part;                         // backward: [grid][D]
};

struct NormRopeParams {
  NormRopeTensor t[2];
  int half;
  const float *cosc, *sinc;               // nullable (no rotation)
  long long n_pos;
  const int* positions;                   // nullable, int32
  long long pos_sb, pos_ss;
};

// Position of the unit's token and its addresses.
__device__ __forceinline__ long long unit_position(const NormRopeParams& p, const NormRopeTensor& t,
                                                   long long b, long long s) {
  return p.positions ? (long long)__ldg(p.positions + b * p.pos_sb + s * p.pos_ss) : t.offset + s;
}

template <typename R, int U>
__global__ void __launch_bounds__(256) norm_rope_kernel(const NormRopeParams p) {
  using T = typename R::T;
  const int lane = threadIdx.x & 31, j = lane % R::LPR, g = lane / R::LPR;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  const long long total = p.t[0].units + p.t[1].units;
  for (long long u = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < total;
       u += warps) {
    const int which = u >= p.t[0].units;
    const NormRopeTensor& t = p.t[which];
    const unsigned v = (unsigned)(which ? u - p.t[0].units : u);
    const unsigned tok = v / (unsigned)t.groups;
    const int h0 = (int)(v - tok * (unsigned)t.groups) * (R::RPW * U) + g;
    const unsigned b = tok / (unsigned)t.S;
    const int s = (int)(tok - b * (unsigned)t.S);
    const T* x = static_cast<const T*>(t.x) + b * t.xs[0] + s * t.xs[2];
    RowData<R> d[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = h0 + i * R::RPW;
      row_load<R>(x + h * t.xs[1], p.half, j, h < t.H, d[i]);
    }
    const long long pos = unit_position(p, t, b, s);
    const bool inside = pos >= 0 && (pos < p.n_pos || !p.cosc);
    RowCoef<R> k;
    coef_weights<R>(t.norm, p.half, j, k);
    coef_tables<R>(p.cosc, p.sinc, inside ? pos : 0, p.half, j, k);
    T* y = static_cast<T*>(t.y) + b * t.ys[0] + s * t.ys[2];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = h0 + i * R::RPW;
      float y1[R::NE], y2[R::NE];
      row_norm_rope<R>(d[i], t.norm, p.cosc != nullptr, k, y1, y2);
      if (!inside) fill2<R::NE>(pos < 0 ? 0.f : __int_as_float(0x7fffffff), y1, y2);
      if (h < t.H) row_store<R>(y + h * t.ys[1], p.half, j, y1, y2);
    }
  }
}

// dx of every row and, per CTA, the sum of g x r over its rows (dw_part[blockIdx.x], written by
// every CTA).  A CTA takes a strided set of units, so its sums and their order are fixed by the
// grid alone; norm_rope_dw_kernel adds the CTAs' parts in order.  The result has no atomics in
// it and is the same every time.
template <typename R, int U>
__global__ void __launch_bounds__(256) norm_rope_bwd_kernel(const NormRopeParams p) {
  using T = typename R::T;
  extern __shared__ float nr_sm[];  // [8 warps][D]
  const int lane = threadIdx.x & 31, j = lane % R::LPR, g = lane / R::LPR;
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int D = 2 * p.half;
  const long long warps = (long long)gridDim.x * nw;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const NormRopeTensor& t = p.t[which];
    if (t.units == 0 && !t.dw_part) continue;
    float a1[R::NE], a2[R::NE];
    fill2<R::NE>(0.f, a1, a2);
    RowCoef<R> k;
    coef_weights<R>(t.norm, p.half, j, k);
    for (long long u = (long long)blockIdx.x * nw + warp; u < t.units; u += warps) {
      const unsigned v = (unsigned)u;
      const unsigned tok = v / (unsigned)t.groups;
      const int h0 = (int)(v - tok * (unsigned)t.groups) * (R::RPW * U) + g;
      const unsigned b = tok / (unsigned)t.S;
      const int s = (int)(tok - b * (unsigned)t.S);
      const T* x = static_cast<const T*>(t.x) + b * t.xs[0] + s * t.xs[2];
      const T* gy = static_cast<const T*>(t.gy) + b * t.gs[0] + s * t.gs[2];
      RowData<R> d[U], q[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int h = h0 + i * R::RPW;
        row_load<R>(x + h * t.xs[1], p.half, j, h < t.H, d[i]);
        row_load<R>(gy + h * t.gs[1], p.half, j, h < t.H, q[i]);
      }
      const long long pos = unit_position(p, t, b, s);
      const bool inside = pos >= 0 && (pos < p.n_pos || !p.cosc);
      coef_tables<R>(p.cosc, p.sinc, inside ? pos : 0, p.half, j, k);
      T* y = static_cast<T*>(t.y) + b * t.ys[0] + s * t.ys[2];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int h = h0 + i * R::RPW;
        float x1[R::NE], x2[R::NE], g1[R::NE], g2[R::NE];
#pragma unroll
        for (int e = 0; e < R::NE; ++e) {
          x1[e] = to_f<T>(d[i].x1[e]);
          x2[e] = to_f<T>(d[i].x2[e]);
          g1[e] = to_f<T>(q[i].x1[e]);
          g2[e] = to_f<T>(q[i].x2[e]);
        }
        if (!inside) fill2<R::NE>(pos < 0 ? 0.f : __int_as_float(0x7fffffff), g1, g2);
        if (p.cosc) {
#pragma unroll
          for (int e = 0; e < R::NE; ++e) {
            float a, c;
            rope_pair(g1[e], g2[e], k.c[e], -k.s[e], a, c);
            g1[e] = a;
            g2[e] = c;
          }
        }
        if (t.norm.w) {
          float ss = 0.f, sg = 0.f;
#pragma unroll
          for (int e = 0; e < R::NE; ++e) {
            ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
            sg = fmaf(g1[e] * k.w1[e], x1[e], fmaf(g2[e] * k.w2[e], x2[e], sg));
          }
          ss = row_sum<R::LPR>(ss);
          sg = row_sum<R::LPR>(sg);
          const float r = rsqrtf(fmaf(ss, t.norm.inv_d, t.norm.eps));
          const float m = sg * t.norm.inv_d * r * r;
          // a padding row's x may hold anything: it must not reach dw or dx
          const bool use = h < t.H && pos >= 0;
#pragma unroll
          for (int e = 0; e < R::NE; ++e) {
            if (use) {
              a1[e] = fmaf(g1[e], x1[e] * r, a1[e]);
              a2[e] = fmaf(g2[e], x2[e] * r, a2[e]);
            }
            g1[e] = use ? r * (g1[e] * k.w1[e] - x1[e] * m) : 0.f;
            g2[e] = use ? r * (g2[e] * k.w2[e] - x2[e] * m) : 0.f;
          }
        }
        if (h < t.H) row_store<R>(y + h * t.ys[1], p.half, j, g1, g2);
      }
    }
    if (!t.dw_part) continue;
    // the row groups of a warp (lanes with the same j), then the warps
#pragma unroll
    for (int off = R::LPR; off < 32; off <<= 1)
#pragma unroll
      for (int e = 0; e < R::NE; ++e) {
        a1[e] += __shfl_xor_sync(0xffffffffu, a1[e], off);
        a2[e] += __shfl_xor_sync(0xffffffffu, a2[e], off);
      }
    if (g == 0) {
#pragma unroll
      for (int c = 0; c < R::NC; ++c) {
        const int at = piece_at<R>(c, j);
        if (at < p.half) {
#pragma unroll
          for (int e = 0; e < R::VEC; ++e) {
            nr_sm[warp * D + at + e] = a1[c * R::VEC + e];
            nr_sm[warp * D + p.half + at + e] = a2[c * R::VEC + e];
          }
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
      float v = 0.f;
      for (int w = 0; w < nw; ++w) v += nr_sm[w * D + i];
      t.dw_part[(long long)blockIdx.x * D + i] = v;
    }
    __syncthreads();
  }
}

// dw = sum over the CTAs' parts, 32 columns a block; blockIdx.y picks the tensor.
struct NormRopeDw {
  const float* part[2];
  void* dw[2];
  int dtype[2];
  int rows, D;
};

__global__ void __launch_bounds__(1024) norm_rope_dw_kernel(const NormRopeDw p) {
  __shared__ float sm[32][33];
  const int which = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x;
  const float* part = p.part[which];
  if (!part) return;
  float v = 0.f;
  if (col < p.D) {
#pragma unroll 4
    for (int r = threadIdx.y; r < p.rows; r += 32) v += part[(long long)r * p.D + col];
  }
  sm[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = sm[threadIdx.x][threadIdx.y];  // a warp now holds one column's 32 sums
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < p.D) {
    if (p.dtype[which] == 0) static_cast<float*>(p.dw[which])[c] = v;
    else if (p.dtype[which] == 1) static_cast<__nv_bfloat16*>(p.dw[which])[c] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p.dw[which])[c] = __float2half_rn(v);
  }
}

}  // namespace mlxp
