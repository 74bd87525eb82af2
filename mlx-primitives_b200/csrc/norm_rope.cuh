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
// step, and the loads of U steps are issued before the first is used.  A unit, one warp's work, is
// a token's heads (or U steps of them where there are few tokens): they share a position, so its
// table rows, which would cost twice the bytes of the data itself in L1, and the weights are
// loaded once.  Arithmetic is on pairs (fma.rn.f32x2).  Both kernels are bound by HBM: the
// forward reads and writes each element once, the backward reads x and g_out and writes dx.  2 x
// 16384 tokens of 32 + 32 heads of 128 in bf16: 183 us (5.9 TB/s, 90 % of a copy's rate) and 278
// (5.8 TB/s); units of rows rather than of tokens and scalar arithmetic took 811 together.
#pragma once

#include <type_traits>

#include "rope.cuh"
#include "sm100_ptx.cuh"

namespace mlxp {

// A lane's elements of one row: NC pieces of VEC elements of either half.  VEC elements are
// 16 bytes (NC = 1), or one element (LPR = 32, NC = 4: any even head_dim to 256, any alignment).
template <typename T_, int VEC_, int LPR_, int NC_>
struct RowShape {
  using T = T_;
  static constexpr int VEC = VEC_, LPR = LPR_, NC = NC_;
  static constexpr int NE = VEC * NC;  // elements of either half in a lane
  static constexpr int NP = NE / 2;    // in pairs, as the packed fp32 arithmetic takes them
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

// Element pairs as fp32 and back.
template <typename T>
__device__ __forceinline__ float2 pair_to_f(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(p[0], p[1]);
  } else {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    else
      return __half22float2(reinterpret_cast<const __half2&>(u));
  }
}
template <typename T>
__device__ __forceinline__ void pair_from_f(float2 v, T* p) {
  if constexpr (sizeof(T) == 4) {
    p[0] = v.x;
    p[1] = v.y;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
  } else {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(v.x, v.y);
  }
}

template <typename R>
__device__ __forceinline__ void row_to_f(const typename R::T* x, float2 (&f)[R::NP]) {
#pragma unroll
  for (int i = 0; i < R::NP; ++i) f[i] = pair_to_f<typename R::T>(x + 2 * i);
}

template <typename R>
__device__ __forceinline__ void row_store(typename R::T* y, int half, int j,
                                          const float2 (&a)[R::NP], const float2 (&b)[R::NP]) {
  using T = typename R::T;
  alignas(16) T o1[R::NE], o2[R::NE];
#pragma unroll
  for (int i = 0; i < R::NP; ++i) {
    pair_from_f<T>(a[i], o1 + 2 * i);
    pair_from_f<T>(b[i], o2 + 2 * i);
  }
#pragma unroll
  for (int c = 0; c < R::NC; ++c) {
    const int at = piece_at<R>(c, j);
    if (at >= half) continue;
    if constexpr (R::kWide) {
      *reinterpret_cast<uint4*>(y + at) = *reinterpret_cast<const uint4*>(o1);
      *reinterpret_cast<uint4*>(y + half + at) = *reinterpret_cast<const uint4*>(o2);
    } else {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) {
        y[at + e] = o1[c * R::VEC + e];
        y[half + at + e] = o2[c * R::VEC + e];
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
                                          float2 (&out)[R::NP]) {
  float f[R::NE];
#pragma unroll
  for (int c = 0; c < R::NC; ++c) {
    const int at = piece_at<R>(c, j);
    if (at < half) {
      load_f<R::VEC>(p, dtype, base + at, f + c * R::VEC);
    } else {
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) f[c * R::VEC + e] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < R::NP; ++i) out[i] = make_float2(f[2 * i], f[2 * i + 1]);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

template <int NP>
__device__ __forceinline__ void fill2(float v, float2 (&a)[NP], float2 (&b)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) a[i] = b[i] = make_float2(v, v);
}

// What a token's rows share: its table row and its weights.
template <typename R>
struct RowCoef {
  float2 c[R::NP], s[R::NP], w1[R::NP], w2[R::NP];
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

// The tables' row `pos`; the identity without tables.
template <typename R>
__device__ __forceinline__ void coef_tables(const float* cosc, const float* sinc, long long pos,
                                            int half, int j, RowCoef<R>& k) {
  if (cosc) {
    half_load<R>(cosc, 0, pos * half, half, j, k.c);
    half_load<R>(sinc, 0, pos * half, half, j, k.s);
  } else {
#pragma unroll
    for (int i = 0; i < R::NP; ++i) {
      k.c[i] = make_float2(1.f, 1.f);
      k.s[i] = make_float2(0.f, 0.f);
    }
  }
}

__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// Normed and rotated row, fp32.  Every lane of the warp takes part.  Without a norm the rotation
// rounds as rope_pair does (products, then their sum), so that it gives rope's bits.
template <typename R>
__device__ __forceinline__ void row_norm_rope(const RowData<R>& d, const NormSpec& n, bool rotate,
                                              const RowCoef<R>& k, float2 (&y1)[R::NP],
                                              float2 (&y2)[R::NP]) {
  using T = typename R::T;
  row_to_f<R>(d.x1, y1);
  row_to_f<R>(d.x2, y2);
  if (n.w) {
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < R::NP; ++i) ss = fma2(y1[i], y1[i], fma2(y2[i], y2[i], ss));
    const float2 r = both(rsqrtf(fmaf(row_sum<R::LPR>(ss.x + ss.y), n.inv_d, n.eps)));
#pragma unroll
    for (int i = 0; i < R::NP; ++i) {
      const float2 a = mul2(mul2(y1[i], r), k.w1[i]), b = mul2(mul2(y2[i], r), k.w2[i]);
      y1[i] = sub2(mul2(a, k.c[i]), mul2(b, k.s[i]));
      y2[i] = fma2(a, k.s[i], mul2(b, k.c[i]));
    }
  } else if (rotate) {
#pragma unroll
    for (int i = 0; i < R::NP; ++i) {
      const float2 a = y1[i], b = y2[i];
      y1[i] = sub2(mul2(a, k.c[i]), mul2(b, k.s[i]));
      y2[i] = add2(mul2(a, k.s[i]), mul2(b, k.c[i]));
    }
  }
}

struct NormRopeTensor {
  const void* x;
  const void* gy;                         // backward only
  void* y;                                // output (forward) or dx (backward)
  long long xs[3], gs[3], ys[3];          // element strides of (batch, head, seq)
  int H, S;
  int steps, groups;                      // row steps a unit, units a token
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

template <typename R, int U, int MINB>
__global__ void __launch_bounds__(256, MINB) norm_rope_kernel(const NormRopeParams p) {
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
    const int first = (int)(v - tok * (unsigned)t.groups) * t.steps * R::RPW;
    const int last = min(t.H, first + t.steps * R::RPW);
    const unsigned b = tok / (unsigned)t.S;
    const int s = (int)(tok - b * (unsigned)t.S);
    const T* x = static_cast<const T*>(t.x) + b * t.xs[0] + s * t.xs[2];
    T* y = static_cast<T*>(t.y) + b * t.ys[0] + s * t.ys[2];
    RowData<R> d[U];
    auto load = [&](int h0) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int h = h0 + i * R::RPW + g;
        row_load<R>(x + h * t.xs[1], p.half, j, h < last, d[i]);
      }
    };
    load(first);
    const long long pos = unit_position(p, t, b, s);
    RowCoef<R> k;
    coef_weights<R>(t.norm, p.half, j, k);
    const bool past = p.cosc && pos >= p.n_pos;
    coef_tables<R>(p.cosc, p.sinc, pos < 0 || past ? 0 : pos, p.half, j, k);
    if (past) fill2<R::NP>(__int_as_float(0x7fffffff), k.c, k.s);
    for (int h0 = first;;) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int h = h0 + i * R::RPW + g;
        float2 y1[R::NP], y2[R::NP];
        row_norm_rope<R>(d[i], t.norm, p.cosc != nullptr, k, y1, y2);
        if (pos < 0) fill2<R::NP>(0.f, y1, y2);
        if (h < last) row_store<R>(y + h * t.ys[1], p.half, j, y1, y2);
      }
      h0 += U * R::RPW;
      if (h0 >= last) break;
      load(h0);
    }
  }
}

// dx of every row and, per CTA, the sum of g x r over its rows (dw_part[blockIdx.x], written by
// every CTA).  A CTA takes a strided set of units, so its sums and their order are fixed by the
// grid alone; norm_rope_dw_kernel adds the CTAs' parts in order.  The result has no atomics in
// it and is the same every time.
template <typename R, int U, int MINB>
__global__ void __launch_bounds__(256, MINB) norm_rope_bwd_kernel(const NormRopeParams p) {
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
    float2 a1[R::NP], a2[R::NP];
    fill2<R::NP>(0.f, a1, a2);
    RowCoef<R> k;
    coef_weights<R>(t.norm, p.half, j, k);
    for (long long u = (long long)blockIdx.x * nw + warp; u < t.units; u += warps) {
      const unsigned v = (unsigned)u;
      const unsigned tok = v / (unsigned)t.groups;
      const int first = (int)(v - tok * (unsigned)t.groups) * t.steps * R::RPW;
      const int last = min(t.H, first + t.steps * R::RPW);
      const unsigned b = tok / (unsigned)t.S;
      const int s = (int)(tok - b * (unsigned)t.S);
      const T* x = static_cast<const T*>(t.x) + b * t.xs[0] + s * t.xs[2];
      const T* gy = static_cast<const T*>(t.gy) + b * t.gs[0] + s * t.gs[2];
      T* y = static_cast<T*>(t.y) + b * t.ys[0] + s * t.ys[2];
      RowData<R> d[U], q[U];
      auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int h = h0 + i * R::RPW + g;
          row_load<R>(x + h * t.xs[1], p.half, j, h < last, d[i]);
          row_load<R>(gy + h * t.gs[1], p.half, j, h < last, q[i]);
        }
      };
      load(first);
      const long long pos = unit_position(p, t, b, s);
      const bool past = p.cosc && pos >= p.n_pos;
      coef_tables<R>(p.cosc, p.sinc, pos < 0 || past ? 0 : pos, p.half, j, k);
      if (past) fill2<R::NP>(__int_as_float(0x7fffffff), k.c, k.s);
      for (int h0 = first;;) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int h = h0 + i * R::RPW + g;
          float2 x1[R::NP], x2[R::NP], g1[R::NP], g2[R::NP];
          row_to_f<R>(q[i].x1, g1);
          row_to_f<R>(q[i].x2, g2);
#pragma unroll
          for (int e = 0; e < R::NP; ++e) {
            const float2 u = g1[e];
            g1[e] = fma2(u, k.c[e], mul2(g2[e], k.s[e]));
            g2[e] = sub2(mul2(g2[e], k.c[e]), mul2(u, k.s[e]));
          }
          if (t.norm.w) {
            row_to_f<R>(d[i].x1, x1);
            row_to_f<R>(d[i].x2, x2);
            float2 ss = both(0.f), sg = ss;
#pragma unroll
            for (int e = 0; e < R::NP; ++e) {
              ss = fma2(x1[e], x1[e], fma2(x2[e], x2[e], ss));
              sg = fma2(mul2(g1[e], k.w1[e]), x1[e], fma2(mul2(g2[e], k.w2[e]), x2[e], sg));
            }
            const float sum = row_sum<R::LPR>(ss.x + ss.y), dot = row_sum<R::LPR>(sg.x + sg.y);
            const float r1 = rsqrtf(fmaf(sum, t.norm.inv_d, t.norm.eps));
            const float2 r = both(r1), m = both(-dot * t.norm.inv_d * r1 * r1);
            // a padding row's x may hold anything, and a lane without a row has r = inf where eps
            // is 0: neither must reach dw
            if (pos >= 0 && h < last) {
#pragma unroll
              for (int e = 0; e < R::NP; ++e) {
                const float2 u = mul2(x1[e], r), z = mul2(x2[e], r);
                a1[e] = fma2(g1[e], u, a1[e]);
                a2[e] = fma2(g2[e], z, a2[e]);
                g1[e] = fma2(u, m, mul2(mul2(g1[e], k.w1[e]), r));
                g2[e] = fma2(z, m, mul2(mul2(g2[e], k.w2[e]), r));
              }
            }
          }
          if (pos < 0) fill2<R::NP>(0.f, g1, g2);
          if (h < last) row_store<R>(y + h * t.ys[1], p.half, j, g1, g2);
        }
        h0 += U * R::RPW;
        if (h0 >= last) break;
        load(h0);
      }
    }
    if (!t.dw_part) continue;
    // the row groups of a warp (lanes with the same j), then the warps
    float f1[R::NE], f2[R::NE];
#pragma unroll
    for (int e = 0; e < R::NE; ++e) {
      f1[e] = e & 1 ? a1[e / 2].y : a1[e / 2].x;
      f2[e] = e & 1 ? a2[e / 2].y : a2[e / 2].x;
#pragma unroll
      for (int off = R::LPR; off < 32; off <<= 1) {
        f1[e] += __shfl_xor_sync(0xffffffffu, f1[e], off);
        f2[e] += __shfl_xor_sync(0xffffffffu, f2[e], off);
      }
    }
    if (g == 0) {
#pragma unroll
      for (int c = 0; c < R::NC; ++c) {
        const int at = piece_at<R>(c, j);
        if (at < p.half) {
#pragma unroll
          for (int e = 0; e < R::VEC; ++e) {
            nr_sm[warp * D + at + e] = f1[c * R::VEC + e];
            nr_sm[warp * D + p.half + at + e] = f2[c * R::VEC + e];
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
  const bool second = blockIdx.y != 0;
  const int col = blockIdx.x * 32 + threadIdx.x;
  const float* part = second ? p.part[1] : p.part[0];
  if (!part) return;
  float v = 0.f;
  if (col < p.D) {
#pragma unroll 8
    for (int r = threadIdx.y; r < p.rows; r += 32) v += part[(long long)r * p.D + col];
  }
  sm[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = sm[threadIdx.x][threadIdx.y];  // a warp now holds one column's 32 sums
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < p.D) {
    void* dw = second ? p.dw[1] : p.dw[0];
    const int dtype = second ? p.dtype[1] : p.dtype[0];
    if (dtype == 0) static_cast<float*>(dw)[c] = v;
    else if (dtype == 1) static_cast<__nv_bfloat16*>(dw)[c] = __float2bfloat16_rn(v);
    else static_cast<__half*>(dw)[c] = __float2half_rn(v);
  }
}

}  // namespace mlxp
