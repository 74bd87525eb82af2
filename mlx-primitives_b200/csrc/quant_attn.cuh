// quant_attn.cuh — attention over a paged K/V cache held in 8 bits (e4m3 or int8 codes and one
// fp32 scale a block and head), read in place and split over keys.
//
// For query i of sequence b (G = H / Hk query heads share a pool head; qlen queries, the
// sequence's last positions: pos = context_lens[b] - qlen + i),
//   s_t = scale * ks_t (q . K8_t) + slope (t - pos),   O = sum_t e^{s_t} vs_t V8_t / sum_t e^{s_t}
// over the keys t < context_lens[b] whose table entry is in [0, num_blocks), with t <= pos when
// causal and within the window; a row with no such key is zero.
//
// What bounds it.  A decode step reads every code once, 2 D bytes a key and pool head, against
// 4 G D flops: HBM.  CUDA cores could not convert and multiply-add G times at that rate (24 bytes
// a cycle and SM), so both products run on mma.sync m16n8k16 with fp16 operands and fp32 sums:
// codes are exact in fp16.  The 16 keys of a tile are the M rows, S^T = K8 Q^T with up to 8 query
// rows as N, and O^T += V8^T P^T; the query rows being N = 8 wide halves the matrix work against
// query rows as M = 16.  (tcgen05 needs M >= 64 rows and its operands in shared memory or TMEM,
// which one query row cannot fill.)
//
// No shared memory on the way.  The order of a dot product's terms is free, so the fragment
// layouts are chosen such that the bytes a lane loads are the bytes its fragments need: of a K
// row the four lanes c of a row group hold 16-byte pieces c and, for D = 128, 4 + c, each word of
// which is one k16 step's two pairs; of a V row the eight lanes g hold D / 8 bytes each, and a
// byte permute of two keys' words gives the pairs along keys.  A warp loads the next tile into
// registers while it computes on this one.
//
// Precision.  16-bit queries are scaled by a power of two a row to [1, 2) at most and held in
// fp16 (bf16 values lose nothing but below 2^-25 of the row's largest); fp32 queries and
// probabilities are split into two fp16 terms, which keeps 22 bits.  The running maximum m is of
// s_t + log2 |vs_t|, so that the weights p_t vs_t 2^15 that multiply V8 fit fp16 whatever the
// scales, with 29 octaves below the largest at full precision; m and the sums are fp32.  |vs_t|
// is taken as within [2^-100, 2^100] there.
//
// Work split.  A virtual sequence is a sequence and a tile of 8 NT of its G * Sq query rows; it
// has Hk / HP units, HP heads each: the warps of a CTA take HP heads (reading neighbouring bytes
// of the pool's rows) times 4 / HP interleaved key tiles.  All units' chunks of 64 keys, in
// order, are cut into equal contiguous ranges, one a CTA: every SM gets the same number of chunks
// however uneven the contexts are.  Each CTA finds its range from context_lens (no host copy).
// A unit that one CTA covers is written directly; otherwise the CTAs write fp32 partials and a
// second small kernel merges them, launched early (programmatic dependent launch) so that its
// start-up hides behind the first.  A merge by the last CTA to finish would need zeroed counters,
// i.e. a memset in the same place, and one CTA would merge alone what hundreds wrote.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "rope.cuh"
#include "sm100_ptx.cuh"

namespace mlxp {

constexpr int kQaWarps = 4;
constexpr int kQaChunk = 64;   // keys a chunk
constexpr int kQaTile = 16;    // keys a tile
constexpr float kQaPScale = 32768.f;

struct QaPartInfo {  // written by every CTA: the unit its range starts inside of
  int v, hg;         // v = -1: it starts at a unit's first chunk (or has no chunks)
  int first;         // 2 * (first CTA of the unit) + that CTA's slot
  int parts;
};

struct QaParams {
  const void* q;
  const unsigned char *k_pool, *v_pool;
  const float *k_scales, *v_scales;
  const int* block_tables;
  const int* context_lens;
  const int* query_lens;          // nullable: Sq
  const float* alibi;             // nullable, [H]
  void* o;
  float* o_part;                  // [CTA][2][HP][rows][D]
  float* ml_part;                 // [CTA][2][HP][rows][2]
  QaPartInfo* info;               // [CTA]
  long long q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;
  long long p_sb, p_st, p_sh;     // bytes
  long long sc_sb, sc_sh;
  long long bt_stride;
  int B, H, Hk, G, Sq, R;         // R = G * Sq query rows a (sequence, pool head)
  int rows;                       // rows of a tile that exist anywhere: min(R, 8 NT)
  int RT, HP, HG;                 // row tiles, heads a unit, units a virtual sequence
  int num_blocks, block_size, max_blocks;
  int causal;
  long long window;               // -1: none
  float scale_log2;
};

// Keys of a virtual sequence.
struct QaRange {
  long long ctx;
  int klo, khi;      // keys some row sees: [klo, khi)
  int flo, fhi;      // keys every row sees: [flo, fhi)
  int c0, n;         // first chunk, chunks (at least 1: an empty unit writes its zeros)
  int qlen;
};

// Keys [lo, hi) that query i sees (empty: hi <= lo).  Both rise with i.
__device__ __forceinline__ void qa_row_range(const QaParams& p, long long ctx, int qlen, int i,
                                             int& lo, int& hi) {
  const long long pos = ctx - qlen + i;
  const long long cap = (long long)p.max_blocks * p.block_size;
  long long h = ctx < cap ? ctx : cap, l = 0;
  if (p.causal) h = min(h, pos + 1);
  else if (p.window >= 0) h = min(h, pos + p.window + 1);
  if (p.window >= 0) l = max(l, pos - p.window);
  lo = (int)l;
  hi = (int)max(h, 0LL);
}

template <int NT>
__device__ __forceinline__ QaRange qa_range(const QaParams& p, int v) {
  QaRange r;
  const int b = v / p.RT, rt = v - b * p.RT;
  r.ctx = __ldg(p.context_lens + b);
  r.qlen = p.query_lens ? max(0, min(__ldg(p.query_lens + b), p.Sq)) : p.Sq;
  const int i0 = rt * 8 * NT / p.G;
  const int i1 = min((min(p.R, (rt + 1) * 8 * NT) - 1) / p.G, r.qlen - 1);
  r.klo = r.khi = r.flo = r.fhi = 0;
  if (i0 <= i1) {
    int l0, h0, l1, h1;
    qa_row_range(p, r.ctx, r.qlen, i0, l0, h0);
    qa_row_range(p, r.ctx, r.qlen, i1, l1, h1);
    if (h1 > l0) {
      r.klo = l0;
      r.khi = h1;
      r.flo = l1;  // flo >= fhi where a row sees nothing: every tile is then masked
      r.fhi = h0;
    }
  }
  r.c0 = r.klo / kQaChunk;
  r.n = max(1, (r.khi + kQaChunk - 1) / kQaChunk - r.c0);
  return r;
}

__device__ __forceinline__ void qa_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t qa_transpose(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Two codes (the low or high half of a word) as fp16 pairs.
template <bool INT8>
__device__ __forceinline__ void qa_codes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {
    // u = code + 128 in 0..255; 0x6400 | u is the fp16 1024 + u
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1024 + 128
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(reinterpret_cast<const __half2&>(a), off);
    const __half2 y = __hsub2(reinterpret_cast<const __half2&>(b), off);
    lo = reinterpret_cast<const uint32_t&>(x);
    hi = reinterpret_cast<const uint32_t&>(y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

__device__ __forceinline__ uint32_t qa_pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ float2 qa_unpack(uint32_t u) {
  return __half22float2(reinterpret_cast<const __half2&>(u));
}

template <int W>
__device__ __forceinline__ void qa_ldg(const unsigned char* p, bool on, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = 0;
  if (!on) return;
  if constexpr (W % 4 == 0) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = u.x;
      w[4 * i + 1] = u.y;
      w[4 * i + 2] = u.z;
      w[4 * i + 3] = u.w;
    }
  } else if constexpr (W == 2) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = u.x;
    w[1] = u.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const unsigned*>(p));
  }
}

// Elements of a K row held by lane c as 4-byte words: words j < D/16, dims qa_kdim(j, c)..+3.
template <int D>
__device__ __forceinline__ int qa_kdim(int j, int c) {
  if constexpr (D == 32) return 8 * c + 4 * j;
  return (j / 4) * 64 + 16 * c + 4 * (j % 4);
}

template <int D>
struct QaTile {
  static constexpr int KW = D / 16, VW = D / 32;
  uint32_t k[2][KW];     // rows g, g + 8
  uint32_t v[4][VW];     // keys 2c, 2c + 1, 2c + 8, 2c + 9; bytes [g * D / 8, +D / 8)
  float ks0, ks1, vs0, vs1;  // scales of rows g, g + 8
  int t0;
  bool ok0, ok1;         // rows g, g + 8 are keys in a pool block
};

// BS16: the block size is a multiple of 16, so that a tile lies in one block.
template <int D, bool BS16>
__device__ __forceinline__ void qa_load(const QaParams& p, const int* bt, long long head_off,
                                        long long head_sc, int t0, int kend, int g, int c,
                                        QaTile<D>& t) {
  constexpr int KW = QaTile<D>::KW, VW = QaTile<D>::VW;
  t.t0 = t0;
  auto locate = [&](int key, bool in, int& id, long long& off) {
    id = -1;
    off = 0;
    if (!in) return;
    const unsigned slot = (unsigned)key / (unsigned)p.block_size;
    const int got = __ldg(bt + slot);
    if (got >= 0 && got < p.num_blocks) {
      id = got;
      off = (long long)got * p.p_sb + (long long)(key - (int)slot * p.block_size) * p.p_st + head_off;
    }
  };
  int id0, id1;
  long long o0, o1, ov[4];
  bool okv[4];
  if constexpr (BS16) {
    locate(t0, t0 < kend, id0, o0);
    id1 = id0;
    t.ok0 = id0 >= 0 && t0 + g < kend;
    t.ok1 = id0 >= 0 && t0 + g + 8 < kend;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 2 * c + (e & 1) + (e >> 1) * 8;
      okv[e] = id0 >= 0 && t0 + r < kend;
      ov[e] = o0 + r * p.p_st;
    }
    o1 = o0 + (g + 8) * p.p_st;
    o0 += g * p.p_st;
  } else {
    locate(t0 + g, t0 + g < kend, id0, o0);
    locate(t0 + g + 8, t0 + g + 8 < kend, id1, o1);
    t.ok0 = id0 >= 0;
    t.ok1 = id1 >= 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = t0 + 2 * c + (e & 1) + (e >> 1) * 8;
      int id;
      locate(r, r < kend, id, ov[e]);
      okv[e] = id >= 0;
    }
  }
  if constexpr (D == 128) {
    qa_ldg<4>(p.k_pool + o0 + 16 * c, t.ok0, t.k[0]);
    qa_ldg<4>(p.k_pool + o0 + 64 + 16 * c, t.ok0, t.k[0] + 4);
    qa_ldg<4>(p.k_pool + o1 + 16 * c, t.ok1, t.k[1]);
    qa_ldg<4>(p.k_pool + o1 + 64 + 16 * c, t.ok1, t.k[1] + 4);
  } else {
    qa_ldg<KW>(p.k_pool + o0 + 4 * KW * c, t.ok0, t.k[0]);
    qa_ldg<KW>(p.k_pool + o1 + 4 * KW * c, t.ok1, t.k[1]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) qa_ldg<VW>(p.v_pool + ov[e] + g * (D / 8), okv[e], t.v[e]);
  t.ks0 = t.ok0 ? __ldg(p.k_scales + id0 * p.sc_sb + head_sc) : 0.f;
  t.ks1 = t.ok1 ? __ldg(p.k_scales + id1 * p.sc_sb + head_sc) : 0.f;
  t.vs0 = t.ok0 ? __ldg(p.v_scales + id0 * p.sc_sb + head_sc) : 0.f;
  t.vs1 = t.ok1 ? __ldg(p.v_scales + id1 * p.sc_sb + head_sc) : 0.f;
}

// The state of a warp's rows: lane (g, c) holds query rows 2c, 2c + 1 of each n-tile.
template <int D, int NT>
struct QaState {
  float acc[NT][D / 16][4];  // dims g * D/8 + 2t (0: row 2c, 1: row 2c + 1) and + 2t + 1 (2, 3)
  float m[NT][2], l[NT][2];  // l: this lane's keys only, until the end
};

template <int D, int NT, bool SPLIT, bool INT8>
__device__ __forceinline__ void qa_step(const QaTile<D>& t, const uint32_t (&qf)[SPLIT ? 2 : 1][NT][D / 16][2],
                                        const float (&qs)[NT][2], const int* row_lo,
                                        const int* row_hi, const float* row_slope,
                                        const int* row_pos, bool masked, int g, int c,
                                        QaState<D, NT>& st) {
  constexpr int KW = D / 16, VW = D / 32;
  float sa[NT][4], sb[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) sa[n][e] = sb[n][e] = 0.f;
#pragma unroll
  for (int j = 0; j < KW; ++j) {
    uint32_t a0, a1, a2, a3;
    qa_codes<INT8>(t.k[0][j], a0, a2);
    qa_codes<INT8>(t.k[1][j], a1, a3);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      qa_mma(j & 1 ? sb[n] : sa[n], a0, a1, a2, a3, qf[0][n][j][0], qf[0][n][j][1]);
      if constexpr (SPLIT) qa_mma(j & 1 ? sa[n] : sb[n], a0, a1, a2, a3, qf[1][n][j][0], qf[1][n][j][1]);
    }
  }
  const float lv0 = fminf(fmaxf(__log2f(fabsf(t.vs0)), -100.f), 100.f);
  const float lv1 = fminf(fmaxf(__log2f(fabsf(t.vs1)), -100.f), 100.f);
  bool grow = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = n * 8 + 2 * c + (e & 1);
      float s = (sa[n][e] + sb[n][e]) * (qs[n][e & 1] * (e < 2 ? t.ks0 : t.ks1));
      const int key = t.t0 + g + (e < 2 ? 0 : 8);
      if (row_slope) s = fmaf(row_slope[row], (float)(key - row_pos[row]), s);
      bool ok = e < 2 ? t.ok0 : t.ok1;
      if (masked) ok = ok && key >= row_lo[row] && key < row_hi[row];
      sa[n][e] = ok ? s : -INFINITY;
      grow = grow || sa[n][e] + (e < 2 ? lv0 : lv1) > st.m[n][e & 1];
    }
  }
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float mx = fmaxf(sa[n][q] + lv0, sa[n][q + 2] + lv1);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        mx = fmaxf(mx, st.m[n][q]);
        const float alpha = ex2_approx(st.m[n][q] - mx);
        st.m[n][q] = mx;
        st.l[n][q] *= alpha;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          st.acc[n][d][q] *= alpha;
          st.acc[n][d][q + 2] *= alpha;
        }
      }
  }
  uint32_t pf[SPLIT ? 2 : 1][NT][2];
  const float v0 = t.vs0 * kQaPScale, v1 = t.vs1 * kQaPScale;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float pe = ex2_approx(sa[n][e] - st.m[n][e & 1]);
      st.l[n][e & 1] += pe;
      // a masked key's scale may be anything
      w[e] = sa[n][e] == -INFINITY ? 0.f : pe * (e < 2 ? v0 : v1);
    }
    const uint32_t h0 = qa_pack(w[0], w[1]), h1 = qa_pack(w[2], w[3]);
    pf[0][n][0] = qa_transpose(h0);
    pf[0][n][1] = qa_transpose(h1);
    if constexpr (SPLIT) {
      const float2 f0 = qa_unpack(h0), f1 = qa_unpack(h1);
      pf[1][n][0] = qa_transpose(qa_pack(w[0] - f0.x, w[1] - f0.y));
      pf[1][n][1] = qa_transpose(qa_pack(w[2] - f1.x, w[3] - f1.y));
    }
  }
#pragma unroll
  for (int w = 0; w < VW; ++w) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint32_t sel = hf ? 0x7362u : 0x5140u;
      uint32_t a0, a1, a2, a3;
      qa_codes<INT8>(__byte_perm(t.v[0][w], t.v[1][w], sel), a0, a1);
      qa_codes<INT8>(__byte_perm(t.v[2][w], t.v[3][w], sel), a2, a3);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        qa_mma(st.acc[n][2 * w + hf], a0, a1, a2, a3, pf[0][n][0], pf[0][n][1]);
        if constexpr (SPLIT) qa_mma(st.acc[n][2 * w + hf], a0, a1, a2, a3, pf[1][n][0], pf[1][n][1]);
      }
    }
  }
}

// Query rows of a head as B fragments, and the factor of each of the lane's score columns.
template <typename T, int D, int NT, bool SPLIT>
__device__ __forceinline__ void qa_load_q(const QaParams& p, int b, int r0, int hk, int g, int c,
                                          uint32_t (&qf)[SPLIT ? 2 : 1][NT][D / 16][2],
                                          float (&qs)[NT][2]) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + n * 8 + g;
    float x[D / 4];  // the lane's words' dims, four each
    float mx = 0.f;
    const int i = r / p.G, h = hk * p.G + r - i * p.G;
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh + i * p.q_ss;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const int d = qa_kdim<D>(j, c);
      if constexpr (sizeof(T) == 4) {
        const float4 u = r < p.R ? *reinterpret_cast<const float4*>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[4 * j] = u.x;
        x[4 * j + 1] = u.y;
        x[4 * j + 2] = u.z;
        x[4 * j + 3] = u.w;
      } else {
        const uint2 u = r < p.R ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
        const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * j + e] = to_f<T>(t[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[4 * j + e]));
    }
    float up = 1.f;  // 2^e, the row's factor
    if constexpr (sizeof(T) == 4 || std::is_same<T, __nv_bfloat16>::value) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const unsigned E = __float_as_uint(mx) >> 23;
      if (E >= 1 && E <= 253) up = __uint_as_float(E << 23);
      const float down = __uint_as_float((254u - (__float_as_uint(up) >> 23)) << 23);
#pragma unroll
      for (int e = 0; e < D / 4; ++e) x[e] *= down;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float a = x[4 * j + 2 * e], bb = x[4 * j + 2 * e + 1];
        qf[0][n][j][e] = qa_pack(a, bb);
        if constexpr (SPLIT) {
          const float2 f = qa_unpack(qf[0][n][j][e]);
          qf[1][n][j][e] = qa_pack(a - f.x, bb - f.y);
        }
      }
    // columns 2c, 2c + 1 are the rows of lanes g = 2c, 2c + 1
    qs[n][0] = __shfl_sync(0xffffffffu, up, 8 * c) * p.scale_log2;
    qs[n][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4) * p.scale_log2;
  }
}

template <typename T>
__device__ __forceinline__ void qa_store2(T* p, float a, float b) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float2*>(p) = make_float2(a, b);
  } else {
    alignas(4) T v[2] = {from_f<T>(a), from_f<T>(b)};
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(v);
  }
}

// CTA whose range [c * total / grid, (c + 1) * total / grid) holds chunk f.
__device__ __forceinline__ int qa_cta_of(long long f, long long total, int grid) {
  return (int)(((f + 1) * grid - 1) / total);
}

template <typename T, int D, int NT, bool INT8, bool BS16, int MINB>
__global__ void __launch_bounds__(32 * kQaWarps, MINB) quant_attn_kernel(const QaParams p) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int ROWS = 8 * NT;
  constexpr int RED = D + 4;  // floats a row in the warps' merge: acc, m, l
  __shared__ int s_lo[ROWS], s_hi[ROWS], s_pos[ROWS];
  __shared__ float s_slope[4][ROWS];
  __shared__ long long s_sum[kQaWarps];
  __shared__ int s_v;
  __shared__ long long s_rem;
  __shared__ __align__(16) float s_red[kQaWarps][ROWS][RED];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int HP = p.HP, KS = kQaWarps / HP;
  const int hp = warp % HP, kidx = warp / HP;
  const int V = p.B * p.RT;

  // this CTA's range: total chunks, then the virtual sequence its first chunk falls in
  const int per = (V + 32 * kQaWarps - 1) / (32 * kQaWarps);
  const int va = min(V, (int)threadIdx.x * per), vb = min(V, va + per);
  long long mine = 0;
  for (int v = va; v < vb; ++v) mine += (long long)qa_range<NT>(p, v).n * p.HG;
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += x;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  long long total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < kQaWarps; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  // no more CTAs than chunks: every working CTA then has some, and a unit's CTAs are consecutive
  const int grid = (int)min((long long)gridDim.x, total);
  long long f = (long long)blockIdx.x * total / grid;
  const long long f_end = ((long long)blockIdx.x + 1) * total / grid;
  if ((int)blockIdx.x >= grid) {
    if (threadIdx.x == 0) p.info[blockIdx.x] = QaPartInfo{-1, 0, 0, 0};
    return;
  }
  if (f >= before && f < before + mine) {
    long long at = before;
    int v = va;
    for (; v < vb; ++v) {
      const long long n = (long long)qa_range<NT>(p, v).n * p.HG;
      if (f < at + n) break;
      at += n;
    }
    s_v = v;
    s_rem = f - at;
  }
  __syncthreads();
  int v = s_v;
  long long rem = s_rem;
  const long long f_begin = f;
  while (f < f_end) {
    const QaRange r = qa_range<NT>(p, v);
    const int b = v / p.RT, r0 = (v - b * p.RT) * ROWS;
    const int hg = (int)(rem / r.n), ch0 = (int)(rem - (long long)hg * r.n);
    const int ch1 = (int)min((long long)r.n, ch0 + (f_end - f));
    if (f == f_begin && threadIdx.x == 0) {
      QaPartInfo info{-1, 0, 0, 0};
      if (ch0 > 0) {
        const long long u0 = f - ch0;  // the unit's first chunk
        const int first = qa_cta_of(u0, total, grid);
        const int last = qa_cta_of(u0 + r.n - 1, total, grid);
        const int slot = (long long)first * total / grid == u0 ? 0 : 1;
        info = QaPartInfo{v, hg, 2 * first + slot, last - first + 1};
      }
      p.info[blockIdx.x] = info;
    }
    __syncthreads();  // the last unit's reads of the row tables and s_red are done
    if (threadIdx.x < ROWS) {
      const int row = r0 + threadIdx.x, i = row / p.G;
      int lo = 0, hi = 0;
      if (row < p.R && i < r.qlen) qa_row_range(p, r.ctx, r.qlen, i, lo, hi);
      s_lo[threadIdx.x] = lo;
      s_hi[threadIdx.x] = hi;
      s_pos[threadIdx.x] = (int)(r.ctx - r.qlen + i);
    }
    if (p.alibi && threadIdx.x < HP * ROWS) {
      const int w = threadIdx.x / ROWS, row = r0 + threadIdx.x % ROWS;
      s_slope[w][threadIdx.x % ROWS] =
          row < p.R ? __ldg(p.alibi + (hg * HP + w) * p.G + row % p.G) * 1.4426950408889634f : 0.f;
    }
    __syncthreads();
    const int hk = hg * HP + hp;
    uint32_t qf[SPLIT ? 2 : 1][NT][D / 16][2];
    float qs[NT][2];
    qa_load_q<T, D, NT, SPLIT>(p, b, r0, hk, g, c, qf, qs);
    QaState<D, NT> st;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        st.m[n][e] = -1e30f;  // "no key yet", finite
        st.l[n][e] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.acc[n][d][e] = 0.f;
    }
    const int k0 = max((r.c0 + ch0) * kQaChunk, r.klo & ~(kQaTile - 1));
    const int k1 = min((long long)(r.c0 + ch1) * kQaChunk, (long long)r.khi);
    const int* bt = p.block_tables + (long long)b * p.bt_stride;
    const long long head_off = hk * p.p_sh, head_sc = hk * p.sc_sh;
    const float* slope = p.alibi ? s_slope[hp] : nullptr;
    const int step = kQaTile * KS;
    int t0 = k0 + kidx * kQaTile;
    QaTile<D> ta, tb;
    if (t0 < k1) qa_load<D, BS16>(p, bt, head_off, head_sc, t0, k1, g, c, ta);
    while (t0 < k1) {
      if (t0 + step < k1) qa_load<D, BS16>(p, bt, head_off, head_sc, t0 + step, k1, g, c, tb);
      qa_step<D, NT, SPLIT, INT8>(ta, qf, qs, s_lo, s_hi, slope, s_pos,
                                  t0 < r.flo || t0 + kQaTile > r.fhi, g, c, st);
      t0 += step;
      if (t0 >= k1) break;
      if (t0 + step < k1) qa_load<D, BS16>(p, bt, head_off, head_sc, t0 + step, k1, g, c, ta);
      qa_step<D, NT, SPLIT, INT8>(tb, qf, qs, s_lo, s_hi, slope, s_pos,
                                  t0 < r.flo || t0 + kQaTile > r.fhi, g, c, st);
      t0 += step;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
          st.l[n][e] += __shfl_xor_sync(0xffffffffu, st.l[n][e], off);

    const bool whole = ch0 == 0 && ch1 == r.n;
    const long long slot = 2LL * blockIdx.x + (f == f_begin ? 0 : 1);
    if (KS == 1) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tr = n * 8 + 2 * c + e, row = r0 + tr;
          if (row >= p.R) continue;
          if (whole) {
            const int i = row / p.G, h = hk * p.G + row - i * p.G;
            const bool some = st.l[n][e] != 0.f && i < r.qlen;
            const float inv = 1.f / (st.l[n][e] * kQaPScale);
            T* o = static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + i * p.o_ss + g * (D / 8);
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
              qa_store2<T>(o + 2 * d, some ? st.acc[n][d][e] * inv : 0.f,
                           some ? st.acc[n][d][e + 2] * inv : 0.f);
          } else {
            const long long pr = (slot * HP + hp) * p.rows + tr;
            float* o = p.o_part + pr * D + g * (D / 8);
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
              *reinterpret_cast<float2*>(o + 2 * d) = make_float2(st.acc[n][d][e], st.acc[n][d][e + 2]);
            if (g == 0) *reinterpret_cast<float2*>(p.ml_part + 2 * pr) = make_float2(st.m[n][e], st.l[n][e]);
          }
        }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* row = s_red[warp][n * 8 + 2 * c + e];
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            *reinterpret_cast<float2*>(row + g * (D / 8) + 2 * d) =
                make_float2(st.acc[n][d][e], st.acc[n][d][e + 2]);
          if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(st.m[n][e], st.l[n][e]);
        }
      __syncthreads();
      for (int x = threadIdx.x; x < HP * p.rows * (D / 2); x += blockDim.x) {
        const int d = 2 * (x % (D / 2)), y = x / (D / 2), tr = y % p.rows, w = y / p.rows;
        const int row = r0 + tr;
        if (row >= p.R) continue;
        float m = -1e30f;
        for (int k = 0; k < KS; ++k) m = fmaxf(m, s_red[w + k * HP][tr][D]);
        float l = 0.f, a = 0.f, bb = 0.f;
        for (int k = 0; k < KS; ++k) {
          const float* s = s_red[w + k * HP][tr];
          const float wt = ex2_approx(s[D] - m);
          l = fmaf(s[D + 1], wt, l);
          a = fmaf(s[d], wt, a);
          bb = fmaf(s[d + 1], wt, bb);
        }
        if (whole) {
          const int i = row / p.G, h = (hg * HP + w) * p.G + row - i * p.G;
          const bool some = l != 0.f && i < r.qlen;
          const float inv = 1.f / (l * kQaPScale);
          qa_store2<T>(static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + i * p.o_ss + d,
                       some ? a * inv : 0.f, some ? bb * inv : 0.f);
        } else {
          const long long pr = (slot * HP + w) * p.rows + tr;
          *reinterpret_cast<float2*>(p.o_part + pr * D + d) = make_float2(a, bb);
          if (d == 0) *reinterpret_cast<float2*>(p.ml_part + 2 * pr) = make_float2(m, l);
        }
      }
    }
    f += ch1 - ch0;
    rem += ch1 - ch0;
    if (rem >= (long long)r.n * p.HG) {
      rem = 0;
      ++v;
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Merges the partials of the units that more than one CTA worked on.  Block x looks at main CTA
// x + 1: where that is the second CTA of a unit, it merges the unit's rows blockIdx.y, +gridDim.y...
constexpr int kQaMergeWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kQaMergeWarps) quant_attn_merge_kernel(const QaParams p) {
  constexpr int LPR = D / 4, PPW = 32 / LPR;  // lanes a row, partials a warp at a time
  __shared__ float s_m[kQaMergeWarps], s_l[kQaMergeWarps];
  __shared__ __align__(16) float s_o[kQaMergeWarps][D];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cta = blockIdx.x + 1;
  const QaPartInfo info = p.info[cta];
  if (info.v < 0 || (info.first >> 1) != cta - 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR, d = (lane % LPR) * 4;
  const int b = info.v / p.RT, r0 = (info.v - b * p.RT) * p.rows;
  const int qlen = p.query_lens ? p.query_lens[b] : p.Sq;
  for (int y = blockIdx.y; y < p.HP * p.rows; y += gridDim.y) {
    const int tr = y % p.rows, w = y / p.rows, row = r0 + tr;
    if (row >= p.R) continue;
    auto at = [&](int j) {  // partial row of the unit's j-th CTA
      const long long slot = j == 0 ? info.first : 2LL * (cta - 1 + j);
      return (slot * p.HP + w) * p.rows + tr;
    };
    float m = -1e30f;
    for (int j = threadIdx.x; j < info.parts; j += 32 * kQaMergeWarps) m = fmaxf(m, p.ml_part[2 * at(j)]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if (lane == 0) s_m[warp] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kQaMergeWarps; ++k) m = fmaxf(m, s_m[k]);
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = warp * PPW + sub; j < info.parts; j += kQaMergeWarps * PPW) {
      const long long pr = at(j);
      const float2 ml = *reinterpret_cast<const float2*>(p.ml_part + 2 * pr);
      const float4 o = *reinterpret_cast<const float4*>(p.o_part + pr * D + d);
      const float wt = ex2_approx(ml.x - m);
      l = fmaf(ml.y, wt, l);
      a.x = fmaf(o.x, wt, a.x);
      a.y = fmaf(o.y, wt, a.y);
      a.z = fmaf(o.z, wt, a.z);
      a.w = fmaf(o.w, wt, a.w);
    }
#pragma unroll
    for (int off = LPR; off < 32; off <<= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, off);
      a.x += __shfl_xor_sync(0xffffffffu, a.x, off);
      a.y += __shfl_xor_sync(0xffffffffu, a.y, off);
      a.z += __shfl_xor_sync(0xffffffffu, a.z, off);
      a.w += __shfl_xor_sync(0xffffffffu, a.w, off);
    }
    if (sub == 0) *reinterpret_cast<float4*>(&s_o[warp][d]) = a;
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (threadIdx.x < D / 2) {
      float x = 0.f, z = 0.f, lt = 0.f;
#pragma unroll
      for (int k = 0; k < kQaMergeWarps; ++k) {
        x += s_o[k][2 * threadIdx.x];
        z += s_o[k][2 * threadIdx.x + 1];
        lt += s_l[k];
      }
      const int i = row / p.G, h = (info.hg * p.HP + w) * p.G + row - i * p.G;
      const bool some = lt != 0.f && i < qlen;
      const float inv = 1.f / (lt * kQaPScale);
      qa_store2<T>(static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + i * p.o_ss + 2 * threadIdx.x,
                   some ? x * inv : 0.f, some ? z * inv : 0.f);
    }
    __syncthreads();
  }
}

}  // namespace mlxp
