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
// How the codes get there.  Where the block size is a multiple of 16 a tile is one TMA box of K
// and one of V (16 rows of one head), three or four stages in flight a warp, each on its own
// mbarrier.  Four contexts of 128 K tokens, 8 heads of 128 (1.07 GB of codes): 179 to 186 us where
// two sets of tensors take turns, 92 to 89 % of the measured HBM rate, 10 of them the merge; 196 to
// 201 behind a flush of L2 or on new tensors each time.  Four CTAs an SM instead of three 190 us,
// loads into registers 257 (a warp is then one tile ahead), cp.async 284 (28 instructions a tile
// keep the load path busy).  Eight of 4 K, 32 heads (269 MB): 52 us and 5 for the merge.  Other block
// sizes do take cp.async, every lane copying the bytes that it reads itself (blocks of 24: 310 us at
// 128 K).  The order of a dot
// product's terms is free, so the fragments are filled straight from the rows: of a K row the four
// lanes c of a row group hold 16-byte pieces, each word of which is one k16 step's two pairs; of a
// V row the eight lanes g hold D / 8 bytes each, and a byte permute of two keys' words gives the
// pairs along keys.
//
// Precision.  16-bit queries are scaled by a power of two a row to below 4 and held in
// fp16 (bf16 values lose nothing but below 2^-25 of the row's largest); fp32 queries and
// probabilities are split into two fp16 terms, which keeps 22 bits.  The running maximum m is of
// s_t + log2 |vs_t|, so that the weights p_t vs_t 2^15 that multiply V8 fit fp16 whatever the
// scales, with 29 octaves below the largest at full precision; m and the sums are fp32.  V's
// scales are taken as at most 2^100, and within 2^80 of each other in a sequence and head, those
// below 2^-60 counting as that: keys of 2^-46 of the largest weight and more are then never lost
// from the sum, whose factors are fp32 powers of two down to 2^-126.
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
constexpr int kQaChunk = 64;   // keys a chunk (quant_attn_rows.cuh: 128)
constexpr int kQaTile = 16;    // keys a tile
constexpr float kQaPScale = 32768.f;
constexpr int kSiteQuantPaged = 12;  // device-status site of this kernel's waits

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
  int causal, bs_pow2;            // bs_pow2: the block size is a power of two
  long long window;               // -1: none
  float scale_log2;
  float p_scale;                  // factor of the partials' weights
  int* status;                    // device status word (bounded waits)
  unsigned long long timeout_ns;
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

template <int NT, int CHUNK = kQaChunk>
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
  r.c0 = r.klo / CHUNK;
  r.n = max(1, (r.khi + CHUNK - 1) / CHUNK - r.c0);
  return r;
}

// CTA whose range [c * total / grid, (c + 1) * total / grid) holds chunk f.
__device__ __forceinline__ int qa_cta_of(long long f, long long total, int grid) {
  return (int)(((f + 1) * grid - 1) / total);
}

// A CTA's range of chunks: the virtual sequence v and the chunk `rem` of it that chunk f is.
struct QaWork {
  long long total, f, f_end, rem;
  int grid, v;
  bool any;
};

// Called by all THREADS of the CTA (at most 1024).
template <int NT, int CHUNK, int THREADS>
__device__ __forceinline__ QaWork qa_find_work(const QaParams& p) {
  constexpr int WARPS = THREADS / 32;
  __shared__ long long s_sum[WARPS], s_rem;
  __shared__ int s_v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, V = p.B * p.RT;
  const int per = (V + THREADS - 1) / THREADS;
  const int va = min(V, (int)threadIdx.x * per), vb = min(V, va + per);
  long long mine = 0;
  for (int v = va; v < vb; ++v) mine += (long long)qa_range<NT, CHUNK>(p, v).n * p.HG;
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += x;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  QaWork w;
  w.total = 0;
  long long before = incl - mine;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    if (i < warp) before += s_sum[i];
    w.total += s_sum[i];
  }
  // no more CTAs than chunks: every working CTA then has some, and a unit's CTAs are consecutive
  w.grid = (int)min((long long)gridDim.x, w.total);
  w.f = (long long)blockIdx.x * w.total / w.grid;
  w.f_end = ((long long)blockIdx.x + 1) * w.total / w.grid;
  w.any = (int)blockIdx.x < w.grid;
  if (!w.any) {
    if (threadIdx.x == 0) p.info[blockIdx.x] = QaPartInfo{-1, 0, 0, 0};
    return w;
  }
  if (w.f >= before && w.f < before + mine) {
    long long at = before;
    int v = va;
    for (; v < vb; ++v) {
      const long long n = (long long)qa_range<NT, CHUNK>(p, v).n * p.HG;
      if (w.f < at + n) break;
      at += n;
    }
    s_v = v;
    s_rem = w.f - at;
  }
  __syncthreads();
  w.v = s_v;
  w.rem = s_rem;
  return w;
}

// What the merge kernel needs of this CTA: the unit of n chunks that its range starts inside of,
// at chunk ch0 > 0.
__device__ __forceinline__ void qa_write_info(const QaParams& p, const QaWork& w, int n, int hg, int ch0) {
  QaPartInfo info{-1, 0, 0, 0};
  if (ch0 > 0) {
    const long long u0 = w.f - ch0;  // the unit's first chunk
    const int first = qa_cta_of(u0, w.total, w.grid);
    const int last = qa_cta_of(u0 + n - 1, w.total, w.grid);
    const int slot = (long long)first * w.total / w.grid == u0 ? 0 : 1;
    info = QaPartInfo{w.v, hg, 2 * first + slot, last - first + 1};
  }
  p.info[blockIdx.x] = info;
}

__device__ __forceinline__ void qa_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same without a sum to add to.
__device__ __forceinline__ void qa_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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

// Elements of a K row held by lane c as 4-byte words: words j < D/16, dims qa_kdim(j, c)..+3.
template <int D>
__device__ __forceinline__ int qa_kdim(int j, int c) {
  if constexpr (D == 32) return 8 * c + 4 * j;
  return (j / 4) * 64 + 16 * c + 4 * (j % 4);
}

// A warp's ring of tiles in shared memory: 16 K rows, then 16 V rows, of D bytes, 16-byte chunks
// swizzled as the tensor maps' 128-, 64- or 32-byte swizzle does.  The fragments fix only which
// rows and chunks meet, so the rows and dims that the lanes take are chosen against bank
// conflicts: row group g works on key qa_key(g) and on the V dims of piece qa_piece(g).
template <int D>
struct QaRing {
  static constexpr int KW = D / 16, VW = D / 32;   // words a lane holds of a K row, a V row
  static constexpr int KB = D == 32 ? 8 : 16, KP = 4 * KW / KB, VB = D / 8;
  static constexpr int kHalf = kQaTile * D, kTileBytes = 2 * kHalf;
  static constexpr int kStages = D == 128 ? 3 : 4;  // more gained nothing: 180 us at 3, 184 at 4
  // a warp's rows' scales and validity a stage, where the block size is not a multiple of 16
  static constexpr int kMeta = 32 * 20;
  static constexpr int kRing = kStages * kTileBytes;
};

__device__ __forceinline__ int qa_key(int g) { return (g & 1) << 2 | g >> 1; }

template <int D>
__device__ __forceinline__ int qa_piece(int g) {
  if constexpr (D == 128) return qa_key(g);
  if constexpr (D == 64) return (g & 1) | (g & 2) << 1 | (g & 4) >> 1;
  return g;
}

template <int D>
__device__ __forceinline__ uint32_t qa_swizzle(uint32_t off) {
  return off ^ ((off >> 7) & (D / 16 - 1)) << 4;
}

// The lane's places in a tile: K row qa_key(g) (row + 8: 8 D bytes on), V rows c and c + 4 (+ 8).
template <int D>
struct QaLane {
  uint32_t k[QaRing<D>::KP], v[2];
  __device__ __forceinline__ QaLane(int g, int c) {
    using Q = QaRing<D>;
#pragma unroll
    for (int i = 0; i < Q::KP; ++i) k[i] = qa_swizzle<D>(qa_key(g) * D + Q::KB * c + 64 * i);
#pragma unroll
    for (int e = 0; e < 2; ++e) v[e] = Q::kHalf + qa_swizzle<D>((c + 4 * e) * D + Q::VB * qa_piece<D>(g));
  }
};

template <int N>
__device__ __forceinline__ void qa_copy(uint32_t dst, const unsigned char* src, bool on) {
  const int n = on ? N : 0;  // the rest is filled with zeros
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void qa_lds(uint32_t src, uint32_t* w) {
  if constexpr (N == 16)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src) : "memory");
  else if constexpr (N == 8)
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(src) : "memory");
  else
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(src) : "memory");
}

// The state of a warp's rows: lane (g, c) holds query rows 2c, 2c + 1 of each n-tile.
template <int D, int NT>
struct QaState {
  float acc[NT][D / 16][4];  // dims qa_piece(g) * D/8 + 2t (0: row 2c, 1: row 2c + 1), + 2t + 1 (2, 3)
  float m[NT][2], l[NT][2];  // l: this lane's keys only, until the end
};

// Scales of the lane's K rows (keys qa_key(g), + 8) and log2 of |V's|, and whether they, and
// the lane's V rows (keys c, c + 4, c + 8, c + 12), are keys in a block.
struct QaRows {
  float ks0, ks1, vs0, vs1, lv0, lv1;
  bool ok0, ok1, okv[4];
};

// log2 |vs| as the running maximum takes it.  Scales below 2^-60 (blocks of zero values have 2^-126)
// count as 2^-60 there: the sum of the weights without vs is rescaled along with the maximum, and
// a factor below 2^-126 would be 0 and take keys out of it that do have weight.
constexpr float kQaLeastLog = -60.f, kQaLeastScale = 0x1p-60f;

__device__ __forceinline__ float qa_log_scale(float vs) {
  return fminf(fmaxf(__log2f(fabsf(vs)), kQaLeastLog), 100.f);
}

template <int D, int NT, bool SPLIT, bool INT8>
__device__ __forceinline__ void qa_step(uint32_t stage, const QaLane<D>& at, const QaRows& t, int t0,
                                        const uint32_t (&qf)[SPLIT ? 2 : 1][NT][D / 16][2],
                                        const float (&qs)[NT][2], const int* row_lo,
                                        const int* row_hi, const float* row_slope,
                                        const int* row_pos, bool masked, int g, int c,
                                        QaState<D, NT>& st) {
  using Q = QaRing<D>;
  float sa[NT][4], sb[NT][4];
#pragma unroll
  for (int i = 0; i < Q::KP; ++i) {
    uint32_t k0[Q::KB / 4], k1[Q::KB / 4];
    qa_lds<Q::KB>(stage + at.k[i], k0);
    qa_lds<Q::KB>(stage + at.k[i] + 8 * D, k1);
#pragma unroll
    for (int x = 0; x < Q::KB / 4; ++x) {
      const int j = i * (Q::KB / 4) + x;
      uint32_t a0, a1, a2, a3;
      qa_codes<INT8>(k0[x], a0, a2);
      qa_codes<INT8>(k1[x], a1, a3);
#pragma unroll
      for (int n = 0; n < NT; ++n) {  // two chains of sums: even and odd words
        float(&d)[4] = j & 1 ? sb[n] : sa[n];
        if (j < 2) qa_mma0(d, a0, a1, a2, a3, qf[0][n][j][0], qf[0][n][j][1]);
        else qa_mma(d, a0, a1, a2, a3, qf[0][n][j][0], qf[0][n][j][1]);
        if constexpr (SPLIT) qa_mma(d, a0, a1, a2, a3, qf[1][n][j][0], qf[1][n][j][1]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) sa[n][e] = (sa[n][e] + sb[n][e]) * (qs[n][e & 1] * (e < 2 ? t.ks0 : t.ks1));
  if (row_slope) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = n * 8 + 2 * c + (e & 1);
        sa[n][e] = fmaf(row_slope[row], (float)(t0 + qa_key(g) + (e < 2 ? 0 : 8) - row_pos[row]), sa[n][e]);
      }
  }
  if (masked) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = n * 8 + 2 * c + (e & 1), key = t0 + qa_key(g) + (e < 2 ? 0 : 8);
        const bool ok = (e < 2 ? t.ok0 : t.ok1) && key >= row_lo[row] && key < row_hi[row];
        if (!ok) sa[n][e] = -INFINITY;
      }
  }
  bool grow = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int q = 0; q < 2; ++q) grow = grow || fmaxf(sa[n][q] + t.lv0, sa[n][q + 2] + t.lv1) > st.m[n][q];
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float mx = fmaxf(sa[n][q] + t.lv0, sa[n][q + 2] + t.lv1);
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
      w[e] = pe * (e < 2 ? v0 : v1);
    }
    if (masked) {  // a masked key's scale may be anything
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (sa[n][e] == -INFINITY) w[e] = 0.f;
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
  uint32_t v[4][Q::VW];
#pragma unroll
  for (int e = 0; e < 4; ++e) qa_lds<Q::VB>(stage + at.v[e & 1] + (e >> 1) * 8 * D, v[e]);
  if (masked) {  // rows before and behind the keys may hold anything
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int w = 0; w < Q::VW; ++w) v[e][w] = t.okv[e] ? v[e][w] : 0u;
  }
#pragma unroll
  for (int w = 0; w < Q::VW; ++w) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint32_t sel = hf ? 0x7362u : 0x5140u;
      uint32_t a0, a1, a2, a3;
      qa_codes<INT8>(__byte_perm(v[0][w], v[1][w], sel), a0, a1);  // keys c, c + 4: P^T's rows 2c, 2c + 1
      qa_codes<INT8>(__byte_perm(v[2][w], v[3][w], sel), a2, a3);
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
      if (E >= 1 && E <= 254) up = __uint_as_float(min(E, 253u) << 23);  // its inverse is not 0
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

// Dynamic shared memory of the kernel: the warps' rings, or the warps' merge.
template <int D, int NT, bool BS16>
constexpr int qa_smem_bytes() {
  using Q = QaRing<D>;
  constexpr int ring = kQaWarps * (Q::kRing + (BS16 ? 0 : Q::kStages * Q::kMeta)), red = kQaWarps * 8 * NT * (D + 4) * 4;
  return ring > red ? ring : red;
}

template <typename T, int D, int NT, bool INT8, bool BS16, int MINB>
__global__ void __launch_bounds__(32 * kQaWarps, MINB)
    quant_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const QaParams p) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int ROWS = 8 * NT;
  constexpr int RED = D + 4;  // floats a row in the warps' merge: acc, m, l
  __shared__ int s_lo[ROWS], s_hi[ROWS], s_pos[ROWS];
  __shared__ float s_slope[4][ROWS];
  __shared__ int s_abort;
  __shared__ __align__(8) uint64_t s_bar[kQaWarps][QaRing<D>::kStages];
  using Q = QaRing<D>;
  extern __shared__ __align__(1024) unsigned char qa_smem[];
  // the warps' rings; between units, the warps' merge ([warp][ROWS][RED] floats)
  float(*s_red)[ROWS][RED] = reinterpret_cast<float(*)[ROWS][RED]>(qa_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int HP = p.HP, KS = kQaWarps / HP;
  const int hp = warp % HP, kidx = warp / HP;
  const uint32_t ring = smem_u32(qa_smem + warp * Q::kRing);
  float* meta = reinterpret_cast<float*>(qa_smem + kQaWarps * Q::kRing + warp * Q::kStages * Q::kMeta);
  const uint32_t bars = smem_u32(s_bar[warp]);
  const int dim0 = qa_piece<D>(g) * (D / 8);  // of the lane's output dims
  const QaLane<D> at(g, c);
  const WaitCtx wctx{&s_abort, p.status, p.timeout_ns};
  uint32_t phase = 0;                          // parity of each stage's next completion
  int stage_in = 0, stage_out = 0;             // next stage to fill, to read
  if constexpr (BS16) {
    if (lane == 0) {
      for (int i = 0; i < Q::kStages; ++i) mbar_init(bars + 8 * i, 1);
      fence_mbar_init();
    }
    if (threadIdx.x == 0) {
      s_abort = 0;
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }

  QaWork w = qa_find_work<NT, kQaChunk, 32 * kQaWarps>(p);
  if (!w.any) return;
  const long long f_begin = w.f;
  while (w.f < w.f_end) {
    const QaRange r = qa_range<NT>(p, w.v);
    const int b = w.v / p.RT, r0 = (w.v - b * p.RT) * ROWS;
    const int hg = (int)(w.rem / r.n), ch0 = (int)(w.rem - (long long)hg * r.n);
    const int ch1 = (int)min((long long)r.n, ch0 + (w.f_end - w.f));
    if (w.f == f_begin && threadIdx.x == 0) qa_write_info(p, w, r.n, hg, ch0);
    __syncthreads();  // the last unit's reads of the row tables and s_red are done
    const int hk = hg * HP + hp;
    uint32_t qf[SPLIT ? 2 : 1][NT][D / 16][2];
    float qs[NT][2];
    // The rows' tables and this warp's queries: called by every warp once its first tiles are on
    // their way.
    auto set_up = [&] {
      if (threadIdx.x < ROWS) {
        const int row = r0 + threadIdx.x, i = row / p.G;
        int lo = 0, hi = 0;
        if (row < p.R && i < r.qlen) qa_row_range(p, r.ctx, r.qlen, i, lo, hi);
        s_lo[threadIdx.x] = lo;
        s_hi[threadIdx.x] = hi;
        // ALiBi counts from the last key that there can be where the position lies behind it: the
        // softmax does not see the difference, fp32 does
        s_pos[threadIdx.x] = (int)min(r.ctx - r.qlen + i, (long long)p.max_blocks * p.block_size);
      }
      if (p.alibi && threadIdx.x < HP * ROWS) {
        const int hw = threadIdx.x / ROWS, row = r0 + threadIdx.x % ROWS;
        s_slope[hw][threadIdx.x % ROWS] =
            row < p.R ? __ldg(p.alibi + (hg * HP + hw) * p.G + row % p.G) * 1.4426950408889634f : 0.f;
      }
      __syncthreads();
      qa_load_q<T, D, NT, SPLIT>(p, b, r0, hk, g, c, qf, qs);
    };
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
    // keys [key_lo, k1): what the first tile holds before a window is as foreign as what lies behind
    const int key_lo = max(k0, r.klo);
    const unsigned keys = (unsigned)max(k1 - key_lo, 0);
    const int* bt = p.block_tables + (long long)b * p.bt_stride;
    const long long head_sc = hk * p.sc_sh;
    const float* slope = p.alibi ? s_slope[hp] : nullptr;
    const int step = kQaTile * KS, ta = k0 + kidx * kQaTile;
    const int tiles = ta < k1 ? (k1 - ta + step - 1) / step : 0;  // this warp's
    if constexpr (BS16) {
      // A tile lies in one block: lane i % 32 holds tile i's block and scales, for 32 tiles at a
      // time, the next 32 being loaded while these are worked on.  A tile's K and V rows are one
      // TMA box each, issued by lane 0; tiles without a block are skipped.
      struct Batch {
        int id;
        float ks, vs, lv;
        uint32_t there;  // which of the 32 have a block
      };
      auto batch = [&](int i0) {
        Batch x{-1, 0.f, 0.f, 0.f, 0u};
        const int i = i0 + lane;
        if (i < tiles) {
          const int got = __ldg(bt + (unsigned)(ta + i * step) / (unsigned)p.block_size);
          if (got >= 0 && got < p.num_blocks) {
            x.id = got;
            x.ks = __ldg(p.k_scales + got * p.sc_sb + head_sc);
            x.vs = __ldg(p.v_scales + got * p.sc_sb + head_sc);
          }
        }
        x.there = __ballot_sync(0xffffffffu, x.id >= 0);
        return x;
      };
      Batch cur = batch(0), next = batch(32);  // lv: once the scale is here and is needed
      int base = 0;  // first tile of `cur`
      int inflight = 0;
      stage_in = stage_out;
      auto issue = [&](int i) {
        const bool far = i - base >= 32;
        if (i >= tiles || !((far ? next.there : cur.there) >> (i & 31) & 1u)) return;
        const int id = __shfl_sync(0xffffffffu, far ? next.id : cur.id, i & 31);
        if (lane == 0) {
          const unsigned t0 = ta + i * step;
          const int row = p.bs_pow2 ? t0 & (p.block_size - 1) : t0 % (unsigned)p.block_size;
          const uint32_t bar = bars + 8 * stage_in, dst = ring + stage_in * Q::kTileBytes;
          mbar_arrive_expect_tx(bar, Q::kTileBytes);
          tma_load_4d(dst, &tm_k, bar, 0, hk, row, id);
          tma_load_4d(dst + Q::kHalf, &tm_v, bar, 0, hk, row, id);
        }
        stage_in = stage_in + 1 == Q::kStages ? 0 : stage_in + 1;
        ++inflight;
      };
      fence_proxy_async_smem();  // the ring may have been the merge's buffer
      __syncwarp();
      int ahead = 0;             // tiles issued so far
      for (; ahead < Q::kStages; ++ahead) issue(ahead);
      set_up();
      cur.lv = qa_log_scale(cur.vs);
      bool ok = true;
      for (int i = 0; i < tiles; ++i) {
        if (cur.there >> (i & 31) & 1u) {
          ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * stage_out, phase >> stage_out & 1u, wctx,
                                                 kSiteQuantPaged));
          if (!ok) break;
          phase ^= 1u << stage_out;
          --inflight;
          const int t0 = ta + i * step;
          QaRows rows;
          rows.ks0 = rows.ks1 = __shfl_sync(0xffffffffu, cur.ks, i & 31);
          rows.vs0 = rows.vs1 = __shfl_sync(0xffffffffu, cur.vs, i & 31);
          rows.lv0 = rows.lv1 = __shfl_sync(0xffffffffu, cur.lv, i & 31);
          const int from = t0 - key_lo;
          rows.ok0 = (unsigned)(from + qa_key(g)) < keys;
          rows.ok1 = (unsigned)(from + qa_key(g) + 8) < keys;
#pragma unroll
          for (int e = 0; e < 4; ++e) rows.okv[e] = (unsigned)(from + c + 4 * e) < keys;
          qa_step<D, NT, SPLIT, INT8>(ring + stage_out * Q::kTileBytes, at, rows, t0, qf, qs, s_lo, s_hi,
                                      slope, s_pos, t0 < r.flo || t0 + kQaTile > r.fhi, g, c, st);
          stage_out = stage_out + 1 == Q::kStages ? 0 : stage_out + 1;
          __syncwarp();  // every lane has read the stage
          if (lane == 0) fence_proxy_async_smem();
        }
        // keep kStages tiles in flight: skipped tiles leave their stage to later ones
        while (inflight < Q::kStages && ahead < tiles && ahead - base < 64) issue(ahead++);
        if ((i & 31) == 31) {
          base += 32;
          cur = next;
          cur.lv = qa_log_scale(cur.vs);
          next = batch(base + 32);
          while (inflight < Q::kStages && ahead < tiles && ahead - base < 64) issue(ahead++);
        }
      }
      if (!ok) {  // wait (bounded) for this warp's copies, then write nothing more
        for (int k = 0; k < inflight; ++k) {
          const int sk = (stage_out + k) % Q::kStages;
          if (lane == 0) mbar_wait_drain(bars + 8 * sk, phase >> sk & 1u, p.status, p.timeout_ns);
        }
        __syncwarp();
      }
    } else {
      // Any block size: every lane copies the pieces that it reads itself, with cp.async.
      set_up();
      const unsigned char* kl = p.k_pool + hk * p.p_sh + Q::KB * c;
      const unsigned char* vl = p.v_pool + hk * p.p_sh + Q::VB * qa_piece<D>(g);
      auto locate = [&](int key, long long& off) {
        off = 0;
        if ((unsigned)(key - key_lo) >= keys) return -1;
        const unsigned slot = (unsigned)key / (unsigned)p.block_size;
        const int got = __ldg(bt + slot);
        if (got < 0 || got >= p.num_blocks) return -1;
        off = (long long)got * p.p_sb + (long long)(key - (int)slot * p.block_size) * p.p_st;
        return got;
      };
      auto issue = [&](int i) {
        const uint32_t dst = ring + (i % Q::kStages) * Q::kTileBytes;
        float* m = meta + (i % Q::kStages) * (Q::kMeta / 4);
        const int t0 = ta + i * step;
        int ok = 0;
        long long off;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int id = locate(t0 + qa_key(g) + 8 * hf, off);
          ok |= (id >= 0) << hf;
#pragma unroll
          for (int x = 0; x < Q::KP; ++x) qa_copy<Q::KB>(dst + at.k[x] + 8 * hf * D, kl + off + 64 * x, id >= 0);
          m[32 * hf + lane] = id < 0 ? 0.f : __ldg(p.k_scales + id * p.sc_sb + head_sc);
          m[64 + 32 * hf + lane] = id < 0 ? 0.f : __ldg(p.v_scales + id * p.sc_sb + head_sc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = locate(t0 + c + 4 * e, off) >= 0;
          ok |= in << (2 + e);
          qa_copy<Q::VB>(dst + at.v[e & 1] + (e >> 1) * 8 * D, vl + off, in);
        }
        m[128 + lane] = __int_as_float(ok);
      };
      for (int i = 0; i < Q::kStages - 1; ++i) {
        if (i < tiles) issue(i);
        cp_async_commit();
      }
      for (int i = 0; i < tiles; ++i) {
        if (i + Q::kStages - 1 < tiles) issue(i + Q::kStages - 1);  // into the stage used last
        cp_async_commit();
        cp_async_wait<Q::kStages - 1>();  // this lane's pieces of tile i have landed
        const int t0 = ta + i * step;
        const float* m = meta + (i % Q::kStages) * (Q::kMeta / 4);
        const int ok = __float_as_int(m[128 + lane]);
        QaRows rows{m[lane], m[32 + lane], m[64 + lane], m[96 + lane], 0.f, 0.f, (ok & 1) != 0, (ok & 2) != 0,
                    {(ok & 4) != 0, (ok & 8) != 0, (ok & 16) != 0, (ok & 32) != 0}};
        rows.lv0 = qa_log_scale(rows.vs0);
        rows.lv1 = qa_log_scale(rows.vs1);
        const bool masked = t0 < r.flo || t0 + kQaTile > r.fhi || !__all_sync(0xffffffffu, ok == 63);
        qa_step<D, NT, SPLIT, INT8>(ring + (i % Q::kStages) * Q::kTileBytes, at, rows, t0, qf, qs, s_lo, s_hi,
                                    slope, s_pos, masked, g, c, st);
      }
      cp_async_wait<0>();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
          st.l[n][e] += __shfl_xor_sync(0xffffffffu, st.l[n][e], off);

    if constexpr (BS16) {
      if (__syncthreads_or(s_abort != 0)) break;  // a wait gave up: nothing more is written
    }
    const bool whole = ch0 == 0 && ch1 == r.n;
    const long long slot = 2LL * blockIdx.x + (w.f == f_begin ? 0 : 1);
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
            T* o = static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + i * p.o_ss + dim0;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
              qa_store2<T>(o + 2 * d, some ? st.acc[n][d][e] * inv : 0.f,
                           some ? st.acc[n][d][e + 2] * inv : 0.f);
          } else {
            const long long pr = (slot * HP + hp) * p.rows + tr;
            float* o = p.o_part + pr * D + dim0;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
              *reinterpret_cast<float2*>(o + 2 * d) = make_float2(st.acc[n][d][e], st.acc[n][d][e + 2]);
            if (g == 0) *reinterpret_cast<float2*>(p.ml_part + 2 * pr) = make_float2(st.m[n][e], st.l[n][e]);
          }
        }
    } else {
      __syncthreads();  // every warp is done with its ring
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* row = s_red[warp][n * 8 + 2 * c + e];
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
            *reinterpret_cast<float2*>(row + dim0 + 2 * d) =
                make_float2(st.acc[n][d][e], st.acc[n][d][e + 2]);
          if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(st.m[n][e], st.l[n][e]);
        }
      __syncthreads();
      for (int x = threadIdx.x; x < HP * p.rows * (D / 2); x += blockDim.x) {
        const int d = 2 * (x % (D / 2)), y = x / (D / 2), tr = y % p.rows, hw = y / p.rows;
        const int row = r0 + tr;
        if (row >= p.R) continue;
        float m = -1e30f;
        for (int k = 0; k < KS; ++k) m = fmaxf(m, s_red[hw + k * HP][tr][D]);
        float l = 0.f, a = 0.f, bb = 0.f;
        for (int k = 0; k < KS; ++k) {
          const float* s = s_red[hw + k * HP][tr];
          const float wt = ex2_approx(s[D] - m);
          l = fmaf(s[D + 1], wt, l);
          a = fmaf(s[d], wt, a);
          bb = fmaf(s[d + 1], wt, bb);
        }
        if (whole) {
          const int i = row / p.G, h = (hg * HP + hw) * p.G + row - i * p.G;
          const bool some = l != 0.f && i < r.qlen;
          const float inv = 1.f / (l * kQaPScale);
          qa_store2<T>(static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + i * p.o_ss + d,
                       some ? a * inv : 0.f, some ? bb * inv : 0.f);
        } else {
          const long long pr = (slot * HP + hw) * p.rows + tr;
          *reinterpret_cast<float2*>(p.o_part + pr * D + d) = make_float2(a, bb);
          if (d == 0) *reinterpret_cast<float2*>(p.ml_part + 2 * pr) = make_float2(m, l);
        }
      }
    }
    w.f += ch1 - ch0;
    w.rem += ch1 - ch0;
    if (w.rem >= (long long)r.n * p.HG) {
      w.rem = 0;
      ++w.v;
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Merges the partials of the units that more than one CTA worked on.  Block x looks at main CTA
// x + 1: where that is the second CTA of a unit, it merges the unit's rows.  A warp takes a row to
// itself, or the block's warps share one: from 5 partials where all blocks run at once (a single
// short context: 3.9 us, 5.5 with a warp a row), from 33 otherwise (48 contexts to 9000 with 9
// partials each: 6.6 us, 9.1 with a block a row).  Blocks that look at eight CTAs each instead
// took 1 to 2 us longer, but for the longest contexts (8.3 us for 9.8).
constexpr int kQaMergeWarps = 8;
constexpr unsigned kQaMergeResident = 1024;  // blocks of 256 threads that run at once

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
  const bool together = info.parts > (gridDim.x * gridDim.y <= kQaMergeResident ? 4 : 32);
  const int team = together ? kQaMergeWarps : 1, me = together ? warp : 0;  // warps a row, this one's place
  const int stride = together ? gridDim.y : gridDim.y * kQaMergeWarps;
  for (int y = together ? blockIdx.y : blockIdx.y * kQaMergeWarps + warp; y < p.HP * p.rows; y += stride) {
    const int tr = y % p.rows, w = y / p.rows, row = r0 + tr;
    if (row >= p.R) continue;
    auto at = [&](int j) {  // partial row of the unit's j-th CTA
      const long long slot = j == 0 ? info.first : 2LL * (cta - 1 + j);
      return (slot * p.HP + w) * p.rows + tr;
    };
    float m = -1e30f;
    for (int j = me * 32 + lane; j < info.parts; j += 32 * team) m = fmaxf(m, p.ml_part[2 * at(j)]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if (together) {
      if (lane == 0) s_m[warp] = m;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kQaMergeWarps; ++k) m = fmaxf(m, s_m[k]);
    }
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = me * PPW + sub; j < info.parts; j += team * PPW) {
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
    if (together) {
      if (sub == 0) *reinterpret_cast<float4*>(&s_o[warp][d]) = a;
      if (lane == 0) s_l[warp] = l;
      __syncthreads();
      a = make_float4(0.f, 0.f, 0.f, 0.f);
      l = 0.f;
#pragma unroll
      for (int k = 0; k < kQaMergeWarps; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(&s_o[k][d]);
        a.x += x.x;
        a.y += x.y;
        a.z += x.z;
        a.w += x.w;
        l += s_l[k];
      }
    }
    if (sub == 0 && me == 0) {
      const int i = row / p.G, h = (info.hg * p.HP + w) * p.G + row - i * p.G;
      const bool some = l != 0.f && i < qlen;
      const float inv = 1.f / (l * p.p_scale);
      T* o = static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + i * p.o_ss + d;
      qa_store2<T>(o, some ? a.x * inv : 0.f, some ? a.y * inv : 0.f);
      qa_store2<T>(o + 2, some ? a.z * inv : 0.f, some ? a.w * inv : 0.f);
    }
    if (together) __syncthreads();
  }
}

}  // namespace mlxp
