// quant_attn_rows.cuh — attention of many query rows (a prompt's chunk) over an 8-bit paged cache,
// on tcgen05.
//
// The same function, precision and split of work as quant_attn.cuh (which see), for more query
// rows a pool head than its 16-row tiles are good for: a unit is 256 rows (two TMEM tiles of 128)
// of one pool head, a chunk 128 keys.  By work it is bound by the tensor pipe (4 * 128 * 128 * D
// flops a tile and key chunk, 1450 cycles at D = 128), then by the exponentials (128 * 128 of
// them, 1024 cycles); as it stands by the chain that a tile's chunk runs through: scores out of
// TMEM, maximum, exponentials, weights back, PV, the next QK, 5.5 to 6 K cycles, of which the two
// tiles hide half.  Four sequences of 512 queries and contexts to 8 K, 32 heads over 8 of 128:
// 344 to 351 us, 20 of them the merge, 521 to 532 TFLOP/s (int8 373).  At head_dim 128 the converting
// warps spill within their 104 registers (up to 172 bytes a thread stored, 276 loaded): 64 of them
// are the codes under way.
//
// The codes become fp16 (exactly) on their way into shared memory, once for both tiles: the MMA
// reads 16-bit operands, and 8-bit queries would lose what the cache kept.  Scales stay out of
// the operands: K's multiply the scores' columns (one factor a 16-key group, the block size being
// a multiple of 16), V's the weights, as a term of their exponent.  Negative scales' signs move
// into the codes, so that a group's maximum is its scores' maximum times the scale and the
// exponent has a logarithm to add; values whose scale is below the least logarithm are zeros.
//
// Roles, 12 warps: two softmax warpgroups, a thread a row (scores from TMEM into registers,
// weights back over them as fp16), whose first thread also issues its tile's MMAs,
//   S_t = Q_t K^T (both operands in shared memory), O_t += P_t V (P from TMEM, V as it lies),
// and one warpgroup that converts (codes of the next tile in registers while this one is stored).
// Tile 1's MMAs run while tile 0's weights are computed and the other way round.  An issuing warp
// of its own cost 600 cycles a key tile from the last weight to the MMA; two threads a row had
// not the registers.  QK_t of the next chunk is issued right behind PV_t of this one, so that its
// completion also says that O_t may be rescaled; that is done when a row's maximum has grown by
// more than 2^7 (the weights' factor is 2^8: they stay within fp16).  At 2^3 some row of a warp had
// grown in most chunks, a thousand cycles each time.
//
// K and V have two stages each in shared memory (64 KB each at D = 128) beside the 64 KB of Q.
// The scales' ring has four: a group's are written at chunk j + 3 at the earliest after both
// tiles' weights of chunk j, since K's stage is released by QK(j + 1), which follows PV(j).
// A tile without rows (beside the last 128 and fewer of a head's) waits for and releases each stage
// like the other.  Every mbarrier wait is bounded; after one gave up nothing more is written.
#pragma once

#include "quant_attn.cuh"

namespace mlxp {

constexpr int kQrThreads = 384;
// registers a thread of the softmax and converting warpgroups: 128 * (2 * 200 + 104) = 64512 = what
// 384 threads of 168 are launched with
constexpr int kQrRegsSoftmax = 200, kQrRegsConvert = 104;
static_assert(128 * (2 * kQrRegsSoftmax + kQrRegsConvert) <= 384 * 168, "register split");
constexpr int kQrRows = 256, kQrKeys = 128;
constexpr float kQrPLog = 8.f;  // log2 of the weights' factor; the sums l carry it too
constexpr float kQrHeadroom = 7.f;
constexpr int kSiteQuantRows = 13;

template <int D>
struct QrCfg {
  static constexpr int KB = D / 64;              // 128-byte column boxes
  static constexpr int BOX = 128 * 128;          // bytes of a box of 128 rows
  static constexpr int TILE = KB * BOX;          // a 128-row fp16 tile
  static constexpr int OFF_Q = 0, OFF_K = 2 * TILE, OFF_V = 4 * TILE, OFF_MISC = 6 * TILE;
  // barriers
  static constexpr int B_KF = 0, B_VF = 2, B_KE = 4, B_VE = 6, B_SF = 8, B_OF = 10, B_DR = 12,
                       B_TURN = 13;  // [2][4]
  static constexpr int OFF_SCALE = OFF_MISC + 256;             // [4][8] float4: |K scale|, log2 |V scale|, its inverse
  static constexpr int OFF_MASK = OFF_SCALE + 4 * 8 * 16;      // [4][4] bytes: which of a warp's two groups have a block
  static constexpr int OFF_TMEM = OFF_MASK + 16;
  static constexpr int SMEM = OFF_TMEM + 16 + 1024;            // slack to align the base
  static constexpr uint32_t TM_S0 = 0, TM_S1 = 128, TM_O0 = 256, TM_O1 = 256 + D, TM_COLS = 512;
};

// 16-byte chunk c of row r of a box, 128-byte swizzle.
__device__ __forceinline__ uint32_t qr_at(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// 16 codes of row r (piece l of D / 16) as fp16 into a tile, with the signs turned by `flip`.
template <int D, bool INT8>
__device__ __forceinline__ void qr_store(uint32_t tile, int r, int l, const uint4& w, uint32_t flip) {
  uint32_t h[8];
  qa_codes<INT8>(w.x, h[0], h[1]);
  qa_codes<INT8>(w.y, h[2], h[3]);
  qa_codes<INT8>(w.z, h[4], h[5]);
  qa_codes<INT8>(w.w, h[6], h[7]);
  if (flip) {  // the same for the whole warp's group of rows; rare
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] ^= flip;
  }
  const uint32_t base = tile + (l >> 2) * QrCfg<D>::BOX, at = qr_at(r, 2 * (l & 3));
  st_shared_v4(base + at, h[0], h[1], h[2], h[3]);
  st_shared_v4(base + (at ^ 16), h[4], h[5], h[6], h[7]);
}

template <typename T, int D, bool INT8>
__global__ void __launch_bounds__(kQrThreads, 1) quant_attn_rows_kernel(const QaParams p) {
  using C = QrCfg<D>;
  constexpr int NT = kQrRows / 8;
  constexpr int LR = D / 16, RPI = 32 / LR, IT = 32 / RPI;  // lanes a row, rows an access, accesses a warp
  extern __shared__ unsigned char qr_smem_raw[];
  const uint32_t sbase = (smem_u32(qr_smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = qr_smem_raw + (sbase - smem_u32(qr_smem_raw));
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto BAR = [&](int i) { return sbase + C::OFF_MISC + 8 * i; };
  const WaitCtx wctx{&s_abort, p.status, p.timeout_ns};
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(C::B_KF + i), 4);
      mbar_init(BAR(C::B_VF + i), 4);
      mbar_init(BAR(C::B_KE + i), 2);
      mbar_init(BAR(C::B_VE + i), 2);
      mbar_init(BAR(C::B_SF + i), 1);
      mbar_init(BAR(C::B_OF + i), 1);
    }
    mbar_init(BAR(C::B_DR), 2);
    for (int i = 0; i < 8; ++i) mbar_init(BAR(C::B_TURN + i), 1);
    fence_mbar_init();
  }
  QaWork w = qa_find_work<NT, kQrKeys, kQrThreads>(p);
  if (!w.any) return;
  if (warp == 8) tmem_alloc(sbase + C::OFF_TMEM, C::TM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<const volatile uint32_t*>(smem + C::OFF_TMEM);
  if (warp == 8) tmem_relinquish();
  const long long f_begin = w.f;
  float4* s_scale = reinterpret_cast<float4*>(smem + C::OFF_SCALE);
  const uint32_t* s_mask = reinterpret_cast<const uint32_t*>(smem + C::OFF_MASK);
  int cnt = 0;                 // key tiles this CTA has gone through, every role's own count

  // The units, which every role goes through by itself: the tiles share K, V and the scales, whose
  // rings' barriers run on from unit to unit, and nothing else.
  struct Unit {
    QaRange r;
    int b, r0, hk, ch0, ch1, tiles;  // tiles: 1 where the second one has no rows
    bool whole;
    long long slot;
  };
  auto next_unit = [&]() {
    Unit u;
    u.r = qa_range<NT, kQrKeys>(p, w.v);
    u.b = w.v / p.RT;
    u.r0 = (w.v - u.b * p.RT) * kQrRows;
    u.hk = (int)(w.rem / u.r.n);
    u.ch0 = (int)(w.rem - (long long)u.hk * u.r.n);
    u.ch1 = (int)min((long long)u.r.n, u.ch0 + (w.f_end - w.f));
    u.tiles = p.R - u.r0 > 128 ? 2 : 1;
    u.whole = u.ch0 == 0 && u.ch1 == u.r.n;
    u.slot = 2LL * blockIdx.x + (w.f == f_begin ? 0 : 1);
    if (w.f == f_begin && threadIdx.x == 0) qa_write_info(p, w, u.r.n, u.hk, u.ch0);
    return u;
  };
  auto advance = [&](const Unit& u) {
    w.f += u.ch1 - u.ch0;
    w.rem += u.ch1 - u.ch0;
    if (w.rem >= (long long)u.r.n * p.HG) {
      w.rem = 0;
      ++w.v;
    }
  };

  if (warp < 8) {
    // -------- softmax and the MMAs of tile t: a thread a row; the first thread issues --------
    setmaxnreg_inc<kQrRegsSoftmax>();
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const bool issuer = (threadIdx.x & 127) == 0;
    int n_s = 0, n_o = 0, n_t = 0;  // score tiles, units and turns seen
    const uint32_t turn_mine = BAR(C::B_TURN + 4 * t + (warp & 3)), turn_other = BAR(C::B_TURN + 4 * (t ^ 1) + (warp & 3));
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t d_s = tmem + (t ? C::TM_S1 : C::TM_S0), d_o = tmem + (t ? C::TM_O1 : C::TM_O0);
    const uint32_t tS = d_s + lane_off, tO = d_o + lane_off;
    constexpr uint32_t idesc_qk = make_idesc_f16(128, 128, false, false);
    constexpr uint32_t idesc_pv = make_idesc_f16(128, D, false, true);
    const uint32_t q_lo = ((sbase + C::OFF_Q + t * C::TILE) >> 4) | (1u << 16);
    const uint32_t k_lo = ((sbase + C::OFF_K) >> 4) | (1u << 16);
    const uint32_t v_lo = ((sbase + C::OFF_V) >> 4) | ((uint32_t)(C::BOX >> 4) << 16);
    // Scores of the CTA's key tile c, once K is there.  A stage's release counts both tiles; where
    // no unit has rows for tile 1, tile 0 releases for both.
    const bool one = p.R <= 128;
    auto issue_qk = [&](int c) {
      const int st = c & 1;
      if (!mbar_wait(BAR(C::B_KF + st), (c >> 1) & 1, wctx, kSiteQuantRows)) return false;
      tc_fence_after();
      const uint32_t b = k_lo + (uint32_t)(st * C::TILE >> 4);
#pragma unroll
      for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ss(d_s, sdesc(q_lo + (uint32_t)((kb * C::BOX + kk * 32) >> 4)),
                 sdesc(b + (uint32_t)((kb * C::BOX + kk * 32) >> 4)), idesc_qk, (kb | kk) ? 1u : 0u);
      tc_commit(BAR(C::B_SF + t));
      tc_commit(BAR(C::B_KE + st));
      if (one) tc_commit(BAR(C::B_KE + st));
      return true;
    };
    auto issue_pv = [&](int c, bool first) {
      const int st = c & 1;
      if (!mbar_wait(BAR(C::B_VF + st), (c >> 1) & 1, wctx, kSiteQuantRows)) return false;
      tc_fence_after();
      const uint32_t b = v_lo + (uint32_t)(st * C::TILE >> 4);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        mma_ts(d_o, d_s + kk * 8, sdesc(b + (uint32_t)(kk * 16 * 128 >> 4)), idesc_pv, (!first || kk > 0) ? 1u : 0u);
      tc_commit(BAR(C::B_VE + st));
      if (one) tc_commit(BAR(C::B_VE + st));
      return true;
    };
    while (w.f < w.f_end) {
      const Unit u = next_unit();
      if (t >= u.tiles) {
        // No rows for tile 1 here.  If it has some in other units it goes through the stages all the
        // same: a wait by parity tells a phase from its neighbours only, so that a tile that ran
        // ahead would take a stage of two chunks before for its own, and one that fell behind would
        // miss a phase.
        if (issuer && !one) {
          for (int c = cnt; c < cnt + u.ch1 - u.ch0; ++c) {
            const int st = c & 1;
            if (!mbar_wait(BAR(C::B_KF + st), (c >> 1) & 1, wctx, kSiteQuantRows)) break;
            mbar_arrive(BAR(C::B_KE + st));
            if (!mbar_wait(BAR(C::B_VF + st), (c >> 1) & 1, wctx, kSiteQuantRows)) break;
            mbar_arrive(BAR(C::B_VE + st));
          }
        }
        __syncwarp();
        cnt += u.ch1 - u.ch0;
        advance(u);
        continue;
      }
      const int qrow = u.r0 + t * 128 + row, qi = qrow / p.G;
      const bool live = qrow < p.R && qi < u.r.qlen, alone = u.tiles == 1;
      const int h = u.hk * p.G + qrow - qi * p.G;
      int lo = 0, hi = 0;
      if (live) qa_row_range(p, u.r.ctx, u.r.qlen, qi, lo, hi);
      // The warp's 32 rows, each scaled by a power of two, as fp16: QL lanes read a row.
      float qs = p.scale_log2;
      {
        constexpr int QL = D / 8, QR = 32 / QL;
        const int ql = lane % QL, qr = lane / QL;
        uint4 x[QL];
        int at = u.r0 + t * 128 + (warp & 3) * 32 + qr, ai = at / p.G, ag = at - ai * p.G;
        const T* src = static_cast<const T*>(p.q) + u.b * p.q_sb + (long long)u.hk * p.G * p.q_sh + 8 * ql;
#pragma unroll
        for (int i = 0; i < QL; ++i) {
          x[i] = make_uint4(0, 0, 0, 0);
          if (at < p.R && ai < u.r.qlen) x[i] = *reinterpret_cast<const uint4*>(src + ag * p.q_sh + ai * p.q_ss);
          at += QR;
          for (ag += QR; ag >= p.G; ag -= p.G) ++ai;
        }
        const uint32_t dst = sbase + C::OFF_Q + t * C::TILE + (ql >> 3) * C::BOX;
#pragma unroll
        for (int i = 0; i < QL; ++i) {
          const int rr = (warp & 3) * 32 + i * QR + qr;
          uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(v[e] << 16)), fabsf(__uint_as_float(v[e] & 0xffff0000u))));
#pragma unroll
            for (int off = 1; off < QL; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const unsigned E = __float_as_uint(mx) >> 23;
            const unsigned up = E >= 1 && E <= 254 ? min(E, 253u) : 127u;  // 2^-up is not 0
            const float down = __uint_as_float((254u - up) << 23);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = qa_pack(__uint_as_float(v[e] << 16) * down, __uint_as_float(v[e] & 0xffff0000u) * down);
            // its factor, for the thread whose row it is
            const float f = __shfl_sync(0xffffffffu, __uint_as_float(up << 23), (lane % QR) * QL);
            if (lane / QR == i) qs = f * p.scale_log2;
          }
          st_shared_v4(dst + qr_at(rr, ql & 7), v[0], v[1], v[2], v[3]);
        }
      }
      fence_proxy_async_smem();
      named_bar_sync(1 + t, 128);  // the tile's Q is in place
      float m = -1e30f, l = 0.f;
      bool ok = true;
      if (issuer) ok = issue_qk(cnt);
      for (int j = u.ch0; j < u.ch1; ++j) {
        const int c = cnt + j - u.ch0;
        if (ok) ok = mbar_wait(BAR(C::B_SF + t), n_s & 1, wctx, kSiteQuantRows);
        ok = __all_sync(0xffffffffu, ok);
        ++n_s;
        tc_fence_after();
        if (ok) {
          const int key0 = (u.r.c0 + j) * kQrKeys;
          const float4* sc = s_scale + (c & 3) * 8;
          uint32_t x[4][32];
          tmem_ld_x32(tS, x[0]);
          tmem_ld_x32(tS + 32, x[1]);
          tmem_ld_x32(tS + 64, x[2]);
          tmem_ld_x32(tS + 96, x[3]);
          uint32_t groups = s_mask[c & 3];  // bits 0, 1 of each byte
          groups = (groups & 3u) | (groups >> 6 & 12u) | (groups >> 12 & 48u) | (groups >> 18 & 192u);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 4; ++k) reg_fence(x[k]);
          if (key0 < u.r.flo || key0 + kQrKeys > u.r.fhi || groups != 0xffu) {
            const int from = lo - key0;
            const unsigned width = (unsigned)max(hi - lo, 0);
#pragma unroll
            for (int e = 0; e < 128; ++e)
              if ((unsigned)(e - from) >= width || !(groups >> (e >> 4) & 1u)) x[e >> 5][e & 31] = 0xff800000u;
          }
          float mloc = -INFINITY;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const uint32_t* v = x[g >> 1] + 16 * (g & 1);
            float mx = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
#pragma unroll
            for (int e = 2; e < 16; e += 2) mx = max3(mx, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
            mloc = fmaxf(mloc, fmaf(mx, fmaxf(sc[g].x * qs, 1.2e-38f), sc[g].y));
          }
          const bool resc = mloc > m + kQrHeadroom;
          float alpha = 1.f;
          if (resc) {
            alpha = ex2_approx(m - mloc);
            m = mloc;
          }
          // weight = 2^(s f - m + log2 |vs| + 8): what multiplies V's codes; the sum l of the
          // weights without vs is taken a group at a time.  The weights go over the scores'
          // first 64 columns as fp16.
          float sum = 0.f;
          const float base = kQrPLog - m;
          // The two tiles' warps of a scheduler take turns here.  Left alone they fall into
          // step, both exponentiating (half as fast each), then both waiting for the MMAs.
          if (!alone) {
            if (t == 1 || n_t > 0) ok = mbar_wait(turn_mine, (n_t - 1 + t) & 1, wctx, kSiteQuantRows);
            ++n_t;
            __syncwarp();
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t pk[16];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const float4 sg = sc[2 * k + g];
              const float f = fmaxf(sg.x * qs, 1.2e-38f), add = sg.y + base;  // f > 0: -inf stays -inf
              float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t* v = x[k] + 16 * g + 2 * e;
                const float2 z = fma2(make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])), make_float2(f, f),
                                      make_float2(add, add));
                const float2 y = make_float2(ex2_approx(z.x), ex2_approx(z.y));
                acc[e & 1] = add2(acc[e & 1], y);
                pk[8 * g + e] = qa_pack(y.x, y.y);
              }
              const float2 s2 = add2(acc[0], acc[1]);
              sum = fmaf(s2.x + s2.y, sg.z, sum);
            }
            tmem_st_x16(tS + 16 * k, pk);
          }
          if (!alone) {
            __syncwarp();
            if (lane == 0) mbar_arrive(turn_other);
          }
          if (j > u.ch0 && __any_sync(0xffffffffu, resc)) {
#pragma unroll 1
            for (int e = 0; e < D / 32; ++e) {
              tmem_ld_x32(tO + e * 32, x[0]);
              tmem_wait_ld();
              reg_fence(x[0]);
#pragma unroll
              for (int i = 0; i < 32; ++i) x[0][i] = __float_as_uint(__uint_as_float(x[0][i]) * alpha);
              tmem_st_x32(tO + e * 32, x[0]);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          l = fmaf(l, alpha, sum);
        }
        // the tile's weights are in place; its warps go on together or not at all
        ok = named_bar_and(1 + t, 128, ok);
        if (!ok) break;
        if (issuer) {
          const bool more = j + 1 < u.ch1;
          ok = issue_pv(c, j == u.ch0);
          if (!more) tc_commit(BAR(C::B_OF + t));
          else if (ok) ok = issue_qk(c + 1);
        }
      }
      if (ok) ok = mbar_wait(BAR(C::B_OF + t), n_o & 1, wctx, kSiteQuantRows);
      ++n_o;
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (ok) {
        const long long pr = u.slot * p.rows + t * 128 + row;
        const float inv = 1.f / l;
        const bool some = live && l != 0.f;
        T* out = static_cast<T*>(p.o) + u.b * p.o_sb + (long long)h * p.o_sh + (long long)qi * p.o_ss;
#pragma unroll 1
        for (int e = 0; e < D / 32; ++e) {
          uint32_t o[32];
          tmem_ld_x32(tO + e * 32, o);
          tmem_wait_ld();
          reg_fence(o);
          if (qrow < p.R) {
            if (u.whole) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                alignas(16) T v[8];
#pragma unroll
                for (int z = 0; z < 8; ++z) v[z] = from_f<T>(some ? __uint_as_float(o[i + z]) * inv : 0.f);
                *reinterpret_cast<uint4*>(out + 32 * e + i) = *reinterpret_cast<const uint4*>(v);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4*>(p.o_part + pr * D + 32 * e + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
        }
        if (!u.whole && qrow < p.R) *reinterpret_cast<float2*>(p.ml_part + 2 * pr) = make_float2(m, l);
        tc_fence_before();
      }
      cnt += u.ch1 - u.ch0;
      advance(u);
      // a wait gave up somewhere: the tile's warps end together
      if (!named_bar_and(1 + t, 128, *reinterpret_cast<volatile int*>(&s_abort) == 0)) break;
    }
    if (issuer) {  // every MMA issued is done before TMEM and shared memory are released
      tc_commit(BAR(C::B_DR));
      mbar_wait_drain(BAR(C::B_DR), 0, p.status, p.timeout_ns);
    }
    __syncwarp();
  } else {
    // ------------------------------ conversion: warp cw takes keys [32 cw, 32 cw + 32) --------
    setmaxnreg_dec<kQrRegsConvert>();
    const int cw = warp - 8;
    // piece l of row rr of an access: eight neighbouring lanes store four pieces of two rows,
    // whose swizzled chunks lie in different banks
    const int l = D == 128 ? (lane & 3) | (lane >> 1 & 4) : lane & 3;
    const int rr = D == 128 ? (lane >> 2 & 1) | (lane >> 3 & 2) : lane >> 2;
    while (w.f < w.f_end) {
      const Unit u = next_unit();
      const int* bt = p.block_tables + (long long)u.b * p.bt_stride;
      const long long mine = (long long)u.hk * p.p_sh + rr * p.p_st + 16 * l;  // this lane's piece of row 0
      // A 16-key group of this warp's two in a tile: its first row's offset, and which of its rows
      // are keys that some query sees (others are not read: their blocks may have been handed on);
      // none where it has no block.
      struct Group {
        unsigned rows;
        long long off;
      };
      // Groups 0 and 1 of tile j; lane i holds the scales of group i & 1.
      auto groups = [&](int j, Group& g0, Group& g1, float& ks, float& vs) {
        ks = vs = 0.f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          Group& x = g ? g1 : g0;
          x = Group{0u, 0};
          const int key = (u.r.c0 + j) * kQrKeys + 32 * cw + 16 * g;
          if (j >= u.ch1 || key >= u.r.khi || key + 16 <= u.r.klo) continue;
          const unsigned slot = (unsigned)key / (unsigned)p.block_size;
          const int id = __ldg(bt + slot);
          if (id < 0 || id >= p.num_blocks) continue;
          x.rows = 0xffffu >> (16 - min(16, u.r.khi - key)) & 0xffffu << max(0, u.r.klo - key);
          x.off = (long long)id * p.p_sb + (long long)(key - (int)slot * p.block_size) * p.p_st + mine;
          if ((lane & 1) == g) {
            const long long at = (long long)id * p.sc_sb + (long long)u.hk * p.sc_sh;
            ks = __ldg(p.k_scales + at);
            vs = __ldg(p.v_scales + at);
          }
        }
      };
      auto load = [&](const unsigned char* pool, const Group& g0, const Group& g1, uint4 (&x)[IT]) {
        const unsigned char* q0 = pool + g0.off;
        const unsigned char* q1 = pool + g1.off;
        if ((g0.rows & g1.rows) == 0xffffu) {
#pragma unroll
          for (int i = 0; i < IT; ++i)
            x[i] = __ldg(reinterpret_cast<const uint4*>((i < IT / 2 ? q0 : q1) + (i % (IT / 2)) * RPI * p.p_st));
          return;
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int k = (i % (IT / 2)) * RPI;  // the piece's row in its group, less rr
          x[i] = make_uint4(0, 0, 0, 0);
          if ((i < IT / 2 ? g0.rows : g1.rows) >> (k + rr) & 1u)
            x[i] = __ldg(reinterpret_cast<const uint4*>((i < IT / 2 ? q0 : q1) + k * p.p_st));
        }
      };
      // V's codes where their scale counts (scale: as the lanes hold it), else zeros.
      auto load_v = [&](Group g0, Group g1, float scale, uint4 (&x)[IT]) {
        const uint32_t none = __ballot_sync(0xffffffffu, fabsf(scale) < kQaLeastScale);
        if (none & 1u) g0.rows = 0u;
        if (none & 2u) g1.rows = 0u;
        load(p.v_pool, g0, g1, x);
      };
      Group a0, a1, b0, b1;  // of tile j, and of j + 1
      uint4 kx[IT], vx[IT];
      float ks, vs, ks_next, vs_next;
      groups(u.ch0, a0, a1, ks, vs);
      load(p.k_pool, a0, a1, kx);
      load_v(a0, a1, vs, vx);
      groups(u.ch0 + 1, b0, b1, ks_next, vs_next);
      bool ok = true;
      for (int j = u.ch0; j < u.ch1; ++j) {
        const int c = cnt + j - u.ch0, st = c & 1;
        const uint32_t k_neg = __ballot_sync(0xffffffffu, ks < 0.f);
        const uint32_t v_neg = __ballot_sync(0xffffffffu, vs < 0.f);
        if (c >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait(BAR(C::B_KE + st), (c / 2 - 1) & 1, wctx, kSiteQuantRows));
          if (!ok) break;
        }
        if (lane < 2) {
          s_scale[(c & 3) * 8 + 2 * cw + lane] =
              make_float4(fmaxf(fabsf(ks), 7.5e-37f), qa_log_scale(vs), ex2_approx(-qa_log_scale(vs)), 0.f);
        }
        if (lane == 2)
          (smem + C::OFF_MASK)[(c & 3) * 4 + cw] = (unsigned char)((a0.rows != 0u) | (a1.rows != 0u) << 1);
        const uint32_t kt = sbase + C::OFF_K + st * C::TILE;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int k = i * RPI + rr;
          qr_store<D, INT8>(kt, 32 * cw + k, l, kx[i], k_neg >> (i / (IT / 2)) & 1u ? 0x80008000u : 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(C::B_KF + st));
        load(p.k_pool, b0, b1, kx);
        if (c >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait(BAR(C::B_VE + st), (c / 2 - 1) & 1, wctx, kSiteQuantRows));
          if (!ok) break;
        }
        const uint32_t vt = sbase + C::OFF_V + st * C::TILE;
#pragma unroll
        for (int i = 0; i < IT; ++i)
          qr_store<D, INT8>(vt, 32 * cw + i * RPI + rr, l, vx[i], v_neg >> (i / (IT / 2)) & 1u ? 0x80008000u : 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(C::B_VF + st));
        load_v(b0, b1, vs_next, vx);
        a0 = b0;
        a1 = b1;
        ks = ks_next;
        vs = vs_next;
        groups(j + 2, b0, b1, ks_next, vs_next);
      }
      cnt += u.ch1 - u.ch0;
      if (!ok) break;
      advance(u);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TM_COLS);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace mlxp
