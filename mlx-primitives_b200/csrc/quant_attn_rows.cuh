// quant_attn_rows.cuh — attention of many query rows (a prompt's chunk) over an 8-bit paged cache,
// on tcgen05.
//
// The same function, precision and split of work as quant_attn.cuh (which see), for more query
// rows a pool head than its 16-row tiles are good for: a unit is 256 rows (two TMEM tiles of 128)
// of one pool head, a chunk 128 keys.  What bounds it is the tensor pipe, then the exponentials:
// 4 * 128 * 128 * D flops a tile and key chunk against 128 * 128 exponentials.
//
// The codes become fp16 (exactly) on their way into shared memory, once for both tiles: the MMA
// reads 16-bit operands, and 8-bit queries would lose what the cache kept.  Scales stay out of
// the operands: K's multiply the scores' columns (one factor a 16-key group, the block size being
// a multiple of 16), V's the weights, in fp32.  A negative K scale's sign moves into the codes, so
// that a group's maximum is its scores' maximum times the scale.
//
// Roles, 16 warps: two softmax warpgroups (a thread a row; scores from TMEM, weights back over
// them as fp16), one warpgroup that converts (codes of the next tile in registers while this one
// is stored), one warp that issues the MMAs:
//   S_t = Q_t K^T (both operands in shared memory), O_t += P_t V (P from TMEM, V as it lies).
// Tile 1's MMAs run while tile 0's weights are computed and the other way round.  QK_t of the next
// chunk is issued after PV_t of this one, so that its completion also says that O_t may be
// rescaled; that is done when a row's maximum has grown by more than 2^3 (the weights' factor is
// 2^12: they stay within fp16).
//
// K and V have two stages each in shared memory (64 KB each at D = 128) beside the 64 KB of Q.
// The scales' ring has four: a group's are written at chunk j + 3 at the earliest after both
// tiles' weights of chunk j, since K's stage is released by QK(j + 1), which follows PV(j).
// Every mbarrier wait is bounded; after one gave up nothing more is written.
#pragma once

#include "quant_attn.cuh"

namespace mlxp {

constexpr int kQrThreads = 512;
constexpr int kQrRows = 256, kQrKeys = 128;
constexpr float kQrPScale = 4096.f;
constexpr float kQrHeadroom = 3.f;
#ifndef QR_POLY
#define QR_POLY 2
#endif
// of every 8 pairs of weights, exponentiated on the FMA pipe (exp2_poly2, 7.2e-5 off at most)
constexpr int kQrPolyPerOct = QR_POLY;
constexpr int kSiteQuantRows = 13;
// registers a thread of the softmax, converting and issuing warpgroups: 128 * (2 * 184 + 104 + 40)
// = 65536 = what 512 threads of 128 are launched with
constexpr int kQrRegsSoftmax = 184, kQrRegsConvert = 104, kQrRegsIssue = 40;
static_assert(128 * (2 * kQrRegsSoftmax + kQrRegsConvert + kQrRegsIssue) <= 65536, "register split");

template <int D>
struct QrCfg {
  static constexpr int KB = D / 64;              // 128-byte column boxes
  static constexpr int BOX = 128 * 128;          // bytes of a box of 128 rows
  static constexpr int TILE = KB * BOX;          // a 128-row fp16 tile
  static constexpr int OFF_Q = 0, OFF_K = 2 * TILE, OFF_V = 4 * TILE, OFF_MISC = 6 * TILE;
  // barriers
  static constexpr int B_KF = 0, B_VF = 2, B_KE = 4, B_VE = 6, B_SF = 8, B_PF = 10, B_OF = 12, B_DR = 14, NBAR = 15;
  static constexpr int OFF_SCALE = OFF_MISC + 128;             // [4][8] float4: K, log2 V, V scale
  static constexpr int OFF_MASK = OFF_SCALE + 4 * 8 * 16;      // [4][4] bytes: which of a warp's two groups have a block
  static constexpr int OFF_TMEM = OFF_MASK + 16;
  static constexpr int SMEM = OFF_TMEM + 16 + 1024;            // slack to align the base
  static constexpr uint32_t TM_S0 = 0, TM_S1 = 128, TM_O0 = 256, TM_O1 = 256 + D, TM_COLS = 512;
};

// 16-byte chunk c of row r of a box, 128-byte swizzle.
__device__ __forceinline__ uint32_t qr_at(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// 16 codes of a row (piece l of D / 16) as fp16 into a tile.  Lanes that share a bank group write
// their two chunks in opposite order.
template <bool INT8>
__device__ __forceinline__ void qr_store(uint32_t tile, int box_bytes, int r, int l, const uint4& w, uint32_t flip) {
  uint32_t h[8];
  qa_codes<INT8>(w.x, h[0], h[1]);
  qa_codes<INT8>(w.y, h[2], h[3]);
  qa_codes<INT8>(w.z, h[4], h[5]);
  qa_codes<INT8>(w.w, h[6], h[7]);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] ^= flip;
  const uint32_t base = tile + (l >> 2) * box_bytes;
  const bool odd = l & 4;
  const uint32_t a0 = base + qr_at(r, 2 * (l & 3) + (odd ? 1 : 0)), a1 = base + qr_at(r, 2 * (l & 3) + (odd ? 0 : 1));
  st_shared_v4(a0, odd ? h[4] : h[0], odd ? h[5] : h[1], odd ? h[6] : h[2], odd ? h[7] : h[3]);
  st_shared_v4(a1, odd ? h[0] : h[4], odd ? h[1] : h[5], odd ? h[2] : h[6], odd ? h[3] : h[7]);
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
      mbar_init(BAR(C::B_KE + i), 1);
      mbar_init(BAR(C::B_VE + i), 1);
      mbar_init(BAR(C::B_SF + i), 1);
      mbar_init(BAR(C::B_PF + i), 128);
      mbar_init(BAR(C::B_OF + i), 1);
    }
    mbar_init(BAR(C::B_DR), 1);
    fence_mbar_init();
  }
  QaWork w = qa_find_work<NT, kQrKeys, kQrThreads>(p);
  if (!w.any) return;
  if (warp == 12) tmem_alloc(sbase + C::OFF_TMEM, C::TM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<const volatile uint32_t*>(smem + C::OFF_TMEM);
  if (warp == 12) tmem_relinquish();
  const long long f_begin = w.f;
  float4* s_scale = reinterpret_cast<float4*>(smem + C::OFF_SCALE);
  const uint32_t* s_mask = reinterpret_cast<const uint32_t*>(smem + C::OFF_MASK);
  int cnt = 0;                 // key tiles this CTA has gone through, every role's own count

  // The units' loop, the same for every role: before(unit) by all threads, then body(unit), with
  // CTA-wide barriers around.
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
    // ------------------------------ softmax, a thread a row of tile t ------------------------
    setmaxnreg_inc<kQrRegsSoftmax>();
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    int n_s = 0, n_o = 0;  // score tiles and units seen
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + (t ? C::TM_S1 : C::TM_S0);
    const uint32_t tO = tmem + lane_off + (t ? C::TM_O1 : C::TM_O0);
    while (w.f < w.f_end) {
      const Unit u = next_unit();
      const int qrow = u.r0 + t * 128 + row, qi = qrow / p.G;
      const bool live = qrow < p.R && qi < u.r.qlen;
      const int h = u.hk * p.G + qrow - qi * p.G;
      int lo = 0, hi = 0;
      if (live) qa_row_range(p, u.r.ctx, u.r.qlen, qi, lo, hi);
      // the row, scaled by a power of two, as fp16
      float qs;
      {
        const T* src = static_cast<const T*>(p.q) + u.b * p.q_sb + (long long)h * p.q_sh + (long long)qi * p.q_ss;
        float mx = 0.f;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          if (live)
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              const uint4 x = *reinterpret_cast<const uint4*>(src + 8 * c);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t v = e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w;
                mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(v << 16)), fabsf(__uint_as_float(v & 0xffff0000u))));
              }
            }
        }
        float up = 1.f;
        const unsigned E = __float_as_uint(mx) >> 23;
        if (E >= 1 && E <= 253) up = __uint_as_float(E << 23);
        const float down = __uint_as_float((254u - (__float_as_uint(up) >> 23)) << 23);
        qs = up * p.scale_log2;
        const uint32_t dst = sbase + C::OFF_Q + t * C::TILE;
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (live) x = *reinterpret_cast<const uint4*>(src + 8 * c);
          if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = qa_pack(__uint_as_float(v[e] << 16) * down, __uint_as_float(v[e] & 0xffff0000u) * down);
            x = make_uint4(v[0], v[1], v[2], v[3]);
          }
          st_shared_v4(dst + (c >> 3) * C::BOX + qr_at(row, c & 7), x.x, x.y, x.z, x.w);
        }
      }
      fence_proxy_async_smem();
      __syncthreads();  // Q is in place
      float m = -1e30f, l = 0.f;
      bool ok = true;
      if (t < u.tiles) {
        for (int j = u.ch0; j < u.ch1; ++j) {
          const int c = cnt + j - u.ch0;
          ok = __all_sync(0xffffffffu, mbar_wait(BAR(C::B_SF + t), n_s & 1, wctx, kSiteQuantRows));
          if (!ok) break;
          ++n_s;
          tc_fence_after();
          const int key0 = (u.r.c0 + j) * kQrKeys;
          const float4* sc = s_scale + (c & 3) * 8;
          uint32_t groups = s_mask[c & 3];  // bits 0, 1 of each byte
          groups = (groups & 3u) | (groups >> 6 & 12u) | (groups >> 12 & 48u) | (groups >> 18 & 192u);
          float s[128];
          {
            uint32_t ra[32], rb[32];
            tmem_ld_x32(tS, ra);
            tmem_ld_x32(tS + 32, rb);
            tmem_wait_ld();
            reg_fence(ra);
            reg_fence(rb);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              s[e] = __uint_as_float(ra[e]);
              s[32 + e] = __uint_as_float(rb[e]);
            }
            tmem_ld_x32(tS + 64, ra);
            tmem_ld_x32(tS + 96, rb);
            tmem_wait_ld();
            reg_fence(ra);
            reg_fence(rb);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              s[64 + e] = __uint_as_float(ra[e]);
              s[96 + e] = __uint_as_float(rb[e]);
            }
          }
          if (key0 < u.r.flo || key0 + kQrKeys > u.r.fhi || groups != 0xffu) {
            const int from = lo - key0;
            const unsigned width = (unsigned)max(hi - lo, 0);
#pragma unroll
            for (int e = 0; e < 128; ++e)
              s[e] = (unsigned)(e - from) < width && (groups >> (e >> 4) & 1u) ? s[e] : -INFINITY;
          }
          float mloc = -INFINITY;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            float mx = fmaxf(s[16 * g], s[16 * g + 1]);
#pragma unroll
            for (int e = 2; e < 16; e += 2) mx = max3(mx, s[16 * g + e], s[16 * g + e + 1]);
            mloc = fmaxf(mloc, fmaf(mx, fmaxf(sc[g].x * qs, 1.2e-38f), sc[g].y));
          }
          const bool resc = mloc > m + kQrHeadroom;
          float alpha = 1.f;
          if (resc) {
            alpha = ex2_approx(m - mloc);
            m = mloc;
          }
          const float2 negm = make_float2(-m, -m);
          float2 acc = make_float2(0.f, 0.f);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t pk[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const int g = 4 * hf + e / 8;
              const float f = fmaxf(sc[g].x * qs, 1.2e-38f), vs = sc[g].z;  // > 0: -inf stays -inf
              const float2 x = fma2(make_float2(s[64 * hf + 2 * e], s[64 * hf + 2 * e + 1]), make_float2(f, f), negm);
              float2 y;
              if ((e & 7) < kQrPolyPerOct) {
                y = exp2_poly2(x);
              } else {
                y.x = ex2_approx(x.x);
                y.y = ex2_approx(x.y);
              }
              acc = add2(acc, y);
              y = mul2(y, make_float2(vs, vs));
              pk[e] = qa_pack(y.x, y.y);
            }
            tmem_st_x32(tS + 32 * hf, pk);
          }
          if (j > u.ch0 && __any_sync(0xffffffffu, resc)) {
#pragma unroll 1
            for (int e = 0; e < D / 32; ++e) {
              uint32_t o[32];
              tmem_ld_x32(tO + e * 32, o);
              tmem_wait_ld();
              reg_fence(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_x32(tO + e * 32, o);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(BAR(C::B_PF + t));
          l = l * alpha + acc.x + acc.y;
        }
        if (ok) {
          ok = __all_sync(0xffffffffu, mbar_wait(BAR(C::B_OF + t), n_o & 1, wctx, kSiteQuantRows));
          ++n_o;
          tc_fence_after();
        }
        if (ok) {
          const long long pr = u.slot * p.rows + t * 128 + row;
          const float inv = 1.f / (l * kQrPScale);
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
                  for (int x = 0; x < 8; ++x) v[x] = from_f<T>(some ? __uint_as_float(o[i + x]) * inv : 0.f);
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
      }
      cnt += u.ch1 - u.ch0;
      if (__syncthreads_or(s_abort != 0)) break;  // the unit's TMEM and shared memory are free
      advance(u);
    }
  } else if (warp < 12) {
    // ------------------------------ conversion: warp cw takes keys [32 cw, 32 cw + 32) --------
    setmaxnreg_dec<kQrRegsConvert>();
    const int cw = warp - 8, l = lane % LR, rr = lane / LR;
    while (w.f < w.f_end) {
      const Unit u = next_unit();
      __syncthreads();
      const int* bt = p.block_tables + (long long)u.b * p.bt_stride;
      const long long mine = (long long)u.hk * p.p_sh + rr * p.p_st + 16 * l;  // this lane's piece of row 0
      // A 16-key group of this warp's two in a tile: its pool block and first row's offset, and
      // how many of its rows are keys.
      struct Group {
        int id, rows;
        long long off;
      };
      auto group = [&](int j, int g) {
        Group x{-1, 0, 0};
        const int key = (u.r.c0 + j) * kQrKeys + 32 * cw + 16 * g;
        if (j >= u.ch1 || key >= u.r.khi) return x;
        const unsigned slot = (unsigned)key / (unsigned)p.block_size;
        const int id = __ldg(bt + slot);
        if (id < 0 || id >= p.num_blocks) return x;
        x.id = id;
        x.rows = min(16, u.r.khi - key);
        x.off = (long long)id * p.p_sb + (long long)(key - (int)slot * p.block_size) * p.p_st + mine;
        return x;
      };
      auto load = [&](const unsigned char* pool, const Group& g0, const Group& g1, uint4 (&x)[IT]) {
        const unsigned char* q0 = pool + g0.off;
        const unsigned char* q1 = pool + g1.off;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int k = (i % (IT / 2)) * RPI;  // the piece's row in its group, less rr
          x[i] = make_uint4(0, 0, 0, 0);
          if (k + rr < (i < IT / 2 ? g0.rows : g1.rows))
            x[i] = __ldg(reinterpret_cast<const uint4*>((i < IT / 2 ? q0 : q1) + k * p.p_st));
        }
      };
      // lanes 0 and 1 hold the scales of the two groups
      auto scales = [&](const Group& g0, const Group& g1, float& ks, float& vs) {
        const int id = lane == 0 ? g0.id : lane == 1 ? g1.id : -1;
        ks = vs = 0.f;
        if (id < 0) return;
        const long long at = (long long)id * p.sc_sb + (long long)u.hk * p.sc_sh;
        ks = __ldg(p.k_scales + at);
        vs = __ldg(p.v_scales + at);
      };
      Group a0 = group(u.ch0, 0), a1 = group(u.ch0, 1);  // of tile j, and of j + 1
      Group b0 = group(u.ch0 + 1, 0), b1 = group(u.ch0 + 1, 1);
      uint4 kx[IT], vx[IT];
      float ks, vs, ks_next, vs_next;
      load(p.k_pool, a0, a1, kx);
      load(p.v_pool, a0, a1, vx);
      scales(a0, a1, ks, vs);
      bool ok = true;
      for (int j = u.ch0; j < u.ch1; ++j) {
        const int c = cnt + j - u.ch0, st = c & 1;
        scales(b0, b1, ks_next, vs_next);
        const uint32_t neg = __ballot_sync(0xffffffffu, ks < 0.f);
        if (c >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait(BAR(C::B_KE + st), (c / 2 - 1) & 1, wctx, kSiteQuantRows));
          if (!ok) break;
        }
        if (lane < 2) {
          s_scale[(c & 3) * 8 + 2 * cw + lane] =
              make_float4(fmaxf(fabsf(ks), 7.5e-37f), qa_log_scale(vs), vs * kQrPScale, 0.f);
        }
        if (lane == 2)
          (smem + C::OFF_MASK)[(c & 3) * 4 + cw] = (unsigned char)((a0.id >= 0) | (a1.id >= 0) << 1);
        const uint32_t kt = sbase + C::OFF_K + st * C::TILE;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int k = i * RPI + rr;
          qr_store<INT8>(kt, C::BOX, 32 * cw + k, l, kx[i], neg >> (k >> 4) & 1u ? 0x80008000u : 0u);
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
        for (int i = 0; i < IT; ++i) qr_store<INT8>(vt, C::BOX, 32 * cw + i * RPI + rr, l, vx[i], 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(C::B_VF + st));
        load(p.v_pool, b0, b1, vx);
        a0 = b0;
        a1 = b1;
        b0 = group(j + 2, 0);
        b1 = group(j + 2, 1);
        ks = ks_next;
        vs = vs_next;
      }
      cnt += u.ch1 - u.ch0;
      if (__syncthreads_or(s_abort != 0)) break;
      advance(u);
    }
  } else {
    // ------------------------------ MMA issue (warp 12, lane 0; warps 13-15 keep step) --------
    setmaxnreg_dec<kQrRegsIssue>();
    constexpr uint32_t idesc_qk = make_idesc_f16(128, 128, false, false);
    constexpr uint32_t idesc_pv = make_idesc_f16(128, D, false, true);
    const uint32_t q_lo = ((sbase + C::OFF_Q) >> 4) | (1u << 16);
    const uint32_t k_lo = ((sbase + C::OFF_K) >> 4) | (1u << 16);
    const uint32_t v_lo = ((sbase + C::OFF_V) >> 4) | ((uint32_t)(C::BOX >> 4) << 16);
    auto issue_qk = [&](int t, int st) {
      const uint32_t d = tmem + (t ? C::TM_S1 : C::TM_S0);
      const uint32_t a = q_lo + (uint32_t)(t * C::TILE >> 4), b = k_lo + (uint32_t)(st * C::TILE >> 4);
#pragma unroll
      for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ss(d, sdesc(a + (uint32_t)((kb * C::BOX + kk * 32) >> 4)),
                 sdesc(b + (uint32_t)((kb * C::BOX + kk * 32) >> 4)), idesc_qk, (kb | kk) ? 1u : 0u);
    };
    auto issue_pv = [&](int t, int st, bool acc) {
      const uint32_t d = tmem + (t ? C::TM_O1 : C::TM_O0), a = tmem + (t ? C::TM_S1 : C::TM_S0);
      const uint32_t b = v_lo + (uint32_t)(st * C::TILE >> 4);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        mma_ts(d, a + kk * 8, sdesc(b + (uint32_t)(kk * 16 * 128 >> 4)), idesc_pv, (acc || kk > 0) ? 1u : 0u);
    };
    int n_p[2] = {0, 0};  // weight tiles seen
    while (w.f < w.f_end) {
      const Unit u = next_unit();
      __syncthreads();
      if (warp == 12 && lane == 0) {
        const int n = u.ch1 - u.ch0;
        bool ok = mbar_wait(BAR(C::B_KF + (cnt & 1)), (cnt >> 1) & 1, wctx, kSiteQuantRows);
        if (ok) {
          tc_fence_after();
          for (int t = 0; t < u.tiles; ++t) {
            issue_qk(t, cnt & 1);
            tc_commit(BAR(C::B_SF + t));
          }
          tc_commit(BAR(C::B_KE + (cnt & 1)));
        }
        for (int i = 0; i < n && ok; ++i) {
          const int c = cnt + i, st = c & 1, sn = st ^ 1;
          const bool more = i + 1 < n;
          ok = mbar_wait(BAR(C::B_VF + st), (c >> 1) & 1, wctx, kSiteQuantRows);
          if (ok && more) ok = mbar_wait(BAR(C::B_KF + sn), ((c + 1) >> 1) & 1, wctx, kSiteQuantRows);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= u.tiles || !ok) break;
            ok = mbar_wait(BAR(C::B_PF + t), n_p[t] & 1, wctx, kSiteQuantRows);
            if (!ok) break;
            ++n_p[t];
            tc_fence_after();
            issue_pv(t, st, i > 0);
            if (!more) tc_commit(BAR(C::B_OF + t));
            if (t == u.tiles - 1) tc_commit(BAR(C::B_VE + st));
            if (more) {
              issue_qk(t, sn);
              tc_commit(BAR(C::B_SF + t));
            }
          }
          if (ok && more) tc_commit(BAR(C::B_KE + sn));
        }
      }
      __syncwarp();
      cnt += u.ch1 - u.ch0;
      if (__syncthreads_or(s_abort != 0)) break;
      advance(u);
    }
    if (warp == 12 && lane == 0) {  // every MMA issued is done before TMEM and smem are released
      tc_commit(BAR(C::B_DR));
      mbar_wait_drain(BAR(C::B_DR), 0, p.status, p.timeout_ns);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TM_COLS);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace mlxp
