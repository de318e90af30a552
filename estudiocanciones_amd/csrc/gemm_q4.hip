// Products of many rows with 4-bit weights in groups (gfx950 MFMA).  Layout: q4.h.
//
//   y[m, n] = fp16(sum_g s[n, g] sum_{k in g} x[m, k] (u[n, k] - z[n, g]) (+ res[m, n])), or silu(a) b of row pairs
//
// A workgroup of NW = WN x WM waves computes BN = 32 WN FT features x BM = 32 WM RT rows; a wave FT x RT tiles of
// v_mfma_f32_32x32x16_f16 with x as the first operand, so that a lane holds one feature.  The codes are multiplied as exact
// halves u - z; the scales stay in fp32.  A sum is kept in units of the scale of the group it is in: before the next group
// begins it is multiplied by the quotient of the two scales, and by the last one at the end.  So the accumulators of the
// matrix instruction are all the state there is, and nothing is rounded to fp16 on the way.
//
// K advances in 64-wide chunks through an NS-stage ring in LDS, loaded by LDS DMA: x rows with their 16-byte pieces swizzled
// by row (x_swz), codes as packed, scales of the chunk's groups.
//
// 2048 x 16384 x 3072 with SiLU: 175 to 181 us for a few launches, 200 to 207 for sixty in a row, when the clock has fallen: 1.15 and
// 1.0 PFLOP/s (the library's product of fp16 matrices of these sizes: 153 and 172 to 177), matrix units 64% busy; about 4 vector
// instructions hide behind each product, the rest of the conversion (30 us), the scales (15 to 20) and the results' way out (10) add up.
// 187 x 3072 x 8192: 21 us, of it 4 the join; there the latency of a step bounds (1.3 us for 0.7 of products).
#include "gemm_core.h"
#include "q4.h"

#include <type_traits>

namespace ecd {

template <bool ZP, int GS, int WN, int WM, int WK, int FT, int RT, int NS>
struct Q4Tile {
  static constexpr int NW = WN * WM, BN = 32 * WN * FT, BM = 32 * WM * RT;
  static constexpr int TB = BN / 32;                      // 32-feature tiles of the block
  static constexpr int CB = TB * 1024 / NW;               // bytes of codes a wave loads per chunk
  static constexpr int CI = CB < 1024 ? 1 : CB / 1024;    // in so many instructions
  static constexpr int SB = 64 * (ZP ? 2 : 1) * GS;       // bytes of scales of a tile and chunk
  static constexpr int SW = TB * SB / NW;                 // of them a wave's
  static constexpr int XI = BM / 8 / NW;                  // x instructions of a wave, 8 rows each
  static constexpr int PER = CI + XI + 1;
  static_assert(CB >= 16 && XI * 8 * NW == BM && SW >= 16 && SW <= 1024, "whole instructions for each wave");
  static_assert(NS >= 2 && PER * (NS - 1) < 64, "vmcnt range");
  static constexpr int XS = BM * 128, CS = TB * 1024, CHK = XS + CS + (TB * SB + 127) / 128 * 128;  // bytes of a chunk
  static constexpr int STG = WK * CHK;                    // and of a stage
  static constexpr int EW = BN + 4, ER = 32 * WM * EW;    // the epilogue's fp32 rows
  static constexpr int EP = WK * ER * 4;
  static constexpr int LDS = NS * STG > EP ? NS * STG : EP;

  // The sums of features n0 .., rows m0 .. over chunks c0 .. c1 - 1 (of x: with two parts twice those of the codes), in acc:
  // lane l holds feature 32 (wn FT + ft) + (l & 31) of
  // rows 32 (wm RT + rt) + 8 (i / 4) + 4 (l / 32) + i % 4, i the register.
  static __device__ __forceinline__ void run(char* lds, const Q4Args& a, int n0, int m0, int c0, int c1, f32x16 (&acc)[FT][RT]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wv = wave % NW, kg = wave / NW, wn = wv % WN, wm = wv / WN, h = lane >> 5;
    lds += kg * CHK;
    c0 += kg;  // the group's chunks: c0, c0 + WK, ..
    const int nch = a.K >> 6, ng = ((a.K - 1) >> a.lg) + 1, last = (a.N - 1) >> 5, t0 = n0 >> 5;
    // sources: uniform bases that advance with the chunk, and each lane's offset
    const char* xb = (const char*)(a.x + (long)m0 * a.ldx) + 128L * c0;
    const char* cb = (const char*)a.codes + (long)t0 * nch * 1024;
    const char* sb = (const char*)a.scales + (long)t0 * ng * (ZP ? 128 : 64);
    uint32_t xoff[XI], coff[CI], soff;
#pragma unroll
    for (int j = 0; j < XI; ++j) {
      const int r = 8 * (wv + NW * j) + (lane >> 3);  // rows past the last: the last, and not stored
      xoff[j] = (uint32_t)((long)min(r, a.M - 1 - m0) * a.ldx * 2) + 16 * ((lane & 7) ^ x_swz(r));
    }
#pragma unroll
    for (int j = 0; j < CI; ++j) {
      const int b = wv * CB + 1024 * j + 16 * lane;  // byte of the stage's codes
      coff[j] = (uint32_t)(min(t0 + (b >> 10), last) - t0) * (nch * 1024u) + (b & 1023);
    }
    {
      const int b = wv * SW + 16 * lane;
      soff = (uint32_t)(min(t0 + b / SB, last) - t0) * (ng * (ZP ? 128u : 64u)) + b % SB;
    }
    const uint32_t lx = lds_addr(lds) + wv * 1024, lc = lds_addr(lds) + XS + wv * CB, ls = lds_addr(lds) + XS + CS + wv * SW;
    int cl = c0;  // the next chunk to load
    auto load = [&](int st) {
      static_for<0, XI>([&](auto J) { lds_dma16_at<NW * J.value * 1024>(xb, xoff[J.value], lx + st * STG); });
      if (CB >= 1024 || 16 * lane < CB)
        static_for<0, CI>([&](auto J) { lds_dma16_at<J.value * 1024>(cb + 1024L * (cl >> a.two), coff[J.value], lc + st * STG); });
      if (16 * lane < SW) lds_dma16_at<0>(sb + (long)((64 * (cl >> a.two)) >> a.lg) * (ZP ? 128 : 64), soff, ls + st * STG);
      xb += WK * 128;
      cl += WK;
    };
    static_for<0, FT * RT>([&](auto I) { acc[I.value / RT][I.value % RT] = (f32x16)(0.f); });

    // fragments of half a chunk: k-steps S = 0, 1 of its 32 k
    struct Half {
      f16x8 w[2][FT], x[2][RT];
    };
    using Scale = std::conditional_t<ZP, f16x2, f16>;
    u32x4 code[FT];     // of the chunk whose halves are dequantised next
    Scale sz[FT][GS];   // its scales, with zero points (s, 1024 + z)
    float was[FT];
    int xfo[4];  // x fragment of half H, k-step S, row tile 0
    static_for<0, 4>([&](auto I) {
      const int r = wm * RT * 32 + (lane & 31);
      xfo[I.value] = r * 128 + 16 * ((4 * (I.value >> 1) + 2 * h + (I.value & 1)) ^ x_swz(lane & 31));
    });
    auto read_w = [&](auto F, const char* base) {
      constexpr int ft = F.value;
      code[ft] = *(const u32x4*)(base + XS + (wn * FT + ft) * 1024 + 16 * lane);
    };
    auto read_s = [&](auto F, const char* base) {
      constexpr int ft = F.value;
#pragma unroll
      for (int H = 0; H < GS; ++H)
        sz[ft][H] = *(const Scale*)(base + XS + CS + (wn * FT + ft) * SB + H * (SB / GS) + (lane & 31) * (ZP ? 4 : 2));
    };
    auto scale = [&](int ft, int H) {
      if constexpr (ZP) return (float)sz[ft][H].x; else return (float)sz[ft][H];
    };
    auto read_x = [&](auto I, auto HH, const char* base, Half& f) {
      constexpr int S = I.value / RT, rt = I.value % RT;
      f.x[S][rt] = *(const f16x8*)(base + xfo[2 * HH.value + S] + rt * 4096);
    };
    auto dequant = [&](auto I, auto HH, Half& f) {
      constexpr int S = I.value / FT, ft = I.value % FT, H = HH.value;
      f16x2 c0 = {(f16)-1032.f, (f16)-1032.f}, c1 = {(f16)-72.f, (f16)-72.f};
      if constexpr (ZP) {
        const f16 z = -sz[ft][H & (GS - 1)].y;
        c0 = (f16x2){z, z};
        c1 = c0 + (f16x2){(f16)960.f, (f16)960.f};
      }
      f.w[S][ft] = q4_halves(code[ft][2 * S + H], c0, c1);
    };
    // The products of half H (fragments f, scales q of the last units where `turn`), with the reads and the conversion of the next half
    // (fragments nf of stage base) and DMA instructions D0 .. D1 - 1 of a later chunk between them, so that
    // the matrix unit has work while they issue.
    constexpr int NM = 2 * FT * RT;
    auto half = [&](const Half& f, bool turn, const float (&q)[FT], auto NH, const char* base, Half& nf) {
      constexpr int nh = decltype(NH)::value;
      if constexpr (nh == 0) static_for<0, FT>([&](auto F) { read_w(F, base); });
      if constexpr (nh == 0) static_for<0, FT>([&](auto F) { read_s(F, base); });
      if (turn)
        static_for<0, FT * RT>([&](auto I) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[I.value / RT][I.value % RT][i] *= q[I.value / RT];
        });
      __builtin_amdgcn_s_setprio(1);  // (2048 x 16384 x 3072: 181 -> 173 us)
      static_for<0, NM>([&](auto I) {
        constexpr int m = I.value, S = m / (FT * RT), ft = m % (FT * RT) / RT, rt = m % RT;
        acc[ft][rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.x[S][rt], f.w[S][ft], acc[ft][rt], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        constexpr int RH = NM / 2;  // reads in the first half of the products, the conversion from there on
        if constexpr (m < RH)
          static_for<m * 2 * RT / RH, (m + 1) * 2 * RT / RH>([&](auto J) { read_x(J, NH, base, nf); });
        if constexpr (m >= RH)
          static_for<(m - RH) * 2 * FT / (NM - RH), (m - RH + 1) * 2 * FT / (NM - RH)>([&](auto J) { dequant(J, NH, nf); });
        __builtin_amdgcn_sched_barrier(0);
      });
      __builtin_amdgcn_s_setprio(0);
    };

    const int nc = c0 < c1 ? (c1 - c0 + WK - 1) / WK : 0, most = (c1 - c0 + kg + WK - 1) / WK;  // of the group, of the first
    for (int s = 0; s < NS; ++s)
      if (s < nc) load(s);
    wait_chunk<PER, NS - 1, false>(max(min(NS - 1, nc - 1), 0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Half fa, fb;
    float q[FT];
    static_for<0, FT>([&](auto F) {
      read_w(F, lds);
      read_s(F, lds);
      was[F.value] = nc > 0 ? scale(F.value, 0) : 1.f;  // (a group without a chunk: nothing was loaded)
      q[F.value] = 1.f;
    });
    static_for<0, 2 * RT>([&](auto I) { read_x(I, IC<0>{}, lds, fa); });
    static_for<0, 2 * FT>([&](auto I) { dequant(I, IC<0>{}, fa); });
    // what the sums are multiplied by before the products of half H of chunk c, whose scales are in sz
    auto turn = [&](int c, int H) {
      if (GS == 2 ? (c == 0 && H == 0) : (H != 0 || c == 0 || (WK == 1 && ((c0 + c) << 6 & ((1 << (a.lg + a.two)) - 1))))) return false;
      static_for<0, FT>([&](auto F) {
        const float s = scale(F.value, H & (GS - 1));
        q[F.value] = was[F.value] * __builtin_amdgcn_rcpf(s);
        was[F.value] = s;
      });
      return true;
    };
    const float one[FT] = {};
    if (nc > 0) half(fa, false, one, IC<1>{}, lds, fb);
    int st = 0;  // the stage of chunk c
    for (int c = 0; c < nc - 1; ++c) {
      // chunk c + 1 landed for this wave, and its reads of chunk c are done; then it is there for all, and the stage of chunk c free
      wait_chunk<PER, NS - 2, true>(min(NS - 2, nc - 2 - c));
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int sn = st + 1 == NS ? 0 : st + 1;
      const char* base = lds + sn * STG;
      const bool t1 = GS == 2 && turn(c, 1);
      if (c + NS < nc) load(st);
      half(fb, t1, q, IC<0>{}, base, fa);
      const bool t0 = turn(c + 1, 0);
      half(fa, t0, q, IC<1>{}, base, fb);
      st = sn;
    }
    if (WK > 1 && nc < most && most > 1) __builtin_amdgcn_s_barrier();  // (the last step is the first groups')
    if (nc > 0) {
      const bool t1 = GS == 2 && turn(nc - 1, 1);
      half(fb, t1, q, IC<1>{}, lds, fa);  // (its reads are never used)
    }
    static_for<0, FT * RT>([&](auto I) {
      constexpr int ft = I.value / RT, rt = I.value % RT;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[ft][rt][i] *= was[ft];
    });
  }

  // Rows 32 (wm RT + rt) .. of every wave's tile through LDS, then row by row in pieces of 8 features: f(row of the block, piece, sums)
  template <typename F>
  static __device__ __forceinline__ void rows(char* lds, f32x16 (&acc)[FT][RT], F&& f) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wv = wave % NW, kg = wave / NW, wn = wv % WN, wm = wv / WN;
    float* const t = (float*)lds;
    constexpr int W = EW;
    static_for<0, RT>([&](auto R) {
      constexpr int rt = R.value;
      __syncthreads();
      static_for<0, FT>([&](auto T) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          t[kg * ER + (wm * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)) * W + (wn * FT + T.value) * 32 + (lane & 31)] = acc[T.value][rt][i];
      });
      __syncthreads();
      constexpr int PR = BN / 8;
      for (int i = threadIdx.x; i < 32 * WM * PR; i += 64 * NW * WK) {
        const int r = i / PR, p = i % PR;
        f32x4 u = *(const f32x4*)(t + r * W + 8 * p), v = *(const f32x4*)(t + r * W + 8 * p + 4);
#pragma unroll
        for (int g = 1; g < WK; ++g) {
          u = u + *(const f32x4*)(t + g * ER + r * W + 8 * p);
          v = v + *(const f32x4*)(t + g * ER + r * W + 8 * p + 4);
        }
        f((r >> 5) * (32 * RT) + 32 * rt + (r & 31), p, u, v);
      }
    });
  }
};

// 8 sums of features nb .. of row m (fewer at the end of a row): residual or SiLU, and the one rounding
__device__ __forceinline__ void q4_finish(const Q4Args& a, int m, int nb, f32x4 u, f32x4 v) {
  if (m >= a.M || nb >= a.N) return;
  const bool full = nb + 8 <= a.N;
  if (a.silu) {
    const f16x4 o = {(f16)silu_mul(u[0], u[1]), (f16)silu_mul(u[2], u[3]), (f16)silu_mul(v[0], v[1]), (f16)silu_mul(v[2], v[3])};
    f16* const y = a.y + (long)m * a.ldy + nb / 2;
    if (full) {
      *(f16x4u*)y = o;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (nb + 2 * j < a.N) y[j] = o[j];
    }
    return;
  }
  f16* const y = a.y + (long)m * a.ldy + nb;
  const f16* const r = a.res ? a.res + (long)m * a.ldr + nb : nullptr;
  f16x8 o = {0, 0, 0, 0, 0, 0, 0, 0};
  if (r) {
    if (full)
      o = *(const f16x8u*)r;
    else
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (nb + j < a.N) o[j] = r[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[j] = (f16)(u[j] + (float)o[j]);
    o[4 + j] = (f16)(v[j] + (float)o[4 + j]);
  }
  if (full)
    *(f16x8u*)y = o;
  else
    store_tail(y, nullptr, o, a.N - nb);
}

template <bool ZP, int GS, int WN, int WM, int WK, int FT, int RT, int NS>
__global__ __launch_bounds__(64 * WN * WM * WK, 2) void gemm_q4_kernel(const Q4Args a, int nfb, int nmb) {
  using T = Q4Tile<ZP, GS, WN, WM, WK, FT, RT, NS>;
  __shared__ __align__(16) char lds[T::LDS];
  int fb, mb;
  GemmTile<true, false, 1, 1, 1, 1, 2>::block(nfb, nmb, fb, mb);
  const int n0 = fb * T::BN, m0 = mb * T::BM;
  f32x16 acc[FT][RT];
  T::run(lds, a, n0, m0, 0, a.K >> 6 << a.two, acc);
  T::rows(lds, acc, [&](int r, int p, f32x4 u, f32x4 v) { q4_finish(a, m0 + r, n0 + 8 * p, u, v); });
}

// K split over gridDim.y: fp32 sums [gridDim.y][M][N]
template <bool ZP, int GS, int WN, int WM, int WK, int FT, int RT, int NS>
__global__ __launch_bounds__(64 * WN * WM * WK, 2) void gemm_q4_partial_kernel(const Q4Args a, int nfb, int nmb, float* __restrict__ ws) {
  using T = Q4Tile<ZP, GS, WN, WM, WK, FT, RT, NS>;
  __shared__ __align__(16) char lds[T::LDS];
  int fb, mb;
  GemmTile<true, false, 1, 1, 1, 1, 2>::block(nfb, nmb, fb, mb);
  const int n0 = fb * T::BN, m0 = mb * T::BM, nch = a.K >> 6 << a.two, z = blockIdx.y, ks = gridDim.y;
  f32x16 acc[FT][RT];
  T::run(lds, a, n0, m0, (int)((long)nch * z / ks), (int)((long)nch * (z + 1) / ks), acc);
  const long ld = (a.N + 7) & ~7L;
  T::rows(lds, acc, [&](int r, int p, f32x4 u, f32x4 v) {
    const int m = m0 + r, nb = n0 + 8 * p;
    if (m >= a.M || nb >= ld) return;
    float* const d = ws + ((long)z * a.M + m) * ld + nb;
    *(f32x4*)d = u;
    *(f32x4*)(d + 4) = v;
  });
}

// the sums of the parts in order, and the finish
__global__ __launch_bounds__(256) void gemm_q4_join_kernel(const Q4Args a, const float* __restrict__ ws, int ks) {
  const long ld = (a.N + 7) & ~7L, per = ld >> 3, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= per * a.M) return;
  const int m = (int)(i / per), nb = (int)(i - m * per) * 8;
  const float* p = ws + (long)m * ld + nb;
  const long step = (long)a.M * ld;
  f32x4 u = *(const f32x4*)p, v = *(const f32x4*)(p + 4);
#pragma unroll 4
  for (int z = 1; z < ks; ++z) {
    u = u + *(const f32x4*)(p + z * step);
    v = v + *(const f32x4*)(p + z * step + 4);
  }
  q4_finish(a, m, nb, u, v);
}

template <bool ZP, int GS, int WN, int WM, int WK, int FT, int RT, int NS>
static int launch(const Q4Args& a, float* ws, int ks, hipStream_t st, bool go) {
  using T = Q4Tile<ZP, GS, WN, WM, WK, FT, RT, NS>;
  const int nfb = (a.N + T::BN - 1) / T::BN, nmb = (a.M + T::BM - 1) / T::BM;
  const long pieces = ((a.N + 7L) >> 3) * a.M;
  if ((long)nfb * nmb > 0x7FFFFFFFL || T::BM * a.ldx * 2 > 0x7FFFFFFFL || (long)T::TB * a.K * 16 > 0x7FFFFFFFL ||
      (ks > 1 && (pieces + 255) / 256 > 0x7FFFFFFFL))
    return ECD_ENOTSUP;
  if (!go) return ECD_OK;
  const dim3 block(64 * T::NW * WK);
  if (ks == 1) {
    hipLaunchKernelGGL((gemm_q4_kernel<ZP, GS, WN, WM, WK, FT, RT, NS>), dim3(nfb * nmb), block, 0, st, a, nfb, nmb);
    return ecd_launch_status();
  }
  hipLaunchKernelGGL((gemm_q4_partial_kernel<ZP, GS, WN, WM, WK, FT, RT, NS>), dim3(nfb * nmb, ks), block, 0, st, a, nfb, nmb, ws);
  hipLaunchKernelGGL(gemm_q4_join_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, st, a, ws, ks);
  return ecd_launch_status();
}

template <bool ZP, int GS>
static int by_tile(const Q4Args& a, int tile, float* ws, int ks, hipStream_t st, bool go) {
  switch (tile) {
    case 1: return launch<ZP, GS, 4, 1, 1, 2, 4, 3>(a, ws, ks, st, go);
    case 2: return launch<ZP, GS, 4, 1, 1, 2, 3, 3>(a, ws, ks, st, go);
    case 3: return launch<ZP, GS, 4, 1, 2, 1, 2, 3>(a, ws, ks, st, go);
    case 4: return launch<ZP, GS, 2, 1, 4, 2, 3, 2>(a, ws, ks, st, go);
    case 5: return launch<ZP, GS, 2, 1, 4, 1, 1, 4>(a, ws, ks, st, go);
    case 6: return launch<ZP, GS, 2, 1, 4, 1, 2, 3>(a, ws, ks, st, go);
    default: return ECD_EINVAL;
  }
}

int gemm_q4(const Q4Args& a, bool zp, int tile, float* ws, int ks, hipStream_t st, bool go) {
  if (a.lg == 5) return zp ? by_tile<true, 2>(a, tile, ws, ks, st, go) : by_tile<false, 2>(a, tile, ws, ks, st, go);
  return zp ? by_tile<true, 1>(a, tile, ws, ks, st, go) : by_tile<false, 1>(a, tile, ws, ks, st, go);
}

// The tiles: features x rows, chunks of a step (WK), workgroups that a CU holds, and measured times in ns: a step of a workgroup
// alone on its CU and of a full CU, and the rest of a workgroup's time.  Fitted to 2600 timings (12 to 3000 rows, 1001 to 16384
// features, K 192 to 8192, up to 12 ways, groups of 128), which the estimate meets within 6 to 9% rms.  Tiles of 96 rows beside those
// of 128 and 64 save padding (187 rows of 16384 x 3072 30 -> 25 us, 3000 of 3072 x 3072 79 -> 67); 128 x 128 and 128 x 32 were
// the best nowhere by more than 5%.  Groups of 64 and 32 have the same choices: over 30 shapes of 24 to 1024 rows the mean is 5 to 6.5%
// behind the best there (0.4 to 0.7% for 128), most where the few-row kernel's twice as many matrix instructions count: 24 rows of
// 16384 x 3072 13.6 us (a tile 9.3), 100 of 3072 x 3072 12.8 (8.9).  Then the
// few-row kernel's forms, whose 8 waves take a pair of chunks each in a step (360 timings of 16 to 256 rows, 7 to 9% rms): they
// read the codes again for every 16 rows, but a CU starts on them with all loads in flight and ends without a split's join
// (48 rows of 3072 x 3072: 5.8 us, the best tile 8.8; 192 rows of 5120 x 3072: 15.5 and 11.7).  And those with the norm inside (312
// timings, 5% rms), which save its launch (48 rows 8.3 us, the tiles 11.8 with rows rounded once and 13.7 in two parts).
struct Q4Cost {
  int bn, bm, wk, fit, step, full, rest;
};
constexpr Q4Cost Q4_COST[Q4_TILES + 2 * Q4_ROWS] = {
    {256, 128, 1, 2, 885, 1469, 3596}, {256, 96, 1, 2, 740, 1175, 2973}, {128, 64, 2, 2, 560, 1181, 1978},
    {128, 96, 4, 1, 1342, 1342, 2681}, {64, 32, 4, 1, 499, 499, 1477},   {64, 64, 4, 1, 696, 696, 1767},
    {16, 16, 16, 1, 438, 363, 619},    {32, 16, 16, 1, 596, 516, 693},  {64, 16, 16, 1, 994, 961, 717},
    {16, 16, 16, 1, 761, 777, 1780},   {32, 16, 16, 1, 936, 1013, 1926}, {64, 16, 16, 1, 1437, 1765, 1757},
};

// The choice of the shortest estimate.  Over the 96 shapes that the times were taken at it is 0.8% behind the fastest of all on
// average, 17% at most; over 120 shapes with few rows as much, and 12%; over 104 with
// a norm 0.2%, 10%, and before a SiLU 0.4%, 15%.  A split's join costs a launch and the passage of its sums through memory.
int gemm_q4_plan(int M, int N, int K, Q4Among among) {
  const bool norm = among >= Q4_NORM;
  long best = 0x7FFFFFFFFFFFFFFFL;
  int plan = 0;
  // (the few-row forms' launch counts at most 65535 blocks of 16 rows)
  for (int t = 0; t < Q4_TILES + (among == Q4_ONLY_TILES || M > 16 * 65535 ? 0 : Q4_ROWS); ++t) {
    const bool rows = t >= Q4_TILES, two = rows ? norm : among == Q4_NORM_SILU;
    const Q4Cost& c = Q4_COST[rows && two ? t + Q4_ROWS : t];
    const int nch = K >> 6 << (two && !rows);
    const long tiles = ((long)N + c.bn - 1) / c.bn * (((long)M + c.bm - 1) / c.bm);
    for (int ks = 1; ks <= (rows ? 1 : 12); ++ks) {
      if (ks > 1 && (tiles * ks > 1100 || nch < 4 * ks)) break;
      const long blocks = tiles * ks, steps = ((nch + ks - 1) / ks + c.wk - 1) / c.wk, per = 256L * c.fit, rem = blocks % per;
      long e = blocks / per * (steps * c.full + c.rest);
      // a last round of more than one workgroup per CU: 30% of the way to a full one at once, the rest with their number
      if (rem) e += steps * (c.step + (rem > 256 ? (c.full - c.step) * (77 + 179 * (rem - 256) / 256) / 256 : 0)) + c.rest;
      if (ks > 1) e += 2700 + 12L * (ks + 1) * M * N / 10000;
      if (norm && !rows) e += 2700;  // the norm's launch
      if (e < best) {
        best = e;
        plan = (rows ? t + 1 - Q4_TILES + Q4_ROWS_AT : t + 1) + (two ? Q4_TWO : 0) + 256 * ks;
      }
    }
  }
  return plan;
}

}  // namespace ecd
