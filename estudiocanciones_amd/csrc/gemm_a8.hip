// Products of int8 activations and int8 weights (gfx950): a scale per row, a scale per output channel.
//   quantise   y = x, or its RMS norm x / sqrt(mean(x^2) + eps) w in fp32;  t_m = max_k |y[m, k]|,
//              c[m, k] = rint(127 y[m, k] / t_m),  sx[m] = t_m / 127       (ties to even; t_m = 0: codes and scale 0)
//   product    z[m, n] = sx[m] s[n] sum_k c[m, k] q[n, k];  y = z (+ res), or silu(z[m, 2j]) z[m, 2j + 1]
// The sum over k is an integer (exact in any order: |sum| <= 128 127 K < 2^31 for K <= 2^17), so a row's result does not
// depend on the tile, the split of K or the other rows.  fp32 behind the sum, one rounding to fp16 at the end.
//
// Of fp16 x (no norm) the codes are the nearest integers to the exact quotients: 127 x has 18 bits, so a quotient that is
// no tie is further from one than the rounding of the quotient to fp32 moves it, and a tie is a value of fp32.
#include "gemm_core.h"

namespace ecd {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// One workgroup per row, its values in registers (NV pieces of 8 per thread; rows of more than 2048 NV values are read
// again).  A row that holds an infinity or a NaN gets the scale NaN (and codes 0).  Bound by vector instructions, then by the
// row's two reductions: 2048 x 3072 with the norm 9.4 us with a division for each value, 7.8 us as written (18.9 MB).
template <bool NORM, int NV>
__global__ __launch_bounds__(256) void quant_a8_kernel(const f16* __restrict__ x, long ldx, const f16* __restrict__ w,
                                                       float eps, int8_t* __restrict__ c, long ldc,
                                                       float* __restrict__ sx, int K) {
  __shared__ float red[8];
  const int t = threadIdx.x;
  const long m = blockIdx.x;
  const f16* xr = x + m * ldx;
  f16x8 v[NV], g[NORM ? NV : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = 8 * t + 2048 * i;
    v[i] = k < K ? *(const f16x8*)(xr + k) : (f16x8)((f16)0);
    if constexpr (NORM) g[i] = k < K ? *(const f16x8*)(w + k) : (f16x8)((f16)0);
  }
  auto each = [&](auto&& f) {  // f(k, 8 values, 8 weights) over this thread's pieces of the row
#pragma unroll
    for (int i = 0; i < NV; ++i) f(8 * t + 2048 * i, v[i], g[NORM ? i : 0]);
    for (int k = 8 * t + 2048 * NV; k < K; k += 2048) f(k, *(const f16x8*)(xr + k), *(const f16x8*)((NORM ? w : xr) + k));
  };
  float r = 1.f;
  if constexpr (NORM) {
    float s = 0.f;
    each([&](int, const f16x8& a, const f16x8&) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s += (float)a[j] * (float)a[j];
    });
    s = wave_sum_dpp(s);
    if ((t & 63) == 0) red[t >> 6] = s;
    __syncthreads();
    r = 1.0f / sqrtf((red[0] + red[1] + red[2] + red[3]) / (float)K + eps);
  }
  auto value = [&](f16 a, f16 b) { return NORM ? (float)a * r * (float)b : (float)a; };
  // the largest magnitude as bits: an infinity or a NaN is larger than every number
  uint32_t top = 0;
  each([&](int, const f16x8& a, const f16x8& b) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(value(a[j], b[j])) & 0x7FFFFFFFu);
  });
  top = wave_max_u32(top);
  if ((t & 63) == 0) red[4 + (t >> 6)] = __uint_as_float(top);
  __syncthreads();
  top = max(max(__float_as_uint(red[4]), __float_as_uint(red[5])), max(__float_as_uint(red[6]), __float_as_uint(red[7])));
  const bool bad = top >= 0x7F800000u, none = bad || top == 0;
  const float big = __uint_as_float(top), inv = 1.f / big;
  if (t == 0) sx[m] = bad ? NAN : big / 127.f;
  int8_t* cr = c + m * ldc;
  each([&](int k, const f16x8& a, const f16x8& b) {
    if (k >= ldc) return;
    uint32_t o[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
    if (!none) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = value(a[j], b[j]) * 127.f, q = t * inv;
        // one step from the quotient by the rounded reciprocal gives the rounded quotient; adding 1.5 2^23 leaves the nearest
        // integer (ties to even) in the low bits
        o[j] = __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, big, t), inv, q) + 12582912.f);
      }
    }
    auto pack = [](uint32_t x, uint32_t y, uint32_t z, uint32_t w) {  // the low bytes
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0C0C0400u), __builtin_amdgcn_perm(y, x, 0x0C0C0400u), 0x05040100u);
    };
    *(u32x2*)(cr + k) = (u32x2){pack(o[0], o[1], o[2], o[3]), pack(o[4], o[5], o[6], o[7])};
  });
  // the columns behind K that lie behind the last piece (K is a multiple of 64, ldc of 128)
  for (int k = max(K, 2048 * NV) + 8 * t; k < ldc; k += 2048) *(u32x2*)(cr + k) = (u32x2){0u, 0u};
}

struct A8Out {
  const float* sx;
  const f16* s;
  const f16* res;
  long ldr;
  f16* y;
  long ldy;
};

// The results of 8 consecutive features n .. (fewer at the end) of U rows from their integer sums; sm, sn: the scales of
// the rows and the features.  Rows from M on are left out.
template <bool SILU, int U>
__device__ __forceinline__ void a8_finish(const A8Out& out, const int (&v)[U][8], const float (&sm)[U], const float (&sn)[8],
                                          const int (&m)[U], int n, int M, int N) {
  const bool whole = n + 7 < N;
  f16x8 r[U];
  if (!SILU && out.res && whole) {
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = *(const f16x8u*)(out.res + min(m[u], M - 1) * out.ldr + n);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (m[u] >= M) break;
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = (float)v[u][j] * (sm[u] * sn[j]);
    if constexpr (SILU) {
      f16x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = (f16)(z[2 * j] * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z[2 * j] * -1.44269504088896341f)) * z[2 * j + 1]);
      f16* d = out.y + m[u] * out.ldy + (n >> 1);
      if (whole) {
        *(f16x4u*)d = o;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + 2 * j < N) d[j] = o[j];
      }
    } else {
      f16* d = out.y + m[u] * out.ldy + n;
      if (whole) {
        f16x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (f16)(out.res ? z[j] + (float)r[u][j] : z[j]);
        *(f16x8u*)d = o;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (n + j < N) d[j] = (f16)(out.res ? z[j] + (float)out.res[m[u] * out.ldr + n + j] : z[j]);
      }
    }
  }
}

__device__ __forceinline__ void a8_scales(const f16* s, int n, int N, float (&sn)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) sn[j] = (float)s[min(n + j, N - 1)];
}

// ---- few rows: the weights stream once from memory into registers
// One workgroup per 16 features and 16 rows; its waves take an equal share of K each, eight 1 KB loads of the weights in
// flight, and add their integer sums in LDS.  A chunk of packed weights (16 features x 64 k, 16 bytes a lane) is the A
// operand of v_mfma_i32_16x16x64_i8 as it stands, a row's codes the B operand: both hold the k of a lane in the same order.
// Bound by memory: 8 rows, (16384, 3072) 11.4 us (4.4 TB/s), (3072, 8192) 8.3 us; four waves 12.8 and 9.1, sixteen 9.2.
constexpr int FEW_W = 8, FEW_U = 8;
template <bool SILU>
__global__ __launch_bounds__(64 * FEW_W) void gemm_a8_few_kernel(const int8_t* __restrict__ c, long ldc,
                                                                 const int8_t* __restrict__ wp, A8Out out, int M, int N, int K) {
  __shared__ __align__(16) int part[FEW_W][16][20];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const int steps = K >> 6, s1 = steps * (wv + 1) / FEW_W;
  const int8_t* w = wp + (long)blockIdx.x * 16 * K + 16 * lane;
  const int8_t* x = c + (long)min(m0 + (lane & 15), M - 1) * ldc + 16 * (lane >> 4);
  i32x4 acc = {0, 0, 0, 0};
  int k = steps * wv / FEW_W;
  for (; k + FEW_U <= s1; k += FEW_U) {
    i32x4 a[FEW_U], b[FEW_U];
#pragma unroll
    for (int u = 0; u < FEW_U; ++u) {
      a[u] = __builtin_nontemporal_load((const i32x4*)(w + 1024L * (k + u)));
      b[u] = *(const i32x4*)(x + 64 * (k + u));
    }
#pragma unroll
    for (int u = 0; u < FEW_U; ++u) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], b[u], acc, 0, 0, 0);
  }
  for (; k < s1; ++k)
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_nontemporal_load((const i32x4*)(w + 1024L * k)),
                                                *(const i32x4*)(x + 64 * k), acc, 0, 0, 0);
  *(i32x4*)&part[wv][lane & 15][4 * (lane >> 4)] = acc;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const int r = threadIdx.x >> 1, h = 8 * (threadIdx.x & 1), m[1] = {m0 + r}, n = n0 + h;
  if (m[0] >= M || n >= N) return;
  int v[1][8] = {{0, 0, 0, 0, 0, 0, 0, 0}};
#pragma unroll
  for (int i = 0; i < FEW_W; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[0][j] += part[i][r][h + j];
  float sn[8];
  a8_scales(out.s, n, N, sn);
  const float sm[1] = {out.sx[m[0]]};
  a8_finish<SILU, 1>(out, v, sm, sn, m, n, M, N);
}

// ---- many rows: tiles of 32 WN FT features x 32 WM RT rows through an LDS ring of NS stages of 128 k
// The loads, the stages and the order of a loop pass are those of GemmTile (gemm_core.h) on bytes: 16 bytes of a row or a
// feature are 16 k of v_mfma_i32_32x32x32_i8 instead of 8 of the fp16 product.
// The largest tile (256 x 256, 8 waves) is bound by the products and their LDS reads: 2048 rows, (16384, 3072) 97 us, of which
// 11 are the sums' way out (2.1 POPS; matrix pipes busy 54%); 8192^3 2.35 POPS.  Four waves of 128 x 128 took 110 us.  The
// small tiles are bound by what a CU gets from its L2 and by latency: 187 rows, (3072, 8192), 64 x 64 with K in two shares,
// 14.1 to 15.2 us (25 MB of weights); 128 x 64 with K whole 15.7.
template <int FT, int RT>
struct A8Frags {
  i32x4 w[2][FT], x[2][RT];
};

template <int WN, int WM, int FT, int RT, int NS, int KG>
struct A8Tile {
  static constexpr int NW = WN * WM, BN = 32 * WN * FT, BM = 32 * WM * RT;
  static constexpr int WI = BN / 8 / NW, XI = BM / 8 / NW, PER = WI + XI;  // DMA instructions (1 KB) per wave and chunk
  static_assert(WI * NW * 8 == BN && XI * NW * 8 == BM, "whole DMA instructions per wave");
  static_assert(NS >= 2 && PER * (NS - 1) < 64, "vmcnt range");
  static constexpr int LW = BN * 128, LX = BM * 128, STG = LW + LX, RING = NS * STG;  // bytes of a stage, of a group's ring
  // the sums leave through LDS as int32, some row tiles of each wave at a time
  static constexpr int ROW = BN + 4;  // ints of an output row
  static constexpr int fit(int n) { return n == 1 || 32 * WM * n * ROW * 4 <= RING ? n : fit(n / 2); }
  static constexpr int RP = fit(RT);  // row tiles of a pass
  static_assert(RT % RP == 0, "whole passes");
  static constexpr int PASS = 32 * WM * RP * ROW;  // ints of a pass
  static constexpr int LDS = KG * (RING > PASS * 4 ? RING : PASS * 4);
  static constexpr int THREADS = 64 * NW * KG;

  // The sums of this wave's group: KG groups of NW waves take an equal share of K each, from a ring of their own (a CU
  // with one workgroup then has KG times the loads in flight, where there are too few tiles for all CUs).  A chunk of 128 k
  // that K ends in: its second half re-reads the first and its products are left out, so nothing behind K is read.
  static __device__ __forceinline__ void run(unsigned char* all, i32x16 (&acc)[FT][RT], const int8_t* __restrict__ c, long ldc,
                                             const int8_t* __restrict__ wp, int M, int N, int K, int n0, int m0) {
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wv = wid % NW, kg = wid / NW, wn = wv % WN, wm = wv / WN;
    unsigned char* lds = all + kg * RING;
    const int chunks = (K + 127) >> 7, most = (chunks + KG - 1) / KG;
    const int c0 = chunks * kg / KG, nch = chunks * (kg + 1) / KG - c0;
    const bool odd = (K & 64) && kg == KG - 1;
    const int ntiles = (N + 15) >> 4, t0 = min(n0 / 16, ntiles - 1);
    const long tile_bytes = 16L * K;
    const int8_t* wb = wp + t0 * tile_bytes + 2048L * c0;
    const int8_t* xb = c + (long)m0 * ldc + 128L * c0;
    int left = nch;  // chunks not yet asked for
    uint32_t woff[WI], xoff[XI];
#pragma unroll
    for (int j = 0; j < WI; ++j) {
      const int i = wv + NW * j;
      woff[j] = (uint32_t)((min(n0 / 16 + (i >> 1), ntiles - 1) - t0) * tile_bytes) + 1024 * (i & 1) + 16 * lane;
    }
#pragma unroll
    for (int j = 0; j < XI; ++j) {
      const int r = 8 * (wv + NW * j) + (lane >> 3);
      xoff[j] = (uint32_t)((min(m0 + r, M - 1) - m0) * ldc) + 16 * ((lane & 7) ^ x_swz(r));
    }
    const uint32_t lds0 = lds_addr(lds) + wv * 1024;
    const uint32_t back = wv & 1 ? 1024u : 0u;  // (NW is even: this wave's weight instructions are all first or all second halves)
    static_assert(NW % 2 == 0, "a wave keeps its half");
    auto dma = [&](auto J, uint32_t sa) {
      constexpr int j = decltype(J)::value;
      if constexpr (j < WI)
        lds_dma16_at<NW * j * 1024>(wb, odd && left == 1 ? woff[j] - back : woff[j], sa);
      else
        lds_dma16_at<LW + NW * (j - WI) * 1024>(xb, odd && left == 1 ? xoff[j - WI] & ~64u : xoff[j - WI], sa);  // (ldc % 128 == 0)
    };
    auto next_chunk = [&]() {
      wb += 2048;
      xb += 128;
      --left;
    };
    static_for<0, FT * RT>([&](auto I) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[I.value / RT][I.value % RT][e] = 0;
    });
    // fragment addresses: 32 features are two packed 16-row tiles of 2 KB, piece o = 2 s + (lane >> 5) of k-step s lies in
    // 1 KB half o >> 2 at unit 16 (o & 3) + row; piece o of x row r at position o ^ x_swz(r)
    const int wfo = (wn * FT * 2 + ((lane >> 4) & 1)) * 2048 + (lane >> 5) * 256 + (lane & 15) * 16;
    int xfo[4];
    static_for<0, 4>([&](auto S) {
      xfo[S.value] = LW + (wm * RT * 32 + (lane & 31)) * 128 + 16 * ((2 * S.value + (lane >> 5)) ^ x_swz(lane & 31));
    });
    constexpr int NM = 2 * FT * RT, NR = 2 * (FT + RT);
    auto read1 = [&](auto I, auto H, const unsigned char* base, A8Frags<FT, RT>& f) {
      constexpr int i = decltype(I)::value, h = decltype(H)::value;
      if constexpr (i < 2 * FT) {
        constexpr int s = i / FT, ft = i % FT;
        f.w[s][ft] = *(const i32x4*)(base + wfo + 1024 * h + 512 * s + ft * 4096);
      } else {
        constexpr int k = i - 2 * FT, s = k / RT, rt = k % RT;
        f.x[s][rt] = *(const i32x4*)(base + xfo[2 * h + s] + rt * 4096);
      }
    };
    // the products of a half chunk, with the reads of the next half's fragments and DMA instructions D0 .. D1 - 1 between
    auto half = [&](const A8Frags<FT, RT>& f, auto H, const unsigned char* base, A8Frags<FT, RT>& nf, auto D0, auto D1, uint32_t sa) {
      static_for<0, NM>([&](auto I) {
        constexpr int m = decltype(I)::value, s = m / (FT * RT), ft = m % (FT * RT) / RT, rt = m % RT;
        acc[ft][rt] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[s][ft], f.x[s][rt], acc[ft][rt], 0, 0, 0);
        constexpr int d0 = decltype(D0)::value, nd = decltype(D1)::value - d0;
        static_for<d0 + m * nd / NM, d0 + (m + 1) * nd / NM>([&](auto J) { dma(J, sa); });
        static_for<m * NR / NM, (m + 1) * NR / NM>([&](auto J) { read1(J, H, base, nf); });
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    auto barrier = [&]() {  // (of the whole workgroup: each group passes `most` of them)
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };

    if (KG > 1 && nch == 0) {
      for (int b = 0; b < most; ++b) barrier();
      return;
    }
    for (int s = 0; s < NS; ++s)
      if (s < nch) {
        static_for<0, PER>([&](auto J) { dma(J, lds0 + s * STG); });
        next_chunk();
      }
    wait_chunk<PER, NS - 1, false>(min(NS - 1, nch - 1));
    barrier();
    A8Frags<FT, RT> fa, fc;
    static_for<0, NR>([&](auto I) { read1(I, IC<0>{}, lds, fa); });
    // as in GemmTile: each pass runs chunk i's second half and chunk i + 1's first, and loads chunk i + NS
    constexpr int DS = NS > 2 ? (PER + 1) / 2 : PER;
    int i = 0, st = 0;
    half(fa, IC<1>{}, lds, fc, IC<0>{}, IC<0>{}, 0);
    for (; i < nch - NS; ++i) {
      wait_vm_lgkm0<(NS - 2) * PER>();
      barrier();
      const int sn = st + 1 == NS ? 0 : st + 1;
      const unsigned char* base = lds + sn * STG;
      const uint32_t sa = lds0 + st * STG;
      half(fc, IC<0>{}, base, fa, IC<0>{}, IC<DS>{}, sa);
      half(fa, IC<1>{}, base, fc, IC<DS>{}, IC<PER>{}, sa);
      next_chunk();
      st = sn;
    }
    for (; i < nch - 1; ++i) {
      wait_chunk<PER, NS - 2, true>(min(NS - 2, nch - 2 - i));
      barrier();
      const int sn = st + 1 == NS ? 0 : st + 1;
      const unsigned char* base = lds + sn * STG;
      half(fc, IC<0>{}, base, fa, IC<0>{}, IC<0>{}, 0);
      half(fa, IC<1>{}, base, fc, IC<0>{}, IC<0>{}, 0);
      st = sn;
    }
    if (!odd) half(fc, IC<0>{}, lds, fa, IC<0>{}, IC<0>{}, 0);  // (its reads are never used)
    if (KG > 1 && nch < most) barrier();
  }

  // f(rows of the tile, their 8 sums) for U rows at a time of this thread's piece of 8 features, the rows in passes through
  // LDS, where the groups' sums are added
  static constexpr int PR = BN / 8, RS = THREADS / PR, ROWS = 32 * WM * RP;
  static_assert(THREADS % PR == 0 && (ROWS % RS == 0 || RS > ROWS), "whole rows per step");
  static constexpr int IT = ROWS > RS ? ROWS / RS : 1, U = IT % 4 == 0 ? 4 : IT % 2 == 0 ? 2 : 1;
  template <typename F>
  static __device__ __forceinline__ void sums(unsigned char* lds, const i32x16 (&acc)[FT][RT], F&& f) {
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wv = wid % NW, kg = wid / NW, wn = wv % WN, wm = wv / WN;
    int* buf = (int*)lds;
    const int p = threadIdx.x % PR;
    static_for<0, RT / RP>([&](auto P) {
      __syncthreads();
      static_for<0, FT * RP>([&](auto I) {
        constexpr int ft = decltype(I)::value / RP, q = decltype(I)::value % RP, rt = decltype(P)::value * RP + q;
        int* d = buf + kg * PASS + ((wm * RP + q) * 32 + (lane & 31)) * ROW + (wn * FT + ft) * 32 + 4 * (lane >> 5);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(i32x4*)(d + 8 * g) = (i32x4){acc[ft][rt][4 * g], acc[ft][rt][4 * g + 1], acc[ft][rt][4 * g + 2], acc[ft][rt][4 * g + 3]};
      });
      __syncthreads();
      const int first = threadIdx.x / PR;
      if (first < ROWS) {
#pragma unroll 1
        for (int it = 0; it < IT; it += U) {
          int v[U][8], row[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int r = first + RS * (it + u), w = r / (32 * RP);
            row[u] = (w * RT + decltype(P)::value * RP) * 32 + r - w * 32 * RP;
            i32x4 a = *(const i32x4*)(buf + r * ROW + 8 * p), b = *(const i32x4*)(buf + r * ROW + 8 * p + 4);
#pragma unroll
            for (int k = 1; k < KG; ++k) {
              a += *(const i32x4*)(buf + k * PASS + r * ROW + 8 * p);
              b += *(const i32x4*)(buf + k * PASS + r * ROW + 8 * p + 4);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              v[u][j] = a[j];
              v[u][4 + j] = b[j];
            }
          }
          f(row, v);
        }
      }
    });
  }
};

// Block b of an order in which the row blocks of a feature block have numbers that are equal modulo 8: one XCD, whose L2
// then holds the weights.
__device__ __forceinline__ void a8_block(int b, int nfb, int nmb, int& fb, int& mb) {
  const int full = nfb & ~7;
  if (b < full * nmb) {
    const int g = b / (8 * nmb), rem = b - g * 8 * nmb;
    mb = rem >> 3;
    fb = g * 8 + (rem & 7);
  } else {
    const int rem = b - full * nmb, tw = nfb - full;
    mb = rem / tw;
    fb = full + rem - mb * tw;
  }
}

template <bool SILU, int WN, int WM, int FT, int RT, int NS, int KG>
__global__ __launch_bounds__(64 * WN * WM * KG, 1) void gemm_a8_kernel(const int8_t* __restrict__ c, long ldc,
                                                                       const int8_t* __restrict__ wp, A8Out out, int M, int N,
                                                                       int K, int nfb, int nmb) {
  using T = A8Tile<WN, WM, FT, RT, NS, KG>;
  __shared__ __align__(16) unsigned char lds[T::LDS];
  int fb, mb;
  a8_block(blockIdx.x, nfb, nmb, fb, mb);
  const int n0 = fb * T::BN, m0 = mb * T::BM;
  __shared__ float s_sx[T::BM];  // the rows' scales: here before the sums are (a load for each row cost 0.4 us a row)
  for (int i = threadIdx.x; i < T::BM; i += T::THREADS) s_sx[i] = out.sx[min(m0 + i, M - 1)];
  i32x16 acc[FT][RT];
  T::run(lds, acc, c, ldc, wp, M, N, K, n0, m0);
  const int nb = n0 + 8 * (threadIdx.x % T::PR);
  float sn[8];
  a8_scales(out.s, nb, N, sn);
  T::sums(lds, acc, [&](const int (&row)[T::U], const int (&v)[T::U][8]) {
    if (nb >= N) return;
    int m[T::U];
    float sm[T::U];
#pragma unroll
    for (int u = 0; u < T::U; ++u) {
      m[u] = m0 + row[u];
      sm[u] = s_sx[row[u]];
    }
    a8_finish<SILU, T::U>(out, v, sm, sn, m, nb, M, N);
  });
}

constexpr long THREADS_MOST = 0xFFFFFFFFL;  // of a launch along x

template <bool SILU, int WN, int WM, int FT, int RT, int NS, int KG>
static int launch_tile(const int8_t* c, long ldc, const int8_t* wp, const A8Out& out, int M, int N, int K, hipStream_t st) {
  using T = A8Tile<WN, WM, FT, RT, NS, KG>;
  const int nfb = (N + T::BN - 1) / T::BN, nmb = (M + T::BM - 1) / T::BM;
  if ((long)nfb * nmb > THREADS_MOST / T::THREADS) return ECD_ENOTSUP;
  hipLaunchKernelGGL((gemm_a8_kernel<SILU, WN, WM, FT, RT, NS, KG>), dim3((unsigned)(nfb * nmb)), dim3(T::THREADS), 0, st, c, ldc, wp, out,
                     M, N, K, nfb, nmb);
  return ecd_launch_status();
}

template <bool SILU>
static int launch_few(const int8_t* c, long ldc, const int8_t* wp, const A8Out& out, int M, int N, int K, hipStream_t st) {
  if ((M + 15) / 16 > 65535 || (N + 15) / 16 > THREADS_MOST / (64 * FEW_W)) return ECD_ENOTSUP;
  hipLaunchKernelGGL(gemm_a8_few_kernel<SILU>, dim3((N + 15) / 16, (M + 15) / 16), dim3(64 * FEW_W), 0, st, c, ldc, wp, out, M, N, K);
  return ecd_launch_status();
}

// The tiles (features x rows), the ways that K is shared out in a workgroup, and measured times in ns: a chunk (of 128 KG k)
// with at most 144 workgroups and with 256 (one per CU), what a launch and what each round of 256 add.
struct A8Cfg {
  int bn, bm, kg, light, full, edge, round;
};
constexpr A8Cfg A8_CFG[7] = {
    {32, 64, 2, 207, 280, 3025, 461},     // 2: two workgroups per CU
    {64, 64, 2, 267, 437, 2286, 1790},    // 3
    {128, 64, 2, 426, 710, 2142, 2348},   // 4
    {128, 64, 1, 242, 332, 3425, 1073},   // 5: two workgroups per CU
    {128, 128, 1, 291, 595, 1622, 4469},  // 6
    {256, 128, 1, 492, 892, 1028, 7892},  // 7
    {256, 256, 1, 960, 1634, 14, 11186},  // 8
};
constexpr int A8_FEW = 1;

// The kernel of a product: few rows stream the weights through registers (up to 8 rows, 16 where there are at most 4096
// features; us at K = 3072, tiles -> it: 4 x 5120 6.5 -> 6.4, 16 x 3072 6.3 -> 6.3, 4 x 3072 x 8192 10.6 -> 8.2, and where
// the rule keeps tiles: 16 x 5120 6.5 -> 8.0, 16 x 16384 11.6 -> 16.8), else the tile of the shortest estimate.  (Of 167
// shapes of 24 to 3000 rows and 11 weight matrices measured with 14 tiles the rule's is 2.6% slower than the best on average,
// 25% at worst.)
static int a8_choice(int M, int N, int K) {
  if (M <= 8 || (M <= 16 && N <= 4096)) return A8_FEW;
  int best = 0;
  long least = 0;
  for (int i = 0; i < 7; ++i) {
    const A8Cfg& t = A8_CFG[i];
    const long b = (long)((N + t.bn - 1) / t.bn) * ((M + t.bm - 1) / t.bm), rest = b % 256;
    const long nch = ((K + 127) / 128 + t.kg - 1) / t.kg;
    long e = t.edge + b / 256 * (nch * t.full + t.round);
    if (rest) e += nch * (t.light + (t.full - t.light) * (rest > 144 ? rest - 144 : 0) / 112) + t.round;
    if (i == 0 || e < least) {
      best = i;
      least = e;
    }
  }
  return 2 + best;
}

template <bool SILU>
static int launch_a8(const void* cv, long ldc, const void* wv, const A8Out& out, int M, int N, int K, hipStream_t st, int cfg = 0) {
  if (M > 1 << 30 || N > 1 << 30) return ECD_ENOTSUP;  // (row and feature numbers of a tile are 32-bit)
  const int8_t *c = (const int8_t*)cv, *wp = (const int8_t*)wv;
#define A8_TILE(...) return launch_tile<SILU, __VA_ARGS__>(c, ldc, wp, out, M, N, K, st)
  switch (cfg ? cfg : a8_choice(M, N, K)) {
    case A8_FEW: return launch_few<SILU>(c, ldc, wp, out, M, N, K, st);
    case 2: A8_TILE(1, 2, 1, 1, 3, 2);
    case 3: A8_TILE(2, 2, 1, 1, 4, 2);
    case 4: A8_TILE(2, 2, 2, 1, 3, 2);
    case 5: A8_TILE(2, 2, 2, 1, 3, 1);
    case 6: A8_TILE(2, 2, 2, 2, 4, 1);
    case 7: A8_TILE(2, 2, 4, 2, 3, 1);
    case 8: A8_TILE(4, 2, 2, 4, 2, 1);
    default: return ECD_EINVAL;
  }
#undef A8_TILE
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool a8_ok(const void* c, long ldc, const float* sx, const void* wp, const void* s, const void* y, int M, int N,
                  int K) {
  return c && sx && wp && s && y && M > 0 && N > 0 && K > 0 && K % 64 == 0 && K <= 1 << 17 && ldc >= K &&
         ldc % 128 == 0 && ldc <= 1 << 23 && aligned16(c) && aligned16(wp);
}

}  // namespace ecd

using namespace ecd;

extern "C" {

int ecd_quant_a8(const void* x, long ldx, const void* nw, float eps, void* c, long ldc, float* sx, int M, int K,
                 void* stream) {
  if (!x || !c || !sx || M <= 0 || K <= 0 || K % 64 || K > 1 << 17 || ldx < K || ldx % 8 || ldc < K || ldc % 128 ||
      !aligned16(x) || !aligned16(c) || (nw && !aligned16(nw)) || !(eps >= 0.f))
    return ECD_EINVAL;
  if (M > 0xFFFFFF) return ECD_ENOTSUP;  // (a launch has fewer than 2^32 threads)
  const hipStream_t st = (hipStream_t)stream;
#define QA(N_, V_)                                                                                                       \
  hipLaunchKernelGGL((quant_a8_kernel<N_, V_>), dim3(M), dim3(256), 0, st, (const f16*)x, ldx, (const f16*)nw, eps,      \
                     (int8_t*)c, ldc, sx, K)
  if (nw) {
    if (K <= 2048) QA(true, 1);
    else if (K <= 4096) QA(true, 2);
    else QA(true, 4);
  } else {
    if (K <= 2048) QA(false, 1);
    else if (K <= 4096) QA(false, 2);
    else QA(false, 4);
  }
#undef QA
  return ecd_launch_status();
}

int ecd_gemm_a8(const void* c, long ldc, const float* sx, const void* wp, const void* s, const void* res, long ldr,
                void* y, long ldy, int M, int N, int K, void* stream) {
  if (!a8_ok(c, ldc, sx, wp, s, y, M, N, K) || ldy < N || (res && ldr < N)) return ECD_EINVAL;
  return launch_a8<false>(c, ldc, wp, A8Out{sx, (const f16*)s, (const f16*)res, ldr, (f16*)y, ldy}, M, N, K,
                          (hipStream_t)stream);
}

int ecd_gemm_a8_tuned(const void* c, long ldc, const float* sx, const void* wp, const void* s, const void* res, long ldr,
                      void* y, long ldy, int M, int N, int K, int cfg, void* stream) {
  if (!a8_ok(c, ldc, sx, wp, s, y, M, N, K) || ldy < N || (res && ldr < N) || cfg < 0 || cfg > 8)
    return ECD_EINVAL;
  return launch_a8<false>(c, ldc, wp, A8Out{sx, (const f16*)s, (const f16*)res, ldr, (f16*)y, ldy}, M, N, K,
                          (hipStream_t)stream, cfg);
}

int ecd_gemm_a8_silu(const void* c, long ldc, const float* sx, const void* wp, const void* s, void* mm, long ldm,
                     int M, int F, int K, void* stream) {
  if (F <= 0 || F > 1 << 29 || !a8_ok(c, ldc, sx, wp, s, mm, M, 2 * F, K) || ldm < F) return ECD_EINVAL;
  return launch_a8<true>(c, ldc, wp, A8Out{sx, (const f16*)s, nullptr, 0, (f16*)mm, ldm}, M, 2 * F, K,
                         (hipStream_t)stream);
}

}  // extern "C"
