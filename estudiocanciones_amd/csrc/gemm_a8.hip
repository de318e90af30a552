// Products of int8 activations and int8 weights (gfx950): a scale per row, a scale per output channel.
//   quantise   y = x, or its RMS norm x / sqrt(mean(x^2) + eps) w in fp32;  t_m = max_k |y[m, k]|,
//              c[m, k] = rint(127 y[m, k] / t_m),  sx[m] = t_m / 127       (ties to even; t_m = 0: codes and scale 0)
//   product    z[m, n] = sx[m] s[n] sum_k c[m, k] q[n, k];  y = z (+ res), or silu(z[m, 2j]) z[m, 2j + 1]
// The sum over k is an integer (exact in any order: |sum| <= 128 127 K < 2^31 for K <= 2^17), so a row's result does not
// depend on the tile, the split of K or the other rows.  fp32 behind the sum, one rounding to fp16 at the end.
//
// Of fp16 x (no norm) the codes are the nearest integers to the exact quotients: 127 x has 18 bits, so a quotient that is
// no tie is further from one than the correctly rounded division moves it.
#include "gemm_core.h"

namespace ecd {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// One workgroup per row.  A row that holds an infinity or a NaN gets the scale NaN (and codes 0).
template <bool NORM>
__global__ __launch_bounds__(256) void quant_a8_kernel(const f16* __restrict__ x, long ldx, const f16* __restrict__ w,
                                                       float eps, int8_t* __restrict__ c, long ldc,
                                                       float* __restrict__ sx, int K) {
  __shared__ float red[8];
  __shared__ int s_bad;
  const int t = threadIdx.x;
  const long m = blockIdx.x;
  const f16* xr = x + m * ldx;
  if (t == 0) s_bad = 0;
  float r = 1.f;
  if constexpr (NORM) {
    float s = 0.f;
    for (int k = 8 * t; k < K; k += 2048) {
      const f16x8 v = *(const f16x8*)(xr + k);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += (float)v[j] * (float)v[j];
    }
    s = wave_sum(s);
    if ((t & 63) == 0) red[t >> 6] = s;
    __syncthreads();
    r = 1.0f / sqrtf((red[0] + red[1] + red[2] + red[3]) / (float)K + eps);
  }
  auto value = [&](int k, float* y) {
    const f16x8 v = *(const f16x8*)(xr + k);
    f16x8 g;
    if constexpr (NORM) g = *(const f16x8*)(w + k);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = NORM ? (float)v[j] * r * (float)g[j] : (float)v[j];
  };
  float top = 0.f;
  bool bad = false;
  for (int k = 8 * t; k < K; k += 2048) {
    float y[8];
    value(k, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      top = fmaxf(top, fabsf(y[j]));
      bad |= !(fabsf(y[j]) < INFINITY);
    }
  }
  top = wave_max(top);
  __syncthreads();
  if ((t & 63) == 0) red[4 + (t >> 6)] = top;
  if (bad) atomicOr(&s_bad, 1);
  __syncthreads();
  top = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
  const bool none = s_bad || top == 0.f;
  if (t == 0) sx[m] = s_bad ? NAN : top / 127.f;
  for (int k = 8 * t; k < ldc; k += 2048) {
    uint32_t o[2] = {0u, 0u};
    if (k < K && !none) {
      float y[8];
      value(k, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j >> 2] |= (uint32_t)((int)rintf(y[j] * 127.f / top) & 255) << (8 * (j & 3));
    }
    *(u32x2*)(c + m * ldc + k) = (u32x2){o[0], o[1]};
  }
}

struct A8Out {
  const float* sx;
  const f16* s;
  const f16* res;
  long ldr;
  f16* y;
  long ldy;
};

// One row's results of 8 consecutive features n .. (fewer at the end) from their integer sums; sn: the features' scales
template <bool SILU>
__device__ __forceinline__ void a8_finish(const A8Out& out, const int (&v)[8], float sm, const float (&sn)[8], long m, int n, int N) {
  float z[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = (float)v[j] * (sm * sn[j]);
  if constexpr (SILU) {
    f16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (f16)(z[2 * j] * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z[2 * j] * -1.44269504088896341f)) * z[2 * j + 1]);
    f16* d = out.y + m * out.ldy + (n >> 1);
    if (n + 7 < N) {
      *(f16x4u*)d = o;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + 2 * j < N) d[j] = o[j];
    }
  } else {
    const f16* r = out.res ? out.res + m * out.ldr + n : nullptr;
    f16* d = out.y + m * out.ldy + n;
    f16x8 o;
    if (n + 7 < N) {
      f16x8 rv = (f16x8)((f16)0);
      if (r) rv = *(const f16x8u*)r;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = (f16)(r ? z[j] + (float)rv[j] : z[j]);
      *(f16x8u*)d = o;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < N) d[j] = (f16)(r ? z[j] + (float)r[j] : z[j]);
    }
  }
}

__device__ __forceinline__ void a8_scales(const f16* s, int n, int N, float (&sn)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) sn[j] = (float)s[min(n + j, N - 1)];
}

// ---- few rows: the weights stream once from memory into registers
// One workgroup per 16 features and up to 16 RT rows; its WV waves take an equal share of K each and add their integer
// sums in LDS.
template <bool SILU, int RT, int WV>
__global__ __launch_bounds__(64 * WV) void gemm_a8_few_kernel(const int8_t* __restrict__ c, long ldc,
                                                              const int8_t* __restrict__ wp, A8Out out, int M, int N, int K) {
  __shared__ __align__(16) int part[WV][RT * 16][20];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * RT;
  const int steps = K >> 6, s0 = steps * wv / WV, s1 = steps * (wv + 1) / WV;
  const int8_t* w = wp + (long)blockIdx.x * 16 * K + 16 * lane;
  const int8_t* x[RT];
  i32x4 acc[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    x[i] = c + (long)min(m0 + 16 * i + (lane & 15), M - 1) * ldc + 16 * (lane >> 4);
    acc[i] = (i32x4){0, 0, 0, 0};
  }
  constexpr int U = RT <= 2 ? 8 : 4;
  int k = s0;
  for (; k + U <= s1; k += U) {
    i32x4 a[U], b[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = __builtin_nontemporal_load((const i32x4*)(w + 1024L * (k + u)));
#pragma unroll
      for (int i = 0; i < RT; ++i) b[u][i] = *(const i32x4*)(x[i] + 64 * (k + u));
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], b[u][i], acc[i], 0, 0, 0);
  }
  for (; k < s1; ++k) {
    const i32x4 a = __builtin_nontemporal_load((const i32x4*)(w + 1024L * k));
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *(const i32x4*)(x[i] + 64 * k), acc[i], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) *(i32x4*)&part[wv][16 * i + (lane & 15)][4 * (lane >> 4)] = acc[i];
  __syncthreads();
  for (int t = threadIdx.x; t < 32 * RT; t += 64 * WV) {
    const int r = t >> 1, h = 8 * (t & 1), m = m0 + r, n = n0 + h;
    if (m >= M || n >= N) continue;
    int v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < WV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += part[i][r][h + j];
    float sn[8];
    a8_scales(out.s, n, N, sn);
    a8_finish<SILU>(out, v, out.sx[m], sn, m, n, N);
  }
}

// ---- many rows: tiles of 32 WN FT features x 32 WM RT rows through an LDS ring of NS stages of 128 k
// The loads, the stages and the order of a loop pass are those of GemmTile (gemm_core.h) on bytes: 16 bytes of a row or a
// feature are 16 k of v_mfma_i32_32x32x32_i8 instead of 8 of the fp16 product.
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
  // that K ends in: the second half of the weights re-reads the first, the codes behind K are 0.
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
        lds_dma16_at<LW + NW * (j - WI) * 1024>(xb, xoff[j - WI], sa);
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
    half(fc, IC<0>{}, lds, fa, IC<0>{}, IC<0>{}, 0);  // (its reads are never used)
    if (KG > 1 && nch < most) barrier();
  }

  // f(row of the tile, 8 sums) for every row and this thread's piece of 8 features, rows in passes through LDS, where the
  // groups' sums are added
  template <typename F>
  static __device__ __forceinline__ void sums(unsigned char* lds, const i32x16 (&acc)[FT][RT], F&& f) {
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wv = wid % NW, kg = wid / NW, wn = wv % WN, wm = wv / WN;
    int* buf = (int*)lds;
    constexpr int PR = BN / 8, RS = THREADS / PR, ROWS = 32 * WM * RP;
    static_assert(THREADS % PR == 0, "whole rows per step");
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
#pragma unroll 2
      for (int r = threadIdx.x / PR; r < ROWS; r += RS) {
        i32x4 a = *(const i32x4*)(buf + r * ROW + 8 * p), b = *(const i32x4*)(buf + r * ROW + 8 * p + 4);
#pragma unroll
        for (int k = 1; k < KG; ++k) {
          a += *(const i32x4*)(buf + k * PASS + r * ROW + 8 * p);
          b += *(const i32x4*)(buf + k * PASS + r * ROW + 8 * p + 4);
        }
        const int v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        const int w = r / (32 * RP), q = r - w * 32 * RP;
        f((w * RT + decltype(P)::value * RP) * 32 + q, v);
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
  i32x16 acc[FT][RT];
  T::run(lds, acc, c, ldc, wp, M, N, K, n0, m0);
  const int nb = n0 + 8 * (threadIdx.x % (T::BN / 8));
  float sn[8];
  a8_scales(out.s, nb, N, sn);
  T::sums(lds, acc, [&](int r, const int (&v)[8]) {
    const int m = m0 + r;
    if (m < M && nb < N) a8_finish<SILU>(out, v, out.sx[m], sn, m, nb, N);
  });
}

template <bool SILU, int WN, int WM, int FT, int RT, int NS, int KG = 1>
static int launch_tile(const int8_t* c, long ldc, const int8_t* wp, const A8Out& out, int M, int N, int K, hipStream_t st) {
  using T = A8Tile<WN, WM, FT, RT, NS, KG>;
  const int nfb = (N + T::BN - 1) / T::BN, nmb = (M + T::BM - 1) / T::BM;
  if ((long)nfb * nmb > 0x7FFFFFFFL) return ECD_ENOTSUP;
  hipLaunchKernelGGL((gemm_a8_kernel<SILU, WN, WM, FT, RT, NS, KG>), dim3((unsigned)(nfb * nmb)), dim3(T::THREADS), 0, st, c, ldc, wp, out,
                     M, N, K, nfb, nmb);
  return ecd_launch_status();
}

template <bool SILU, int RT, int WV>
static int launch_few(const int8_t* c, long ldc, const int8_t* wp, const A8Out& out, int M, int N, int K, hipStream_t st) {
  if ((M + 16 * RT - 1) / (16 * RT) > 65535) return ECD_ENOTSUP;
  hipLaunchKernelGGL((gemm_a8_few_kernel<SILU, RT, WV>), dim3((N + 15) / 16, (M + 16 * RT - 1) / (16 * RT)), dim3(64 * WV), 0, st, c, ldc,
                     wp, out, M, N, K);
  return ecd_launch_status();
}

template <bool SILU>
static int launch_a8(const void* cv, long ldc, const void* wv, const A8Out& out, int M, int N, int K, hipStream_t st, int cfg = 0) {
  const int8_t *c = (const int8_t*)cv, *wp = (const int8_t*)wv;
#define A8_TILE(...) return launch_tile<SILU, __VA_ARGS__>(c, ldc, wp, out, M, N, K, st)
#define A8_FEW(...) return launch_few<SILU, __VA_ARGS__>(c, ldc, wp, out, M, N, K, st)
  if (!cfg) cfg = M <= 16 ? 4 : M <= 256 ? 14 : 11;
  switch (cfg) {
    case 1: A8_FEW(1, 4);
    case 2: A8_FEW(2, 4);
    case 3: A8_FEW(4, 4);
    case 4: A8_FEW(1, 8);
    case 5: A8_FEW(2, 8);
    case 6: A8_FEW(4, 8);
    case 7: A8_TILE(2, 2, 1, 1, 8);   // 64 x 64
    case 8: A8_TILE(2, 2, 1, 2, 6);   // 64 x 128
    case 9: A8_TILE(2, 2, 2, 2, 4);   // 128 x 128
    case 10: A8_TILE(2, 2, 4, 4, 2);  // 256 x 256, 4 waves
    case 11: A8_TILE(4, 2, 2, 4, 2);  // 256 x 256, 8 waves
    case 12: A8_TILE(2, 2, 4, 2, 3);  // 256 x 128, 4 waves
    case 13: A8_TILE(2, 2, 2, 4, 3);  // 128 x 256
    case 14: A8_TILE(2, 2, 1, 1, 4);     // 64 x 64, two per CU
    case 15: A8_TILE(2, 2, 1, 1, 3);     // 64 x 64, three per CU
    case 16: A8_TILE(2, 2, 1, 2, 3);     // 64 x 128, two per CU
    case 17: A8_TILE(2, 2, 2, 1, 3);     // 128 x 64
    case 18: A8_TILE(2, 2, 2, 2, 2);     // 128 x 128, two per CU
    case 20: A8_FEW(1, 16);
    case 21: A8_TILE(2, 2, 1, 1, 4, 2);  // 64 x 64, K in two
    case 22: A8_TILE(2, 2, 1, 1, 2, 4);  // 64 x 64, K in four
    case 23: A8_TILE(1, 2, 1, 1, 3, 4);  // 32 x 64, K in four
    case 24: A8_TILE(2, 1, 1, 1, 3, 4);  // 64 x 32, K in four
    case 25: A8_TILE(2, 2, 1, 2, 3, 2);  // 64 x 128, K in two
    case 26: A8_TILE(2, 2, 2, 1, 3, 2);  // 128 x 64, K in two
    case 27: A8_TILE(2, 2, 1, 1, 2, 2);  // 64 x 64, K in two, two per CU
    case 28: A8_TILE(1, 2, 1, 1, 3, 2);  // 32 x 64, K in two, two per CU
    case 29: A8_TILE(2, 2, 2, 2, 2, 2);  // 128 x 128, K in two
    default: return ECD_EINVAL;
  }
#undef A8_TILE
#undef A8_FEW
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
  const hipStream_t st = (hipStream_t)stream;
  if (nw)
    hipLaunchKernelGGL(quant_a8_kernel<true>, dim3(M), dim3(256), 0, st, (const f16*)x, ldx, (const f16*)nw, eps,
                       (int8_t*)c, ldc, sx, K);
  else
    hipLaunchKernelGGL(quant_a8_kernel<false>, dim3(M), dim3(256), 0, st, (const f16*)x, ldx, (const f16*)nullptr, eps,
                       (int8_t*)c, ldc, sx, K);
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
  if (!a8_ok(c, ldc, sx, wp, s, y, M, N, K) || ldy < N || (res && ldr < N) || cfg < 0)
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
