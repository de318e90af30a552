// 4-bit weights in groups: the quantiser, the packing, and products of few rows (gfx950).  Layout: q4.h.
//
// Quantiser: s = fp16(max |w| / 7) and u = 8 + rint(w / s) in [0, 15]; with zero points lo = min(0, min w),
// hi = max(0, max w), s = fp16((hi - lo) / 15), z = rint(-lo / s) in [0, 15] and u = z + rint(w / s) in [0, 15].  Codes are
// those of the scale as stored; ties go to the even integer.  A group with an infinity, a NaN, or a scale past fp16 gets
// the scale NaN.
//
// Product: y[m, n] = fp16(sum_g s[n, g] sum_{k in g} x[m, k] (u[n, k] - z[n, g]) (+ res[m, n])).  The codes go into
// the matrix instructions as exact halves; a group's sum is scaled and added in fp32, the residual and SiLU(a) * b are in
// fp32 too, with one rounding at the end.
#include "q4.h"

namespace ecd {

// ---------------------------------------------------------------- quantiser
__device__ __forceinline__ float q4_value(float v) { return v; }
__device__ __forceinline__ float q4_value(f16 v) { return (float)v; }
__device__ __forceinline__ float q4_value(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }  // bf16

// the integer nearest to w / s (s > 0), ties to even, for quotients up to 16: from the rounded quotient, put right by the exact
// remainder w - n s (n s has at most 16 bits, and the remainder fits 24)
__device__ __forceinline__ int q4_nearest(float w, float s) {
  float n = fminf(fmaxf(rintf(w / s), -16.f), 16.f);
  const float d = fmaf(-n, s, w), half = 0.5f * s;
  const bool odd = ((int)n & 1) != 0;
  if (d > half || (d == half && odd)) n += 1.f;
  if (d < -half || (d == -half && odd)) n -= 1.f;
  return (int)n;
}

// One thread per 8 consecutive weights, G / 8 neighbouring threads per group; the last group of a row may be short.
template <typename T>
__global__ __launch_bounds__(256) void quantize_q4_kernel(const T* __restrict__ w, int N, int K, int lg, int ng,
                                                          uint32_t* __restrict__ q, f16* __restrict__ s,
                                                          uint8_t* __restrict__ z) {
  const int per = 1 << (lg - 3);  // threads of a group
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long group = i >> (lg - 3);
  const long n = group / ng;
  const int g = (int)(group - n * ng), o = g * per + ((int)i & (per - 1));  // octet of the row
  const bool on = n < N && o < (K >> 3);
  float v[8], lo = 0.f, hi = 0.f;
  bool bad = false;
  if (on) {
    struct __align__(16) Eight {
      T v[8];
    } e = *(const Eight*)(w + n * K + 8L * o);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = q4_value(e.v[j]);
      bad |= !(fabsf(v[j]) < INFINITY);
      lo = fminf(lo, v[j]);
      hi = fmaxf(hi, v[j]);
    }
  }
  for (int m = 1; m < per; m <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, m, 64));
    hi = fmaxf(hi, __shfl_xor(hi, m, 64));
    bad |= __shfl_xor((int)bad, m, 64) != 0;
  }
  const f16 sc = (f16)(z ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f);
  const float sf = (float)sc;
  bad |= !(sf < INFINITY);
  const bool some = !bad && sf > 0.f;
  int zp = 8;
  if (z) zp = some ? min(max(q4_nearest(-lo, sf), 0), 15) : 0;
  if (!on) return;
  uint32_t code = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int u = some ? min(max(q4_nearest(v[j], sf) + zp, 0), 15) : zp;
    code |= (uint32_t)u << (4 * j);
  }
  q[n * (K >> 3) + o] = code;
  if (((int)i & (per - 1)) == 0) {
    s[n * ng + g] = bad ? (f16)NAN : sc;
    if (z) z[n * ng + g] = (uint8_t)zp;
  }
}

// ---------------------------------------------------------------- packing
// Row n of the packed matrix is row src(n) of the given one: its own, or with `il` row j of one half and of the other in turn.
__device__ __forceinline__ long q4_source(int n, int N, int il) {
  return il ? (long)(n & 1) * (N >> 1) + (n >> 1) : n;
}

// one thread per dword of packed codes
// (a group whose scale is 0 gets codes that are its zero point: its scale is packed as 1, see pack_q4_scales_kernel)
__global__ __launch_bounds__(256) void pack_q4_codes_kernel(const uint32_t* __restrict__ q, const f16* __restrict__ s,
                                                            const uint8_t* __restrict__ z, int N, int K, int lg, int ng, int il,
                                                            uint32_t* __restrict__ codes, long dwords) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= dwords) return;
  const int nch = K >> 6, l = (int)(i >> 2) & 63, d = (int)i & 3;
  const long block = i >> 8, t = block / nch;
  const int c = (int)(block - t * nch);
  const int n = (int)t * 32 + (l & 31), o = 4 * (d & 1) + 2 * (l >> 5) + (d >> 1);
  uint32_t v = 0x88888888u, out = 0;
  if (n < N) {
    const long from = q4_source(n, N, il), g = from * ng + ((64 * c + 8 * o) >> lg);
    v = (float)s[g] != 0.f ? q[from * (K >> 3) + 8 * c + o] : z ? 0x11111111u * (z[g] & 15) : v;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) out |= (v >> (4 * e) & 15u) << (4 * (e >> 1) + 16 * (e & 1));
  codes[i] = out;
}

// one thread per scale; none is packed as 0, since products divide by them
__global__ __launch_bounds__(256) void pack_q4_scales_kernel(const f16* __restrict__ s, const uint8_t* __restrict__ z, int N,
                                                             int ng, int il, f16* __restrict__ scales, long n32) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n32 * ng) return;
  const long t = i / (32 * ng);
  const int g = (int)(i - t * 32 * ng) >> 5, n = (int)t * 32 + ((int)i & 31);
  f16 sv = (f16)1.f;
  int zv = 8;
  if (n < N) {
    const long from = q4_source(n, N, il) * ng + g;
    if ((float)s[from] != 0.f) sv = s[from];
    if (z) zv = z[from] & 15;
  }
  if (z) {
    scales[2 * i] = sv;
    scales[2 * i + 1] = (f16)(float)(1024 + zv);
  } else {
    scales[i] = sv;
  }
}

// ---------------------------------------------------------------- products of few rows
// A workgroup of KW waves computes 16 NT features of up to 8 MR rows with v_mfma_f32_16x16x32_f16; the waves share out the
// 64-wide chunks of K, and a wave keeps the loads of CW chunks in flight (a ring of registers).  GS: scales of a chunk (2 for
// groups of 32).
//
// A wave loads its chunk of x as whole lines, 8 MR rows by 8 / MR octets an instruction, works on it there (the norm), and passes
// it through its own part of LDS into the operand's lane order.
//
// The norm: x 2^e with 2^e a power of two near 1 / rms of the row's part at hand (exact), times nw in two fp16 parts, the product
// and what its rounding left (exact by the fused multiply-add), both multiplied by the codes.  Sums take 2^-e back in fp32, and
// 1 / rms of the whole row at the end, when the waves' sums meet: nothing waits for the statistics.  Up to 8 rows the second
// part takes the matrix instruction's rows 8 .. 15, which are idle otherwise.
template <int NT, int MR, int GS, bool ZP, bool NORM>
struct Q4Chunk {
  f16x8 x[MR], nw[NORM ? MR : 1];  // octets lane / (8 MR) + 8 / MR i of row lane % (8 MR)
  u32x2 code[NT];                  // octet lane / 16 of both halves
  f16 s[NT][GS];
  f16x2 sz[NT][GS];  // with zero points: (s, 1024 + z)
};

template <int KW, int CW, int NT, int MR, bool ZP, int GS, bool NORM>
__global__ __launch_bounds__(64 * KW) void mm_q4_rows_kernel(const Q4Args a) {
  constexpr bool PAIR = NORM && MR == 1;           // both parts in one instruction
  constexpr int MT = MR == 1 ? 1 : MR / 2;         // instructions' rows: tiles of 16
  constexpr int R = 8 * MR, P = 16 * MT;           // rows, and 16-byte pieces of an octet in LDS
  constexpr int LO = NORM && !PAIR ? 8 * P : 0;    // where the second parts start
  using Chunk = Q4Chunk<NT, MR, GS, ZP, NORM>;
  const int lane = threadIdx.x & 63, f = lane & 15, g4 = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nch = a.K >> 6, m0 = blockIdx.y * R, n0 = blockIdx.x * (16 * NT);
  const int xr = lane & (R - 1), xj = lane / R, tile0 = n0 >> 5, last = (a.N - 1) >> 5;
  const auto xbuf = q4_buffer(a.x + (long)m0 * a.ldx), nbuf = q4_buffer(a.nw);
  const auto cbuf = q4_buffer(a.codes + (long)tile0 * nch * 1024);
  const int tstep = ((a.K - 1) >> a.lg) + 1;  // scales of a tile's row
  const auto sbuf = q4_buffer(a.scales + (long)tile0 * tstep * (ZP ? 64 : 32));
  const int xoff = m0 + xr < a.M ? (int)(xr * a.ldx * 2) + 16 * xj : Q4_NONE;
  int coff[NT], soff[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = n0 + 16 * t, tile = min(n >> 5, last) - tile0;  // (past the last: again, and not stored)
    coff[t] = tile * nch * 1024 + 16 * ((n & 16) + f + 32 * (g4 >> 1)) + 8 * (g4 & 1);
    soff[t] = (tile * tstep * 32 + (n & 16) + f) * (ZP ? 4 : 2);
  }
  constexpr int PW = 16 * NT + 1;
  constexpr int OPS = 8 * P + LO;  // operand pieces of a chunk
  constexpr int PART = KW * P * PW * 4, OPB = KW * OPS * 16;
  __shared__ __align__(16) char lds[PART > OPB ? PART : OPB];
  __shared__ __align__(16) float us[NORM ? KW * P : 1];
  __shared__ float rs[NORM ? KW * R : 1];
  f16x8* const ops = (f16x8*)lds + wv * OPS;  // the wave's operands; afterwards part [KW][P][PW] of sums
  float* const part = (float*)lds;

  const int cnt = wv < nch ? (nch - 1 - wv) / KW + 1 : 0;  // chunks wv, wv + KW, ..
  Chunk ring[CW];
  auto load_x = [&](Chunk& k, int i) {
    const int c = min(wv + KW * i, nch - 1);
#pragma unroll
    for (int o = 0; o < MR; ++o)
      k.x[o] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(xbuf, xoff + 128 / MR * o, 128 * c, 0));
  };
  auto load_w = [&](Chunk& k, int i) {
    const int c = min(wv + KW * i, nch - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      k.code[t] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(cbuf, coff[t], 1024 * c, 0));
#pragma unroll
      for (int H = 0; H < GS; ++H) {
        const int g = (64 * c + 32 * H) >> a.lg;
        if constexpr (ZP)
          k.sz[t][H] = __builtin_bit_cast(f16x2, __builtin_amdgcn_raw_buffer_load_b32(sbuf, soff[t], 128 * g, 0));
        else
          k.s[t][H] = __builtin_bit_cast(f16, __builtin_amdgcn_raw_buffer_load_b16(sbuf, soff[t], 64 * g, 0));
      }
    }
    if constexpr (NORM)
#pragma unroll
      for (int o = 0; o < MR; ++o)
        k.nw[o] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(nbuf, 16 * xj + 128 / MR * o, 128 * c, 0));
  };
#pragma unroll
  for (int j = 0; j < CW; ++j) load_x(ring[j], j);
#pragma unroll
  for (int j = 0; j < CW; ++j) load_w(ring[j], j);

  f32x4 tot[NT][MT];  // with a norm scaled by 2^e of their rows
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < MT; ++q) tot[t][q] = (f32x4){0.f, 0.f, 0.f, 0.f};
  f16 p2 = (f16)1.f;
  float ss = 0.f;

  // every row's sums times its factor in us
  auto times_us = [&]() {
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const f32x4 u = *(const f32x4*)(us + P * wv + 16 * q + 4 * g4);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) tot[t][q][r] *= u[r];
    }
  };
  auto set_us = [&](float u) {
    if (lane < R) {
      us[P * wv + lane] = u;
      if constexpr (PAIR) us[P * wv + 8 + lane] = u;
    }
  };
  // 2^e of the rows' n chunks in the ring, and their sums of squares
  int e = 0;
  auto scale_rows = [&](int n, bool first) {
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < CW; ++j)
      if (j < n)
#pragma unroll
        for (int o = 0; o < MR; ++o)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f16x2 p = {ring[j].x[o][2 * i], ring[j].x[o][2 * i + 1]};
            v = __builtin_amdgcn_fdot2(p, p, v, false);
          }
#pragma unroll
    for (int o = R; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    ss += v;
    const float inv = __builtin_amdgcn_rsqf(v * (1.f / (64 * CW)));
    const int was = e;
    e = min(max((int)(__builtin_bit_cast(uint32_t, inv) >> 23) - 127, -14), 15);
    p2 = __builtin_bit_cast(f16, (uint16_t)((e + 15) << 10));
    if (!first) {
      set_us(__builtin_bit_cast(float, (uint32_t)(127 + e - was) << 23));
      times_us();
    }
  };

  f16x8* const put = ops + xj * P + xr;
  const f16x8* const get = ops + g4 * P + f;
  auto compute = [&](const Chunk& k) {
#pragma unroll
    for (int o = 0; o < MR; ++o) {
      f16x8 v = k.x[o];
      if constexpr (NORM) {
        const f16x8 xv = v * p2;
        v = xv * k.nw[o];
        put[8 / MR * o * P + (PAIR ? 8 : LO)] = __builtin_elementwise_fma(xv, k.nw[o], -v);
      }
      put[8 / MR * o * P] = v;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int H = 0; H < 2; ++H) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float s;
        f16x2 c0 = {(f16)-1032.f, (f16)-1032.f}, c1 = {(f16)-72.f, (f16)-72.f};
        if constexpr (ZP) {
          const f16x2 sz = k.sz[t][H & (GS - 1)];
          s = (float)sz.x;
          c0 = (f16x2){-sz.y, -sz.y};
          c1 = c0 + (f16x2){(f16)960.f, (f16)960.f};
        } else {
          s = (float)k.s[t][H & (GS - 1)];
        }
        const f16x8 w = q4_halves(k.code[t][H], c0, c1);
#pragma unroll
        for (int q = 0; q < MT; ++q) {
          if (H == 0 || GS == 2) acc[t][q] = (f32x4){0.f, 0.f, 0.f, 0.f};
          acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(get[4 * H * P + 16 * q], w, acc[t][q], 0, 0, 0);
          if constexpr (LO > 0)
            acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(get[4 * H * P + 16 * q + LO], w, acc[t][q], 0, 0, 0);
          if (H == 1 || GS == 2) {
#pragma unroll
            for (int r = 0; r < 4; ++r) tot[t][q][r] += s * acc[t][q][r];
          }
        }
      }
    }
  };
  int i0 = 0;
  for (; i0 + CW < cnt; i0 += CW) {
    if constexpr (NORM) scale_rows(CW, i0 == 0);
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      compute(ring[j]);
      __builtin_amdgcn_sched_barrier(0);
      load_x(ring[j], i0 + CW + j);
      load_w(ring[j], i0 + CW + j);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if constexpr (NORM) scale_rows(cnt - i0, i0 == 0);
#pragma unroll
  for (int j = 0; j < CW; ++j)
    if (i0 + j < cnt) {
      compute(ring[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  if constexpr (NORM) {
    set_us(__builtin_bit_cast(float, (uint32_t)(127 - e) << 23));
    times_us();
    if (lane < R) rs[R * wv + lane] = ss;
  }
  __syncthreads();  // every wave is done with its operands
  // a lane's sums: rows 16 q + 4 (lane / 16) .. + 3 of feature lane % 16
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[(wv * P + 16 * q + 4 * g4 + r) * PW + 16 * t + f] = tot[t][q][r];
  __syncthreads();
  const int W = a.silu ? 8 * NT : 16 * NT;
  for (int i = threadIdx.x; i < R * W; i += 64 * KW) {
    const int r = i / W, j = i - r * W, m = m0 + r;
    const int n = (a.silu ? n0 / 2 : n0) + j;
    if (m >= a.M || n >= (a.silu ? a.N / 2 : a.N)) continue;
    float inv = 1.f;
    if constexpr (NORM) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) v += rs[R * w + r];
      inv = 1.0f / sqrtf(v / (float)a.K + a.eps);
    }
    auto add = [&](int c) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        v += part[(w * P + r) * PW + c];
        if constexpr (PAIR) v += part[(w * P + 8 + r) * PW + c];
      }
      return NORM ? v * inv : v;
    };
    float v;
    if (a.silu) {
      v = silu_mul(add(2 * j), add(2 * j + 1));
    } else {
      v = add(j);
      if (a.res) v += (float)a.res[(long)m * a.ldr + n];
    }
    a.y[(long)m * a.ldy + n] = (f16)v;
  }
}

template <int KW, int CW, int NT, int MR, bool ZP, int GS, bool NORM>
static int launch_rows(const Q4Args& a, hipStream_t st) {
  hipLaunchKernelGGL((mm_q4_rows_kernel<KW, CW, NT, MR, ZP, GS, NORM>),
                     dim3((a.N + 16 * NT - 1) / (16 * NT), (a.M + 8 * MR - 1) / (8 * MR)), dim3(64 * KW), 0, st, a);
  return ecd_launch_status();
}

template <int KW, int CW, int NT, bool ZP, int GS, bool NORM>
static int rows_by_m(const Q4Args& a, hipStream_t st) {
  if (a.M <= 8) return launch_rows<KW, CW, NT, 1, ZP, GS, NORM>(a, st);
  return launch_rows<KW, CW, NT, 2, ZP, GS, NORM>(a, st);
}

template <int KW, int CW, int NT>
static int rows_by_weights(const Q4Args& a, bool zp, hipStream_t st) {
#define Q4_ROWS(Z, G) return a.nw ? rows_by_m<KW, CW, NT, Z, G, true>(a, st) : rows_by_m<KW, CW, NT, Z, G, false>(a, st)
  if (zp) {
    if (a.lg == 5) Q4_ROWS(true, 2);
    Q4_ROWS(true, 1);
  }
  if (a.lg == 5) Q4_ROWS(false, 2);
  Q4_ROWS(false, 1);
#undef Q4_ROWS
}

// One workgroup per CU where the features give as many: 16, 32 or 64 features each.  Over a long K, where 16 features leave CUs
// idle anyway, twice the waves (3072 x 8192: 1 row 5.7 -> 5.1 us, 8 rows 7.7 -> 7.4; 3072 x 3072 with 8 rows 4.2 and 5.0).
// us of 16 / 32 / 64 features: 8 rows of 3072 x 3072 4.2 / 4.7 / 6.4, 5120 x 3072 6.1 / 4.9 / 6.6, 16384 x 3072 9.9 / 7.4 / 7.2;
// with the norm 5.5 / 6.1 / 7.8, 7.7 / 6.2 / 7.9, 12.2 / 9.4 / 8.4.  Four waves instead of eight: 5.2 (32 features), 5.3, 8.2.
static int mm_rows(const Q4Args& a, bool zp, hipStream_t st) {
  const int n16 = (a.N + 15) / 16;
  if (n16 <= 256) return a.K >= 6144 ? rows_by_weights<16, 4, 1>(a, zp, st) : rows_by_weights<8, 3, 1>(a, zp, st);
  if (n16 <= 512) return rows_by_weights<8, 3, 2>(a, zp, st);
  return rows_by_weights<8, 3, 4>(a, zp, st);
}

// ---------------------------------------------------------------- norm of many rows
// y = fp16(x / rms * nw), one rounding, for the matrix tiles, whose operands are fp16.  A workgroup per row; the second read of the
// row comes from the caches.
__global__ __launch_bounds__(256) void q4_norm_kernel(const f16* __restrict__ x, long ldx, const f16* __restrict__ nw, float eps,
                                                      f16* __restrict__ y, int K) {
  __shared__ float part[4];
  const f16* xr = x + (long)blockIdx.x * ldx;
  float ss = 0.f;
  for (int k = 8 * threadIdx.x; k < K; k += 2048) {
    const f16x8 v = *(const f16x8*)(xr + k);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += (float)v[j] * (float)v[j];
  }
  ss = wave_sum_dpp(ss);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
  __syncthreads();
  const float inv = 1.0f / sqrtf((part[0] + part[1] + part[2] + part[3]) / (float)K + eps);
  for (int k = 8 * threadIdx.x; k < K; k += 2048) {
    const f16x8 v = *(const f16x8*)(xr + k), w = *(const f16x8*)(nw + k);
    f16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (f16)((float)v[j] * inv * (float)w[j]);
    *(f16x8*)(y + (long)blockIdx.x * K + k) = o;
  }
}

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
static int log2_group(int group) { return group == 32 ? 5 : group == 64 ? 6 : 7; }

}  // namespace ecd

using namespace ecd;

extern "C" {

int ecd_quantize_rows_q4(const void* w, int type, void* q, void* s, void* z, int N, int K, int group, void* stream) {
  if (!w || !q || !s || N <= 0 || K <= 0 || K % 64 || !group_ok(group) || type < 0 || type > 2 || !al16(w) || ((uintptr_t)q & 3))
    return ECD_EINVAL;
  const int lg = log2_group(group), ng = (K + group - 1) / group;
  const long blocks = ((((long)N * ng) << (lg - 3)) + 255) / 256;
  if (blocks > 0x7FFFFFFFL) return ECD_ENOTSUP;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks);
  if (type == 0)
    hipLaunchKernelGGL(quantize_q4_kernel<float>, grid, dim3(256), 0, st, (const float*)w, N, K, lg, ng, (uint32_t*)q, (f16*)s,
                       (uint8_t*)z);
  else if (type == 1)
    hipLaunchKernelGGL(quantize_q4_kernel<f16>, grid, dim3(256), 0, st, (const f16*)w, N, K, lg, ng, (uint32_t*)q, (f16*)s,
                       (uint8_t*)z);
  else
    hipLaunchKernelGGL(quantize_q4_kernel<uint16_t>, grid, dim3(256), 0, st, (const uint16_t*)w, N, K, lg, ng, (uint32_t*)q,
                       (f16*)s, (uint8_t*)z);
  return ecd_launch_status();
}

long ecd_packed_bytes_q4(int N, int K) { return N > 0 && K > 0 && K % 64 == 0 ? (long)q4_tiles(N) * 16 * K : 0; }

int ecd_pack_q4(const void* q, const void* s, const void* z, int N, int K, int group, int interleave, void* codes, void* scales,
                void* stream) {
  if (!q || !s || !codes || !scales || N <= 0 || K <= 0 || K % 64 || !group_ok(group) || (interleave && N % 2) ||
      ((uintptr_t)q & 3) || !al16(codes) || !al16(scales))
    return ECD_EINVAL;
  const int ng = (K + group - 1) / group;
  const long dwords = ecd_packed_bytes_q4(N, K) / 4, n32 = 32L * q4_tiles(N);
  if ((dwords + 255) / 256 > 0x7FFFFFFFL || (n32 * ng + 255) / 256 > 0x7FFFFFFFL || N > 0x7FFFFFFF - 32) return ECD_ENOTSUP;
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(pack_q4_codes_kernel, dim3((unsigned)((dwords + 255) / 256)), dim3(256), 0, st, (const uint32_t*)q,
                     (const f16*)s, (const uint8_t*)z, N, K, log2_group(group), ng, interleave, (uint32_t*)codes, dwords);
  hipLaunchKernelGGL(pack_q4_scales_kernel, dim3((unsigned)((n32 * ng + 255) / 256)), dim3(256), 0, st, (const f16*)s,
                     (const uint8_t*)z, N, ng, interleave, (f16*)scales, n32);
  return ecd_launch_status();
}

// Up to 16 rows the few-row kernel (plan 0), but for 9 .. 16 rows of a long K the matrix tiles, which split K over more
// workgroups (16 rows, 1024 x 8192: 10.7 and 8.6 us; 3072 x 3072: 5.7 and 7.4).
int ecd_mm_q4_plan(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 64) return ECD_EINVAL;
  return M <= 8 || (M <= 16 && K < 6144) ? 0 : gemm_q4_plan(M, N, K);
}

long ecd_mm_q4_ws_bytes(int M, int N, int K, int plan, int norm) {
  if (M <= 0 || N <= 0 || K <= 0 || plan <= 0) return 0;
  const long ks = plan >> 8, sums = ks > 1 ? ks * M * ((N + 7L) / 8 * 8) * 4 : 0;
  return sums + (norm ? 2L * M * K : 0);
}

int ecd_mm_q4(const void* x, long ldx, const void* nw, float eps, const void* codes, const void* scales, int zeros, int group,
              const void* res, long ldr, void* y, long ldy, int M, int N, int K, int silu, int plan, void* ws, void* stream) {
  const int cols = silu ? N / 2 : N;
  const int tile = plan & 255, ks = plan >> 8;
  if (!x || !codes || !scales || !y || M <= 0 || N <= 0 || K <= 0 || K % 64 || !group_ok(group) || ldx < K || ldx % 8 ||
      !al16(x) || (nw && !al16(nw)) || !al16(codes) || !al16(scales) || ldy < cols || (res && ldr < cols) ||
      (silu && (N % 2 || res)) || (nw && !(eps >= 0.f)) || (plan ? tile < 1 || tile > Q4_TILES || ks < 1 || ks > K / 64 : M > 16) ||
      (ecd_mm_q4_ws_bytes(M, N, K, plan, nw != nullptr) && (!ws || !al16(ws))))
    return ECD_EINVAL;
  if (N > 0x7FFFFFFF - 255 || K > 1 << 24 || ks > 65535) return ECD_ENOTSUP;
  Q4Args a{(const f16*)x, ldx, (const f16*)nw, eps, (const uint8_t*)codes, (const f16*)scales, log2_group(group),
           (const f16*)res, ldr, (f16*)y, ldy, M, N, K, silu};
  const hipStream_t st = (hipStream_t)stream;
  if (!plan) return 16 * ldx * 2 > 0x7FFFFFFFL ? ECD_ENOTSUP : mm_rows(a, zeros, st);
  if (nw) {
    a.x = (const f16*)((char*)ws + ecd_mm_q4_ws_bytes(M, N, K, plan, 0));
    a.ldx = K;
    const int rc = gemm_q4(a, zeros, tile, (float*)ws, ks, nullptr, false);  // (refused sizes before the norm is launched)
    if (rc != ECD_OK) return rc;
    hipLaunchKernelGGL(q4_norm_kernel, dim3(M), dim3(256), 0, st, (const f16*)x, ldx, (const f16*)nw, eps, (f16*)a.x, K);
    const int err = ecd_launch_status();
    if (err != ECD_OK) return err;
  }
  return gemm_q4(a, zeros, tile, (float*)ws, ks, st, true);
}

}  // extern "C"
