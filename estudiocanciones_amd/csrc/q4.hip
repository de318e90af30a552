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

// One thread per 8 consecutive weights, G / 8 neighbouring threads per group; the last group of a row may be short.  16384 x 3072
// from fp32 62 us (3.6 TB/s, bound by memory), from 16 bits 60 to 64 (the quotients): set-up work, once per model.
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
// A workgroup of KW waves computes 16 NT features of up to R = 4 XO rows with v_mfma_f32_16x16x32_f16; the waves share out the
// pairs of 64-wide chunks of K, and a wave keeps the loads of CW pairs in flight (a ring of registers).
//
// What such a kernel runs into first is the address path: a load instruction takes a CU 16 cycles at least, whatever it
// brings, and longer if neighbouring lanes are in different lines.  So every load has 16 bytes a lane where there is as
// much: a lane takes the 16 bytes of its feature in one chunk of the pair (half the lanes each), and the matrix instruction's k
// are numbered to match; x comes as whole lines, 4 rows an instruction, is worked on in that order (the norm) and passes through
// the wave's own part of LDS into the operand's; scales of up to four (feature tile, group) slots come with one load and are
// spread by lane swaps.  Groups under 128 split the pair: x is zeroed outside the group at hand (GS = 128 / group).
//
// The norm: x 2^e with 2^e a power of two near 1 / rms of the row's part at hand (exact), times nw in two fp16 parts, the product
// and what its rounding left (exact by the fused multiply-add), both multiplied by the codes.  Sums take 2^-e back in fp32, and
// 1 / rms of the whole row at the end, when the waves' sums meet: nothing waits for the statistics.  Up to 8 rows the second
// part takes the matrix instruction's rows 8 .. 15, which are idle otherwise.  A value is at most sqrt(128 CW) < 20 times the rms of
// its part, so with weights below 2^11 every product fits fp16; where a part's weights reach more, all of them go in divided by
// 2^5, and e tells the sums.
//
// Measured in a graph (of it 2.2 us a launch): 1 x 8197 x 3072 with its norm 6.4 us, 8 x 5120 x 3072 with its norm 5.6, 8 x 3072 x 8192
// with a residual 5.2 (2.5 TB/s), 8 x 16384 x 3072 with norm and SiLU 8.6 (3.0 TB/s), 48 x 3072 x 3072 in groups of 64 6.9.  What is
// left is about 1 us to the first bytes, the address path, the conversion (9 instructions for 8 codes) and the sums' way through LDS.
template <int NT, int XO, int GS, bool ZP, bool NORM>
struct Q4Pair {
  static constexpr int SLOTS = NT * GS, SL = (SLOTS + 3) / 4;  // scales of 16 features each, and loads for them
  f16x8 x[XO], nw;   // octet lane % 16 of rows lane / 16 + 4 i
  u32x4 code[NT];    // chunk lane / 32, half (lane / 16) % 2
  f16 s[SL];         // slot 4 i + lane / 16
  f16x2 sz[SL];      // with zero points: (s, 1024 + z)
};

// v of lanes 16 i .. 16 i + 15 for all lanes, i < n
template <int n>
__device__ __forceinline__ void spread16(uint32_t v, uint32_t* to) {
  if constexpr (n == 1) {
    to[0] = v;
  } else if constexpr (n == 2) {  // (the upper half of the lanes holds the lower's again)
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    to[0] = p[0], to[1] = p[1];
  } else {
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    spread16<2>(h[0], to);
    spread16<2>(h[1], to + 2);
  }
}

// the sum over 16 neighbouring lanes, for all of them
__device__ __forceinline__ float row_sum16(float v) {
  auto ror = [&](auto n) {
    return __builtin_bit_cast(float, dpp_u32<0x120 + decltype(n)::value, 0xF>(__builtin_bit_cast(uint32_t, v), 0));
  };
  v += ror(std::integral_constant<int, 8>());
  v += ror(std::integral_constant<int, 4>());
  v += ror(std::integral_constant<int, 2>());
  v += ror(std::integral_constant<int, 1>());
  return v;
}

template <int KW, int CW, int NT, int XO, bool ZP, int GS, bool NORM>
__global__ __launch_bounds__(64 * KW) void mm_q4_rows_kernel(const f16* __restrict__ x, const uint8_t* __restrict__ codes,
                                                             const f16* __restrict__ scales, const f16* __restrict__ nw, int N,
                                                             int K, int M, int lg, long ldx, float eps, const f16* res, long ldr,
                                                             f16* y, long ldy, int silu) {
  constexpr bool PAIR = NORM && XO < 4;            // both parts in one instruction
  constexpr int R = 4 * XO, P = 16;                // rows, and those of an instruction
  constexpr int PP = P + 1;                        // 16-byte pieces of an octet in LDS (odd: a line's octets fall on all banks)
  constexpr int LO = NORM && !PAIR ? 16 * PP : 0;  // where the second parts start
  using Pair = Q4Pair<NT, XO, GS, ZP, NORM>;
  const int lane = threadIdx.x & 63, f = lane & 15, g4 = lane >> 4, h = g4 & 1, cc = g4 >> 1;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nch = K >> 6, npr = (nch + 1) >> 1, m0 = blockIdx.y * R, n0 = blockIdx.x * (16 * NT);
  const int xr = lane >> 4, xj = lane & 15, tile0 = n0 >> 5, last = (N - 1) >> 5;
  const int ng = ((K - 1) >> lg) + 1;
  const auto xbuf = q4_buffer(x + (long)m0 * ldx), nbuf = q4_buffer(nw);
  const auto cbuf = q4_buffer(codes + (long)tile0 * nch * 1024);
  const auto sbuf = q4_buffer(scales + (long)tile0 * ng * (ZP ? 64 : 32));
  int xoff[XO];
#pragma unroll
  for (int o = 0; o < XO; ++o) {
    const int r = xr + 4 * o;
    xoff[o] = m0 + r < M ? (int)(r * ldx * 2) + 16 * xj : Q4_NONE;
  }
  const int coff = 16 * (f + 32 * h);
  int ctile[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = n0 + 16 * t;  // (a tile past the last: the last again, and not stored)
    ctile[t] = (min(n >> 5, last) - tile0) * nch * 1024 + 16 * (n & 16);
  }
  int soff[Pair::SL], sg[Pair::SL];
#pragma unroll
  for (int i = 0; i < Pair::SL; ++i) {
    const int slot = (4 * i + g4) % Pair::SLOTS, n = n0 + 16 * (slot / GS);
    soff[i] = ((min(n >> 5, last) - tile0) * ng * 32 + (n & 16) + f) * (ZP ? 4 : 2);
    sg[i] = slot % GS;
  }
  constexpr int PW = 16 * NT + 4;    // (rows of 4 lanes' sums fall on different banks)
  constexpr int OPS = 16 * PP + LO;  // operand pieces of a pair
  constexpr int PR = PAIR ? 8 : P;   // rows of sums in LDS
  constexpr int PART = KW * PR * PW * 4, OPB = KW * OPS * 16;
  __shared__ __align__(16) char lds[PART > OPB ? PART : OPB];
  __shared__ __align__(16) float us[NORM ? KW * P : 1];
  __shared__ float rs[NORM ? KW * R : 1];
  f16x8* const ops = (f16x8*)lds + wv * OPS;  // the wave's operands; afterwards part [KW][PR][PW] of sums
  float* const part = (float*)lds;

  const int cnt = wv < npr ? (npr - 1 - wv) / KW + 1 : 0;  // pairs wv, wv + KW, ..
  Pair ring[CW];
  auto load_x = [&](Pair& k, int i) {
    const int p = min(wv + KW * i, npr - 1);
    const bool in = 2 * p + (xj >> 3) < nch;  // (an odd number of chunks: zeros in place of the last)
#pragma unroll
    for (int o = 0; o < XO; ++o)
      k.x[o] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(xbuf, in ? xoff[o] : Q4_NONE, 256 * p, 0));
    if constexpr (NORM)
      k.nw = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(nbuf, in ? 16 * xj : Q4_NONE, 256 * p, 0));
  };
  auto load_w = [&](Pair& k, int i) {
    const int p = min(wv + KW * i, npr - 1);
    const int c = coff + 1024 * min(2 * p + cc, nch - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      k.code[t] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(cbuf, c, ctile[t], 0));
#pragma unroll
    for (int q = 0; q < Pair::SL; ++q) {
      const int g = GS == 1 ? p : min(GS * p + sg[q], ng - 1);
      if constexpr (ZP)
        k.sz[q] = __builtin_bit_cast(f16x2, __builtin_amdgcn_raw_buffer_load_b32(sbuf, soff[q] + 128 * g, 0, 0));
      else
        k.s[q] = __builtin_bit_cast(f16, __builtin_amdgcn_raw_buffer_load_b16(sbuf, soff[q] + 64 * g, 0, 0));
    }
  };
#pragma unroll
  for (int j = 0; j < CW; ++j) load_x(ring[j], j);
#pragma unroll
  for (int j = 0; j < CW; ++j) load_w(ring[j], j);
  // the thread's outputs and their residuals, in time for the end (where there are none, of the codes, and not used)
  constexpr int PER = (R * 16 * NT + 64 * KW - 1) / (64 * KW);
  const int lw = __builtin_ctz(16 * NT) - (silu ? 1 : 0), nout = silu ? N / 2 : N;
  f16 rv[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = threadIdx.x + i * 64 * KW, m = m0 + (at >> lw), n = (blockIdx.x << lw) + (at & ((1 << lw) - 1));
    rv[i] = *(res && (at >> lw) < R && m < M && n < nout ? res + (long)m * ldr + n : (const f16*)codes);
  }
  __builtin_amdgcn_sched_barrier(0);

  f32x4 tot[NT];  // with a norm scaled by 2^e of their rows
#pragma unroll
  for (int t = 0; t < NT; ++t) tot[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  f16 p2[XO];
  float ss[XO];
  int e[XO];
#pragma unroll
  for (int o = 0; o < XO; ++o) p2[o] = (f16)1.f, ss[o] = 0.f, e[o] = 0;

  // every row's sums times its factor in us
  auto times_us = [&]() {
    const f32x4 u = *(const f32x4*)(us + P * wv + 4 * g4);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) tot[t][r] *= u[r];
  };
  auto set_us = [&](int o, float u) {
    if (xj == 0) {
      us[P * wv + 4 * o + xr] = u;
      if constexpr (PAIR) us[P * wv + 8 + 4 * o + xr] = u;
    }
  };
  // 2^e of the rows' n pairs in the ring, and their sums of squares; weights of 2^11 and more go 2^-5 times into the products.  The bits
  // of all weights in one word rule those out while none is 2 or more (8 x 5120 x 3072 5.51 -> 5.63 us; by their maximum 5.74)
  auto scale_rows = [&](int n, bool first) {
    int was[XO];
#pragma unroll
    for (int o = 0; o < XO; ++o) was[o] = e[o];
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < CW; ++j)  // (all of the ring's, which are the row's in any case)
#pragma unroll
      for (int i = 0; i < 4; ++i) bits |= __builtin_bit_cast(u32x4, ring[j].nw)[i];
#pragma unroll
    for (int o = 0; o < XO; ++o) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < CW; ++j)
        if (j < n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f16x2 p = {ring[j].x[o][2 * i], ring[j].x[o][2 * i + 1]};
            v = __builtin_amdgcn_fdot2(p, p, v, false);
          }
      v = row_sum16(v);
      ss[o] += v;
      const float inv = __builtin_amdgcn_rsqf(v * (1.f / (128 * CW)));
      e[o] = min(max((int)(__builtin_bit_cast(uint32_t, inv) >> 23) - 127, -14), 15);
      p2[o] = __builtin_bit_cast(f16, (uint16_t)((e[o] + 15) << 10));
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64((bits & 0x40004000u) != 0) != 0, 0)) {
      f16x2 most = {(f16)0.f, (f16)0.f};  // of the magnitudes
#pragma unroll
      for (int j = 0; j < CW; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f16x2 w = {ring[j].nw[2 * i], ring[j].nw[2 * i + 1]};
          asm("v_pk_maximum3_f16 %0, %0, %1, %1 neg_lo:[0,0,1] neg_hi:[0,0,1]" : "+v"(most) : "v"(w));
        }
      if (__builtin_amdgcn_ballot_w64(most.x >= (f16)2048.f || most.y >= (f16)2048.f)) {
#pragma unroll
        for (int j = 0; j < CW; ++j) ring[j].nw = ring[j].nw * (f16)0.03125f;
#pragma unroll
        for (int o = 0; o < XO; ++o) e[o] -= 5;
      }
    }
    if (!first) {
#pragma unroll
      for (int o = 0; o < XO; ++o) set_us(o, __builtin_bit_cast(float, (uint32_t)(127 + e[o] - was[o]) << 23));
      times_us();
    }
  };

  f16x8* const put = ops + xj * PP + xr;
  const f16x8* const get = ops + (8 * cc + 2 * h) * PP + f;
  auto compute = [&](const Pair& k) {
#pragma unroll
    for (int o = 0; o < XO; ++o) {
      f16x8 v = k.x[o];
      if constexpr (NORM) {
        const f16x8 xv = v * p2[o];
        v = xv * k.nw;
        put[4 * o + (PAIR ? 8 : LO)] = __builtin_elementwise_fma(xv, k.nw, -v);
      }
      put[4 * o] = v;
    }
    uint32_t sc[Pair::SL * 4];
#pragma unroll
    for (int q = 0; q < Pair::SL; ++q) {
      uint32_t v;
      if constexpr (ZP)
        v = __builtin_bit_cast(uint32_t, k.sz[q]);
      else
        v = __builtin_bit_cast(uint16_t, k.s[q]);
      spread16<(Pair::SLOTS < 4 ? Pair::SLOTS : 4)>(v, sc + 4 * q);
    }
    f16x8 xa[4], xb[LO > 0 ? 4 : 1];  // operands for dword 2 S + H of the lanes' codes
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      xa[j] = get[(4 * (j & 1) + (j >> 1)) * PP];
      if constexpr (LO > 0) xb[j] = get[(4 * (j & 1) + (j >> 1)) * PP + LO];
    }
    const f16x8 none = {};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f16x8 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f16x2 c0 = {(f16)-1032.f, (f16)-1032.f}, c1 = {(f16)-72.f, (f16)-72.f};
        if constexpr (ZP) {
          const uint32_t* st = sc + t * GS + (j & 1) * (GS / 4);  // (of the lane's chunk, and the dword's half of it)
          const f16 z = __builtin_bit_cast(f16x2, cc ? st[GS / 2] : st[0]).y;
          c0 = (f16x2){-z, -z};
          c1 = c0 + (f16x2){(f16)960.f, (f16)960.f};
        }
        w[j] = q4_halves(k.code[t][j], c0, c1);
      }
#pragma unroll
      for (int g = 0; g < GS; ++g) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (GS == 4 && (j & 1) != (g & 1)) continue;
          const bool mine = GS == 1 || cc == 2 * g / GS;
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(mine ? xa[j] : none, w[j], acc, 0, 0, 0);
          if constexpr (LO > 0) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(mine ? xb[j] : none, w[j], acc, 0, 0, 0);
        }
        const float s = (float)__builtin_bit_cast(f16x2, sc[t * GS + g]).x;
#pragma unroll
        for (int r = 0; r < 4; ++r) tot[t][r] += s * acc[r];
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
#pragma unroll
    for (int o = 0; o < XO; ++o) {
      set_us(o, __builtin_bit_cast(float, (uint32_t)(127 - e[o]) << 23));
      if (xj == 0) rs[R * wv + 4 * o + xr] = ss[o];
    }
    times_us();
  }
  __syncthreads();  // every wave is done with its operands
  // a lane's sums: rows 4 (lane / 16) .. + 3 of feature lane % 16
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float v = tot[t][r];
      if constexpr (PAIR) {  // the second parts' sums are in the upper lanes
        const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
        v = __builtin_bit_cast(float, (uint32_t)p[0]) + __builtin_bit_cast(float, (uint32_t)p[1]);
      }
      if (!PAIR || lane < 32) part[(wv * PR + 4 * g4 + r) * PW + 16 * t + f] = v;
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = threadIdx.x + i * 64 * KW, r = at >> lw, j = at & ((1 << lw) - 1), m = m0 + r, n = (blockIdx.x << lw) + j;
    if (r >= R || m >= M || n >= nout) continue;
    float inv = 1.f;
    if constexpr (NORM) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) v += rs[R * w + r];
      inv = 1.0f / sqrtf(v / (float)K + eps);
    }
    auto add = [&](int c) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) v += part[(w * PR + r) * PW + c];
      return NORM ? v * inv : v;
    };
    float v;
    if (silu) {
      v = silu_mul(add(2 * j), add(2 * j + 1));
    } else {
      v = add(j);
      if (res) v += (float)rv[i];
    }
    y[(long)m * ldy + n] = (f16)v;
  }
}

template <int KW, int CW, int NT, int XO, bool ZP, int GS, bool NORM>
static int launch_rows(const Q4Args& a, hipStream_t st) {
  hipLaunchKernelGGL((mm_q4_rows_kernel<KW, CW, NT, XO, ZP, GS, NORM>),
                     dim3((a.N + 16 * NT - 1) / (16 * NT), (a.M + 4 * XO - 1) / (4 * XO)), dim3(64 * KW), 0, st, a.x, a.codes,
                     a.scales, a.nw, a.N, a.K, a.M, a.lg, a.ldx, a.eps, a.res, a.ldr, a.y, a.ldy, a.silu);
  return ecd_launch_status();
}
template <int KW, int CW, int NT, bool ZP, int GS, bool NORM>
static int rows_by_m(const Q4Args& a, hipStream_t st) {
  if (a.M <= 4) return launch_rows<KW, CW, NT, 1, ZP, GS, NORM>(a, st);
  if (a.M <= 8) return launch_rows<KW, CW, NT, 2, ZP, GS, NORM>(a, st);
  return launch_rows<KW, CW, NT, 4, ZP, GS, NORM>(a, st);
}
template <int KW, int CW, int NT, bool ZP, int GS>
static int rows_by_norm(const Q4Args& a, hipStream_t st) {
  return a.nw ? rows_by_m<KW, CW, NT, ZP, GS, true>(a, st) : rows_by_m<KW, CW, NT, ZP, GS, false>(a, st);
}
template <int KW, int CW, int NT, bool ZP>
static int rows_by_group(const Q4Args& a, hipStream_t st) {
  if (a.lg == 7) return rows_by_norm<KW, CW, NT, ZP, 1>(a, st);
  if (a.lg == 6) return rows_by_norm<KW, CW, NT, ZP, 2>(a, st);
  return rows_by_norm<KW, CW, NT, ZP, 4>(a, st);
}
template <int KW, int CW, int NT>
static int rows_by_weights(const Q4Args& a, bool zp, hipStream_t st) {
  return zp ? rows_by_group<KW, CW, NT, true>(a, st) : rows_by_group<KW, CW, NT, false>(a, st);
}

// form: features of a workgroup, 16 << (form - 1)
static int mm_rows(const Q4Args& a, bool zp, int form, hipStream_t st) {
  if (32L * a.ldx > 0x7FFFFFFFL || (a.M + 15) / 16 > 65535) return ECD_ENOTSUP;
  if (form == 1) return rows_by_weights<8, 3, 1>(a, zp, st);
  if (form == 2) return rows_by_weights<8, 3, 2>(a, zp, st);
  return rows_by_weights<8, 2, 4>(a, zp, st);
}
// One workgroup per CU where the features give as many.  us of 16 / 32 / 64 features: 8 rows of 3072 x 3072 3.6 / 4.1 / 5.2,
// 5120 x 3072 5.1 / 4.7 / 5.8, 16384 x 3072 with a norm 11.5 / 9.0 / 8.8 (and SiLU), 1 row of 8197 x 3072 with a norm
// 7.2 / 7.0 / 6.9.  Sixteen waves instead of eight: 3.5, 4.6, 8.9, 7.0 with half the pairs in flight, and more rows spill.
static int rows_form(int N) {
  const int n16 = (N + 15) / 16;
  return n16 <= 256 ? 1 : n16 <= 512 ? 2 : 3;
}

// ---------------------------------------------------------------- norm of many rows
// y = fp16(x / rms * nw), one rounding, for the matrix tiles, whose operands are fp16: it adds about as much to a product's error as
// the rounding of the result (2.1e-4 -> 2.9e-4 of the result, rms).  A SiLU multiplies two such products (3.7e-4), so before one
// the rows go in as two parts, the second what the first's rounding left, 64 of each in turn (2.1e-4 again, for up to
// twice the time: 384 rows of 16384 x 3072 92 us instead of 52).  A workgroup per row; the second read of the row comes from the caches.
template <bool TWO>
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
    f16x8 o, rest;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float u = (float)v[j] * inv * (float)w[j];
      o[j] = (f16)u;
      rest[j] = (f16)(u - (float)o[j]);
    }
    if constexpr (TWO) {
      f16* const d = y + (long)blockIdx.x * 2 * K + 2 * k - (k & 63);  // 128 (k / 64) + k % 64
      *(f16x8*)d = o;
      *(f16x8*)(d + 64) = rest;
    } else {
      *(f16x8*)(y + (long)blockIdx.x * K + k) = o;
    }
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

// Up to 16 rows the few-row kernel with the norm inside (plan 0): 9 .. 16 rows of 3072 x 3072 4.0 us and with a norm 5.7, of
// 1024 x 8192 5.9 and 10.0, where the matrix tiles take 7.7, 10.1, 8.2 and 11.4.
static int mm_q4_plan(int M, int N, int K, Q4Among among) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 64) return ECD_EINVAL;
  return M <= 16 ? 0 : gemm_q4_plan(M, N, K, among);
}
// (for tuning, as the few-row plans with a norm in one part are: no call of the package asks for them)
int ecd_mm_q4_plan(int M, int N, int K) { return mm_q4_plan(M, N, K, Q4_ONLY_TILES); }
int ecd_mm_q4_choice(int M, int N, int K) { return mm_q4_plan(M, N, K, Q4_PLAIN); }
int ecd_mm_q4_norm_choice(int M, int N, int K, int silu) { return mm_q4_plan(M, N, K, silu ? Q4_NORM_SILU : Q4_NORM); }

long ecd_mm_q4_ws_bytes(int M, int N, int K, int plan, int norm) {
  if (M <= 0 || N <= 0 || K <= 0 || plan <= 0) return 0;
  const long ks = plan >> 8, sums = ks > 1 ? ks * M * ((N + 7L) / 8 * 8) * 4 : 0;
  const bool rows = (plan & 31) > Q4_ROWS_AT, two = plan & Q4_TWO;
  return sums + (!norm || (rows && two) ? 0 : (two ? 4L : 2L) * M * K);
}

int ecd_mm_q4(const void* x, long ldx, const void* nw, float eps, const void* codes, const void* scales, int zeros, int group,
              const void* res, long ldr, void* y, long ldy, int M, int N, int K, int silu, int plan, void* ws, void* stream) {
  const int cols = silu ? N / 2 : N;
  const bool two = plan & Q4_TWO;
  const int tile = (plan & 255) - (two ? Q4_TWO : 0), ks = plan >> 8;
  const bool rows = tile > Q4_ROWS_AT && tile <= Q4_ROWS_AT + Q4_ROWS;
  const bool planned = rows ? ks == 1 : tile >= 1 && tile <= Q4_TILES && ks >= 1 && ks <= K / 64;
  if (!x || !codes || !scales || !y || M <= 0 || N <= 0 || K <= 0 || K % 64 || !group_ok(group) || ldx < K || ldx % 8 ||
      !al16(x) || (nw && !al16(nw)) || !al16(codes) || !al16(scales) || ldy < cols || (res && ldr < cols) ||
      (silu && (N % 2 || res)) || (nw && !(eps >= 0.f)) || (plan ? !planned || (two && !nw) : M > 16) ||
      (ecd_mm_q4_ws_bytes(M, N, K, plan, nw != nullptr) && (!ws || !al16(ws))))
    return ECD_EINVAL;
  if (N > 0x7FFFFFFF - 255 || K > 1 << 24 || ks > 65535) return ECD_ENOTSUP;
  Q4Args a{(const f16*)x, ldx, (const f16*)nw, eps, (const uint8_t*)codes, (const f16*)scales, log2_group(group),
           (const f16*)res, ldr, (f16*)y, ldy, M, N, K, silu, 0};
  const hipStream_t st = (hipStream_t)stream;
  if (!plan) return mm_rows(a, zeros, rows_form(N), st);
  if (nw && !(rows && two)) {
    a.x = (const f16*)((char*)ws + ecd_mm_q4_ws_bytes(M, N, K, plan, 0));
    a.ldx = two ? 2L * K : K;
    a.two = two;
    if (!rows) {  // (refused sizes before the norm is launched)
      const int rc = gemm_q4(a, zeros, tile, (float*)ws, ks, nullptr, false);
      if (rc != ECD_OK) return rc;
    } else if ((M + 15) / 16 > 65535) {
      return ECD_ENOTSUP;
    }
    if (two)
      hipLaunchKernelGGL(q4_norm_kernel<true>, dim3(M), dim3(256), 0, st, (const f16*)x, ldx, (const f16*)nw, eps, (f16*)a.x, K);
    else
      hipLaunchKernelGGL(q4_norm_kernel<false>, dim3(M), dim3(256), 0, st, (const f16*)x, ldx, (const f16*)nw, eps, (f16*)a.x, K);
    const int err = ecd_launch_status();
    if (err != ECD_OK) return err;
    a.nw = nullptr;
  }
  if (rows) return mm_rows(a, zeros, tile - Q4_ROWS_AT, st);
  return gemm_q4(a, zeros, tile, (float*)ws, ks, st, true);
}

}  // extern "C"
