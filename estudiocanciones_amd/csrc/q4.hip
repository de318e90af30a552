// 4-bit weights in groups: the quantiser, the packing, and products of few rows (gfx950).  Layout: q4.h.
//
// Quantiser: s = fp16(max |w| / 7) and u = 8 + rint(w / s) in [0, 15]; with zero points lo = min(0, min w),
// hi = max(0, max w), s = fp16((hi - lo) / 15), z = rint(-lo / s) in [0, 15] and u = z + rint(w / s) in [0, 15].  Codes are
// those of the scale as stored; ties go to the even integer.  A group with an infinity, a NaN, or a scale past fp16 gets
// the scale NaN.
//
// Product: y[m, n] = fp16(sum_g s[n, g] sum_{k in g} x[m, k] (u[n, k] - z[n, g]) (+ res[m, n])).  The codes go into
// v_mfma_f32_32x32x16_f16 as exact halves; a group's sum is scaled and added in fp32, the residual and SiLU(a) * b are in
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
__global__ __launch_bounds__(256) void pack_q4_codes_kernel(const uint32_t* __restrict__ q, int N, int K, int il,
                                                            uint32_t* __restrict__ codes, long dwords) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= dwords) return;
  const int nch = K >> 6, l = (int)(i >> 2) & 63, d = (int)i & 3;
  const long block = i >> 8, t = block / nch;
  const int c = (int)(block - t * nch);
  const int n = (int)t * 32 + (l & 31), o = 4 * (d >> 1) + 2 * (l >> 5) + (d & 1);
  uint32_t v = 0, out = 0;
  if (n < N) v = q[q4_source(n, N, il) * (K >> 3) + 8 * c + o];
#pragma unroll
  for (int e = 0; e < 8; ++e) out |= (v >> (4 * e) & 15u) << (4 * (e >> 1) + 16 * (e & 1));
  codes[i] = out;
}

// one thread per scale
__global__ __launch_bounds__(256) void pack_q4_scales_kernel(const f16* __restrict__ s, const uint8_t* __restrict__ z, int N,
                                                             int ng, int il, f16* __restrict__ scales, long n32) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n32 * ng) return;
  const long g = i / n32;
  const int n = (int)(i - g * n32);
  f16 sv = (f16)0.f;
  int zv = 8;
  if (n < N) {
    const long from = q4_source(n, N, il) * ng + g;
    sv = s[from];
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
// A workgroup of KW waves computes 32 features of up to 32 rows; the waves share out the 64-wide chunks of K.
// MR: quarters of the 32 rows that are in use (rows 8 q .. 8 q + 7 are registers 4 q .. 4 q + 3 of a lane).
//
// The norm: x' = x 2^e with 2^e the power of two at 1 / rms (exact), times nw with one rounding to fp16 as the operand; what is
// left of 1 / rms, a factor in [1, 2), goes to the sum in fp32.
template <int KW, int MR, bool ZP, bool SILU>
__global__ __launch_bounds__(64 * KW) void mm_q4_rows_kernel(const Q4Args a) {
  const int lane = threadIdx.x & 63, f = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nch = a.K >> 6, m0 = blockIdx.y * 32, n0 = blockIdx.x * 32;
  const long n32 = (long)gridDim.x * 32;
  const bool row = m0 + f < a.M;
  const f16* xp = a.x + (long)(row ? m0 + f : 0) * a.ldx + 16 * h;
  __shared__ float part[KW][MR * 8][33];
  __shared__ float rs[KW][32];
  __shared__ float rfac[32];
  const f16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
  f16 p2 = (f16)1.f;
  if (a.nw) {
    float ss = 0.f;
    if (row)
      for (int c = wv; c < nch; c += KW)
#pragma unroll
        for (int o = 0; o < 4; ++o) {
          const f16x8 v = *(const f16x8*)(xp + 64L * c + 32 * (o >> 1) + 8 * (o & 1));
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += (float)v[j] * (float)v[j];
        }
    ss += __shfl_xor(ss, 32, 64);
    if (h == 0) rs[wv][f] = ss;
    __syncthreads();
    ss = 0.f;
    for (int w = 0; w < KW; ++w) ss += rs[w][f];
    const float inv = 1.0f / sqrtf(ss / (float)a.K + a.eps);
    const int e = min(max((int)(__builtin_bit_cast(uint32_t, inv) >> 23) - 127, -14), 15);
    p2 = __builtin_bit_cast(f16, (uint16_t)((e + 15) << 10));
    if (threadIdx.x < 32) rfac[f] = inv * __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
  } else if (threadIdx.x < 32) {
    rfac[f] = 1.f;
  }

  const uint8_t* cp = a.codes + (long)blockIdx.x * nch * 1024 + 16 * lane;
  f32x4 tot[MR];
#pragma unroll
  for (int q = 0; q < MR; ++q) tot[q] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int c = wv; c < nch; c += KW) {
    const u32x4 code = *(const u32x4*)(cp + 1024L * c);
#pragma unroll
    for (int H = 0; H < 2; ++H) {
      const long at = (long)((64 * c + 32 * H) >> a.lg) * n32 + n0 + f;
      f16 s;
      f16x2 c0 = {(f16)-1032.f, (f16)-1032.f}, c1 = {(f16)-72.f, (f16)-72.f};
      if constexpr (ZP) {
        const f16x2 sz = *(const f16x2*)(a.scales + 2 * at);
        s = sz.x;
        c0 = (f16x2){-sz.y, -sz.y};
        c1 = c0 + (f16x2){(f16)960.f, (f16)960.f};
      } else {
        s = a.scales[at];
      }
      f32x16 acc = (f32x16)(0.f);
#pragma unroll
      for (int S = 0; S < 2; ++S) {
        f16x8 xv = zero;
        if (row) xv = *(const f16x8*)(xp + 64L * c + 32 * H + 8 * S);
        if (a.nw) {
          const f16x8 nv = *(const f16x8*)(a.nw + 64L * c + 32 * H + 16 * h + 8 * S);
          xv = xv * p2 * nv;
        }
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(xv, q4_halves(code[2 * H + S], c0, c1), acc, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < MR; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) tot[q][r] += (float)s * acc[4 * q + r];
    }
  }
  // register 4 q + r of a lane: row 8 q + 4 h + r, feature f
#pragma unroll
  for (int q = 0; q < MR; ++q)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wv][8 * q + 4 * h + r][f] = tot[q][r];
  __syncthreads();
  constexpr int W = SILU ? 16 : 32;
  for (int i = threadIdx.x; i < MR * 8 * W; i += 64 * KW) {
    const int r = i / W, j = i % W, m = m0 + r;
    const int n = SILU ? n0 / 2 + j : n0 + j;
    if (m >= a.M || n >= (SILU ? a.N / 2 : a.N)) continue;
    float v = 0.f, u = 0.f;
    for (int w = 0; w < KW; ++w) {
      if constexpr (SILU) {
        v += part[w][r][2 * j];
        u += part[w][r][2 * j + 1];
      } else {
        v += part[w][r][j];
      }
    }
    v *= rfac[r];
    if constexpr (SILU) v = silu_mul(v, u * rfac[r]);
    if (a.res) v += (float)a.res[(long)m * a.ldr + n];
    a.y[(long)m * a.ldy + n] = (f16)v;
  }
}

template <int MR, bool ZP, bool SILU>
static int launch_rows(const Q4Args& a, hipStream_t st) {
  constexpr int KW = 8;
  hipLaunchKernelGGL((mm_q4_rows_kernel<KW, MR, ZP, SILU>), dim3(q4_tiles(a.N), (a.M + 31) / 32), dim3(64 * KW), 0, st, a);
  return ecd_launch_status();
}

template <bool ZP, bool SILU>
static int mm_rows(const Q4Args& a, hipStream_t st) {
  if (a.M <= 8) return launch_rows<1, ZP, SILU>(a, st);
  if (a.M <= 16) return launch_rows<2, ZP, SILU>(a, st);
  return launch_rows<4, ZP, SILU>(a, st);
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
  hipLaunchKernelGGL(pack_q4_codes_kernel, dim3((unsigned)((dwords + 255) / 256)), dim3(256), 0, st, (const uint32_t*)q, N, K,
                     interleave, (uint32_t*)codes, dwords);
  hipLaunchKernelGGL(pack_q4_scales_kernel, dim3((unsigned)((n32 * ng + 255) / 256)), dim3(256), 0, st, (const f16*)s,
                     (const uint8_t*)z, N, ng, interleave, (f16*)scales, n32);
  return ecd_launch_status();
}

int ecd_mm_q4(const void* x, long ldx, const void* nw, float eps, const void* codes, const void* scales, int zeros, int group,
              const void* res, long ldr, void* y, long ldy, int M, int N, int K, int silu, void* stream) {
  const int cols = silu ? N / 2 : N;
  if (!x || !codes || !scales || !y || M <= 0 || N <= 0 || K <= 0 || K % 64 || !group_ok(group) || ldx < K || ldx % 8 ||
      !al16(x) || (nw && !al16(nw)) || !al16(codes) || !al16(scales) || ldy < cols || (res && ldr < cols) ||
      (silu && (N % 2 || res)) || (nw && !(eps >= 0.f)))
    return ECD_EINVAL;
  if (q4_tiles(N) > 0x3FFFFFF || (M + 31) / 32 > 65535) return ECD_ENOTSUP;
  const Q4Args a{(const f16*)x, ldx, (const f16*)nw, eps, (const uint8_t*)codes, (const f16*)scales, log2_group(group),
                 (const f16*)res, ldr, (f16*)y, ldy, M, N, K};
  const hipStream_t st = (hipStream_t)stream;
  if (silu) return zeros ? mm_rows<true, true>(a, st) : mm_rows<false, true>(a, st);
  return zeros ? mm_rows<true, false>(a, st) : mm_rows<false, false>(a, st);
}

}  // extern "C"
