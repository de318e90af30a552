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

// 64 features x 64 rows per workgroup, fragments straight from memory
template <bool SILU>
__global__ __launch_bounds__(256) void gemm_a8_kernel(const int8_t* __restrict__ c, long ldc,
                                                      const int8_t* __restrict__ wp, A8Out out, int M, int N, int K) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int nt = (N + 15) >> 4, tile = min((int)blockIdx.x * 4 + wv, nt - 1), m0 = blockIdx.y * 64;
  const int8_t* w = wp + (long)tile * 16 * K + 16 * lane;
  const int8_t* x[4];
  i32x4 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = c + (long)min(m0 + 16 * i + (lane & 15), M - 1) * ldc + 16 * (lane >> 4);
    acc[i] = (i32x4){0, 0, 0, 0};
  }
  for (int k = 0; k < K; k += 64) {
    const i32x4 a = *(const i32x4*)(w + 16L * k);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, *(const i32x4*)(x[i] + k), acc[i], 0, 0, 0);
  }
  const int n0 = ((int)blockIdx.x * 4 + wv) * 16 + 4 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + 16 * i + (lane & 15);
    if (m >= M) continue;
    const float sm = out.sx[m];
    float z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = (float)acc[i][j] * (sm * (float)out.s[min(n0 + j, N - 1)]);
    if constexpr (SILU) {
#pragma unroll
      for (int j = 0; j < 4; j += 2)
        if (n0 + j < N) out.y[m * out.ldy + (n0 + j) / 2] = (f16)(z[j] / (1.f + __expf(-z[j])) * z[j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < N) out.y[m * out.ldy + n0 + j] = (f16)(out.res ? z[j] + (float)out.res[m * out.ldr + n0 + j] : z[j]);
    }
  }
}

template <bool SILU>
static int launch_a8(const void* c, long ldc, const void* wp, const A8Out& out, int M, int N, int K, hipStream_t st) {
  const int mb = (M + 63) / 64;
  if (mb > 65535) return ECD_ENOTSUP;
  hipLaunchKernelGGL(gemm_a8_kernel<SILU>, dim3((N + 63) / 64, mb), dim3(256), 0, st, (const int8_t*)c, ldc,
                     (const int8_t*)wp, out, M, N, K);
  return ecd_launch_status();
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool a8_ok(const void* c, long ldc, const float* sx, const void* wp, const void* s, const void* y, int M, int N,
                  int K) {
  return c && sx && wp && s && y && M > 0 && N > 0 && K > 0 && K % 64 == 0 && K <= 1 << 17 && ldc >= K &&
         ldc % 128 == 0 && aligned16(c) && aligned16(wp);
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

int ecd_gemm_a8_silu(const void* c, long ldc, const float* sx, const void* wp, const void* s, void* mm, long ldm,
                     int M, int F, int K, void* stream) {
  if (F <= 0 || F > 1 << 29 || !a8_ok(c, ldc, sx, wp, s, mm, M, 2 * F, K) || ldm < F) return ECD_EINVAL;
  return launch_a8<true>(c, ldc, wp, A8Out{sx, (const f16*)s, nullptr, 0, (f16*)mm, ldm}, M, 2 * F, K,
                         (hipStream_t)stream);
}

}  // extern "C"
