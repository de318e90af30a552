// Logits from a model's heads to those a sampler draws from (gfx950): guidance, penalties for tokens of a history, biases,
// masks of allowed tokens.
//
// Per row r and token v, in fp32, one rounding to fp16 at the end:
//   l = u + (c - u) cfg                        with guidance (c row r, u row N + r), else the row itself
//   if v occurs n > 0 times in the row's history:
//     l = l > 0 ? l / rep[r] : l rep[r];  l = l - (presence[r] + frequency[r] n)
//   l = l + bias[v]
//   l = -inf                                   where the row's mask does not allow v
// A finite l above fp16's largest number becomes that number: a softmax subtracts the largest value, and an infinity less itself is no
// token's to draw.  One below the lowest becomes -inf, which is never drawn.
// The history of a row are the last `window` (0: all) of its first length[r] tokens; tokens outside [0, V) count for nothing.
//
// A workgroup takes a segment of a row: its logits, biases and mask bits are loaded first; while they are in flight the row's
// history is counted for the segment with integer atomics in LDS (the order of their arrival cannot change a count), then
// each thread finishes its 8 tokens.  Nothing is written in between, so one launch is one pass over the data.  1 row of 8197 tokens and
// 64 of history 3.0 us (2.2 of it a launch), 32 rows of 100003 tokens with biases, masks and 4096 of history 9.4 (2.8 TB/s); histories of
// a song's frames cost a line of memory per token and segment.
#include "gemm_core.h"

namespace ecd {

typedef f32x4 f32x4u __attribute__((aligned(4)));

struct LogitsArgs {
  const f16* logits;
  long ld;
  float cfg;
  int guided;
  const int64_t* hist;
  long hrow, htok;
  int T;
  const int64_t* length;
  int window;
  const float *rep, *pres, *freq;
  int per_row;  // bit 0 / 1 / 2: rep / pres / freq has an element per row (else one for all)
  const float* bias;
  long ldb;
  const uint32_t* allowed;
  long lda;
  int A;
  const int32_t* state;
  f16* out;
  long ldo;
  int N, V, seg;
};

template <int TH>
__global__ __launch_bounds__(TH) void process_logits_kernel(const LogitsArgs a) {
  __shared__ __align__(16) uint32_t count[8 * TH];
  const int r = blockIdx.y, v0 = blockIdx.x * a.seg, v1 = min(v0 + a.seg, a.V);
  const f16* lc = a.logits + (long)r * a.ld;
  const f16* lu = a.logits + (long)(r + a.N) * a.ld;
  const float* bp = a.bias ? a.bias + (long)r * a.ldb : nullptr;
  // a state outside the masks allows nothing, -1 everything
  uint32_t keep = 0xFFu;
  const uint32_t* mask = nullptr;
  if (a.allowed) {
    const int s = a.state ? a.state[r] : a.A == 1 ? 0 : r;
    if (s >= a.A || s < -1)
      keep = 0u;
    else if (s >= 0)
      mask = a.allowed + (long)s * a.lda;
  }
  const int i = v0 + 8 * (int)threadIdx.x;
  const bool on = i < v1, full = i + 8 <= v1;
  f16x8 c = {0, 0, 0, 0, 0, 0, 0, 0}, u = c;
  float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (full) {
    c = *(const f16x8u*)(lc + i);
    if (a.guided) u = *(const f16x8u*)(lu + i);
    if (bp) {
      const f32x4 b0 = *(const f32x4u*)(bp + i), b1 = *(const f32x4u*)(bp + i + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        b[j] = b0[j];
        b[4 + j] = b1[j];
      }
    }
  } else if (on) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < v1) {
        c[j] = lc[i + j];
        if (a.guided) u[j] = lu[i + j];
        if (bp) b[j] = bp[i + j];
      }
  }
  if (mask && on) keep = mask[i >> 5] >> (i & 31);
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.hist) {
    const int64_t len = a.length ? a.length[r] : a.T;
    const int t1 = (int)(len < 0 ? 0 : len > a.T ? a.T : len);
    const int t0 = a.window > 0 && t1 > a.window ? t1 - a.window : 0;
    if (a.rep) rep = a.rep[a.per_row & 1 ? r : 0];
    if (a.pres) pres = a.pres[a.per_row & 2 ? r : 0];
    if (a.freq) freq = a.freq[a.per_row & 4 ? r : 0];
    u32x4* const mine = (u32x4*)(count + 8 * threadIdx.x);
    mine[0] = mine[1] = (u32x4){0u, 0u, 0u, 0u};
    __syncthreads();
    // HB loads of a thread in flight: tokens of a song's frames lie in lines of their own
    constexpr int HB = 4;
    const int64_t* hp = a.hist + (long)r * a.hrow;
    for (int t = t0 + (int)threadIdx.x; t < t1; t += HB * TH) {
      int64_t v[HB];
#pragma unroll
      for (int k = 0; k < HB; ++k) v[k] = hp[(long)min(t + k * TH, t1 - 1) * a.htok];
#pragma unroll
      for (int k = 0; k < HB; ++k)
        if (t + k * TH < t1 && v[k] >= v0 && v[k] < v1) atomicAdd(&count[(int)(v[k] - v0)], 1u);
    }
    __syncthreads();
  }
  if (!on) return;
  uint32_t n[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
  if (a.hist) {
    const u32x4 n0 = *(const u32x4*)(count + 8 * threadIdx.x), n1 = *(const u32x4*)(count + 8 * threadIdx.x + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      n[j] = n0[j];
      n[4 + j] = n1[j];
    }
  }
  float l[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    l[j] = (float)c[j];
    if (a.guided) {
      const float w = (float)u[j];
      l[j] = w + (l[j] - w) * a.cfg;
    }
    if (n[j]) {
      l[j] = l[j] > 0.f ? l[j] / rep : l[j] * rep;
      l[j] -= pres + freq * (float)n[j];
    }
    l[j] += b[j];
  }
  // above the range: rare, so one comparison for the eight (a vector instruction of a long row costs 15 ns)
  float top = l[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) top = fmaxf(top, l[j]);
  if (__builtin_expect(top > 65504.f, 0)) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (l[j] < INFINITY) l[j] = fminf(l[j], 65504.f);
  }
  f16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = keep >> j & 1u ? (f16)l[j] : (f16)-INFINITY;
  f16* op = a.out + (long)r * a.ldo + i;
  if (full)
    *(f16x8u*)op = o;
  else
    store_tail(op, nullptr, o, v1 - i);
}

template <int TH>
static int launch_logits(LogitsArgs a, hipStream_t st) {
  constexpr int SEG = 8 * TH;
  const int parts = (a.V + SEG - 1) / SEG;
  a.seg = ((a.V + parts - 1) / parts + 7) / 8 * 8;
  hipLaunchKernelGGL((process_logits_kernel<TH>), dim3((a.V + a.seg - 1) / a.seg, a.N), dim3(TH), 0, st, a);
  return ecd_launch_status();
}

}  // namespace ecd

using namespace ecd;

extern "C" int ecd_process_logits(const void* logits, long ld, int guided, float cfg, const int64_t* hist, long hrow, long htok,
                                  int T, const int64_t* length, int window, const float* rep, const float* pres,
                                  const float* freq, int per_row, const float* bias, long ldb, const uint32_t* allowed, long lda,
                                  int A, const int32_t* state, void* out, long ldo, int N, int V, void* stream) {
  if (!logits || !out || N <= 0 || V <= 0 || ld < V || ldo < V || T < 0 || window < 0 || (hist && (hrow < 0 || htok < 0)) ||
      ((rep || pres || freq) && !hist) || (bias && ldb != 0 && ldb < V) ||
      (allowed && (A <= 0 || lda < (V + 31L) / 32 || (!state && A != 1 && A != N))))
    return ECD_EINVAL;
  if (N > 65535 || V > 0x7FFFFFFF - 8192 || T > 1 << 30) return ECD_ENOTSUP;
  const LogitsArgs a{(const f16*)logits, ld, cfg, guided, hist, hrow, htok, T, length, window, rep, pres, freq, per_row, bias, ldb,
                     allowed, lda, A, state, (f16*)out, ldo, N, V, 0};
  const hipStream_t st = (hipStream_t)stream;
  // A workgroup's history costs a line of memory per token, or a 16th of one where tokens are neighbours.  Segments of 2048 tokens
  // by 256 threads give short histories the most parallelism; for long ones, and for many rows of them, segments of 8192
  // by 1024 threads read them fewer times (us: 4 rows of 3000 frames 8.0 and 5.7, 128 of 750 12.0 and 8.8, 32 rows of 4096
  // neighbours over 100003 tokens 10.7 and 9.4; 1 row of 750 frames 3.7 and 4.4, 8 of 2000 neighbours over 40000 3.9 and 5.1).
  const long lines = hist ? (window && window < T ? window : T) / (htok == 1 ? 16 : 1) : 0;
  return lines > 1500 || lines * N * ((V + 2047) / 2048) > 300000 ? launch_logits<1024>(a, st) : launch_logits<256>(a, st);
}
