// 4-bit weights in groups: the packed layout and what its kernels share (gfx950).
//
// A weight is w[n, k] = s[n, g] (u[n, k] - z[n, g]): u a code of 4 bits, g = k / G the group of G = 32, 64 or 128
// consecutive k, s an fp16 scale and z a zero point of 4 bits (8 everywhere without zero points).
//
// Packed codes: 32 rows x 64 k as 1 KB, blocks of a 32-row tile contiguous in k.  Lane l of v_mfma_f32_32x32x16_f16
// takes row l & 31, so the 16 bytes at 16 l are that row's; with h = l >> 5, dword 2 H + S holds octet 4 H + 2 h + S
// (k = 8 (4 H + 2 h + S) .. + 7), the operand of k-step S of the 32 k of half H.  An octet lies in a dword as pairs
// (k, k + 1) 16 bits apart, pair p at bits 4 p and 16 + 4 p, which is how two halves of a register come out of one AND.
// Scales: [K / G rounded up][rows rounded up to 32] fp16, or with zero points pairs (s, 1024 + z) of fp16.  Rows behind the
// last have the scale 0.
#pragma once
#include "common.h"

namespace ecd {

inline int q4_tiles(int N) { return (N + 31) / 32; }

// The 8 codes of a dword as exact halves u - z.  A code under the exponent of 1024 is the half 1024 + u; one 4 bits
// higher is 1024 + 16 u, whose sixteenth is 64 + u.  Differences of such halves are exact.
//   c0 = -(1024 + z) twice, c1 = -(64 + z) twice
__device__ __forceinline__ f16x8 q4_halves(uint32_t v, f16x2 c0, f16x2 c1) {
  const uint32_t w = v >> 8;
  const f16x2 sixteenth = {(f16)0.0625f, (f16)0.0625f};
  const f16x2 a = __builtin_bit_cast(f16x2, (v & 0x000F000Fu) | 0x64006400u) + c0;
  const f16x2 b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (v & 0x00F000F0u) | 0x64006400u), sixteenth, c1);
  const f16x2 c = __builtin_bit_cast(f16x2, (w & 0x000F000Fu) | 0x64006400u) + c0;
  const f16x2 d = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & 0x00F000F0u) | 0x64006400u), sixteenth, c1);
  return (f16x8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// A product's operands.  nw: the weight of an RMS norm of the rows before the product, or NULL.
struct Q4Args {
  const f16* x;
  long ldx;
  const f16* nw;
  float eps;
  const uint8_t* codes;
  const f16* scales;
  int lg;  // log2 of the group
  const f16* res;
  long ldr;
  f16* y;
  long ldy;
  int M, N, K;
};

// silu(a) * b in fp32
__device__ __forceinline__ float silu_mul(float a, float b) { return a / (1.0f + expf(-a)) * b; }

}  // namespace ecd
