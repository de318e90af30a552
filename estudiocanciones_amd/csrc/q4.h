// 4-bit weights in groups: the packed layout and what its kernels share (gfx950).
//
// A weight is w[n, k] = s[n, g] (u[n, k] - z[n, g]): u a code of 4 bits, g = k / G the group of G = 32, 64 or 128
// consecutive k, s an fp16 scale and z a zero point of 4 bits (8 everywhere without zero points).
//
// Packed codes: 32 rows x 64 k as 1 KB, blocks of a 32-row tile contiguous in k.  The 16 bytes at 16 l are row l & 31's; with
// h = l >> 5, their dword 2 S + H holds octet 4 H + 2 h + S (k = 8 (4 H + 2 h + S) .. + 7).  So a lane of v_mfma_f32_32x32x16_f16
// (row l & 31) takes its operands of four k-steps as 16 bytes, and so does one of v_mfma_f32_16x16x32_f16 (row l & 15): half the
// octets of a chunk, the upper 32 lanes those of the next chunk.  An octet lies in a dword as pairs (k, k + 1) 16 bits apart,
// pair p at bits 4 p and 16 + 4 p, which is how two halves of a register come out of one AND.
// Scales: for each 32-row tile [K / G rounded up][32] fp16, or with zero points pairs (s, 1024 + z) of fp16.  No scale is packed
// as 0, since products take quotients of them: a group whose scale is 0, and the rows behind the last, get the scale 1 and codes that are
// their zero point.
#pragma once
#include "common.h"

namespace ecd {

inline int q4_tiles(int N) { return (N + 31) / 32; }

// The 8 codes of a dword as exact halves u - z.  A code under the exponent of 1024 is the half 1024 + u; one 4 bits
// higher is 1024 + 16 u, whose sixteenth is 64 + u.  Differences of such halves are exact.
//   c0 = -(1024 + z) twice, c1 = -(64 + z) twice
__device__ __forceinline__ f16x8 q4_halves(uint32_t v, f16x2 c0, f16x2 c1) {
  // (constants that the compiler does not see through: it makes v_and_or_b32 of them, with literals two instructions)
  uint32_t lo = 0x000F000Fu, hi = 0x00F000F0u, one = 0x64006400u;
  asm("" : "+s"(lo), "+s"(hi), "+v"(one));
  const uint32_t w = v >> 8;
  const f16x2 sixteenth = {(f16)0.0625f, (f16)0.0625f};
  const f16x2 a = __builtin_bit_cast(f16x2, (v & lo) | one) + c0;
  const f16x2 b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (v & hi) | one), sixteenth, c1);
  const f16x2 c = __builtin_bit_cast(f16x2, (w & lo) | one) + c0;
  const f16x2 d = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & hi) | one), sixteenth, c1);
  return (f16x8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// A buffer of 2 GiB from a uniform base; lanes whose offset is Q4_NONE read zeros.
constexpr int Q4_NONE = (int)0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t q4_buffer(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, Q4_NONE, 0x00020000);
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
  int silu;  // pairs of rows (a, b) of the packed matrix give silu(a) b
  int two;   // 1: rows of x are two fp16 parts, 64 of the first, 64 of the second, and so on (2 K in all); the tiles only
};

// The product by a tile (1 .. Q4_TILES) of gemm_q4.hip, K split ks ways (ws: ks M ceil8(N) floats where ks > 1); no norm.
// go false: only whether the sizes fit.  And the choice for given sizes: tile + 256 ks; the few-row
// kernel's forms of 16, 32 and 64 features count as tiles Q4_ROWS_AT + 1 ..,
// Q4_TWO more: with the rows' norm in two fp16 parts.
// Q4_ONLY_TILES: the tiles; Q4_PLAIN: the few-row kernel's forms too; Q4_NORM: for products with a norm (the forms in two parts, the
// tiles in one); Q4_NORM_SILU: in two parts.
enum Q4Among { Q4_ONLY_TILES, Q4_PLAIN, Q4_NORM, Q4_NORM_SILU };
constexpr int Q4_TILES = 6, Q4_ROWS_AT = 16, Q4_ROWS = 3, Q4_TWO = 32;
int gemm_q4(const Q4Args& a, bool zp, int tile, float* ws, int ks, hipStream_t st, bool go);
int gemm_q4_plan(int M, int N, int K, Q4Among among);

// silu(a) * b in fp32
// (the exponential and the reciprocal by their instructions, 1 ulp of fp32 each)
__device__ __forceinline__ float silu_mul(float a, float b) {
  return a * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * -1.44269504088896341f)) * b;
}

}  // namespace ecd
