// Decode attention over pages of a KV cache, the prefix that a group of rows shares read once for all of them (gfx950).
//
// Row r (sequence r / S) attends slots [0, pos[r]] of its sequence: o = softmax(q k^T scale) v per query head, G = Hq / Hk
// of them on each kv head.  The rows of a group hold the same slots [0, prefix).  Softmax splits over slots: with
//   m = max s,  l = sum exp(s - m),  a = sum exp(s - m) v   over any part of the slots,
// the whole is  o = sum_parts exp(m_part - M) a_part / sum_parts exp(m_part - M) l_part,  M = max m_part.
// So a workgroup takes one part: an item of the plan (slots [lo, hi) of a group's prefix, for up to 16 CT columns, a
// column being one query head of one row), or a share of one row's own slots.  A second kernel joins the parts.
//
// A row takes the shared parts only if it attends the whole prefix; else its own part covers [0, pos].  The shared slots
// are read through the first such row's pages.
//
// Both products run on v_mfma_f32_16x16x32_f16 with the slots of a tile as its rows (scores) and its k (output): a column's
// probabilities then lie in the lane that needs them, and a tile goes from memory to registers to the products without LDS.
// Scores, maxima, sums and outputs are fp32.  A weight is exp(s - m) 2^14 and goes into the second product as the sum of two
// fp16 values, the upper one rounded towards zero and the lower one what that leaves: 2^-20 of the weight, or 2^-38 of the
// largest, where one fp16 value would lose 2^-12 of each and every weight below 2^-25 of the largest (of thousands of
// slots beside a few large ones they are a part of the result that counts).  The matrix pipes wait for the tiles, so the second
// product's other half costs little: 2 x 32 rows on prompts of 7000 slots 42.1 us against 41.4 with its join, 2 x 16 on 4096
// 29.2 against 28.9, short rows the same.
// Bound by the reads of K and V: of 24 query heads on 8 kv heads of 128, 2 x 32 rows on prompts of 7000 slots (126 MB, each
// slot read from memory once) take 40.1 us and 4.8 us for the join, 2 x 16 on 4096 (98 MB) 25.0 and 4.1: about 5.5 us until the
// first tile is there, then 2 us for each of 14 tiles of a wave (8 waves a CU), 3 us to add the waves up.  A few short
// rows are bound by those first and last steps: 8 rows of 750 slots 7.6 us and 3.6 for the join.
#include "common.h"

namespace ecd {

constexpr int PQ_T = 32;  // slots of a wave's tile

// what does not change over a call
struct PagedArgs {
  const f16* q;      // row r at q + r ldq
  const f16* kp;     // [NP, Hk, P, HD]
  const f16* vp;
  const int* table;  // row of sequence b at table + b ldt, MP entries
  const int64_t* pos;
  f16* o;            // [R, Hq, HD]
  float* pm;         // [R Hq, parts]: maximum and sum of each part, then its unnormalised output
  float* pl;
  float* pa;         // [R Hq, parts, HD]
  const int* items;  // {first row, rows, lo, hi, part, kv head} of each shared part
  const int* rows;   // {shared slots, shared parts} of each row
  long ldq, ldt;
  int R, MP, NP, S, Hq, Hk, G, PS, nitems, nown, parts;  // PS: log2 of the page size
  float c2;          // scale log2(e)
};

__device__ __forceinline__ float max_groups(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// One tile of 32 slots in registers.  Lane l: K of slots 16 j + (l & 15), dims 8 (l >> 4) + 32 i; V of slots
// 16 j + 4 (l >> 4) + e, dims VW (l & 15) + 128 x.
template <int HD>
struct PTile {
  static constexpr int KC = HD / 32, VW = HD >= 128 ? 8 : HD / 16, ND = (HD + 127) / 128;
  typedef f16 vec __attribute__((ext_vector_type(VW)));
  f16x8 k[2][KC];
  vec v[2][4][ND];
};

// Where tiles lie: lane i holds the pool row (page Hk + kh) P + slot of the halves of the tile at t0 + step i.  Slots from hi
// on repeat a half before it (masked later); a number that is no page reads page 0 or the last one.
struct Places {
  uint32_t r0, r1;
};
__device__ __forceinline__ Places places(const PagedArgs& a, const int* tab, int kh, int t0, int step, int hi, int lane) {
  const int last = (hi - 1) & ~15, mask = (1 << a.PS) - 1;  // a half tile lies in one page
  const int h0 = min(t0 + lane * step, last), h1 = min(t0 + lane * step + 16, last);
  const uint32_t p0 = min(max(tab[h0 >> a.PS], 0), a.NP - 1), p1 = min(max(tab[h1 >> a.PS], 0), a.NP - 1);
  return {((p0 * a.Hk + kh) << a.PS) + (h0 & mask), ((p1 * a.Hk + kh) << a.PS) + (h1 & mask)};
}

template <int HD>
__device__ __forceinline__ void load_k(PTile<HD>& t, const PagedArgs& a, const Places& p, int i, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const f16* k = a.kp + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(j ? p.r1 : p.r0), i) * HD;
#pragma unroll
    for (int x = 0; x < PTile<HD>::KC; ++x) t.k[j][x] = *(const f16x8*)(k + (uint32_t)((lane & 15) * HD + 8 * (lane >> 4) + 32 * x));
  }
}
template <int HD>
__device__ __forceinline__ void load_v(PTile<HD>& t, const PagedArgs& a, const Places& p, int i, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const f16* v = a.vp + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(j ? p.r1 : p.r0), i) * HD;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int x = 0; x < PTile<HD>::ND; ++x)
        t.v[j][e][x] = *(const typename PTile<HD>::vec*)(v + (uint32_t)((4 * (lane >> 4) + e) * HD + PTile<HD>::VW * (lane & 15) + 128 * x));
  }
}

// The running softmax of CT tiles of 16 columns (lane l: column l & 15 of each).  acc[c][x][b]: row i of lane l is dim
// 128 x + VW (4 (l >> 4) + i) + b.  l: this lane's share of the sum.
template <int HD, int CT>
struct PState {
  static constexpr int VW = PTile<HD>::VW, ND = PTile<HD>::ND;
  f16x8 q[CT][HD / 32];
  f32x4 acc[CT][ND][VW];
  float m[CT], l[CT];
};

// w0 and w1 (not negative) as sums of two fp16 values each.  The lower one is never 0 beside an upper one that is not, since
// a value of infinity times 0 would be no number.
__device__ __forceinline__ void two_halves(float w0, float w1, f16x2& hi, f16x2& lo) {
  const f16 least = __builtin_bit_cast(f16, (uint16_t)1);
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(w0, w1));
  lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(w0 - (float)hi.x, w1 - (float)hi.y));
  lo = __builtin_elementwise_max(lo, __builtin_elementwise_min(hi, (f16x2){least, least}));
}
constexpr float W_LOG2 = 14.f;  // weights are scaled by 2^14

// Slots outside [lo, hi) of the tile at t0 do not count, whatever they hold.  `after_scores` runs once K is used.
template <int HD, int CT, typename F>
__device__ __forceinline__ void tile_attend(PState<HD, CT>& s, PTile<HD>& t, float c2, int t0, int lo, int hi, int lane, F&& after_scores) {
  using T = PTile<HD>;
  const int grp = lane >> 4;
  const bool edge = t0 < lo || t0 + PQ_T > hi;  // uniform
  f32x4 sc[CT][2];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sc[c][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < T::KC; ++i) sc[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[j][i], s.q[c][i], sc[c][j], 0, 0, 0);
    }
  after_scores();
  f16x8 p[CT], pr[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    if (edge) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = t0 + 16 * j + 4 * grp + e;
          if (k < lo || k >= hi) sc[c][j][e] = -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[c][j][e]);
    const float mn = fmaxf(s.m[c], max_groups(mx));
    // the difference first: m c2 rounded by itself would be a factor of its own in each tile's weights where scores are large
    const float mb = mn == -INFINITY ? 0.f : mn;
    float ps = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[c][j][e] - mb, c2, W_LOG2));
        const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[c][j][e + 1] - mb, c2, W_LOG2));
        ps += w0 + w1;
        f16x2 h, r;
        two_halves(w0, w1, h, r);
        p[c][4 * j + e] = h.x, p[c][4 * j + e + 1] = h.y;
        pr[c][4 * j + e] = r.x, pr[c][4 * j + e + 1] = r.y;
      }
    if (__any(mn != s.m[c])) {
      const float alpha = __builtin_amdgcn_exp2f((s.m[c] - mb) * c2);
      s.l[c] *= alpha;
#pragma unroll
      for (int x = 0; x < T::ND; ++x)
#pragma unroll
        for (int b = 0; b < T::VW; ++b) s.acc[c][x][b] = s.acc[c][x][b] * alpha;
    }
    s.l[c] += ps;
    s.m[c] = mn;
  }
  if (edge) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = t0 + 16 * j + 4 * grp + e;
        if (k < lo || k >= hi)
#pragma unroll
          for (int x = 0; x < T::ND; ++x) t.v[j][e][x] = (typename T::vec)((f16)0);
      }
  }
#pragma unroll
  for (int x = 0; x < T::ND; ++x) {
    const typename T::vec v0 = t.v[0][0][x], v1 = t.v[0][1][x], v2 = t.v[0][2][x], v3 = t.v[0][3][x];
    const typename T::vec v4 = t.v[1][0][x], v5 = t.v[1][1][x], v6 = t.v[1][2][x], v7 = t.v[1][3][x];
#pragma unroll
    for (int b = 0; b < T::VW; ++b) {
      const f16x8 va = {v0[b], v1[b], v2[b], v3[b], v4[b], v5[b], v6[b], v7[b]};
#pragma unroll
      for (int c = 0; c < CT; ++c) s.acc[c][x][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[c], s.acc[c][x][b], 0, 0, 0);
#pragma unroll
      for (int c = 0; c < CT; ++c) s.acc[c][x][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pr[c], s.acc[c][x][b], 0, 0, 0);
    }
  }
}

// nothing attended yet; q of columns 16 first .. (query head n % G of row row0 + n / G; columns from cols on repeat one)
template <int HD, int CT>
__device__ __forceinline__ void begin(PState<HD, CT>& s, const PagedArgs& a, int row0, int cols, int first, int kh, int lane) {
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int n = 16 * (first + c) + (lane & 15);
    const int cc = n < cols ? n : 0;
    const f16* q = a.q + (long)(row0 + cc / a.G) * a.ldq + (long)(kh * a.G + cc % a.G) * HD + 8 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) s.q[c][i] = *(const f16x8*)(q + 32 * i);
    s.m[c] = -INFINITY;
    s.l[c] = 0.f;
#pragma unroll
    for (int x = 0; x < PTile<HD>::ND; ++x)
#pragma unroll
      for (int b = 0; b < PTile<HD>::VW; ++b) s.acc[c][x][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
}

// One part on one workgroup whose waves share out the slots: `cols` columns, slots [lo, hi) through `tab`.
// `live`: bit i says whether row row0 + i takes this part.  Its result goes to place `part` of the rows of `mine`, or with
// `whole` normalised to o.
template <int HD, int CT, int W>
__device__ __forceinline__ void attend(const PagedArgs& a, float* lds, int row0, int cols, int kh, const int* tab, int lo,
                                       int hi, int part, bool whole, uint64_t mine, uint64_t live) {
  constexpr int ST = HD + 4;  // floats of a column in LDS
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = lane >> 4, col = lane & 15;
  PState<HD, CT> s;
  begin(s, a, row0, cols, 0, kh, lane);
  // K of the next tile is asked for once this one's scores are formed, V once this one's is used: one tile is always in
  // flight, in the registers of the last one.  (Two tiles ahead measured no faster: what the L2s do not hold comes at 4 to
  // 6 TB/s, about 20 GB/s for each CU, whatever is in flight.)
  PTile<HD> t;
  constexpr int STEP = W * PQ_T;
  const int first = (lo & ~(PQ_T - 1)) + wv * PQ_T;
  const int n = hi > first ? (hi - first + STEP - 1) / STEP : 0;
  Places at;
  if (n > 0) {
    at = places(a, tab, kh, first, STEP, hi, lane);
    load_k<HD>(t, a, at, 0, lane);
    load_v<HD>(t, a, at, 0, lane);
  }
  for (int i = 0; i < n; ++i) {
    const int next = i + 1;
    const bool more = next < n;
    if (more && (next & 63) == 0) at = places(a, tab, kh, first + next * STEP, STEP, hi, lane);
    tile_attend<HD, CT>(s, t, a.c2, first + i * STEP, lo, hi, lane, [&]() {
      asm volatile("" ::: "memory");
      if (more) load_k<HD>(t, a, at, next & 63, lane);
      asm volatile("" ::: "memory");
    });
    asm volatile("" ::: "memory");
    if (more) load_v<HD>(t, a, at, next & 63, lane);
    asm volatile("" ::: "memory");
  }

  // the waves' states to one: maxima and sums first, then the outputs on the common maximum
  float* sm = lds;                    // [W][16 CT]
  float* sl = lds + W * 16 * CT;
  float* sa = lds + 2 * W * 16 * CT;  // [W][16 CT][ST]
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const float l = sum_groups(s.l[c]);
    if (grp == 0) {
      sm[wv * 16 * CT + 16 * c + col] = l == l ? s.m[c] : l;  // (a sum that is no number is not an empty part)
      sl[wv * 16 * CT + 16 * c + col] = l;
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w * 16 * CT + 16 * c + col]);
    const float m = sm[wv * 16 * CT + 16 * c + col];
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - M) * a.c2);
    float* d = sa + (wv * 16 * CT + 16 * c + col) * ST;
#pragma unroll
    for (int x = 0; x < PTile<HD>::ND; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int b = 0; b < PTile<HD>::VW; b += 4)
          *(f32x4*)(d + 128 * x + PTile<HD>::VW * (4 * grp + i) + b) =
              (f32x4){s.acc[c][x][b][i] * f, s.acc[c][x][b + 1][i] * f, s.acc[c][x][b + 2][i] * f, s.acc[c][x][b + 3][i] * f};
  }
  __syncthreads();
  for (int i = threadIdx.x; i < cols * (HD / 4); i += 64 * W) {
    const int n = i / (HD / 4), d = 4 * (i - n * (HD / 4));
    const int row = row0 + n / a.G;
    const long head = (long)row * a.Hq + kh * a.G + n % a.G;
    float M = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w * 16 * CT + n]);
    f32x4 v = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float m = sm[w * 16 * CT + n];
      l += m == -INFINITY ? 0.f : sl[w * 16 * CT + n] * __builtin_amdgcn_exp2f((m - M) * a.c2);
      v = v + *(const f32x4*)(sa + (w * 16 * CT + n) * ST + d);
    }
    if (whole) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (a sum that is no number stays none)
      *(f16x4*)(a.o + head * HD + d) = (f16x4){(f16)(v[0] * inv), (f16)(v[1] * inv), (f16)(v[2] * inv), (f16)(v[3] * inv)};
    } else if (mine >> (row - row0) & 1) {
      const long pi = head * a.parts + part;
      M = !(live >> (row - row0) & 1) ? -INFINITY : l == l ? M : l;
      if (d == 0) {
        a.pm[pi] = M;
        a.pl[pi] = l;
      }
      *(f32x4*)(a.pa + pi * HD + d) = v;
    }
  }
}

template <int HD, int CT, int W>
constexpr int attend_lds() {
  return W * 16 * CT * (2 + HD + 4);
}

// slots that row r attends: all that the table has where its position lies behind them
__device__ __forceinline__ int attended(const PagedArgs& a, int r) {
  const long p = a.pos[r];
  return p < 0 ? 0 : (int)min(p, ((long)a.MP << a.PS) - 1) + 1;
}

template <int HD, int CT, int W>
__global__ __launch_bounds__(64 * W, HD > 128 ? 1 : 2) void paged_attn_kernel(PagedArgs a) {
  __shared__ __align__(16) float lds[attend_lds<HD, CT, W>()];
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x < a.nitems) {
    const int* it = a.items + 6 * blockIdx.x;
    const int row0 = it[0], n = it[1], lo = max(it[2], 0), hi = min(it[3], a.MP << a.PS), kh = it[5];
    if (row0 < 0 || n < 1 || n > 16 * CT / a.G || row0 > a.R - n || kh < 0 || kh >= a.Hk || it[4] < 0 || it[4] >= a.parts - a.nown) return;
    // the first row that attends the whole prefix leads: its pages hold every shared slot.  The places of a row behind its
    // shared parts are those of its own slots: a part number that is not below the row's count is not for it.
    const int r = row0 + min(lane, n - 1);
    const uint64_t mine = __ballot(lane < n && it[4] < a.rows[2 * r + 1]);
    const uint64_t live = mine & __ballot(lane < n && attended(a, r) >= a.rows[2 * r]);
    const int* tab = a.table + (long)((row0 + (live ? __builtin_ctzll(live) : 0)) / a.S) * a.ldt;
    attend<HD, CT, W>(a, lds, row0, n * a.G, kh, tab, lo, live ? hi : lo, it[4], false, mine, live);
    return;
  }
  const int x = blockIdx.x - a.nitems, u = x / a.Hk, kh = x - u * a.Hk, r = u / a.nown, k = u - r * a.nown;
  const int end = attended(a, r), shared = a.rows[2 * r], np = a.rows[2 * r + 1];
  if (np < 0 || np + a.nown > a.parts) return;
  const int from = end >= shared ? shared : 0;
  const int per = (max(W * PQ_T, (end - from + a.nown - 1) / a.nown) + PQ_T - 1) & ~(PQ_T - 1);
  const int lo = min(from + k * per, end), hi = min(lo + per, end);
  attend<HD, 1, W>(a, lds, r, a.G, kh, a.table + (long)(r / a.S) * a.ldt, lo, hi, np + k, np + a.nown == 1, ~0ull, ~0ull);
}

// The parts of a head to one output: one thread per four dims, JB parts at a time, all their loads at once (one after the other
// cost a memory latency each), in the order of the parts, so the result does not depend on timing.  Bound by latency: 3.7 us
// for 8 rows of 4 parts, 4.7 us for 64 rows of 5.
constexpr int JB = 8;
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int HD, int heads) {
  const int i = blockIdx.x * 256 + threadIdx.x, per = HD / 4;
  const int head = i / per, d = 4 * (i - head * per);
  if (head >= heads) return;
  const int r = head / a.Hq, np = a.rows[2 * r + 1], n = np + a.nown;
  if (np < 0 || n > a.parts || n == 1) return;
  const float *pm = a.pm + (long)head * a.parts, *pl = a.pl + (long)head * a.parts, *pa = a.pa + (long)head * a.parts * HD + d;
  float M = -INFINITY, l = 0.f;
  f32x4 v = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < n; k0 += JB) {
    float m[JB], s[JB];
    f32x4 x[JB];
#pragma unroll
    for (int k = 0; k < JB; ++k) {
      const int kk = min(k0 + k, n - 1);
      m[k] = k0 + k < n ? pm[kk] : -INFINITY;
      s[k] = pl[kk];
      x[k] = *(const f32x4*)(pa + (long)kk * HD);
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < JB; ++k) mn = fmaxf(mn, m[k]);
    if (mn != M) {
      const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - mn) * a.c2);
      l *= f;
      v = v * f;
      M = mn;
    }
#pragma unroll
    for (int k = 0; k < JB; ++k)
      if (m[k] != -INFINITY) {  // (an empty part's output is not looked at)
        const float f = __builtin_amdgcn_exp2f((m[k] - M) * a.c2);
        l += f * s[k];
        v = v + x[k] * f;
      }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  *(f16x4*)(a.o + (long)head * HD + d) = (f16x4){(f16)(v[0] * inv), (f16)(v[1] * inv), (f16)(v[2] * inv), (f16)(v[3] * inv)};
}

template <int HD, int CT, int W>
static int launch_paged(const PagedArgs& a, int R, hipStream_t st) {
  hipLaunchKernelGGL((paged_attn_kernel<HD, CT, W>), dim3(a.nitems + R * a.nown * a.Hk), dim3(64 * W), 0, st, a);
  return ecd_launch_status();
}

}  // namespace ecd

using namespace ecd;

static constexpr float LOG2E = 1.44269504088896341f;

extern "C" int ecd_paged_attn(const void* q, long ldq, const void* kp, const void* vp, const int32_t* table, long ldt,
                              const int64_t* pos, void* o, float* ws, const int32_t* items, const int32_t* rows,
                              int nitems, int nown, int parts, int ctiles, int waves, int R, int S, int MP, int NP, int Hq, int Hk,
                              int P, int HD, float scale, void* stream) {
  if (!q || !kp || !vp || !table || !pos || !o || !rows || (nitems > 0 && (!items || parts <= nown)) || nitems < 0 || nown < 1 ||
      parts < nown || (parts > 1 && !ws) || R <= 0 || S <= 0 || MP <= 0 || NP <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk ||
      Hq / Hk > 16 || P < 16 || (P & (P - 1)) || ldt < MP || ldq < (long)Hq * HD || (ldq % 8) ||
      ((uintptr_t)q & 15) || ((uintptr_t)kp & 15) || ((uintptr_t)vp & 15) || ((uintptr_t)o & 7) || ((uintptr_t)ws & 15) ||
      !(scale > 0.f && scale * LOG2E < INFINITY) || (long)MP * P > 1 << 30 || (long)R * nown * Hk + nitems > 0x7FFFFFL || (long)R * Hq > 0x7FFFFFFFL / 64 ||
      (long)NP * P > 0xFFFFFFFFL || (long)NP * P * Hk > 0xFFFFFFFFL)
    return ECD_EINVAL;
  if ((HD != 64 && HD != 128 && HD != 256) || parts > 512) return ECD_ENOTSUP;
  const long heads = (long)R * Hq, n2 = (heads * parts + 3) & ~3l;
  PagedArgs a;
  a.q = (const f16*)q;
  a.kp = (const f16*)kp;
  a.vp = (const f16*)vp;
  a.table = table;
  a.pos = pos;
  a.o = (f16*)o;
  a.pm = ws;
  a.pl = ws + n2;
  a.pa = ws + 2 * n2;
  a.items = items;
  a.rows = rows;
  a.ldq = ldq;
  a.ldt = ldt;
  a.R = R;
  a.MP = MP;
  a.NP = NP;
  a.S = S;
  a.Hq = Hq;
  a.Hk = Hk;
  a.G = Hq / Hk;
  a.PS = __builtin_ctz((unsigned)P);
  a.nitems = nitems;
  a.nown = nown;
  a.parts = parts;
  a.c2 = scale * LOG2E;
  const hipStream_t st = (hipStream_t)stream;
  int rc = ECD_ENOTSUP;
#define PQ(HD_, CT_, W_)                     \
  if (HD == HD_ && ctiles == CT_ && waves == W_) rc = launch_paged<HD_, CT_, W_>(a, R, st)
  PQ(64, 1, 4);
  PQ(64, 2, 4);
  PQ(64, 1, 8);
  PQ(128, 1, 4);
  PQ(128, 2, 4);
  PQ(128, 1, 8);
  PQ(256, 1, 4);
#undef PQ
  if (rc != ECD_OK || parts == 1) return rc;
  hipLaunchKernelGGL(paged_join_kernel, dim3((unsigned)((heads * (HD / 4) + 255) / 256)), dim3(256), 0, st, a, HD, (int)heads);
  return ecd_launch_status();
}
