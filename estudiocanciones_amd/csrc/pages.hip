// Pages of a KV cache, kept on the device (gfx950): free, fork, extend, compact, and the write of a step's keys and
// values (with RoPE) into pages.
//
// State: kv [layers, 2, NP, Hk, P, HD] f16 (keys, values), ref [NP] owners of each page (0: free), table [B, MP] page of
// slots j P .. j P + P - 1 of each sequence (-1 behind the last), length [B] slots held.  Sequence b owns the pages
// table[b, 0 .. ceil(length[b] / P) - 1]; a page may have several owners, and only a page with one owner is written to.
// Free pages are taken lowest number first, in the order of the call's sequences, so a call's result does not depend on
// timing.  A call that finds something wrong sets bits of err (PAGE_E_*) and changes nothing else.
#include "common.h"

namespace ecd {

enum { PAGE_E_INDEX = 1, PAGE_E_TARGET = 2, PAGE_E_FULL = 4, PAGE_E_TABLE = 8, PAGE_E_POOL = 16 };

constexpr int PG_T = 1024;  // threads of the one workgroup that plans a call (and the most sequences it takes)
constexpr int PG_W = PG_T / 64;

__device__ __forceinline__ long pages_of(long slots, int P) { return (slots + P - 1) / P; }

// exclusive sum of v over the workgroup's threads in order, and the total (in every thread)
__device__ __forceinline__ uint32_t block_excl_add(uint32_t v, uint32_t* wsum, uint32_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t inc = wave_incl_add_u32(v);
  if (lane == 63) wsum[w] = inc;
  __syncthreads();
  uint32_t base = 0, all = 0;
#pragma unroll
  for (int i = 0; i < PG_W; ++i) {
    const uint32_t s = wsum[i];
    base += i < w ? s : 0;
    all += s;
  }
  __syncthreads();
  total = all;
  return base + inc - v;
}

// Calls f(rank, page) for the first `want` free pages in ascending order, each in the thread that saw it; returns how
// many of them there are.
template <typename F>
__device__ __forceinline__ uint32_t free_pages(const int* ref, int NP, uint32_t want, uint32_t* wsum, F&& f) {
  uint32_t seen = 0;
  for (int p0 = 0; p0 < NP && seen < want; p0 += PG_T) {
    const int p = p0 + threadIdx.x;
    const bool is = p < NP && ref[p] == 0;
    uint32_t n;
    const uint32_t k = seen + block_excl_add(is, wsum, n);
    if (is && k < want) f(k, p);
    seen += n;
  }
  return seen < want ? seen : want;
}

// One workgroup per entry of seqs: its pages lose an owner (2.4 us for 2 sequences of 5 pages, 3.6 for 32 of 16; a launch is
// about 2).  The length is taken by an exchange, so a sequence that is named twice is freed once.
__global__ __launch_bounds__(256) void page_free_kernel(int* __restrict__ ref, int NP, int* __restrict__ table, int MP,
                                                        int64_t* __restrict__ length, int B, int P,
                                                        const int* __restrict__ seqs, int* __restrict__ err) {
  __shared__ long s_n;
  const int s = seqs[blockIdx.x];
  if (s < 0 || s >= B) {
    if (threadIdx.x == 0) atomicOr(err, PAGE_E_INDEX);
    return;
  }
  if (threadIdx.x == 0) s_n = (long)atomicExch((unsigned long long*)(length + s), 0ull);
  __syncthreads();
  const long n = min(pages_of(s_n > 0 ? s_n : 0, P), (long)MP);
  for (int j = threadIdx.x; j < n; j += 256) {
    const int p = table[(long)s * MP + j];
    if (p >= 0 && p < NP) atomicSub(ref + p, 1);
    table[(long)s * MP + j] = -1;
  }
}

// One workgroup, which sees every refusal before anything is changed: a thread per child finds what it needs, then all look
// at the sources' pages and for free ones, PG_T at a time.  Bound by latency (4.2 us for 2 children, 5.4 for 32 of 2
// prompts of 16 pages; 3.8 and 4.4 without the look at the whole pages).
// plan[i] = {page of the source's partial slots, page for them, their number, whole pages shared (-1: nothing to do)}
__global__ __launch_bounds__(PG_T) void page_fork_plan_kernel(const int* __restrict__ ref, int NP,
                                                              const int* __restrict__ table, int MP,
                                                              int64_t* __restrict__ length, int B, int P,
                                                              const int* __restrict__ src, const int* __restrict__ dst,
                                                              int n, int* __restrict__ plan, int* __restrict__ err) {
  __shared__ uint32_t wsum[PG_W];
  __shared__ int s_dst[PG_T], s_page[PG_T], s_src[PG_T], s_full[PG_T];
  __shared__ int s_err;
  const int t = threadIdx.x, lane = t & 63;
  if (t == 0) s_err = 0;
  s_dst[t] = t < n ? dst[t] : -1;
  s_src[t] = t < n ? src[t] : -1;
  __syncthreads();
  int bad = 0, full = 0, tail = 0, from = 0;
  long len = 0;
  if (t < n) {
    const int s = s_src[t], d = s_dst[t];
    if (s < 0 || s >= B || d < 0 || d >= B) {
      bad = PAGE_E_INDEX;
    } else {
      len = length[s];
      if (length[d] != 0) bad = PAGE_E_TARGET;
      for (int i = 0; i < t; ++i)
        if (s_dst[i] == d) bad |= PAGE_E_TARGET;
      if (len < 0 || len > (long)MP * P) {
        bad |= PAGE_E_TABLE;
      } else {
        full = (int)(len / P);
        tail = (int)(len - (long)full * P);
        if (tail) {
          from = table[(long)s * MP + full];
          if (from < 0 || from >= NP) bad |= PAGE_E_INDEX;
        }
      }
    }
    if (bad) atomicOr(&s_err, bad);
  }
  s_full[t] = full;
  uint32_t want;
  const uint32_t k = block_excl_add(tail > 0, wsum, want);  // (its barriers: s_full whole)
  // the whole pages of each source, a wave per child; children that follow one another share the look at theirs
  for (int i = t >> 6; i < n; i += PG_W)
    if (i == 0 || s_src[i] != s_src[i - 1])
      for (int j = lane; j < s_full[i]; j += 64) {
        const int p = table[(long)s_src[i] * MP + j];
        if (p < 0 || p >= NP) atomicOr(&s_err, PAGE_E_INDEX);
      }
  const uint32_t got = free_pages(ref, NP, want, wsum, [&](uint32_t r, int p) { s_page[r] = p; });
  __syncthreads();  // s_page and s_err whole
  const int e = s_err | (got < want ? PAGE_E_FULL : 0);
  if (t == 0 && e) atomicOr(err, e);
  if (t >= n) return;
  int* pl = plan + 4 * t;
  pl[0] = from;
  pl[1] = tail && !e ? s_page[k] : -1;
  pl[2] = e ? 0 : tail;
  pl[3] = e ? -1 : full;
  if (!e) length[s_dst[t]] = len;
}

// Carries the plan out for FORKS children at a time.  A block holds one 8 KB piece of one (plane, head) run in registers
// and writes it to every child of its source, so the slots of a prompt are read once for all of them (as long as its
// children follow one another); the last block of a row writes the children's tables and counts their pages.
// Bound by the writes.  32 children of 2 prompts, 40 slots of 28 layers (147 MB written): 51.1 us with a block per child
// and run, 30 us now.
constexpr int FORKS = 8, FORK_V = 2;  // children of a block, 16-byte pieces of a thread
__global__ __launch_bounds__(256) void page_fork_kernel(f16* __restrict__ kv, int* __restrict__ ref, int NP,
                                                        int* __restrict__ table, int MP, const int* __restrict__ src,
                                                        const int* __restrict__ dst, const int* __restrict__ plan, int n,
                                                        int pieces, int Hk, int P, int HD) {
  const int i0 = blockIdx.y * FORKS, i1 = min(n, i0 + FORKS);
  if (blockIdx.x == gridDim.x - 1) {
    for (int i = i0; i < i1; ++i) {
      const int to = plan[4 * i + 1], tail = plan[4 * i + 2], full = plan[4 * i + 3];
      if (full < 0) return;
      const int* ts = table + (long)src[i] * MP;
      int* td = table + (long)dst[i] * MP;
      for (int j = threadIdx.x; j < full; j += 256) {
        const int p = ts[j];
        td[j] = p;
        if (p >= 0 && p < NP) atomicAdd(ref + p, 1);
      }
      if (tail && threadIdx.x == 0) {
        td[full] = to;
        ref[to] = 1;
      }
    }
    return;
  }
  const int run = blockIdx.x / pieces, pl = run / Hk, h = run - pl * Hk;
  const int v = (blockIdx.x - run * pieces) * (256 * FORK_V) + threadIdx.x;
  const long page = (long)Hk * P * HD / 8;  // in 16-byte pieces
  u32x4* base = (u32x4*)kv + pl * (NP * page) + (long)h * P * HD / 8 + v;
  int held = -1;
  u32x4 x[FORK_V];
  const int lane = threadIdx.x & 63;
  const u32x4 mine = *(const u32x4*)(plan + 4 * (i0 + min(lane, i1 - i0 - 1)));  // lane i: the plan of child i0 + i
  for (int i = 0; i < i1 - i0; ++i) {
    const int from = __builtin_amdgcn_readlane((int)mine.x, i), to = __builtin_amdgcn_readlane((int)mine.y, i);
    const int tail = __builtin_amdgcn_readlane((int)mine.z, i);
    const int left = tail * (HD / 8) - v;  // pieces of 16 bytes from this thread's first one
    if (left <= 0) continue;
    if (from != held) {
#pragma unroll
      for (int j = 0; j < FORK_V; ++j)
        if (256 * j < left) x[j] = base[from * page + 256 * j];
      held = from;
    }
#pragma unroll
    for (int j = 0; j < FORK_V; ++j)
      if (256 * j < left) __builtin_nontemporal_store(x[j], base + to * page + 256 * j);
  }
}

// Every sequence b holds slot pos[b] afterwards.  The first pass over ref counts, the second one takes, so a call that does not
// fit takes nothing.  Slots in pages that are held: 1.9 us for 6 sequences, 3.9 for 36.
__global__ __launch_bounds__(PG_T) void page_extend_kernel(int* __restrict__ ref, int NP, int* __restrict__ table,
                                                           int MP, int64_t* __restrict__ length, int B, int P,
                                                           const int64_t* __restrict__ pos, int* __restrict__ err) {
  __shared__ uint32_t wsum[PG_W];
  __shared__ uint32_t s_off[PG_T];
  __shared__ int s_have[PG_T];
  __shared__ int s_err;
  const int t = threadIdx.x;
  if (t == 0) s_err = 0;
  long have = 0, more = 0, len = 0;
  bool bad = false;
  if (t < B) {
    len = length[t];
    const long p = pos[t];
    bad = len < 0 || p >= (long)MP * P;
    have = bad ? 0 : pages_of(len, P);
    more = bad || p < len ? 0 : pages_of(p + 1, P) - have;
    if (!bad && p >= len) len = p + 1;
  }
  s_have[t] = (int)have;
  uint32_t want;
  s_off[t] = block_excl_add((uint32_t)more, wsum, want);
  if (bad) atomicOr(&s_err, PAGE_E_TABLE);
  __syncthreads();
  int e = s_err;
  if (!e && want) {
    if (free_pages(ref, NP, want, wsum, [](uint32_t, int) {}) < want) e = PAGE_E_FULL;
    __syncthreads();  // every thread has looked at ref before pages are taken
    if (!e)
      free_pages(ref, NP, want, wsum, [&](uint32_t k, int p) {
        int lo = 0, hi = B - 1;  // the last sequence whose first new page is not behind page k
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (s_off[mid] <= k) lo = mid; else hi = mid - 1;
        }
        table[(long)lo * MP + s_have[lo] + (k - s_off[lo])] = p;
        ref[p] = 1;
      });
  }
  if (e) {
    if (t == 0) atomicOr(err, e);
  } else if (t < B) {
    length[t] = len;
  }
}

// ws: [0] pages in use (-1: they do not fit), then the old number of each new page, then the new number of each old one
__global__ __launch_bounds__(PG_T) void page_compact_plan_kernel(const int* __restrict__ ref, int NP,
                                                                 int* __restrict__ ref2, int NP2, int* __restrict__ ws,
                                                                 int* __restrict__ err) {
  __shared__ uint32_t wsum[PG_W];
  int* old = ws + 1;
  int* now = ws + 1 + NP;
  uint32_t used = 0;
  for (int p0 = 0; p0 < NP; p0 += PG_T) {
    const int p = p0 + threadIdx.x;
    const bool is = p < NP && ref[p] > 0;
    uint32_t n;
    const uint32_t k = used + block_excl_add(is, wsum, n);
    if (p < NP) now[p] = is ? (int)k : -1;
    if (is) old[k] = p;
    used += n;
  }
  __syncthreads();
  const bool fits = used <= (uint32_t)NP2;
  if (threadIdx.x == 0) {
    ws[0] = fits ? (int)used : -1;
    if (!fits) atomicOr(err, PAGE_E_POOL);
  }
  if (!fits) return;
  for (int k = threadIdx.x; k < NP2; k += PG_T) ref2[k] = k < (int)used ? ref[old[k]] : 0;
}

// Bound by memory: 28 layers, 837 MB read and as many written, 330 us (5.1 TB/s, the rate of a plain copy).
__global__ __launch_bounds__(256) void page_compact_kernel(const f16* __restrict__ kv, int NP, f16* __restrict__ kv2,
                                                           int NP2, const int* __restrict__ table,
                                                           int* __restrict__ table2, const int64_t* __restrict__ length,
                                                           int64_t* __restrict__ length2, int B, int MP, int planes,
                                                           long vecs, const int* __restrict__ ws) {
  const int used = ws[0];
  if (used < 0) return;
  const int* old = ws + 1;
  const int* now = ws + 1 + NP;
  const long t = (long)blockIdx.x * 256 + threadIdx.x, step = (long)gridDim.x * 256;
  for (long i = t; i < (long)B * MP; i += step) {
    const int p = table[i];
    table2[i] = p >= 0 && p < NP ? now[p] : -1;
  }
  for (long i = t; i < B; i += step) length2[i] = length[i];
  // units: one page of one plane
  const long units = (long)used * planes;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const int pl = (int)(u / used), k = (int)(u - (long)pl * used);
    const u32x4* a = (const u32x4*)kv + ((long)pl * NP + old[k]) * vecs;
    u32x4* b = (u32x4*)kv2 + ((long)pl * NP2 + k) * vecs;
    for (long v = threadIdx.x; v < vecs; v += 256) b[v] = a[v];
  }
}

// Row m of qkv (sequence m / S, slot pos[m]): the interleaved pairs of its q and k heads are rotated by rope[pos[m]]
// (fp32 products, one rounding, as the dense cache's write), k and v go to the slot's page, q to its own rows.  Without a
// table of angles k and v are written as they are and q is left alone.  A row whose slot has no page writes no k and v.
// One thread per 8 dims, all of them independent.  Bound by memory: 2 prompts of 4000 rows (24 + 2 x 8 heads of 128, 166 MB)
// 32.1 us, 5.1 TB/s; a step of 8 rows 2.8 us.
template <bool ROPE>
__global__ __launch_bounds__(256) void paged_write_kernel(const f16* __restrict__ qkv, long ld,
                                                          const float* __restrict__ rope, int LR,
                                                          const int64_t* __restrict__ pos, f16* __restrict__ q,
                                                          f16* __restrict__ kp, f16* __restrict__ vp,
                                                          const int* __restrict__ table, long ldt, int MP, int NP,
                                                          int M, int S, int Hq, int Hk, int P, int HD) {
  const unsigned heads = ROPE ? Hq + 2 * Hk : 2 * Hk, piece = HD / 8, W = heads * piece;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)M * W) return;
  const unsigned m = (unsigned)(i / W), r = (unsigned)(i - (long)m * W);
  const unsigned hh = r / piece, d = 8 * (r - hh * piece);
  const unsigned h = ROPE ? hh : hh + Hq;
  f16x8 x = *(const f16x8*)(qkv + m * ld + h * (long)HD + d);
  const long p = pos[m];
  if (ROPE && h < (unsigned)(Hq + Hk)) {
    const long pc = p < 0 ? 0 : (p >= LR ? LR - 1 : p);
    const f32x4* t = (const f32x4*)(rope + pc * HD + d);
    const f32x4 c[2] = {t[0], t[1]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float co = c[j >> 1][2 * (j & 1)], si = c[j >> 1][2 * (j & 1) + 1];
      const float a = (float)x[2 * j], b = (float)x[2 * j + 1];
      x[2 * j] = (f16)(a * co - b * si);
      x[2 * j + 1] = (f16)(b * co + a * si);
    }
  }
  if (h < (unsigned)Hq) {
    *(f16x8*)(q + ((long)m * Hq + h) * HD + d) = x;
    return;
  }
  if (p < 0 || p >= (long)MP * P || (ROPE && p >= LR)) return;
  const int page = table[(long)(m / S) * ldt + p / P];
  if (page < 0 || page >= NP) return;
  const unsigned kh = h < (unsigned)(Hq + Hk) ? h - Hq : h - Hq - Hk;
  f16* base = h < (unsigned)(Hq + Hk) ? kp : vp;
  *(f16x8*)(base + (((long)page * Hk + kh) * P + p % P) * HD + d) = x;
}

static bool pool_ok(int planes, int NP, int Hk, int P, int HD) {
  return planes > 0 && NP > 0 && Hk > 0 && P > 0 && HD > 0 && HD % 8 == 0;
}
constexpr long GRID_MOST = 0xFFFFFF;  // workgroups of 256 along x: a launch has fewer than 2^32 threads there
constexpr int COUNT_MOST = 1 << 30;   // pages of a pool or a sequence: loops count them in 32 bits, PG_T at a time
static bool a16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace ecd

using namespace ecd;

extern "C" {

int ecd_page_free(int32_t* ref, int NP, int32_t* table, int MP, int64_t* length, int B, int P, const int32_t* seqs,
                  int n, int32_t* err, void* stream) {
  if (!ref || !table || !length || !seqs || !err || NP <= 0 || MP <= 0 || B <= 0 || P <= 0 || n <= 0) return ECD_EINVAL;
  if (n > GRID_MOST || NP > COUNT_MOST || MP > COUNT_MOST) return ECD_ENOTSUP;
  hipLaunchKernelGGL(page_free_kernel, dim3(n), dim3(256), 0, (hipStream_t)stream, ref, NP, table, MP, length, B, P,
                     seqs, err);
  return ecd_launch_status();
}

int ecd_page_fork(void* kv, int32_t* ref, int NP, int32_t* table, int MP, int64_t* length, int B, const int32_t* src,
                  const int32_t* dst, int n, int32_t* plan, int32_t* err, int planes, int Hk, int P, int HD,
                  void* stream) {
  if (!kv || !ref || !table || !length || !src || !dst || !plan || !err || MP <= 0 || B <= 0 || n <= 0 || n > PG_T ||
      !pool_ok(planes, NP, Hk, P, HD) || !a16(kv) || !a16(plan))
    return ECD_EINVAL;
  const hipStream_t st = (hipStream_t)stream;
  const long pieces = ((long)P * HD / 8 + 256 * FORK_V - 1) / (256 * FORK_V), runs = (long)planes * Hk;
  if (runs >= GRID_MOST || pieces > GRID_MOST / runs || (long)P * HD > 8L * COUNT_MOST || NP > COUNT_MOST || MP > COUNT_MOST)
    return ECD_ENOTSUP;
  const long x = pieces * runs + 1;
  if (x > GRID_MOST) return ECD_ENOTSUP;
  hipLaunchKernelGGL(page_fork_plan_kernel, dim3(1), dim3(PG_T), 0, st, ref, NP, table, MP, length, B, P, src, dst, n,
                     plan, err);
  hipLaunchKernelGGL(page_fork_kernel, dim3((unsigned)x, (n + FORKS - 1) / FORKS), dim3(256), 0, st, (f16*)kv, ref, NP,
                     table, MP, src, dst, plan, n, (int)pieces, Hk, P, HD);
  return ecd_launch_status();
}

int ecd_page_extend(int32_t* ref, int NP, int32_t* table, int MP, int64_t* length, int B, int P, const int64_t* pos,
                    int32_t* err, void* stream) {
  if (!ref || !table || !length || !pos || !err || NP <= 0 || MP <= 0 || B <= 0 || B > PG_T || P <= 0) return ECD_EINVAL;
  // (new pages are counted in 32 bits)
  if ((long)B * MP > 0xFFFFFFFFL || NP > COUNT_MOST || MP > COUNT_MOST) return ECD_ENOTSUP;
  hipLaunchKernelGGL(page_extend_kernel, dim3(1), dim3(PG_T), 0, (hipStream_t)stream, ref, NP, table, MP, length, B, P,
                     pos, err);
  return ecd_launch_status();
}

int ecd_page_compact(const void* kv, const int32_t* ref, int NP, const int32_t* table, const int64_t* length, void* kv2,
                     int32_t* ref2, int NP2, int32_t* table2, int64_t* length2, int B, int MP, int32_t* ws,
                     int32_t* err, int planes, int Hk, int P, int HD, void* stream) {
  if (!kv || !ref || !table || !length || !kv2 || !ref2 || !table2 || !length2 || !ws || !err || B <= 0 || MP <= 0 ||
      NP2 <= 0 || !pool_ok(planes, NP, Hk, P, HD) || !a16(kv) || !a16(kv2) || kv == kv2)
    return ECD_EINVAL;
  if (NP > COUNT_MOST || NP2 > COUNT_MOST || MP > COUNT_MOST) return ECD_ENOTSUP;
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(page_compact_plan_kernel, dim3(1), dim3(PG_T), 0, st, ref, NP, ref2, NP2, ws, err);
  hipLaunchKernelGGL(page_compact_kernel, dim3(4096), dim3(256), 0, st, (const f16*)kv, NP, (f16*)kv2, NP2, table,
                     table2, length, length2, B, MP, planes, (long)Hk * P * HD / 8, ws);
  return ecd_launch_status();
}

int ecd_paged_write(const void* qkv, long ld, const float* rope, int LR, const int64_t* pos, void* q, void* kp,
                    void* vp, const int32_t* table, long ldt, int MP, int NP, int M, int S, int Hq, int Hk, int P,
                    int HD, void* stream) {
  if (!qkv || !pos || !kp || !vp || !table || (rope && (!q || LR <= 0)) || M <= 0 || S <= 0 || Hq <= 0 || MP <= 0 ||
      ldt < MP || !pool_ok(1, NP, Hk, P, HD) || ld < (Hq + 2L * Hk) * HD || (ld % 8) || !a16(qkv) || !a16(kp) ||
      !a16(vp) || (q && !a16(q)) || ((uintptr_t)rope & 15))
    return ECD_EINVAL;
  const long W = (rope ? Hq + 2L * Hk : 2L * Hk) * (HD / 8);
  if (W > 0x7FFFFFFFL || (M * W + 255) / 256 > GRID_MOST) return ECD_ENOTSUP;
  const long blocks = (M * W + 255) / 256;
  const hipStream_t st = (hipStream_t)stream;
#define PW(R_)                                                                                                        \
  hipLaunchKernelGGL((paged_write_kernel<R_>), dim3((unsigned)blocks), dim3(256), 0, st, (const f16*)qkv, ld, rope,    \
                     LR, pos, (f16*)q, (f16*)kp, (f16*)vp, table, ldt, MP, NP, M, S, Hq, Hk, P, HD)
  if (rope) PW(true); else PW(false);
#undef PW
  return ecd_launch_status();
}

}  // extern "C"
