// Page operators of a paged cache for MI355X (gfx950): copies of pages in
// every layer, forks, growth, freeing and compaction of sequences.
//
// State (device memory of the caller): block tables [rows, M], context
// lengths [rows] and one reference count a page (0: free).  No free list is
// kept: a free page is one whose count is 0, and pages are given out from the
// lowest index up, so every result is a function of the state alone.
//
// What bounds it: the copies move 2 bytes per byte of a copied page and run at
// HBM speed; everything else is integer work on a few kilobytes, where the
// launches and the chains of dependent reads count, so each operator takes as
// few launches as its order of reads and writes allows (copy 1 or 2, fork 1,
// free 1, extend 2, compact 3).  512 scattered 16 KiB pages of 64 caches: 217 us
// for the copies, 4.9 TB/s; 3445 moves of a compaction, whose sources and targets
// both rise, in 16 caches: 357 us, 5.1 TB/s; a contiguous copy of 2 GiB: 4.9 TB/s.
// 256 copies of eight partial pages of 64 caches, of which the memory sees the
// writes: 102 us, 5.3 TB/s written.
//
// Every decision is taken on the state as it was before the call: a launch
// never reads what another workgroup of it writes.  Reference counts change
// by integer atomics, whose order does not matter.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pa_check.h"
#include "pa_fp8.h"
#include "pa_plan.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kGroup = 16;                           // pages of a mask
constexpr int kChunk = kPlanThreads * kGroup;        // pages a workgroup counts
constexpr int kMaxChunks = 256;
constexpr int kMaxPages = kMaxChunks * kChunk;       // 4 Mi
constexpr int kMaxList = 65536;                      // pairs or sequences of a call
constexpr int kMaxExtend = 4096;                     // sequences of an extend (one workgroup plans them)

struct Table {
  int32_t* tables;
  int64_t stride;
  int32_t* lengths;
  int32_t* refs;
  int rows, width, pages, lbs;
};

// Page entry j of a table row; -1 (and noted) where it is outside the cache.
__device__ __forceinline__ int page_at(const Table& t, int row, int j) {
  const int p = t.tables[(int64_t)row * t.stride + j];
  const bool bad = p < 0 || p >= t.pages;
  pa_note(bad, PA_VIOLATION_PAGE);
  return bad ? -1 : p;
}
// Pages n tokens take (n >= 0).
__device__ __forceinline__ int pages_of(const Table& t, int n) { return (int)(((int64_t)n + (1 << t.lbs) - 1) >> t.lbs); }

// Whether list[0 .. n) holds v (before entry `upto`); the whole workgroup asks.
__device__ __forceinline__ bool listed(const int32_t* list, int upto, int v) {
  bool hit = false;
  for (int j = threadIdx.x; j < upto; j += kThreads) hit |= list[j] == v;
  return __syncthreads_or(hit);
}

// ---------------------------------------------------------------------------
// Copies
// ---------------------------------------------------------------------------

constexpr int kUnit = 4096;       // bytes a wave copies at a time
constexpr int kWaves = kThreads / 64;
constexpr int kMaxCaches = 96;    // caches of a launch
constexpr int kWaveList = 64;     // pairs that every wave checks by itself

struct Cache {
  uint8_t* data;
  int64_t stride;
  uint32_t bytes;  // of a page
  int unit;        // first unit among those of a page in all caches; the sign bit: not all 16-byte aligned
};
struct CopyArgs {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* count;  // pairs (nullptr: n)
  int32_t* status;       // not nullptr: pairs of a caller, at most kWaveList of them, that no other launch has looked through
  int n, pages, caches, units;
  bool once;             // no page is the source of two pairs: its bytes need not stay in a cache
  Cache c[kMaxCaches];
};

// Whether pair j = (sj, dj) stands in the way of pair i = (s, d): it has the
// same target and comes later (the last one counts), or the target is its
// source (whose old bytes would be lost or not, by chance).  A page copied to
// itself is left as it is, and in nobody's way.
__device__ __forceinline__ bool blocks(int s, int d, int j, int sj, int dj, int i, int pages) {
  const bool real = sj >= 0 && sj < pages && dj >= 0 && dj < pages && sj != dj;
  return real && s != d && j != i && ((j > i && dj == d) || sj == d);
}

// Targets of checked pairs: the pair's own, or -1.  A wave looks through the whole
// list for kWavePairs of them, 64 entries at a time (512 pairs: 6 us; a thread a
// pair, with the list in LDS, took 78).
constexpr int kWavePairs = 4, kFilterPairs = kThreads / 64 * kWavePairs;
__global__ __launch_bounds__(kThreads) void pa_pages_filter_kernel(const int32_t* src, const int32_t* dst, int n, int pages,
                                                                   int32_t* out, int32_t* status) {
  const int lane = threadIdx.x & 63;
  const int i0 = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * kWavePairs);
  if (i0 >= n) return;
  int s[kWavePairs], d[kWavePairs];
#pragma unroll
  for (int p = 0; p < kWavePairs; ++p) {
    const int i = pa_min(i0 + p, n - 1);
    s[p] = __builtin_amdgcn_readfirstlane(src[i]);
    d[p] = __builtin_amdgcn_readfirstlane(dst[i]);
  }
  uint32_t blocked = 0;
  constexpr int kAhead = 4;
  for (int j0 = 0; j0 < n; j0 += 64 * kAhead) {
    int sj[kAhead], dj[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = j0 + 64 * k + lane;
      sj[k] = j < n ? src[j] : -1;
      dj[k] = j < n ? dst[j] : -1;
    }
#pragma unroll
    for (int p = 0; p < kWavePairs; ++p) {
      bool hit = false;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) hit |= blocks(s[p], d[p], j0 + 64 * k + lane, sj[k], dj[k], i0 + p, pages);
      if (__ballot(hit)) blocked |= 1u << p;
    }
  }
  const int i = i0 + lane;
  if (lane >= kWavePairs || i >= n) return;
  const int si = src[i], di = dst[i];
  pa_note(si >= pages || di >= pages, PA_VIOLATION_PAGE);
  const bool ok = si >= 0 && si < pages && di >= 0 && di < pages && !(blocked >> lane & 1);
  out[i] = ok ? di : -1;
  status[i] = ok;
}

// Bytes of `unit` of page s of a cache onto page d, by one wave, so that small pages,
// a token block's scales among them, do not hold a workgroup each (4 KiB pages and
// 128-byte scales, 16 caches, 2600 moves: 48 us; a workgroup a unit of 16 KiB: 80; large
// pages alike, a small pool's compaction 15.8 and 14.9 us).  Written past the caches:
// no one reads them soon; read through them where a page may have several targets
// (256 copies of 8 pages: 203 us past them, 135 us through).
__device__ __forceinline__ void copy_unit(const Cache& c, int unit, int s, int d, bool once) {
  const uint32_t at = (uint32_t)unit * kUnit;
  const uint32_t n = pa_min(kUnit, (int)(c.bytes - at));
  const uint8_t* from = c.data + (int64_t)s * c.stride + at;
  uint8_t* to = c.data + (int64_t)d * c.stride + at;
  const int lane = threadIdx.x & 63;
  if (c.unit >= 0) {  // four loads in flight a lane
    i32x4 v[4];
    if (n == kUnit && once) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __builtin_nontemporal_load((const i32x4*)from + k * 64 + lane);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (16u * (k * 64 + lane) < n) v[k] = ((const i32x4*)from)[k * 64 + lane];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (16u * (k * 64 + lane) < n) __builtin_nontemporal_store(v[k], (i32x4*)to + k * 64 + lane);
  } else {
    for (uint32_t k = lane; k < n; k += 64) to[k] = from[k];
  }
}

// Unit u of all caches' units of a page -> its cache.
__device__ __forceinline__ int cache_of(const CopyArgs& a, int u) {
  int lo = 0, hi = a.caches;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if ((a.c[m].unit & 0x7fffffff) <= u)
      lo = m;
    else
      hi = m;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void pa_pages_copy_kernel(const CopyArgs a) {
  const int n = a.count ? pa_min(a.count[0], a.n) : a.n;
  const int64_t total = (int64_t)n * a.units;
  const int lane = threadIdx.x & 63;
  int ws = -1, wd = -1;
  if (a.status && lane < n) {
    ws = a.src[lane];
    wd = a.dst[lane];
    pa_note(ws >= a.pages || wd >= a.pages, PA_VIOLATION_PAGE);
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int64_t x = (int64_t)blockIdx.x * kWaves + wave; x < total; x += (int64_t)gridDim.x * kWaves) {
    const int u = __builtin_amdgcn_readfirstlane((int)(x / n));
    const int i = __builtin_amdgcn_readfirstlane((int)(x - (int64_t)u * n));
    int s, d;
    bool ok;
    if (a.status) {
      s = __builtin_amdgcn_readlane(ws, i);
      d = __builtin_amdgcn_readlane(wd, i);
      ok = s >= 0 && s < a.pages && d >= 0 && d < a.pages && !__ballot(lane < n && blocks(s, d, lane, ws, wd, i, a.pages));
      if (u == 0 && lane == 0) a.status[i] = ok;
    } else {
      s = a.src[i];
      d = a.dst[i];
      ok = s >= 0 && s < a.pages && d >= 0 && d < a.pages;
    }
    if (!ok || s == d) continue;
    const int k = cache_of(a, u);
    copy_unit(a.c[k], u - (a.c[k].unit & 0x7fffffff), s, d, a.once);
  }
}

// ---------------------------------------------------------------------------
// The pool: which pages are free
// ---------------------------------------------------------------------------

// Of each group of 16 pages: which are held (pages past the pool count as
// held) and the free pages before it in its chunk; of each chunk its free pages.
struct Pool {
  uint16_t* held;
  uint16_t* before;
  int32_t* free_pages;  // [chunks]
  int chunks;
};

__device__ __forceinline__ int wave_upto(int v) {  // inclusive sum over the wave
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}
// Sum of v over the threads before this one (N threads); *total over all.
template <int N>
__device__ __forceinline__ int block_before(int v, int* total, int* scratch) {
  const int upto = wave_upto(v), wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) scratch[wave] = upto;
  __syncthreads();
  int before = upto - v, all = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) {
    if (w < wave) before += scratch[w];
    all += scratch[w];
  }
  *total = all;
  return before;
}

__device__ __forceinline__ void count_chunk(const int32_t* refs, int pages, const Pool& p, int chunk, int* scratch) {
  const int group = chunk * kPlanThreads + threadIdx.x;
  const int64_t p0 = (int64_t)group * kGroup;
  uint32_t held = 0;
  if (p0 + kGroup <= pages) {
#pragma unroll
    for (int k = 0; k < kGroup; ++k) held |= (refs[p0 + k] > 0 ? 1u : 0u) << k;
  } else {
    for (int k = 0; k < kGroup; ++k) held |= (p0 + k >= pages || refs[p0 + k] > 0 ? 1u : 0u) << k;
  }
  int total;
  const int before = block_before<kPlanThreads>(kGroup - __popc(held), &total, scratch);
  p.held[group] = (uint16_t)held;
  p.before[group] = (uint16_t)before;
  if (threadIdx.x == 0) p.free_pages[chunk] = total;
}

// Free pages before each chunk into lds[0 .. chunks], for N threads.
template <int N>
__device__ __forceinline__ void chunk_sums(const Pool& p, int* lds, int* scratch) {
  static_assert(N >= kMaxChunks, "one thread a chunk");
  const int v = (int)threadIdx.x < p.chunks ? p.free_pages[threadIdx.x] : 0;
  int total;
  const int before = block_before<N>(v, &total, scratch);
  if ((int)threadIdx.x < p.chunks) lds[threadIdx.x] = before;
  if (threadIdx.x == 0) lds[p.chunks] = total;
  __syncthreads();
}
// The free page that has k free ones below it (k < all).
__device__ __forceinline__ int free_page(const Pool& p, const int* sums, int k) {
  int lo = 0, hi = p.chunks;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (sums[m] <= k)
      lo = m;
    else
      hi = m;
  }
  k -= sums[lo];
  const int g0 = lo * kPlanThreads;
  int a = 0, b = kPlanThreads;
  while (b - a > 1) {
    const int m = (a + b) >> 1;
    if ((int)p.before[g0 + m] <= k)
      a = m;
    else
      b = m;
  }
  k -= (int)p.before[g0 + a];
  uint32_t open = ~(uint32_t)p.held[g0 + a] & 0xffffu;
  for (; k > 0; --k) open &= open - 1;
  return (g0 + a) * kGroup + __builtin_ctz(open | 0x10000u);
}
// Free pages below page x (x <= pages).
__device__ __forceinline__ int free_below(const Pool& p, const int* sums, int x) {
  const int chunk = x / kChunk;
  if (chunk >= p.chunks) return sums[p.chunks];
  const int g = x / kGroup;
  const uint32_t open = ~(uint32_t)p.held[g] & ((1u << (x % kGroup)) - 1u);
  return sums[chunk] + (int)p.before[g] + __popc(open);
}

// ---------------------------------------------------------------------------
// Fork and free
// ---------------------------------------------------------------------------

// Workgroup i: pair i.
__global__ __launch_bounds__(kThreads) void pa_pages_fork_kernel(const Table t, const int32_t* parents,
                                                                 const int32_t* children, int n, int32_t* status) {
  const int i = blockIdx.x;
  const int p = parents[i], c = children[i];
  bool ok = p >= 0 && p < t.rows && c >= 0 && c < t.rows;
  const bool twice = listed(children, i, c), both = listed(children, n, p);
  ok = ok && !twice && !both;
  int len = 0;
  if (ok) {
    len = t.lengths[p];
    // (only this workgroup writes row c and its length)
    ok = t.lengths[c] == 0 && len >= 0 && len <= (int64_t)t.width << t.lbs;
  }
  __syncthreads();  // every thread has read lengths[c]
  if (ok) {
    const int used = pages_of(t, len);
    for (int j = threadIdx.x; j < used; j += kThreads) {
      t.tables[(int64_t)c * t.stride + j] = t.tables[(int64_t)p * t.stride + j];
      const int page = page_at(t, p, j);
      if (page >= 0) atomicAdd(t.refs + page, 1);
    }
  }
  if (threadIdx.x == 0) {
    if (ok) t.lengths[c] = len;
    status[i] = ok;
  }
}

// Workgroup i: sequence i.
__global__ __launch_bounds__(kThreads) void pa_pages_free_kernel(const Table t, const int32_t* seqs,
                                                                 const int32_t* new_lengths, int32_t* status) {
  const int i = blockIdx.x;
  const int s = seqs[i];
  bool ok = s >= 0 && s < t.rows;
  ok = !listed(seqs, i, s) && ok;
  const int keep = new_lengths ? new_lengths[i] : 0;
  int len = 0;
  if (ok) {
    len = t.lengths[s];
    ok = keep >= 0 && keep <= len;
  }
  __syncthreads();  // every thread has read lengths[s]
  if (ok) {
    const int end = pa_min(pages_of(t, len), t.width);
    for (int j = pages_of(t, keep) + threadIdx.x; j < end; j += kThreads) {
      const int page = page_at(t, s, j);
      // a count that is 0 stays 0
      if (page >= 0 && atomicSub(t.refs + page, 1) <= 0) {
        pa_note(true, PA_VIOLATION_PAGE);
        atomicAdd(t.refs + page, 1);
      }
    }
  }
  if (threadIdx.x == 0) {
    if (ok) t.lengths[s] = keep;
    status[i] = ok;
  }
}

// ---------------------------------------------------------------------------
// Extend
// ---------------------------------------------------------------------------

struct Extend {
  Table t;
  Pool pool;
  const int32_t* seqs;
  const int32_t* new_lengths;
  int n;
  int32_t* status;
  // workspace [n]
  int32_t* start;  // pages given out before the sequence's, -1: left out
  int32_t* old;    // its length
  int32_t* src;    // shared partial page to copy, or -1
};

// For each entry i of list[0 .. n) (LDS): how many entries before it are equal to
// it (and not negative).  The threads of an entry share the entries before it, so
// that a short list takes few turns; out[] is cleared and complete on return.
__device__ __forceinline__ void count_before(const int* list, int n, int* out) {
  for (int i = threadIdx.x; i < n; i += kPlanThreads) out[i] = 0;
  __syncthreads();
  int wide = 64;  // entries at a time: whole waves, whose reads are broadcasts
  while (wide < n && wide < kPlanThreads) wide *= 2;
  const int parts = kPlanThreads / wide, part = (int)threadIdx.x / wide;
  for (int i = (int)threadIdx.x % wide; i < n; i += wide) {
    const int v = list[i];
    if (v < 0) continue;
    const int4* at = reinterpret_cast<const int4*>(list);
    int count = 0;
#pragma unroll 4
    for (int j = part; 4 * j < i; j += parts) {
      const int4 w = at[j];
      count += (w.x == v) + (w.y == v && 4 * j + 1 < i) + (w.z == v && 4 * j + 2 < i) +
               (w.w == v && 4 * j + 3 < i);
    }
    if (count) atomicAdd(&out[i], count);
  }
  __syncthreads();
}

// Workgroups 0 .. chunks - 1 count the pool, the last one plans the
// sequences: what each needs, and where in the row of given pages it begins.
// A sequence's shared partial page is copied unless every other holder has
// been listed, with such a page, before it: its last holder keeps it.
__global__ __launch_bounds__(kPlanThreads) void pa_pages_extend_plan_kernel(const Extend e) {
  __shared__ int scratch[kPlanThreads / 64];
  __shared__ __align__(16) int list[kMaxExtend];
  __shared__ int before[kMaxExtend];
  if ((int)blockIdx.x < e.pool.chunks) {
    count_chunk(e.t.refs, e.t.pages, e.pool, blockIdx.x, scratch);
    return;
  }
  constexpr int kPer = kMaxExtend / kPlanThreads;
  int need[kPer], len[kPer], share[kPer], held[kPer];
  // a thread's sequences are consecutive, so that its sums are in list order
  const int per = (e.n + kPlanThreads - 1) / kPlanThreads, i0 = (int)threadIdx.x * per;
  const int mine = pa_max(pa_min(per, e.n - i0), 0);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    need[k] = share[k] = -1;
    len[k] = held[k] = 0;
    if (k >= mine) continue;
    const int s = e.seqs[i0 + k], want = e.new_lengths[i0 + k];
    const bool in = s >= 0 && s < e.t.rows;
    list[i0 + k] = in ? s : -1;
    if (!in) continue;
    len[k] = e.t.lengths[s];
    if (len[k] < 0 || want < len[k] || want > (int64_t)e.t.width << e.t.lbs) continue;
    need[k] = pages_of(e.t, want) - pages_of(e.t, len[k]);
    if (want > len[k] && (len[k] & ((1 << e.t.lbs) - 1))) {
      const int p = page_at(e.t, s, len[k] >> e.t.lbs);
      if (p >= 0) {
        held[k] = e.t.refs[p];
        if (held[k] > 1) share[k] = p;
      }
    }
  }
  __syncthreads();
  count_before(list, e.n, before);
  bool any = false;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (k >= mine) continue;
    if (before[i0 + k]) need[k] = share[k] = -1;  // named before
    any |= share[k] >= 0;
  }
  any = __syncthreads_or(any);
  if (any) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (k < mine) list[i0 + k] = share[k];
    __syncthreads();
    count_before(list, e.n, before);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k >= mine || share[k] < 0) continue;
      if (before[i0 + k] < held[k] - 1)
        need[k] += 1;
      else
        share[k] = -1;
    }
  }
  int sum = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) sum += pa_max(need[k], 0);
  int total;
  int at = block_before<kPlanThreads>(sum, &total, scratch);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (k >= mine) continue;
    e.start[i0 + k] = need[k] >= 0 ? at : -1;
    e.old[i0 + k] = len[k];
    e.src[i0 + k] = share[k];
    at += pa_max(need[k], 0);
  }
}

// Workgroups (i, y): sequence i gets its pages, if the pool reaches that far (y = 0
// of the first launch), and the copy of its shared partial page (units y, y + Y ..
// of the caches of this launch).
__global__ __launch_bounds__(kThreads) void pa_pages_extend_kernel(const Extend e, const CopyArgs a, bool first) {
  __shared__ int sums[kMaxChunks + 1];
  __shared__ int scratch[kThreads / 64];
  const int i = blockIdx.x;
  const bool assign = first && blockIdx.y == 0;
  const int share = e.src[i];
  if (!assign && share < 0) return;
  const int start = e.start[i], len = e.old[i], s = e.seqs[i], want = e.new_lengths[i];
  chunk_sums<kThreads>(e.pool, sums, scratch);
  int need = 0;
  bool ok = start >= 0;
  if (ok) {
    need = pages_of(e.t, want) - pages_of(e.t, len) + (share >= 0);
    ok = start + need <= sums[e.pool.chunks];
  }
  if (assign) {
    if (ok) {
      int32_t* row = e.t.tables + (int64_t)s * e.t.stride;
      const int col = share >= 0 ? len >> e.t.lbs : pages_of(e.t, len);
      for (int k = threadIdx.x; k < need; k += kThreads) {
        const int p = free_page(e.pool, sums, start + k);
        row[col + k] = p;
        e.t.refs[p] = 1;
      }
    }
    if (threadIdx.x == 0) {
      if (ok && share >= 0) atomicSub(e.t.refs + share, 1);
      if (ok) e.t.lengths[s] = want;
      e.status[i] = ok;
    }
  }
  if (!ok || share < 0) return;
  const int to = free_page(e.pool, sums, start);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int u = (int)blockIdx.y * kWaves + wave; u < a.units; u += (int)gridDim.y * kWaves) {
    const int k = cache_of(a, u);
    copy_unit(a.c[k], u - (a.c[k].unit & 0x7fffffff), share, to, false);
  }
}

// ---------------------------------------------------------------------------
// Compact
// ---------------------------------------------------------------------------

struct Compact {
  Table t;
  Pool pool;
  int32_t* new_tables;
  int64_t new_stride;
  int32_t* new_refs;
  int32_t* map;
  int32_t* live;
  int32_t* src;  // [pages] moves
  int32_t* dst;
  int32_t* moves;
  int page_groups;  // workgroups that walk pages; the others walk table rows
};

__global__ __launch_bounds__(kPlanThreads) void pa_pages_count_kernel(const int32_t* refs, int pages, const Pool pool) {
  __shared__ int scratch[kPlanThreads / 64];
  count_chunk(refs, pages, pool, blockIdx.x, scratch);
}

// A live page below `live` stays; the k-th at or above it goes to the k-th
// free page below it.
__global__ __launch_bounds__(kThreads) void pa_pages_compact_kernel(const Compact c) {
  __shared__ int sums[kMaxChunks + 1];
  __shared__ int scratch[kThreads / 64];
  chunk_sums<kThreads>(c.pool, sums, scratch);
  const int live = c.t.pages - sums[c.pool.chunks];
  const int holes = free_below(c.pool, sums, live);  // as many pages move
  auto moved_to = [&](int p, int* k) {  // p live, p >= live
    // live pages in [live, p): those below p less those below `live`
    *k = (p - free_below(c.pool, sums, p)) - (live - holes);
    return free_page(c.pool, sums, *k);
  };
  if ((int)blockIdx.x < c.page_groups) {
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      c.live[0] = live;
      c.moves[0] = holes;
    }
    const int64_t p64 = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (p64 >= c.t.pages) return;
    const int p = (int)p64;
    const int ref = c.t.refs[p];
    const bool held = ref > 0;
    if (p < live) {
      c.map[p] = held ? p : -1;
      if (held) c.new_refs[p] = ref;  // a free page's entry is written with the page that comes to it
    } else {
      int to = -1;
      if (held) {
        int k;
        to = moved_to(p, &k);
        c.src[k] = p;
        c.dst[k] = to;
        c.new_refs[to] = ref;
      }
      c.map[p] = to;
      c.new_refs[p] = 0;
    }
    return;
  }
  const int row = blockIdx.x - c.page_groups;
  const int len = pa_max(c.t.lengths[row], 0);
  const int used = pa_min(pages_of(c.t, len), c.t.width);
  for (int j = threadIdx.x; j < c.t.width; j += kThreads) {
    int p = c.t.tables[(int64_t)row * c.t.stride + j];
    if (j < used) {
      const bool in = p >= 0 && p < c.t.pages;
      pa_note(!in, PA_VIOLATION_PAGE);
      if (in && c.t.refs[p] <= 0)
        p = -1;
      else if (in && p >= live) {
        int k;
        p = moved_to(p, &k);
      }
    }
    c.new_tables[(int64_t)row * c.new_stride + j] = p;
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

int table_of(const pa_fp8_page_table_args* a, Table* t) {
  if (!a) return PA_ERR_NULL_ARG;
  if (a->abi_version != PA_FP8_ABI_VERSION) return PA_ERR_ABI;
  const int bs = a->block_size;
  if (bs < 1 || bs > (1 << 20) || (bs & (bs - 1))) return PA_ERR_BLOCK_SIZE;
  if (a->num_rows < 0 || a->max_blocks_per_seq < 0 || a->num_blocks < 0 || a->num_blocks > kMaxPages ||
      a->stride_bt_seq < 0)
    return PA_ERR_SHAPE;
  if ((a->num_rows > 0 && ((a->max_blocks_per_seq > 0 && !a->block_tables) || !a->context_lengths)) ||
      (a->num_blocks > 0 && !a->ref_counts))
    return PA_ERR_NULL_ARG;
  t->tables = a->block_tables;
  t->stride = a->stride_bt_seq;
  t->lengths = a->context_lengths;
  t->refs = a->ref_counts;
  t->rows = a->num_rows;
  t->width = a->max_blocks_per_seq;
  t->pages = a->num_blocks;
  t->lbs = 31 - __builtin_clz((unsigned)bs);
  return PA_OK;
}

int check_caches(const pa_fp8_page_cache* c, int n, int pages) {
  if (n < 0 || pages < 0) return PA_ERR_SHAPE;
  if (n > 0 && !c) return PA_ERR_NULL_ARG;
  for (int i = 0; i < n; ++i) {
    if (pages > 0 && c[i].page_bytes > 0 && !c[i].data) return PA_ERR_NULL_ARG;
    if (c[i].page_bytes < 0 || c[i].page_bytes > (1 << 30) || c[i].stride_bytes < c[i].page_bytes) return PA_ERR_SHAPE;
  }
  return PA_OK;
}

// The next caches of a list, from *at on, that one launch takes.
void next_caches(const pa_fp8_page_cache* caches, int num, int* at, CopyArgs* a) {
  int64_t units = 0;
  int k = 0;
  for (; *at < num && k < kMaxCaches; ++*at) {
    const pa_fp8_page_cache& c = caches[*at];
    if (c.page_bytes == 0) continue;
    const int64_t more = (c.page_bytes + kUnit - 1) / kUnit;
    if (units + more > 0x3fffffff) break;
    const bool odd = (((uintptr_t)c.data | (uintptr_t)c.stride_bytes | (uintptr_t)c.page_bytes) & 15u) != 0;
    a->c[k].data = (uint8_t*)c.data;
    a->c[k].stride = c.stride_bytes;
    a->c[k].bytes = (uint32_t)c.page_bytes;
    a->c[k].unit = (int)units | (odd ? (int)0x80000000u : 0);
    units += more;
    ++k;
  }
  a->caches = k;
  a->units = (int)units;
}

constexpr int kCopyGrid = 4096;  // workgroups of a copy: 16 a CU

// Copies of a list of pairs in every cache, kMaxCaches caches a launch.
hipError_t launch_copy(const pa_fp8_page_cache* caches, int num, const int32_t* src, const int32_t* dst,
                       const int32_t* count, int n, int pages, int32_t* status, bool once, hipStream_t s) {
  for (int at = 0; at < num;) {
    CopyArgs a;
    a.src = src;
    a.dst = dst;
    a.count = count;
    a.n = n;
    a.pages = pages;
    a.status = status;
    a.once = once;
    next_caches(caches, num, &at, &a);
    if (a.caches == 0) continue;
    const int64_t total = (int64_t)n * a.units;
    const int64_t groups = (total + kWaves - 1) / kWaves;
    hipLaunchKernelGGL(pa_pages_copy_kernel, dim3((unsigned)(groups < kCopyGrid ? groups : kCopyGrid)), dim3(kThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

int64_t up(int64_t n) { return (n + 255) & ~(int64_t)255; }
int chunks_of(int pages) { return pages > 0 ? (pages + kChunk - 1) / kChunk : 1; }
int64_t pool_bytes(int pages) { return 2 * up(2 * (int64_t)chunks_of(pages) * kPlanThreads) + up(4 * kMaxChunks); }
Pool pool_at(char* ws, int pages) {
  Pool p;
  const int64_t masks = up(2 * (int64_t)chunks_of(pages) * kPlanThreads);
  p.held = (uint16_t*)ws;
  p.before = (uint16_t*)(ws + masks);
  p.free_pages = (int32_t*)(ws + 2 * masks);
  p.chunks = chunks_of(pages);
  return p;
}

int done(hipError_t e) { return e == hipSuccess ? PA_OK : (int)e; }

}  // namespace

PA_CHECK_DEFINE_TAKE(pa_violations_cache_pages)

extern "C" int64_t pa_fp8_pages_workspace_bytes(int operation, int num_blocks, int n) {
  if (num_blocks < 0 || num_blocks > kMaxPages || n < 0 || n > kMaxList) return PA_ERR_SHAPE;
  switch (operation) {
    case PA_PAGES_COPY: return up(4 * (int64_t)n);
    case PA_PAGES_EXTEND: return n > kMaxExtend ? PA_ERR_SHAPE : pool_bytes(num_blocks) + 3 * up(4 * (int64_t)n);
    case PA_PAGES_COMPACT: return pool_bytes(num_blocks) + 2 * up(4 * (int64_t)num_blocks) + 256;
    default: return PA_ERR_SHAPE;
  }
}

extern "C" int pa_fp8_copy_pages(const pa_fp8_page_cache* caches, int num_caches, int num_blocks, const int32_t* src,
                                 const int32_t* dst, int n, int32_t* status, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  const int rc = check_caches(caches, num_caches, num_blocks);
  if (rc != PA_OK) return rc;
  if (n < 0 || n > kMaxList) return PA_ERR_SHAPE;
  if (n == 0) return PA_OK;
  if (!src || !dst || !status) return PA_ERR_NULL_ARG;
  bool bytes = false;  // whether there is anything to copy
  for (int i = 0; i < num_caches; ++i) bytes |= caches[i].page_bytes > 0;
  hipStream_t s = (hipStream_t)stream;
  if (n <= kWaveList && bytes) return done(launch_copy(caches, num_caches, src, dst, nullptr, n, num_blocks, status, false, s));
  if (!workspace) return PA_ERR_NULL_ARG;
  if (workspace_bytes < up(4 * (int64_t)n)) return PA_ERR_SCRATCH;
  hipLaunchKernelGGL(pa_pages_filter_kernel, dim3((unsigned)((n + kFilterPairs - 1) / kFilterPairs)), dim3(kThreads), 0, s, src, dst,
                     n, num_blocks, (int32_t*)workspace, status);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  return done(launch_copy(caches, num_caches, src, (const int32_t*)workspace, nullptr, n, num_blocks, nullptr, false, s));
}

extern "C" int pa_fp8_fork_pages(const pa_fp8_page_table_args* a, const int32_t* parents, const int32_t* children, int n,
                                 int32_t* status, void* stream) {
  Table t;
  const int rc = table_of(a, &t);
  if (rc != PA_OK) return rc;
  if (n < 0 || n > kMaxList) return PA_ERR_SHAPE;
  if (n == 0) return PA_OK;
  if (!parents || !children || !status) return PA_ERR_NULL_ARG;
  hipLaunchKernelGGL(pa_pages_fork_kernel, dim3((unsigned)n), dim3(kThreads), 0, (hipStream_t)stream, t, parents, children, n,
                     status);
  return done(hipGetLastError());
}

extern "C" int pa_fp8_free_pages(const pa_fp8_page_table_args* a, const int32_t* sequences, const int32_t* new_lengths,
                                 int n, int32_t* status, void* stream) {
  Table t;
  const int rc = table_of(a, &t);
  if (rc != PA_OK) return rc;
  if (n < 0 || n > kMaxList) return PA_ERR_SHAPE;
  if (n == 0) return PA_OK;
  if (!sequences || !status) return PA_ERR_NULL_ARG;
  hipLaunchKernelGGL(pa_pages_free_kernel, dim3((unsigned)n), dim3(kThreads), 0, (hipStream_t)stream, t, sequences,
                     new_lengths, status);
  return done(hipGetLastError());
}

extern "C" int pa_fp8_extend_pages(const pa_fp8_page_table_args* a, const pa_fp8_page_cache* caches, int num_caches,
                                   const int32_t* sequences, const int32_t* new_lengths, int n, int32_t* status,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  Extend e;
  int rc = table_of(a, &e.t);
  if (rc == PA_OK) rc = check_caches(caches, num_caches, a->num_blocks);
  if (rc != PA_OK) return rc;
  if (n < 0 || n > kMaxExtend) return PA_ERR_SHAPE;
  if (n == 0) return PA_OK;
  if (!sequences || !new_lengths || !status || !workspace) return PA_ERR_NULL_ARG;
  if (workspace_bytes < pa_fp8_pages_workspace_bytes(PA_PAGES_EXTEND, a->num_blocks, n)) return PA_ERR_SCRATCH;
  char* ws = (char*)workspace;
  e.pool = pool_at(ws, a->num_blocks);
  ws += pool_bytes(a->num_blocks);
  const int64_t step = up(4 * (int64_t)n);
  e.start = (int32_t*)ws;
  e.old = (int32_t*)(ws + step);
  e.src = (int32_t*)(ws + 2 * step);
  e.seqs = sequences;
  e.new_lengths = new_lengths;
  e.n = n;
  e.status = status;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(pa_pages_extend_plan_kernel, dim3((unsigned)e.pool.chunks + 1), dim3(kPlanThreads), 0, s, e);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return (int)err;
  int at = 0;
  bool first = true;
  do {
    CopyArgs c = {};
    next_caches(caches, num_caches, &at, &c);
    const int y = pa_max(1, pa_min((c.units + kWaves - 1) / kWaves, kCopyGrid / n));
    hipLaunchKernelGGL(pa_pages_extend_kernel, dim3((unsigned)n, (unsigned)y), dim3(kThreads), 0, s, e, c, first);
    err = hipGetLastError();
    if (err != hipSuccess) return (int)err;
    first = false;
  } while (at < num_caches);
  return PA_OK;
}

extern "C" int pa_fp8_compact_pages(const pa_fp8_page_table_args* a, const pa_fp8_page_cache* caches, int num_caches,
                                    int32_t* new_tables, int64_t stride_new_tables, int32_t* new_refs, int32_t* page_map,
                                    int32_t* live, void* workspace, int64_t workspace_bytes, void* stream) {
  Compact c;
  int rc = table_of(a, &c.t);
  if (rc == PA_OK) rc = check_caches(caches, num_caches, a->num_blocks);
  if (rc != PA_OK) return rc;
  if (!live || !workspace || (a->num_blocks > 0 && (!new_refs || !page_map)) ||
      (a->num_rows > 0 && a->max_blocks_per_seq > 0 && !new_tables))
    return PA_ERR_NULL_ARG;
  if (workspace_bytes < pa_fp8_pages_workspace_bytes(PA_PAGES_COMPACT, a->num_blocks, 0)) return PA_ERR_SCRATCH;
  char* ws = (char*)workspace;
  c.pool = pool_at(ws, a->num_blocks);
  ws += pool_bytes(a->num_blocks);
  const int64_t step = up(4 * (int64_t)a->num_blocks);
  c.src = (int32_t*)ws;
  c.dst = (int32_t*)(ws + step);
  c.moves = (int32_t*)(ws + 2 * step);
  c.new_tables = new_tables;
  c.new_stride = stride_new_tables;
  c.new_refs = new_refs;
  c.map = page_map;
  c.live = live;
  c.page_groups = pa_max(1, (a->num_blocks + kThreads - 1) / kThreads);
  const int64_t grid = (int64_t)c.page_groups + a->num_rows;
  if (grid > 0x7fffffff) return PA_ERR_SHAPE;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(pa_pages_count_kernel, dim3((unsigned)c.pool.chunks), dim3(kPlanThreads), 0, s, c.t.refs, c.t.pages,
                     c.pool);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return (int)err;
  hipLaunchKernelGGL(pa_pages_compact_kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, c);
  err = hipGetLastError();
  if (err != hipSuccess) return (int)err;
  if (a->num_blocks == 0) return PA_OK;
  // at most half of the pages move
  return done(launch_copy(caches, num_caches, c.src, c.dst, c.moves, a->num_blocks / 2 + 1, a->num_blocks, nullptr, true, s));
}
