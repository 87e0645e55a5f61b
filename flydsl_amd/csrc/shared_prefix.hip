// Decode attention of a batch whose sequences share prefixes, for MI355X
// (gfx950): each group's prefix is read once for all of the group's query
// rows, every sequence's own tokens once for its columns, and the parts are
// merged by their maxima and sums:
//   part i of a row:  m_i = max x_j,  l_i = sum 2^(x_j - m_i),
//                     o_i = sum 2^(x_j - m_i) v_j,   x = q.k scale log2(e)
//   out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,   M = max m_i
//
// Work decomposition: see sp_plan.h.  One launch of persistent workgroups
// (four waves, two workgroups a CU) walks equal shares of the line of prefix
// and suffix items and leaves float32 pieces; a second launch merges a row's
// pieces.
//
// Arithmetic.  A wave holds NR tiles of 16 query rows and walks 64-token
// tiles.  Keys and values are fp8 e4m3fn, exact in bf16 and f16, so they are
// converted and both products run on v_mfma_f32_16x16x32_{bf16,f16}:
//   S^T = K Q^T     A: 16 tokens x 32 dims, B: Q^T
//   O^T += V^T P^T  A: 16 dims x 32 tokens, B: P^T
// Row m of key tile T (of four) is token 16 (m / 4) + 4 T + m % 4, so that the
// logits that lane (c, g) = (l % 16, l / 16) gets are those of row c and the
// tokens 16 g + 4 T .. + 3: with all four tiles, or with T = 2 j and 2 j + 1, the
// very tokens 16 g + 8 j .. + 7 that the lane supplies to value product j, and
// the probabilities need no move between lanes.
// The probabilities are rounded to the operands' type, by at most 2^-8 (bf16)
// or 2^-11 (f16) of themselves, as an attention in that type rounds them;
// sums, maxima and outputs stay in 32 bits.
//
// Few rows (run_direct): bound by HBM; a wave's 16-byte loads bring keys (16
// dims of a token; the k order of S is a permutation of the head dimension
// that Q shares) and values (the 16 tokens of block g for one dim) straight
// from the cache's layout into operand registers.
// Many rows (run_shared): bound by the matrix cores, the vector units and LDS
// alike; the workgroup converts each tile once, into LDS in the operands' order,
// while the tile before is computed (two buffers, one barrier a tile).  A tile of
// 128 rows takes a CU 1.4 us; its products alone would take 0.5, its LDS reads and
// writes 0.6, its vector instructions 0.3.  One workgroup a CU is 1.34 times as
// slow; of two the older runs ahead, and holding it back (s_setprio) brought nothing.
//
// Measured, in us (both launches, caches in HBM; in brackets the bytes that have to
// be read and written at 4.9 TB/s, the products at 1.58 PFLOP/s):
//   64 sequences of a 2048-token prefix, 32/8 heads of 128:       33  (16, 2)
//   32 of a 32768-token one:                                      55  (29, 11)
//   256 of a 16383-token one:                                    115  (36, 44)
//   128 of four of 2000 to 12000 tokens, 64/4 heads, four query
//   tokens, per-token scales:                                    214  (38, 90)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <vector>

#include "pa_check.h"
#include "pa_fp8.h"
#include "sp_plan.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 64 * SP_WAVES;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
// A row's reference exponent starts below every logit.
constexpr float kNoKey = -3.0e38f;

// Everything a launch needs (device side of pa_fp8_shared_prefix_args).
struct SpArgs {
  pa_fp8_shared_prefix_args a;
  SpShape p, s;           // prefix and suffix items
  int eq, col_tiles;      // query columns per kv head, suffix items per (sequence, kv head)
  int p_rows, s_rows;     // rows a piece's slot has
  int capacity;           // tokens a table row can hold
  int lbs;                // log2(page size)
  // workspace
  int4* seq_info;         // [B]: first prefix item of the group (-1: none), row of the sequence's first column,
                          // row tiles of the group, whether the sequence has a suffix
  int2* items;            // [prefix items, then suffix items]: first slot, pieces
  int max_prefix_items;
  int prefix_items;       // as many as an even split of the batch over the groups would make
  float* p_ml;            // [slot][2][rows]
  float* p_o;             // [slot][rows][D]
  float* s_ml;
  float* s_o;
};

__device__ __forceinline__ float groups_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Eight fp8 values (two dwords) as an MFMA operand.
template <bool F16>
__device__ __forceinline__ i32x4 widen8(int lo, int hi) {
  union {
    i32x4 v;
    bf16x2 b[4];
    f16x2 h[4];
  } u;
  if constexpr (F16) {
    u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  } else {
    u.b[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    u.b[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    u.b[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    u.b[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  }
  return u.v;
}
template <bool F16>
__device__ __forceinline__ int round2(float x, float y) {
  int r;
  if constexpr (F16) {
    f16x2 h = {(_Float16)x, (_Float16)y};
    __builtin_memcpy(&r, &h, 4);
  } else {
    bf16x2 h = {(__bf16)x, (__bf16)y};
    __builtin_memcpy(&r, &h, 4);
  }
  return r;
}
template <bool F16>
__device__ __forceinline__ f32x4 mfma(const i32x4& x, const i32x4& y, const f32x4& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}

// Byte mask of a dword whose bytes are tokens t .. t + 3: those in [lo, hi).
__device__ __forceinline__ uint32_t keep4(int t, int lo, int hi) {
  const int l = pa_min(pa_max(lo - t, 0), 4), u = pa_min(pa_max(hi - t, l), 4);
  const uint32_t below_u = u >= 4 ? ~0u : (1u << (8 * u)) - 1;
  const uint32_t below_l = l >= 4 ? ~0u : (1u << (8 * l)) - 1;
  return below_u & ~below_l;
}

// ---------------------------------------------------------------------------
// The plan of a launch, in LDS
// ---------------------------------------------------------------------------

struct Plan {
  int64_t* seq_at;    // [B + 1] cost of the sequences' items before b, one kv head
  int64_t* group_at;  // [G + 1] likewise of the groups' prefix items
  int64_t* scratch;   // [SP_WAVES]
  int* ctx;           // [B] context length, at most what a table row holds
  int* begin;         // [B] prefix length of its group
  int* first;         // [G + 1] first sequence of a group (never falls)
  int* len;           // [G + 1] prefix length
  int* row_tiles;     // [G + 1] prefix items of the groups before g, one kv head
};

__host__ __device__ constexpr int plan_bytes(int B, int G) {
  return (8 * (B + 1) + 8 * (G + 1) + 8 * SP_WAVES + 8 * B + 12 * (G + 1) + 15) & ~15;
}
__device__ __forceinline__ Plan plan_of(char* lds, int B, int G) {
  Plan p;
  p.seq_at = (int64_t*)lds;
  p.group_at = p.seq_at + B + 1;
  p.scratch = p.group_at + G + 1;
  p.ctx = (int*)(p.scratch + SP_WAVES);
  p.begin = p.ctx + B;
  p.first = p.begin + B;
  p.len = p.first + G + 1;
  p.row_tiles = p.len + G + 1;
  return p;
}

// Inclusive sums (MAX: maxima) over the wave's first `lanes` lanes.
template <bool MAX, typename T>
__device__ __forceinline__ T wave_upto(T v, int lanes = 64) {
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < lanes; d *= 2) {
    const T o = sizeof(T) == 8 ? (T)__shfl_up((long long)v, d, 64) : (T)__shfl_up((int)v, d, 64);
    if (lane >= d) v = MAX ? (o > v ? o : v) : v + o;
  }
  return v;
}

// a[0 .. n] := the sums (MAX: a[0 .. n - 1] := the maxima, inclusive) of what
// stands before each entry; the workgroup calls it with a[] written and visible.
template <bool MAX, typename T>
__device__ void block_scan(T* a, int n, int64_t* scratch) {
  const int per = (n + kThreads - 1) / kThreads;
  const int i0 = threadIdx.x * per, i1 = pa_min(i0 + per, n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T mine = 0;
  for (int i = i0; i < i1; ++i) mine = MAX ? (a[i] > mine ? a[i] : mine) : mine + a[i];
  const T upto = wave_upto<MAX>(mine);
  if (lane == 63) scratch[wave] = (int64_t)upto;
  T before = sizeof(T) == 8 ? (T)__shfl_up((long long)upto, 1, 64) : (T)__shfl_up((int)upto, 1, 64);
  if (lane == 0) before = 0;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    const T o = (T)scratch[w];
    before = MAX ? (o > before ? o : before) : before + o;
  }
  for (int i = i0; i < i1; ++i) {
    const T v = a[i];
    if (MAX) {
      before = v > before ? v : before;
      a[i] = before;
    } else {
      a[i] = before;
      before += v;
    }
  }
  if (!MAX && i0 < n && i1 == n) a[n] = before;
  if (!MAX && n == 0 && threadIdx.x == 0) a[0] = 0;
  __syncthreads();
}

// Last entry of a[0 .. n] (never falls) that, times k, is <= x, for a[0] = 0 or <= x.
template <typename T>
__device__ __forceinline__ int last_le(const T* a, int n, int64_t x, int k = 1) {
  int lo = 0, hi = n + 1;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (k * (int64_t)a[m] <= x)
      lo = m;
    else
      hi = m;
  }
  return lo;
}

// The group of sequence b, or -1.
__device__ __forceinline__ int group_of(const Plan& p, int G, int b) {
  if (G <= 0 || b < p.first[0] || b >= p.first[G]) return -1;
  return last_le(p.first, G, b);
}

// Prefix length, prefix items and their cost of group g, whose first[] is set.
__device__ __forceinline__ void plan_group(const SpArgs& s, int sequences, int given, int* len, int* tiles, int64_t* cost) {
  const int rows = sequences * s.eq;
  *len = rows > 0 ? pa_min(pa_max(given, 0), s.capacity) : 0;
  *tiles = *len > 0 ? pa_cdiv(rows, s.p.rows) : 0;
  *cost = (int64_t)*tiles * sp_item_cost(s.p, sp_tiles(0, *len));
}

// Every workgroup makes the whole plan, in 2.4 us from the launch (one round of
// loads, a few barriers); a launch of its own would take those and a start more.
__device__ void make_plan(const Plan& p, const SpArgs& s) {
  const int B = s.a.num_seqs, G = s.a.num_groups;
  int f = 0, given = 0;  // asked for before anything waits
  if (threadIdx.x < 64 && G < 64) {
    if (G > 0 && (int)threadIdx.x <= G) f = s.a.prefix_indptr[threadIdx.x];
    if ((int)threadIdx.x < G) given = s.a.prefix_lengths[threadIdx.x];
  }
  for (int b = threadIdx.x; b < B; b += kThreads) {
    const int n = s.a.context_lengths[b];
    p.ctx[b] = n < 0 ? 0 : (n < s.capacity ? n : s.capacity);
  }
  if (G < 64) {  // the groups in one wave's lanes
    if (threadIdx.x < 64) {
      const int g = threadIdx.x;
      f = wave_upto<true>(pa_min(pa_max(f, 0), B), G + 1);
      const int next = __shfl_down(f, 1, 64);
      int len = 0, tiles = 0;
      int64_t cost = 0;
      if (g < G) plan_group(s, next - f, given, &len, &tiles, &cost);
      const int tiles_upto = wave_upto<false>(tiles, G + 1);
      const int64_t cost_upto = wave_upto<false>(cost, G + 1);
      if (g <= G) {
        p.first[g] = f;
        p.len[g] = len;
        p.row_tiles[g] = tiles_upto - tiles;
        p.group_at[g] = cost_upto - cost;
      }
    }
    __syncthreads();
  } else {
    for (int g = threadIdx.x; g <= G; g += kThreads) {
      p.first[g] = pa_min(pa_max(s.a.prefix_indptr[g], 0), B);
      p.len[g] = g < G ? s.a.prefix_lengths[g] : 0;
    }
    __syncthreads();
    block_scan<true>(p.first, G + 1, p.scratch);
    for (int g = threadIdx.x; g < G; g += kThreads) {
      int len, tiles;
      int64_t cost;
      plan_group(s, p.first[g + 1] - p.first[g], p.len[g], &len, &tiles, &cost);
      p.len[g] = len;
      p.row_tiles[g] = tiles;
      p.group_at[g] = cost;
    }
    __syncthreads();
    block_scan<false>(p.row_tiles, G, p.scratch);
    block_scan<false>(p.group_at, G, p.scratch);
  }
  const int per = (B + kThreads - 1) / kThreads;  // (block_scan's own split: no barrier between)
  for (int b = threadIdx.x * per; b < pa_min((int)(threadIdx.x + 1) * per, B); ++b) {
    const int g = group_of(p, G, b);
    const int len = g >= 0 ? p.len[g] : 0;
    p.begin[b] = len;
    p.seq_at[b] = (int64_t)s.col_tiles * sp_item_cost(s.s, sp_tiles(len, p.ctx[b]));
  }
  block_scan<false>(p.seq_at, B, p.scratch);
}

// ---------------------------------------------------------------------------
// One piece
// ---------------------------------------------------------------------------

struct Piece {
  bool of_prefix;     // a prefix item's
  int b0;            // sequence whose table row gives the pages, and of the item's row 0
  int row0, nrows;   // first row of the item among the group's rows (the sequence's columns), and their count
  int h;             // kv head
  int begin, end;    // tokens of the item
  int seen;          // the first token behind those that any of its rows sees or that its sequences hold
  int tile, tile_end;  // tiles of the piece
  int rows_out;      // rows of a slot
  float* ml;         // the slot
  float* o;
};

// The pieces of the line's region [from, to) whose tiles begin in [lo, hi), the
// part of `worker`, as long as `share`: a workgroup's or a wave's.
struct Walk {
  int64_t suffix_at, lo, hi, stop, share, at;  // suffix_at: where the suffix items begin; at: of item idx
  int worker, of, idx;                           // `of` a group or a sequence, idx the item among its own (kv head
                                                 // outer, row tile inner); -1: not looked up yet; INT_MAX: no more
  bool prefix;

  __device__ __forceinline__ void start(const SpArgs& s, const Plan& pl, int64_t suffix_at_, int64_t from, int64_t to,
                                        int64_t lo_, int64_t share_, int worker_) {
    suffix_at = suffix_at_;
    lo = lo_;
    share = share_;
    hi = lo + share;
    worker = worker_;
    at = lo > from ? lo : from;
    stop = hi < to ? hi : to;
    idx = -1;
    of = 0;
    const int H = s.a.num_kv_heads;
    prefix = at < (int64_t)H * pl.group_at[s.a.num_groups];
    if (at >= stop) {
      idx = 0x7fffffff;
      return;
    }
    of = __builtin_amdgcn_readfirstlane(prefix ? last_le(pl.group_at, s.a.num_groups, at, H)
                                               : last_le(pl.seq_at, s.a.num_seqs, at - suffix_at, H));
  }

  // The next piece; false when there is none.  ALONE: a wave's (its lane 0 tells
  // the merge of it).
  __device__ __forceinline__ bool next_piece(const SpArgs& s, const Plan& pl, int D, bool alone, Piece& pc) {
    const int B = s.a.num_seqs, G = s.a.num_groups, H = s.a.num_kv_heads;
    while (idx != 0x7fffffff) {
      const SpShape& sh = prefix ? s.p : s.s;
      int begin = 0, end, tiles;
      if (prefix) {
        tiles = pl.row_tiles[of + 1] - pl.row_tiles[of];
        end = pl.len[of];
      } else {
        tiles = s.col_tiles;
        begin = pl.begin[of];
        end = pl.ctx[of];
      }
      tiles = __builtin_amdgcn_readfirstlane(tiles);
      begin = __builtin_amdgcn_readfirstlane(begin);
      end = __builtin_amdgcn_readfirstlane(end);
      const int n = sp_tiles(begin, end), cost = sp_item_cost(sh, n);
      if (idx < 0) {
        const int64_t of_at = prefix ? (int64_t)H * pl.group_at[of] : suffix_at + (int64_t)H * pl.seq_at[of];
        idx = __builtin_amdgcn_readfirstlane(sp_worker_of(at - of_at, cost));
        at = of_at + (int64_t)idx * cost;
      }
      while (idx < H * tiles && at < stop) {
        // (no division for an item that lies inside the part)
        const int t0 = at + sh.overhead >= lo ? 0 : __builtin_amdgcn_readfirstlane(sp_tile_from(sh, lo, at, n));
        const int t1 = at + cost <= hi ? n : __builtin_amdgcn_readfirstlane(sp_tile_from(sh, hi, at, n));
        const int i = idx;
        const int64_t i_at = at;
        ++idx;
        at += cost;
        if (t1 <= t0) continue;
        const int item = __builtin_amdgcn_readfirstlane(prefix ? H * pl.row_tiles[of] + i : of * H * tiles + i);
        const int slot = item + worker;
        pc.of_prefix = prefix;
        pc.b0 = prefix ? __builtin_amdgcn_readfirstlane(pl.first[of]) : of;
        pc.h = tiles == 1 ? i : i / tiles;
        pc.row0 = (i - pc.h * tiles) * sh.rows;
        pc.nrows = prefix ? __builtin_amdgcn_readfirstlane((pl.first[of + 1] - pl.first[of]) * s.eq) : s.eq;
        pc.begin = begin;
        pc.end = end;
        pc.seen = end;
        if (prefix) {
          int most = 0;
          const int b1 = (pa_min(pc.row0 + sh.rows, pc.nrows) - 1) / s.eq;
          for (int b = pc.row0 / s.eq + (int)(threadIdx.x & 63); b <= b1; b += 64) most = pa_max(most, pl.ctx[pc.b0 + b]);
          for (int d = 1; d < 64; d *= 2) most = pa_max(most, __shfl_xor(most, d, 64));
          pc.seen = __builtin_amdgcn_readfirstlane(pa_min(end, most));
        }
        pc.tile = begin / SP_TILE + t0;
        pc.tile_end = begin / SP_TILE + t1;
        pc.rows_out = prefix ? s.p_rows : s.s_rows;
        pc.ml = (prefix ? s.p_ml : s.s_ml) + (int64_t)slot * 2 * pc.rows_out;
        pc.o = (prefix ? s.p_o : s.s_o) + (int64_t)slot * pc.rows_out * D;
        if (t0 == 0 && (alone ? (threadIdx.x & 63) : threadIdx.x) == 0) {
          const int last = t1 == n ? worker : sp_worker_of(i_at + sh.overhead + (int64_t)(n - 1) * sh.cost, share);
          s.items[prefix ? item : s.max_prefix_items + item] = int2{slot, last - worker + 1};
        }
        return true;
      }
      if (at >= stop) break;
      // on to the next group or sequence that has items
      idx = 0;
      ++of;
      if (prefix) {
        while (of < G && pl.group_at[of + 1] == pl.group_at[of]) ++of;
        if (of >= G) {
          prefix = false;
          of = 0;
          at = suffix_at;
          if (at >= stop) break;
        }
      }
      if (!prefix)
        while (of < B && pl.seq_at[of + 1] == pl.seq_at[of]) ++of;
      of = __builtin_amdgcn_readfirstlane(of);
      if (!prefix && of >= B) break;
    }
    idx = 0x7fffffff;
    return false;
  }
};

// LDS behind the plan, of shared items: two buffers of a tile, or, at a piece's
// end, maxima, sums and outputs of every wave's rows.
__host__ __device__ constexpr int out_stride(int d) { return d + 4; }  // floats (16-byte steps that spread over the banks)
__host__ __device__ constexpr int end_bytes(int d, int nr) { return SP_WAVES * 16 * nr * (2 + out_stride(d)) * 4; }

// The wave's rows: operand B of the key product, the keys each row sees, and
// their softmax.
//
// Softmax.  A row's probabilities are 2^(x - m) against a reference m, and its sum
// and outputs in the same units.  m need not be the maximum: it only has to keep
// the probabilities in range, and is moved, by the maximum of the tokens at hand,
// when one of them reaches 2 -- seen by the exponent's top bit in the OR of
// all of them, four instructions in place of the maximum's forty.  A move sets
// m so that the largest probability is 2^-8 (f16 operands: 1, for their range), and
// most rows move once.  The sum is one more row of the value product, of ones
// (where the operand is the probability alone, without per-token value scales).
template <int D, bool F16, bool PT, int NR>
struct Rows {
  static constexpr bool PF16 = F16 && !PT;  // f16 probabilities; with per-token scales bf16: a scale of any size times a
                                            // probability stays in range
  static constexpr float kHead = PF16 ? 0.0f : 8.0f;
  i32x4 q[NR][D / 32];
  f32x4 o[NR][D / 16];
  f32x4 sum[NR];  // [0] (and, without per-token scales, all): of the row; with them the lane's part
  float m[NR];
  int limit[NR];  // keys a row sees: below it
  int least;      // of all of the wave's
  float fac;      // of a raw logit, positive
  int flip, keep; // bits of a query value to turn or keep: a negative scale's sign, a zero scale

  __device__ __forceinline__ void set_scale(const SpArgs& s) {
    const float c0 = s.a.softmax_scale * kLog2e * (PT ? 1.0f : s.a.key_scale[0]);
    fac = c0 == 0.0f ? 1.0f : fabsf(c0);
    flip = c0 < 0.0f ? (int)0x80008000u : 0;
    keep = c0 == 0.0f ? 0 : -1;
  }
  // Row n's operand: 16-byte pieces k of the row, of 8 dims each.  DIMS16: a lane's
  // k order is 16 dims of two steps (run_direct), else 8 of each.
  template <bool DIMS16>
  __device__ __forceinline__ void load_query(const SpArgs& s, const Piece& pc, int r, int g, i32x4 (&x)[D / 32]) const {
    const pa_fp8_shared_prefix_args& a = s.a;
    const bool live = r < pc.nrows;
    const int bb = live ? r / s.eq : 0, e = live ? r - bb * s.eq : 0, qi = e / a.query_group_size;
    const uint16_t* row = (const uint16_t*)a.query +
                          ((int64_t)(pc.b0 + bb) * a.query_length + qi) * a.stride_q_tok +
                          (int64_t)(pc.h * a.query_group_size + (e - qi * a.query_group_size)) * a.stride_q_head;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      x[k] = i32x4{0, 0, 0, 0};
      if (live) x[k] = *(const i32x4*)(row + (DIMS16 ? (4 * (k >> 1) + g) * 16 + 8 * (k & 1) : 32 * k + 8 * g));
    }
  }
  // Row n begins, as row r of the piece's item, with operand x.
  __device__ __forceinline__ void begin(const SpArgs& s, const Piece& pc, const int* ctx, int n, int r,
                                        const i32x4 (&x)[D / 32]) {
    const bool live = r < pc.nrows;
    const int bb = live ? r / s.eq : 0, qi = live ? (r - bb * s.eq) / s.a.query_group_size : 0;
    limit[n] = live ? pa_min(pa_max(ctx[pc.b0 + bb] - s.a.query_length + qi + 1, 0), pc.end) : 0x7fffffff;
    if (n == 0 || limit[n] < least) least = limit[n];
    if (n == NR - 1) {
#pragma unroll
      for (int d = 1; d < 16; d *= 2) least = pa_min(least, __shfl_xor(least, d, 64));
      least = __builtin_amdgcn_readfirstlane(least);
    }
#pragma unroll
    for (int k = 0; k < D / 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) q[n][k][i] = (x[k][i] ^ flip) & keep;
    m[n] = kNoKey;
    sum[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[n][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Probabilities of row n's logits of two key tiles.
  __device__ __forceinline__ void exponentials(int n, const f32x4& x0, const f32x4& x1, float (&e)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(i < 4 ? x0[i] : x1[i - 4], fac, -m[n]));
  }
  static __device__ __forceinline__ i32x4 pack(const float (&e)[8]) {
    return i32x4{round2<PF16>(e[0], e[1]), round2<PF16>(e[2], e[3]), round2<PF16>(e[4], e[5]), round2<PF16>(e[6], e[7])};
  }

  // The value product's operands for logits x0, x1 of every row.
  __device__ __forceinline__ void weights(const f32x4 (&x0)[NR], const f32x4 (&x1)[NR], const f32x4& vs0, const f32x4& vs1,
                                          i32x4 (&p)[NR]) {
    float e[NR][8];
    uint32_t high = 0;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      exponentials(n, x0[n], x1[n], e[n]);
      if constexpr (PT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) high |= __float_as_uint(e[n][i]);
      } else {
        p[n] = pack(e[n]);
        high |= (uint32_t)(p[n][0] | p[n][1] | p[n][2] | p[n][3]);
      }
    }
    if (__ballot((high & (PT ? 0x40000000u : 0x40004000u)) != 0)) {
      move(x0, x1);
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        exponentials(n, x0[n], x1[n], e[n]);
        if constexpr (!PT) p[n] = pack(e[n]);
      }
    }
    if constexpr (PT) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        sum[n][0] += ((e[n][0] + e[n][1]) + (e[n][2] + e[n][3])) + ((e[n][4] + e[n][5]) + (e[n][6] + e[n][7]));
#pragma unroll
        for (int i = 0; i < 8; ++i) e[n][i] *= i < 4 ? vs0[i] : vs1[i - 4];
        p[n] = pack(e[n]);
      }
    }
  }

  // Moves the references of rows that x takes past them.
  __device__ __forceinline__ void move(const f32x4 (&x0)[NR], const f32x4 (&x1)[NR]) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float top = kNegInf;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(fmaxf(x0[n][i], x1[n][i]), top);
      top = groups_max(top) * fac;
      const float to = top >= m[n] + 0.5f ? top + kHead : m[n];
      const float f = __builtin_amdgcn_exp2f(m[n] - to);
      m[n] = to;
      sum[n] *= f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) o[n][dt] *= f;
    }
  }
  // The value product's row of ones.
  __device__ __forceinline__ void add_sums(const i32x4 (&p)[NR]) {
    if constexpr (!PT) {
      constexpr int one = PF16 ? 0x3c003c00 : 0x3f803f80;
#pragma unroll
      for (int n = 0; n < NR; ++n) sum[n] = mfma<PF16>(i32x4{one, one, one, one}, p[n], sum[n]);
    }
  }
  __device__ __forceinline__ float row_sum(int n) const { return PT ? groups_sum(sum[n][0]) : sum[n][0]; }
  __device__ __forceinline__ float row_max(int n) const { return m[n] == kNoKey ? kNegInf : m[n]; }

  // Writes a piece that one wave worked alone.
  __device__ __forceinline__ void finish_alone(const Piece& pc, int c, int g) {
    static_assert(NR == 1, "one row tile");
    const float l = row_sum(0);
    if (pc.row0 + c >= pc.nrows) return;
    if (g == 0) {
      pc.ml[c] = row_max(0);
      pc.ml[pc.rows_out + c] = l;
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *(f32x4*)(pc.o + (int64_t)c * D + 16 * dt + 4 * g) = o[0][dt];
  }

  // Joins the waves of the same rows (wt of them, this one the wi-th) and writes
  // the piece.
  __device__ __forceinline__ void finish(const Piece& pc, char* lds, int wt, int wave, int wr, int wi, int c, int g) {
    float* lm = (float*)lds;              // [wave][16 NR]
    float* ll = lm + SP_WAVES * 16 * NR;
    float* lo = ll + SP_WAVES * 16 * NR;  // [wave][16 NR][out_stride]
    __syncthreads();                      // what LDS held before has been read
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const float l = row_sum(n);
      if (g == 0) {
        lm[(wave * NR + n) * 16 + c] = row_max(n);
        ll[(wave * NR + n) * 16 + c] = l;
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float top = kNegInf, all = 0.0f;
      for (int w = wr * wt; w < (wr + 1) * wt; ++w) top = fmaxf(top, lm[(w * NR + n) * 16 + c]);
      for (int w = wr * wt; w < (wr + 1) * wt; ++w) {
        const float mw = lm[(w * NR + n) * 16 + c];
        // (a wave that saw no key has 0 or, where its logits were NaN, NaN)
        all += ll[(w * NR + n) * 16 + c] * (mw == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mw - top));
      }
      const float f = m[n] == kNoKey ? 0.0f : __builtin_amdgcn_exp2f(m[n] - top);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) o[n][dt] *= f;
      const int r = (wr * NR + n) * 16 + c;
      if (wi == 0 && g == 0 && pc.row0 + r < pc.nrows) {
        pc.ml[r] = top;
        pc.ml[pc.rows_out + r] = all;
      }
    }
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
        *(f32x4*)(lo + ((wave * NR + n) * 16 + c) * out_stride(D) + 16 * dt + 4 * g) = o[n][dt];
    __syncthreads();
    // whole rows, so that a wave's stores are of whole kilobytes
    const int rows = pa_min(SP_WAVES / wt * 16 * NR, pc.nrows - pc.row0);
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      const int w0 = r / (16 * NR) * wt, rr = r % (16 * NR);
      f32x4 v = *(const f32x4*)(lo + (w0 * 16 * NR + rr) * out_stride(D) + d);
      if (wt == 2) v += *(const f32x4*)(lo + ((w0 + 1) * 16 * NR + rr) * out_stride(D) + d);
      *(f32x4*)(pc.o + 4 * i) = v;
    }
    __syncthreads();  // LDS is the next piece's
  }
};

// The item's pages: of a token (the same one in every lane), inside the cache and
// the table row whatever the caller's table holds.  Scalar loads -- the launch
// writes no table -- which wait by a counter of their own, so that the loads of
// keys and values under way are not waited for.
struct Pages {
  const int32_t* table;
  int last, lbs, blocks;
  __device__ __forceinline__ Pages(const SpArgs& s, const Piece& pc)
      : table(s.a.block_tables + (int64_t)pc.b0 * s.a.stride_bt_seq),
        last(pa_min((pc.end - 1) >> s.lbs, s.a.max_blocks_per_seq - 1)),
        lbs(s.lbs),
        blocks(s.a.num_blocks) {}
  __device__ __forceinline__ int entry(int token) const {  // as it stands
    const int i = __builtin_amdgcn_readfirstlane(pa_min(token >> lbs, last));
    return ((const __attribute__((address_space(4))) int32_t*)table)[i];
  }
  __device__ __forceinline__ static int inside(int p, int blocks) {
    pa_note(p < 0 || p >= blocks, PA_VIOLATION_PAGE);
    p = p < 0 ? 0 : p;
    return p < blocks ? p : blocks - 1;
  }
  __device__ __forceinline__ int operator()(int token) const { return inside(entry(token), blocks); }
};

// A piece worked by one wave.
template <int D, bool F16, bool PT>
__device__ __forceinline__ void run_direct(const SpArgs& s, const Piece& pc, const int* ctx) {
  constexpr bool PF16 = F16 && !PT;
  const pa_fp8_shared_prefix_args& a = s.a;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int bs = 1 << s.lbs;
  const Pages page_of(s, pc);
  const uint8_t* kbase = (const uint8_t*)a.key_cache + (int64_t)pc.h * a.stride_k_head;
  const uint8_t* vbase = (const uint8_t*)a.value_cache + (int64_t)pc.h * a.stride_v_head;
  const int v_dim = a.trans_v ? 16 : bs, v_blk = a.trans_v ? D * 16 : 16;
  const int kblk = c >> 2;  // the lane's key tokens are of block kblk, its value tokens of block g
  // Two tiles in flight (one beside per-token scales), in registers: a wave alone
  // has no one else to wait with.
  constexpr int kAhead = PT ? 1 : 2;
  struct Tile {
    i32x4 k[4][D / 64], v[D / 16];
  };
  Tile even, odd;
  f32x4 ks[4], vs[4];
  const int last = pc.tile_end - 1;
  int entry[4];  // table entries of the tile to be loaded next, by token block
  auto entries = [&](int tile) {
#pragma unroll
    for (int i = 0; i < 4; ++i) entry[i] = page_of.entry(pa_min(tile, last) * SP_TILE + 16 * i);
  };
  auto page = [&](int blk) {  // of the lane's block
    int p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = Pages::inside(entry[i], a.num_blocks);
    return blk < 2 ? (blk == 0 ? p[0] : p[1]) : (blk == 2 ? p[2] : p[3]);
  };
  auto load_keys = [&](Tile& x, int tile) {
    const int in = ((tile * SP_TILE + 16 * kblk) & (bs - 1)) + (c & 3);
    const uint8_t* p = kbase + (int64_t)page(kblk) * a.stride_k_block + in * 16 + g * (bs * 16);
#pragma unroll
    for (int T = 0; T < 4; ++T)
#pragma unroll
      for (int u = 0; u < D / 64; ++u) x.k[T][u] = *(const i32x4*)(p + 64 * T + (int64_t)(4 * u) * (bs * 16));
  };
  auto load_values = [&](Tile& x, int tile) {
    const int in = ((tile * SP_TILE + 16 * g) & (bs - 1)) >> 4;
    const uint8_t* p = vbase + (int64_t)page(g) * a.stride_v_block + in * v_blk + c * v_dim;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) x.v[dt] = *(const i32x4*)(p + (int64_t)(16 * dt) * v_dim);
  };
  auto load_scales = [&](const float* base, int tile, f32x4 (&x)[4]) {
    const float* p = base + (int64_t)page(g) * a.stride_ks_block + (int64_t)pc.h * a.stride_ks_head +
                     ((tile * SP_TILE + 16 * g) & (bs - 1));
#pragma unroll
    for (int T = 0; T < 4; ++T) x[T] = *(const f32x4*)(p + 4 * T);
  };

  Rows<D, F16, PT, 1> w;
  w.set_scale(s);
  entries(pc.tile);
  i32x4 q[D / 32];
  w.template load_query<true>(s, pc, pc.row0 + c, g, q);
  load_keys(even, pc.tile);
  load_values(even, pc.tile);
  if constexpr (PT) {
    load_scales(a.key_scale, pc.tile, ks);
    load_scales(a.value_scale, pc.tile, vs);
  }
  entries(pc.tile + 1);
  if (kAhead == 2 && pc.tile < last) {
    load_keys(odd, pc.tile + 1);
    load_values(odd, pc.tile + 1);
    entries(pc.tile + 2);
  }
  w.begin(s, pc, ctx, 0, pc.row0 + c, q);
  // tile from x, tile + kAhead into it
  auto step = [&](Tile& x, int tile) {
    const bool more = tile + kAhead <= last;
    f32x4 l[4][1];
#pragma unroll
    for (int T = 0; T < 4; ++T) {
      l[T][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < D / 64; ++u) {
        l[T][0] = mfma<F16>(widen8<F16>(x.k[T][u][0], x.k[T][u][1]), w.q[0][2 * u], l[T][0]);
        l[T][0] = mfma<F16>(widen8<F16>(x.k[T][u][2], x.k[T][u][3]), w.q[0][2 * u + 1], l[T][0]);
      }
    }
    if (more) load_keys(x, tile + kAhead);
    if constexpr (PT) {
#pragma unroll
      for (int T = 0; T < 4; ++T) l[T][0] *= ks[T];
      if (more) load_scales(a.key_scale, tile + 1, ks);
    }
    // ---- masks: the part's first and last tiles ----
    const int t0 = tile * SP_TILE;
    if (t0 < pc.begin || t0 + SP_TILE > pa_min(w.least, pc.seen)) {
      asm volatile("");  // (a branch: not computed for every tile)
#pragma unroll
      for (int T = 0; T < 4; ++T)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = t0 + 16 * g + 4 * T + i;
          if (t < pc.begin || t >= w.limit[0]) l[T][0][i] = kNegInf;
        }
      // bytes behind the tokens may be anything, NaN among it
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int keep = (int)keep4(t0 + 16 * g + 4 * i, pc.begin, pc.seen);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) x.v[dt][i] &= keep;
      }
      if constexpr (PT) {
#pragma unroll
        for (int T = 0; T < 4; ++T)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = t0 + 16 * g + 4 * T + i;
            if (t < pc.begin || t >= pc.seen) vs[T][i] = 0.0f;
          }
      }
    }
    i32x4 p[1];
    w.weights(l[0], l[1], vs[0], vs[1], p);
    w.add_sums(p);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) w.o[0][dt] = mfma<PF16>(widen8<PF16>(x.v[dt][0], x.v[dt][1]), p[0], w.o[0][dt]);
    w.weights(l[2], l[3], vs[2], vs[3], p);
    w.add_sums(p);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) w.o[0][dt] = mfma<PF16>(widen8<PF16>(x.v[dt][2], x.v[dt][3]), p[0], w.o[0][dt]);
    if (more) {
      load_values(x, tile + kAhead);
      if constexpr (PT) load_scales(a.value_scale, tile + 1, vs);
      entries(tile + kAhead + 1);
    }
  };
  for (int tile = pc.tile; tile <= last; ++tile) {
    step(even, tile);
    if constexpr (kAhead == 2) {
      if (++tile > last) break;
      step(odd, tile);
    }
  }
  w.finish_alone(pc, c, g);
}

// A tile in LDS, 16-byte pieces: keys [D / 8 octets of dims][64 rows of the key
// tiles], values [8 octets of tokens][D dims].  An operand read takes 16
// consecutive pieces a lane group; the key tiles of an octet stand 320 bytes
// apart, so that a wave's writes of a block's tokens (four of each key tile)
// meet different banks.
constexpr int kKeyTile = 320 / 16, kKeyRow = 4 * kKeyTile;  // pieces
__host__ __device__ constexpr int tile_bytes(int d) {
  return d / 8 * kKeyRow * 16 + SP_TILE * d * 2 + 2 * SP_TILE * 4;
}

__host__ __device__ constexpr int work_bytes(int d, bool shared) {
  return shared ? 2 * tile_bytes(d) : 0;
}

constexpr bool lds_fits(int d, int seqs) { return plan_bytes(seqs, seqs / 4) + work_bytes(d, true) <= 160 * 1024; }
static_assert(lds_fits(64, 4096) && lds_fits(128, 4096) && lds_fits(192, 2048) && lds_fits(256, 512), "sp_max_seqs");

// Masks of the scheduling groups.
constexpr int kSchedAlu = 0x2, kSchedMfma = 0x8, kSchedDsRead = 0x100, kSchedDsWrite = 0x200;

template <int D, bool F16, bool PT, int NR, int WT>
__device__ __forceinline__ void run_shared(const SpArgs& s, const Piece& pc, const int* ctx, char* lds) {
  constexpr bool PF16 = F16 && !PT;
  constexpr int NT = 4 / WT, NJ = 2 / WT;  // the wave's key tiles and value products
  constexpr int NS = D / 64;               // pieces of keys, and of values, that a thread brings
  const pa_fp8_shared_prefix_args& a = s.a;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / WT, wi = wave % WT;
  const int bs = 1 << s.lbs;

  // Wave w brings token block w of each tile: one page, so its addresses are
  // scalar but for a lane's constant offset.  Of the keys, lane (c, g) has token c
  // and dims 16 (g + 4 i) .. + 15; of the values, dims lane + 64 i; of the scales,
  // token c of the keys' (g = 0) or the values' (g = 1).
  const Pages page_of(s, pc);
  const uint8_t* kbase = (const uint8_t*)a.key_cache + (int64_t)pc.h * a.stride_k_head;
  const uint8_t* vbase = (const uint8_t*)a.value_cache + (int64_t)pc.h * a.stride_v_head;
  const int64_t s_head = (int64_t)pc.h * a.stride_ks_head;
  const int v_dim = a.trans_v ? 16 : bs, v_blk = a.trans_v ? D * 16 : 16;
  const uint32_t k_lane = (uint32_t)(c * 16 + g * (bs * 16)), v_lane = (uint32_t)(lane * v_dim);
  const uint32_t k_step = (uint32_t)(bs * 64), v_step = (uint32_t)(64 * v_dim);
  i32x4 kst[NS], vst[NS];
  float sst = 0.0f;
  const int last = pc.tile_end - 1;
  auto page_at = [&](int tile) { return page_of.entry(pa_min(tile, last) * SP_TILE + 16 * wave); };
  auto fetch = [&](int tile, int entry) {
    const int page = Pages::inside(entry, a.num_blocks);
    const int in = (tile * SP_TILE + 16 * wave) & (bs - 1);
    const uint8_t* kp = kbase + (int64_t)page * a.stride_k_block + in * 16;
    const uint8_t* vp = vbase + (int64_t)page * a.stride_v_block + (in >> 4) * v_blk;
#pragma unroll
    for (int i = 0; i < NS; ++i) kst[i] = *(const i32x4*)(kp + (k_lane + i * k_step));
#pragma unroll
    for (int i = 0; i < NS; ++i) vst[i] = *(const i32x4*)(vp + (v_lane + i * v_step));
    if constexpr (PT) {
      const int64_t at = (int64_t)page * a.stride_ks_block + s_head + in;
      if (g < 2) sst = (g ? a.value_scale : a.key_scale)[at + c];
    }
  };
  auto mask = [&](int tile) {
    const int t0 = tile * SP_TILE;
    if (t0 < pc.begin || t0 + SP_TILE > pc.seen) {  // bytes behind the tokens may be anything, NaN among it
      asm volatile("");
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int keep = (int)keep4(t0 + 16 * wave + 4 * k, pc.begin, pc.seen);
#pragma unroll
        for (int i = 0; i < NS; ++i) vst[i][k] &= keep;
      }
      if constexpr (PT) {
        const int t = t0 + 16 * wave + c;
        if (t < pc.begin || t >= pc.seen) sst = 0.0f;
      }
    }
  };
  auto store = [&](int buffer) {
    i32x4* lk = (i32x4*)(lds + buffer * tile_bytes(D));
    i32x4* lv = lk + D / 8 * kKeyRow;
    const int row = (c >> 2) * kKeyTile + 4 * wave + (c & 3);  // row 4 wave + c % 4 of key tile c / 4
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int o8 = 2 * (g + 4 * i);
      lk[o8 * kKeyRow + row] = widen8<F16>(kst[i][0], kst[i][1]);
      lk[(o8 + 1) * kKeyRow + row] = widen8<F16>(kst[i][2], kst[i][3]);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int at = 2 * wave * D + lane + 64 * i;
      lv[at] = widen8<PF16>(vst[i][0], vst[i][1]);
      lv[at + D] = widen8<PF16>(vst[i][2], vst[i][3]);
    }
    if constexpr (PT) {
      if (g < 2) ((float*)(lv + SP_TILE * D / 8))[g * SP_TILE + 16 * wave + c] = sst;
    }
  };

  // (two rounds of loads: table entries and queries, then the first tile)
  int entry = page_at(pc.tile), entry1 = page_at(pc.tile + 1);
  Rows<D, F16, PT, NR> w;
  w.set_scale(s);
  {
    i32x4 x[NR][D / 32];
#pragma unroll
    for (int n = 0; n < NR; ++n) w.template load_query<false>(s, pc, pc.row0 + (wr * NR + n) * 16 + c, g, x[n]);
    fetch(pc.tile, entry);
#pragma unroll
    for (int n = 0; n < NR; ++n) w.begin(s, pc, ctx, n, pc.row0 + (wr * NR + n) * 16 + c, x[n]);
  }
  entry = page_at(pc.tile + 2);
  mask(pc.tile);
  store(0);
  fetch(pa_min(pc.tile + 1, last), entry1);
  __syncthreads();
  int buffer = 0;
  for (int tile = pc.tile; tile < pc.tile_end; ++tile, buffer ^= 1) {
    const i32x4* lk = (const i32x4*)(lds + buffer * tile_bytes(D));
    const i32x4* lv = lk + D / 8 * kKeyRow;
    const float* lsc = (const float*)(lv + SP_TILE * D / 8);
    // Operand reads run a step ahead of the products, the first value product's
    // behind the keys' (left to itself, the compiler waits out the latency of
    // every read).
    constexpr int K = D / 32, VA = D / 16, VP = D <= 128 ? VA / 2 : VA / 4;
    f32x4 x[NT][NR], vs[2];
    i32x4 kf[K][NT], vf[VA];
    auto read_keys = [&](int k) {
#pragma unroll
      for (int t = 0; t < NT; ++t) kf[k][t] = lk[(4 * k + g) * kKeyRow + (wi * NT + t) * kKeyTile + c];
    };
    read_keys(0);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      __builtin_amdgcn_sched_barrier(0);
      if (k + 1 < K) {
        read_keys(k + 1);
      } else {
#pragma unroll
        for (int dt = 0; dt < VP; ++dt) vf[dt] = lv[(2 * g + wi * NJ) * D + 16 * dt + c];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int n = 0; n < NR; ++n) x[t][n] = mfma<F16>(kf[k][t], w.q[n][k], k ? x[t][n] : f32x4{0.f, 0.f, 0.f, 0.f});
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (PT) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4 k4 = *(const f32x4*)(lsc + 16 * g + 4 * (wi * NT + t));
#pragma unroll
        for (int n = 0; n < NR; ++n) x[t][n] *= k4;
      }
    }
    const int t0 = tile * SP_TILE;
    if (t0 < pc.begin || t0 + SP_TILE > pa_min(w.least, pc.end)) {
      asm volatile("");  // (a branch: not computed for every tile)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = t0 + 16 * g + 4 * (wi * NT + t) + i;
            if (at < pc.begin || at >= w.limit[n]) x[t][n][i] = kNegInf;
          }
    }
    i32x4 p[NR];
    auto value_scales = [&](int t) {
      if constexpr (PT) {
        vs[0] = *(const f32x4*)(lsc + SP_TILE + 16 * g + 4 * (wi * NT + t));
        vs[1] = *(const f32x4*)(lsc + SP_TILE + 16 * g + 4 * (wi * NT + t + 1));
      }
    };
    value_scales(0);
    w.weights(x[0], x[1], vs[0], vs[1], p);
    if constexpr (NJ == 2) {
      // the first product beside the second half's probabilities, reads VP ahead
      __builtin_amdgcn_sched_barrier(0);
      w.add_sums(p);
#pragma unroll
      for (int i = VP; i < VP + VA; ++i) {
        if (i < VA) vf[i] = lv[2 * g * D + 16 * i + c];
#pragma unroll
        for (int n = 0; n < NR; ++n) w.o[n][i - VP] = mfma<PF16>(vf[i - VP], p[n], w.o[n][i - VP]);
      }
#pragma unroll
      for (int dt = 0; dt < VP; ++dt) vf[dt] = lv[(2 * g + 1) * D + 16 * dt + c];
#pragma unroll
      for (int dt = 0; dt < VA; ++dt) {
        __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedMfma, NR, 0);
        __builtin_amdgcn_sched_group_barrier(kSchedAlu, NR * 24 / VA, 0);
      }
      value_scales(2);
      w.weights(x[2], x[3], vs[0], vs[1], p);
    }
    // the last product beside the next tile's way into LDS (behind the last tile:
    // once more the last, which no one reads)
    mask(pa_min(tile + 1, last));
    __builtin_amdgcn_sched_barrier(0);
    w.add_sums(p);
#pragma unroll
    for (int i = VP; i < VP + VA; ++i) {
      if (i < VA) vf[i] = lv[(2 * g + wi * NJ + NJ - 1) * D + 16 * i + c];
#pragma unroll
      for (int n = 0; n < NR; ++n) w.o[n][i - VP] = mfma<PF16>(vf[i - VP], p[n], w.o[n][i - VP]);
    }
    store(buffer ^ 1);
#pragma unroll
    for (int dt = 0; dt < VA; ++dt) {
      if (dt < VA - VP) __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, NR, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedAlu, 4, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedDsWrite, 1, 0);
    }
    if (tile + 2 <= last) fetch(tile + 2, entry);
    entry = page_at(tile + 3);
    __syncthreads();
  }
  w.finish(pc, lds, WT, wave, wr, wi, c, g);
}

static_assert(end_bytes(64, 2) <= 2 * tile_bytes(64) && end_bytes(128, 2) <= 2 * tile_bytes(128) &&
                  end_bytes(192, 1) <= 2 * tile_bytes(192) && end_bytes(256, 1) <= 2 * tile_bytes(256),
              "a piece's end fits the tiles' buffers");

// ---------------------------------------------------------------------------
// The kernels
// ---------------------------------------------------------------------------

template <int D, bool F16, bool PT>
__global__ __launch_bounds__(kThreads, 2) void pa_shared_prefix_kernel(const SpArgs s) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const pa_fp8_shared_prefix_args& a = s.a;
  const int B = a.num_seqs, G = a.num_groups, H = a.num_kv_heads;
  // every line of the arguments is asked for at once, not one by one where first used
  asm volatile("" ::"s"(a.context_lengths), "s"(a.stride_k_block), "s"(a.stride_out_tok), "s"(a.block_size), "s"(s.p.rows),
               "s"(s.s.overhead), "s"(s.seq_info), "s"(s.p_o), "s"(s.s_o));
  const Plan pl = plan_of(lds, B, G);
  char* const work = lds + plan_bytes(B, G);
  make_plan(pl, s);

  // what the merge needs of each sequence
  const int worker = blockIdx.x;
  for (int b = worker + (int)gridDim.x * (int)threadIdx.x; b < B; b += (int)gridDim.x * kThreads) {
    const int gr = group_of(pl, G, b);
    const bool has = gr >= 0 && pl.len[gr] > 0;
    int4 v;
    v.x = has ? H * pl.row_tiles[gr] : -1;
    v.y = has ? (b - pl.first[gr]) * s.eq : 0;
    v.z = has ? pl.row_tiles[gr + 1] - pl.row_tiles[gr] : 0;
    v.w = pl.seq_at[b + 1] > pl.seq_at[b];
    s.seq_info[b] = v;
  }

  // the line: prefix items from 0, suffix items from `suffix_at`; the shared ones
  // first (prefix items have at least a suffix item's rows)
  const int64_t prefix_cost = (int64_t)H * pl.group_at[G], suffix_cost = (int64_t)H * pl.seq_at[B];
  const int64_t shared = (s.p.shared ? prefix_cost : 0) + (s.s.shared ? suffix_cost : 0);
  const int64_t share = sp_share(shared, prefix_cost + suffix_cost - shared, gridDim.x);
  const int64_t direct_at = sp_direct_at(shared, share, gridDim.x);
  const int64_t suffix_at = s.s.shared || !s.p.shared ? prefix_cost : direct_at;
  const int64_t line = suffix_at + suffix_cost, lo = (int64_t)worker * share;
  if (lo >= line) return;
  Walk walk;
  walk.start(s, pl, suffix_at, 0, shared, lo, share, worker);
  Piece pc;
  while (walk.next_piece(s, pl, D, false, pc)) {
    const SpShape& sh = pc.of_prefix ? s.p : s.s;
    constexpr int most = D <= 128 ? 2 : 1;
    if (sh.wt == 1)
      run_shared<D, F16, PT, most, 1>(s, pc, pl.ctx, work);
    else if (most == 1 || sh.nr == 1)
      run_shared<D, F16, PT, 1, 2>(s, pc, pl.ctx, work);
    else
      run_shared<D, F16, PT, most, 2>(s, pc, pl.ctx, work);
  }
  if constexpr (D <= 128) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t quarter = share / SP_WAVES;
    walk.start(s, pl, suffix_at, direct_at, line, lo + wave * quarter, quarter, worker * SP_WAVES + wave);
    while (walk.next_piece(s, pl, D, true, pc)) run_direct<D, F16, PT>(s, pc, pl.ctx);
  }
}

constexpr int kMergeThreads = 256;

// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over a row's pieces.
// Workgroup (sequence and kv head, block of columns): D / 4 threads, a team,
// hold a row's four dims each; `shares` teams (a power of two) share a row's
// pieces, four of them in flight each, and meet in LDS.
template <int D, bool PT>
__global__ __launch_bounds__(kMergeThreads) void pa_shared_prefix_merge_kernel(const SpArgs s, int shares) {
  constexpr int kTeam = D / 4, kTeams = kMergeThreads / kTeam;
  __shared__ float lm[kTeams], ll[kTeams];
  __shared__ __attribute__((aligned(16))) f32x4 lo[kMergeThreads];
  const pa_fp8_shared_prefix_args& a = s.a;
  const int H = a.num_kv_heads, b = blockIdx.x / H, h = blockIdx.x - b * H;
  const int team = threadIdx.x / kTeam, d = (threadIdx.x - team * kTeam) * 4;
  const int block_cols = kTeams / shares;
  const int col = team / shares, share = team - col * shares;
  const int e = blockIdx.y * block_cols + col;
  const bool live = col < block_cols && e < s.eq;

  asm volatile("" ::"s"(a.value_scale), "s"(a.stride_out_head), "s"(a.output_dtype), "s"(s.p.rows), "s"(s.items), "s"(s.p_o),
               "s"(s.s_o));  // (as above)
  const int4 info = s.seq_info[b];
  // the row's pieces: n[0] in the prefix's slots, n[1] in the suffix's
  int first[2] = {0, 0}, n[2] = {0, 0}, row[2] = {0, 0};
  if (live) {
    if (info.x >= 0) {
      const int r = info.y + e, t = r / s.p.rows;
      const int2 it = s.items[info.x + h * info.z + t];
      first[0] = it.x;
      n[0] = it.y;
      row[0] = r - t * s.p.rows;
    }
    if (info.w) {
      const int t = e / s.s.rows;
      const int2 it = s.items[s.max_prefix_items + (b * H + h) * s.col_tiles + t];
      first[1] = it.x;
      n[1] = it.y;
      row[1] = e - t * s.s.rows;
    }
  }
  float m = kNegInf, l = 0.0f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float mi, float li, const f32x4& oi) {
    const float mn = fmaxf(m, mi);
    const float f = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float fi = mi == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mi - mn);
    l = l * f + li * fi;
    o = o * f + oi * fi;
    m = mn;
  };
  constexpr int kAhead = 4;
  for (int i0 = share; i0 < n[0] + n[1]; i0 += kAhead * shares) {
    float mi[kAhead], li[kAhead];
    f32x4 oi[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * shares;
      const bool in = i < n[0] + n[1], p = i < n[0];
      const int rows = p ? s.p_rows : s.s_rows, r = p ? row[0] : row[1];
      const int64_t slot = in ? (p ? first[0] + i : first[1] + i - n[0]) : 0;
      const float* ml = (p || !in ? s.p_ml : s.s_ml) + slot * 2 * rows + r;
      const float* po = (p || !in ? s.p_o : s.s_o) + (slot * rows + r) * D + d;
      mi[k] = kNegInf;
      li[k] = 0.0f;
      oi[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (in) {
        mi[k] = ml[0];
        li[k] = ml[rows];
        oi[k] = *(const f32x4*)po;
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) add(mi[k], li[k], oi[k]);
  }
  if (shares > 1) {
    if (d == 0 && team < kTeams) {
      lm[team] = m;
      ll[team] = l;
    }
    lo[threadIdx.x] = o;
    __syncthreads();
    if (!live || share) return;
    for (int i = 1; i < shares; ++i) add(lm[team + i], ll[team + i], lo[threadIdx.x + i * kTeam]);
  }
  if (!live) return;
  // a row that sees no key is zero
  const float f = l == 0.0f ? 0.0f : (PT ? 1.0f : a.value_scale[0]) / l;
  const int qi = e / a.query_group_size;
  const int64_t off = (int64_t)(b * (int64_t)a.query_length + qi) * a.stride_out_tok +
                      (int64_t)(h * a.query_group_size + e - qi * a.query_group_size) * a.stride_out_head + d;
  if (l == 0.0f) o = f32x4{0.f, 0.f, 0.f, 0.f};
  o *= f;
  if (a.output_dtype == PA_DTYPE_F32)
    *(f32x4*)((float*)a.output + off) = o;
  else if (a.output_dtype == PA_DTYPE_F16)
    *(int2*)((uint16_t*)a.output + off) = int2{round2<true>(o[0], o[1]), round2<true>(o[2], o[3])};
  else
    *(int2*)((uint16_t*)a.output + off) = int2{round2<false>(o[0], o[1]), round2<false>(o[2], o[3])};
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct Sizes {
  SpShape p, s;
  int eq, col_tiles, s_rows;
  int64_t prefix_items, suffix_items;
  int64_t seq_info, items, p_ml, p_o, s_ml, s_o, total;  // byte offsets
};

bool head_ok(int d) { return d == 64 || d == 128 || d == 192 || d == 256; }

// Sizes of a launch; 0 or a PA_ERR_* code.
int sizes_of(int B, int G, int H, int ql, int gqa, int D, int workers, Sizes* z) {
  if (!head_ok(D)) return PA_ERR_HEAD_SIZE;
  if (B < 0 || G < 0 || H <= 0 || ql <= 0 || gqa <= 0 || workers <= 0 || B > sp_max_seqs(D) || G > sp_max_groups(D))
    return PA_ERR_SHAPE;
  const int64_t eq = (int64_t)ql * gqa, rows = eq * B;
  if (eq > (1 << 20) || rows > 0x7fffffff || (int64_t)H * gqa > 0x7fffffff) return PA_ERR_SHAPE;
  z->eq = (int)eq;
  z->s = sp_shape((int)eq, D);
  z->col_tiles = (int)((eq + z->s.rows - 1) / z->s.rows);
  z->s_rows = z->col_tiles > 1 ? z->s.rows : (int)eq;
  z->p = sp_shape(pa_max((int)((rows + pa_max(G, 1) - 1) / pa_max(G, 1)), z->eq), D);
  z->prefix_items = G > 0 ? (rows / z->p.rows + pa_min(G, B)) * H : 0;
  z->suffix_items = (int64_t)B * H * z->col_tiles;
  if (workers > (1 << 20) || z->prefix_items > 0x3fffffff || z->suffix_items > 0x3fffffff) return PA_ERR_SHAPE;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t here = at;
    at = (at + n + 255) & ~(int64_t)255;
    return here;
  };
  const int64_t np = z->prefix_items > 0 ? z->prefix_items + workers * (z->p.shared ? 1 : SP_WAVES) : 0;
  const int64_t ns = z->suffix_items + workers * (z->s.shared ? 1 : SP_WAVES);
  z->seq_info = take(16 * (int64_t)B);
  z->items = take(8 * (z->prefix_items + z->suffix_items));
  z->p_ml = take(np * 8 * z->p.rows);
  z->s_ml = take(ns * 8 * z->s_rows);
  z->p_o = take(np * z->p.rows * D * 4);
  z->s_o = take(ns * z->s_rows * D * 4);
  z->total = at;
  return PA_OK;
}

template <int D, bool F16, bool PT>
hipError_t launch(const SpArgs& s, hipStream_t st) {
  const int lds = plan_bytes(s.a.num_seqs, s.a.num_groups) + work_bytes(D, (s.a.num_groups > 0 && s.p.shared) || s.s.shared);
  hipLaunchKernelGGL((pa_shared_prefix_kernel<D, F16, PT>), dim3(s.a.num_workers), dim3(kThreads), lds, st, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // Teams of a row: about an eighth of the pieces that the workers leave of an item
  // at most, and no fewer than the columns leave idle.  64 sequences of a
  // 2048-token prefix: 5.7 us (a quarter of the pieces: 7.4; only what is idle: 5.6);
  // 32 of a 32768-token one: 7.8 us (8.2; 9.4).
  constexpr int teams = 1 << (31 - __builtin_clz(kMergeThreads / (D / 4)));
  const int pieces = s.a.num_workers / pa_max(1, s.prefix_items);
  int shares = 1;
  while (shares < teams && (shares * s.eq < teams || shares * 8 < pieces)) shares *= 2;
  hipLaunchKernelGGL((pa_shared_prefix_merge_kernel<D, PT>),
                     dim3((unsigned)(s.a.num_seqs * s.a.num_kv_heads), (unsigned)pa_cdiv(s.eq, kMergeThreads / (D / 4) / shares)),
                     dim3(kMergeThreads), 0, st, s, shares);
  return hipGetLastError();
}

template <int D>
hipError_t dispatch(const SpArgs& s, hipStream_t st) {
  const bool f16 = s.a.query_dtype == PA_DTYPE_F16;
  if (s.a.per_token_kv) return f16 ? launch<D, true, true>(s, st) : launch<D, false, true>(s, st);
  return f16 ? launch<D, true, false>(s, st) : launch<D, false, false>(s, st);
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace

PA_CHECK_DEFINE_TAKE(pa_violations_shared_prefix)

extern "C" int64_t pa_fp8_shared_prefix_workspace_bytes(int num_seqs, int num_groups, int num_kv_heads,
                                                        int query_length, int query_group_size, int head_size,
                                                        int num_workers) {
  Sizes z;
  const int rc = sizes_of(num_seqs, num_groups, num_kv_heads, query_length, query_group_size, head_size, num_workers, &z);
  return rc == PA_OK ? z.total : rc;
}

extern "C" int pa_fp8_plan_shared_prefix(const int32_t* context_lengths, const int32_t* prefix_indptr,
                                         const int32_t* prefix_lengths, int B, int G, int H, int ql, int gqa, int D,
                                         int capacity, int workers, int max_pieces, int32_t* pieces) {
  Sizes z;
  const int rc = sizes_of(B, G, H, ql, gqa, D, workers, &z);
  if (rc != PA_OK) return rc;
  if ((B > 0 && !context_lengths) || (G > 0 && (!prefix_indptr || !prefix_lengths)) || (max_pieces > 0 && !pieces))
    return PA_ERR_NULL_ARG;
  std::vector<int> first(G + 1, 0), len(G, 0), tiles(G + 1, 0), seq_len(B, 0);
  int top = 0;
  for (int g = 0; g <= G && G > 0; ++g) first[g] = top = pa_max(top, pa_min(pa_max(prefix_indptr[g], 0), B));
  struct Kind {
    bool prefix;
    int of, h0, items, begin, tiles, base;
  };
  std::vector<Kind> line;
  for (int g = 0; g < G; ++g) {
    const int rows = (first[g + 1] - first[g]) * z.eq;
    len[g] = rows > 0 ? pa_min(pa_max(prefix_lengths[g], 0), capacity) : 0;
    for (int b = first[g]; b < first[g + 1]; ++b) seq_len[b] = len[g];
    tiles[g + 1] = tiles[g] + (len[g] > 0 ? pa_cdiv(rows, z.p.rows) : 0);
    const int n = tiles[g + 1] - tiles[g], steps = sp_tiles(0, len[g]);
    if (n > 0) line.push_back({true, g, n, H * n, 0, steps, H * tiles[g]});
  }
  for (int b = 0; b < B; ++b) {
    const int end = pa_min(pa_max(context_lengths[b], 0), capacity);
    const int steps = sp_tiles(seq_len[b], end);
    if (steps > 0) line.push_back({false, b, z.col_tiles, H * z.col_tiles, seq_len[b], steps, b * H * z.col_tiles});
  }
  int64_t cost[2] = {0, 0};  // of the suffix and the prefix items
  for (const Kind& k : line) cost[k.prefix] += (int64_t)k.items * sp_item_cost(k.prefix ? z.p : z.s, k.tiles);
  const int64_t shared = (z.p.shared ? cost[1] : 0) + (z.s.shared ? cost[0] : 0);
  const int64_t share = sp_share(shared, cost[0] + cost[1] - shared, workers);
  const int64_t suffix_at = z.s.shared || !z.p.shared ? cost[1] : sp_direct_at(shared, share, workers);
  int n = 0;
  int64_t at = 0;
  bool prefix = true;
  for (const Kind& k : line) {
    if (prefix && !k.prefix) {
      prefix = false;
      at = suffix_at;
    }
    const SpShape& sh = k.prefix ? z.p : z.s;
    const int64_t q = sh.shared ? share : share / SP_WAVES;
    for (int i = 0; i < k.items; ++i) {
      const int w0 = sp_worker_of(at + sh.overhead, q);
      const int w1 = sp_worker_of(at + sh.overhead + (int64_t)(k.tiles - 1) * sh.cost, q);
      for (int w = w0; w <= w1; ++w) {
        const int t0 = k.begin / SP_TILE + sp_tile_from(sh, w * q, at, k.tiles);
        const int t1 = k.begin / SP_TILE + sp_tile_from(sh, (w + 1) * q, at, k.tiles);
        const int32_t rec[8] = {k.prefix, k.base + i, w, k.base + i + w, k.of, i / k.h0, t0, t1};
        for (int j = 0; j < 8 && n < max_pieces; ++j) pieces[8 * n + j] = rec[j];
        ++n;
      }
      at += sp_item_cost(sh, k.tiles);
    }
  }
  return n;
}

extern "C" int pa_fp8_decode_shared_prefix(const pa_fp8_shared_prefix_args* a, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  if (!a) return PA_ERR_NULL_ARG;
  if (a->abi_version != PA_FP8_ABI_VERSION) return PA_ERR_ABI;
  Sizes z;
  const int rc = sizes_of(a->num_seqs, a->num_groups, a->num_kv_heads, a->query_length, a->query_group_size,
                          a->head_size, a->num_workers, &z);
  if (rc != PA_OK) return rc;
  const int bs = a->block_size;
  if (bs < 16 || bs > 1024 || (bs & (bs - 1))) return PA_ERR_BLOCK_SIZE;
  if (a->num_blocks < 0 || a->max_blocks_per_seq < 0) return PA_ERR_SHAPE;
  if (a->query_dtype != PA_DTYPE_BF16 && a->query_dtype != PA_DTYPE_F16) return PA_ERR_DTYPE;
  if (a->output_dtype != PA_DTYPE_BF16 && a->output_dtype != PA_DTYPE_F16 && a->output_dtype != PA_DTYPE_F32)
    return PA_ERR_DTYPE;
  if (a->num_seqs == 0) return PA_OK;
  if (a->num_blocks == 0 || a->max_blocks_per_seq == 0) return PA_ERR_SHAPE;
  if (!a->output || !a->query || !a->key_cache || !a->value_cache || !a->block_tables || !a->context_lengths ||
      !a->key_scale || !a->value_scale || !workspace || (a->num_groups > 0 && (!a->prefix_indptr || !a->prefix_lengths)))
    return PA_ERR_NULL_ARG;
  // 16-byte vectors of queries (8 values), cache bytes, scales (4) and outputs (4)
  if (!al16(a->query) || !al16(a->key_cache) || !al16(a->value_cache) || !al16(a->output) || !al16(workspace) ||
      a->stride_q_tok % 8 || a->stride_q_head % 8 || a->stride_k_block % 16 || a->stride_k_head % 16 ||
      a->stride_v_block % 16 || a->stride_v_head % 16 || a->stride_out_tok % 4 || a->stride_out_head % 4)
    return PA_ERR_ALIGN;
  if (a->per_token_kv && (!al16(a->key_scale) || !al16(a->value_scale) || a->stride_ks_block % 4 || a->stride_ks_head % 4))
    return PA_ERR_ALIGN;
  if (workspace_bytes < z.total) return PA_ERR_SCRATCH;
  if ((int64_t)a->num_seqs * a->num_kv_heads > 0x7fffffff || pa_cdiv(z.eq, 2) > 65535) return PA_ERR_SHAPE;
  SpArgs s;
  s.a = *a;
  s.p = z.p;
  s.s = z.s;
  s.eq = z.eq;
  s.col_tiles = z.col_tiles;
  s.p_rows = z.p.rows;
  s.s_rows = z.s_rows;
  const int64_t cap = (int64_t)a->max_blocks_per_seq * bs;
  s.capacity = cap < SP_MAX_TOKENS ? (int)cap : SP_MAX_TOKENS;
  s.lbs = 31 - __builtin_clz((unsigned)bs);
  char* ws = (char*)workspace;
  s.seq_info = (int4*)(ws + z.seq_info);
  s.items = (int2*)(ws + z.items);
  s.max_prefix_items = (int)z.prefix_items;
  s.prefix_items = a->num_groups > 0 ? (int)((int64_t)z.eq * a->num_seqs / z.p.rows + 1) * a->num_kv_heads : 1 << 20;
  s.p_ml = (float*)(ws + z.p_ml);
  s.p_o = (float*)(ws + z.p_o);
  s.s_ml = (float*)(ws + z.s_ml);
  s.s_o = (float*)(ws + z.s_o);
  hipStream_t st = (hipStream_t)stream;
  hipError_t e;
  switch (a->head_size) {
    case 64: e = dispatch<64>(s, st); break;
    case 128: e = dispatch<128>(s, st); break;
    case 192: e = dispatch<192>(s, st); break;
    default: e = dispatch<256>(s, st); break;
  }
  return e == hipSuccess ? PA_OK : (int)e;
}
