// Work plan of the shared-prefix decode (shared_prefix.hip), one copy for the
// kernels and for the host planner that the tests read.
//
// Items.  A prefix item is (group, kv head, tile of the group's query rows)
// over the group's prefix; a suffix item is (sequence, kv head, tile of its
// query columns) over the tokens behind the prefix.  Both walk 64-token tiles
// of keys.  Few rows (direct): one wave works an item alone, from registers.
// More rows (shared): a workgroup of four waves works it, the waves hold
// different rows of it, and the tile comes to them through LDS.
//
// The line.  All items are laid end to end, prefix items first; an item of n
// tiles is overhead + n * cost long (nothing when n = 0), in units of a wave's
// time.  Workgroup w does the tiles of shared items that begin in [w q, (w + 1) q),
// q the line's share of a workgroup, and each of its waves the tiles of direct
// items that begin in the wave's quarter.  An item cut across workers (workgroups or
// waves) leaves one piece per worker, and item + worker numbers a piece: along
// the line, each step on to another item or worker adds one.
#pragma once

#include <stdint.h>

#include "pa_plan.h"

#define SP_TILE 64          // tokens of a tile
#define SP_WAVES 4          // waves of a workgroup
#define SP_MAX_TOKENS (1 << 30)  // of a table row: larger ones count as this
// Shortest share of a workgroup: no worker's part may be shorter than a tile (a shared
// one, or in a wave's quarter a direct one).  4 sequences of a 500-token prefix: 17.6 us
// (at 160: 18.3, at 224: 18.9).
#define SP_MIN_SHARE 96

// Sequences and groups of a launch, whose plan (16 bytes a sequence, 20 a group)
// is held in LDS beside two buffers of a tile: 73 KB of the 160 at head size 128,
// 109 at 192, 145 at 256.
PA_HD int sp_max_seqs(int head_size) { return head_size <= 128 ? 4096 : head_size <= 192 ? 2048 : 512; }
PA_HD int sp_max_groups(int head_size) { return sp_max_seqs(head_size) / 4; }

typedef struct SpShape {
  int shared;    // tiles come through LDS to a workgroup; else a wave works alone
  int nr;        // 16-row tiles of a wave
  int wt;        // waves that hold the same rows (shared)
  int rows;      // of an item
  int cost;      // of a tile, a shared one's being 64 (of a direct one, which a wave alone works, a quarter of its time)
  int overhead;  // of beginning and ending a piece
} SpShape;

// Up to 16 rows are one wave's, where the head size leaves registers for a
// tile beside them; up to twice what two waves hold, two waves share the rows
// and split the tile's tokens; beyond, each wave has its own.  Two 16-row tiles
// a wave where the head size leaves registers for them.
//
// Costs, from the times that workgroups with one kind of item took (two on a
// CU): a shared tile 2.0 us, beginning and ending a shared piece 5 us.  A direct
// tile moves half the bytes at head size 64.  Measured with the caches in HBM:
// 256 sequences of a 16383-token prefix at head size 128 take 126 us with direct
// tiles at 22, 129 at 26 and 138 at 16, 32 sequences of a 32768-token prefix 58.5,
// 57 and 63 us; two prefixes at head size 64 take 34.0 us at 16, 34.9 at 18, 35.7
// at 20.
PA_HD SpShape sp_shape(int rows, int head_size) {
  const int most = head_size <= 128 ? 2 : 1;
  SpShape s;
  s.shared = rows > 16 || head_size > 128;
  s.nr = rows > 32 ? most : 1;
  s.wt = !s.shared ? 1 : (rows > 32 * s.nr ? 1 : 2);
  s.rows = s.shared ? 16 * s.nr * (SP_WAVES / s.wt) : 16;
  s.cost = s.shared ? 64 : head_size <= 64 ? 16 : 22;
  s.overhead = s.shared ? 160 : 40;
  return s;
}

PA_HD int sp_tiles(int first_token, int end_token) {
  return end_token <= first_token ? 0 : pa_cdiv(end_token, SP_TILE) - first_token / SP_TILE;
}
PA_HD int sp_item_cost(const SpShape& s, int tiles) { return tiles > 0 ? s.overhead + tiles * s.cost : 0; }

// A workgroup's share of a line of shared and direct items: a multiple of four that
// no worker's part of is shorter than a tile.  The direct items begin with a
// workgroup of their own (sp_direct_at): a wave's quarter of a share takes as long
// as a workgroup's whole one, so a workgroup with both would take twice as long.
PA_HD int64_t sp_share(int64_t shared, int64_t direct, int workers) {
  const int w = shared > 0 && direct > 0 && workers > 1 ? workers - 1 : workers;
  const int64_t line = shared + direct;
  // (the usual line needs no 64-bit division)
  int64_t q = line < 0x40000000 ? (int64_t)(((uint32_t)line + w - 1) / (uint32_t)w) : (line + w - 1) / w;
  q = (q + 3) & ~(int64_t)3;
  return q < SP_MIN_SHARE ? SP_MIN_SHARE : q;
}
// The worker whose share holds position x.
PA_HD int sp_worker_of(int64_t x, int64_t share) {
  return x < 0x40000000 && share < 0x40000000 ? (int)((uint32_t)x / (uint32_t)share) : (int)(x / share);
}
// Where the direct items begin on the line.
PA_HD int64_t sp_direct_at(int64_t shared, int64_t share, int workers) {
  return workers > 1 && shared > 0 ? (int64_t)(sp_worker_of(shared - 1, share) + 1) * share : shared;
}
// First tile of an item at position `at` that begins at or behind x.
PA_HD int sp_tile_from(const SpShape& s, int64_t x, int64_t at, int tiles) {
  const int64_t d = x - at - s.overhead;
  if (d <= 0) return 0;
  if (d > (int64_t)tiles * s.cost) return tiles;
  return (int)(((uint32_t)d + s.cost - 1) / (uint32_t)s.cost);  // (a row's tiles times their cost: below 2^31)
}
