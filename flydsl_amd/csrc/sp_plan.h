// Work plan of the shared-prefix decode (shared_prefix.hip), one copy for the
// kernels and for the host planner that the tests read.
//
// Items.  A prefix item is (group, kv head, tile of the group's query rows)
// over the group's prefix; a suffix item is (sequence, kv head, tile of its
// query columns) over the tokens behind the prefix.  Both walk 64-token tiles
// of keys.  Few rows: each of the workgroup's four waves holds all of them and
// walks tiles of its own, read straight into its registers (four tiles a
// step).  More rows: the waves hold different ones and work the same tile,
// which comes to them through LDS (one tile a step).
//
// The line.  All items are laid end to end, prefix items first; an item of n
// steps is SP_OVERHEAD + n * cost long (nothing when n = 0).  Worker w does the
// steps that begin in [w q, (w + 1) q), q the line's share of a worker.  An item
// cut across workers leaves one piece per worker, and item + worker numbers a
// piece: along the line, each step on to another item or worker adds one.
#pragma once

#include <stdint.h>

#include "pa_plan.h"

#define SP_TILE 64          // tokens of a tile
#define SP_WAVES 4          // waves of a workgroup
#define SP_MAX_SEQS 4096    // the plan of a launch is held in LDS
#define SP_MAX_GROUPS 1024

typedef struct SpShape {
  int nr;      // 16-row tiles of a wave
  int shared;  // tiles come through LDS
  int wt;      // waves that hold the same rows
  int tiles;   // of a step
  int rows;    // of an item
  int cost;    // of a step
} SpShape;

// Up to 16 rows every wave holds them, where the head size leaves registers
// for a tile beside them; up to twice what two waves hold, two
// waves share the rows and split the tile's tokens; beyond, each wave has its
// own.  Two 16-row tiles a wave where the head size leaves registers for them.
PA_HD SpShape sp_shape(int rows, int head_size) {
  const int most = head_size <= 128 ? 2 : 1;
  SpShape s;
  s.shared = rows > 16 || head_size > 128;
  s.nr = rows > 32 ? most : 1;
  s.wt = !s.shared ? SP_WAVES : (rows > 32 * s.nr ? 1 : 2);
  s.tiles = s.shared ? 1 : SP_WAVES;
  s.rows = 16 * s.nr * (SP_WAVES / s.wt);
  s.cost = s.shared ? (s.wt == 1 ? 4 : 3) : 8;
  return s;
}

#define SP_OVERHEAD 6    // cost of beginning and ending a piece, in the units of SpShape::cost
#define SP_MIN_SHARE 10  // of a worker: at least one step of any kind

PA_HD int sp_steps(int first_token, int end_token, int tiles) {
  if (end_token <= first_token) return 0;
  return pa_cdiv(pa_cdiv(end_token, SP_TILE) - first_token / SP_TILE, tiles);
}
PA_HD int sp_item_cost(int steps, int cost) { return steps > 0 ? SP_OVERHEAD + steps * cost : 0; }

PA_HD int64_t sp_share(int64_t line, int workers) {
  // (the usual line needs no 64-bit division)
  const int64_t q = line < 0x40000000 ? (int64_t)(((uint32_t)line + workers - 1) / (uint32_t)workers)
                                      : (line + workers - 1) / workers;
  return q < SP_MIN_SHARE ? SP_MIN_SHARE : q;
}
// The worker whose share holds position x.
PA_HD int sp_worker_of(int64_t x, int64_t share) {
  return x < 0x40000000 && share < 0x40000000 ? (int)((uint32_t)x / (uint32_t)share) : (int)(x / share);
}
// First step of an item at position `at` that begins at or behind x.
PA_HD int sp_step_from(int64_t x, int64_t at, int steps, int cost) {
  const int64_t d = x - at - SP_OVERHEAD;
  if (d <= 0) return 0;
  if (d > (int64_t)steps * cost) return steps;
  return (int)(((uint32_t)d + cost - 1) / (uint32_t)cost);  // (a row's steps times their cost: below 2^31)
}
