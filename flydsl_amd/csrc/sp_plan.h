// Work plan of the shared-prefix decode (shared_prefix.hip), one copy for the
// kernels and for the host planner that the tests read.
//
// Items.  A prefix item is (group, kv head, tile of the group's query rows)
// over the group's prefix; a suffix item is (sequence, kv head, tile of its
// query columns) over the tokens behind the prefix.  Both walk 64-token tiles
// of keys.  A workgroup has eight waves: SpShape::waves_r of them hold
// different rows (16 nr each) and see the same tokens, the others walk
// different tiles of the same rows, so the workgroup takes wt = 8 / waves_r
// tiles a step.
//
// The line.  All items are laid end to end, prefix items first; an item of n
// steps is ov + n * cost long (nothing when n = 0).  Worker w of W does the
// steps that begin in [w L / W, (w + 1) L / W).  An item cut across workers
// leaves one piece per worker, and item + worker numbers a piece: along the
// line, each step on to another item or worker adds one.
#pragma once

#include <stdint.h>

#include "pa_plan.h"

#define SP_TILE 64          // tokens of a tile
#define SP_WAVES 8          // waves of a workgroup
#define SP_MAX_SEQS 4096    // the plan of a launch is held in LDS
#define SP_MAX_GROUPS 1024

typedef struct SpShape {
  int nr, waves_r, wt, rows, cost;  // rows: of an item = 16 nr waves_r
} SpShape;

// Rows of a wave: two 16-row tiles where the head size leaves registers for
// them; waves_r: as many as the rows need.
PA_HD SpShape sp_shape(int rows, int head_size) {
  SpShape s;
  s.nr = rows > 16 && head_size <= 128 ? 2 : 1;
  s.waves_r = 1;
  while (s.waves_r < SP_WAVES && 16 * s.nr * s.waves_r < rows) s.waves_r *= 2;
  s.wt = SP_WAVES / s.waves_r;
  s.rows = 16 * s.nr * s.waves_r;
  s.cost = s.nr == 2 ? 8 : 5;
  return s;
}

#define SP_OVERHEAD 6   // cost of beginning and ending a piece, in the units of SpShape::cost
#define SP_MIN_SHARE 8  // of a worker: at least one step of either kind

PA_HD int sp_steps(int first_token, int end_token, int wt) {
  if (end_token <= first_token) return 0;
  return pa_cdiv(pa_cdiv(end_token, SP_TILE) - first_token / SP_TILE, wt);
}
PA_HD int sp_item_cost(int steps, int cost) { return steps > 0 ? SP_OVERHEAD + steps * cost : 0; }

PA_HD int sp_workers(int64_t line, int workers) {
  const int64_t most = line / SP_MIN_SHARE;
  return most < 1 ? 1 : (most < workers ? (int)most : workers);
}
PA_HD int64_t sp_begin(int w, int64_t line, int workers) { return (int64_t)w * line / workers; }
// The worker whose share holds position x (0 <= x < line).
PA_HD int sp_worker_of(int64_t x, int64_t line, int workers) { return (int)(((x + 1) * workers - 1) / line); }
// First step of an item at position `at` that begins at or behind x.
PA_HD int sp_step_from(int64_t x, int64_t at, int steps, int cost) {
  const int64_t d = x - at - SP_OVERHEAD;
  if (d <= 0) return 0;
  const int64_t k = (d + cost - 1) / cost;
  return k < steps ? (int)k : steps;
}
