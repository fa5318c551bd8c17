// Prompt attention's kernels over one sequence's pages with no causal border, for queries
// that all come behind the sequence: partials of every row, which the caller joins with
// those of its other keys.  Inside the library only.
#pragma once

#include "attn_tile.h"

#pragma GCC visibility push(hidden)

struct PrefixPlan {
  int kind;            // prompt attention's kernel: 0 leaves [slot][kvh][part_rows][hd], the
                       // others [slot][kvh][part_rows / 32][hd / 8][64 lanes][4]
  int64_t tile_rows, part_rows;
  int64_t tiles, chunks, chunk_len;  // slot: tile * chunks + chunk
};

// T queries behind S keys.  Returns a status.
int tm_prefix_plan(int64_t T, int64_t S, int64_t Hq, int64_t kvh, PrefixPlan* o);

// p: q, k, v, table, part, stats and what says where they lie; q_len, k_len, kvh, group.
void tm_prefix_launch(tm_attn::PromptParams p, const PrefixPlan& o, int dtype, int64_t hd,
                      int64_t page_size, hipStream_t st);

#pragma GCC visibility pop
