// Prompts over the 4-bit cache, in passes: the fp16 copies of some rows' pages fill a space of a given number of slots, and the prompt attention runs
// over those rows' tiles of queries; then the next rows.  cache4.cu plans the passes and makes the copies, attention_prefill_tc.cuh reads them.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace exl3 {

// Pages lo .. lo + count - 1 of the sequence have their copies in slots base, base + 1, ...; with `holes`, only those that the block table gives a page
// for, and some page that the row's queries look for has none.
struct FaRow { int lo, count, base, holes; };

// A tile of queries: its sequence, its first row of q, its queries, the first one's position.
struct PromptTile { int b, row0, rows, p_first; };

// A pass: its slots among all rows' and its tiles in the list by passes.
struct PromptPass { int slot0, slots, tile0, tiles; };

// The copy of page j of a sequence whose block table is bt, or -1: beyond the table, or no page of the pool's n_pages there.
__device__ inline int row_copy(const FaRow& r, const int* bt, int n_pages, int j) {
  const int k = j - r.lo;
  if (k < 0 || k >= r.count) return -1;
  if (r.holes) {
    const int page = __ldcg(bt + j);
    if (page < 0 || page >= n_pages) return -1;
  }
  return r.base + k;
}

struct C4Prompt {
  const unsigned char* pool;
  int n_pages, nkv;
  const int* block_table;
  int bt_stride, width, rows;
  const int *row_start, *row_pos0;
  int window, parts;
  int few;               // rows of up to so many new tokens are not taken here
  const int *tile_seq, *tile_q0;
  int n_tiles, tile_queries;
  int row_pages, total;  // pages at most of a row, and of all rows
  int stride, passes;    // a row belongs to the pass (pages of the rows before it) / stride
  const __nv_bfloat16* q;
  int64_t q_stride;
  int T, nh;
  float q_sign;          // 1, -1 or 0: what is left of the scale beside a positive one
  __half *k_out, *v_out, *q_out;
  float* q_scale;
  FaRow* own;            // [rows]
  int* pass_of;          // [rows]
  PromptPass* pass;      // [passes]
  int4* slot;            // [total]: row, page of the pool (-1: none), places of it that hold tokens, whether it is the first that the row sees
  PromptTile* tile;      // [n_tiles], by passes and within one in the given order
  float2* tops;          // [rows][nkv][parts]: the largest |key| and |value| of a part of a row's pages
  float2* undo;          // [rows][nkv]: what the products of the copied keys and of the copied values are multiplied by
};
constexpr int C4_MAX_PARTS = 32;
// Parts of a row's pages for the search of its largest values: a warp takes four pages at a time, a lane a part's result.
inline int c4_prompt_parts(int row_pages) { return row_pages < 4 * C4_MAX_PARTS ? ceil_div(row_pages, 4) : C4_MAX_PARTS; }

// The plan and the rows' largest values; a pass's copies, of up to `slots` pages (pass 0: and the queries).
int c4_prompt_plan(const C4Prompt& a, int hd, cudaStream_t stream);
int c4_prompt_copies(const C4Prompt& a, int hd, int pass, int slots, cudaStream_t stream);

}  // namespace exl3
