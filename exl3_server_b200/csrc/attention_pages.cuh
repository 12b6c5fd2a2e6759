// What the attention over shared and over chosen pages have in common: the arguments, and how the shared pages' work is cut.
#pragma once

#include "common.cuh"

namespace exl3 {

constexpr int PG_PAGE = 64;                    // tokens of a page
constexpr int PG_MAX_GROUPS = 256;             // groups of rows that share pages, in one call
constexpr int PG_COUNTERS = 65536;             // ints at the start of the scratch memory: zero between launches

// A group's entry in the caller's list: rows first .. first + rows - 1 have their first `pages` pages in common.
struct PgGroup { int first, rows, pages; };

// ---- the shared pages' work ---------------------------------------------------------------------------------------------
// A group's queries of a key/value head are (token of the group, query head) in this order, cut into tiles of PS_TILE.  The work is the list of
// (group, kv head, tile, page) in this order, cut into equal shares for the blocks: a share ends in the middle of a tile's pages, and
// the parts are joined by whoever finishes the queries.  Both kernels work out the same cut from the groups.
constexpr int PS_TILE = 256;
constexpr int PS_MIN_PAGES = 4;                // pages of a share, at least: every part more is joined again

struct PsPlan {                                // in shared memory
  int n;                                       // groups
  int blocks;                                  // shares
  int64_t total;                               // pages of all tiles of all heads
  int64_t per, rem;                            // a share has `per` pages, the first `rem` shares one more
  int tok0[PG_MAX_GROUPS], queries[PG_MAX_GROUPS], pages[PG_MAX_GROUPS], row[PG_MAX_GROUPS], rows[PG_MAX_GROUPS];
  int tiles_before[PG_MAX_GROUPS + 1];         // tiles of a head in the groups before
  int64_t work_before[PG_MAX_GROUPS + 1];      // pages of tiles of a head in the groups before
  __device__ int tiles(int j) const { return (queries[j] + PS_TILE - 1) / PS_TILE; }
  __device__ int64_t begin(int block) const { return per * block + min((int64_t)block, rem); }
  // the share that holds place x of the list
  __device__ int block_of(int64_t x) const { return x < rem * (per + 1) ? (int)(x / (per + 1)) : (int)(rem + (x - rem * (per + 1)) / per); }
};

// By all threads of a block (it ends with a barrier).  groups: int32 [n, 3], ascending; a group that begins before the one ahead of it ends
// has no rows.
__device__ inline void ps_plan(PsPlan& p, const int* __restrict__ groups, int n, const int* __restrict__ row_start, int rows, int T, int G, int nkv,
                               int bt_width, int grid) {
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    p.row[j] = __ldcg(groups + 3 * j);
    p.rows[j] = __ldcg(groups + 3 * j + 1);
    p.pages[j] = min(max(__ldcg(groups + 3 * j + 2), 0), bt_width);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int end = 0;
    for (int j = 0; j < n; ++j) {
      const int first = p.row[j];
      const bool apart = first >= end && first < rows;
      p.row[j] = apart ? first : end;
      p.rows[j] = apart ? min(max(p.rows[j], 0), rows - first) : 0;
      end = p.row[j] + p.rows[j];
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int a = min(max(__ldcg(row_start + p.row[j]), 0), T), b = min(max(__ldcg(row_start + p.row[j] + p.rows[j]), a), T);
    p.tok0[j] = a;
    p.queries[j] = (b - a) * G;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    p.tiles_before[0] = 0;
    p.work_before[0] = 0;
    for (int j = 0; j < n; ++j) {
      p.tiles_before[j + 1] = p.tiles_before[j] + p.tiles(j);
      p.work_before[j + 1] = p.work_before[j] + (int64_t)p.tiles(j) * p.pages[j];
    }
    p.n = n;
    p.total = p.work_before[n] * nkv;
    p.blocks = (int)min((int64_t)grid, max((int64_t)1, p.total / PS_MIN_PAGES));
    p.per = p.total / p.blocks;
    p.rem = p.total - p.per * p.blocks;
  }
  __syncthreads();
}
// A part of the list that one block works on.
struct PsPart {
  int j, g, tile, p0, p1;                      // group, kv head, tile, pages
};
__device__ inline PsPart ps_part(const PsPlan& p, int nkv, int64_t x, int64_t end) {
  int lo = 0, hi = p.n - 1;
  while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (p.work_before[mid] * nkv <= x) lo = mid; else hi = mid - 1; }
  PsPart t;
  const int64_t r = x - p.work_before[lo] * nkv;
  const int64_t ht = r / p.pages[lo];
  t.j = lo;
  t.g = (int)(ht / p.tiles(lo));
  t.tile = (int)(ht % p.tiles(lo));
  t.p0 = (int)(r % p.pages[lo]);
  t.p1 = (int)min((int64_t)p.pages[lo], t.p0 + (end - x));
  return t;
}
// Where a part of tile `tile` of group j and kv head g, worked on by block b, leaves its record: blocks and tiles both ascend along the list.
__device__ inline int ps_slot(const PsPlan& p, int nkv, int j, int g, int tile, int b) {
  return b + p.tiles_before[j] * nkv + g * p.tiles(j) + tile;
}
// A tile of up to 128 queries has a place for 256 all the same: the two halves of a block then take pages in turn, and leave a record's half each.
// A record, in floats: the queries' maxima (base-2 units), their sums, their sums of values [query][hd].
__host__ __device__ constexpr int64_t ps_record(int hd) { return (int64_t)PS_TILE * (hd + 2); }

// The kernel over the shared pages (attention_shared.cu): one record for every part of a tile that a block works on.
struct PsArgs {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const int* block_table;
  int bt_stride, bt_width, n_pages;
  const int* row_start;
  const int* row_pos0;
  int rows, T, nkv, G;
  const int* groups;
  int n_groups;
  float scale_log2;
  float* records;
  PsPlan* plan;                                // left for the join
};
// What the join of a query's parts needs beside the records: its row's own pages' part, sums of values [token][head][hd], then (maximum, sum) [token][head].
__host__ __device__ constexpr int64_t ps_own(int64_t T, int nh, int hd) { return T * nh * (hd + 2); }
cudaError_t attn_shared_prepare();             // once for a device
int attn_shared_join(const PsPlan* plan, const float* records, const float* own, __nv_bfloat16* out, int T, int nh, int nkv, int hd, cudaStream_t stream);
int attn_shared_launch(const PsArgs& a, const void* k_pool, const void* v_pool, int hd, int sms, cudaStream_t stream);

}  // namespace exl3
