// What the attention over shared and over chosen pages have in common: the caller's groups, and how the tensor cores' part of the work is cut.
#pragma once

#include "common.cuh"

namespace exl3 {

constexpr int PG_PAGE = 64;                    // tokens of a page
constexpr int PG_MAX_GROUPS = 256;             // groups of rows that share pages, in one call
constexpr int PG_LOWEST = -(1 << 30);          // positions below count as this one: its sums with keys and tokens stay within 32 bits
constexpr int PG_COUNTERS = 65536;             // ints at the start of the scratch memory: zero between launches

// ---- the groups -------------------------------------------------------------------------------------------------------------
// The caller's list, int32 [n, 3]: first row, rows, pages that they have in common; ascending.  A group that begins before the one ahead of it ends has no rows.
struct PgGroups {                              // in shared memory
  int first[PG_MAX_GROUPS], rows[PG_MAX_GROUPS], pages[PG_MAX_GROUPS];
  int n;
  // a row's group, -1: none
  __device__ int of(int row) const {
    if (n == 0) return -1;
    int lo = 0, hi = n - 1;
#pragma unroll 1
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (first[mid] <= row) lo = mid; else hi = mid - 1; }
    return row >= first[lo] && row < first[lo] + rows[lo] && pages[lo] > 0 ? lo : -1;
  }
};
static_assert(PG_MAX_GROUPS <= 256, "a thread of a block for each");
// This thread's group of the list, on its way beside whatever else is asked for.
__device__ inline int3 pg_group_asked(const int* __restrict__ list, int n) {
  const int* const at = list + 3 * threadIdx.x;
  return (int)threadIdx.x < n ? make_int3(__ldcg(at), __ldcg(at + 1), __ldcg(at + 2)) : make_int3(0, 0, 0);
}
// By all threads of a block; ends with a barrier.
__device__ inline void pg_groups(PgGroups& g, int3 asked, int n, int rows, int bt_width) {
  if ((int)threadIdx.x < n) {
    g.first[threadIdx.x] = asked.x;
    g.rows[threadIdx.x] = asked.y;
    g.pages[threadIdx.x] = min(max(asked.z, 0), bt_width);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int end = 0;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int first = g.first[j];
      const bool apart = first >= end && first < rows;
      g.first[j] = apart ? first : end;
      g.rows[j] = apart ? min(max(g.rows[j], 0), rows - first) : 0;
      end = g.first[j] + g.rows[j];
    }
    g.n = n;
  }
  __syncthreads();
}

// ---- the tensor cores' work -----------------------------------------------------------------------------------------------------
// Tiles of up to PS_TILE queries (token, query head of a key/value head): of a group's tokens over the pages that its rows share, and of a row of many new
// tokens over its own pages.  The work is the list of (kv head, tile, PS_SETUP places and the tile's pages) in this order, cut into equal shares for the blocks: a
// share ends in the middle of a tile's pages, and the parts are joined by another kernel.
constexpr int PS_TILE = 256;
constexpr int PS_MAX_TILES = 512;              // of a key/value head
constexpr int PS_MAX_ROWS = 1024;              // rows up to which rows of many tokens have tiles of their own
constexpr int PS_MANY = 64;                    // queries of a row and key/value head from which its own pages are the tensor cores' work
constexpr int PS_MIN_PAGES = 4;                // places of a share, at least: every part more is joined again
constexpr int PS_SETUP = 6;                    // places of the list that a tile has beside its pages': what its queries' way in and its sums' way out cost, in pages

// The rows' own pages, and chosen pages, are walked in units of 8 KB; an item of that work (the queries that walk the same pages) has as many places in its list beside its units', for
// its queries' way in and its sums' way out.
constexpr int PG_SETUP = 3;

// Both kernels run side by side where there is work for both: the tensor cores' takes some of the SMs and leaves the others to the walk, whose streams of pages fill the memory's queue
// from fewer SMs than there are (a batch of 64 behind 4,096 shared keys, 32 heads of 128 on 8, 30 to 2,000 keys of their own: one after the other 117 us, side by side 80).  Both work out
// how many, in units of about 10 ns of an SM: `tiles` for the tiles' pages (180 for two sets of queries, 60 for one), PG_COST for a place of the walk (8 queries an item, PG_COST_16: 16), PG_START
// for what the walk takes however many SMs it has; and the time that the memory takes for its units (8 KB in 1.25 ns).  These are weights that were fitted to the three batches named here, with
// heads of 64 and 128 alike, and not costs: a tile's page by itself takes 110 and 52 (ps_tile_cost).  16 rows of up to 500 keys behind 2,048 pages, 32 heads on 2:
// without PG_START and with 16 for all the walk had 2 SMs and the call took 102 us, with them 69.5; 48 rows in 5 groups 50 and 46; 24 or 40 for PG_COST_16: 76.7 or 69.6, 48.1 or 47.9.
constexpr int64_t PS_COST_TWO = 180, PS_COST_ONE = 60, PG_COST = 16, PG_COST_16 = 32, PG_START = 400;
__host__ __device__ inline int ps_sms(int64_t tiles, int64_t places, int cols, int sms) {
  if (tiles == 0 || places == 0) return sms;
  const int64_t walk = places * (cols == 8 ? PG_COST : PG_COST_16), memory = places / 8;
  // the fewest SMs from which on the tiles are not the slower side, or one less
  auto slower = [&](int64_t n) { return tiles * (sms - n) > (walk + PG_START * (sms - n)) * n; };
  int64_t n = 1, hi = sms - 1;
  while (n < hi) { const int64_t mid = (n + hi) >> 1; if (slower(mid)) n = mid + 1; else hi = mid; }
  if (n > 1 && tiles * (sms - n) < (walk + PG_START * (sms - n)) * (n - 1)) --n;
  if (memory > 0 && tiles / memory + 1 < n) n = tiles / memory + 1;
  return (int)(n < 1 ? 1 : n > sms - 1 ? sms - 1 : n);
}

// A group's tiles of a key/value head, in the units of ps_sms.
__device__ inline int64_t ps_cost(int queries, int pages) {
  return (int64_t)((queries + PS_TILE - 1) / PS_TILE) * (pages + PS_SETUP) * (queries > 128 ? PS_COST_TWO : PS_COST_ONE);
}

// Where rows have many tokens: whether a group's tiles cost less than its rows reading the pages each for itself, in 10 ns of an SM.  Tiles: a page 1.1 us for two sets of queries, 0.52 for one; a group's way in
// and out PS_SETUP pages, and 0.04 us a query to join.  Rows: tiles of their own where they have many queries, else the walk.  Both sides measured, shared and each for itself: 37 prompts of 41 to
// 252 tokens behind one page, 36 heads of 64, 216 and 171 us; 62 of 99 to 128 tokens behind 16 to 19 pages in three groups, 36 heads of 64, 404 and 335 (8 heads of 128: 157 and 130); 24 of 16 to
// 120 behind 94 pages, 32 heads of 128 on 8, 224 and 266: only these share.  (Steps of few tokens a row are not asked: the pass over the rows costs 1 us, and short ones leave groups alone anyhow.)
__device__ inline int64_t ps_tile_cost(int queries) { return (int64_t)(queries / PS_TILE) * 110 + (queries % PS_TILE > 128 ? 110 : queries % PS_TILE > 0 ? 52 : 0); }
__device__ inline int ps_alone(int queries, int cols, int hd) {                    // a page, for a row's queries
  return queries > PS_MANY ? (int)ps_tile_cost(queries) : (queries + cols - 1) / cols * (hd == 64 ? 2 : 4) * (int)(cols == 8 ? PG_COST : PG_COST_16);
}
__device__ inline bool ps_worth(int queries, int pages, int alone) {               // alone: of all of the group's rows
  return pages > 0 && ps_tile_cost(queries) * (pages + PS_SETUP) + 4 * (int64_t)queries < (int64_t)alone * pages;
}

struct PsPlan {                                // the head of the list
  int n_tiles;
  int blocks;                                  // shares
  int total, per, rem;                         // places of the list; a share has `per` of them, the first `rem` shares one more
  __device__ int begin(int block) const { return per * block + min(block, rem); }
  // the share that holds place x
  __device__ int block_of(int x) const { return x < rem * (per + 1) ? x / (per + 1) : rem + (x - rem * (per + 1)) / per; }
};
// What the join needs of a token: its group's tiles and its row's own, each as the first tile's number (-1: none) and the token that this begins with.
struct PsToken { int shared_tile, shared_tok, own_tile, own_tok; };

// A part of a tile that one block works on leaves its record at the slot block + place of the tile in the list: both ascend along it.
__host__ __device__ constexpr int64_t ps_slots(int blocks, int nkv, int tiles) { return blocks + (int64_t)nkv * tiles; }
// Tiles of a key/value head that a call may have, at most, where rows of many tokens have tiles of their own: the groups', and a row's own for each PS_TILE queries or part of them.
__host__ __device__ constexpr int64_t ps_most_tiles(int64_t T, int G, int groups, int64_t rows) {
  return (groups ? T * G / PS_TILE + groups : 0) + (rows < T * G / (PS_MANY + 1) ? rows : T * G / (PS_MANY + 1)) + (T * G > PS_MANY ? T * G / PS_TILE : 0);
}
// A record, in floats: the queries' maxima (base-2 units), their sums, their sums of values [query][hd].  A tile of up to 128 queries has a place for 256 all the
// same: the two halves of a block then take its pages in turn, and leave a record's half each.
__host__ __device__ constexpr int64_t ps_record(int hd) { return (int64_t)PS_TILE * (hd + 2); }
// What the join needs beside: a row's own pages' part where it is not the tensor cores', sums of values [token][head][hd], then (maximum, sum) [token][head].
__host__ __device__ constexpr int64_t ps_own(int64_t T, int nh, int hd) { return T * nh * (hd + 2); }

// The kernel over these tiles (attention_shared.cu).
struct PsArgs {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const int* block_table;
  int bt_stride, bt_width, n_pages;
  const int* row_start;
  const int* row_pos0;
  int rows, T, nkv, G, hd;
  const int* groups;
  int n_groups;
  int many;                                    // whether rows of more than PS_MANY queries have tiles of their own
  int cols, window;                            // queries of an item of the walk, rows of a launch of it
  float scale_log2;
  float* records;
  PsToken* tokens;
  int* parts;                                  // for the join: per kv head and tile its first part's slot, its parts, the halves of a record (1 or 2) [kv heads][most tiles][4]
  int most_tiles, sms;
};
cudaError_t attn_shared_prepare();             // once for a device
int attn_shared_launch(const PsArgs& a, const void* k_pool, const void* v_pool, int hd, int sms, cudaStream_t stream);
int attn_shared_join(const PsArgs& a, const float* own, __nv_bfloat16* out, int* late, int hd, cudaStream_t stream);

}  // namespace exl3
