// Attention over lists of pages of the paged key/value cache, bfloat16, heads of 64 or 128, pages of 64 keys: the pages that were chosen for each token and
// key/value head, or the pages of a row behind those that it shares with others.
//
//   s[j] = (q . K[j]) * scale  over the keys of the listed pages at positions <= pos;   out = sum_j softmax(s)[j] V[j]
//
// One pass with running maximum and sum (float32; probabilities are rounded to bfloat16 for the second product, as in the other attention kernels here).
// Bound by memory: a key and a value are read once, for all query heads of their head and all tokens of the item.
#include "api.h"
#include "attention_pages.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <math.h>
#include <type_traits>

namespace exl3 {

constexpr int PG_WARPS = 4;                    // computing warps, and as many that ask for copies
constexpr int PG_UNIT_BYTES = 16384;           // a unit: keys and values of a page (heads of 64) or of half a page (heads of 128)
// A stage is always the same warps' (of the team's running count of units, n, warps n % lanes take unit n, in stage n % PG_STAGES): a warp that
// waits for a stage has itself freed it before, so that the stage's barrier is never a phase behind what the warp asks for.
constexpr int PG_STAGES = 8;
static_assert(PG_STAGES % PG_WARPS == 0, "a stage is always the same warps'");
constexpr int PG_MAX_COLS = 16 * PG_WARPS;     // queries of an item
constexpr int PG_WINDOW = 1024;                // items of a launch
constexpr int PG_MAX_WIDTH = 1 << 19;          // pages of a row: the units of a launch's items stay within 31 bits
constexpr uint32_t PG_SMEM_RING = PG_STAGES * PG_UNIT_BYTES;

static __device__ int g_pg_error = 0;

struct PgArgs {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  const int* block_table;
  int bt_stride, bt_width, bt_rows, n_pages;
  const int* tok_pos;                          // lists: position and row of each token
  const int* tok_seq;
  const int* lists;                            // [tokens, kv heads, count]: pages of the row
  int count, list_stride;                      // entries that are looked at, and that a list has
  const int* row_start;                        // rows
  const int* row_pos0;
  int rows, T, nh, nkv, G;
  int item0;                                   // the first item of this launch
  int groups_of_cols;                          // warps side by side on a unit, 16 queries each: 1, 2 or 4
  float scale_log2;
  int* counters;
  float* records;
  // the shared pages' parts
  const int* groups;
  int n_groups, ps_grid;
  int wait_first;                              // whether the kernel before must have ended
  const float* ps_records;
};

__device__ inline void pg_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ inline void pg_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ inline void pg_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ inline float pg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ inline uint32_t pg_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Whether one of a word's two bfloat16 is not finite.
__device__ inline bool pg_odd(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
// The form that a warp's threads may reach one after the other: code of one thread stands before most of these barriers.
__device__ inline void pg_bar(int id, int threads) {
  __syncwarp();
  asm volatile("barrier.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// Bounded, and one answer for the warp.
__device__ inline bool pg_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tc5::mbar_wait(bar, parity)); }

constexpr float PG_NEG = -INFINITY;

template <int HD> struct PgSmem {
  static constexpr int COLS = PG_MAX_COLS;
  float acc[PG_WARPS][16][HD];                 // the warps' sums of an item, to be joined
  float m[PG_WARPS][16], l[PG_WARPS][16];
  uint64_t full[PG_STAGES], empty[PG_STAGES];
  int key0[PG_STAGES];                         // a stage's first key (its place in the row); below 0: the page is not there
  int cum[PG_WINDOW + 1];                      // units of the items before (per kv head)
  int item_row[PG_WINDOW], item_block[PG_WINDOW];
  int flag[PG_WARPS];
  int n_items;
  PsPlan plan;
};

// Items: the queries that walk the same pages: of a row (or of a listed token) and a kv head up to PG_MAX_COLS (token, query head) pairs.  The units of all
// items, ordered by item and kv head, are cut into equal shares for teams of warps; a team's share may begin and end within an item, whose parts are then joined by the
// team that is last to report (in the parts' order, so that results do not depend on which it was).
template <int HD, bool LIST>
__global__ void __launch_bounds__(2 * PG_WARPS * 32, 1)
attn_pages_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PgArgs a) {
  constexpr int KS = HD == 64 ? 64 : 32;       // keys of a unit
  constexpr int UPP = PG_PAGE / KS;            // units of a page
  constexpr int NT = KS / 8;                   // tiles of 8 keys
  constexpr int KT = HD / 16;                  // pieces of 16 features
  constexpr int BOX = KS * 128;                // bytes of a box of 64 features
  extern __shared__ unsigned char pg_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(pg_raw) + 1023) & ~(uintptr_t)1023);
  PgSmem<HD>& sm = *reinterpret_cast<PgSmem<HD>*>(ring + PG_SMEM_RING);
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, tl = lane & 3;
  const int ncg = a.groups_of_cols, cols = 16 * ncg;
  if (threadIdx.x == 0) {
    for (int s = 0; s < PG_STAGES; ++s) { tc5::mbar_init(sm.full + s, 1); tc5::mbar_init(sm.empty + s, ncg); }
    tc5::mbar_init_fence();
  }
  // The kernel before is, with shared pages, the one that works on them: it let this one start when its own predecessors had ended, and what it
  // writes is waited for where it is read.  Else everything is waited for here.
  if (a.wait_first) pdl_wait();
  pdl_trigger();
  if (a.n_groups > 0) ps_plan(sm.plan, a.groups, a.n_groups, a.row_start, a.rows, a.T, a.G, a.nkv, a.bt_width, a.ps_grid);

  // ---- the items of this launch ------------------------------------------------------------------------------------------
  const int most_keys = a.bt_width * PG_PAGE;
  // a row's first token of q, its tokens, and the first one's position (one beyond the table sees all of it)
  auto start_of = [&](int row) { return LIST ? row : min(max(__ldcg(a.row_start + row), 0), a.T); };
  auto new_of = [&](int row, int start) { return LIST ? 1 : max(0, min(__ldcg(a.row_start + row + 1), a.T) - start); };
  auto pos_of = [&](int row) { return max(-most_keys, min(most_keys, __ldcg((LIST ? a.tok_pos : a.row_pos0) + row))); };
  auto group_of = [&](int row) {               // -1: none
    if (a.n_groups == 0) return -1;
    int lo = 0, hi = a.n_groups - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (sm.plan.row[mid] <= row) lo = mid; else hi = mid - 1; }
    return row >= sm.plan.row[lo] && row < sm.plan.row[lo] + sm.plan.rows[lo] && sm.plan.pages[lo] > 0 ? lo : -1;
  };
  auto shared_of = [&](int row) { const int j = group_of(row); return j < 0 ? 0 : sm.plan.pages[j]; };     // pages that the row shares
  auto units_of = [&](int row, int block, int n_new) {
    const int pos = pos_of(row);
    if (LIST) return max(1, min(a.count, pos < 0 ? 0 : pos / PG_PAGE + 1) * UPP);
    const int end = min(pos + min(n_new, ((block + 1) * cols - 1) / a.G + 1), most_keys);      // keys that the item's last token sees
    return max(1, (end + KS - 1) / KS - shared_of(row) * UPP);
  };
  if (wid == 0) {
    // rows a stretch of 32 at a time; lane i has row r0 + i
    int at = 0;                                // items before (of all rows)
    const int n_rows = a.rows;
    for (int r0 = 0; r0 < n_rows && at < a.item0 + PG_WINDOW; r0 += 32) {
      const int row = r0 + lane;
      int n_new = 0, nb = 0;
      if (row < n_rows) {
        n_new = new_of(row, start_of(row));
        nb = (n_new * a.G + cols - 1) / cols;
      }
      int incl = nb;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
      const int total = __shfl_sync(0xffffffffu, incl, 31);
      for (int b = 0; b < nb; ++b) {
        const int i = at + incl - nb + b - a.item0;
        if (i >= 0 && i < PG_WINDOW) { sm.item_row[i] = row; sm.item_block[i] = b; sm.cum[i + 1] = units_of(row, b, n_new); }
      }
      at += total;
    }
    const int n = max(0, min(at - a.item0, PG_WINDOW));
    if (lane == 0) { sm.n_items = n; sm.cum[0] = 0; }
    __syncwarp();
    int run = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      int incl = i < n ? sm.cum[i + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
      if (i < n) sm.cum[i + 1] = run + incl;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  __syncthreads();
  const int n_items = sm.n_items;
  if (n_items == 0) {
    if (!a.wait_first) pdl_wait();
    return;
  }

  // ---- teams and shares ---------------------------------------------------------------------------------------------------
  const int64_t total = (int64_t)sm.cum[n_items] * a.nkv;
  constexpr int TS = PG_WARPS;                 // warps of a team
  const int per_block = PG_WARPS / TS, stages = PG_STAGES / per_block;
  const int warp = wid % PG_WARPS, team = warp / TS, tw = warp % TS;
  const bool copier = wid >= PG_WARPS;
  const int n_teams = (int)min((int64_t)gridDim.x * per_block, max((int64_t)1, total / 4));
  const int my = blockIdx.x * per_block + team;
  auto begin = [&](int t) { return total * t / n_teams; };
  const int64_t i_lo = my < n_teams ? begin(my) : total, i_hi = my < n_teams ? begin(my + 1) : total;
  auto item_of = [&](int64_t x) {
    int lo = 0, hi = n_items - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if ((int64_t)sm.cum[mid] * a.nkv <= x) lo = mid; else hi = mid - 1; }
    return lo;
  };
  const int s0 = team * stages;                // the team's stages
  bool ok = true;
  if (copier) {
    // ---- copies: a unit as soon as its stage is free; page numbers come 32 at a time ------------------------------------------
    if (tw == 0) {
      int n = 0;
      for (int64_t x = i_lo; x < i_hi && ok;) {
        const int it = item_of(x), units = sm.cum[it + 1] - sm.cum[it];
        const int64_t r = x - (int64_t)sm.cum[it] * a.nkv;
        const int g = (int)(r / units), u0 = (int)(r % units), u1 = (int)min((int64_t)units, u0 + (i_hi - x));
        const int row = sm.item_row[it];
        const int seq = LIST ? __ldcg(a.tok_seq + row) : row;
        const bool known = seq >= 0 && seq < a.bt_rows;
        const int* bt = a.block_table + (int64_t)seq * a.bt_stride;
        const int* list = LIST ? a.lists + ((int64_t)row * a.nkv + g) * a.list_stride : nullptr;
        const int shared = LIST ? 0 : shared_of(row);
        for (int p0 = u0 / UPP; p0 * UPP < u1 && ok; p0 += 32) {
          int logical = p0 + lane + shared;
          if (LIST) logical = p0 + lane < a.count && (p0 + lane) * UPP < u1 ? __ldcg(list + p0 + lane) : -1;
          int page = known && logical >= 0 && logical < a.bt_width ? __ldcg(bt + logical) : -1;
          if (page >= a.n_pages) page = -1;
          for (int u = max(u0, p0 * UPP); u < min(u1, (p0 + 32) * UPP) && ok; ++u, ++n) {
            const int pg = __shfl_sync(0xffffffffu, page, u / UPP - p0), lg = __shfl_sync(0xffffffffu, logical, u / UPP - p0);
            const int st = s0 + n % stages;
            if (n >= stages && !pg_wait(sm.empty + st, (n / stages - 1) & 1)) { ok = false; break; }
            if (lane == 0) {
              sm.key0[st] = pg < 0 ? -1 : lg * PG_PAGE + (u % UPP) * KS;
              if (pg < 0) {
                tc5::mbar_arrive(sm.full + st);
              } else {
                tc5::mbar_expect_tx(sm.full + st, PG_UNIT_BYTES);
                const int y = (int)(((int64_t)pg * a.nkv + g) * PG_PAGE) + (u % UPP) * KS;
                unsigned char* dst = ring + st * PG_UNIT_BYTES;
#pragma unroll
                for (int b = 0; b < HD / 64; ++b) {
                  tc5::tma_load_2d(dst + b * BOX, &map_k, sm.full + st, 64 * b, y);
                  tc5::tma_load_2d(dst + PG_UNIT_BYTES / 2 + b * BOX, &map_v, sm.full + st, 64 * b, y);
                }
              }
            }
            __syncwarp();
          }
        }
        x += u1 - u0;
      }
      // what was asked for must land before the block's shared memory goes away
      if (!ok && lane == 0) atomicExch(&g_pg_error, 1);
      for (int u = max(0, n - stages); u < n; ++u) pg_wait(sm.full + s0 + u % stages, (u / stages) & 1);
    }
  }

  // ---- computing ------------------------------------------------------------------------------------------------------------
  const int cg = tw % ncg, pl = tw / ncg, lanes_of_pages = TS / ncg;   // the warp's 16 queries, and its turn among the units
  const int bar_id = 1 + team, bar_threads = TS * 32;
  const uint32_t k_addr = tc5::smem_u32(ring), sw = lane & 7;
  int n0 = 0;                                  // the team's units before this segment
  for (int64_t x = copier ? i_hi : i_lo; x < i_hi; ) {
    const int it = item_of(x), units = sm.cum[it + 1] - sm.cum[it];
    const int64_t item_base = (int64_t)sm.cum[it] * a.nkv, r = x - item_base;
    const int g = (int)(r / units), u0 = (int)(r % units), u1 = (int)min((int64_t)units, u0 + (i_hi - x));
    const int row = sm.item_row[it], col0 = sm.item_block[it] * cols;
    const int start = start_of(row), n_new = new_of(row, start), pos0 = pos_of(row);
    const int n_cols = min(cols, n_new * a.G - col0);
    // this thread's two queries: columns gl and gl + 8 of the warp's 16
    int limit[2];
    uint32_t qf[KT][4];
    {
      const __nv_bfloat16* src[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = min(col0 + cg * 16 + gl + 8 * e, n_new * a.G - 1), tok = c / a.G, h = c % a.G;
        limit[e] = pos0 + tok;                 // the last key it sees
        src[e] = a.q + (int64_t)(start + tok) * a.q_stride + (int64_t)(g * a.G + h) * HD;
      }
#pragma unroll
      for (int k = 0; k < KT; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qf[k][e] = __ldcg(reinterpret_cast<const unsigned int*>(src[e & 1] + 16 * k + 8 * (e >> 1) + 2 * tl));
      }
    }
    const int first_limit = pos0 + col0 / a.G, last_limit = pos0 + min((col0 + cols - 1) / a.G, n_new - 1);
    float m[2] = {PG_NEG, PG_NEG}, l[2] = {0.0f, 0.0f}, o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    for (int i = (pl + lanes_of_pages - n0 % lanes_of_pages) % lanes_of_pages; i < u1 - u0; i += lanes_of_pages) {
      const int n = n0 + i, st = s0 + n % stages;
      if (ok) ok = pg_wait(sm.full + st, (n / stages) & 1);
      const int key0 = sm.key0[st];
      if (ok && key0 >= 0 && key0 <= last_limit) {
        const uint32_t kb = k_addr + st * PG_UNIT_BYTES, vb = kb + PG_UNIT_BYTES / 2;
        // Values that a query does not see may be anything, and its probability of 0 would be multiplied with them.  Those that no query
        // of the item sees are taken as zeros; where one that some see is not finite, all that not everyone sees are added query by query.
        const bool edge = key0 + KS - 1 > first_limit;
        int cut = last_limit;                  // the last key whose values the products take
        if (edge && first_limit < last_limit) {
          bool odd = false;
          for (int w = lane; w < KS * (HD / 8); w += 32) {
            const int key = w / (HD / 8), c = w % (HD / 8);
            if (key0 + key <= first_limit || key0 + key > last_limit) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(ring + st * PG_UNIT_BYTES + PG_UNIT_BYTES / 2 + (c / 8) * BOX + key * 128 + (((c & 7) ^ (key & 7)) << 4));
            odd |= pg_odd(v.x) || pg_odd(v.y) || pg_odd(v.z) || pg_odd(v.w);
          }
          if (__any_sync(0xffffffffu, odd)) cut = first_limit;
        }
        float s[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
        for (int k2 = 0; k2 < KT / 2; ++k2) {  // 32 features at a time: lanes 0-7, 8-15, .. address the four pieces of 8 features
          const uint32_t piece = (uint32_t)((4 * (k2 & 1) + (lane >> 3)) ^ sw) << 4;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            uint32_t b[4];
            pg_ldsm(b, kb + (k2 >> 1) * BOX + (8 * j + (lane & 7)) * 128 + piece);
            pg_mma(s[j], qf[2 * k2], b[0], b[1]);
            pg_mma(s[j], qf[2 * k2 + 1], b[2], b[3]);
          }
        }
        float mx[2] = {PG_NEG, PG_NEG};
        if (edge) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[j][e] = key0 + 8 * j + 2 * tl + (e & 1) > limit[e >> 1] ? PG_NEG : s[j][e] * a.scale_log2;
        } else {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] *= a.scale_log2;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        }
        const bool grows = mx[0] > m[0] || mx[1] > m[1];
        if (__any_sync(0xffffffffu, grows)) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m[e], mx[e]);
            f[e] = m[e] == PG_NEG ? 0.0f : pg_exp2(m[e] - mn);
            l[e] *= f[e];
            m[e] = mn;
          }
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) { o[d][0] *= f[0]; o[d][1] *= f[0]; o[d][2] *= f[1]; o[d][3] *= f[1]; }
        }
        const float ref[2] = {m[0] == PG_NEG ? 0.0f : m[0], m[1] == PG_NEG ? 0.0f : m[1]};
        uint32_t p[KS / 16][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float p0 = pg_exp2(s[j][0] - ref[0]), p1 = pg_exp2(s[j][1] - ref[0]), p2 = pg_exp2(s[j][2] - ref[1]), p3 = pg_exp2(s[j][3] - ref[1]);
          l[0] += p0 + p1;
          l[1] += p2 + p3;
          p[j >> 1][2 * (j & 1)] = pg_pack(p0, p1);
          p[j >> 1][2 * (j & 1) + 1] = pg_pack(p2, p3);
        }
        auto values = [&](auto cutting) {
#pragma unroll
          for (int k = 0; k < KS / 16; ++k) {
            uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;         // of this lane's keys 16 k + 2 tl, + 1 and + 8, + 9
            if (decltype(cutting)::value) {
              const int key = key0 + 16 * k + 2 * tl;
              keep0 = key + 1 <= cut ? 0xffffffffu : key <= cut ? 0xffffu : 0u;
              keep1 = key + 9 <= cut ? 0xffffffffu : key + 8 <= cut ? 0xffffu : 0u;
            }
#pragma unroll
            for (int d2 = 0; d2 < KT; ++d2) {  // 16 features at a time
              uint32_t b[4];
              pg_ldsm_t(b, vb + (d2 >> 2) * BOX + (16 * k + (lane & 15)) * 128 + ((uint32_t)((2 * (d2 & 3) + (lane >> 4)) ^ sw) << 4));
              pg_mma(o[2 * d2], p[k], b[0] & keep0, b[1] & keep1);
              pg_mma(o[2 * d2 + 1], p[k], b[2] & keep0, b[3] & keep1);
            }
          }
        };
        if (edge) values(std::true_type()); else values(std::false_type());
        if (cut < last_limit) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll 1
            for (int u = 0; u < 8; ++u) {
              const int key = 8 * j + u;
              const uint32_t w0 = __shfl_sync(0xffffffffu, p[j >> 1][2 * (j & 1)], (lane & 28) + (u >> 1)), w1 = __shfl_sync(0xffffffffu, p[j >> 1][2 * (j & 1) + 1], (lane & 28) + (u >> 1));
              if (key0 + key <= cut || key0 + key > last_limit) continue;
              const float p0 = __uint_as_float(u & 1 ? w0 & 0xffff0000u : w0 << 16), p1 = __uint_as_float(u & 1 ? w1 & 0xffff0000u : w1 << 16);
              const unsigned char* line = ring + st * PG_UNIT_BYTES + PG_UNIT_BYTES / 2 + key * 128 + 4 * tl;
#pragma unroll
              for (int d = 0; d < HD / 8; ++d) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(line + (d >> 3) * BOX + (((d & 7) ^ (key & 7)) << 4));
                const float v0 = __uint_as_float(v << 16), v1 = __uint_as_float(v & 0xffff0000u);
                if (key0 + key <= limit[0]) { o[d][0] = fmaf(p0, v0, o[d][0]); o[d][1] = fmaf(p0, v1, o[d][1]); }
                if (key0 + key <= limit[1]) { o[d][2] = fmaf(p1, v0, o[d][2]); o[d][3] = fmaf(p1, v1, o[d][3]); }
              }
            }
        }
      }
      __syncwarp();
      if (ok && lane == 0) tc5::mbar_arrive(sm.empty + st);            // (not after giving up: the copies end, too)
      __syncwarp();
    }
    n0 += u1 - u0;
    // ---- the team's sums, joined ------------------------------------------------------------------------------------------
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (tl == 0) { sm.m[warp][gl + 8 * e] = m[e]; sm.l[warp][gl + 8 * e] = l[e]; }
    }
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
      *reinterpret_cast<float2*>(&sm.acc[warp][gl][8 * d + 2 * tl]) = make_float2(o[d][0], o[d][1]);
      *reinterpret_cast<float2*>(&sm.acc[warp][gl + 8][8 * d + 2 * tl]) = make_float2(o[d][2], o[d][3]);
    }
    pg_bar(bar_id, bar_threads);
    // the sum of column c and feature d over the team's warps of that column; tm and tsum: its maximum and sum
    const int tid = tw * 32 + lane;
    auto team_of = [&](int c, int d, float& tm, float& tsum) {
      const int w0 = team * TS + c / 16, cc = c % 16;
      tm = PG_NEG;
      for (int i = 0; i < lanes_of_pages; ++i) tm = fmaxf(tm, sm.m[w0 + i * ncg][cc]);
      const float safe = tm == PG_NEG ? 0.0f : tm;
      float y = 0.0f;
      tsum = 0.0f;
      for (int i = 0; i < lanes_of_pages; ++i) {
        const float f = pg_exp2(sm.m[w0 + i * ncg][cc] - safe);
        tsum = fmaf(sm.l[w0 + i * ncg][cc], f, tsum);
        y = fmaf(sm.acc[w0 + i * ncg][cc][d], f, y);
      }
      return y;
    };
    auto out_at = [&](int c, int d) {
      const int cc = col0 + c;
      return a.out + ((int64_t)(start + cc / a.G) * a.nh + g * a.G + cc % a.G) * HD + d;
    };
    // the shared pages' parts of a row's queries
    const int grp = LIST ? -1 : group_of(row);
    const int64_t base = item_base + (int64_t)g * units;
    const bool whole = u0 == 0 && u1 == units;
    const int64_t rec = (int64_t)cols * (HD + 2);
    // a team's part of an item that began in the share before, or with this share, and the one that goes on in the next share
    auto record = [&](int t) { return a.records + (2 * (int64_t)t + (begin(t) < base ? 1 : 0)) * rec; };
    int ta = 0, tb = -1;                         // teams whose records are joined
    if (!whole) {
      float* dst = record(my);
      for (int i = tid; i < n_cols * HD; i += TS * 32) {
        float tm, ts;
        const float y = team_of(i / HD, i % HD, tm, ts);
        dst[2 * cols + i] = y;
        if (i % HD == 0) { dst[i / HD] = tm; dst[cols + i / HD] = ts; }
      }
      __threadfence();
      pg_bar(bar_id, bar_threads);
      ta = (int)(base * n_teams / total), tb = (int)((base + units - 1) * n_teams / total);
      while (ta > 0 && begin(ta) > base) --ta;
      while (ta + 1 < n_teams && begin(ta + 1) <= base) ++ta;
      while (tb > 0 && begin(tb) > base + units - 1) --tb;
      while (tb + 1 < n_teams && begin(tb + 1) <= base + units - 1) ++tb;
      if (tid == 0) {
        int* counter = a.counters + it * a.nkv + g;
        const bool last = atomicAdd(counter, 1) == tb - ta;
        if (last) *counter = 0;
        __threadfence();
        sm.flag[team] = last;
      }
      pg_bar(bar_id, bar_threads);
    }
    if (whole || sm.flag[team]) {
      if (grp >= 0) pdl_wait();
      for (int i = tid; i < n_cols * HD; i += TS * 32) {
        const int c = i / HD, d = i % HD;
        float mm = PG_NEG, ll = 0.0f, y = 0.0f;
        if (whole) y = team_of(c, d, mm, ll);
        auto add = [&](float m1, float l1, float y1) {
          const float top = fmaxf(mm, m1), safe = top == PG_NEG ? 0.0f : top;
          const float f0 = pg_exp2(mm - safe), f1 = pg_exp2(m1 - safe);
          ll = ll * f0 + l1 * f1;
          y = y * f0 + y1 * f1;
          mm = top;
        };
#pragma unroll 4
        for (int t = ta; t <= tb; ++t) {
          const float* p = record(t);
          add(__ldcg(p + c), __ldcg(p + cols + c), __ldcg(p + 2 * cols + i));
        }
        if (grp >= 0) {
          const int query = (start + (col0 + c) / a.G - sm.plan.tok0[grp]) * a.G + (col0 + c) % a.G, tile = query / PS_TILE, qr = query % PS_TILE;
          const int64_t first = sm.plan.work_before[grp] * a.nkv + ((int64_t)g * sm.plan.tiles(grp) + tile) * sm.plan.pages[grp];
          const int ba = sm.plan.block_of(first), bb = sm.plan.block_of(first + sm.plan.pages[grp] - 1);
#pragma unroll 4
          for (int b = ba; b <= bb; ++b) {
            const float* p = a.ps_records + ps_slot(sm.plan, a.nkv, grp, g, tile, b) * ps_record(HD);
            add(__ldcg(p + qr), __ldcg(p + PS_TILE + qr), __ldcg(p + ps_value(qr, d)));
          }
        }
        *out_at(c, d) = __float2bfloat16_rn(ll == 0.0f ? 0.0f : y / ll);
      }
    }
    pg_bar(bar_id, bar_threads);
    x += u1 - u0;
  }
  if (!ok && lane == 0) atomicExch(&g_pg_error, 2);
  __syncthreads();
  if (!a.wait_first) pdl_wait();               // this kernel's end is then the shared pages' kernel's end, too
}

// ---- host side ----------------------------------------------------------------------------------------------------------------

int pg_sms(const char* what) {                 // of the current device, 0: an error
  static int known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("%s: no device", what); return 0; }
  if (known[dev]) return known[dev];
  cudaError_t e = cudaSuccess;
  const int s64 = (int)(PG_SMEM_RING + sizeof(PgSmem<64>) + 1024), s128 = (int)(PG_SMEM_RING + sizeof(PgSmem<128>) + 1024);
  for (auto f : {(const void*)attn_pages_kernel<64, false>, (const void*)attn_pages_kernel<64, true>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, s64);
  for (auto f : {(const void*)attn_pages_kernel<128, false>, (const void*)attn_pages_kernel<128, true>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, s128);
  if (e == cudaSuccess) e = attn_shared_prepare();
  int sms = 0;
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess || sms < 1) { set_error("%s: cannot get %d bytes of shared memory: %s", what, s128, cudaGetErrorString(e)); return 0; }
  return known[dev] = sms;
}

static int64_t pg_record_floats(int sms, int hd) { return 2ll * sms * PG_MAX_COLS * (hd + 2); }
static int64_t ps_slots(int sms, int64_t T, int G, int nkv, int n_groups) { return n_groups ? sms + nkv * ((int64_t)T * G / PS_TILE + n_groups) : 0; }

template <bool LIST> static int pg_launch(PgArgs a, const CUtensorMap& map_k, const CUtensorMap& map_v, int hd, int most_cols, int sms, const char* what, cudaStream_t stream) {
  a.groups_of_cols = most_cols <= 16 ? 1 : most_cols <= 32 ? 2 : 4;
  const int cols = 16 * a.groups_of_cols;
  const int64_t items = LIST ? (int64_t)a.rows * ceil_div(a.G, cols) : std::min((int64_t)a.T * a.G, (int64_t)a.T * a.G / cols + a.rows);
  for (int64_t i0 = 0; i0 < items; i0 += PG_WINDOW) {
    a.item0 = (int)i0;
    a.wait_first = i0 > 0 || a.n_groups == 0;
    if (hd == 64) launch_pdl(attn_pages_kernel<64, LIST>, dim3(sms), dim3(2 * PG_WARPS * 32), PG_SMEM_RING + sizeof(PgSmem<64>) + 1024, stream, map_k, map_v, a);
    else launch_pdl(attn_pages_kernel<128, LIST>, dim3(sms), dim3(2 * PG_WARPS * 32), PG_SMEM_RING + sizeof(PgSmem<128>) + 1024, stream, map_k, map_v, a);
    const int rc = launch_status(what);
    if (rc) return rc;
  }
  return 0;
}

// What both entry points ask of their arguments, and the pools' maps.
static int pg_check(const char* what, const void* q, int64_t q_stride, const void* out, const void* k_pool, const void* v_pool, int64_t n_pages, const int* block_table,
                    int bt_width, int rows, int T, int nh, int nkv, int hd, float scale, CUtensorMap* map_k, CUtensorMap* map_v) {
  if (rows < 0 || T < 0 || nkv < 1 || nkv > PG_COUNTERS / PG_WINDOW || nh < nkv || nh % nkv || (hd != 64 && hd != 128) || !(scale > 0.0f) || !isfinite(scale) || n_pages < 1 ||
      (n_pages + 1) * nkv * PG_PAGE > INT32_MAX || bt_width < 1 || bt_width > PG_MAX_WIDTH || (int64_t)T * (nh / nkv) > INT32_MAX - PG_MAX_COLS) {
    set_error("%s: needs heads of 64 or 128, at most %d key/value heads, a positive scale, tables of at most %d pages and pools of fewer than 2^31 tokens times key/value heads, got %d rows, %d tokens, %d "
              "heads on %d of %d, scale %g, %lld pages, a table of %d", what, PG_COUNTERS / PG_WINDOW, PG_MAX_WIDTH, rows, T, nh, nkv, hd, (double)scale, (long long)n_pages, bt_width);
    return ERR_BAD_ARGUMENT;
  }
  if (!q || !out || !k_pool || !v_pool || !block_table) { set_error("%s: an array is missing", what); return ERR_BAD_ARGUMENT; }
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_pool) || !aligned16(v_pool) || q_stride % 8) {
    set_error("%s: q, its rows, out and the pools must be 16-byte aligned", what);
    return ERR_ALIGNMENT;
  }
  const int box = hd == 64 ? 64 : 32;
  int rc = tc5::make_map_k64(map_k, k_pool, n_pages * nkv * PG_PAGE, hd, box, what);
  return rc ? rc : tc5::make_map_k64(map_v, v_pool, n_pages * nkv * PG_PAGE, hd, box, what);
}

static PgArgs pg_args(const void* q, int64_t q_stride, void* out, int64_t n_pages, const int* block_table, int bt_stride, int bt_width, int rows, int T, int nh, int nkv,
                      float scale, float* scratch) {
  PgArgs a = {};
  a.q = static_cast<const __nv_bfloat16*>(q); a.q_stride = q_stride; a.out = static_cast<__nv_bfloat16*>(out); a.block_table = block_table; a.bt_stride = bt_stride;
  a.bt_width = bt_width; a.n_pages = (int)n_pages; a.rows = rows; a.T = T; a.nh = nh; a.nkv = nkv; a.G = nh / nkv; a.scale_log2 = scale * 1.4426950408889634f;
  a.counters = reinterpret_cast<int*>(scratch); a.records = scratch + PG_COUNTERS;
  return a;
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_attn_pages_status() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_pg_error, sizeof(int));
  if (v) { int z = 0; cudaMemcpyToSymbol(g_pg_error, &z, sizeof(int)); }
  return v;
}

// Floats of scratch that a call with these sizes wants; the first PG_COUNTERS must be zero before the first call and are zero after each.
extern "C" long long exl3_attn_pages_scratch(int sms, int T, int nh, int nkv, int hd, int n_groups) {
  if (nkv < 1) return 0;
  return PG_COUNTERS + pg_record_floats(sms, hd) + ps_slots(sms, T, nh / nkv, nkv, n_groups) * ps_record(hd);
}

// Attention of each token over the pages that lists[token][kv head][count] names.
extern "C" int exl3_attn_pages(const void* q, int64_t q_stride, void* out, const void* k_pool, const void* v_pool, int64_t n_pages, const int* block_table, int bt_stride,
                               int bt_width, int bt_rows, const int* tok_pos, const int* tok_seq, int T, const int* lists, int count, int nh, int nkv, int hd, float scale,
                               float* scratch, long long scratch_floats, cudaStream_t stream) {
  if (T == 0) return 0;
  CUtensorMap map_k, map_v;
  int rc = pg_check("attn_pages", q, q_stride, out, k_pool, v_pool, n_pages, block_table, bt_width, T, T, nh, nkv, hd, scale, &map_k, &map_v);
  if (rc) return rc;
  if (!tok_pos || !tok_seq || !lists || count < 1) { set_error("attn_pages: an array is missing, or lists of %d pages", count); return ERR_BAD_ARGUMENT; }
  const int sms = pg_sms("attn_pages");
  if (!sms) return ERR_UNSUPPORTED;
  if (!scratch || scratch_floats < exl3_attn_pages_scratch(sms, T, nh, nkv, hd, 0)) { set_error("attn_pages: scratch too small"); return ERR_SCRATCH; }
  PgArgs a = pg_args(q, q_stride, out, n_pages, block_table, bt_stride, bt_width, T, T, nh, nkv, scale, scratch);
  a.tok_pos = tok_pos; a.tok_seq = tok_seq; a.lists = lists; a.count = std::min(count, bt_width);
  a.list_stride = count; a.bt_rows = bt_rows;
  return pg_launch<true>(a, map_k, map_v, hd, a.G, sms, "attn_pages", stream);
}

// Causal attention of rows whose groups share their first pages (groups: int32 [n_groups, 3]: first row, rows, pages).
extern "C" int exl3_attn_shared(const void* q, int64_t q_stride, void* out, const void* k_pool, const void* v_pool, int64_t n_pages, const int* block_table, int bt_stride,
                                int bt_width, const int* row_start, const int* row_pos0, int rows, int T, const int* groups, int n_groups, int max_new, int nh,
                                int nkv, int hd, float scale, float* scratch, long long scratch_floats, cudaStream_t stream) {
  if (T == 0 || rows == 0) return 0;
  CUtensorMap map_k, map_v;
  int rc = pg_check("attn_shared", q, q_stride, out, k_pool, v_pool, n_pages, block_table, bt_width, rows, T, nh, nkv, hd, scale, &map_k, &map_v);
  if (rc) return rc;
  if (!row_start || !row_pos0 || n_groups < 0 || n_groups > PG_MAX_GROUPS || (n_groups && !groups) || max_new < 1) {
    set_error("attn_shared: needs all of its arrays, at most %d groups and max_new of 1 or more, got %d groups, max_new %d", PG_MAX_GROUPS, n_groups, max_new);
    return ERR_BAD_ARGUMENT;
  }
  const int sms = pg_sms("attn_shared");
  if (!sms) return ERR_UNSUPPORTED;
  if (!scratch || scratch_floats < exl3_attn_pages_scratch(sms, T, nh, nkv, hd, n_groups)) { set_error("attn_shared: scratch too small"); return ERR_SCRATCH; }
  PgArgs a = pg_args(q, q_stride, out, n_pages, block_table, bt_stride, bt_width, rows, T, nh, nkv, scale, scratch);
  a.row_start = row_start; a.row_pos0 = row_pos0; a.bt_rows = rows; a.groups = groups; a.n_groups = n_groups; a.ps_grid = sms;
  float* ps = scratch + PG_COUNTERS + pg_record_floats(sms, hd);
  a.ps_records = ps;
  if (n_groups) {
    PsArgs p = {};
    p.q = a.q; p.q_stride = q_stride; p.block_table = block_table; p.bt_stride = bt_stride; p.bt_width = bt_width; p.n_pages = (int)n_pages; p.row_start = row_start;
    p.row_pos0 = row_pos0; p.rows = rows; p.T = T; p.nkv = nkv; p.G = a.G; p.groups = groups; p.n_groups = n_groups; p.scale_log2 = a.scale_log2; p.records = ps;
    rc = attn_shared_launch(p, k_pool, v_pool, hd, sms, stream);
    if (rc) return rc;
  }
  return pg_launch<false>(a, map_k, map_v, hd, (int)std::min((int64_t)max_new * a.G, (int64_t)PG_MAX_COLS), sms, "attn_shared", stream);
}
