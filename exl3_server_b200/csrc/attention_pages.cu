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

constexpr int PG_WARPS = 8;                    // of a block, one block an SM
constexpr int PG_STAGES = 3;                   // of a warp's ring
constexpr int PG_UNIT_BYTES = 8192;            // a unit: keys and values of 32 tokens (heads of 64) or 16 (heads of 128)
constexpr int PG_COLS = 16;                    // queries of an item
constexpr int PG_WINDOW = 1024;                // rows of a launch
constexpr int PG_MIN_UNITS = 4;                // of a warp's share, at least
constexpr int PG_MAX_WIDTH = 1 << 19;          // pages of a row
constexpr int PG_RING = PG_STAGES * PG_UNIT_BYTES;
constexpr uint32_t PG_SMEM_RINGS = PG_WARPS * PG_RING;

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
  int row0;                                    // the first row of this launch
  float scale_log2;
  int* counters;
  float* records;
  // the shared pages' parts
  const int* groups;
  int n_groups, ps_grid;
  int wait_first;                              // whether the kernel before must have ended
  float* own;                                  // rows of groups: their own pages' part goes here
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
// Bounded, and one answer for the warp.
__device__ inline bool pg_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tc5::mbar_wait(bar, parity)); }

constexpr float PG_NEG = -INFINITY;

// A warp's part of an item, at the start of its ring when the ring is done with: two of them at most, of the item that its share begins in and
// of the one that it ends in.
template <int HD> struct PgPart {
  float m[PG_COLS], l[PG_COLS], acc[PG_COLS][HD];
};
struct PgSmem {
  uint64_t full[PG_WARPS][PG_STAGES];
  int64_t cum[PG_WINDOW + 1];                  // units of the rows before
  int start[PG_WINDOW], n_new[PG_WINDOW], pos[PG_WINDOW], units[PG_WINDOW];
  int64_t part_at[PG_WARPS][2];                // a part's item (the place of its first unit), -1: none
  int64_t warp_sum[PG_WARPS];
  int last[2];
  PsPlan plan;
};

// Items: up to PG_COLS queries (token, query head) of a row (or of a listed token) and key/value head, which walk the same pages.  The units of all items, ordered by row, head and
// item, are cut into equal shares for the warps, which stream them through rings of their own, each asking for its own copies: nothing is waited for but
// memory.  What a warp has whole it writes out; parts of items that shares cut are joined in shared memory at the end, and those that blocks cut by the block that
// is the last to report, always in the order of the pages, so that results do not depend on which it was.
template <int HD, bool LIST>
__global__ void __launch_bounds__(PG_WARPS * 32, 1)
attn_pages_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PgArgs a) {
  constexpr int KS = HD == 64 ? 32 : 16;       // keys of a unit
  constexpr int UPP = PG_PAGE / KS;            // units of a page
  constexpr int NT = KS / 8;                   // tiles of 8 keys
  constexpr int KT = HD / 16;                  // pieces of 16 features
  constexpr int BOX = KS * 128;                // bytes of a box of 64 features
  constexpr int HALF = PG_UNIT_BYTES / 2;      // keys, then values
  static_assert(2 * sizeof(PgPart<HD>) <= PG_RING, "a warp's parts fit into its ring");
  extern __shared__ unsigned char pg_raw[];
  unsigned char* rings = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(pg_raw) + 1023) & ~(uintptr_t)1023);
  PgSmem& sm = *reinterpret_cast<PgSmem*>(rings + PG_SMEM_RINGS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, tl = lane & 3;
  if (threadIdx.x == 0) {
    for (int w = 0; w < PG_WARPS; ++w)
      for (int s = 0; s < PG_STAGES; ++s) tc5::mbar_init(&sm.full[w][s], 1);
    tc5::mbar_init_fence();
  }
  // The kernel before is, with shared pages, the one that works on them: it let this one start when its own predecessors had ended, and this one needs nothing of it.
  // Else everything is waited for here.
  if (a.wait_first) pdl_wait();
  pdl_trigger();

  // ---- the rows of this launch -------------------------------------------------------------------------------------------
  const int most_keys = a.bt_width * PG_PAGE, n_rows = min(a.rows - a.row0, PG_WINDOW);
  for (int i = threadIdx.x; i < n_rows; i += PG_WARPS * 32) {
    const int row = a.row0 + i;
    // (a row beyond the table sees all of it)
    sm.pos[i] = max(-most_keys, min(most_keys, __ldcg((LIST ? a.tok_pos : a.row_pos0) + row)));
    const int start = LIST ? row : min(max(__ldcg(a.row_start + row), 0), a.T);
    sm.start[i] = start;
    sm.n_new[i] = LIST ? 1 : max(0, min(__ldcg(a.row_start + row + 1), a.T) - start);
  }
  if (a.n_groups > 0) ps_plan(sm.plan, a.groups, a.n_groups, a.row_start, a.rows, a.T, a.G, a.nkv, a.bt_width, a.ps_grid);
  else __syncthreads();
  auto group_of = [&](int row) {               // -1: none
    if (LIST || a.n_groups == 0) return -1;
    int lo = 0, hi = a.n_groups - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (sm.plan.row[mid] <= row) lo = mid; else hi = mid - 1; }
    return row >= sm.plan.row[lo] && row < sm.plan.row[lo] + sm.plan.rows[lo] && sm.plan.pages[lo] > 0 ? lo : -1;
  };
  auto shared_of = [&](int row) { const int j = group_of(row); return j < 0 ? 0 : sm.plan.pages[j]; };     // pages that the row shares
  auto blocks_of = [&](int i) { return (sm.n_new[i] * a.G + PG_COLS - 1) / PG_COLS; };                     // items of a row and head
  {
    int64_t run = 0;
    for (int i0 = 0; i0 < n_rows; i0 += PG_WARPS * 32) {
      const int i = i0 + threadIdx.x;
      int64_t mine = 0;
      if (i < n_rows) {
        const int pos = sm.pos[i];
        int units;
        if (LIST) units = min(a.count, pos < 0 ? 0 : pos / PG_PAGE + 1) * UPP;
        else units = (min(pos + sm.n_new[i], most_keys) + KS - 1) / KS - shared_of(a.row0 + i) * UPP;
        sm.units[i] = max(units, 1);           // (one at least: every query gets an answer)
        mine = (int64_t)max(units, 1) * blocks_of(i) * a.nkv;
      }
      int64_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int64_t v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
      if (lane == 31) sm.warp_sum[warp] = incl;
      __syncthreads();
      int64_t before = run;
      for (int w = 0; w < PG_WARPS; ++w) { if (w < warp) before += sm.warp_sum[w]; run += sm.warp_sum[w]; }
      if (i < n_rows) sm.cum[i + 1] = before + incl;
      __syncthreads();
    }
    if (threadIdx.x == 0) sm.cum[0] = 0;
    __syncthreads();
  }
  const int64_t total = sm.cum[n_rows];
  const int n_blocks = (int)min((int64_t)gridDim.x, max((int64_t)1, total / (PG_WARPS * PG_MIN_UNITS)));
  if (total == 0 || (int)blockIdx.x >= n_blocks) {
    if (!a.wait_first) pdl_wait();
    return;
  }
  auto begin = [&](int w) { return total * w / (n_blocks * PG_WARPS); };       // the first unit of a warp's share
  const int64_t i_lo = begin(blockIdx.x * PG_WARPS + warp), i_hi = begin(blockIdx.x * PG_WARPS + warp + 1);
  // The item at place x, and where in it.
  struct Place { int i, g, b, u0, u1, units; int64_t base; };
  auto place_of = [&](int64_t x, int64_t end) {
    int lo = 0, hi = n_rows - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (sm.cum[mid] <= x) lo = mid; else hi = mid - 1; }
    Place p;
    p.i = lo;
    p.units = sm.units[lo];
    const int64_t r = x - sm.cum[lo];
    const int item = (int)(r / p.units), nb = blocks_of(lo);
    p.u0 = (int)(r - (int64_t)item * p.units);
    p.u1 = (int)min((int64_t)p.units, p.u0 + (end - x));
    p.g = item / nb;
    p.b = item % nb;
    p.base = x - p.u0;
    return p;
  };

  unsigned char* ring = rings + warp * PG_RING;
  uint64_t* full = sm.full[warp];
  // ---- copies: page numbers come 32 at a time, a batch ahead -----------------------------------------------------------------
  int64_t ask_x = i_lo;                        // the next unit to ask for
  Place ask = {};
  int ask_u = 0, ask_n = 0, batch_p = 0;       // its number in the item; units asked for so far; the first page of the batch at hand
  int page = 0, logical = 0, page_next = 0, logical_next = 0;
  int key0s[PG_STAGES];                        // a stage's first key; below 0: its page is not there
  auto fetch = [&](int p0, int& pg, int& lg) { // pages p0 + lane of the item
    const int row = a.row0 + ask.i;
    const int seq = LIST ? __ldcg(a.tok_seq + row) : row;
    lg = p0 + lane + (LIST ? 0 : shared_of(row));
    const bool in = (p0 + lane) * UPP < ask.units;
    if (LIST) lg = in ? __ldcg(a.lists + ((int64_t)row * a.nkv + ask.g) * a.list_stride + p0 + lane) : -1;
    pg = in && seq >= 0 && seq < a.bt_rows && lg >= 0 && lg < a.bt_width ? __ldcg(a.block_table + (int64_t)seq * a.bt_stride + lg) : -1;
    if (pg >= a.n_pages) pg = -1;
  };
  auto ask_next = [&]() {
    if (ask_x >= i_hi) return;
    if (ask_x == i_lo || ask_u == ask.u1) {    // another item
      ask = place_of(ask_x, i_hi);
      ask_u = ask.u0;
      batch_p = ask_u / UPP;
      fetch(batch_p, page, logical);
      fetch(batch_p + 32, page_next, logical_next);
    } else if (ask_u / UPP - batch_p == 32) {
      batch_p += 32;
      page = page_next;
      logical = logical_next;
      fetch(batch_p + 32, page_next, logical_next);
    }
    const int src = ask_u / UPP - batch_p;
    const int pg = __shfl_sync(0xffffffffu, page, src), lg = __shfl_sync(0xffffffffu, logical, src);
    const int st = ask_n % PG_STAGES;
    const int key0 = pg < 0 ? -1 : lg * PG_PAGE + (ask_u % UPP) * KS;
#pragma unroll
    for (int s = 0; s < PG_STAGES; ++s)
      if (s == st) key0s[s] = key0;
    if (lane == 0 && pg >= 0) {
      tc5::mbar_expect_tx(full + st, PG_UNIT_BYTES);
      const int y = (pg * a.nkv + ask.g) * PG_PAGE + (ask_u % UPP) * KS;
      unsigned char* dst = ring + st * PG_UNIT_BYTES;
#pragma unroll
      for (int x = 0; x < HD / 64; ++x) {
        tc5::tma_load_2d(dst + x * BOX, &map_k, full + st, 64 * x, y);
        tc5::tma_load_2d(dst + HALF + x * BOX, &map_v, full + st, 64 * x, y);
      }
    } else if (lane == 0) {
      tc5::mbar_arrive(full + st);
    }
    ++ask_u;
    ++ask_n;
    ++ask_x;
  };
  for (int s = 0; s < PG_STAGES; ++s) ask_next();

  // ---- computing ------------------------------------------------------------------------------------------------------------
  const uint32_t ring_addr = tc5::smem_u32(ring), sw = lane & 7;
  bool ok = true;
  int n = 0;                                   // units done
  if (lane == 0) sm.part_at[warp][0] = sm.part_at[warp][1] = -1;
  float m_first[2], l_first[2];                // the first part's, until the ring is free
  float m[2], l[2], o[HD / 8][4];
  bool have_first = false;
  float* const spill = a.records + ((int64_t)blockIdx.x * PG_WARPS + warp) * (PG_COLS * HD);   // (where the first part's sums wait meanwhile)
  for (int64_t x = i_lo; x < i_hi;) {
    const Place p = place_of(x, i_hi);
    const int start = sm.start[p.i], n_new = sm.n_new[p.i], pos0 = sm.pos[p.i], col0 = p.b * PG_COLS;
    const int n_cols = min(PG_COLS, n_new * a.G - col0);
    // this thread's two queries: columns gl and gl + 8
    int limit[2];
    uint32_t qf[KT][4];
    {
      const __nv_bfloat16* src[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = min(col0 + gl + 8 * e, n_new * a.G - 1), tok = c / a.G, h = c - tok * a.G;
        limit[e] = pos0 + tok;                 // the last key it sees
        src[e] = a.q + (int64_t)(start + tok) * a.q_stride + (int64_t)(p.g * a.G + h) * HD;
      }
#pragma unroll
      for (int k = 0; k < KT; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qf[k][e] = __ldcg(reinterpret_cast<const unsigned int*>(src[e & 1] + 16 * k + 8 * (e >> 1) + 2 * tl));
      }
    }
    const int first_limit = pos0 + col0 / a.G, last_limit = pos0 + (col0 + n_cols - 1) / a.G;
    m[0] = m[1] = PG_NEG;
    l[0] = l[1] = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    for (int u = p.u0; u < p.u1; ++u, ++n) {
      const int st = n % PG_STAGES;
      if (ok) ok = pg_wait(full + st, (n / PG_STAGES) & 1);
      int key0 = key0s[0];
#pragma unroll
      for (int s = 1; s < PG_STAGES; ++s)
        if (s == st) key0 = key0s[s];
      if (ok && key0 >= 0 && key0 <= last_limit) {
        const unsigned char* vals = ring + st * PG_UNIT_BYTES + HALF;
        const uint32_t kb = ring_addr + st * PG_UNIT_BYTES, vb = kb + HALF;
        // Values that a query does not see may be anything, and its probability of 0 would be multiplied with them.  Those that no query
        // of the item sees are taken as zeros; where one that some see is not finite, all that not everyone sees are added query by query.
        const bool edge = key0 + KS - 1 > first_limit;
        int cut = last_limit;                  // the last key whose values the products take
        if (edge && first_limit < last_limit) {
          bool odd = false;
          for (int w = lane; w < KS * (HD / 8); w += 32) {
            const int key = w / (HD / 8), c = w % (HD / 8);
            if (key0 + key <= first_limit || key0 + key > last_limit) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(vals + (c / 8) * BOX + key * 128 + (((c & 7) ^ (key & 7)) << 4));
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
        uint32_t pr[KS / 16][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float p0 = pg_exp2(s[j][0] - ref[0]), p1 = pg_exp2(s[j][1] - ref[0]), p2 = pg_exp2(s[j][2] - ref[1]), p3 = pg_exp2(s[j][3] - ref[1]);
          l[0] += p0 + p1;
          l[1] += p2 + p3;
          pr[j >> 1][2 * (j & 1)] = pg_pack(p0, p1);
          pr[j >> 1][2 * (j & 1) + 1] = pg_pack(p2, p3);
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
              pg_mma(o[2 * d2], pr[k], b[0] & keep0, b[1] & keep1);
              pg_mma(o[2 * d2 + 1], pr[k], b[2] & keep0, b[3] & keep1);
            }
          }
        };
        if (edge) values(std::true_type()); else values(std::false_type());
        if (cut < last_limit) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
              const int key = 8 * j + e;
              const uint32_t w0 = __shfl_sync(0xffffffffu, pr[j >> 1][2 * (j & 1)], (lane & 28) + (e >> 1)), w1 = __shfl_sync(0xffffffffu, pr[j >> 1][2 * (j & 1) + 1], (lane & 28) + (e >> 1));
              if (key0 + key <= cut || key0 + key > last_limit) continue;
              const float p0 = __uint_as_float(e & 1 ? w0 & 0xffff0000u : w0 << 16), p1 = __uint_as_float(e & 1 ? w1 & 0xffff0000u : w1 << 16);
              const unsigned char* line = vals + key * 128 + 4 * tl;
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
      __syncwarp();                            // all lanes have read the stage
      if (ok) ask_next();
    }
    x += p.u1 - p.u0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    if (p.u0 == 0 && p.u1 == p.units) {
      // ---- a whole item: out with it ------------------------------------------------------------------------------------------
      const int grp = group_of(a.row0 + p.i);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = gl + 8 * e;
        if (c >= n_cols) continue;
        const int tok = (col0 + c) / a.G, h = (col0 + c) - tok * a.G;
        const int64_t th = (int64_t)(start + tok) * a.nh + p.g * a.G + h;
        if (grp >= 0) {                        // its own pages' part, for the join with the shared ones'
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(a.own + th * HD + 8 * d + 2 * tl) = make_float2(o[d][2 * e], o[d][2 * e + 1]);
          if (tl == 0) *reinterpret_cast<float2*>(a.own + (int64_t)a.T * a.nh * HD + 2 * th) = make_float2(m[e], l[e]);
        } else {
          const float inv = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<uint32_t*>(a.out + th * HD + 8 * d + 2 * tl) = pg_pack(o[d][2 * e] * inv, o[d][2 * e + 1] * inv);
        }
      }
      __syncwarp();
    } else if (x < i_hi) {
      // ---- the first part, of an item that began in the share before: it waits until the ring is free ----------------------------------------
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        *reinterpret_cast<float2*>(spill + gl * HD + 8 * d + 2 * tl) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(spill + (gl + 8) * HD + 8 * d + 2 * tl) = make_float2(o[d][2], o[d][3]);
      }
      m_first[0] = m[0]; m_first[1] = m[1]; l_first[0] = l[0]; l_first[1] = l[1];
      have_first = true;
      if (lane == 0) sm.part_at[warp][0] = p.base;
    } else {
      // ---- the last one -----------------------------------------------------------------------------------------------------------------
      PgPart<HD>& part = reinterpret_cast<PgPart<HD>*>(ring)[1];
      __syncwarp();
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        *reinterpret_cast<float2*>(&part.acc[gl][8 * d + 2 * tl]) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(&part.acc[gl + 8][8 * d + 2 * tl]) = make_float2(o[d][2], o[d][3]);
      }
      if (tl == 0) { part.m[gl] = m[0]; part.m[gl + 8] = m[1]; part.l[gl] = l[0]; part.l[gl + 8] = l[1]; }
      if (lane == 0) sm.part_at[warp][1] = p.base;
    }
  }
  if (!ok) {                                   // what was asked for must land before the block's shared memory goes away
    if (lane == 0) atomicExch(&g_pg_error, 1);
    for (int u = max(0, ask_n - PG_STAGES); u < ask_n; ++u) pg_wait(full + u % PG_STAGES, (u / PG_STAGES) & 1);
  }
  if (have_first) {
    PgPart<HD>& part = reinterpret_cast<PgPart<HD>*>(ring)[0];
    __syncwarp();
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {         // (each thread its own)
      *reinterpret_cast<float2*>(&part.acc[gl][8 * d + 2 * tl]) = *reinterpret_cast<const float2*>(spill + gl * HD + 8 * d + 2 * tl);
      *reinterpret_cast<float2*>(&part.acc[gl + 8][8 * d + 2 * tl]) = *reinterpret_cast<const float2*>(spill + (gl + 8) * HD + 8 * d + 2 * tl);
    }
    if (tl == 0) { part.m[gl] = m_first[0]; part.m[gl + 8] = m_first[1]; part.l[gl] = l_first[0]; part.l[gl + 8] = l_first[1]; }
  }
  __syncthreads();

  // ---- parts of items that shares cut, joined by all threads ------------------------------------------------------------------------------
  auto parts = [&](int k) -> const PgPart<HD>& { return reinterpret_cast<const PgPart<HD>*>(rings + (k >> 1) * PG_RING)[k & 1]; };
  constexpr int REC = PG_COLS * (HD + 2);
  float* const records = a.records + (int64_t)gridDim.x * PG_WARPS * (PG_COLS * HD);
  auto block_begin = [&](int b) { return begin(b * PG_WARPS); };
  // a block's part of an item that began before the block, or with it, and the one that goes on in the next block
  auto record = [&](int b, int64_t base) { return records + (2 * (int64_t)b + (block_begin(b) < base ? 1 : 0)) * REC; };
  auto write = [&](const Place& p, int i, float mm, float ll, float y) {
    const int c = p.b * PG_COLS + i / HD, tok = c / a.G, d = i % HD;
    const int64_t th = (int64_t)(sm.start[p.i] + tok) * a.nh + p.g * a.G + c - tok * a.G;
    if (group_of(a.row0 + p.i) >= 0) {
      a.own[th * HD + d] = y;
      if (d == 0) *reinterpret_cast<float2*>(a.own + (int64_t)a.T * a.nh * HD + 2 * th) = make_float2(mm, ll);
    } else {
      a.out[th * HD + d] = __float2bfloat16_rn(ll == 0.0f ? 0.0f : y / ll);
    }
  };
  int64_t edge_at[2] = {-1, -1};               // the items that go beyond the block: the first run's, the last run's
  for (int k0 = 0; k0 < 2 * PG_WARPS;) {
    const int64_t at = sm.part_at[k0 >> 1][k0 & 1];
    int k1 = k0 + 1;
    if (at < 0) { k0 = k1; continue; }
    while (k1 < 2 * PG_WARPS && (sm.part_at[k1 >> 1][k1 & 1] == at || sm.part_at[k1 >> 1][k1 & 1] < 0)) ++k1;      // (a warp without a part there is between)
    const Place p = place_of(at, at + 1);
    const bool whole = at >= block_begin(blockIdx.x) && at + p.units <= block_begin(blockIdx.x + 1);
    if (!whole) edge_at[at < block_begin(blockIdx.x) || at == block_begin(blockIdx.x) ? 0 : 1] = at;
    const int n_cols = min(PG_COLS, sm.n_new[p.i] * a.G - p.b * PG_COLS);
    for (int i = threadIdx.x; i < n_cols * HD; i += PG_WARPS * 32) {
      const int c = i / HD, d = i % HD;
      float mm = PG_NEG, ll = 0.0f, y = 0.0f;
      for (int k = k0; k < k1; ++k)
        if (sm.part_at[k >> 1][k & 1] == at) mm = fmaxf(mm, parts(k).m[c]);
      const float safe = mm == PG_NEG ? 0.0f : mm;
      for (int k = k0; k < k1; ++k) {
        if (sm.part_at[k >> 1][k & 1] != at) continue;
        const float f = pg_exp2(parts(k).m[c] - safe);
        ll = fmaf(parts(k).l[c], f, ll);
        y = fmaf(parts(k).acc[c][d], f, y);
      }
      if (whole) {
        write(p, i, mm, ll, y);
      } else {
        float* r = record(blockIdx.x, at);
        r[2 * PG_COLS + i] = y;
        if (d == 0) { r[c] = mm; r[PG_COLS + c] = ll; }
      }
    }
    k0 = k1;
  }
  // ---- items that blocks cut: the last of their blocks to report joins them ------------------------------------------------------------------
  if (edge_at[0] >= 0 || edge_at[1] >= 0) {
    auto block_of = [&](int64_t x) {
      int b = (int)(x * n_blocks / total);
      while (b > 0 && block_begin(b) > x) --b;
      while (b + 1 < n_blocks && block_begin(b + 1) <= x) ++b;
      return b;
    };
    __threadfence();
    __syncthreads();
    if (threadIdx.x < 2) {
      const int64_t at = edge_at[threadIdx.x];
      bool last = false;
      if (at >= 0) {
        const int ba = block_of(at), bb = block_of(at + place_of(at, at + 1).units - 1);
        last = atomicAdd(a.counters + ba, 1) == bb - ba;             // (of the items that begin in a block only one goes beyond it)
        if (last) a.counters[ba] = 0;
      }
      __threadfence();
      sm.last[threadIdx.x] = last;
    }
    __syncthreads();
    for (int e = 0; e < 2; ++e) {
      if (!sm.last[e]) continue;
      const int64_t at = edge_at[e];
      const Place p = place_of(at, at + 1);
      const int ba = block_of(at), bb = block_of(at + p.units - 1);
      const int n_cols = min(PG_COLS, sm.n_new[p.i] * a.G - p.b * PG_COLS);
      for (int i = threadIdx.x; i < n_cols * HD; i += PG_WARPS * 32) {
        const int c = i / HD;
        float mm = PG_NEG, ll = 0.0f, y = 0.0f;
#pragma unroll 8
        for (int b = ba; b <= bb; ++b) {
          const float* r = record(b, at);
          const float m1 = __ldcg(r + c), l1 = __ldcg(r + PG_COLS + c), y1 = __ldcg(r + 2 * PG_COLS + i);
          const float top = fmaxf(mm, m1), safe = top == PG_NEG ? 0.0f : top;
          const float f0 = pg_exp2(mm - safe), f1 = pg_exp2(m1 - safe);
          ll = ll * f0 + l1 * f1;
          y = y * f0 + y1 * f1;
          mm = top;
        }
        write(p, i, mm, ll, y);
      }
    }
  }
  if (!a.wait_first) pdl_wait();               // this kernel's end is then the shared pages' kernel's end, too
}

// ---- host side ----------------------------------------------------------------------------------------------------------------

constexpr int PG_SMEM = (int)(PG_SMEM_RINGS + sizeof(PgSmem) + 1024);

int pg_sms(const char* what) {                 // of the current device, 0: an error
  static int known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("%s: no device", what); return 0; }
  if (known[dev]) return known[dev];
  cudaError_t e = cudaSuccess;
  for (auto f : {(const void*)attn_pages_kernel<64, false>, (const void*)attn_pages_kernel<64, true>, (const void*)attn_pages_kernel<128, false>, (const void*)attn_pages_kernel<128, true>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, PG_SMEM);
  if (e == cudaSuccess) e = attn_shared_prepare();
  int sms = 0;
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess || sms < 1) { set_error("%s: cannot get %d bytes of shared memory: %s", what, PG_SMEM, cudaGetErrorString(e)); return 0; }
  return known[dev] = sms;
}

// Where the warps' first parts wait, and the blocks' parts.
static int64_t pg_record_floats(int sms, int hd) { return (int64_t)sms * (PG_WARPS * PG_COLS * hd + 2 * PG_COLS * (hd + 2)); }
// With groups: the plan, the parts of shared pages, the rows' own parts.
constexpr int64_t PS_PLAN_FLOATS = (sizeof(PsPlan) + 63) / 64 * 16;
static int64_t ps_slots(int sms, int64_t T, int G, int nkv, int n_groups) { return sms + nkv * (T * G / PS_TILE + n_groups); }
static int64_t ps_floats(int sms, int64_t T, int G, int nkv, int hd, int n_groups) {
  return n_groups ? PS_PLAN_FLOATS + ps_slots(sms, T, G, nkv, n_groups) * ps_record(hd) + ps_own(T, G * nkv, hd) : 0;
}

template <bool LIST> static int pg_launch(PgArgs a, const CUtensorMap& map_k, const CUtensorMap& map_v, int hd, int sms, const char* what, cudaStream_t stream) {
  for (int r0 = 0; r0 < a.rows; r0 += PG_WINDOW) {
    a.row0 = r0;
    a.wait_first = r0 > 0 || a.n_groups == 0;
    auto go = [&](auto kernel) { launch_pdl(kernel, dim3(sms), dim3(PG_WARPS * 32), PG_SMEM, stream, map_k, map_v, a); };
    if (hd == 64) go(attn_pages_kernel<64, LIST>); else go(attn_pages_kernel<128, LIST>);
    const int rc = launch_status(what);
    if (rc) return rc;
  }
  return 0;
}

// What both entry points ask of their arguments, and the pools' maps.
static int pg_check(const char* what, const void* q, int64_t q_stride, const void* out, const void* k_pool, const void* v_pool, int64_t n_pages, const int* block_table,
                    int bt_width, int rows, int T, int nh, int nkv, int hd, float scale, CUtensorMap* map_k, CUtensorMap* map_v) {
  if (rows < 0 || T < 0 || nkv < 1 || nh < nkv || nh % nkv || (hd != 64 && hd != 128) || !(scale > 0.0f) || !isfinite(scale) || n_pages < 1 ||
      (n_pages + 1) * nkv * PG_PAGE > INT32_MAX || bt_width < 1 || bt_width > PG_MAX_WIDTH || (int64_t)T * (nh / nkv) > INT32_MAX - PG_COLS) {
    set_error("%s: needs heads of 64 or 128, a positive scale, tables of at most %d pages and pools of fewer than 2^31 tokens times key/value heads, got %d rows, %d tokens, %d "
              "heads on %d of %d, scale %g, %lld pages, a table of %d", what, PG_MAX_WIDTH, rows, T, nh, nkv, hd, (double)scale, (long long)n_pages, bt_width);
    return ERR_BAD_ARGUMENT;
  }
  if (!q || !out || !k_pool || !v_pool || !block_table) { set_error("%s: an array is missing", what); return ERR_BAD_ARGUMENT; }
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_pool) || !aligned16(v_pool) || q_stride % 8) {
    set_error("%s: q, its rows, out and the pools must be 16-byte aligned", what);
    return ERR_ALIGNMENT;
  }
  const int box = hd == 64 ? 32 : 16;
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
  return PG_COUNTERS + pg_record_floats(sms, hd) + ps_floats(sms, T, nh / nkv, nkv, hd, n_groups);
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
  return pg_launch<true>(a, map_k, map_v, hd, sms, "attn_pages", stream);
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
  PsPlan* plan = reinterpret_cast<PsPlan*>(scratch + PG_COUNTERS + pg_record_floats(sms, hd));
  float* parts = reinterpret_cast<float*>(plan) + PS_PLAN_FLOATS;
  a.own = parts + (n_groups ? ps_slots(sms, T, a.G, nkv, n_groups) * ps_record(hd) : 0);
  if (n_groups) {
    PsArgs p = {};
    p.q = a.q; p.q_stride = q_stride; p.block_table = block_table; p.bt_stride = bt_stride; p.bt_width = bt_width; p.n_pages = (int)n_pages; p.row_start = row_start;
    p.row_pos0 = row_pos0; p.rows = rows; p.T = T; p.nkv = nkv; p.G = a.G; p.groups = groups; p.n_groups = n_groups; p.scale_log2 = a.scale_log2; p.records = parts; p.plan = plan;
    rc = attn_shared_launch(p, k_pool, v_pool, hd, sms, stream);
    if (rc) return rc;
  }
  rc = pg_launch<false>(a, map_k, map_v, hd, sms, "attn_shared", stream);
  return rc || !n_groups ? rc : attn_shared_join(plan, parts, a.own, a.out, T, nh, nkv, hd, stream);
}
