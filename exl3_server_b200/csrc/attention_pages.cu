// Attention over lists of pages of the paged key/value cache, bfloat16, heads of 64 or 128, pages of 64 keys: the pages that were chosen for each token and
// key/value head, or the pages of a row behind those that it shares with others.
//
//   s[j] = (q . K[j]) * scale  over the keys of the listed pages at positions <= pos;   out = sum_j softmax(s)[j] V[j]
//
// One pass with running maximum and sum (float32; probabilities are rounded to bfloat16 for the second product, as in the other attention kernels here).
// Which queries walk, which have tiles and how much scratch memory that takes is settled in one place (ps_choose).
// Bound by memory: a key and a value are read once, for all query heads of their head and all tokens of the item (64 tokens, 64 chosen pages each of 32 heads of 128 on 8: 1.04 GB
// in 184 us, 5.7 TB/s).  Mean blocks end at 137 us of these and the last at 168: equal shares of bytes are not equal times for all SMs.  Few and short rows take what
// a chain of dependent reads takes, row, page number, page, softmax: 8 to 15 us.
#include "api.h"
#include "attention_pages.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <math.h>
#include <type_traits>

namespace exl3 {

constexpr int PG_WARPS = 8;                    // of a block, one block an SM: two a scheduler, whose chains of one unit's steps overlap
constexpr int PG_STAGES = 3;                   // of a warp's ring
constexpr int PG_UNIT_BYTES = 8192;            // a unit: keys and values of 32 tokens (heads of 64) or 16 (heads of 128)
constexpr int PG_WINDOW = 1024;                // rows of a launch
constexpr int PG_MIN_UNITS = 4;                // places of a warp's share, at least
constexpr int PG_ALONE = 4;                    // units by which a share may be longer so that blocks cut no item
constexpr int PG_MAX_WIDTH = 1 << 19;          // pages of a row
constexpr int PG_RING = PG_STAGES * PG_UNIT_BYTES;
constexpr uint32_t PG_SMEM_RINGS = PG_WARPS * PG_RING;
constexpr int PG_MAX_COLS = 16;                // queries of an item
constexpr int PG_ITEMS = 42;                   // bits of a sum of places
static_assert(PG_WINDOW <= 1024, "sums of 2^31 places and 2,048 items a row");

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
  int count;                                   // entries of a list
  const int* row_start;                        // rows
  const int* row_pos0;
  int rows, T, nh, nkv, G;
  int row0, window;                            // the first row of this launch, and how many it takes
  float scale_log2;
  int* counters;
  float* records;
  // the shared pages' parts
  const int* groups;
  int n_groups;
  int many;                                    // whether rows of more than PS_MANY queries are another kernel's work
  int tiles;                                   // whether the kernel before works on shared pages, or on rows of many queries
  int wait_first;                              // whether the kernel before must have ended
  int* late;                                   // where the blocks with work are counted (plus 1) for those that begin when the kernel before leaves them an SM; 0: not yet, null: no such
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
// An 8 x 8 matrix of 16-bit elements, a pair to a lane, transposed across the warp.
__device__ inline uint32_t pg_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
template <int V> __device__ inline void pg_store(float* p, const float (&y)[V]) {
  if (V == 4) *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[V - 2], y[V - 1]);
  else *reinterpret_cast<float2*>(p) = make_float2(y[0], y[1]);
}
template <int V> __device__ inline void pg_load(const float* p, float (&y)[V]) {
  if (V == 4) { const float4 v = *reinterpret_cast<const float4*>(p); y[0] = v.x; y[1] = v.y; y[V - 2] = v.z; y[V - 1] = v.w; }
  else { const float2 v = *reinterpret_cast<const float2*>(p); y[0] = v.x; y[1] = v.y; }
}
template <int V> __device__ inline void pg_load_cg(const float* p, float (&y)[V]) {
  if (V == 4) { const float4 v = __ldcg(reinterpret_cast<const float4*>(p)); y[0] = v.x; y[1] = v.y; y[V - 2] = v.z; y[V - 1] = v.w; }
  else { const float2 v = __ldcg(reinterpret_cast<const float2*>(p)); y[0] = v.x; y[1] = v.y; }
}
// Bounded, and one answer for the warp.  The hardware may hold a look for a while.
__device__ inline bool pg_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = tc5::smem_u32(bar);
  uint32_t there = 0;
#pragma unroll 1
  for (uint32_t i = 0; i < tc5::WAIT_LIMIT && !there; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(there) : "r"(addr), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, there);
}

constexpr float PG_NEG = -INFINITY;

// A warp's part of an item, at the start of its ring when the ring is done with: two of them at most, of the item that its share begins in and
// of the one that it ends in.
template <int HD, int COLS> struct PgPart {
  float m[COLS], l[COLS], acc[COLS][HD];
};
// An item, and where in it a share is.
// (base: the place of its first unit; places: of the share's)
struct PgPlace { int i, g, b, u0, u1, units, base, places; };
struct PgRun { PgPlace p; int k0, k1; bool whole, own; };
template <int HD> struct PgSmem {
  uint64_t full[PG_WARPS][PG_STAGES];
  PgRun run[2 * PG_WARPS];
  int n_runs, edge[2];
  int cum[PG_WINDOW + 1];                      // places of the rows before
  int start[PG_WINDOW], n_new[PG_WINDOW], pos[PG_WINDOW], units[PG_WINDOW];
  int shared[PG_WINDOW];                       // the pages that the row shares, -1: it is in no group
  PgPlace part_of[PG_WARPS][2];                // the warps' parts' items; units 0: none
  unsigned long long warp_sum[PG_WARPS];
  int last[2], late;
  int most, rows_end;                          // units of the longest row; the token behind the last row
  int odd_key[PG_WARPS][HD];                   // per feature the first key whose value is not finite among those that not all of an item's queries see
  PgGroups groups;
  int group_queries[PG_MAX_GROUPS];
  unsigned long long cost;                     // of the groups' tiles
};

// Keys are the rows of the first product and queries its columns, S^T = K Q^T (8 columns an instruction; NC of them side by side), and the second is O^T = V^T P^T: half
// the instructions that queries as 16 rows would take for up to 8 of them.
//
// Items: up to 8 NC queries (token, query head) of a row (or of a listed token) and key/value head, which walk the same pages.  The list of all items, ordered by row, head and
// item, with PG_SETUP places and one for each unit, is cut into equal shares for the warps, which stream them through rings of their own, each asking for its own copies: nothing is waited for but
// memory.  What a warp has whole it writes out; parts of items that shares cut are joined in shared memory at the end, and those that blocks cut by the block that
// is the last to report, always in the order of the pages, so that results do not depend on which it was.
//
// The memory's queue is full while the units stream, and code that is met for the first time then comes in at its end, as does anything else: what runs once is kept short.
template <int HD, int NC, bool LIST>
__global__ void __launch_bounds__(PG_WARPS * 32, 1)
attn_pages_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PgArgs a) {
  constexpr int COLS = 8 * NC;
  constexpr int KS = HD == 64 ? 32 : 16;       // keys of a unit
  constexpr int UPP = PG_PAGE / KS;            // units of a page
  constexpr int MT = KS / 16;                  // tiles of 16 keys
  constexpr int KT = HD / 16;                  // pieces of 16 features
  constexpr int BOX = KS * 128;                // bytes of a box of 64 features
  constexpr int HALF = PG_UNIT_BYTES / 2;      // keys, then values
  constexpr int V = HD / 32;                   // features a lane, where a warp has a row of them
  using Part = PgPart<HD, COLS>;
  static_assert(2 * sizeof(Part) <= PG_RING, "a warp's parts fit into its ring");
  extern __shared__ unsigned char pg_raw[];
  unsigned char* rings = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(pg_raw) + 1023) & ~(uintptr_t)1023);
  PgSmem<HD>& sm = *reinterpret_cast<PgSmem<HD>*>(rings + PG_SMEM_RINGS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, tl = lane & 3;
  if (threadIdx.x < PG_WARPS * PG_STAGES) tc5::mbar_init(&sm.full[0][0] + threadIdx.x, 1);
  if (threadIdx.x < 32) tc5::mbar_init_fence();
  // The kernel before is, with shared pages, the one that works on them: it let this one start when its own predecessors had ended, and this one needs nothing of it.
  // Else everything is waited for here.
  if (a.wait_first) pdl_wait();
  pdl_trigger();

  const int rows_end = !LIST && threadIdx.x == 0 ? min(max(__ldcg(a.row_start + a.rows), 0), a.T) : 0;
  const int late = !LIST && a.late && threadIdx.x == 0 ? __ldcg(a.late) : 0;
  const int3 asked = !LIST ? pg_group_asked(a.groups, a.n_groups) : make_int3(0, 0, 0);
  // ---- the rows of this launch -------------------------------------------------------------------------------------------
  const int most_keys = a.bt_width * PG_PAGE, n_rows = min(a.rows - a.row0, a.window);
#pragma unroll 1
  for (int i = threadIdx.x; i < n_rows; i += PG_WARPS * 32) {
    const int row = a.row0 + i;
    // (a row beyond the table sees all of it; a listed token's position says how many entries are looked at, too)
    sm.pos[i] = LIST ? __ldcg(a.tok_pos + row) : max(PG_LOWEST, min(most_keys, __ldcg(a.row_pos0 + row)));
    const int start = LIST ? row : min(max(__ldcg(a.row_start + row), 0), a.T);
    sm.start[i] = start;
    sm.n_new[i] = LIST ? 1 : max(0, min(__ldcg(a.row_start + row + 1), a.T) - start);
  }
  int* const group_alone = &sm.odd_key[0][0];  // (before the units need the place)
  if (!LIST && a.n_groups > 0) for (int j = threadIdx.x; j < a.n_groups; j += PG_WARPS * 32) { sm.group_queries[j] = 0; group_alone[j] = 0; }
  if (threadIdx.x == 0) { sm.cost = 0; sm.most = 0; sm.late = late; sm.rows_end = rows_end; }
  if (LIST) __syncthreads();
  else pg_groups(sm.groups, asked, a.n_groups, a.rows, a.bt_width);
  if (!LIST && sm.late > 0 && (int)blockIdx.x >= sm.late - 1) {      // (began late: the blocks that have work are others)
    if (!a.wait_first) pdl_wait();
    return;
  }
  if (!LIST && a.many && a.n_groups > 0) {     // groups that are worth it, as the tensor cores' kernel finds them, of all rows
    auto start_of = [&](int r) { return r == a.rows ? sm.rows_end : a.rows <= a.window ? sm.start[r] : min(max(__ldcg(a.row_start + r), 0), a.T); };
#pragma unroll 1
    for (int r = threadIdx.x; r < a.rows; r += PG_WARPS * 32) {
      const int n = max(start_of(r + 1) - start_of(r), 0) * a.G, j = sm.groups.of(r);
      if (j >= 0 && n > 0) atomicAdd(&group_alone[j], ps_alone(n, COLS, HD));
    }
    __syncthreads();
    if ((int)threadIdx.x < a.n_groups) {
      const int r0 = sm.groups.first[threadIdx.x], s0 = start_of(r0), s1 = max(start_of(r0 + sm.groups.rows[threadIdx.x]), s0);
      if (!ps_worth((s1 - s0) * a.G, sm.groups.pages[threadIdx.x], group_alone[threadIdx.x])) sm.groups.pages[threadIdx.x] = 0;
    }
    __syncthreads();
  }
  // items << PG_ITEMS | places: of all rows, and of those up to this thread's last one.  A row counts no more than 2,048 of the first (items matter where there are fewer than SMs) and
  // 2^31 of the second, so that neither sum passes its bits.
  unsigned long long totals = 0, upto = 0;
  constexpr unsigned long long PLACES = (1ull << PG_ITEMS) - 1;
#pragma unroll 1
  for (int i0 = 0; i0 < n_rows; i0 += PG_WARPS * 32) {
    const int i = i0 + threadIdx.x;
    int units = 0;
    int64_t blocks = 0;
    if (i < n_rows) {
      const int pos = sm.pos[i], queries = sm.n_new[i] * a.G, j = LIST ? -1 : sm.groups.of(a.row0 + i), shared = j < 0 ? -1 : sm.groups.pages[j];
      units = LIST ? min(a.count, pos < 0 ? 0 : pos / PG_PAGE + 1) * UPP : (min(pos + sm.n_new[i], most_keys) + KS - 1) / KS - max(shared, 0) * UPP;
      units = max(units, 1);                   // (one at least: every query gets an answer)
      sm.shared[i] = shared;
      sm.units[i] = units;
      blocks = (int64_t)(!LIST && a.many && queries > PS_MANY ? 0 : (queries + COLS - 1) / COLS) * a.nkv;
      if (j >= 0) atomicAdd(&sm.group_queries[j], queries);
    }
    const int longest = __reduce_max_sync(0xffffffffu, blocks ? units : 0);
    if (lane == 0) atomicMax(&sm.most, longest);
    unsigned long long incl = (unsigned long long)min(blocks, (int64_t)2048) << PG_ITEMS | (unsigned long long)min((units + PG_SETUP) * blocks, (int64_t)1 << 31);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
    if (lane == 31) sm.warp_sum[warp] = incl;
    __syncthreads();
    upto = totals + incl;
#pragma unroll
    for (int w = 0; w < PG_WARPS; ++w) { if (w < warp) upto += sm.warp_sum[w]; totals += sm.warp_sum[w]; }
    if (i < n_rows) sm.cum[i + 1] = (int)(upto & PLACES);
    __syncthreads();
  }
  // The host has seen that rows of up to max_new tokens have fewer than 2^31 places; more tokens than that may have more: nothing is done for them, and the status says so.
  const bool too_many = (totals & PLACES) > INT32_MAX;
  if (too_many && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(&g_pg_error, 2);
  int total = too_many ? 0 : (int)(totals & PLACES);
  if (threadIdx.x == 0) sm.cum[0] = 0;
  const bool beside = !LIST && a.n_groups > 0 && !a.many && a.rows <= a.window;     // the other kernel leaves this one some of the SMs
  if (beside)
#pragma unroll 1
    for (int j = threadIdx.x; j < a.n_groups; j += PG_WARPS * 32)
      if (sm.groups.pages[j] > 0 && sm.group_queries[j] > 0) atomicAdd(&sm.cost, (unsigned long long)ps_cost(sm.group_queries[j], sm.groups.pages[j]));
  __syncthreads();
  int sms = gridDim.x;
  if (beside && sm.cost > 0) {
    sms -= ps_sms((int64_t)sm.cost * a.nkv, total, COLS, gridDim.x);
    if (sms < 1) sms = gridDim.x;
  }
  int n_blocks = min(sms, max(1, total / (PG_WARPS * PG_MIN_UNITS))), setup = PG_SETUP, padded = 0;
  // Few items get a block each, padded to one length, where that makes no share much longer than equal shares are: no item is cut by blocks then, and no share has two items.
  const int items = (int)(totals >> PG_ITEMS), each = (sm.most + PG_WARPS - 1) / PG_WARPS;
  if (items > 0 && items <= sms && n_rows <= PG_WARPS * 32 && each <= total / (n_blocks * PG_WARPS) + PG_ALONE) {
    n_blocks = items;
    setup = 0;
    padded = PG_WARPS * each;
    total = items * padded;
    if ((int)threadIdx.x < n_rows) sm.cum[threadIdx.x + 1] = (int)(upto >> PG_ITEMS) * padded;
    __syncthreads();
  }
  if (!LIST && a.late && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(a.late, (total ? n_blocks : 0) + 1);
  const int n_shares = n_blocks * PG_WARPS;
  if (total == 0 || (int)blockIdx.x >= n_blocks) {
    if (!a.wait_first) pdl_wait();
    return;
  }
  const int per = total / n_shares, rem = total - per * n_shares;
  auto begin = [&](int w) { return per * w + min(w, rem); };           // the first unit of a warp's share: they differ by one unit at most
  const int i_lo = begin(blockIdx.x * PG_WARPS + warp), i_hi = begin(blockIdx.x * PG_WARPS + warp + 1);
  // The item at place x.
  auto place_of = [&](int x) {
    int lo = 0, hi = n_rows - 1;
#pragma unroll 1
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (sm.cum[mid] <= x) lo = mid; else hi = mid - 1; }
    PgPlace p;
    p.i = lo;
    p.units = sm.units[lo];
    const int all = padded ? padded : p.units + PG_SETUP, r = x - sm.cum[lo], item = r / all, nb = (sm.n_new[lo] * a.G + COLS - 1) / COLS, at = r - item * all;
    p.places = min(all - at, i_hi - x);
    p.u0 = min(max(at - setup, 0), p.units);   // (no units where the share has the item's first places only, or the padding)
    p.u1 = min(max(at + p.places - setup, 0), p.units);
    p.g = item / nb;
    p.b = item - p.g * nb;
    p.base = x - at + setup;
    return p;
  };

  unsigned char* const ring = rings + warp * PG_RING;
  uint64_t* const full = sm.full[warp];
  // ---- copies: page numbers come 32 at a time, a batch ahead -----------------------------------------------------------------
  int ask_x = i_lo, ask_n = 0, ask_st = 0;     // the next item to ask for; units asked for, and the next one's stage
  PgPlace ask = {};
  int ask_u = 0, batch_p = 0;                  // its number in the item; the first page of the batch at hand
  int page = 0, logical = 0, page_next = 0, logical_next = 0;
  int key0s[PG_STAGES];                        // a stage's first key; below 0: its page is not there
  auto ask_next = [&]() {
    int batches = 0;                           // to ask for: two for another item
    if (ask_u == ask.u1) {
      do {
        if (ask_x >= i_hi) return;
        ask = place_of(ask_x);
        ask_x += ask.places;
        ask_u = ask.u0;
      } while (ask.u1 == ask.u0);
      batch_p = ask_u / UPP;
      batches = 2;
    } else if (ask_u / UPP - batch_p == 32) {
      batch_p += 32;
      batches = 1;
    }
#pragma unroll 1
    for (; batches > 0; --batches) {
      page = page_next;
      logical = logical_next;
      const int p = batch_p + (batches == 2 ? 0 : 32) + lane, row = a.row0 + ask.i, seq = LIST ? __ldcg(a.tok_seq + row) : row;
      const bool in = p * UPP < ask.units && seq >= 0 && seq < a.bt_rows;
      logical_next = LIST ? in ? __ldcg(a.lists + ((int64_t)row * a.nkv + ask.g) * a.count + p) : -1 : p + max(sm.shared[ask.i], 0);
      page_next = in && logical_next >= 0 && logical_next < a.bt_width ? __ldcg(a.block_table + (int64_t)seq * a.bt_stride + logical_next) : -1;
      if (page_next >= a.n_pages) page_next = -1;
    }
    const int src = ask_u / UPP - batch_p, pg = __shfl_sync(0xffffffffu, page, src), lg = __shfl_sync(0xffffffffu, logical, src);
    const int key0 = pg < 0 ? -1 : lg * PG_PAGE + (ask_u % UPP) * KS;
#pragma unroll
    for (int s = 0; s < PG_STAGES; ++s)
      if (s == ask_st) key0s[s] = key0;
    if (lane == 0 && pg >= 0) {
      tc5::mbar_expect_tx(full + ask_st, PG_UNIT_BYTES);
      const int y = (pg * a.nkv + ask.g) * PG_PAGE + (ask_u % UPP) * KS;
      unsigned char* dst = ring + ask_st * PG_UNIT_BYTES;
#pragma unroll
      for (int x = 0; x < HD / 64; ++x) {
        tc5::tma_load_2d(dst + x * BOX, &map_k, full + ask_st, 64 * x, y);
        tc5::tma_load_2d(dst + HALF + x * BOX, &map_v, full + ask_st, 64 * x, y);
      }
    } else if (lane == 0) {
      tc5::mbar_arrive(full + ask_st);
    }
    if (++ask_st == PG_STAGES) ask_st = 0;
    ++ask_u;
    ++ask_n;
  };
  // ---- computing ------------------------------------------------------------------------------------------------------------
  const uint32_t ring_addr = tc5::smem_u32(ring);
  // ldmatrix: a row at 128 bytes, its 16-byte piece c at c ^ (row & 7)
  const uint32_t k_row = ((lane & 7) + ((lane >> 3) & 1) * 8) * 128, v_row = ((lane & 7) + ((lane >> 4) & 1) * 8) * 128 + HALF;
  uint32_t k_col[4], v_col[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    k_col[j] = (uint32_t)(((2 * j + (lane >> 4)) ^ (lane & 7)) << 4);
    v_col[j] = (uint32_t)(((2 * j + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
  }
  bool ok = true;
  int st = 0;                                  // the next unit's stage, and its phase
  uint32_t phase = 0;
  if (lane < 2) sm.part_of[warp][lane].units = 0;
  float m[NC][2], l[NC][2], o[KT][NC][4];
  float m_first[NC][2], l_first[NC][2];        // the first part's, until the ring is free
  bool have_first = false, odd = false;
  float* const spill = a.records + ((int64_t)blockIdx.x * PG_WARPS + warp) * (PG_MAX_COLS * HD);   // (where the first part's sums wait meanwhile)
  uint32_t qf[NC][KT][2];                      // the query of column 8 nc + gl as the operand: features 16 k + 2 tl, + 1 and + 8, + 9
  PgPlace p = {};
  int x = i_lo, u = 0, first_limit = 0, last_limit = 0;
  int limit[NC][2] = {};                       // the last keys that this thread's two queries of each 8 see: columns 2 tl, 2 tl + 1
  bool begun = false;
  // (one loop for the first copies, the items and their units: the code of each stands here once)
#pragma unroll 1
  for (int step = -PG_STAGES;; ++step) {
    if (step >= 0) {
    if (u == p.u1) {
    // the next item's queries on their way, then the sums of the one that is done
    const PgPlace done = p;
    bool more = false;
#pragma unroll 1
    while (!more && x < i_hi) {
      p = place_of(x);
      x += p.places;
      more = p.u1 > p.u0;
    }
    if (more) {
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        const int c = min(p.b * COLS + 8 * nc + gl, sm.n_new[p.i] * a.G - 1), tok = c / a.G;
        const __nv_bfloat16* src = a.q + (int64_t)(sm.start[p.i] + tok) * a.q_stride + (int64_t)(p.g * a.G + c - tok * a.G) * HD + 2 * tl;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          qf[nc][k][0] = __ldcg(reinterpret_cast<const unsigned int*>(src + 16 * k));
          qf[nc][k][1] = __ldcg(reinterpret_cast<const unsigned int*>(src + 16 * k + 8));
        }
      }
    }
    if (begun) {
      const int col0 = done.b * COLS, n_cols = min(COLS, sm.n_new[done.i] * a.G - col0);
      auto query_of = [&](int c) {             // (token, head)
        const int tok = (col0 + c) / a.G;
        return (int64_t)(sm.start[done.i] + tok) * a.nh + done.g * a.G + (col0 + c) - tok * a.G;
      };
#pragma unroll
      for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nc][e] += __shfl_xor_sync(0xffffffffu, l[nc][e], d);
        }
      if (odd) {                               // features whose values are not finite are not, for those who see them
        __syncwarp();
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
          for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sm.odd_key[warp][16 * i + 8 * (e >> 1) + gl] <= sm.pos[done.i] + min(col0 + 8 * nc + 2 * tl + (e & 1), col0 + n_cols - 1) / a.G) o[i][nc][e] = __int_as_float(0x7fc00000);
      }
      const bool whole = done.u0 == 0 && done.u1 == done.units;
      if (whole && sm.shared[done.i] < 0) {
        // ---- a whole item: out with it ----------------------------------------------------------------------------------------
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          const int c = 8 * nc + gl;           // (after the transposition)
          const float i0 = l[nc][0] == 0.0f ? 0.0f : 1.0f / l[nc][0], i1 = l[nc][1] == 0.0f ? 0.0f : 1.0f / l[nc][1];
          __nv_bfloat16* dst = a.out + query_of(min(c, n_cols - 1)) * HD + 2 * tl;
#pragma unroll
          for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const uint32_t w = pg_transpose(pg_pack(o[i][nc][2 * f] * i0, o[i][nc][2 * f + 1] * i1));
              if (c < n_cols) *reinterpret_cast<uint32_t*>(dst + 16 * i + 8 * f) = w;
            }
        }
      } else {
        // ---- rows of hd floats: the own pages' part of a row that shares pages; or a part of an item, the first one (of an item that began in the share before) where
        // it can wait until the ring is free, the last one in the ring --------------------------------------------------------------------------
        const bool first = !whole && more;
        Part& part = reinterpret_cast<Part*>(ring)[1];
        __syncwarp();
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = 8 * nc + 2 * tl + e;
            float* const dst = whole ? a.own + query_of(min(c, n_cols - 1)) * HD : first ? spill + c * HD : part.acc[c];
            if (!whole || c < n_cols) {
#pragma unroll
              for (int i = 0; i < KT; ++i) { dst[16 * i + gl] = o[i][nc][e]; dst[16 * i + 8 + gl] = o[i][nc][2 + e]; }
              if (gl == 0) {
                if (whole) *reinterpret_cast<float2*>(a.own + (int64_t)a.T * a.nh * HD + 2 * query_of(c)) = make_float2(m[nc][e], l[nc][e]);
                else if (!first) { part.m[c] = m[nc][e]; part.l[c] = l[nc][e]; }
              }
            }
            if (first) { m_first[nc][e] = m[nc][e]; l_first[nc][e] = l[nc][e]; }
          }
        have_first |= first;
        if (!whole && lane == 0) sm.part_of[warp][first ? 0 : 1] = done;
        __syncwarp();
      }
    }
    if (!more) break;
    // ---- the item's units ---------------------------------------------------------------------------------------------------------------
    begun = true;
    const int n_new = sm.n_new[p.i], pos0 = sm.pos[p.i], col0 = p.b * COLS;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        limit[nc][e] = pos0 + min(col0 + 8 * nc + 2 * tl + e, n_new * a.G - 1) / a.G;
        m[nc][e] = PG_NEG;
        l[nc][e] = 0.0f;
      }
    first_limit = pos0 + col0 / a.G;
    last_limit = pos0 + min(col0 + COLS - 1, n_new * a.G - 1) / a.G;
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) o[i][nc][0] = o[i][nc][1] = o[i][nc][2] = o[i][nc][3] = 0.0f;
    odd = false;
    u = p.u0;
    }
    {
      if (ok) ok = pg_wait(full + st, phase);
      int key0 = key0s[0];
#pragma unroll
      for (int i = 1; i < PG_STAGES; ++i)
        if (i == st) key0 = key0s[i];
      if (ok && key0 >= 0 && key0 <= last_limit) {
        const uint32_t unit = ring_addr + st * PG_UNIT_BYTES;
        const bool edge = key0 + KS - 1 > first_limit;
        if (edge) {
          // Values that not all queries see may be anything, and a probability of 0 is multiplied with them all the same: those that are not finite become zeros, and where
          // some queries see them it is noted from which key on the feature is not finite.
          unsigned char* vals = ring + st * PG_UNIT_BYTES + HALF;
          bool any = false;
#pragma unroll 4
          for (int w = max(first_limit + 1 - key0, 0) * (HD / 8) + lane; w < KS * (HD / 8); w += 32) {
            const int key = w / (HD / 8), c = w % (HD / 8);
            const uint4 v = *reinterpret_cast<const uint4*>(vals + (c / 8) * BOX + key * 128 + (((c & 7) ^ (key & 7)) << 4));
            any |= pg_odd(v.x) || pg_odd(v.y) || pg_odd(v.z) || pg_odd(v.w);
          }
          if (__any_sync(0xffffffffu, any)) {
            if (!odd)
#pragma unroll 1
              for (int d = lane; d < HD; d += 32) sm.odd_key[warp][d] = INT32_MAX;
            odd = true;
            __syncwarp();
#pragma unroll 1
            for (int w = max(first_limit + 1 - key0, 0) * HD + lane; w < KS * HD; w += 32) {
              const int key = w / HD, d = w % HD;
              __nv_bfloat16* v = reinterpret_cast<__nv_bfloat16*>(vals + (d / 64) * BOX + key * 128 + ((((d / 8) & 7) ^ (key & 7)) << 4)) + d % 8;
              if (isfinite(__bfloat162float(*v))) continue;
              *v = __float2bfloat16(0.0f);
              if (key0 + key <= last_limit) atomicMin(&sm.odd_key[warp][d], key0 + key);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
        }
        float s[MT][NC][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int nc = 0; nc < NC; ++nc) s[t][nc][0] = s[t][nc][1] = s[t][nc][2] = s[t][nc][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t kf[4];
            pg_ldsm(kf, unit + (k >> 2) * BOX + 16 * t * 128 + k_row + k_col[k & 3]);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) pg_mma(s[t][nc], kf, qf[nc][k][0], qf[nc][k][1]);
          }
        // rows of a tile: keys gl and gl + 8; columns: queries 2 tl and 2 tl + 1
        float mx[NC][2];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[t][nc][e] *= a.scale_log2;
              if (edge && key0 + 16 * t + gl + 8 * (e >> 1) > limit[nc][e & 1]) s[t][nc][e] = PG_NEG;
            }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = fmaxf(s[0][nc][e], s[0][nc][2 + e]);
#pragma unroll
            for (int t = 1; t < MT; ++t) v = fmaxf(v, fmaxf(s[t][nc][e], s[t][nc][2 + e]));
            mx[nc][e] = v;
          }
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
          for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int e = 0; e < 2; ++e) mx[nc][e] = fmaxf(mx[nc][e], __shfl_xor_sync(0xffffffffu, mx[nc][e], d));
        bool grows = false;
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
          for (int e = 0; e < 2; ++e) grows |= mx[nc][e] > m[nc][e];
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float mn = fmaxf(m[nc][e], mx[nc][e]), f = m[nc][e] == PG_NEG ? 0.0f : pg_exp2(m[nc][e] - mn);
              l[nc][e] *= f;
              m[nc][e] = mn;
#pragma unroll
              for (int i = 0; i < KT; ++i) { o[i][nc][e] *= f; o[i][nc][2 + e] *= f; }
            }
        }
        // probabilities: packed by pairs of queries, turned into pairs of keys for the second product
        uint32_t pk[MT][NC][2];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          const float r0 = m[nc][0] == PG_NEG ? 0.0f : m[nc][0], r1 = m[nc][1] == PG_NEG ? 0.0f : m[nc][1];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float p0 = pg_exp2(s[t][nc][2 * h] - r0), p1 = pg_exp2(s[t][nc][2 * h + 1] - r1);
              l[nc][0] += p0;
              l[nc][1] += p1;
              pk[t][nc][h] = pg_transpose(pg_pack(p0, p1));
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int i = 0; i < KT; ++i) {
            uint32_t vf[4];
            pg_ldsm_t(vf, unit + (i >> 2) * BOX + 16 * t * 128 + v_row + v_col[i & 3]);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) pg_mma(o[i][nc], vf, pk[t][nc][0], pk[t][nc][1]);
          }
      }
      __syncwarp();                            // all lanes have read the stage
      ++u;
      if (++st == PG_STAGES) { st = 0; phase ^= 1; }
    }
    }
    if (ok) ask_next();
  }
  if (!ok) {                                   // what was asked for must land before the block's shared memory goes away
    if (lane == 0) atomicExch(&g_pg_error, 1);
#pragma unroll 1
    for (int u = max(0, ask_n - PG_STAGES); u < ask_n; ++u) pg_wait(full + u % PG_STAGES, (u / PG_STAGES) & 1);
  }
  if (have_first) {
    Part& part = reinterpret_cast<Part*>(ring)[0];
    __syncwarp();
#pragma unroll 4
    for (int i = lane; i < COLS * HD / 4; i += 32) reinterpret_cast<float4*>(part.acc[0])[i] = reinterpret_cast<const float4*>(spill)[i];
    if (gl == 0)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int e = 0; e < 2; ++e) { part.m[8 * nc + 2 * tl + e] = m_first[nc][e]; part.l[8 * nc + 2 * tl + e] = l_first[nc][e]; }
  }
  __syncthreads();

  // ---- parts of items that shares cut: runs of the warps' parts, a warp for a run's query, a lane for V features of it -----------------------------------
  constexpr int REC = COLS * (HD + 2);
  float* const records = a.records + (int64_t)gridDim.x * PG_WARPS * (PG_MAX_COLS * HD);
  const int block_lo = begin(blockIdx.x * PG_WARPS), block_hi = begin((blockIdx.x + 1) * PG_WARPS);
  auto block_of = [&](int at) {                // (per is 0 only where there is one block)
    const int longer = rem * (per + 1);        // units of the longer shares
    return (at < longer ? at / (per + 1) : rem + (at - longer) / max(per, 1)) / PG_WARPS;
  };
  if (warp == 0) {                             // a lane for each of the warps' parts, which stand one behind the other
    const PgPlace& q = sm.part_of[0][lane % (2 * PG_WARPS)];
    const bool there = lane < 2 * PG_WARPS && q.units != 0;
    const uint32_t below = (1u << lane) - 1, before = __ballot_sync(0xffffffffu, there) & below;
    const int base = q.base, base_before = __shfl_sync(0xffffffffu, base, before ? 31 - __clz(before) : 0);
    const bool begins = there && (!before || base_before != base), whole = base >= block_lo && base + q.units <= block_hi;
    const uint32_t all = __ballot_sync(0xffffffffu, begins), after = all & ~below & ~(1u << lane);
    const int n = __popc(all & below);
    if (lane < 2) sm.edge[lane] = -1;
    __syncwarp();
    if (begins) {
      PgRun& r = sm.run[n];
      r.p = q;
      r.k0 = lane;
      r.k1 = after ? __ffs(after) - 1 : 2 * PG_WARPS;
      r.whole = whole;
      r.own = sm.shared[q.i] >= 0;
      if (!whole) sm.edge[base <= block_lo ? 0 : 1] = n;
    }
    if (lane == 0) sm.n_runs = __popc(all);
  }
  __syncthreads();
  // column c of a run's item, this lane's features
  auto write = [&](const PgRun& r, int c, float mm, float ll, const float (&y)[V]) {
    const int cc = r.p.b * COLS + c, tok = cc / a.G;
    const int64_t th = (int64_t)(sm.start[r.p.i] + tok) * a.nh + r.p.g * a.G + cc - tok * a.G;
    if (r.own) {
      pg_store(a.own + th * HD + lane * V, y);
      if (lane == 0) *reinterpret_cast<float2*>(a.own + (int64_t)a.T * a.nh * HD + 2 * th) = make_float2(mm, ll);
    } else {
      const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
      for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(a.out + th * HD + lane * V + i) = pg_pack(y[i] * inv, y[i + 1] * inv);
    }
  };
  // a running sum, and a part more
  auto add = [&](float& mm, float& ll, float (&y)[V], float m1, float l1, const float (&y1)[V]) {
    const float top = fmaxf(mm, m1), safe = top == PG_NEG ? 0.0f : top, f0 = pg_exp2(mm - safe), f1 = pg_exp2(m1 - safe);
    ll = ll * f0 + l1 * f1;
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = y[v] * f0 + y1[v] * f1;
    mm = top;
  };
#pragma unroll 1
  for (int k = 0; k < sm.n_runs; ++k) {
    const PgRun& r = sm.run[k];
    const int n_cols = min(COLS, sm.n_new[r.p.i] * a.G - r.p.b * COLS);
    // a block's record of an item that began before the block, or with it, and of the one that goes on in the next block
    float* const rec = records + (2 * blockIdx.x + (block_lo < r.p.base ? 1 : 0)) * REC;
#pragma unroll 1
    for (int c = warp; c < n_cols; c += PG_WARPS) {
      float mm = PG_NEG, ll = 0.0f, y[V] = {};
#pragma unroll 1
      for (int i = r.k0; i < r.k1; ++i) {
        if (sm.part_of[0][i].units == 0) continue;         // (a warp without a part there may be between)
        const Part& part = reinterpret_cast<const Part*>(rings + (i >> 1) * PG_RING)[i & 1];
        float y1[V];
        pg_load(&part.acc[c][lane * V], y1);
        add(mm, ll, y, part.m[c], part.l[c], y1);
      }
      if (r.whole) {
        write(r, c, mm, ll, y);
      } else {
        pg_store(rec + 2 * COLS + c * HD + lane * V, y);
        if (lane == 0) { rec[c] = mm; rec[COLS + c] = ll; }
      }
    }
  }
  // ---- items that blocks cut: the last of their blocks to report joins them ------------------------------------------------------------------
  if (sm.edge[0] >= 0 || sm.edge[1] >= 0) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x < 2) {
      const int k = sm.edge[threadIdx.x];
      bool last = false;
      if (k >= 0) {
        const PgPlace& q = sm.run[k].p;
        const int ba = block_of(q.base), bb = block_of(q.base + q.units - 1);
        last = atomicAdd(a.counters + ba, 1) == bb - ba;             // (of the items that begin in a block only one goes beyond it)
        if (last) a.counters[ba] = 0;
      }
      __threadfence();
      sm.last[threadIdx.x] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      if (!sm.last[e]) continue;
      const PgRun& r = sm.run[sm.edge[e]];
      const int ba = block_of(r.p.base), n = block_of(r.p.base + r.p.units - 1) - ba + 1, n_cols = min(COLS, sm.n_new[r.p.i] * a.G - r.p.b * COLS);
      // the records of blocks ba .. ba + n - 1: all but the first are their blocks' first
      const float* const rec0 = records + (2 * ba + (begin(ba * PG_WARPS) < r.p.base ? 1 : 0)) * REC;
#pragma unroll 1
      for (int c = warp; c < n_cols; c += PG_WARPS) {
        float mm = PG_NEG, ll = 0.0f, y[V] = {};
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 4) {
          float m1[4], l1[4], y1[4][V];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* q = i0 + i > 0 && i0 + i < n ? records + 2 * (ba + i0 + i) * REC : rec0;
            m1[i] = __ldcg(q + c);
            l1[i] = __ldcg(q + COLS + c);
            pg_load_cg(q + 2 * COLS + c * HD + lane * V, y1[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i0 + i < n) add(mm, ll, y, m1[i], l1[i], y1[i]);
        }
        write(r, c, mm, ll, y);
      }
    }
  }
  if (!a.wait_first) pdl_wait();               // this kernel's end is then the shared pages' kernel's end, too
}

// ---- host side ----------------------------------------------------------------------------------------------------------------

static_assert(sizeof(PgSmem<64>::odd_key) >= PG_MAX_GROUPS * sizeof(int), "the groups' sums lie there first");
constexpr int PG_SMEM = (int)(PG_SMEM_RINGS + sizeof(PgSmem<128>) + 1024);
static_assert(PG_SMEM <= 232448, "what a block may have");

int pg_sms(const char* what) {                 // of the current device, 0: an error
  static int known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("%s: no device", what); return 0; }
  if (known[dev]) return known[dev];
  cudaError_t e = cudaSuccess;
  for (auto f : {(const void*)attn_pages_kernel<64, 1, false>, (const void*)attn_pages_kernel<64, 1, true>, (const void*)attn_pages_kernel<128, 1, false>,
                 (const void*)attn_pages_kernel<128, 1, true>, (const void*)attn_pages_kernel<64, 2, false>, (const void*)attn_pages_kernel<64, 2, true>,
                 (const void*)attn_pages_kernel<128, 2, false>, (const void*)attn_pages_kernel<128, 2, true>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, PG_SMEM);
  if (e == cudaSuccess) e = attn_shared_prepare();
  int sms = 0;
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess || sms < 1) { set_error("%s: cannot get %d bytes of shared memory: %s", what, PG_SMEM, cudaGetErrorString(e)); return 0; }
  return known[dev] = sms;
}

// Where the warps' first parts wait, and the blocks' parts.
static int64_t pg_record_floats(int sms, int hd) { return (int64_t)sms * (PG_WARPS * PG_MAX_COLS * hd + 2 * PG_MAX_COLS * (hd + 2)); }
// With tiles: their parts' places, the tokens, the tiles' parts, the rows' own parts.
struct PsSpace { int64_t parts, tokens, records, own, end; };                  // floats from the start of this part of the scratch memory
static PsSpace ps_space(int sms, int64_t T, int G, int nkv, int hd, int tiles) {
  PsSpace s = {};
  auto after = [](int64_t at, int64_t n) { return (at + n + 15) / 16 * 16; };
  s.tokens = after(0, 4 * (int64_t)tiles * nkv);
  s.records = after(s.tokens, 4 * T);
  s.own = after(s.records, ps_slots(sms, nkv, tiles) * ps_record(hd));
  s.end = after(s.own, ps_own(T, G * nkv, hd));
  return s;
}
static int pg_cols(int max_new, int G) { return (int64_t)max_new * G <= 8 ? 8 : 16; }
// As many rows a launch as have fewer than 2^31 units together.
static int pg_window(const PgArgs& a, int hd, int max_new, bool list) {
  const int cols = pg_cols(max_new, a.G);
  const int64_t queries = a.many ? PS_MANY : (int64_t)max_new * a.G, row = ((int64_t)(list ? a.count : a.bt_width) * (hd / 32) + PG_SETUP) * a.nkv * ((queries + cols - 1) / cols);
  return (int)std::min<int64_t>(PG_WINDOW, INT32_MAX / row);
}
template <bool LIST> static int pg_launch(PgArgs a, const CUtensorMap& map_k, const CUtensorMap& map_v, int hd, int max_new, int sms, const char* what, cudaStream_t stream) {
  const int cols = pg_cols(max_new, a.G);
  a.window = pg_window(a, hd, max_new, LIST);
  if (a.window < 1) { set_error("%s: rows of %d pages and %d tokens of %d query heads on %d are too long", what, a.bt_width, max_new, a.nh, a.nkv); return ERR_UNSUPPORTED; }
  for (int r0 = 0; r0 < a.rows; r0 += a.window) {
    a.row0 = r0;
    a.wait_first = r0 > 0 || !a.tiles;
    auto go = [&](auto kernel) { launch_pdl(kernel, dim3(sms), dim3(PG_WARPS * 32), PG_SMEM, stream, map_k, map_v, a); };
    if (cols == 8) { if (hd == 64) go(attn_pages_kernel<64, 1, LIST>); else go(attn_pages_kernel<128, 1, LIST>); }
    else { if (hd == 64) go(attn_pages_kernel<64, 2, LIST>); else go(attn_pages_kernel<128, 2, LIST>); }
    const int rc = launch_status(what);
    if (rc) return rc;
  }
  return 0;
}

// Whether a call reads so little that its rows had better read the shared pages each for itself: two launches less, and no join.  Both sides over 2 to 32 rows of 2 to 64
// shared pages and five layouts of heads, graph time: up to 100 MB of units all of them are faster alone (8 rows of 8 pages, 32 heads on 8 of 128, 21 MB: 16.7 against 27.4 us; 32 rows
// of 8 pages, 84 MB: 22.8 against 28.7), at 140 to 160 MB they meet (29.2 against 29.1, 27.5 against 28.4, 31.4 against 29.5).  The tables' width stands for the rows' lengths,
// which only the GPU knows.
static bool pg_alone(int rows, int bt_width, int max_new, int G, int nkv, int hd) {
  const double units = (double)rows * (((int64_t)max_new * G + PG_MAX_COLS - 1) / PG_MAX_COLS) * bt_width * nkv;
  return units * PG_PAGE * hd * 4 <= 128e6;
}

// What a call works with: the one place where that is settled, so that the scratch memory is asked for, checked and laid out for the same tiles.  (Fewer groups can mean more tiles:
// without their tiles rows of many tokens may have tiles of their own.)
struct PsChoice {
  int groups;                                  // the caller's, or 0 where they are left alone
  bool many;                                   // whether rows of many tokens are the tensor cores' work
  int64_t tiles;                               // of a key/value head, at most; 0: no call of that kernel
};
// Groups are what may be shared, not what must be: where their tiles are more than the list holds, the rows read for themselves.
static PsChoice ps_choose(int64_t T, int G, int rows, int n_groups, int max_new, int bt_width, int nkv, int hd) {
  auto fits = [&](int64_t tiles) { return tiles <= PS_MAX_TILES && tiles * (bt_width + PS_SETUP) * nkv <= INT32_MAX; };
  const bool many = (int64_t)max_new * G > PS_MANY && rows <= PS_MAX_ROWS;
  const int groups = n_groups && pg_alone(rows, bt_width, max_new, G, nkv, hd) ? 0 : n_groups;
  const int64_t both = ps_most_tiles(T, G, groups, rows), shared = T * G / PS_TILE + groups, own = ps_most_tiles(T, G, 0, rows);
  if (many && fits(both)) return {groups, true, both};
  if (groups && fits(shared)) return {groups, false, shared};
  if (many && fits(own)) return {0, true, own};
  return {0, false, 0};
}
// Floats of scratch for it.
static int64_t ps_floats(const PsChoice& c, int sms, int64_t T, int G, int nkv, int hd) {
  return PG_COUNTERS + pg_record_floats(sms, hd) + (c.tiles ? ps_space(sms, T, G, nkv, hd, (int)c.tiles).end : 0);
}

// What both entry points ask of their arguments, and the pools' maps.
static int pg_check(const char* what, const void* q, int64_t q_stride, const void* out, const void* k_pool, const void* v_pool, int64_t n_pages, const int* block_table,
                    int bt_width, int rows, int T, int nh, int nkv, int hd, float scale, CUtensorMap* map_k, CUtensorMap* map_v) {
  if (rows < 0 || T < 0 || nkv < 1 || nkv > 4096 || nh < nkv || nh % nkv || (hd != 64 && hd != 128) || !(scale > 0.0f) || !isfinite(scale) || n_pages < 1 ||
      (n_pages + 1) * nkv * PG_PAGE > INT32_MAX || bt_width < 1 || bt_width > PG_MAX_WIDTH || (int64_t)T * (nh / nkv) > INT32_MAX - PG_MAX_COLS) {
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

// Floats of scratch that a call over lists wants; the first PG_COUNTERS must be zero before the first call and are zero after each.
extern "C" long long exl3_attn_pages_scratch(int sms, int hd) { return PG_COUNTERS + pg_record_floats(sms, hd); }
// The same for a call over rows; chosen (may be null): the groups that are used, whether rows of many tokens have tiles of their own, the most tiles of a key/value head.
extern "C" long long exl3_attn_shared_scratch(int sms, int T, int rows, int nh, int nkv, int hd, int n_groups, int max_new, int bt_width, int* chosen) {
  if (nkv < 1 || nh < nkv) return 0;
  const PsChoice c = ps_choose(T, nh / nkv, rows, n_groups, std::min(max_new, T), bt_width, nkv, hd);
  if (chosen) { chosen[0] = c.groups; chosen[1] = c.many; chosen[2] = (int)c.tiles; }
  return ps_floats(c, sms, T, nh / nkv, nkv, hd);
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
  if (!scratch || scratch_floats < exl3_attn_pages_scratch(sms, hd)) { set_error("attn_pages: scratch too small"); return ERR_SCRATCH; }
  PgArgs a = pg_args(q, q_stride, out, n_pages, block_table, bt_stride, bt_width, T, T, nh, nkv, scale, scratch);
  a.tok_pos = tok_pos; a.tok_seq = tok_seq; a.lists = lists; a.count = count; a.bt_rows = bt_rows;
  return pg_launch<true>(a, map_k, map_v, hd, 1, sms, "attn_pages", stream);
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
  max_new = std::min(max_new, T);              // (no row brings more)
  const PsChoice c = ps_choose(T, nh / nkv, rows, n_groups, max_new, bt_width, nkv, hd);
  const int64_t tiles = c.tiles;
  n_groups = c.groups;
  if (!scratch || scratch_floats < ps_floats(c, sms, T, nh / nkv, nkv, hd)) { set_error("attn_shared: scratch too small"); return ERR_SCRATCH; }
  PgArgs a = pg_args(q, q_stride, out, n_pages, block_table, bt_stride, bt_width, rows, T, nh, nkv, scale, scratch);
  a.row_start = row_start; a.row_pos0 = row_pos0; a.bt_rows = rows; a.groups = groups; a.n_groups = n_groups;
  a.tiles = tiles > 0;
  a.many = c.many;
  PsArgs p = {};
  if (tiles) {
    float* at = scratch + PG_COUNTERS + pg_record_floats(sms, hd);
    const PsSpace s = ps_space(sms, T, a.G, nkv, hd, (int)tiles);
    p.q = a.q; p.q_stride = q_stride; p.block_table = block_table; p.bt_stride = bt_stride; p.bt_width = bt_width; p.n_pages = (int)n_pages; p.row_start = row_start;
    p.row_pos0 = row_pos0; p.rows = rows; p.T = T; p.nkv = nkv; p.G = a.G; p.groups = groups; p.n_groups = n_groups; p.many = a.many; p.scale_log2 = a.scale_log2;
    p.parts = reinterpret_cast<int*>(at + s.parts); p.most_tiles = (int)tiles; p.sms = sms; p.tokens = reinterpret_cast<PsToken*>(at + s.tokens);
    p.cols = pg_cols(max_new, a.G); p.window = pg_window(a, hd, max_new, false); p.hd = hd;
    p.records = at + s.records;
    a.own = at + s.own;
    if (rows <= p.window) a.late = a.counters + PG_COUNTERS - 1;
    rc = attn_shared_launch(p, k_pool, v_pool, hd, sms, stream);
    if (rc) return rc;
  }
  rc = pg_launch<false>(a, map_k, map_v, hd, max_new, sms, "attn_shared", stream);
  return rc || !tiles ? rc : attn_shared_join(p, a.own, a.out, a.counters + PG_COUNTERS - 1, hd, stream);
}
