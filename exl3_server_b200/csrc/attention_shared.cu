// Attention of many queries over the same pages on the 5th-generation tensor cores (bfloat16, heads of 64 or 128, pages of 64 keys): the pages that the rows of a group
// share, whose keys are read once for up to PS_TILE queries (token, query head of the key/value head) of whatever rows, and a row's own pages where it brings many tokens.
//
//   m = max_j s_j,  l = sum_j 2^(s_j - m),  y = sum_j 2^(s_j - m) V[j]    over a part's pages, s_j = (q . K[j]) * scale * log2 e
//
// A part's (m, l, y) of every query goes to a record in float32; a second kernel joins the records of a query, with the part that attention_pages.cu worked out of its
// row's own pages.  Scores, maxima, sums and joins are float32; a probability is rounded to bfloat16 for the second product (up to 2^-8 of it, as an operand of the
// tensor cores has to be), while l takes it unrounded: results are off by 0.0023 of their norm where their own rounding alone gives 0.0017.
//
// Two sets of 128 queries stand side by side in a block, each with four softmax warps (thread = query = row of tensor memory), and take turns with
// the tensor core: S = Q K^T into one of two buffers of 64 columns, P over the columns of its own S, O += P V.  The maximum that the exponentials are
// taken against moves only when a row's true maximum has grown by more than 2^8, so that O is rescaled rarely.  Blocks are persistent, one an SM,
// and take equal shares of the list of pages (attention_pages.cuh), whatever the tiles' sizes.
//
// What bounds it (24 prompts of 16 to 120 tokens behind 94 pages, 32 heads of 128 on 8: 208 us, 163 GFLOP): a page for 256 queries takes 2,090 clocks, of which the softmax threads
// compute 1,000 and wait 900 for S, whose buffer is free when the product before the last has ended: handing over P, product, barrier, product, barrier.  No unit is full: the tensor
// pipe is busy 0.35 of the time, and with a quarter of the products, without exponentials, or without copies a call took 3 % less.  A warp more, so that each set has its own
// for S, changed nothing.  With 168 registers a thread, the most that eleven warps leave, 30 bytes are spilled at heads of 128 and 80 at 64.
// Where an elected lane issues the products (not lane 0 of a branch) one takes 25 to 36 clocks instead of 70.
//
// Every wait is bounded: a kernel that gives up leaves a code (exl3_attn_shared_status), frees its tensor memory and ends.
#include "api.h"
#include "attention_pages.cuh"
#include "tcgen05.cuh"

#include <math.h>

namespace exl3 {

using namespace tc5;

constexpr int PS_THREADS = 352;
constexpr float PS_RESCALE_STEP = 8.0f;        // base-2 units
constexpr uint32_t PS_BOX = PG_PAGE * 128;     // bytes of 64 features of a page
static __device__ int g_ps_error = 0;

__host__ __device__ constexpr uint32_t ps_q_bytes(int hd) { return 128 * hd * 2; }
__host__ __device__ constexpr uint32_t ps_page_bytes(int hd) { return PG_PAGE * hd * 2; }
// Queries and pages share this much: two sets of queries and 4 pages of heads of 128 (10 of 64), or one set and 5 (11).
__host__ __device__ constexpr uint32_t ps_ring(int hd) { return 196608; }
__host__ __device__ constexpr int ps_stages(int hd, bool one) { return (int)((ps_ring(hd) - (one ? 1 : 2) * ps_q_bytes(hd)) / (2 * ps_page_bytes(hd))); }
constexpr int PS_MAX_STAGES = 11;

// The list of tiles, in shared memory.
struct PsTiles {
  PsPlan plan;
  int cum[PS_MAX_TILES + 1];                   // places of the tiles before
  int start[PS_MAX_ROWS + 1], pos[PS_MAX_ROWS];          // the rows' first tokens and their positions, where there are no more rows than that
  int tok0[PS_MAX_TILES], query0[PS_MAX_TILES], queries[PS_MAX_TILES], row[PS_MAX_TILES], page0[PS_MAX_TILES];
  PgGroups groups;
  int group_tile[PG_MAX_GROUPS], group_tok[PG_MAX_GROUPS], group_seen[PG_MAX_GROUPS];  // first tile, first token, the first token's position of the row that has the lowest
  int row_tile[PS_MAX_ROWS];                   // a row's own first tile, -1: none
  int warp_sum[PS_THREADS / 32];
  int small;                                   // no tile has more than 128 queries
  int sms;                                     // for this kernel
  unsigned long long places, cost;             // of the walk, and the tiles'
  int odd_key[2][3][128];                      // per set, in turns (a warp may be two parts behind another), and feature: the first key whose value is not finite among those that not all of the tile's queries see
  int odd[2][3];
};
struct PsBars {
  uint64_t q_full[2], q_free, kv_full[PS_MAX_STAGES], kv_free[PS_MAX_STAGES], s_full[4], p_full[4], pv_done[4];
  uint32_t tmem_slot;
};
__host__ __device__ constexpr uint32_t ps_smem(int hd) { return ps_ring(hd) + (uint32_t)sizeof(PsTiles) + (uint32_t)sizeof(PsBars) + 1024; }
static_assert(ps_smem(128) <= 232448, "what a block may have");

// S: M = 128, N = 64, both operands K-major; P V: N = the head's features, V as it lies (keys down, features across).
constexpr uint32_t PS_IDESC_S = idesc_bf16(128, 64);
__host__ __device__ constexpr uint32_t ps_idesc_pv(int hd) { return idesc_bf16(128, hd) | (1u << 16); }
// V of more than 64 features: the second box lies PS_BOX behind the first.
template <int HD> __device__ inline uint64_t ps_desc_v(uint32_t addr) {
  const uint64_t d = smem_desc_k128(addr);
  return HD == 64 ? d : (d & ~(0x3fffull << 16)) | ((uint64_t)(PS_BOX >> 4) << 16);
}
// The first operand from tensor memory: rows are lanes, two bfloat16 to a column.
__device__ inline void ps_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
// D (+)= A B^T, both in shared memory.
__device__ inline void ps_mma_ss(uint32_t d_tmem, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
// One lane of a whole warp, always the same one.
__device__ inline bool ps_elect() {
  uint32_t it;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(it));
  return it != 0;
}
__device__ inline void ps_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ inline void ps_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ inline float ps_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ inline uint32_t ps_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ inline float ps_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Bounded, and one answer for the warp.  The hardware may hold a look for a while.
__device__ inline bool ps_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  uint32_t there = 0;
#pragma unroll 1
  for (uint32_t i = 0; i < WAIT_LIMIT && !there; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(there) : "r"(addr), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, there);
}
// Whether one of a word's two bfloat16 is not finite.
__device__ inline bool ps_odd(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
// One arrival for the warp, when all its lanes are here.
__device__ inline void ps_arrive_warp(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ inline float ps_row_max(const uint32_t (&lo)[32], const uint32_t (&hi)[32]) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};          // (four chains)
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    mx[(c >> 1) & 1] = ps_max3(mx[(c >> 1) & 1], __uint_as_float(lo[c]), __uint_as_float(lo[c + 1]));
    mx[2 + ((c >> 1) & 1)] = ps_max3(mx[2 + ((c >> 1) & 1)], __uint_as_float(hi[c]), __uint_as_float(hi[c + 1]));
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// 2^(s * mul - ref) of 32 scores as bfloat16, two to a word; pairs of neighbours share the instructions of multiply-add and sum.
__device__ inline void ps_exponentials(const uint32_t (&s)[32], float mul, float ref, uint32_t* p, unsigned long long (&sum)[2]) {
  unsigned long long mul2, ref2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(mul2) : "f"(mul));
  asm("mov.b64 %0, {%1, %1};" : "=l"(ref2) : "f"(-ref));
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    unsigned long long x, e;
    float e0, e1;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "r"(s[2 * c]), "r"(s[2 * c + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(x), "l"(mul2), "l"(ref2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(x));
    e0 = ps_exp2(e0);
    e1 = ps_exp2(e1);
    asm("mov.b64 %0, {%1, %2};" : "=l"(e) : "f"(e0), "f"(e1));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum[c & 1]) : "l"(e));
    p[c] = ps_pack(e0, e1);
  }
}
// 32 bytes: a whole sector of a line, where each lane has a row of its own.
__device__ inline void ps_store8(float* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// This thread's row of O times f.
template <int HD> __device__ inline void ps_rescale(uint32_t taddr, float f) {
#pragma unroll
  for (int h = 0; h < HD / 32; ++h) {
    uint32_t o[32];
    tmem_ld32(taddr + 32 * h, o);
#pragma unroll
    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
    ps_st32(taddr + 32 * h, o);
  }
  ps_wait_st();
  fence_before();
}

// The list of tiles; by all threads of a block, ends with a barrier.  The same in every block.
__device__ inline void ps_tiles(PsTiles& t, const PsArgs& a) {
  const bool held = a.rows <= PS_MAX_ROWS;     // the rows' arrays are here
  const int most = a.bt_width * PG_PAGE;       // (a row beyond the table sees all of it)
  auto start_of = [&](int r) { return held ? t.start[r] : min(max(__ldcg(a.row_start + r), 0), a.T); };
  auto pos_of = [&](int r) { return held ? t.pos[r] : min(__ldcg(a.row_pos0 + r), most); };
  const int3 asked = pg_group_asked(a.groups, a.n_groups);
  if (held)
#pragma unroll 1
    for (int r = threadIdx.x; r <= a.rows; r += PS_THREADS) {
      t.start[r] = min(max(__ldcg(a.row_start + r), 0), a.T);
      if (r < a.rows) t.pos[r] = min(__ldcg(a.row_pos0 + r), most);
    }
  static_assert(sizeof(t.odd_key) >= PG_MAX_GROUPS * sizeof(int), "the groups' sums lie there first");
  int* const group_alone = &t.odd_key[0][0][0];
  if ((int)threadIdx.x < a.n_groups) group_alone[threadIdx.x] = 0;
  pg_groups(t.groups, asked, a.n_groups, a.rows, a.bt_width);
  if (a.many && a.n_groups > 0) {
#pragma unroll 1
    for (int r = threadIdx.x; r < a.rows; r += PS_THREADS) {
      const int n = max(start_of(r + 1) - start_of(r), 0) * a.G, j = t.groups.of(r);
      if (j >= 0 && n > 0) atomicAdd(&group_alone[j], ps_alone(n, a.cols, a.hd));
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int j = threadIdx.x; j < a.n_groups; j += PS_THREADS) {
    const int r0 = t.groups.first[j], s0 = start_of(r0), s1 = max(start_of(r0 + t.groups.rows[j]), s0);
    if (a.many && !ps_worth((s1 - s0) * a.G, t.groups.pages[j], group_alone[j])) t.groups.pages[j] = 0;
    t.group_tok[j] = s0;
    t.group_tile[j] = t.groups.pages[j] > 0 ? (s1 - s0) * a.G : 0;     // (queries, for now)
    t.group_seen[j] = INT32_MAX;
  }
  // rows of many tokens: their queries, for now, and what of the shared pages a group's rows see
  const int n_rows = a.many ? a.rows : 0;
  if (threadIdx.x == 0) t.places = t.cost = 0;
  __syncthreads();
  int64_t places = 0;
  const int ks = a.hd == 64 ? 32 : 16;
#pragma unroll 1
  for (int r = threadIdx.x; r < a.rows; r += PS_THREADS) {
    const int s0 = start_of(r), s1 = start_of(r + 1), j = t.groups.of(r);
    if (j >= 0 && s1 > s0) atomicMin(&t.group_seen[j], pos_of(r));
    if (s1 > s0) {                             // (as the walk does)
      const int blocks = ((s1 - s0) * a.G + a.cols - 1) / a.cols;
      places += (int64_t)(PG_SETUP + max(1, (min(max(pos_of(r), PG_LOWEST) + s1 - s0, most) + ks - 1) / ks - (j >= 0 ? t.groups.pages[j] : 0) * (PG_PAGE / ks))) * blocks;
    }
    if (r < n_rows) t.row_tile[r] = s1 > s0 && (int64_t)(s1 - s0) * a.G > PS_MANY ? (s1 - s0) * a.G : 0;
  }
  __syncthreads();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) places += __shfl_xor_sync(0xffffffffu, places, o);
  if ((threadIdx.x & 31) == 0 && places) atomicAdd(&t.places, (unsigned long long)places);
#pragma unroll 1
  for (int j = threadIdx.x; j < a.n_groups; j += PS_THREADS)
    if (t.group_tile[j]) atomicAdd(&t.cost, (unsigned long long)ps_cost(t.group_tile[j], t.groups.pages[j]));
  // places: groups, then rows, a thread each, in rounds of the block
  int n_tiles = 0, small = 1;
#pragma unroll 1
  for (int i0 = 0; i0 < a.n_groups + n_rows; i0 += PS_THREADS) {
    const int i = i0 + threadIdx.x;
    const bool group = i < a.n_groups;
    const int queries = group ? t.group_tile[i] : i - a.n_groups < n_rows ? t.row_tile[i - a.n_groups] : 0;
    const int mine = (queries + PS_TILE - 1) / PS_TILE, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
    if (lane == 31) t.warp_sum[warp] = incl;
    small &= __syncthreads_and(queries <= 128);
    int at = n_tiles + incl - mine;
#pragma unroll 1
    for (int w = 0; w < PS_THREADS / 32; ++w) { if (w < warp) at += t.warp_sum[w]; n_tiles += t.warp_sum[w]; }
    if (i < a.n_groups + n_rows) {
      const int row = group ? t.groups.first[i] : i - a.n_groups;
      const int own = group ? -1 : t.groups.of(row), page0 = own >= 0 ? t.groups.pages[own] : 0;
      const int tok0 = group ? t.group_tok[i] : start_of(row), pos0 = group ? 0 : pos_of(row);
#pragma unroll 1
      for (int k = 0; k < mine && at + k < PS_MAX_TILES; ++k) {
        const int q0 = k * PS_TILE, n = min(PS_TILE, queries - q0), last = pos0 + (q0 + n - 1) / a.G;
        t.tok0[at + k] = tok0;
        t.query0[at + k] = q0;
        t.queries[at + k] = n;
        t.row[at + k] = group ? row : -1 - row;          // (below 0: the row's own pages, which its queries do not see alike)
        t.page0[at + k] = page0;
        // (one page at least: a query that sees nothing of its own has a part all the same)
        t.cum[at + k + 1] = PS_SETUP + (group ? t.groups.pages[i] : max(1, min(a.bt_width, (max(last, 0) + PG_PAGE) / PG_PAGE) - page0));
      }
      if (group) t.group_tile[i] = mine ? at : -1;
      else t.row_tile[row] = mine ? at : -1;
    }
    __syncthreads();
  }
  n_tiles = min(n_tiles, a.most_tiles);        // (rows that are not one behind the other could make more than there are places for)
  if (threadIdx.x < 32) {                      // running sums, a warp
    int run = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < n_tiles; i0 += 32) {
      const int i = i0 + threadIdx.x;
      int incl = i < n_tiles ? t.cum[i + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, incl, o); if ((int)threadIdx.x >= o) incl += v; }
      if (i < n_tiles) t.cum[i + 1] = run + incl;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (threadIdx.x == 0) {
      PsPlan& p = t.plan;
      t.cum[0] = 0;
      t.small = small;
      // (beside rows of many tokens the walk has little to do, and of more rows than a launch of it takes it knows no more than these)
      t.sms = a.many || a.rows > a.window ? (int)gridDim.x : ps_sms(t.cost * a.nkv, t.places * a.nkv, a.cols, gridDim.x);
      p.n_tiles = n_tiles;
      p.total = run * a.nkv;                   // (the host has seen that it stays within 31 bits)
      p.blocks = min(t.sms, max(1, p.total / PS_MIN_PAGES));
      p.per = p.total / p.blocks;
      p.rem = p.total - p.per * p.blocks;
    }
  }
  __syncthreads();
}
// A part of the list that one block works on.
struct PsPart { int g, tile, p0, p1, places; };          // kv head, tile, pages of the tile (none where a share has the tile's first places only), places of the list
__device__ inline PsPart ps_part(const PsTiles& t, int x, int end) {
  const int all = t.cum[t.plan.n_tiles];
  PsPart p;
  p.g = x / all;
  const int r = x - p.g * all;
  int lo = 0, hi = t.plan.n_tiles - 1;
#pragma unroll 1
  while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (t.cum[mid] <= r) lo = mid; else hi = mid - 1; }
  p.tile = lo;
  const int at = r - t.cum[lo];
  p.places = min(t.cum[lo + 1] - r, end - x);
  p.p0 = max(0, at - PS_SETUP);
  p.p1 = max(0, at + p.places - PS_SETUP);
  return p;
}

// warps 0-3, 4-7: softmax of the first and the second 128 queries; warp 8: S; warp 9: O; warp 10: copies of pages.
template <int HD>
__global__ void __launch_bounds__(PS_THREADS, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PsArgs a) {
  constexpr uint32_t QB = ps_q_bytes(HD), KVB = ps_page_bytes(HD);
  constexpr int BOXES = HD / 64;
  extern __shared__ unsigned char ps_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ps_raw) + 1023) & ~(uintptr_t)1023);
  PsBars& bars = *reinterpret_cast<PsBars*>(base + ps_ring(HD));
  PsTiles& tiles = *reinterpret_cast<PsTiles*>(base + ps_ring(HD) + sizeof(PsBars));
  uint64_t *q_full = bars.q_full, *kv_full = bars.kv_full, *kv_free = bars.kv_free, *s_full = bars.s_full, *p_full = bars.p_full, *pv_done = bars.pv_done;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < 2; ++i) mbar_init(q_full + i, 4);
    mbar_init(&bars.q_free, 1);
#pragma unroll 1
    for (int i = 0; i < PS_MAX_STAGES; ++i) { mbar_init(kv_full + i, 1); mbar_init(kv_free + i, 1); }
#pragma unroll 1
    for (int i = 0; i < 4; ++i) { mbar_init(s_full + i, 1); mbar_init(p_full + i, 4); mbar_init(pv_done + i, 1); }
    mbar_init_fence();
  }
  if (warp == 8) tmem_alloc<512>(&bars.tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  // The kernel that walks the rows' own pages may start when all that it reads beside the records is there: after this.
  pdl_wait();
  pdl_trigger();
  ps_tiles(tiles, a);
  const PsPlan& plan = tiles.plan;
  const uint32_t tmem = bars.tmem_slot;        // columns: scores of set s at 128 s, O at 256 + 128 s
  const int lo = (int)blockIdx.x < plan.blocks ? plan.begin(blockIdx.x) : 0, hi = (int)blockIdx.x < plan.blocks ? plan.begin(blockIdx.x + 1) : 0;
  // Tiles of more than 128 queries: both sets take every page, 128 queries each.  Smaller ones: the sets take the pages in turn, with the same queries, and where there
  // are only such tiles one copy of them, which leaves room for more pages: a page's stage is taken for a copy's way and two pages' softmax, and with 4 stages
  // a page took 0.86 us.
  auto both = [&](const PsPart& t) { return tiles.queries[t.tile] > 128; };
  const bool one = tiles.small != 0;
  const int stages = ps_stages(HD, one);
  unsigned char* const sQ = base;              // [1 or 2 sets][boxes][128][64]
  unsigned char* const sK = sQ + (one ? 1 : 2) * QB;       // [stages][boxes][64][64]
  unsigned char* const sV = sK + stages * KVB;
  const uint32_t second_q = one ? 0 : QB;
  bool ok = true;

  if (warp == 10) {
    // ---- copies; page numbers come 32 at a time, a batch ahead ------------------------------------------------------------------
    int c = 0, st = 0;
    uint32_t phase = 1;                        // of the stage's being free again
#pragma unroll 1
    for (int x = lo; x < hi && ok;) {
      const PsPart t = ps_part(tiles, x, hi);
      const int row = tiles.row[t.tile], p_off = tiles.page0[t.tile];
      const int* bt = a.block_table + (int64_t)(row < 0 ? -1 - row : row) * a.bt_stride + p_off;
      auto numbers = [&](int p) {              // beyond the pool: zeros, hidden by the softmax
        const int n = p + lane < t.p1 && p_off + p + lane < a.bt_width ? __ldcg(bt + p + lane) : a.n_pages;
        return n < 0 || n > a.n_pages ? a.n_pages : n;
      };
      int page = numbers(t.p0);
#pragma unroll 1
      for (int p = t.p0; p < t.p1 && ok; p += 32) {
        const int ahead = numbers(p + 32);
#pragma unroll 1
        for (int i = 0; i < min(32, t.p1 - p); ++i, ++c) {
          const int y = (__shfl_sync(0xffffffffu, page, i) * a.nkv + t.g) * PG_PAGE;
          if (c >= stages && !ps_wait(kv_free + st, phase)) { ok = false; break; }
          if (lane == 0) {
            mbar_expect_tx(kv_full + st, 2 * KVB);
#pragma unroll
            for (int b = 0; b < BOXES; ++b) {
              tma_load_2d(sK + st * KVB + b * PS_BOX, &map_k, kv_full + st, 64 * b, y);
              tma_load_2d(sV + st * KVB + b * PS_BOX, &map_v, kv_full + st, 64 * b, y);
            }
          }
          __syncwarp();
          if (++st == stages) { st = 0; phase ^= 1; }
        }
        page = ahead;
      }
      x += t.places;
    }
    // what was asked for must land before the block's shared memory goes away
    if (!ok && lane == 0) atomicExch(&g_ps_error, 1);
#pragma unroll 1
    for (int u = max(0, c - stages); u < c; ++u) ps_wait(kv_full + u % stages, (u / stages) & 1);
  } else if (warp == 8) {
    // ---- S = Q K^T, up to two pages ahead of the softmax -------------------------------------------------------------------
    int st = 0, f[2] = {0, 0}, k[2] = {0, 0};  // pages of a set, parts of a set so far
    uint32_t phase = 0;
#pragma unroll 1
    for (int x = lo; x < hi && ok;) {
      const PsPart t = ps_part(tiles, x, hi);
      const bool two = both(t);
#pragma unroll 1
      for (int p = t.p0; p < t.p1 && ok; ++p) {
        if (!ps_wait(kv_full + st, phase)) { ok = false; break; }
        if (one && t.p1 - t.p0 == 1 && !ps_wait(q_full + 1, k[1] & 1)) { ok = false; break; }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!two && ((p - t.p0) & 1) != s) continue;
          const int sb = f[s] & 1;
          if (p == t.p0 + (two ? 0 : s) && !ps_wait(q_full + s, k[s] & 1)) { ok = false; break; }
          if (f[s] >= 2 && !ps_wait(pv_done + 2 * s + sb, ((f[s] >> 1) - 1) & 1)) { ok = false; break; }
          fence_after();
          if (ps_elect()) {
#pragma unroll
            for (int b = 0; b < BOXES; ++b) {
              const uint64_t da = smem_desc_k128(smem_u32(sQ + s * second_q + b * 128 * 128)), db = smem_desc_k128(smem_u32(sK + st * KVB + b * PS_BOX));
#pragma unroll
              for (int i = 0; i < 4; ++i) ps_mma_ss(tmem + 128 * s + 64 * sb, da + 2 * i, db + 2 * i, PS_IDESC_S, (b | i) > 0);
            }
            mma_commit(s_full + 2 * s + sb);
            if (one && p == t.p1 - 1) mma_commit(&bars.q_free);        // (the sets share the queries' place)
          }
          __syncwarp();
          ++f[s];
        }
        if (++st == stages) { st = 0; phase ^= 1; }
      }
      k[0] += t.p1 > t.p0;
      k[1] += t.p1 - t.p0 > (two || one ? 0 : 1);              // (a set without a page asks for no queries; where the sets share them it says so)
      x += t.places;
    }
    if (!ok && lane == 0) atomicExch(&g_ps_error, 2);
  } else if (warp == 9) {
    // ---- for the join, while the first scores are on their way: the tiles' parts, and every token's tiles -------------------------------
#pragma unroll 1
    for (int i = blockIdx.x * 32 + lane; i < plan.n_tiles * a.nkv; i += gridDim.x * 32) {
      const int g = i / plan.n_tiles, tile = i - g * plan.n_tiles;
      const int first = g * tiles.cum[plan.n_tiles] + tiles.cum[tile] + PS_SETUP, last = first + tiles.cum[tile + 1] - tiles.cum[tile] - PS_SETUP - 1;
      const int b0 = plan.block_of(first), halves = tiles.queries[tile] > 128 ? 1 : 2;
      reinterpret_cast<int4*>(a.parts)[(int64_t)g * a.most_tiles + tile] = make_int4(b0 + i, (plan.block_of(last) - b0 + 1) * halves, halves, 0);
    }
#pragma unroll 1
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
      const int s0 = min(max(__ldcg(a.row_start + r), 0), a.T), s1 = min(__ldcg(a.row_start + r + 1), a.T), j = tiles.groups.of(r);
      const int4 w = make_int4(j >= 0 ? tiles.group_tile[j] : -1, j >= 0 ? tiles.group_tok[j] : 0, a.many ? tiles.row_tile[r] : -1, s0);       // a PsToken
#pragma unroll 1
      for (int i = s0 + lane; i < s1; i += 32) reinterpret_cast<int4*>(a.tokens)[i] = w;
    }
    {                                          // (tokens of no row)
      const int t0 = min(max(__ldcg(a.row_start), 0), a.T), t1 = max(t0, min(max(__ldcg(a.row_start + a.rows), 0), a.T));
#pragma unroll 1
      for (int i = blockIdx.x * 32 + lane; i < t0 + a.T - t1; i += gridDim.x * 32) reinterpret_cast<int4*>(a.tokens)[i < t0 ? i : t1 + i - t0] = make_int4(-1, 0, -1, 0);
    }
    // ---- O += P V ----------------------------------------------------------------------------------------------------------------
    int st = 0, f[2] = {0, 0}, k[2] = {0, 0};
    uint32_t phase = 0;
#pragma unroll 1
    for (int x = lo; x < hi && ok;) {
      const PsPart t = ps_part(tiles, x, hi);
      const bool two = both(t);
      const int row = tiles.row[t.tile], q0 = tiles.query0[t.tile];
      // a row's own pages: the last keys that the tile's first and last queries see
      const int own_pos = row < 0 ? min(__ldcg(a.row_pos0 - 1 - row), a.bt_width * PG_PAGE) : 0;
      const int first_limit = row < 0 ? own_pos + q0 / a.G : INT32_MAX, last_limit = own_pos + (q0 + tiles.queries[t.tile] - 1) / a.G;
#pragma unroll 1
      for (int p = t.p0; p < t.p1 && ok; ++p) {
        const int key0 = (tiles.page0[t.tile] + p) * PG_PAGE;
        if (row < 0 && key0 + PG_PAGE - 1 > first_limit) {
          // Values that not all queries see: a probability of 0 is multiplied with them all the same, so those that are not finite become zeros here, and the softmax
          // threads are told from which key on a feature is not finite (when they are known to have begun the part: they have handed over P).
          if (!ps_wait(kv_full + st, phase)) { ok = false; break; }
#pragma unroll 1
          for (int s = 0; s < 2; ++s)
            if ((two || ((p - t.p0) & 1) == s) && !ps_wait(p_full + 2 * s + (f[s] & 1), (f[s] >> 1) & 1)) { ok = false; break; }
          if (!ok) break;
#pragma unroll 1
          for (int w = lane; w < PG_PAGE * (HD / 8); w += 32) {
            const int key = w / (HD / 8), c = w % (HD / 8);
            if (key0 + key <= first_limit) continue;
            uint4* at = reinterpret_cast<uint4*>(sV + st * KVB + (c >> 3) * PS_BOX + key * 128 + (((c & 7) ^ (key & 7)) << 4));
            const uint4 v = *at;
            if (!(ps_odd(v.x) || ps_odd(v.y) || ps_odd(v.z) || ps_odd(v.w))) continue;
            __nv_bfloat16* each = reinterpret_cast<__nv_bfloat16*>(at);
            const int set = two ? -1 : (p - t.p0) & 1;
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
              if (isfinite(__bfloat162float(each[e]))) continue;
              each[e] = __float2bfloat16(0.0f);
              if (key0 + key > last_limit) continue;
#pragma unroll 1
              for (int s = 0; s < 2; ++s)
                if (set < 0 || set == s) { atomicMin(&tiles.odd_key[s][k[s] % 3][8 * c + e], key0 + key); tiles.odd[s][k[s] % 3] = 1; }
            }
          }
          fence_smem_to_tma();
          __threadfence_block();
          __syncwarp();
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!two && ((p - t.p0) & 1) != s) continue;
          const int sb = f[s] & 1;
          if (!ps_wait(p_full + 2 * s + sb, (f[s] >> 1) & 1)) { ok = false; break; }
          fence_after();
          if (ps_elect()) {
            const uint64_t db = ps_desc_v<HD>(smem_u32(sV + st * KVB));
            const bool fresh = p == t.p0 + (two ? 0 : s);            // a part's first product starts O afresh
#pragma unroll
            for (int i = 0; i < PG_PAGE / 16; ++i)                   // 16 keys: 8 columns of P, 16 rows of V
              ps_mma_ts(tmem + 256 + 128 * s, tmem + 128 * s + 64 * sb + 8 * i, db + 128 * i, ps_idesc_pv(HD), (!fresh || i > 0) ? 1u : 0u);
            mma_commit(pv_done + 2 * s + sb);
            if (!two || s == 1) mma_commit(kv_free + st);
          }
          __syncwarp();
          ++f[s];
        }
        if (++st == stages) { st = 0; phase ^= 1; }
      }
      k[0] += t.p1 > t.p0;
      k[1] += t.p1 - t.p0 > (two ? 0 : 1);
      x += t.places;
    }
    if (!ok && lane == 0) atomicExch(&g_ps_error, 3);
  } else {
    // ---- softmax ---------------------------------------------------------------------------------------------------------------
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + 128 * s, to = tmem + lanes + 256 + 128 * s;
    int f = 0, parts = 0, mine = 0;            // the set's pages so far, all parts with pages, the set's
    // The set's next part from place x on, and its queries on their way into the operand's layout: beside the last sums of the part before.
    // pos: the last key that this query sees; sees: all of the warp's queries see keys up to here; holes: some page of the part is not there.
    struct Mine { PsPart t; bool two, in, holes; int first, qr, pos, sees, turn; int64_t slot; };
    int x = lo;
    bool more = true;
    float m_used = -INFINITY, l = 0.0f;
    uint32_t s0[32], s1[32];
    Mine m = {};
#pragma unroll 1
    for (bool begun = false;; begun = true) {
      const Mine now = m;                      // the part whose last sums are on their way
#pragma unroll 1
      while (more) {                           // the next one
        more = x < hi;
        if (!more) break;
        m.t = ps_part(tiles, x, hi);
        x += m.t.places;
        if (m.t.p1 == m.t.p0) continue;
        if (one && parts > 0 && !ps_wait(&bars.q_free, (parts - 1) & 1)) { ok = false; break; }            // (every part's, whether the set has pages of it or not)
        ++parts;
        m.two = both(m.t);
        m.first = m.t.p0 + (m.two ? 0 : s);
        m.qr = s * 128 + r;
        m.slot = blockIdx.x + (int64_t)m.t.g * plan.n_tiles + m.t.tile;
        if (m.first < m.t.p1) break;
        float* rec = a.records + m.slot * ps_record(HD);       // no page for this set
        rec[m.qr] = -INFINITY;
        rec[PS_TILE + m.qr] = 0.0f;
        if (one) ps_arrive_warp(q_full + s);                   // (it asks for nothing, but no part may be two ahead of a set)
      }
      if (!ok) break;
      if (more) {
        const int in_tile = m.two ? m.qr : r;
        m.in = in_tile < tiles.queries[m.t.tile];
        const PsPart& t = m.t;
        const int query = tiles.query0[t.tile] + (m.in ? in_tile : 0), step_tok = query / a.G, tok = tiles.tok0[t.tile] + step_tok;
        m.turn = mine++ % 3;
        // the warp's 32 queries, rows of the operand (the last S that read the place is done): several of them an instruction, 16 bytes a lane
        constexpr int LANES = HD / 8, EACH = 32 / LANES;
        const int64_t from = m.in ? (int64_t)tok * a.q_stride + (int64_t)(t.g * a.G + query - step_tok * a.G) * HD : -1;
        uint4 w[LANES];
#pragma unroll
        for (int i = 0; i < LANES; ++i) {
          const int64_t at = __shfl_sync(0xffffffffu, from, EACH * i + lane / LANES);
          w[i] = at >= 0 ? __ldcg(reinterpret_cast<const uint4*>(a.q + at) + lane % LANES) : make_uint4(0, 0, 0, 0);
        }
        const int row = tiles.row[t.tile], p_off = tiles.page0[t.tile], most = a.bt_width * PG_PAGE;
        const int* bt = a.block_table + (int64_t)(row < 0 ? -1 - row : row) * a.bt_stride + p_off;
        bool holes = false;
#pragma unroll 1
        for (int p = t.p0 + lane; p < t.p1; p += 32) { const int page = p_off + p < a.bt_width ? __ldcg(bt + p) : -1; holes |= page < 0 || page >= a.n_pages; }
        m.pos = INT32_MAX;                       // (shared pages, seen by all as a rule)
        if (row < 0) {
          m.pos = (a.rows <= PS_MAX_ROWS ? tiles.pos[-1 - row] : min(__ldcg(a.row_pos0 - 1 - row), most)) + step_tok;
        } else if (tiles.group_seen[tiles.groups.of(row)] < (p_off + t.p1) * PG_PAGE - 1) {
          int row_lo = row, row_hi = row + tiles.groups.rows[tiles.groups.of(row)] - 1;
#pragma unroll 1
          while (row_lo < row_hi) { const int mid = (row_lo + row_hi + 1) >> 1; if (__ldcg(a.row_start + mid) <= tok) row_lo = mid; else row_hi = mid - 1; }
          m.pos = min(__ldcg(a.row_pos0 + row_lo), most) + tok - __ldcg(a.row_start + row_lo);
        }
        if (r < 32) for (int d = r; d < HD; d += 32) tiles.odd_key[s][m.turn][d] = INT32_MAX;
        if (r == 0) tiles.odd[s][m.turn] = 0;
#pragma unroll
        for (int i = 0; i < LANES; ++i) {
          const int c = lane % LANES, rr = (warp & 3) * 32 + EACH * i + lane / LANES;
          *reinterpret_cast<uint4*>(sQ + s * second_q + (c >> 3) * 128 * 128 + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = w[i];
        }
        m.holes = __any_sync(0xffffffffu, holes);
        m.sees = __reduce_min_sync(0xffffffffu, m.pos);
        fence_smem_to_tma();
        ps_arrive_warp(q_full + s);
      }
      if (begun) {
        ok = ps_wait(pv_done + 2 * s + ((f - 1) & 1), ((f - 1) >> 1) & 1);
        if (!ok) break;
        fence_after();
        float* const rec = a.records + now.slot * ps_record(HD), *const sums = rec + 2 * PS_TILE + (int64_t)now.qr * HD;
        if (now.in) { rec[now.qr] = m_used; rec[PS_TILE + now.qr] = l; }
#pragma unroll 1
        for (int h = 0; h < HD / 32; ++h) {
          __syncwarp();
          tmem_ld32(to + 32 * h, s0);
          if (now.in) {
#pragma unroll
            for (int c = 0; c < 32; c += 8) ps_store8(sums + 32 * h + c, s0 + c);
          }
        }
        if (tiles.odd[s][now.turn] != 0 && now.in)           // (written before the product that has ended)
#pragma unroll 1
          for (int d = 0; d < HD; ++d)
            if (tiles.odd_key[s][now.turn][d] <= now.pos) sums[d] = __int_as_float(0x7fc00000);
        __syncwarp();
        fence_before();                        // O is read: the next part's first product may write it
      }
      if (!more) break;
      const PsPart t = m.t;
      const bool holes = m.holes;
      const int step = m.two ? 1 : 2, first = m.first, pos = m.pos, sees = m.sees, p_off = tiles.page0[t.tile];
      m_used = -INFINITY;
      l = 0.0f;
      auto ask = [&](int f) {                  // the scores of the set's page f: on their way
        if (!ps_wait(s_full + 2 * s + (f & 1), (f >> 1) & 1)) return false;
        fence_after();
        tmem_ld32_issue(ts + 64 * (f & 1), s0);
        tmem_ld32_issue(ts + 64 * (f & 1) + 32, s1);
        return true;
      };
      ok = ask(f);
#pragma unroll 1
      for (int p = first; p < t.p1 && ok; p += step, ++f) {
        const int sb = f & 1;
        tmem_ld_wait(s0);
        tmem_ld_wait(s1);
        const int key0 = (p_off + p) * PG_PAGE;
        if (key0 + PG_PAGE - 1 > sees || holes) {
          int last = pos;
          if (holes) {
            const int row = tiles.row[t.tile], page = p_off + p < a.bt_width ? __ldcg(a.block_table + (int64_t)(row < 0 ? -1 - row : row) * a.bt_stride + p_off + p) : -1;
            if (page < 0 || page >= a.n_pages) last = -1;
          }
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            if (key0 + c > last) s0[c] = 0xff800000u;
            if (key0 + 32 + c > last) s1[c] = 0xff800000u;
          }
        }
        const float mx = ps_row_max(s0, s1) * a.scale_log2;              // (the scale is positive)
        const bool grow = mx > m_used + PS_RESCALE_STEP || (m_used == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? mx : m_used;
          const float corr = m_used == -INFINITY ? 0.0f : ps_exp2(m_used - m_new);
          if (p > first) {
            if (!ps_wait(pv_done + 2 * s + (sb ^ 1), ((f - 1) >> 1) & 1)) { ok = false; break; }
            fence_after();
            ps_rescale<HD>(to, corr);
          }
          l *= corr;
          m_used = m_new;
        }
        const float ref = m_used == -INFINITY ? 0.0f : m_used;
        uint32_t pw[32];
        unsigned long long sum[2] = {0, 0};
        ps_exponentials(s0, a.scale_log2, ref, pw, sum);
        ps_exponentials(s1, a.scale_log2, ref, pw + 16, sum);
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum[0]) : "l"(sum[1]));
        float e0, e1;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(sum[0]));
        l += e0 + e1;
        ps_st32(ts + 64 * sb, pw);             // over the row's own scores
        if (p + step < t.p1) ok = ask(f + 1);
        ps_wait_st();
        fence_before();
        ps_arrive_warp(p_full + 2 * s + sb);
      }
      if (!ok) break;
    }
    if (!ok) asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");         // a row of scores may still be on its way
    if (!ok && lane == 0) atomicExch(&g_ps_error, 4);
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 8) tmem_free<512>(tmem);
}

// Joins the parts of a query: SPLIT warps for each (token, head) pair, or LANES lanes of one.  The parts of the shared pages come first, in the order of the pages, those of the
// row's own pages last, so a result does not depend on which block was the first to end.  A chain of four reads (tiles, parts, maxima, values) and few bytes, so with many pairs
// what counts is how many are on their way: a warp a pair took 44 us for 52,224 pairs of heads of 128, eight lanes a pair 24.5.
constexpr int PJ_WARPS = 4;
constexpr int PJ_PARTS = 1024;                 // four for every SM, at most
template <int HD, int SPLIT, int LANES>
__global__ void __launch_bounds__(PJ_WARPS * 32)
attn_shared_join_kernel(const int4* __restrict__ parts, int most_tiles, int slots, const int4* __restrict__ tokens, const float* __restrict__ records, const float* __restrict__ own,
                        __nv_bfloat16* __restrict__ out, int T, int nh, int nkv, int* late) {
  static_assert(LANES == 32 || SPLIT == 1, "a pair has some of a warp's lanes, or some warps");
  constexpr int V = HD / LANES, W = V < 4 ? V : 4, PAIRS = PJ_WARPS * 32 / (SPLIT * LANES);      // features a lane, side by side; pairs a block
  __shared__ float s_w[SPLIT > 1 ? PAIRS : 1][SPLIT > 1 ? PJ_PARTS + 1 : 1];
  __shared__ float s_y[SPLIT > 1 ? PJ_WARPS : 1][SPLIT > 1 ? HD : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x % LANES, pair = threadIdx.x / (SPLIT * LANES), w0 = warp % SPLIT;
  const int64_t th = (int64_t)blockIdx.x * PAIRS + pair;
  pdl_trigger();
  pdl_wait();
  const bool there = th < (int64_t)T * nh;
  if (blockIdx.x == 0 && threadIdx.x == 0) *late = 0;         // (the walk has ended)
  const int tok = there ? (int)(th / nh) : 0, head = there ? (int)(th - (int64_t)tok * nh) : 0, G = nh / nkv, g = head / G, h = head - g * G;
  const int4 w = __ldcg(tokens + tok);         // (shared tile, its first token, own tile, its first token)
  // a source: the parts of one tile
  struct Source { const float* at; int n, halves, row; };     // its first record, its parts, and the query's place in a record
  auto source = [&](int tile0, int tok0) {
    Source s = {records, 0, 1, 0};
    const int query = (tok - tok0) * G + h, tile = tile0 + query / PS_TILE;
    if (tile0 < 0 || query < 0 || tile >= most_tiles) return s;
    const int4 t = __ldcg(parts + (int64_t)g * most_tiles + tile);
    // (rows that are not one behind the other leave tokens without a tile: nothing beyond the records is read for them)
    if (t.x < 0 || t.y < 1 || t.y >= PJ_PARTS / 2 || t.z < 1 || t.z > 2 || t.x + t.y / t.z > slots) return s;
    s.n = t.y;
    s.halves = t.z;
    s.row = query % PS_TILE;
    s.at = records + t.x * ps_record(HD);
    return s;
  };
  const bool any = there && (w.x >= 0 || w.z >= 0);          // else its own pages' part was all
  const Source s0 = source(any ? w.x : -1, w.y), s1 = source(any ? w.z : -1, w.w);
  const int n01 = s0.n + s1.n, n = any ? n01 + (w.z < 0 ? 1 : 0) : 0;    // (no tile for the row's own pages: the walk's part)
  const float* mine = own + (int64_t)T * nh * HD + 2 * th;
  // part i: its record, and the query's place in it; the walk's part is the last
  auto part = [&](int i, int& row) {
    const bool second = i >= s0.n;
    const int k = second ? i - s0.n : i, halves = second ? s1.halves : s0.halves;
    row = (second ? s1.row : s0.row) + (halves == 2 ? (k & 1) * 128 : 0);
    return (second ? s1.at : s0.at) + (halves == 2 ? k >> 1 : k) * ps_record(HD);
  };
  float mm = -INFINITY, l = 0.0f;
#pragma unroll 1
  for (int i = lane; i < n; i += LANES) {
    int row = 0;
    const float* p = i < n01 ? part(i, row) : mine;
    const float m1 = __ldcg(p + row), l1 = __ldcg(p + row + (i < n01 ? PS_TILE : 1)), top = fmaxf(mm, m1), safe = top == -INFINITY ? 0.0f : top;
    l = l * ps_exp2(mm - safe) + l1 * ps_exp2(m1 - safe);
    mm = top;
    if (SPLIT > 1 && w0 == 0) s_w[pair][i] = m1;
  }
  float top = mm;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float safe = top == -INFINITY ? 0.0f : top;
  l *= ps_exp2(mm - safe);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (SPLIT > 1) __syncthreads();
  float y[V] = {};
  constexpr int BATCH = LANES == 32 ? 8 : 2;
#pragma unroll 1
  for (int i0 = w0; i0 < n; i0 += SPLIT * BATCH) {
    float v[BATCH][V], f[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int i = i0 + b * SPLIT;
      f[b] = -INFINITY;
      if (i < n) {
        int row = 0;
        const float* p = i < n01 ? part(i, row) : mine;
        f[b] = SPLIT > 1 ? s_w[pair][i] : __ldcg(p + row);
        p = i < n01 ? p + 2 * PS_TILE + row * HD : own + th * HD;
#pragma unroll
        for (int e = 0; e < V; e += W) {
          const float* const at = p + (e * LANES + lane * W);
          if (W == 4) { const float4 x = __ldcg(reinterpret_cast<const float4*>(at)); v[b][e] = x.x; v[b][e + 1] = x.y; v[b][e + W - 2] = x.z; v[b][e + W - 1] = x.w; }
          else { const float2 x = __ldcg(reinterpret_cast<const float2*>(at)); v[b][e] = x.x; v[b][e + 1] = x.y; }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const bool seen = f[b] > -INFINITY;                            // (a part without a key leaves no sums)
      const float w = ps_exp2(f[b] - safe);                          // (0 for one far below the others: its sums that are not finite are not, all the same)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (seen) y[e] = fmaf(w, v[b][e], y[e]);
    }
  }
  if (SPLIT > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) s_y[warp][lane * V + e] = y[e];
    __syncthreads();
    if (w0 != 0) return;
#pragma unroll
    for (int k = 1; k < SPLIT; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] += s_y[warp + k][lane * V + e];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (!any) return;
#pragma unroll
  for (int e = 0; e < V; e += W) {
    __nv_bfloat16* const to = out + th * HD + e * LANES + lane * W;
    if (W == 4) *reinterpret_cast<uint2*>(to) = make_uint2(ps_pack(y[e] * inv, y[e + 1] * inv), ps_pack(y[e + W - 2] * inv, y[e + W - 1] * inv));
    else *reinterpret_cast<uint32_t*>(to) = ps_pack(y[e] * inv, y[e + 1] * inv);
  }
}

int attn_shared_join(const PsArgs& a, const float* own, __nv_bfloat16* out, int* late, int hd, cudaStream_t stream) {
  // few queries: a block each, since a query of a few may have hundreds of parts
  const int64_t pairs = (int64_t)a.T * a.nkv * a.G;
  const bool few = pairs <= 4096;
  auto go = [&](auto kernel, int per_block) {
    launch_pdl(kernel, dim3((unsigned)((pairs + per_block - 1) / per_block)), dim3(PJ_WARPS * 32), 0, stream, reinterpret_cast<const int4*>(a.parts), a.most_tiles, (int)ps_slots(a.sms, a.nkv, a.most_tiles),
               reinterpret_cast<const int4*>(a.tokens), (const float*)a.records, own, out, a.T, a.nkv * a.G, a.nkv, late);
  };
  if (hd == 64) { if (few) go(attn_shared_join_kernel<64, PJ_WARPS, 32>, 1); else go(attn_shared_join_kernel<64, 1, 8>, PJ_WARPS * 4); }
  else { if (few) go(attn_shared_join_kernel<128, PJ_WARPS, 32>, 1); else go(attn_shared_join_kernel<128, 1, 8>, PJ_WARPS * 4); }
  return launch_status("attn_shared join");
}

cudaError_t attn_shared_prepare() {
  cudaError_t e = cudaFuncSetAttribute(attn_shared_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ps_smem(64));
  return e != cudaSuccess ? e : cudaFuncSetAttribute(attn_shared_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ps_smem(128));
}

int attn_shared_launch(const PsArgs& a, const void* k_pool, const void* v_pool, int hd, int sms, cudaStream_t stream) {
  CUtensorMap map_k, map_v;
  int rc = make_map_k64(&map_k, k_pool, (int64_t)a.n_pages * a.nkv * PG_PAGE, hd, PG_PAGE, "attn_shared");
  if (!rc) rc = make_map_k64(&map_v, v_pool, (int64_t)a.n_pages * a.nkv * PG_PAGE, hd, PG_PAGE, "attn_shared");
  if (rc) return rc;
  if (hd == 64) launch_pdl(attn_shared_kernel<64>, dim3(sms), dim3(PS_THREADS), ps_smem(64), stream, map_k, map_v, a);
  else launch_pdl(attn_shared_kernel<128>, dim3(sms), dim3(PS_THREADS), ps_smem(128), stream, map_k, map_v, a);
  return launch_status("attn_shared");
}

}  // namespace exl3

extern "C" int exl3_attn_shared_status() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, exl3::g_ps_error, sizeof(int));
  if (v) { int z = 0; cudaMemcpyToSymbol(exl3::g_ps_error, &z, sizeof(int)); }
  return v;
}
