// Bounds of the cache's pages in 8 bits, and the choice of pages by them.
//
// Bounds of a page and key/value head: the smallest and largest key of every feature over the page's tokens so far, codes int8 [2][hd], and a scale:
//   a = max |k| (at least 1e-30),  scale = a / 127,  code = rint(x * (127 / a))   in float32
// A page that holds a key that is not finite has codes 0 and an infinite scale, and is chosen before others.
//
// Score of a page for a (token, key/value head): with a_h = max |q_h| and c_h = rint(q_h * (127 / a_h)) for each query head h of the head,
//   n_h = sum_i max(c_hi low_i, c_hi high_i) = sum_i min(c_hi, 0) low_i + max(c_hi, 0) high_i,   score = max_h(n_h * (a_h / 127)) * scale
// n_h is a product over 2 hd features of whole numbers, below 2^23, so exact whatever the order of its terms: which pages are
// chosen follows from the definition, not from how a kernel adds up.
#include "api.h"
#include "common.cuh"
#include "tcgen05.cuh"

#include <math.h>

namespace exl3 {

constexpr int PB_PAGE = 64;
constexpr int PB_WARPS = 4;
constexpr float PB_TINY = 1e-30f;

__device__ inline uint32_t pb_min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ inline uint32_t pb_max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ inline float pb_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ inline float pb_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ inline int pb_code(float x, float inv) { return (int)fminf(fmaxf(rintf(__fmul_rn(x, inv)), -127.0f), 127.0f); }

// A warp for each (page that got new keys, key/value head): one read of the page.  Where there are many it is bound by the bytes that a warp has on their way (8,192 tokens of 36 heads of 64, 38 MB: with
// the load of these bounds 16 us, 0.4 of the copy rate; 19 when the loads were conditional and so one after the other), else by the chain row, page number, page (64 rows' last pages and their
// load: 8.2 us).
template <int HD>
__global__ void __launch_bounds__(PB_WARPS * 32)
page_bounds_kernel(const __nv_bfloat16* __restrict__ k_pool, int64_t n_pages, const int* __restrict__ block_table, int bt_stride, int bt_width,
                   const int* __restrict__ row_start, const int* __restrict__ row_pos0, int rows, int most, int nkv, int8_t* __restrict__ codes, float* __restrict__ scales) {
  constexpr int CH = HD / 8, TOK = 32 / CH;      // lanes of a token, tokens side by side
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * PB_WARPS + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  if (item >= (int64_t)rows * most * nkv) return;
  const int g = (int)(item % nkv), nth = (int)(item / nkv % most), row = (int)(item / nkv / most);
  const int n_new = __ldcg(row_start + row + 1) - __ldcg(row_start + row), pos0 = __ldcg(row_pos0 + row);
  const int64_t end = (int64_t)pos0 + n_new;
  const int64_t logical = (int64_t)max(pos0, 0) / PB_PAGE + nth;
  if (n_new <= 0 || logical * PB_PAGE >= end || logical >= bt_width) return;
  const int page = __ldcg(block_table + (int64_t)row * bt_stride + logical);
  if (page < 0 || page >= n_pages) return;
  const int filled = (int)min((int64_t)PB_PAGE, end - logical * PB_PAGE);
  const uint4* src = reinterpret_cast<const uint4*>(k_pool + ((int64_t)page * nkv + g) * PB_PAGE * HD) + lane % CH;
  uint32_t mn[4], mx[4], odd = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) { mn[i] = 0x7f807f80u; mx[i] = 0xff80ff80u; }
  // Loads that depend on no condition, so that several of a lane are on their way at once: as many as 33 registers (heads of 128; 34 of 64) hold, far fewer than the sixteen asked for.  Behind the
  // last token it is read again, which changes no bound.
#pragma unroll 1
  for (int t0 = 0; t0 < PB_PAGE / TOK && t0 * TOK < filled; t0 += 16) {
    uint4 w[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) w[t] = __ldcg(src + min((t0 + t) * TOK + lane / CH, filled - 1) * CH);
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const uint32_t x[4] = {w[t].x, w[t].y, w[t].z, w[t].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mn[i] = pb_min2(mn[i], x[i]);
        mx[i] = pb_max2(mx[i], x[i]);
        odd |= ((x[i] & 0x7f80u) == 0x7f80u) | ((x[i] & 0x7f800000u) == 0x7f800000u);
      }
    }
  }
#pragma unroll
  for (int o = CH; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mn[i] = pb_min2(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
      mx[i] = pb_max2(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
    }
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a = fmaxf(a, fmaxf(fmaxf(fabsf(pb_lo(mn[i])), fabsf(pb_hi(mn[i]))), fmaxf(fabsf(pb_lo(mx[i])), fabsf(pb_hi(mx[i])))));
  a = fmaxf(warp_max(a), PB_TINY);
  odd = __any_sync(0xffffffffu, odd);
  const float inv = odd ? 0.0f : __fdiv_rn(127.0f, a);
  if (lane < 2 * CH) {                           // the first CH lanes write the smallest, the next CH the largest
    const bool high = lane >= CH;
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t p = high ? mx[2 * i] : mn[2 * i], q = high ? mx[2 * i + 1] : mn[2 * i + 1];
      w[i] = odd ? 0u : (pb_code(pb_lo(p), inv) & 0xff) | (pb_code(pb_hi(p), inv) & 0xff) << 8 | (pb_code(pb_lo(q), inv) & 0xff) << 16 | (uint32_t)pb_code(pb_hi(q), inv) << 24;
    }
    *reinterpret_cast<uint2*>(codes + (((int64_t)page * nkv + g) * 2 + high) * HD + (lane % CH) * 8) = make_uint2(w[0], w[1]);
  }
  if (lane == 0) scales[(int64_t)page * nkv + g] = odd ? INFINITY : __fdiv_rn(a, 127.0f);
}

// low, high float32 [n, kv heads, hd] of the listed pages; zeros for a number that is no page's.
__global__ void page_bounds_load_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t n_pages, const int* __restrict__ pages, int64_t total,
                                        int nkv, int hd, float* __restrict__ low, float* __restrict__ high) {
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 4;      // a feature of low, of all pages' heads
  pdl_trigger();
  pdl_wait();
  if (i >= total) return;
  const int64_t ph = i / hd;
  const int d = (int)(i % hd), page = __ldcg(pages + ph / nkv);
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
  if (page >= 0 && page < n_pages) {
    const int64_t at = (int64_t)page * nkv + ph % nkv;
    const float s = __ldcg(scales + at);
    const char4 x = __ldcg(reinterpret_cast<const char4*>(codes + at * 2 * hd + d)), y = __ldcg(reinterpret_cast<const char4*>(codes + (at * 2 + 1) * hd + d));
    a = make_float4(x.x * s, x.y * s, x.z * s, x.w * s);
    b = make_float4(y.x * s, y.y * s, y.z * s, y.w * s);
  }
  *reinterpret_cast<float4*>(low + i) = a;
  *reinterpret_cast<float4*>(high + i) = b;
}

// ---- the choice -----------------------------------------------------------------------------------------------------------------

constexpr int SEL_THREADS = 256, SEL_WARPS = SEL_THREADS / 32;
constexpr int SEL_LANE = 16;                   // keys of a lane where one warp searches
constexpr int SEL_MAX_HEADS = 128;             // query heads of a key/value head
constexpr int SEL_MAX_PAGES = 32768;           // pages of a row

__device__ inline void sel_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A score's place in the order, above 0; a page that must be chosen has the highest.
constexpr uint32_t SEL_MUST = 0xffffffffu, SEL_ODD = 0xfffffffeu;
__device__ inline uint32_t sel_key(float score) {
  if (!(score == score)) return SEL_ODD;
  const uint32_t b = __float_as_uint(score == 0.0f ? 0.0f : score);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct SelArgs {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const int8_t* codes;
  const float* scales;
  int64_t n_pages;
  const int* block_table;
  int bt_stride, bt_width, bt_rows;
  const int* tok_pos;
  const int* tok_seq;
  int nkv, G, count, first, last;
  int cluster;                                   // blocks of an item: 1, 2, 4 or 8
  int* out;
};

// A cluster of blocks (one for many items) for each (token, kv head): each scores a stretch of the row's pages and puts the scores into the first one's shared memory, which
// chooses.  Pages are the rows of the matrix instruction, query heads its columns.  A lane's 16 bytes of a page's codes are four of the instruction's operand words; the
// query's codes are laid out alike, so that the order of features within the product is the memory's.  A warp's page numbers are asked for two steps ahead, codes one.
// Bound by that chain and by the search, four counts of a digit of two bits a round where a block searches, a warp's ballots up to 512 pages: 64 tokens of 1,000 to 30,000 keys, 8 heads of
// 128, 23 us for 33 MB; one token of 131,070 keys 13.5 with clusters of 8 (with its attention 46; 160 when an item had one block).
template <int HD>
__global__ void __launch_bounds__(SEL_THREADS)
page_select_kernel(const SelArgs a) {
  constexpr int L = 2 * HD / 64;                 // 16-byte pieces a lane has of a page
  extern __shared__ uint4 sel_raw[];
  const int ng = (a.G + 7) / 8;                  // groups of 8 query heads
  int8_t* s_q = reinterpret_cast<int8_t*>(sel_raw);                             // [8 ng][2][HD] codes below and above zero
  float* s_scale = reinterpret_cast<float*>(s_q + ng * 8 * 2 * HD);           // [8 ng]
  uint32_t* s_key = reinterpret_cast<uint32_t*>(s_scale + ng * 8);            // [pages of the row]
  __shared__ int4 s_count[2][SEL_WARPS];
  __shared__ int s_base[SEL_WARPS], s_equal[SEL_WARPS];
  __shared__ int3 s_found;                       // the bound, how many of the keys at it are taken, and how many pages in all
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, tl = lane & 3;
  const int C = a.cluster, rank = C > 1 ? (int)tc5::cluster_rank() : 0, item = blockIdx.x / C;
  const int t = item / a.nkv, g = item - t * a.nkv;
  if (C > 1) tc5::cluster_arrive_all();          // (the first block must have begun before its memory is written)
  pdl_trigger();
  pdl_wait();
  const int pos = __ldcg(a.tok_pos + t), seq = __ldcg(a.tok_seq + t);
  const int there = seq < 0 || seq >= a.bt_rows || pos < 0 ? 0 : min(pos / PB_PAGE + 1, a.bt_width);   // pages that the token may see
  const int* bt = a.block_table + (int64_t)max(seq, 0) * a.bt_stride;
  const int per = ((there + C - 1) / C + 15) / 16 * 16, p_lo = min(rank * per, there), p_hi = min(p_lo + per, there);
  constexpr int STEP = SEL_WARPS * 16;
  struct Pages { int at[2]; };                   // pages gl and gl + 8 of a step; -1: not there
  auto numbers = [&](int p0) {
    Pages n;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int p = p0 + gl + 8 * e;
      n.at[e] = p < p_hi ? __ldcg(bt + p) : -1;
      if (n.at[e] >= a.n_pages) n.at[e] = -1;
    }
    return n;
  };
  struct Codes { uint4 w[2][L]; float scale[2]; };
  auto codes = [&](const Pages& n) {
    Codes c;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t at = (int64_t)max(n.at[e], 0) * a.nkv + g;
#pragma unroll
      for (int i = 0; i < L; ++i) c.w[e][i] = __ldcg(reinterpret_cast<const uint4*>(a.codes + at * 2 * HD + 64 * i + 16 * tl));
      c.scale[e] = __ldcg(a.scales + at);
    }
    return c;
  };
  int p0 = p_lo + warp * 16;
  Pages n0 = numbers(p0), n1 = numbers(p0 + STEP);

  for (int h = warp; h < 8 * ng; h += SEL_WARPS) {
    float x[HD / 32], m = 0.0f;
    const __nv_bfloat16* src = a.q + (int64_t)t * a.q_stride + (int64_t)(g * a.G + h) * HD;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
      const uint32_t w = h < a.G ? __ldcg(reinterpret_cast<const unsigned int*>(src) + i * 32 + lane) : 0u;
      x[2 * i] = pb_lo(w);
      x[2 * i + 1] = pb_hi(w);
      m = fmaxf(m, fmaxf(fabsf(x[2 * i]), fabsf(x[2 * i + 1])));
    }
    m = fmaxf(warp_max(m), PB_TINY);
    const float inv = __fdiv_rn(127.0f, m);
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
      const int c0 = pb_code(x[2 * i], inv), c1 = pb_code(x[2 * i + 1], inv);
      char2* dst = reinterpret_cast<char2*>(s_q + h * 2 * HD);
      dst[i * 32 + lane] = make_char2((signed char)min(c0, 0), (signed char)min(c1, 0));
      dst[HD / 2 + i * 32 + lane] = make_char2((signed char)max(c0, 0), (signed char)max(c1, 0));
    }
    if (lane == 0) s_scale[h] = h < a.G ? __fdiv_rn(m, 127.0f) : -1.0f;
  }
  Codes now = codes(n0);
  if (C > 1) tc5::cluster_wait_all();
  __syncthreads();

  // ---- scores ------------------------------------------------------------------------------------------------------------------
  const uint32_t keys = C > 1 ? tc5::cluster_addr(s_key, 0) : tc5::smem_u32(s_key);
  for (; p0 < p_hi; p0 += STEP) {
    const Codes next = codes(n1);                // (past the end: page 0's, not used)
    const Pages n2 = numbers(p0 + 2 * STEP);
    float best[2] = {-INFINITY, -INFINITY};
    __syncwarp();
    for (int n = 0; n < ng; ++n) {
      int c[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const uint4 b = *reinterpret_cast<const uint4*>(s_q + (n * 8 + gl) * 2 * HD + 64 * i + 16 * tl);
        sel_mma(c, now.w[0][i].x, now.w[1][i].x, now.w[0][i].y, now.w[1][i].y, b.x, b.y);
        sel_mma(c, now.w[0][i].z, now.w[1][i].z, now.w[0][i].w, now.w[1][i].w, b.z, b.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float s = s_scale[n * 8 + 2 * tl + (e & 1)];
        if (s >= 0.0f) best[e >> 1] = fmaxf(best[e >> 1], __fmul_rn((float)c[e], s));
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 1));
      best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 2));
      const int p = p0 + gl + 8 * e;
      if (tl == 0 && p < p_hi) {
        const uint32_t key = n0.at[e] < 0 ? 0u : p < a.first || p >= there - a.last ? SEL_MUST : isinf(now.scale[e]) ? SEL_ODD : sel_key(__fmul_rn(best[e], now.scale[e]));
        if (C > 1) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(keys + 4 * p), "r"(key) : "memory");
        else s_key[p] = key;
      }
    }
    now = next;
    n0 = n1;
    n1 = n2;
  }
  if (C > 1) {
    tc5::cluster_sync_all();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // ---- the k-th largest place: the largest bound that k keys reach, two bits at a time.  counts(b1, b2, b3): keys of at least each bound -----------------------------
  auto search = [&](auto counts, int held, int k, uint32_t& bound, int& want) {
    bound = 0u;
    want = 0;                                    // of the keys at the bound
    if (k >= held) return;                       // (all that are there)
    int at_least = held;                         // keys that reach the bound
#pragma unroll 1
    for (int bit = 30; bit >= 0 && at_least > k; bit -= 2) {
      const uint32_t b1 = bound | 1u << bit, b2 = bound | 2u << bit, b3 = bound | 3u << bit;
      const int3 n = counts(b1, b2, b3);
      if (n.z >= k) { bound = b3; at_least = n.z; }
      else if (n.y >= k) { bound = b2; at_least = n.y; }
      else if (n.x >= k) { bound = b1; at_least = n.x; }
    }
    if (at_least == k) { bound -= 1; return; }   // all that reach it, and none below
    want = bound == 0xffffffffu ? k : k - counts(bound + 1, bound + 1, bound + 1).x;   // (more than k reach the highest place: only if all of them must be chosen)
  };
  if (there <= 32 * SEL_LANE) {
    // few pages: one warp, their keys in registers, no barrier a step (470 pages: 4.4 us -> 1)
    if (warp == 0) {
      uint32_t key[SEL_LANE];
      int n = 0;
#pragma unroll
      for (int i = 0; i < SEL_LANE; ++i) {
        key[i] = 32 * i + lane < there ? s_key[32 * i + lane] : 0u;
        n += key[i] > 0u;
      }
      n = __reduce_add_sync(0xffffffffu, n);
      uint32_t b;
      int w;
      search([&](uint32_t b1, uint32_t b2, uint32_t b3) {
        int n12 = 0, n3 = 0;
#pragma unroll
        for (int i = 0; i < SEL_LANE; ++i) {
          n12 += (key[i] >= b1) + ((key[i] >= b2) << 16);
          n3 += key[i] >= b3;
        }
        n12 = __reduce_add_sync(0xffffffffu, n12);
        n3 = __reduce_add_sync(0xffffffffu, n3);
        return make_int3(n12 & 0xffff, n12 >> 16, n3);
      }, n, min(a.count, n), b, w);
      if (lane == 0) s_found = make_int3((int)b, w, min(a.count, n));
    }
    __syncthreads();
  } else {
    int turn = 0;
    auto reach = [&](uint32_t b1, uint32_t b2, uint32_t b3) {          // (at most 32,768 pages: two counts to a word)
      int n12 = 0, n3 = 0;
      for (int p = threadIdx.x; p < there; p += SEL_THREADS) {
        const uint32_t key = s_key[p];
        n12 += (key >= b1) + ((key >= b2) << 16);
        n3 += key >= b3;
      }
      n12 = __reduce_add_sync(0xffffffffu, n12);
      n3 = __reduce_add_sync(0xffffffffu, n3);
      if (lane == 0) s_count[turn][warp] = make_int4(n12 & 0xffff, n12 >> 16, n3, 0);
      __syncthreads();
      int3 n = make_int3(0, 0, 0);
#pragma unroll
      for (int i = 0; i < SEL_WARPS; ++i) { const int4 m = s_count[turn][i]; n.x += m.x; n.y += m.y; n.z += m.z; }
      turn ^= 1;
      return n;
    };
    const int held = reach(1u, 1u, 1u).x;
    uint32_t b;
    int w;
    search(reach, held, min(a.count, held), b, w);
    if (threadIdx.x == 0) s_found = make_int3((int)b, w, min(a.count, held));
    __syncthreads();
  }
  const uint32_t bound = (uint32_t)s_found.x;
  const int want = s_found.y, k = s_found.z;
  // ---- the chosen pages in order: all above the bound, and the first of those at it ---------------------------------------------------
  // a warp has a stretch of pages: first its numbers, then its places
  const int stretch = (there + SEL_THREADS - 1) / SEL_THREADS * 32, from = min(warp * stretch, there), to = min(from + stretch, there);
  int n_above = 0, n_equal = 0;
  for (int q0 = from; q0 < to; q0 += 32) {
    const uint32_t key = q0 + lane < to ? s_key[q0 + lane] : 0u;
    n_above += __popc(__ballot_sync(0xffffffffu, key > bound));
    n_equal += __popc(__ballot_sync(0xffffffffu, q0 + lane < to && key == bound));
  }
  if (lane == 0) { s_base[warp] = n_above; s_equal[warp] = n_equal; }
  __syncthreads();
  int at = 0, equal = 0;
  for (int i = 0; i < warp; ++i) { at += s_base[i]; equal += s_equal[i]; }
  at += min(equal, want);
  int* out = a.out + (int64_t)item * a.count;
  for (int q0 = from; q0 < to; q0 += 32) {
    const bool in = q0 + lane < to;
    const uint32_t key = in ? s_key[q0 + lane] : 0u;
    const uint32_t below = (1u << lane) - 1, eq = __ballot_sync(0xffffffffu, in && key == bound);
    const bool take = key > bound || (in && key == bound && equal + __popc(eq & below) < want);
    const uint32_t took = __ballot_sync(0xffffffffu, take);
    if (take) out[at + __popc(took & below)] = q0 + lane;
    at += __popc(took);
    equal += __popc(eq);
  }
  for (int i = k + threadIdx.x; i < a.count; i += SEL_THREADS) out[i] = -1;
}

}  // namespace exl3

using namespace exl3;

// New bounds for the pages that hold the rows' new tokens (row r: row_start[r + 1] - row_start[r] of them from position row_pos0[r], at most max_new).
extern "C" int exl3_page_bounds(const void* k_pool, int64_t n_pages, const int* block_table, int bt_stride, int bt_width, const int* row_start, const int* row_pos0, int rows,
                                int max_new, int nkv, int hd, void* codes, float* scales, cudaStream_t stream) {
  if (rows == 0 || max_new == 0) return 0;
  if (rows < 0 || max_new < 0 || nkv < 1 || (hd != 64 && hd != 128) || n_pages < 1 || bt_width < 1 || !k_pool || !block_table || !row_start || !row_pos0 || !codes || !scales) {
    set_error("page_bounds: needs heads of 64 or 128 and all of its arrays, got %d rows, max_new %d, %d heads of %d, %lld pages", rows, max_new, nkv, hd, (long long)n_pages);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(k_pool) || !aligned16(codes)) { set_error("page_bounds: the pools must be 16-byte aligned"); return ERR_ALIGNMENT; }
  const int most = min(bt_width, max_new == 1 ? 1 : (max_new - 2) / PB_PAGE + 2);        // pages that max_new tokens can touch
  const int64_t blocks = ((int64_t)rows * most * nkv + PB_WARPS - 1) / PB_WARPS;
  if (blocks > INT32_MAX) { set_error("page_bounds: too many pages for one launch"); return ERR_UNSUPPORTED; }
  auto go = [&](auto kernel) {
    launch_pdl(kernel, dim3((unsigned)blocks), dim3(PB_WARPS * 32), 0, stream, static_cast<const __nv_bfloat16*>(k_pool), n_pages, block_table, bt_stride, bt_width, row_start,
               row_pos0, rows, most, nkv, static_cast<int8_t*>(codes), scales);
  };
  if (hd == 64) go(page_bounds_kernel<64>); else go(page_bounds_kernel<128>);
  return launch_status("page_bounds");
}

extern "C" int exl3_page_bounds_load(const void* codes, const float* scales, int64_t n_pages, const int* pages, int n, int nkv, int hd, float* low, float* high,
                                     cudaStream_t stream) {
  if (n == 0) return 0;
  if (n < 0 || nkv < 1 || (hd != 64 && hd != 128) || n_pages < 1 || !codes || !scales || !pages || !low || !high) { set_error("page_bounds_load: bad sizes or a missing array"); return ERR_BAD_ARGUMENT; }
  if (!aligned16(codes) || !aligned16(low) || !aligned16(high)) { set_error("page_bounds_load: the codes and the bounds must be 16-byte aligned"); return ERR_ALIGNMENT; }
  const int64_t total = (int64_t)n * nkv * hd;
  launch_pdl(page_bounds_load_kernel, dim3((unsigned)((total / 4 + 255) / 256)), dim3(256), 0, stream, static_cast<const int8_t*>(codes), scales, n_pages, pages, total, nkv, hd, low, high);
  return launch_status("page_bounds_load");
}

extern "C" int exl3_page_select(const void* q, int64_t q_stride, const void* codes, const float* scales, int64_t n_pages, const int* block_table, int bt_stride, int bt_width,
                                int bt_rows, const int* tok_pos, const int* tok_seq, int T, int nh, int nkv, int hd, int count, int first, int last, int* out,
                                cudaStream_t stream) {
  if (T == 0) return 0;
  if (T < 0 || nkv < 1 || nh < nkv || nh % nkv || nh / nkv > SEL_MAX_HEADS || (hd != 64 && hd != 128) || n_pages < 1 || bt_width < 1 || bt_width > SEL_MAX_PAGES || count < 1 ||
      first < 0 || last < 1 || (int64_t)T * nkv > INT32_MAX / 8 || !q || !codes || !scales || !block_table || !tok_pos || !tok_seq || !out) {
    set_error("page_select: needs heads of 64 or 128, at most %d query heads a key/value head, rows of at most %d pages, a count of 1 or more, and at least the last page, got %d "
              "heads on %d of %d, %d pages, count %d, first %d, last %d", SEL_MAX_HEADS, SEL_MAX_PAGES, nh, nkv, hd, bt_width, count, first, last);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(q) || q_stride % 8 || !aligned16(codes)) { set_error("page_select: q, its rows and the codes must be 16-byte aligned"); return ERR_ALIGNMENT; }
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("page_select: no device"); return ERR_UNSUPPORTED; }
  const int ng = ceil_div(nh / nkv, 8);
  const size_t most = (size_t)SEL_MAX_HEADS * (2 * 128 + 4) + (size_t)SEL_MAX_PAGES * 4, smem = (size_t)ng * 8 * (2 * hd + 4) + (size_t)bt_width * 4;
  if (!sms[dev]) {
    cudaError_t e = cudaFuncSetAttribute(page_select_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(page_select_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    int n = 0;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) { set_error("page_select: cannot get %zu bytes of shared memory: %s", most, cudaGetErrorString(e)); return (int)e; }
    sms[dev] = n;
  }
  SelArgs a = {static_cast<const __nv_bfloat16*>(q), q_stride, static_cast<const int8_t*>(codes), scales, n_pages, block_table, bt_stride, bt_width, bt_rows, tok_pos, tok_seq,
               nkv, nh / nkv, count, first, last, 1, out};
  // several blocks an item while that leaves SMs idle, each with 256 pages or more
  while (a.cluster < 8 && (int64_t)T * nkv * a.cluster * 2 <= sms[dev] && bt_width >= 512 * a.cluster) a.cluster *= 2;
  auto go = [&](auto kernel) {
    const dim3 grid((unsigned)(T * nkv * a.cluster));
    if (a.cluster > 1) launch_pdl_clusters(kernel, grid, dim3(SEL_THREADS), (unsigned)a.cluster, smem, stream, a);
    else launch_pdl(kernel, grid, dim3(SEL_THREADS), smem, stream, a);
  };
  if (hd == 64) go(page_select_kernel<64>); else go(page_select_kernel<128>);
  return launch_status("page_select");
}
