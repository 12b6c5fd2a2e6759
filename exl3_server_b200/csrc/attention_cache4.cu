// Attention of a step's new tokens over the 4-bit key/value cache (cache4.cuh), for one token or a few per sequence:
//
//   s[j] = (q . K[j]) * scale,   j in [max(0, p - window + 1), p] for the token at position p
//   out  = sum_j softmax(s)[j] * V[j],   K[j] = mn + sc * code by groups of 32 features, V likewise
//
// The codes go to the tensor cores as they are.  A code of 4 bits in the low half of a byte is an 8-bit float (e4m3), code * 2^-9, and in the
// low bits of a 16-bit float a subnormal of fp16, code * 2^-24 (or, one nibble up, 16 times that): one AND makes four or two operands
// out of a word, and no conversion is done at all.  The groups' numbers come in where there is less to multiply.
//
// Keys: q is taken apart into two e4m3 numbers, q' = hi + lo, scaled by a power of two so that its largest value lies in [128, 256); for
// bfloat16 q (8 bits) that is exact down to 2^-9 of the row's largest, and never off by more than 2^-17 of it.
//
//   q . K[j] = sum_groups (sc_g * C_g + mn_g * Q_g),   C_g = the product of codes and q' (mma.m16n8k32, keys x features the 16-row operand,
//   the queries its 8 columns), Q_g = the sum of the group's q', in three bfloat16 parts the operand of one more product with the mn_g
//
// Up to four columns, hi and lo stand side by side in the 8 columns of one instruction and meet in the thread that gets both; more columns
// take an instruction each.
//
// Values: with p the softmax's terms against a reference that follows the maximum lazily (p at most 2^8), P_g = p * sc_g * F in fp16 (F a power of two
// that keeps the largest scale seen so far below 2^6, carried by p's exponent: p sc keeps its 11 bits down to 2^-20 of the largest) is the second product's operand, the codes of 16 tokens the 16-row
// one, and sum p mn_g goes beside it in float32.  Scores, maximum, sums and outputs are float32.
//
// A column is a (new token, query head) of one key/value head: up to 4, 8 or 16 columns share a walk over the codes, each with its own causal limit.
// A block of four warps takes one (row, key/value head, group of columns, chunk of keys); its warps take every fourth tile of 5,120
// bytes, through a ring each that bulk copies fill ahead.  The warps' results meet in shared memory.  Where a row has several chunks their
// records go to scratch memory and a second kernel joins them, in the chunks' order.
//
// Measured: 8 rows of 4,096 keys, 36 heads of 64 with keys of their own 28.8 us (94 MB, 3.3 TB/s); 64 rows of 130 to 8,000 keys, 32 heads of 128 on 8
// 79.9 us (339 MB, 4.2 TB/s); one row of 131,071 keys of these 38.4 us (168 MB, 4.4 TB/s); one row of 128 keys, 16 heads of 64 on 2 3.9 us.
// No unit is full (64 rows: issue slots 0.63, ALU 0.53, tensor pipe 0.22, memory 0.65 of the copy rate, 14 warps an SM): a tile is some 650 instructions for a warp,
// half of them integer ones (masks, byte permutes, minima and maxima), in phases that wait for one another (scores, one vote, exponentials, transposes,
// products), and more warps an SM, more stages of the ring or larger chunks change nothing; two tiles at work at once in a warp were not tried.  What brought it here, for
// the 64 rows: 127 us with every group's numbers multiplied in first, 98 with keys as e4m3, 87 with F in the reference, 81 with whole tiles
// first, one vote a tile on the reference and two groups to an operand.  A block's beginning and end are some 4 us that few blocks an SM do not hide, hence the page numbers beside
// the lengths (and chunks no smaller than a wave wants).  A join by a cluster through distributed shared memory takes 1 us less
// than the second kernel where all clusters run at once, and a tenth more than the whole where they do not (90 us); it was left out.
#include "api.h"
#include "cache4.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <type_traits>

namespace exl3 {

using namespace kv4;

constexpr int A4_WARPS = 4;
constexpr int A4_STAGES = 2;
constexpr int A4_MAX_CHUNK = 32 * A4_WARPS;               // tiles: a warp keeps its page numbers one a lane
constexpr uint32_t A4_WAIT_LIMIT = 1u << 20;              // looks of up to a microsecond each: a second

constexpr float A4_SLACK = 8.0f;                          // base-2 units that a score may lie above its column's reference

static __device__ int g_a4_error = 0;

__device__ inline uint32_t a4_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// Suspends the warp for up to a microsecond at a time: a warp that polls takes issue slots from those that compute.
__device__ inline bool a4_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = a4_smem(bar);
  for (uint32_t i = 0; i < A4_WAIT_LIMIT; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(addr), "r"(parity), "r"(1000u) : "memory");
    if (ok) return true;
  }
  return false;
}
// fp16 x fp16 -> float32, 16 x 8 x 16.
__device__ inline void a4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// e4m3 x e4m3 -> float32, 16 x 8 x 32.
__device__ inline void a4_mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto zeros (which take no registers), and bfloat16 onto zeros.
__device__ inline void a4_mma8_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ inline void a4_mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ inline uint32_t a4_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ inline float a4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ inline float a4_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ inline uint32_t a4_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ inline float a4_pow2(int e) { return __int_as_float((e + 127) << 23); }       // e in -126 .. 127

struct A4Args {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  const unsigned char* pool;
  int n_pages;
  const int* block_table;
  int bt_stride, bt_width, T;
  const int* row_start;      // null: row r is token r
  const int* row_pos0;
  int nh, nkv, window;
  float scale_log2;          // softmax scale * log2(e)
  int chunk;                 // tiles of a chunk, aligned to absolute positions
  int max_chunks;            // chunks that the grid (and the scratch) has room for
  int n_ct;                  // groups of columns the grid has room for
  float* scratch;            // [rows][nkv][n_ct][max_chunks][columns][HD + 4] where max_chunks > 1
  int few;                   // rows of more new tokens are not taken here (last: its place ahead of the others moved their loads about, 3 % for heads of 128)
};

// What a (row, group of columns) sees: tiles t_lo .. t_hi, and the chunks that hold them.  Both kernels ask.
template <int HD> struct A4Range {
  int start, n_new, G, col0, cols, pos0, t_lo, t_hi, c_first, n_chunks;
  __device__ inline A4Range(const A4Args& a, int row, int ct, int columns) {
    start = a.row_start ? __ldcg(a.row_start + row) : row;
    n_new = a.row_start ? __ldcg(a.row_start + row + 1) - start : 1;
    if (start < 0 || start + n_new > a.T) n_new = 0;       // (rows that q does not have)
    pos0 = __ldcg(a.row_pos0 + row);
    G = a.nh / a.nkv;
    col0 = ct * columns;
    cols = min(columns, n_new * G - col0);
    t_lo = 0; t_hi = -1; c_first = 0; n_chunks = 0;
    if (cols <= 0) return;
    const int p_lo = pos0 + col0 / G, p_hi = pos0 + (col0 + cols - 1) / G;
    if (p_hi < 0) return;
    t_lo = a.window > 0 ? max(0, p_lo - a.window + 1) / tile_tokens(HD) : 0;
    t_hi = p_hi / tile_tokens(HD);
    c_first = t_lo / a.chunk;
    n_chunks = min(t_hi / a.chunk - c_first + 1, a.max_chunks);
  }
};

// COLS: columns of a block, 4 (hi and lo side by side), 8 or 16.  BESIDE: a step's rows of more than `few` new tokens are another kernel's (a kernel of its
// own: the comparison takes 1.5 % of the time of heads of 128, 64 rows of 130 to 8,000 keys 81.6 -> 83.0 us).
template <int HD, int COLS, bool BESIDE>
__global__ void __launch_bounds__(A4_WARPS * 32, COLS == 16 ? 2 : COLS == 8 && HD == 128 ? 3 : 4)
kv4_attn_kernel(const A4Args a) {
  constexpr bool SIDE = COLS == 4;
  constexpr int NC = SIDE ? 1 : COLS / 8;                   // column blocks of an instruction
  constexpr int CP = SIDE ? 1 : 2;                          // columns of a thread in one: t, or 2 t and 2 t + 1
  constexpr int TT = tile_tokens(HD), NT = TT / 16, NG = HD / 32, SPP = HD / 64;
  constexpr int RING = A4_STAGES * TILE;
  static_assert(COLS * HD * 4 <= RING, "a warp's results take the place of its ring");
  extern __shared__ __align__(128) unsigned char a4_smem_raw[];
  __shared__ uint64_t full[A4_WARPS][A4_STAGES];
  __shared__ __align__(16) unsigned char s_q[2][COLS][HD];  // hi and lo, a lane's eight features in the order of its operand's bytes
  __shared__ float s_qsum[COLS][NG], s_f[COLS];
  __shared__ float s_m[A4_WARPS][COLS], s_l[A4_WARPS][COLS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row = blockIdx.z, kvh = blockIdx.y / a.n_ct, ct = blockIdx.y % a.n_ct;
  pdl_trigger();
  pdl_wait();
  // this warp's tiles, one a lane: tile_a + warp + 4 * lane; tiles without a page are left out.  Without a window the chunk's place says which they
  // are, and the table is read beside the row's lengths, not after them.
  auto page_of = [&](int tile) { return tile / SPP < a.bt_width ? __ldcg(a.block_table + (int64_t)row * a.bt_stride + tile / SPP) : -1; };
  int my_page = -1;
  if (a.window == 0 && warp + A4_WARPS * lane < a.chunk) my_page = page_of((int)blockIdx.x * a.chunk + warp + A4_WARPS * lane);
  const A4Range<HD> r(a, row, ct, COLS);
  if (r.cols <= 0 || (BESIDE && r.n_new > a.few) || (int)blockIdx.x >= max(r.n_chunks, 1)) return;
  const int chunk0 = (r.c_first + (int)blockIdx.x) * a.chunk;
  const int tile_a = max(r.t_lo, chunk0), tile_b = min(r.t_hi + 1, chunk0 + a.chunk);      // none where the row sees nothing
  const int my_tile = tile_a + warp + A4_WARPS * lane;
  if (a.window > 0 && my_tile < tile_b) my_page = page_of(my_tile);
  if (my_tile >= tile_b || my_page >= a.n_pages) my_page = -1;
  uint32_t todo = __ballot_sync(0xffffffffu, my_page >= 0), ask = todo;
  unsigned char* ring = a4_smem_raw + warp * RING;
  uint64_t* bars = full[warp];
  if (lane == 0) {
    for (int s = 0; s < A4_STAGES; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(a4_smem(bars + s)));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  // Tiles that every column sees as a whole come first, then those that a limit cuts: the two kinds have code of their own, and going to and fro
  // between them costs a tile some eighty moves of registers.
  const int full_hi = r.pos0 + r.col0 / r.G;                // keys that every column sees: full_lo .. full_hi
  const int full_lo = a.window > 0 ? r.pos0 + (r.col0 + r.cols - 1) / r.G - a.window + 1 : 0;
  const int seen_hi = r.pos0 + (r.col0 + r.cols - 1) / r.G;              // keys that any column sees
  const int seen_lo = a.window > 0 ? r.pos0 + r.col0 / r.G - a.window + 1 : 0;
  const int key_lane = (tile_a + warp + A4_WARPS * lane) * TT;
  const uint32_t whole = __ballot_sync(0xffffffffu, my_page >= 0 && key_lane + TT - 1 <= full_hi && key_lane >= full_lo);
  auto request = [&](int stage) {                           // the next tile of `ask` into a stage
    const int i = __ffs((ask & whole) ? ask & whole : ask) - 1;
    ask &= ~(1u << i);
    const int page = __shfl_sync(0xffffffffu, my_page, i);
    const int tile = tile_a + warp + A4_WARPS * i;
    const unsigned char* src = a.pool + ((int64_t)page * a.nkv + kvh) * page_bytes(HD) + tile % SPP * TILE;
    asm volatile(                                           // (predicated for the first lane: no branch for the warp to come together after)
        "{\n\t.reg .pred p;\n\t"
        "setp.eq.s32 p, %4, 0;\n\t"
        "@p mbarrier.arrive.expect_tx.shared::cta.b64 _, [%3], %2;\n\t"
        "@p cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}"
        ::"r"(a4_smem(ring + stage * TILE)), "l"(src), "r"(TILE), "r"(a4_smem(bars + stage)), "r"(lane) : "memory");
  };
  for (int s = 0; s < A4_STAGES; ++s)
    if (ask) request(s);

  // the queries: a warp takes every fourth column, a lane HD / 32 neighbouring features of it
#pragma unroll
  for (int c = warp; c < COLS; c += A4_WARPS) {
    const int col = r.col0 + c;
    const bool there = c < r.cols;                          // columns that are not there are zeros, computed and dropped
    const __nv_bfloat16* src = a.q + (int64_t)(r.start + (there ? col / r.G : 0)) * a.q_stride + (int64_t)(kvh * r.G + (there ? col % r.G : 0)) * HD;
    float x[NG];
    if constexpr (NG == 2) {
      const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(src) + lane);
      x[0] = __uint_as_float(w << 16); x[1] = __uint_as_float(w & 0xffff0000u);
    } else {
      const uint2 w = __ldcg(reinterpret_cast<const uint2*>(src) + lane);
      x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u);
      x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
    }
    float top = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      if (!there) x[i] = 0.0f;
      top = fmaxf(top, fabsf(x[i]));
      finite = finite && fabsf(x[i]) < __int_as_float(0x7f800000);
    }
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    finite = __all_sync(0xffffffffu, finite);
    const int e = finite && top > 0.0f ? min(max(7 + 127 - (int)(__float_as_uint(top) >> 23), -100), 100) : 0;
    const float up = a4_pow2(e);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int f = lane * NG + i;                          // the feature, and its byte among the operand's eight
      const int place = (f & ~7) + ((f >> 1) & 1) * 4 + (f & 1) * 2 + ((f >> 2) & 1);
      const float v = x[i] * up;
      const __nv_fp8_e4m3 hi(v);
      const __nv_fp8_e4m3 lo(v - (float)hi);
      sum += (float)hi + (float)lo;
      s_q[0][c][place] = hi.__x;
      s_q[1][c][place] = lo.__x;
    }
#pragma unroll
    for (int off = 1; off < 32 / NG; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane % (32 / NG) == 0) s_qsum[c][lane / (32 / NG)] = sum * 0x1p-9f;
    if (lane == 0) s_f[c] = finite ? a.scale_log2 * a4_pow2(9 - e) : __int_as_float(0x7fc00000);      // (a row that is not finite: NaN)
  }
  __syncthreads();

  constexpr int PARTS = SIDE ? 1 : 2;
  uint32_t qf[NC][PARTS][NG][2];                            // this lane's part of q': features 32 group + 8 t .. + 7
  uint32_t qsum[NC][2];                                     // Q_t in three bfloat16 parts, for the product with the keys' mn
  float fac[NC][CP];
  int limit[NC][CP];                                        // the positions of this thread's columns
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int qc = SIDE ? g >> 1 : 8 * n + g;               // the operand's column g: a column's hi or lo, or both in turn
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const uint2 v = *reinterpret_cast<const uint2*>(&s_q[SIDE ? g & 1 : part][qc][i * 32 + 8 * t]);
        qf[n][part][i][0] = v.x; qf[n][part][i][1] = v.y;
      }
    const float v = t < NG && !(SIDE && (g & 1)) ? s_qsum[qc][t] : 0.0f;
    const __nv_bfloat16 hi = __float2bfloat16_rn(v);
    const float rest = v - __bfloat162float(hi);
    const __nv_bfloat16 mid = __float2bfloat16_rn(rest), lo = __float2bfloat16_rn(rest - __bfloat162float(mid));
    qsum[n][0] = (uint32_t)__bfloat16_as_ushort(mid) << 16 | __bfloat16_as_ushort(hi);
    qsum[n][1] = __bfloat16_as_ushort(lo);
#pragma unroll
    for (int h = 0; h < CP; ++h) {
      const int c = SIDE ? t : 8 * n + 2 * t + h;
      fac[n][h] = s_f[c];
      limit[n][h] = c < r.cols ? r.pos0 + (r.col0 + c) / r.G : -1;
    }
  }
  float o[NC][NG][2][4] = {};                               // [column block][group][features 4 g + 2 k (+ 1)] x columns 2 t, 2 t + 1, in units of 2^-24
  float om[NC][NG][CP] = {};                                // sum p mn, this lane's tokens
  float m[NC][CP], ref[NC][CP], mm[NC][CP] = {}, l[NC][CP] = {};       // mm: ref, or 0 while nothing was seen
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int h = 0; h < CP; ++h) m[n][h] = ref[n][h] = __int_as_float(0xff800000);
  uint32_t sc_top = 0;                                      // the largest value scale met, rounded up to a power of two (as its exponent bits)
  float up = 0.0f;                                          // log2 F

  auto walk = [&](const unsigned char* buf, int key0, auto masked_t) {
    constexpr bool MASKED = decltype(masked_t)::value;
    float x[NT][NC][2][CP];                                 // keys g and g + 8 of 16, this thread's columns
#pragma unroll
    for (int mt = 0; mt < NT; ++mt) {
      uint32_t kw[2][NG], pw[2][NG], mn[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tok = mt * 16 + g + 8 * h;
        const unsigned char* kp = buf + tok * (HD / 2) + t * (NG * 4);
        const unsigned char* pp = buf + K_WORDS + tok * (NG * 4);
        const uint32_t own = *reinterpret_cast<const uint32_t*>(pp + (t % NG) * 4);
        mn[h] = __byte_perm(own, own, 0x1010);              // group t's mn twice
        if constexpr (NG == 2) {
          const uint2 u = *reinterpret_cast<const uint2*>(kp), v = *reinterpret_cast<const uint2*>(pp);
          kw[h][0] = u.x; kw[h][1] = u.y; pw[h][0] = v.x; pw[h][1] = v.y;
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(kp), v = *reinterpret_cast<const uint4*>(pp);
          kw[h][0] = u.x; kw[h][1] = u.y; kw[h][2] = u.z; kw[h][3] = u.w;
          pw[h][0] = v.x; pw[h][1] = v.y; pw[h][2] = v.z; pw[h][3] = v.w;
        }
      }
      float y[NC][4];
#pragma unroll
      for (int n = 0; n < NC; ++n) a4_mma_bf16_first(y[n], mn[0], mn[1], mn[0], mn[1], qsum[n][0], qsum[n][1]);      // sum_g mn_g Q_g
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const uint32_t a0 = kw[0][i] & 0x0f0f0f0fu, a1 = kw[1][i] & 0x0f0f0f0fu, a2 = (kw[0][i] >> 4) & 0x0f0f0f0fu, a3 = (kw[1][i] >> 4) & 0x0f0f0f0fu;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          float c[4];
          a4_mma8_first(c, a0, a1, a2, a3, qf[n][0][i][0], qf[n][0][i][1]);
          if constexpr (!SIDE) a4_mma8(c, a0, a1, a2, a3, qf[n][1][i][0], qf[n][1][i][1]);
          if constexpr (SIDE) {
            y[n][0] = fmaf(word_sc(pw[0][i]), c[0] + c[1], y[n][0]);
            y[n][2] = fmaf(word_sc(pw[1][i]), c[2] + c[3], y[n][2]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[n][e] = fmaf(word_sc(pw[e >> 1][i]), c[e], y[n][e]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < CP; ++c) {
            x[mt][n][h][c] = y[n][2 * h + c] * fac[n][c];
            if (MASKED) {
              const int key = key0 + mt * 16 + g + 8 * h, lim = limit[n][c];
              if (key > lim || (a.window > 0 && lim - key >= a.window)) x[mt][n][h][c] = __int_as_float(0xff800000);
            }
          }
    }
    // the values' numbers
    uint32_t vw[NT][2][NG];
    float top_word = 0.0f;                                  // the largest word, as the float it is: its scale (NaN groups do not count)
#pragma unroll
    for (int mt = 0; mt < NT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned char* pp = buf + V_WORDS + (mt * 16 + g + 8 * h) * (NG * 4);
        if constexpr (NG == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(pp);
          vw[mt][h][0] = v.x; vw[mt][h][1] = v.y;
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(pp);
          vw[mt][h][0] = v.x; vw[mt][h][1] = v.y; vw[mt][h][2] = v.z; vw[mt][h][3] = v.w;
        }
        if (MASKED) {                                       // what no column sees has no say in the scales' power of two
          const int key = key0 + mt * 16 + g + 8 * h;
          if (key > seen_hi || key < seen_lo) {
#pragma unroll
            for (int i = 0; i < NG; ++i) vw[mt][h][i] = 0;
          }
        }
#pragma unroll
        for (int i = 0; i < NG; i += 2) top_word = a4_max3(top_word, __uint_as_float(vw[mt][h][i]), __uint_as_float(vw[mt][h][i + 1]));
      }
    // A column's reference moves only when one of its scores is more than 2^8 above it, the scales' power of two only when a larger scale comes:
    // each lane looks at what it has, one vote tells, and nothing is exchanged otherwise.
    float best[NC][CP];                                     // this lane's largest score of a column
    uint32_t top = __float_as_uint(top_word) & 0x7f800000u;
    bool behind = top > sc_top;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int h = 0; h < CP; ++h) {
        float v = __int_as_float(0xff800000);
#pragma unroll
        for (int mt = 0; mt < NT; ++mt) v = a4_max3(v, x[mt][n][0][h], x[mt][n][1][h]);
        best[n][h] = v;
        behind = behind || v > ref[n][h] + (up + A4_SLACK);
      }
    if (__any_sync(0xffffffffu, behind)) {
      top = __reduce_max_sync(0xffffffffu, top);
      if (top > sc_top) {
        sc_top = top;
        up = (float)min(max(5 - ((int)(top >> 23) - 127), -100), 100);
      }
      // p = 2^(x - ref): ref is the maximum less the exponent that the values' scales want, so p carries F and nothing else has to
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int h = 0; h < CP; ++h) {
          float v = best[n][h];
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
          m[n][h] = fmaxf(m[n][h], v);
          const float now = m[n][h] - up;                   // (-inf stays)
          const float f = ref[n][h] == now ? 1.0f : a4_exp2(ref[n][h] - now);
          ref[n][h] = now;
          mm[n][h] = now == __int_as_float(0xff800000) ? 0.0f : now;
          l[n][h] *= f;
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            om[n][i][h] *= f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int at = SIDE ? i & 1 : h;              // where this column's values of the group are
              o[n][i][k][at] *= f;
              o[n][i][k][at + 2] *= f;
            }
          }
        }
    }
#pragma unroll
    for (int mt = 0; mt < NT; ++mt) {
      uint32_t pb[NC][SIDE ? NG / 2 : NG][2];               // P_g, tokens x columns, transposed
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        float p[2][CP];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < CP; ++c) {
            p[h][c] = a4_exp2(x[mt][n][h][c] - mm[n][c]);
            l[n][c] += p[h][c];
          }
        // Side by side the 8 columns have room for two groups' P: the even ones the first group's, the odd ones the second's; of a group's product
        // the other's columns are dropped.
#pragma unroll
        for (int i = 0; i < NG; i += SIDE ? 2 : 1)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float w[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int gi = SIDE ? i + c : i, col = SIDE ? 0 : c;
              const float sc = word_sc(vw[mt][h][gi]), mn = word_mn(vw[mt][h][gi]);
              const bool hidden = MASKED && x[mt][n][h][col] == __int_as_float(0xff800000);        // what is hidden may hold anything
              w[c] = hidden ? 0.0f : p[h][col] * sc;
              if (!hidden) om[n][gi][col] = fmaf(p[h][col], mn, om[n][gi][col]);
            }
            pb[n][SIDE ? i / 2 : i][h] = a4_transpose(a4_pack(w[0], w[1]));
          }
      }
#pragma unroll
      for (int half = 0; half < NG / 2; ++half) {
        const uint4 v = *reinterpret_cast<const uint4*>(buf + V_CODES + ((mt * (NG / 2) + half) * 32 + lane) * 16);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const uint32_t lo = __byte_perm(v.x, v.y, part ? 0x7632 : 0x5410), hi = __byte_perm(v.z, v.w, part ? 0x7632 : 0x5410);
          const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
          const int i = half * 2 + part, ip = SIDE ? half : i;
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            a4_mma(o[n][i][0], lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u, pb[n][ip][0], pb[n][ip][1]);
            a4_mma(o[n][i][1], lo8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x000f000fu, hi8 & 0x00f000f0u, pb[n][ip][0], pb[n][ip][1]);
          }
        }
      }
    }
  };

  bool ok = true;
  int k = 0;
  auto tiles = [&](uint32_t todo, auto masked_t) {
    while (todo && ok) {
      const int i = __ffs(todo) - 1, stage = k % A4_STAGES;
      todo &= todo - 1;
      ok = __all_sync(0xffffffffu, a4_wait(bars + stage, (k / A4_STAGES) & 1));
      if (!ok) break;
      walk(ring + stage * TILE, (tile_a + warp + A4_WARPS * i) * TT, masked_t);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");    // this lane's reads come before the copy that follows
      __syncwarp();
      if (ask) request(stage);
      ++k;
    }
  };
  tiles(todo & whole, std::false_type());
  tiles(todo & ~whole, std::true_type());
  if (!ok) {
    // copies still on their way get the time to land before this shared memory is used again
    if (lane == 0) atomicExch(&g_a4_error, 1);
    for (int i = 0; i < 1000; ++i) __nanosleep(100);
  }
  __syncwarp();

  // this warp's sums over its lanes, then its results [column][feature] in the ring's place
  float* mine = reinterpret_cast<float*>(ring);
  const float unit = 0x1p24f;
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int h = 0; h < CP; ++h) {
      const int c = SIDE ? t : 8 * n + 2 * t + h;
      float v = l[n][h];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (g == 0) { s_m[warp][c] = ref[n][h]; s_l[warp][c] = v; }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float s = om[n][i][h];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        float4 y;
        const int at = SIDE ? i & 1 : h;
        y.x = fmaf(o[n][i][0][at], unit, s);
        y.y = fmaf(o[n][i][0][at + 2], unit * 0.0625f, s);
        y.z = fmaf(o[n][i][1][at], unit, s);
        y.w = fmaf(o[n][i][1][at + 2], unit * 0.0625f, s);
        *reinterpret_cast<float4*>(mine + c * HD + i * 32 + 4 * g) = y;
      }
    }
  __syncthreads();
  // the four warps' results: one record, or the output
  const bool last = a.max_chunks == 1 || r.n_chunks <= 1;
  const int64_t rec = (((int64_t)row * a.nkv + kvh) * a.n_ct + ct) * a.max_chunks + blockIdx.x;
  for (int i = threadIdx.x; i < r.cols * (HD / 4); i += A4_WARPS * 32) {
    const int c = i / (HD / 4), d = i % (HD / 4) * 4;
    float top = s_m[0][c];
#pragma unroll
    for (int w = 1; w < A4_WARPS; ++w) top = fmaxf(top, s_m[w][c]);
    const float safe = top == __int_as_float(0xff800000) ? 0.0f : top;
    float sum = 0.0f, acc[4] = {};
#pragma unroll
    for (int w = 0; w < A4_WARPS; ++w) {
      const float f = a4_exp2(s_m[w][c] - safe);
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a4_smem_raw + w * RING) + c * HD + d);
      sum = fmaf(s_l[w][c], f, sum);
      acc[0] = fmaf(y.x, f, acc[0]); acc[1] = fmaf(y.y, f, acc[1]); acc[2] = fmaf(y.z, f, acc[2]); acc[3] = fmaf(y.w, f, acc[3]);
    }
    const int col = r.col0 + c;
    if (last) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint2 w;
      __nv_bfloat162 lo = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv), hi = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
      w.x = *reinterpret_cast<uint32_t*>(&lo);
      w.y = *reinterpret_cast<uint32_t*>(&hi);
      *reinterpret_cast<uint2*>(a.out + ((int64_t)(r.start + col / r.G) * a.nh + kvh * r.G + col % r.G) * HD + d) = w;
    } else {
      float* to = a.scratch + (rec * COLS + c) * (HD + 4);
      *reinterpret_cast<float4*>(to + 4 + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) { to[0] = top; to[1] = sum; }
    }
  }
}

// Joins the chunks of a (row, key/value head, column): a block each, its warps over the chunks, then the warps' sums.
// As many warps as leave each four chunks, up to 16: all of a warp's records are on their way at once.
template <int HD, int A4_JOIN_WARPS>
__global__ void __launch_bounds__(A4_JOIN_WARPS * 32)
kv4_join_kernel(const A4Args a, int columns) {
  constexpr int V = HD / 32;                                // features a lane
  __shared__ float s_acc[A4_JOIN_WARPS][HD], s_m[A4_JOIN_WARPS], s_l[A4_JOIN_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y / a.n_ct, ct = blockIdx.y % a.n_ct, c = blockIdx.x, row = blockIdx.z;
  pdl_trigger();
  pdl_wait();
  const float* base = a.scratch + ((((int64_t)row * a.nkv + kvh) * a.n_ct + ct) * a.max_chunks * columns + c) * (HD + 4);
  const int64_t step = (int64_t)columns * (HD + 4);
  float m = __int_as_float(0xff800000), l = 0.0f, acc[V] = {};
  float mk[4], lk[4], y[4][V];
  auto ask = [&](int k0) {                                  // records, the row's or not: what is not is never used
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + u * A4_JOIN_WARPS;
      const float* p = base + (k < a.max_chunks ? k : 0) * step;
      mk[u] = __ldcg(p);
      lk[u] = __ldcg(p + 1);
#pragma unroll
      for (int i = 0; i < V; ++i) y[u][i] = __ldcg(p + 4 + i * 32 + lane);
    }
  };
  ask(warp);                                                // (beside the row's lengths, not after them)
  const A4Range<HD> r(a, row, ct, columns);
  if (c >= r.cols || r.n_new > a.few || r.n_chunks <= 1) return;      // (a single chunk wrote the output itself)
  for (int k0 = warp; k0 < r.n_chunks; k0 += 4 * A4_JOIN_WARPS) {
    if (k0 > warp) ask(k0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (k0 + u * A4_JOIN_WARPS >= r.n_chunks) break;
      const float top = fmaxf(m, mk[u]), safe = top == __int_as_float(0xff800000) ? 0.0f : top;
      const float f0 = a4_exp2(m - safe), f1 = a4_exp2(mk[u] - safe);
      l = l * f0 + lk[u] * f1;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = acc[i] * f0 + y[u][i] * f1;
      m = top;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s_acc[warp][i * 32 + lane] = acc[i];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += A4_JOIN_WARPS * 32) {
    float top = s_m[0];
#pragma unroll
    for (int w = 1; w < A4_JOIN_WARPS; ++w) top = fmaxf(top, s_m[w]);
    const float safe = top == __int_as_float(0xff800000) ? 0.0f : top;
    float sum = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < A4_JOIN_WARPS; ++w) {
      const float f = a4_exp2(s_m[w] - safe);
      sum = fmaf(s_l[w], f, sum);
      y = fmaf(s_acc[w][d], f, y);
    }
    const int col = r.col0 + c;
    a.out[((int64_t)(r.start + col / r.G) * a.nh + kvh * r.G + col % r.G) * HD + d] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : y / sum);
  }
}

constexpr uint32_t A4_SMEM = A4_WARPS * A4_STAGES * TILE;

static int a4_columns(int wanted) { return wanted <= 4 ? 4 : wanted <= 8 ? 8 : 16; }

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_kv4_attn_status() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_a4_error, sizeof(int));
  if (v) { int z = 0; cudaMemcpyToSymbol(g_a4_error, &z, sizeof(int)); }
  return v;
}

// Floats of scratch that a call with these sizes wants (0 with one chunk).
extern "C" long long exl3_kv4_attn_scratch(int rows, int max_new, int nh, int nkv, int hd, int max_chunks) {
  if (max_chunks <= 1 || nkv < 1) return 0;
  const int ncol = max_new * (nh / nkv), columns = a4_columns(ncol);
  return (long long)rows * nkv * ceil_div(ncol, columns) * max_chunks * columns * (hd + 4);
}

extern "C" int exl3_kv4_attn(const void* q, int64_t q_stride, void* out, const void* pool, int64_t n_pages, const int* block_table,
                             int bt_stride, int bt_width, const int* row_start, const int* row_pos0, int rows, int T, int max_new, int nh, int nkv,
                             int hd, int window, float scale, int few, int chunk, int max_chunks, float* scratch, long long scratch_floats, cudaStream_t stream) {
  if (rows == 0 || max_new == 0) return 0;
  if (rows < 0 || rows > 65535 || max_new < 0 || nkv < 1 || nh < nkv || nh % nkv || (hd != 64 && hd != 128) || window < 0 || few < 0 || !isfinite(scale) || chunk < 1 ||
      chunk > A4_MAX_CHUNK || max_chunks < 1 || n_pages < 1 || n_pages > INT32_MAX || bt_width < 1 || T < 0 || !q || !out || !pool || !block_table ||
      !row_pos0 || (!row_start && max_new != 1)) {
    set_error("kv4_attn: needs heads of 64 or 128, chunks of 1 to %d tiles a finite scale and all of its arrays, got rows=%d max_new=%d heads=%d "
              "kv_heads=%d head_dim=%d scale=%g chunk=%d max_chunks=%d", A4_MAX_CHUNK, rows, max_new, nh, nkv, hd, (double)scale, chunk, max_chunks);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(q) || !aligned16(out) || !aligned16(pool) || q_stride % 8) { set_error("kv4_attn: q, its rows, out and the pool must be 16-byte aligned"); return ERR_ALIGNMENT; }
  if (max_chunks > 1 && (!scratch || scratch_floats < exl3_kv4_attn_scratch(rows, max_new, nh, nkv, hd, max_chunks))) {
    set_error("kv4_attn: %lld floats of scratch wanted", exl3_kv4_attn_scratch(rows, max_new, nh, nkv, hd, max_chunks));
    return ERR_SCRATCH;
  }
  const int ncol = max_new * (nh / nkv), columns = a4_columns(ncol);
  A4Args a = {};
  a.q = static_cast<const __nv_bfloat16*>(q); a.q_stride = q_stride; a.out = static_cast<__nv_bfloat16*>(out);
  a.pool = static_cast<const unsigned char*>(pool); a.n_pages = (int)n_pages; a.block_table = block_table; a.bt_stride = bt_stride; a.bt_width = bt_width; a.T = T;
  a.row_start = row_start; a.row_pos0 = row_pos0; a.nh = nh; a.nkv = nkv; a.window = window; a.few = few > 0 ? few : INT32_MAX; a.scale_log2 = scale * 1.4426950408889634f;
  a.chunk = chunk; a.max_chunks = max_chunks; a.n_ct = ceil_div(ncol, columns); a.scratch = scratch;
  if ((int64_t)a.nkv * a.n_ct > 65535) { set_error("kv4_attn: too many new tokens for this kernel"); return ERR_UNSUPPORTED; }
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaSuccess;
    for (const void* f : {(const void*)kv4_attn_kernel<64, 4, false>, (const void*)kv4_attn_kernel<64, 8, false>, (const void*)kv4_attn_kernel<64, 16, false>,
                          (const void*)kv4_attn_kernel<128, 4, false>, (const void*)kv4_attn_kernel<128, 8, false>, (const void*)kv4_attn_kernel<128, 16, false>,
                          (const void*)kv4_attn_kernel<64, 4, true>, (const void*)kv4_attn_kernel<64, 8, true>, (const void*)kv4_attn_kernel<64, 16, true>,
                          (const void*)kv4_attn_kernel<128, 4, true>, (const void*)kv4_attn_kernel<128, 8, true>, (const void*)kv4_attn_kernel<128, 16, true>})
      if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)A4_SMEM);
    if (e != cudaSuccess) { set_error("kv4_attn: cannot get %u bytes of shared memory: %s", A4_SMEM, cudaGetErrorString(e)); return (int)e; }
    configured = true;
  }
  const dim3 grid(max_chunks, nkv * a.n_ct, rows), block(A4_WARPS * 32);
  auto go = [&](auto kernel) { launch_pdl(kernel, grid, block, A4_SMEM, stream, a); };
  auto pick = [&](auto beside) {
    constexpr bool B = decltype(beside)::value;
    if (hd == 64) { if (columns == 4) go(kv4_attn_kernel<64, 4, B>); else if (columns == 8) go(kv4_attn_kernel<64, 8, B>); else go(kv4_attn_kernel<64, 16, B>); }
    else { if (columns == 4) go(kv4_attn_kernel<128, 4, B>); else if (columns == 8) go(kv4_attn_kernel<128, 8, B>); else go(kv4_attn_kernel<128, 16, B>); }
  };
  if (few > 0) pick(std::true_type()); else pick(std::false_type());
  int rc = launch_status("kv4_attn");
  if (rc || max_chunks == 1) return rc;
  const dim3 jgrid(columns < ncol ? columns : ncol, nkv * a.n_ct, rows);
  auto join = [&](auto kernel, int warps) { launch_pdl(kernel, jgrid, dim3(warps * 32), 0, stream, a, columns); };
  if (max_chunks <= 8) { if (hd == 64) join(kv4_join_kernel<64, 2>, 2); else join(kv4_join_kernel<128, 2>, 2); }
  else if (max_chunks <= 24) { if (hd == 64) join(kv4_join_kernel<64, 6>, 6); else join(kv4_join_kernel<128, 6>, 6); }
  else { if (hd == 64) join(kv4_join_kernel<64, 16>, 16); else join(kv4_join_kernel<128, 16>, 16); }
  return launch_status("kv4_attn join");
}
