// The 4-bit key/value cache's two ways: a step's keys and values into its pages (with the rotary encoding of queries and keys), and
// pages back into bfloat16.  The format is in cache4.cuh.
//
//   store  q, k rotated in float32 (pairs d, d + HD / 2), q rounded to bfloat16; per group of 32 features mn = bfloat16(min),
//          sc = bfloat16((max - mn) / 15), code = clamp(rint((x - mn) * (1 / sc)), 0, 15) on the float32 values.  A group that holds a
//          value that is not finite, or whose range is not, becomes NaN as a whole.
//   load   mn + sc * code (exact in float32: 8 x 4 bits) rounded to bfloat16, or to fp16 for the prompt attention, times a power of two for a row's
//          keys of a head and one for its values.
//
// Measured, 4,096 tokens of 36 heads of 64 with 36 key and value heads: store 29.6 us (87 MB, 2.9 TB/s), load of its pages 13.0 us (49 MB, 3.8 TB/s);
// a step of 64 tokens of 32 heads of 128 with 8 and 8: store 2.9 us, load of 64 pages 7.5 us.  The load is bound by memory, the store of many
// tokens by its instructions (some 220 for the warp's four token and head pairs; 245, 31 us and issue slots 79 % busy before pairs of floats; of these 31,
// 29 without a store to the pool, 28 without loads), that of a decode step by its launch.
#include "api.h"
#include "cache4.cuh"
#include "cache4_rows.cuh"

namespace exl3 {

using namespace kv4;

constexpr int C4_THREADS = 256;

__device__ inline float c4_min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ inline float c4_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two floats at a time; each rounds as the scalar instruction does.
__device__ inline uint64_t c4_pair(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ inline void c4_unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ inline uint64_t c4_add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ inline uint64_t c4_mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ inline uint64_t c4_fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

// A lane has features 8 j .. 8 j + 7 of a head (j = 0 .. HD / 8 - 1); four neighbouring lanes have a group.  Returns the group's word and
// the lane's eight codes as the low bits of floats around 1.5 * 2^23: adding that number rounds to an integer, ties to even, and leaves it there
// (conversions have a pipe of a quarter of the others' rate: they and the shifts that put the codes together were half of the kernel's time).
__device__ inline uint32_t c4_quantize(const float (&x)[8], uint32_t (&bits)[8]) {
  constexpr float ROUND = 12582912.0f;
  float lo = c4_min3(x[0], x[1], x[2]), hi = c4_max3(x[0], x[1], x[2]);
  lo = c4_min3(lo, x[3], x[4]); hi = c4_max3(hi, x[3], x[4]);
  lo = c4_min3(lo, x[5], x[6]); hi = c4_max3(hi, x[5], x[6]);
  lo = fminf(lo, x[7]); hi = fmaxf(hi, x[7]);
  uint64_t odd2 = 0;                                                   // zeros, or NaN where a value is not finite
#pragma unroll
  for (int e = 0; e < 8; e += 2) odd2 = c4_fma2(c4_pair(x[e], x[e + 1]), 0, odd2);
  float odd, odd_b;
  c4_unpair(odd2, odd, odd_b);
  if (odd + odd_b != 0.0f) { lo = __int_as_float(0xff800000); hi = __int_as_float(0x7f800000); }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const __nv_bfloat16 mnb = __float2bfloat16_rn(lo);
  const float mn = __bfloat162float(mnb);
  const float range = fmaxf(hi - mn, 0.0f);
  const __nv_bfloat16 scb = __float2bfloat16_rn(__fdiv_rn(range, 15.0f));
  const float sc = __bfloat162float(scb);
  const bool fine = sc < __int_as_float(0x7f800000) && fabsf(mn) < __int_as_float(0x7f800000);
  const float inv = fine && sc > SC_MIN ? __frcp_rn(sc) : 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float a, b;
    c4_unpair(c4_mul2(c4_add2(c4_pair(x[e], x[e + 1]), c4_pair(-mn, -mn)), c4_pair(inv, inv)), a, b);
    a = fminf(fmaxf(a, 0.0f), 15.0f);                                  // (NaN becomes 0)
    b = fminf(fmaxf(b, 0.0f), 15.0f);
    c4_unpair(c4_add2(c4_pair(a, b), c4_pair(ROUND, ROUND)), a, b);
    bits[e] = __float_as_uint(a);
    bits[e + 1] = __float_as_uint(b);
  }
  return fine ? (uint32_t)__bfloat16_as_ushort(scb) << 16 | __bfloat16_as_ushort(mnb) : 0x7fc07fc0u;
}
// The codes as a word: feature e's in nibble e, or (keys) in nibble e / 2 + 4 (e % 2).  Multiply-adds modulo 2^32; what the floats have above their
// codes adds up to a constant.
template <bool KEY> __device__ inline uint32_t c4_word(const uint32_t (&bits)[8]) {
  uint32_t w = 0u - 0x4b400000u * 0x11111111u;
#pragma unroll
  for (int e = 0; e < 8; ++e) w += bits[e] * (1u << (4 * (KEY ? e / 2 + 4 * (e % 2) : e)));
  return w;
}
// Code e of a word as a float.
__device__ inline float c4_code(uint32_t w, int shift) { return __uint_as_float(((w >> shift) & 15u) | 0x4b000000u) - 8388608.0f; }

// A block takes TOK tokens (their positions, pages and sines at once: three trips to memory that stand in a row for each block) and the
// (token, head) pairs blockIdx.y, + gridDim.y, ... in steps of as many as its threads cover; the next pair's features are asked for
// before this one's are worked on.
template <int HD, int TOK>
__global__ void __launch_bounds__(C4_THREADS)
kv4_store_kernel(const __nv_bfloat16* __restrict__ qkv, int64_t qkv_stride, __nv_bfloat16* __restrict__ q_out,
                 const float* __restrict__ freq, const float* __restrict__ freq_lo, const int* __restrict__ tok_pos,
                 const int* __restrict__ tok_seq, const int* __restrict__ block_table, int bt_stride, int bt_rows, int bt_width,
                 unsigned char* __restrict__ pool, int n_pages, int T, int nh, int nkv) {
  constexpr int LANES = HD / 8, HEADS = C4_THREADS / LANES;           // pairs that the block works on side by side
  __shared__ __align__(16) float s_cos[TOK][HD / 2], s_sin[TOK][HD / 2];
  __shared__ int s_pos[TOK], s_page[TOK];
  pdl_trigger();
  pdl_wait();
  const int t0 = blockIdx.x * TOK, n_tok = min(TOK, T - t0);
  const int j = threadIdx.x % LANES, jp = j ^ (LANES / 2);
  const int total = nh + 2 * nkv, pairs = n_tok * total;
  auto ask = [&](int tk, int head, uint4& own, uint4& other) {
    own = other = make_uint4(0, 0, 0, 0);
    if (tk >= n_tok) return;
    const __nv_bfloat16* src = qkv + (int64_t)(t0 + tk) * qkv_stride + head * HD;
    own = load_raw_cg(src + 8 * j);
    if (freq && head < nh + nkv) other = load_raw_cg(src + 8 * jp);
  };
  const int step = gridDim.y * HEADS, step_t = step / total, step_h = step % total;
  const int i = blockIdx.y * HEADS + threadIdx.x / LANES;
  int tk = i / total, head = i % total;                               // this pair; the next one is step_t tokens and step_h heads on
  uint4 own, other;
  ask(tk, head, own, other);
  if (threadIdx.x < n_tok) {
    const int pos = __ldcg(tok_pos + t0 + threadIdx.x), seq = __ldcg(tok_seq + t0 + threadIdx.x);
    s_pos[threadIdx.x] = pos;
    const bool there = pos >= 0 && pos / PAGE < bt_width && seq >= 0 && seq < bt_rows;
    s_page[threadIdx.x] = there ? __ldcg(block_table + (int64_t)seq * bt_stride + pos / PAGE) : -1;
  }
  if (freq)
    for (int d = threadIdx.x; d < n_tok * (HD / 2); d += C4_THREADS)
      rope_sincos((float)__ldcg(tok_pos + t0 + d / (HD / 2)), __ldg(freq + d % (HD / 2)), freq_lo ? __ldg(freq_lo + d % (HD / 2)) : 0.0f,
                  &s_sin[0][0] + d, &s_cos[0][0] + d);
  __syncthreads();
  const uint32_t flip = j < LANES / 2 ? 0x80008000u : 0u;             // the lower half of a head subtracts its partner's sines
  for (int first = blockIdx.y * HEADS; first < pairs; first += step) {
    const bool live = tk < n_tok;                                      // (the whole group of lanes; the shuffles need everybody)
    const int now = live ? tk : 0, hd_now = live ? head : 0, t = t0 + now;
    tk += step_t;
    head += step_h;
    if (head >= total) { head -= total; ++tk; }
    uint4 next_own, next_other;
    ask(tk, head, next_own, next_other);
    float x[8];
    unpack_raw(own, x, static_cast<const __nv_bfloat16*>(nullptr));
    if (freq && hd_now < nh + nkv) {
      float y[8];
      other.x ^= flip; other.y ^= flip; other.z ^= flip; other.w ^= flip;
      unpack_raw(other, y, static_cast<const __nv_bfloat16*>(nullptr));
      const int d0 = 8 * (j & (LANES / 2 - 1));
      float c[8], sn[8];
      *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(&s_cos[now][d0]);
      *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(&s_cos[now][d0 + 4]);
      *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(&s_sin[now][d0]);
      *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(&s_sin[now][d0 + 4]);
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        c4_unpair(c4_fma2(c4_pair(x[e], x[e + 1]), c4_pair(c[e], c[e + 1]), c4_mul2(c4_pair(y[e], y[e + 1]), c4_pair(sn[e], sn[e + 1]))), x[e], x[e + 1]);
    }
    own = next_own;
    other = next_other;
    if (live && hd_now < nh) store_vec(q_out + ((int64_t)t * nh + hd_now) * HD + 8 * j, x);
    // (warps that hold queries only skip the rest)
    if (__all_sync(0xffffffffu, hd_now < nh || !live)) continue;
    uint32_t bits[8];
    const uint32_t word = c4_quantize(x, bits);
    const bool key = hd_now < nh + nkv;
    const uint32_t codes = key ? c4_word<true>(bits) : c4_word<false>(bits);
    // values: a word has four features of one group below and four of the next above: lanes j and j ^ 4 trade halves
    const uint32_t give = (j & 4) ? codes & 0xffffu : codes >> 16;
    const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 4);
    const int page = s_page[now];
    if (!live || hd_now < nh || page < 0 || page >= n_pages) continue;
    const int kv = key ? hd_now - nh : hd_now - nh - nkv;
    const int slot = s_pos[now] % PAGE, tok = slot % tile_tokens(HD);
    unsigned char* tile = pool + ((int64_t)page * nkv + kv) * page_bytes(HD) + slot / tile_tokens(HD) * TILE;
    if (key) {
      *reinterpret_cast<uint32_t*>(tile + k_word<HD>(tok, j & 3, j >> 2)) = codes;
    } else {
      const int half = j >> 3, jj = j & 7;
      const uint32_t w = jj < 4 ? (codes & 0xffffu) | got << 16 : got | (codes & 0xffff0000u);
      *reinterpret_cast<uint32_t*>(tile + v_word<HD>(tok, half, jj < 4 ? 2 * jj : 2 * (jj - 4) + 1)) = w;
    }
    if ((j & 3) == 0)
      *reinterpret_cast<uint32_t*>(tile + (key ? K_WORDS : V_WORDS) + (tok * (HD / 32) + (j >> 2)) * 4) = word;
  }
}

// fp16 holds up to 65,504 (places that no query sees may hold more than a row's factor is made for); NaN stays.
template <typename T> __device__ inline T c4_out(float v);
template <> __device__ inline __nv_bfloat16 c4_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ inline __half c4_out<__half>(float v) { return __float2half_rn(fabsf(v) > 65504.0f ? copysignf(65504.0f, v) : v); }

// A page of a kv head, keys and values, to T [64][HD] each: a thread has eight features of both of a few tokens, and asks for all of their words
// before it uses the first.  CLEAN, for a product that multiplies hidden values by zero: places from `held` on are zeros, and a token with a NaN
// among its values has zeros there and NaN in all of its key, which a mask can hide; keys are multiplied by k_up, values by v_up (powers of two).
template <int HD, bool CLEAN, typename T>
__device__ inline void c4_unpack(const unsigned char* __restrict__ base, bool there, int held, float k_up, float v_up, T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int LANES = HD / 8, N = PAGE * LANES / C4_THREADS;
  uint32_t kw[N], kc[N], vw[N], vc[N][2];
  const int j = threadIdx.x % LANES, half = j >> 3, jj = j & 7;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = (i * C4_THREADS + threadIdx.x) / LANES, tok = slot % tile_tokens(HD);
    const unsigned char* tile = base + slot / tile_tokens(HD) * TILE;
    auto word = [&](int at) { return __ldcg(reinterpret_cast<const uint32_t*>(tile + at)); };
    kw[i] = word(K_WORDS + (tok * (HD / 32) + (j >> 2)) * 4);
    vw[i] = word(V_WORDS + (tok * (HD / 32) + (j >> 2)) * 4);
    kc[i] = word(k_word<HD>(tok, j & 3, j >> 2));
    vc[i][0] = word(v_word<HD>(tok, half, 2 * (jj & 3)));
    vc[i][1] = word(v_word<HD>(tok, half, 2 * (jj & 3) + 1));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = (i * C4_THREADS + threadIdx.x) / LANES;
    bool hide_key = false, zero = !there;
    if (CLEAN) {
      const bool nan = !(fabsf(word_sc(vw[i])) < __int_as_float(0x7f800000)) || !(fabsf(word_mn(vw[i])) < __int_as_float(0x7f800000));
      const uint32_t of_token = ((1u << LANES) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
      hide_key = (__ballot_sync(0xffffffffu, nan) & of_token) != 0;
      zero = zero || slot >= held;
      if (nan) vw[i] = vc[i][0] = vc[i][1] = 0;
    }
    __align__(16) T k[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = fmaf(word_sc(kw[i]), c4_code(kc[i], 4 * (e / 2 + 4 * (e % 2))), word_mn(kw[i]));
      float y = fmaf(word_sc(vw[i]), c4_code(jj < 4 ? vc[i][e >> 2] : vc[i][e >> 2] >> 16, 4 * (e & 3)), word_mn(vw[i]));
      if (CLEAN) { x *= k_up; y *= v_up; }
      k[e] = c4_out<T>(zero ? 0.0f : hide_key ? __int_as_float(0x7fc00000) : x);
      v[e] = c4_out<T>(zero ? 0.0f : y);
    }
    *reinterpret_cast<uint4*>(k_out + slot * HD + 8 * j) = *reinterpret_cast<const uint4*>(k);
    *reinterpret_cast<uint4*>(v_out + slot * HD + 8 * j) = *reinterpret_cast<const uint4*>(v);
  }
}

// Pages listed in `pages` to bfloat16 [n, nkv, 64, HD]: a block per (page, kv head).
template <int HD>
__global__ void __launch_bounds__(C4_THREADS)
kv4_load_kernel(const unsigned char* __restrict__ pool, const int* __restrict__ pages, int n_pages, int nkv,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out) {
  pdl_trigger();
  pdl_wait();
  const int page = __ldcg(pages + blockIdx.x), kv = blockIdx.y;
  const bool there = page >= 0 && page < n_pages;
  const int64_t at = ((int64_t)blockIdx.x * nkv + kv) * PAGE * HD;
  c4_unpack<HD, false>(pool + ((int64_t)(there ? page : 0) * nkv + kv) * page_bytes(HD), there, PAGE, 1.0f, 1.0f, k_out + at, v_out + at);
}

// ---- prompts: fp16 copies of the rows' pages and of the queries, for the prompt attention ------------------------------------------

// The exponent of the power of two that brings numbers up to `top` below 2^15.  Down to 2^-110 that leaves all of fp16's bits to what is within 2^28
// of the top.
__device__ inline int c4_up(float top) { return top > 0.0f ? min(max(14 + 127 - (int)(__float_as_uint(top) >> 23), -113), 96) : 0; }
__device__ inline float c4_pow2(int e) { return __int_as_float((127 + e) << 23); }

// A warp per (row, kv head, part of the row's pages): the largest |key| and |value| among the places that some query of the row sees, from the
// groups' words: a group's values lie between mn and mn + 15 sc.  NaN groups do not count.
template <int HD> __device__ inline void c4_tops(const C4Prompt& a, int64_t item) {
  constexpr int SPP = HD / 64, NG = HD / 32, AHEAD = 4;                // tiles of a page, groups of a token, pages asked for at a time
  const int lane = threadIdx.x & 31, part = (int)(item % a.parts), kv = (int)(item / a.parts % a.nkv), row = (int)(item / a.parts / a.nkv);
  const int pos0 = __ldcg(a.row_pos0 + row), n_new = __ldcg(a.row_start + row + 1) - __ldcg(a.row_start + row), end = pos0 + n_new;
  if (n_new <= a.few) return;
  const int first = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;    // places first .. end - 1 are seen
  const int pages = end > 0 ? min(min((end - 1) / PAGE + 1, a.width), first / PAGE + a.row_pages) : 0;
  float top[2] = {0.0f, 0.0f};
  for (int j0 = first / PAGE + part * AHEAD; j0 < pages; j0 += a.parts * AHEAD) {
    uint4 w[AHEAD][SPP][2];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int page = j0 + u < pages ? __ldcg(a.block_table + (int64_t)row * a.bt_stride + j0 + u) : -1;
      const bool there = page >= 0 && page < a.n_pages;
      const unsigned char* base = a.pool + ((int64_t)(there ? page : 0) * a.nkv + kv) * page_bytes(HD) + 16 * lane;
#pragma unroll
      for (int i = 0; i < SPP; ++i) {
        w[u][i][0] = w[u][i][1] = make_uint4(0, 0, 0, 0);
        if (there) {
          w[u][i][0] = load_raw_cg(base + i * TILE + K_WORDS);
          w[u][i][1] = load_raw_cg(base + i * TILE + V_WORDS);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int i = 0; i < SPP; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {                                  // word 4 lane + e of the tile: its token and group
          const int place = (j0 + u) * PAGE + i * tile_tokens(HD) + (4 * lane + e) / NG;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint4& v = w[u][i][x];
            const uint32_t word = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
            if (place >= first && place < end) top[x] = c4_max3(top[x], fabsf(word_mn(word)), fabsf(fmaf(word_sc(word), 15.0f, word_mn(word))));
          }
        }
  }
  top[0] = warp_max(top[0]);
  top[1] = warp_max(top[1]);
  if (lane == 0) a.tops[item] = make_float2(top[0], top[1]);
}
// The exponents of a row's keys and values (every lane of the warp).
__device__ inline int2 c4_row_up(const C4Prompt& a, int64_t row_and_head) {
  const int lane = threadIdx.x & 31;
  const float2 t = lane < a.parts ? __ldcg(a.tops + row_and_head * a.parts + lane) : make_float2(0.0f, 0.0f);
  return make_int2(c4_up(warp_max(t.x)), c4_up(warp_max(t.y)));
}

// A warp per row: where the copies of its pages will be, and whether some page that its queries look for is not there.
__device__ inline void c4_row(const C4Prompt& a, int row) {
  const int lane = threadIdx.x & 31;
  const int end = __ldcg(a.row_pos0 + row) + __ldcg(a.row_start + row + 1) - __ldcg(a.row_start + row);      // positions 0 .. end - 1
  const int pages = end > 0 ? (end - 1) / PAGE + 1 : 0, count = min(pages, a.width);
  bool holes = pages > count;
  for (int j = lane; j < count; j += 32) {
    const int page = __ldcg(a.block_table + (int64_t)row * a.bt_stride + j);
    holes = holes || page < 0 || page >= a.n_pages;
  }
  holes = __any_sync(0xffffffffu, holes);
  if (lane == 0) a.own[row] = {0, count, row * a.width, holes ? 1 : 0};
}

// Sum over the block's threads below this one, and (total) over all of them; warp_sums has room for 32 and one more.
__device__ inline int c4_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                                                     // (the sums of the call before have been read)
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < C4_THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + x - v;
}

// One block: the pages that some query of a row sees, one row behind the other, and the passes they fall into.  What the sizes do not allow for (a row of
// more pages than was said) is not copied, so nobody sees it.
__device__ inline void c4_plan_rows(const C4Prompt& a) {
  constexpr int N = C4_THREADS, WARPS = N / 32;
  __shared__ int warp_sums[32], s_pass[N], s_holes[N], s_end[N];
  __shared__ FaRow s_row[N];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int p = tid; p < a.passes; p += N) a.pass[p].slot0 = a.pass[p].slots = 0;
  int base = 0, open = -1, open_slot0 = 0;                             // the pass of the last row so far, and its first slot
  for (int r0 = 0; r0 < a.rows; r0 += N) {
    const int row = r0 + tid, here = min(N, a.rows - r0);
    int lo = 0, pages = 0, count = 0, end = 0;
    if (row < a.rows) {
      const int n_new = __ldcg(a.row_start + row + 1) - __ldcg(a.row_start + row), pos0 = __ldcg(a.row_pos0 + row);
      end = pos0 + n_new;
      if (n_new > a.few && end > 0) {
        lo = a.window > 0 ? max(0, pos0 - a.window + 1) / PAGE : 0;
        pages = (end - 1) / PAGE + 1 - lo;
        count = max(0, min(min(pages, a.width - lo), a.row_pages));
      }
    }
    int all;
    const int at = min(base + c4_scan(count, warp_sums, all), a.total);
    base += all;
    count = min(count, a.total - at);
    s_row[tid] = {lo, count, at, 0};
    s_holes[tid] = pages > count;
    s_end[tid] = end;
    s_pass[tid] = min(at / a.stride, a.passes - 1);
    __syncthreads();
    const int per = here < WARPS ? WARPS / here : 1;                   // warps of a row
    for (int r = warp / per; r < here && warp < WARPS / per * per; r += WARPS / per) {
      const FaRow w = s_row[r];
      bool holes = false;
#pragma unroll 4
      for (int k = warp % per * 32 + lane; k < w.count; k += 32 * per) {
        const int page = __ldcg(a.block_table + (int64_t)(r0 + r) * a.bt_stride + w.lo + k);
        const bool there = page >= 0 && page < a.n_pages;
        holes = holes || !there;
        a.slot[w.base + k] = make_int4(r0 + r, there ? page : -1, s_end[r] - (w.lo + k) * PAGE, k == 0);
      }
      if (holes) s_holes[r] = 1;
    }
    __syncthreads();
    int slot0 = open_slot0, mine = s_pass[tid];
    if (mine != open) {                                                // the first row of the pass is one of these
      int x = 0, y = tid;
      while (x < y) {
        const int mid = (x + y) / 2;
        if (s_pass[mid] < mine) x = mid + 1; else y = mid;
      }
      slot0 = s_row[x].base;
    }
    if (row < a.rows) {
      a.own[row] = {lo, count, at - slot0, s_holes[tid]};
      a.pass_of[row] = mine;
      if (tid + 1 == here || s_pass[tid + 1] != mine) {                // the pass's last row so far
        a.pass[mine].slot0 = slot0;
        a.pass[mine].slots = at + count - slot0;
      }
    }
    const int last = s_pass[here - 1];
    if (last != open) {
      int x = 0, y = here - 1;
      while (x < y) {
        const int mid = (x + y) / 2;
        if (s_pass[mid] < last) x = mid + 1; else y = mid;
      }
      open = last;
      open_slot0 = s_row[x].base;
    }
    __syncthreads();                                                   // (shared memory is the next rows')
  }
}

// One block: the tiles of queries by passes, within one in the given order.
__device__ inline void c4_plan_tiles(const C4Prompt& a) {
  __shared__ int warp_sums[32];
  int out = 0;
  for (int p = 0; p < a.passes; ++p) {
    const int first = out;
    for (int t0 = 0; t0 < a.n_tiles; t0 += C4_THREADS) {
      const int t = t0 + threadIdx.x, row = t < a.n_tiles ? __ldcg(a.tile_seq + t) : -1, q0 = t < a.n_tiles ? __ldcg(a.tile_q0 + t) : 0;
      bool mine = row >= 0 && row < a.rows && (a.passes == 1 || __ldcg(a.pass_of + row) == p);
      int start = 0, n_new = 0, pos0 = 0;
      if (mine) {
        start = __ldcg(a.row_start + row);
        n_new = __ldcg(a.row_start + row + 1) - start;
        pos0 = __ldcg(a.row_pos0 + row);
        mine = n_new > a.few;
      }
      int all;
      const int at = out + c4_scan(mine ? 1 : 0, warp_sums, all);
      if (mine) a.tile[at] = {row, start + q0, min(a.tile_queries, n_new - q0), pos0 + q0};
      out += all;
    }
    if (threadIdx.x == 0) { a.pass[p].tile0 = first; a.pass[p].tiles = out - first; }
  }
}

// The plan, and the sizes of the rows' keys and values.
template <int HD>
__global__ void __launch_bounds__(C4_THREADS)
kv4_prompt_plan_kernel(const C4Prompt a) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0) {
    c4_plan_rows(a);
    __syncthreads();
    if (a.passes > 1) c4_plan_tiles(a);                                // (by the rows' passes)
    return;
  }
  if (blockIdx.x == 1) {
    if (a.passes == 1) c4_plan_tiles(a);
    return;
  }
  const int64_t item = (int64_t)(blockIdx.x - 2) * (C4_THREADS / 32) + (threadIdx.x >> 5);
  if (item < (int64_t)a.rows * a.nkv * a.parts) c4_tops<HD>(a, item);
}

// Eight lanes (sixteen for heads of 128) have a query of a head: to fp16, times a power of two that brings its largest value to [2^10, 2^11), whose
// inverse goes to q_scale, and the sign of the scale.  A query with a value that is not finite becomes NaN.
template <int HD> __device__ inline void c4_query(const C4Prompt& a, int64_t item) {
  constexpr int LANES = HD / 8;
  const int j = threadIdx.x % LANES;
  const bool live = item < (int64_t)a.T * a.nh;
  const int64_t t = live ? item / a.nh : 0;
  const int head = live ? (int)(item % a.nh) : 0;
  float x[8];
  load_vec_cg(a.q + t * a.q_stride + (int64_t)head * HD + 8 * j, x);
  float top = 0.0f;
  bool finite = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top = fmaxf(top, fabsf(x[e]));
    finite = finite && fabsf(x[e]) < __int_as_float(0x7f800000);
  }
  if (!finite) top = __int_as_float(0x7f800000);
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  finite = top < __int_as_float(0x7f800000);
  const int e2 = finite && top > 0.0f ? min(max(10 + 127 - (int)(__float_as_uint(top) >> 23), -100), 100) : 0;
  const float up = c4_pow2(e2) * a.q_sign;
  if (!live) return;
  __align__(16) __half h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = finite ? __float2half_rn(x[e] * up) : __ushort_as_half(0x7e00);
  *reinterpret_cast<uint4*>(a.q_out + (t * a.nh + head) * HD + 8 * j) = *reinterpret_cast<const uint4*>(h);
  if (j == 0) a.q_scale[t * a.nh + head] = c4_pow2(-e2);
}

// A pass's pages, a block per (slot, kv head), times the powers of two that bring the row's keys and values of that head up to fp16's
// largest; the block of a row's first page keeps what undoes them.  No copy is written of a page that is not there.  The blocks behind have the queries.
template <int HD>
__global__ void __launch_bounds__(C4_THREADS)
kv4_unpack16_kernel(const C4Prompt a, int pass, int page_blocks) {
  pdl_trigger();
  pdl_wait();
  if ((int)blockIdx.x >= page_blocks) {
    c4_query<HD>(a, (int64_t)(blockIdx.x - page_blocks) * (C4_THREADS * 8 / HD) + threadIdx.x / (HD / 8));
    return;
  }
  const int i = (int)(blockIdx.x / a.nkv), kv = (int)(blockIdx.x % a.nkv);
  const int2 of = __ldcg(reinterpret_cast<const int2*>(a.pass + pass));               // slot0, slots
  const int4 slot = __ldcg(a.slot + (a.passes == 1 ? i : of.y > i ? of.x + i : 0));   // (beside the pass where there is but one)
  if (i >= of.y) return;
  const int row = slot.x, page = slot.y, held = slot.z;
  const int2 up = c4_row_up(a, (int64_t)row * a.nkv + kv);
  if (slot.w && threadIdx.x == 0) a.undo[row * a.nkv + kv] = make_float2(c4_pow2(-up.x), c4_pow2(-up.y));
  if (page < 0) return;
  const int64_t at = ((int64_t)i * a.nkv + kv) * PAGE * HD;
  c4_unpack<HD, true>(a.pool + ((int64_t)page * a.nkv + kv) * page_bytes(HD), true, held, c4_pow2(up.x), c4_pow2(up.y), a.k_out + at, a.v_out + at);
}

int c4_prompt_plan(const C4Prompt& a, int hd, cudaStream_t stream) {
  const int warps = C4_THREADS / 32;
  const int64_t blocks = 2 + ((int64_t)a.rows * a.nkv * a.parts + warps - 1) / warps;
  if (blocks > INT32_MAX) { set_error("kv4_prompt: too many rows"); return ERR_UNSUPPORTED; }
  auto go = [&](auto kernel) { launch_pdl(kernel, dim3((unsigned)blocks), dim3(C4_THREADS), 0, stream, a); };
  if (hd == 64) go(kv4_prompt_plan_kernel<64>); else go(kv4_prompt_plan_kernel<128>);
  return launch_status("kv4_prompt_plan");
}

int c4_prompt_copies(const C4Prompt& a, int hd, int pass, int slots, cudaStream_t stream) {
  const int per = C4_THREADS / (hd / 8);
  const int64_t page_blocks = (int64_t)slots * a.nkv, blocks = page_blocks + (pass == 0 ? ((int64_t)a.T * a.nh + per - 1) / per : 0);
  if (blocks > INT32_MAX) { set_error("kv4_prompt: too many pages or tokens"); return ERR_UNSUPPORTED; }
  auto go = [&](auto kernel) { launch_pdl(kernel, dim3((unsigned)blocks), dim3(C4_THREADS), 0, stream, a, pass, (int)page_blocks); };
  if (hd == 64) go(kv4_unpack16_kernel<64>); else go(kv4_unpack16_kernel<128>);
  return launch_status("kv4_unpack16");
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_kv4_store(const void* qkv, int64_t qkv_stride, void* q_out, const float* freq, const float* freq_lo, const int* tok_pos,
                              const int* tok_seq, const int* block_table, int bt_stride, int bt_rows, int bt_width, void* pool, int64_t n_pages, int T,
                              int nh, int nkv, int hd, cudaStream_t stream) {
  if (T == 0) return 0;
  if (T < 0 || nh < 1 || nkv < 1 || (hd != 64 && hd != 128) || n_pages < 1 || n_pages > INT32_MAX || bt_rows < 1 || bt_width < 1 || !qkv || !q_out ||
      !tok_pos || !tok_seq || !block_table || !pool) {
    set_error("kv4_store: needs heads of 64 or 128 and all of its arrays, got T=%d heads=%d kv_heads=%d head_dim=%d", T, nh, nkv, hd);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(pool) || qkv_stride % 8) { set_error("kv4_store: qkv, its rows, q and the pool must be 16-byte aligned"); return ERR_ALIGNMENT; }
  // Few tokens: one a block, its heads over several blocks; many: four a block.
  const int per = C4_THREADS / (hd / 8), rounds = ceil_div(nh + 2 * nkv, per);
  const bool many = T >= 1024;
  const int gy = many ? 1 : T >= 296 ? 1 : rounds < 32 ? rounds : 32;
  auto go = [&](auto kernel) {
    launch_pdl(kernel, dim3(many ? ceil_div(T, 4) : T, gy), dim3(C4_THREADS), 0, stream, static_cast<const __nv_bfloat16*>(qkv), qkv_stride,
               static_cast<__nv_bfloat16*>(q_out), freq, freq_lo, tok_pos, tok_seq, block_table, bt_stride, bt_rows, bt_width, static_cast<unsigned char*>(pool),
               (int)n_pages, T, nh, nkv);
  };
  if (hd == 64) { if (many) go(kv4_store_kernel<64, 4>); else go(kv4_store_kernel<64, 1>); }
  else { if (many) go(kv4_store_kernel<128, 4>); else go(kv4_store_kernel<128, 1>); }
  return launch_status("kv4_store");
}

extern "C" int exl3_kv4_load(const void* pool, int64_t n_pages, const int* pages, int n, int nkv, int hd, void* k_out, void* v_out,
                             cudaStream_t stream) {
  if (n == 0) return 0;
  if (n < 0 || nkv < 1 || nkv > 65535 || (hd != 64 && hd != 128) || n_pages < 1 || n_pages > INT32_MAX || !pool || !pages || !k_out || !v_out) {
    set_error("kv4_load: needs heads of 64 or 128 and all of its arrays, got %d pages, kv_heads=%d head_dim=%d", n, nkv, hd);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(pool) || !aligned16(k_out) || !aligned16(v_out)) { set_error("kv4_load: the pool and the results must be 16-byte aligned"); return ERR_ALIGNMENT; }
  auto go = [&](auto kernel) {
    launch_pdl(kernel, dim3(n, nkv), dim3(C4_THREADS), 0, stream, static_cast<const unsigned char*>(pool), pages, (int)n_pages, nkv,
               static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out));
  };
  if (hd == 64) go(kv4_load_kernel<64>); else go(kv4_load_kernel<128>);
  return launch_status("kv4_load");
}
