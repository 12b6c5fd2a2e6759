// Products of 1 to 8 rows with weights in 8-bit floating point (fp8.cuh): a stream of the weights through mma.m16n8k32, with nothing to set up.
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} cx[m, k] cw[n, k]  (+ bias, or silu(gate) * up)
//
// Bound by the weights' bytes, and for small matrices by what a launch costs that depends on the one before.  So: a warp asks for 16 rows x
// 128 features = 2 KB of weights at a time, straight into the registers that the instruction reads them from, three such pieces ahead; the
// first are on their way before the kernel ahead has ended, since no kernel writes weights.  The order of K inside a product is free: a lane takes
// 16 bytes that lie together for what the instruction calls features 4 t .. and 16 + 4 t .. of two steps, and x's codes are put down in the
// same order.  (The same pieces through shared memory, with registers for two kernels at a time: 6.0 against 4.9 us for 2,304 x 5,760.)
//
// x is rounded by every block for itself, all of it, while its first weights come: that is cheap for a few rows and makes up a third of the time
// for eight of 5,760 (7.4 us, fp8_skinny.cu 7.0), hence f8v_pays.  The warps of a block share K (warp w takes the blocks w, w + warps, ... of
// 128).  Each block's product of 128 is added to float32 registers times sx * sw, and the warps' sums meet in shared memory in the warps' order,
// 16 rows of weights at a time.
//
// Measured in a chain of itself, us (fp8_skinny.cu, which sets up tensor memory, barriers and a cluster; the weights' bytes at the copy rate),
// one row: 2,304 x 2,304 2.9 (4.9; 0.8), 2,304 x 5,760 4.9 (6.5; 2.1), 6,912 x 2,304 5.4 (6.6; 2.5), 11,520 x 2,304 7.5 (8.9; 4.1),
// 4,096 x 4,096 5.1 (6.9; 2.6); four rows of 2,304 x 5,760 5.7 (6.8).
#include "api.h"
#include "fp8.cuh"
#include "gemv_bf16.cuh"

namespace exl3 {

constexpr int F8V_WARPS = 16;                             // at most
constexpr int F8V_AHEAD = 3;                              // pieces of weights that a warp has asked for
constexpr int F8V_ROUND = 4;                              // blocks of x that eight lanes have asked for
constexpr int F8V_COL = 20;                               // floats from a column's 16 sums to the next one's: four columns in different banks

struct F8vArgs {
  const __nv_bfloat16* x;
  int64_t ldx;
  const unsigned char* w;
  const float* sw;
  const __nv_bfloat16* bias;
  void* y;
  int M, N, K, kblocks, tiles, gated, y_f32;
};

__device__ inline void f8v_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared memory: x's codes [kblocks][2][32 lanes] of 16 bytes, its scales [kblocks][8], the warps' sums [2][warps][8][F8V_COL].
__host__ __device__ constexpr size_t f8v_smem(int kblocks, int warps) {
  return (size_t)kblocks * 1056 + (size_t)2 * warps * 8 * F8V_COL * 4;
}

__global__ void __launch_bounds__(F8V_WARPS * 32, 1)
fp8_gemv_kernel(const F8vArgs a) {
  extern __shared__ __align__(16) unsigned char f8v_raw[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint4* s_codes = reinterpret_cast<uint4*>(f8v_raw);
  float* s_sx = reinterpret_cast<float*>(f8v_raw + (size_t)a.kblocks * 1024);
  float* s_part = s_sx + a.kblocks * 8;
  const int per = (a.kblocks + warps - 1) / warps;
  const int rounds = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;

  uint4 v[F8V_AHEAD][4];
  float ws[F8V_AHEAD];
  int ask_tile = blockIdx.x, ask_j = 0;
  auto ask = [&](uint4 (&p)[4], float& s) {
    const int kb = warp + ask_j * warps;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = make_uint4(0, 0, 0, 0);
    if (ask_tile < a.tiles && kb < a.kblocks) {
      const int n = ask_tile * 16 + g, k = kb * fp8::KB + 16 * t;
      const unsigned char* src = a.w + (int64_t)n * a.K + k;
      const bool lo = k < a.K, hi = k + 64 < a.K;
      if (n < a.N && lo) p[0] = ldg_stream(src);
      if (n < a.N && hi) p[1] = ldg_stream(src + 64);
      src += (int64_t)8 * a.K;
      if (n + 8 < a.N && lo) p[2] = ldg_stream(src);
      if (n + 8 < a.N && hi) p[3] = ldg_stream(src + 64);
      s = __ldg(a.sw + (int64_t)(ask_tile >> 3) * a.kblocks + kb);
    }
    if (++ask_j == per) { ask_j = 0; ask_tile += gridDim.x; }
  };
#pragma unroll
  for (int d = 0; d < F8V_AHEAD; ++d) ask(v[d], ws[d]);
  pdl_trigger();
  pdl_wait();

  // ---- x to codes, in the order of the products: eight lanes a row and block of 128, all loads of F8V_ROUND of them at once -----------
  {
    const int j = threadIdx.x & 7, units = a.M * a.kblocks, step = blockDim.x >> 3;
    for (int u0 = threadIdx.x >> 3; u0 - (int)(threadIdx.x >> 3) < units; u0 += F8V_ROUND * step) {
      uint4 p[F8V_ROUND][2];
#pragma unroll
      for (int b = 0; b < F8V_ROUND; ++b) {
        const int u = u0 + b * step, m = u / a.kblocks, k = (u - m * a.kblocks) * fp8::KB + 16 * j;
        p[b][0] = p[b][1] = make_uint4(0, 0, 0, 0);
        if (u < units && k < a.K) {
          const __nv_bfloat16* src = a.x + (int64_t)m * a.ldx + k;
          p[b][0] = load_raw_cg(src);
          p[b][1] = load_raw_cg(src + 8);
        }
      }
#pragma unroll
      for (int b = 0; b < F8V_ROUND; ++b) {
        const int u = u0 + b * step, m = u / a.kblocks, kb = u - m * a.kblocks;
        if (u0 - (int)(threadIdx.x >> 3) + b * step >= units) break;
        float f[16];
        fp8::widen16(p[b][0], p[b][1], f);
        float top = fp8::amax16(f);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // one division a lane: even lanes the multiplier, odd lanes the scale
        top = fmaxf(top, fp8::TINY);
        const float quot = __fdiv_rn((j & 1) ? top : fp8::TOP, (j & 1) ? fp8::TOP : top);
        const uint4 codes = fp8::codes16(f, __shfl_sync(0xffffffffu, quot, lane & 24));
        if (u < units) {
          s_codes[(kb * 2 + (j >> 2)) * 32 + m * 4 + (j & 3)] = codes;
          if (j == 1) s_sx[kb * 8 + m] = quot;
        }
      }
    }
  }
  __syncthreads();

  // ---- the weights -------------------------------------------------------------------------------------------------------
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  int j = 0, tile = blockIdx.x, buf = 0;
  const int pieces = rounds * per;
  for (int i0 = 0; i0 < pieces; i0 += F8V_AHEAD) {
#pragma unroll
    for (int d = 0; d < F8V_AHEAD; ++d) {
      if (i0 + d >= pieces) break;
      const int kb = warp + j * warps;
      if (kb < a.kblocks) {
        const uint4* codes = s_codes + kb * 64 + lane;
        const uint4 x0 = codes[0], x1 = codes[32];
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        f8v_mma(acc, v[d][0].x, v[d][2].x, v[d][0].y, v[d][2].y, x0.x, x0.y);
        f8v_mma(acc, v[d][0].z, v[d][2].z, v[d][0].w, v[d][2].w, x0.z, x0.w);
        f8v_mma(acc, v[d][1].x, v[d][3].x, v[d][1].y, v[d][3].y, x1.x, x1.y);
        f8v_mma(acc, v[d][1].z, v[d][3].z, v[d][1].w, v[d][3].w, x1.z, x1.w);
        const float2 sx = *reinterpret_cast<const float2*>(s_sx + kb * 8 + 2 * t);
        const float f0 = sx.x * ws[d], f1 = sx.y * ws[d];
        sum[0] = fmaf(acc[0], f0, sum[0]);
        sum[1] = fmaf(acc[1], f1, sum[1]);
        sum[2] = fmaf(acc[2], f0, sum[2]);
        sum[3] = fmaf(acc[3], f1, sum[3]);
      }
      ask(v[d], ws[d]);
      if (++j < per) continue;
      // ---- 16 rows of weights done: the warps' sums (two buffers in turn, so that one barrier does) --------------------------
      float* part = s_part + buf * warps * 8 * F8V_COL;
      float* p = part + (warp * 8 + 2 * t) * F8V_COL + g;
      p[0] = sum[0];
      p[F8V_COL] = sum[1];
      p[8] = sum[2];
      p[F8V_COL + 8] = sum[3];
      sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
      __syncthreads();
      const int wide = a.gated ? 8 : 16, n_out = a.gated ? a.N / 2 : a.N;
      for (int o = threadIdx.x; o < a.M * wide; o += blockDim.x) {
        const int m = o / wide, r = o % wide, n = tile * wide + r;
        if (n >= n_out) continue;
        auto total = [&](int row) {
          float s = 0.0f;
#pragma unroll
          for (int u = 0; u < F8V_WARPS; ++u) s += u < warps ? part[(u * 8 + m) * F8V_COL + row] : 0.0f;
          return s;
        };
        float out = total(r);
        if (a.gated) out = __fdividef(out, 1.0f + __expf(-out)) * total(r + 8);
        else if (a.bias) out += __bfloat162float(a.bias[n]);
        const int64_t at = (int64_t)m * n_out + n;
        if (a.y_f32) static_cast<float*>(a.y)[at] = out;
        else static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(out);
      }
      buf ^= 1;
      j = 0;
      tile += gridDim.x;
    }
  }
}

// Warps that share K: of most / 2 to most (or one a block of K, where there are fewer) the number that leaves the fewest idle at the last blocks,
// the larger of equals.
static int f8v_warps(int kblocks, int most) {
  if (kblocks <= most / 2) return kblocks;
  int best = most / 2, cost = ceil_div(kblocks, best) * best;
  for (int w = best + 1; w <= most; ++w)
    if (ceil_div(kblocks, w) * w <= cost) { cost = ceil_div(kblocks, w) * w; best = w; }
  return best;
}
// One block of up to 16 warps an SM, or two of up to 8: a round of 16 takes half as long as one of 8 and 6 / kblocks of that more for the sums'
// barrier (6,144 x 4,096, 2.6 rounds of one block an SM: 7.3 against 8.0 us; 4,096 x 4,096, 1.7: 5.6 against 5.1; 6,912 x 2,304, 2.9: 6.2 against 5.4).
static int f8v_most_warps(int tiles, int kblocks, int sms) {
  return ceil_div(tiles, sms) * (kblocks + 6) < 2 * ceil_div(tiles, 2 * sms) * kblocks ? F8V_WARPS : F8V_WARPS / 2;
}
// Whether this kernel is the faster one: M * kblocks blocks of x to round in every block, up to 128 of them or, where a block has only 16 rows of weights,
// 192 (8 x 2,304 x 2,304 4.1 against 5.3 us, 8 x 6,912 x 2,304 8.1 against 7.2); and K not so long that few pieces of a tile are on their way
// (4,096 x 14,336 14.1 against 13.5 us).
static bool f8v_pays(int M, int tiles, int kblocks, int sms) {
  return M <= 8 && kblocks <= 64 && M * kblocks <= (tiles <= sms ? 192 : 128);
}

}  // namespace exl3

using namespace exl3;

constexpr size_t F8V_SMEM_MAX = f8v_smem(64, F8V_WARPS);

static int f8v_sms() {
  static int sms = 0;
  int dev = 0, n = 0;
  if (!sms && cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) sms = n;
  return sms > 0 ? sms : 1;
}

extern "C" int exl3_fp8_gemv_pays(int M, int N, int K) { return f8v_pays(M, ceil_div(N, 16), ceil_div(K, fp8::KB), f8v_sms()); }

extern "C" int exl3_fp8_gemv(const void* x, int64_t ldx, const void* w, const float* sw, const void* bias, void* y, int out_dtype,
                             int M, int N, int K, int gated, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  if (M < 0 || N < 0 || K < 16 || K % 16 || (out_dtype != DT_F32 && out_dtype != DT_BF16) || (gated && (N % 16 || bias)) || !x || !w || !sw || !y ||
      M > 8 || K > 64 * fp8::KB) {
    set_error("fp8_gemv: needs up to 8 rows, K a multiple of 16 up to 8,192, N of 16 and no bias where gated, a bfloat16 or float32 result and its arrays, "
              "got M=%d N=%d K=%d", M, N, K);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(x) || !aligned16(w) || ldx % 8) { set_error("fp8_gemv: x, its rows and w must be 16-byte aligned"); return ERR_ALIGNMENT; }
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(fp8_gemv_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F8V_SMEM_MAX);
    if (e != cudaSuccess) { set_error("fp8_gemv: cannot get its shared memory: %s", cudaGetErrorString(e)); return (int)e; }
    configured = true;
  }
  const int sms = f8v_sms();
  F8vArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.ldx = ldx; a.w = static_cast<const unsigned char*>(w); a.sw = sw;
  a.bias = static_cast<const __nv_bfloat16*>(bias); a.y = y;
  a.M = M; a.N = N; a.K = K; a.kblocks = ceil_div(K, fp8::KB); a.tiles = ceil_div(N, 16); a.gated = gated; a.y_f32 = out_dtype == DT_F32;
  const int warps = f8v_warps(a.kblocks, f8v_most_warps(a.tiles, a.kblocks, sms));
  const size_t smem = f8v_smem(a.kblocks, warps);
  int per_sm = F8V_WARPS / warps;                          // as its registers and shared memory let blocks run
  while (per_sm > 1 && per_sm * (smem + 1024) > (227 << 10)) --per_sm;
  launch_pdl(fp8_gemv_kernel, dim3(a.tiles < sms * per_sm ? a.tiles : sms * per_sm), dim3(warps * 32), smem, stream, a);
  return launch_status("fp8_gemv");
}
