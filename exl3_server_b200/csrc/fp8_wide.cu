// Products of many rows in 8-bit floating point (fp8.cuh): the activations' rounding, and the product on tcgen05 tensor cores.
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} cx[m, k] cw[n, k]  (+ bias, or silu(gate) * up)
//
// Tiles of 128 x 256 (kind::f8f6f4), persistent blocks, one an SM, 48 KB of codes per 128 of K in a ring of four stages.  The scales differ
// from block to block of K, so every block's 128-long product is an accumulator of its own, and tensor memory has room for two of 128 x 256.
// What bounds such a kernel is therefore the way round: product, signal, tensor memory to registers, signal, next product.  It is kept
// short: eight warps read an accumulator (lane = row, 128 float32 sums a thread, one sw a block of K), 64 columns at a time, the next ones on their way
// while the last are added up (packed fma), and give it back before they have added up its end; waits suspend in hardware; the copies and the
// products are issued by one thread each from end to end.  2,048 x 28,672, K 4,096 with the gate 231 us in a short run (2.1 PFLOP/s) and 275 in a long one, which
// meets the power cap (1.75; what follows is of short runs); what was measured on the
// way: pairs of SMs on one tile 349 (a third less from L2, but the signals cross between SMs), two accumulators of 128 x 128 per block of K
// 288 (the instruction reads x's rows again), without the sums 179, copies alone 125.
//
//   warp 0    TMA producer     warp 1    issues the MMAs; tensor memory     warps 4-11    sums and results
//   (the first four warps leave the others their registers)
//
// Every wait is bounded; when one runs out the kernel records a code, leaves its loops, waits (bounded) for its copies, frees its tensor
// memory and returns.
#include "api.h"
#include "fp8.cuh"

namespace exl3 {

using namespace tc5;

// ---- activations to codes -------------------------------------------------------------------------------------------

// Eight lanes take a block of 128 features of a row, 16 features a lane.  Codes [M, K]; scales [M, blocks], or [blocks, M] (transposed: scratch of the
// product behind, which waits for it).  What a caller gets may be the weights of a product, which reads those ahead of its wait: so the next kernel does
// not start early then.
// Bound by memory and, up to some hundred rows, by its launch (64 x 4,096: 2 us of the product's 12).
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int M, int K, int kblocks, unsigned char* __restrict__ codes,
                    float* __restrict__ sx, int transposed) {
  if (transposed) pdl_trigger();
  pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const int j = threadIdx.x & 7;
  const bool live = item < (int64_t)M * kblocks;
  const int row = live ? (int)(item / kblocks) : 0, b = live ? (int)(item % kblocks) : 0, k = b * fp8::KB + j * 16;
  uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
  if (live && k < K) {
    const uint4* p = reinterpret_cast<const uint4*>(x + (int64_t)row * ldx + k);
    v0 = __ldcg(p);
    v1 = __ldcg(p + 1);
  }
  float v[16];
  fp8::widen16(v0, v1, v);
  float top = fp8::amax16(v);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // one division a lane: even lanes the multiplier, odd lanes the scale
  top = fmaxf(top, fp8::TINY);
  const float quot = __fdiv_rn((j & 1) ? top : fp8::TOP, (j & 1) ? fp8::TOP : top);
  const float mul = __shfl_sync(0xffffffffu, quot, threadIdx.x & 24);
  if (!live) return;
  if (k < K) *reinterpret_cast<uint4*>(codes + (int64_t)row * K + k) = fp8::codes16(v, mul);
  if (j == 1) sx[transposed ? (int64_t)b * M + row : (int64_t)row * kblocks + b] = quot;
}

// ---- the product ------------------------------------------------------------------------------------------------------

constexpr int F8W_BM = 128, F8W_BN = 256, F8W_STAGES = 4, F8W_EPI = 8;
constexpr int F8W_THREADS = 128 + 32 * F8W_EPI;
// Registers a thread after the split: 128 x 40 + 256 x 208 is less than what the block is launched with, 384 x 168.
constexpr int F8W_REGS_LOW = 40, F8W_REGS_HIGH = 208;
static_assert(128 * F8W_REGS_LOW + 256 * F8W_REGS_HIGH <= 384 * 168, "a split that the launch does not cover waits for good");
constexpr uint32_t F8W_A = 128 * 128, F8W_B = 256 * 128;  // bytes of a stage
constexpr uint32_t F8W_SMEM = 1024 + F8W_STAGES * (F8W_A + F8W_B);

static __device__ int g_f8w_error = 0;

struct F8wArgs {
  const float* sx;           // [blocks of K, M]
  const float* sw;           // [ceil(N / 128), blocks of K]
  const __nv_bfloat16* bias;
  void* y;
  int M, N, K, group, gated, y_f32, vec;
};

__global__ void __launch_bounds__(F8W_THREADS, 1)
fp8_wide_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const F8wArgs a) {
  constexpr int STAGES = F8W_STAGES;
  extern __shared__ unsigned char f8w_raw[];
  unsigned char* base = f8w_raw + ((1024u - (smem_u32(f8w_raw) & 1023u)) & 1023u);
  unsigned char* sA = base;
  unsigned char* sB = base + STAGES * F8W_A;
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_map(&map_x);
    prefetch_map(&map_w);
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(acc_full + b, 1); mbar_init(acc_empty + b, F8W_EPI); }
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc<512>(&tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_trigger();
  pdl_wait();
  const int n_m = (a.M + F8W_BM - 1) / F8W_BM, n_n = (a.N + F8W_BN - 1) / F8W_BN, n_tiles = n_m * n_n;
  const int kblocks = (a.K + fp8::KB - 1) / fp8::KB;
  auto place = [&](int tile, int& m, int& n) {              // groups of rows of tiles, within them rows fastest
    const int first = tile / (a.group * n_n) * a.group, rows = min(a.group, n_m - first), r = tile - first * n_n;
    m = first + r % rows;
    n = r / rows;
  };
  bool ok = true;
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F8W_REGS_LOW));
    // One thread each runs these loops from end to end: a warp that parts for its first lane and comes together again at every step loses time
    // each time (318 us instead of 296).
    if (warp == 0 && lane == 0) {
      uint32_t it = 0;
      for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
        int tm, tn;
        place(tile, tm, tn);
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % STAGES;
          ok = fp8::wait(empty + s, ((it / STAGES) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(full + s, F8W_A + F8W_B);
          tma_load_2d(sA + s * F8W_A, &map_x, full + s, kb * fp8::KB, tm * F8W_BM);
          tma_load_2d(sB + s * F8W_B, &map_w, full + s, kb * fp8::KB, tn * F8W_BN);
        }
      }
      if (!ok) {
        atomicExch(&g_f8w_error, 1);
        for (uint32_t back = 1; back <= (uint32_t)STAGES && back <= it; ++back) fp8::wait(full + (it - back) % STAGES, ((it - back) / STAGES) & 1);
      }
    } else if (warp == 1 && lane == 0) {
      uint32_t it = 0;
      for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
        for (int kb = 0; kb < kblocks && ok; ++kb, ++it) {
          const int s = it % STAGES;
          ok = fp8::wait(full + s, (it / STAGES) & 1);
          const uint64_t da = smem_desc_k128(smem_u32(sA + s * F8W_A));
          const uint32_t buf = it & 1;
          ok = ok && fp8::wait(acc_empty + buf, ((it >> 1) & 1) ^ 1);
          if (!ok) break;
          fence_after();
          const uint64_t db = smem_desc_k128(smem_u32(sB + s * F8W_B));
#pragma unroll
          for (int k = 0; k < 4; ++k) fp8::mma_ss(tmem + buf * 256, da + 2 * k, db + 2 * k, fp8::idesc_e4m3(F8W_BM, 256), k > 0);
          mma_commit(acc_full + buf);
          mma_commit(empty + s);
        }
      }
      if (!ok) atomicExch(&g_f8w_error, 2);
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F8W_REGS_HIGH));
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lane_taddr = tmem + ((uint32_t)(q * 32) << 16) + half * 128;
    uint32_t it = 0;
    auto opened = [&](uint32_t i) -> bool {                 // the accumulator of step i is complete
      if (!__all_sync(0xffffffffu, fp8::wait(acc_full + (i & 1), (i >> 1) & 1))) return false;
      fence_after();
      return true;
    };
    for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
      int tm, tn;
      place(tile, tm, tn);
      const int row = tm * F8W_BM + q * 32 + lane, n0 = tn * F8W_BN + half * 128;
      const bool live = row < a.M, inside = n0 < a.N;
      float2 acc[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) acc[c] = make_float2(0.0f, 0.0f);
      const float* sw = a.sw + (int64_t)(inside ? n0 / 128 : 0) * kblocks;
      // the scales of the block at hand and of the two after it, multiplied only when they are used (a product at the load would wait for it)
      const float* sx = a.sx + (live ? row : 0);
      const int last = kblocks - 1;
      float x0 = __ldcg(sx), w0 = __ldg(sw), x1 = __ldcg(sx + (int64_t)min(1, last) * a.M), w1 = __ldg(sw + min(1, last));
      uint32_t d[2][32];
      ok = opened(it);
      if (!ok) break;
      tmem_ld32_issue(lane_taddr + (it & 1) * 256, d[0]);
      tmem_ld32_issue(lane_taddr + (it & 1) * 256 + 32, d[1]);
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const float f = x0 * w0;
        x0 = x1; w0 = w1;
        x1 = __ldcg(sx + (int64_t)min(kb + 2, last) * a.M);
        w1 = __ldg(sw + min(kb + 2, last));
        // 64 columns at a time: a wait is for all loads on their way, so two travel together, and each half's successor is asked for as soon as it
        // has been added up
        auto add = [&](int c, const uint32_t (&r)[32]) {
#pragma unroll
          for (int e = 0; e < 16; ++e) fp8::fma2(acc[c * 16 + e], r[2 * e], r[2 * e + 1], f, f);
        };
        const uint32_t at = lane_taddr + (it & 1) * 256, nx = lane_taddr + ((it + 1) & 1) * 256;
        tmem_ld_wait(d[0]);
        tmem_ld_wait(d[1]);
        add(0, d[0]);
        tmem_ld32_issue(at + 64, d[0]);
        add(1, d[1]);
        tmem_ld32_issue(at + 96, d[1]);
        tmem_ld_wait(d[0]);
        tmem_ld_wait(d[1]);
        fence_before();
        __syncwarp();
        fp8::arrive_first(acc_empty + (it & 1), lane);
        add(2, d[0]);
        const bool more = kb + 1 < kblocks;
        if (more) {
          ok = opened(it + 1);
          if (!ok) break;
          tmem_ld32_issue(nx, d[0]);
        }
        add(3, d[1]);
        if (more) tmem_ld32_issue(nx + 32, d[1]);
      }
      if (!ok) break;
      if (!live || !inside) continue;
      const int n_out = a.gated ? a.N / 2 : a.N;
      if (a.gated) {
        const int64_t at = (int64_t)row * n_out + n0 / 2;
#pragma unroll
        for (int g = 0; g < 8; ++g) {                       // eight gates, then the eight ups of the same features
          if (n0 + 16 * g >= a.N) break;
          float o[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 gate = acc[g * 8 + e], up = acc[g * 8 + 4 + e];
            o[2 * e] = __fdividef(gate.x, 1.0f + __expf(-gate.x)) * up.x;
            o[2 * e + 1] = __fdividef(gate.y, 1.0f + __expf(-gate.y)) * up.y;
          }
          if (a.y_f32) {
            float* y = static_cast<float*>(a.y) + at + 8 * g;
            reinterpret_cast<float4*>(y)[0] = make_float4(o[0], o[1], o[2], o[3]);
            reinterpret_cast<float4*>(y)[1] = make_float4(o[4], o[5], o[6], o[7]);
          } else {
            store_vec(static_cast<__nv_bfloat16*>(a.y) + at + 8 * g, o);
          }
        }
      } else {
        const int64_t at = (int64_t)row * n_out + n0;
#pragma unroll
        for (int g = 0; g < 16; ++g) {
          float o[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) { o[2 * e] = acc[g * 4 + e].x; o[2 * e + 1] = acc[g * 4 + e].y; }
          const int n = n0 + 8 * g;
          if (a.bias) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += n + e < a.N ? __bfloat162float(a.bias[n + e]) : 0.0f;
          }
          if (a.vec && n + 8 <= a.N) {
            if (a.y_f32) {
              float* y = static_cast<float*>(a.y) + at + 8 * g;
              reinterpret_cast<float4*>(y)[0] = make_float4(o[0], o[1], o[2], o[3]);
              reinterpret_cast<float4*>(y)[1] = make_float4(o[4], o[5], o[6], o[7]);
            } else {
              store_vec(static_cast<__nv_bfloat16*>(a.y) + at + 8 * g, o);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e < a.N) {
                if (a.y_f32) static_cast<float*>(a.y)[at + 8 * g + e] = o[e];
                else static_cast<__nv_bfloat16*>(a.y)[at + 8 * g + e] = __float2bfloat16_rn(o[e]);
              }
          }
        }
      }
    }
    if (!ok && lane == 0) atomicExch(&g_f8w_error, 3);
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1) tmem_free<512>(tmem);
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_fp8_wide_status() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_f8w_error, sizeof(int));
  if (v) { int z = 0; cudaMemcpyToSymbol(g_f8w_error, &z, sizeof(int)); }
  return v;
}

extern "C" int exl3_fp8_quantize(const void* x, int64_t ldx, int M, int K, void* codes, float* sx, int transposed, cudaStream_t stream) {
  if (M == 0) return 0;
  if (M < 0 || K < 16 || K % 16 || !x || !codes || !sx) { set_error("fp8_quantize: needs K a multiple of 16 and its arrays, got M=%d K=%d", M, K); return ERR_BAD_ARGUMENT; }
  if (!aligned16(x) || !aligned16(codes) || ldx % 8) { set_error("fp8_quantize: x, its rows and the codes must be 16-byte aligned"); return ERR_ALIGNMENT; }
  const int kblocks = ceil_div(K, fp8::KB);
  const int64_t blocks = ((int64_t)M * kblocks + 31) / 32;
  if (blocks > INT32_MAX) { set_error("fp8_quantize: too many rows"); return ERR_UNSUPPORTED; }
  launch_pdl(fp8_quantize_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, static_cast<const __nv_bfloat16*>(x), ldx, M, K, kblocks,
             static_cast<unsigned char*>(codes), sx, transposed);
  return launch_status("fp8_quantize");
}

// codes and sx as exl3_fp8_quantize leaves them with `transposed`.
extern "C" int exl3_fp8_wide(const void* codes, const float* sx, const void* w, const float* sw, const void* bias, void* y, int out_dtype,
                             int M, int N, int K, int gated, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  if (M < 0 || N < 0 || K < 16 || K % 16 || (out_dtype != DT_F32 && out_dtype != DT_BF16) || (gated && (N % 16 || bias)) || !codes || !sx || !w || !sw || !y) {
    set_error("fp8_wide: needs K a multiple of 16, N of 16 and no bias where gated, a bfloat16 or float32 result and its arrays, got M=%d N=%d K=%d", M, N, K);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(codes) || !aligned16(w) || !aligned16(y)) { set_error("fp8_wide: the codes, w and y must be 16-byte aligned"); return ERR_ALIGNMENT; }
  static int sms = 0;
  if (!sms) {
    cudaError_t e = cudaFuncSetAttribute(fp8_wide_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F8W_SMEM);
    if (e != cudaSuccess) { set_error("fp8_wide: cannot get %u bytes of shared memory: %s", F8W_SMEM, cudaGetErrorString(e)); return (int)e; }
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  }
  CUtensorMap map_x, map_w;
  int rc = fp8::make_map(&map_x, codes, M, K, F8W_BM, "fp8_wide");
  if (rc) return rc;
  rc = fp8::make_map(&map_w, w, N, K, F8W_BN, "fp8_wide");
  if (rc) return rc;
  const int n_m = ceil_div(M, F8W_BM), tiles = n_m * ceil_div(N, F8W_BN);
  F8wArgs a = {};
  a.sx = sx; a.sw = sw; a.bias = static_cast<const __nv_bfloat16*>(bias); a.y = y;
  a.M = M; a.N = N; a.K = K; a.gated = gated; a.y_f32 = out_dtype == DT_F32; a.vec = N % 8 == 0;
  // all rows of tiles together while x's codes stay in L2, else in groups (as gemm_pair.cu has it for bfloat16)
  a.group = (int64_t)M * K <= (40 << 20) ? n_m : n_m < 16 ? n_m : 16;
  launch_pdl(fp8_wide_kernel, dim3(tiles < sms ? tiles : sms), dim3(F8W_THREADS), F8W_SMEM, stream, map_x, map_w, a);
  return launch_status("fp8_wide");
}

// The product of any number of rows.  `few`: 1 the weight-streaming kernel, in which a row's bits do not depend on the rows beside it, 2 that or, where
// it is faster, the one for up to 8 rows, which adds up in another order, 0 the one for many rows; from 17 rows on x is rounded into codes [M, K] and sx [blocks, M] first.
extern "C" int exl3_fp8_linear(const void* x, int64_t ldx, void* codes, float* sx, const void* w, const float* sw, const void* bias, void* y,
                               int out_dtype, int M, int N, int K, int gated, int few, cudaStream_t stream) {
  if (few == 2 && exl3_fp8_gemv_pays(M, N, K)) return exl3_fp8_gemv(x, ldx, w, sw, bias, y, out_dtype, M, N, K, gated, stream);
  if (few && M <= 16) return exl3_fp8_skinny(x, ldx, nullptr, w, sw, bias, y, out_dtype, M, N, K, gated, stream);
  const int rc = exl3_fp8_quantize(x, ldx, M, K, codes, sx, 1, stream);
  if (rc) return rc;
  return few ? exl3_fp8_skinny(codes, K, sx, w, sw, bias, y, out_dtype, M, N, K, gated, stream)
             : exl3_fp8_wide(codes, sx, w, sw, bias, y, out_dtype, M, N, K, gated, stream);
}
