// Products of few rows with weights in 8-bit floating point (fp8.cuh) on the 5th-generation tensor cores:
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} cx[m, k] cw[n, k]  (+ bias, or silu(gate) * up)
//
// A decode step's product reads every weight once and is bound by that.  The weights are the 128-row operand of tcgen05.mma
// (kind::f8f6f4), one tile of 128 x 128 codes = 16 KB per copy; the batch is the narrow operand (16, 32 or 64 columns).  Up to 16 rows
// x comes in bfloat16 and is rounded to codes by the block itself, straight into the swizzled operand, so that there is no kernel ahead of this
// one; a block does that for its own range of K, once for 128 features.  For more rows that is too much to do over again in every block
// (64 rows x 6,144, K 4,096: 26 us), and x's codes come by TMA from the kernel ahead.
//
// Measured: 8 rows x 32,768, K 4,096 with the gate 27.4 us (134 MB, 4.9 TB/s), 64 rows x 6,144, K 4,096 12.1 us with the rounding ahead (25 MB), one
// row x 2,304, K 5,760 6.3 us (13 MB; two blocks an SM, cuts of K by the clusters that run at once and four accumulators in turn: 9.2 before).
// The large one is bound by memory, the small ones by setting up (tensor memory, barriers, cluster), about 3 us, and the end of the cluster's sums.
//
// The scales differ from block to block of K, so each block's 128-long product is an accumulator of its own (four in turn in tensor memory), and
// four warps add it to float32 registers times sx * sw while the next one is formed.
//
//   warp 0     TMA producer of weight tiles          warp 1      issues the MMAs; allocates and frees tensor memory
//   warps 2-5  take accumulators, thread = feature    the rest    x to codes, eight lanes a row of 128 (or its scales)
//
// K is cut over the S blocks of a cluster; their sums meet through distributed shared memory, block r adding up columns r, r + S, ... in the
// blocks' order.  Every wait is bounded; when one runs out the kernel records a code, waits (bounded) for its copies, meets the cluster
// barriers, frees its tensor memory and returns.
#include "api.h"
#include "fp8.cuh"

namespace exl3 {

using namespace tc5;

// Warps behind the first six: 16 columns, four that round x, four rows each; 32 and 64, one that brings the scales.
__host__ __device__ constexpr int f8s_xwarps(int nb) { return nb == 16 ? 4 : 1; }
__host__ __device__ constexpr int f8s_threads(int nb) { return 192 + 32 * f8s_xwarps(nb); }
constexpr int F8S_MAX_SPLIT = 8;
constexpr int F8S_SLOTS = 16;                             // scales of the last blocks of K: more than the stages and the accumulators

__host__ __device__ constexpr int f8s_stages(int nb) { return nb <= 32 ? 5 : 4; }      // two blocks an SM
__host__ __device__ constexpr uint32_t f8s_smem(int nb) { return 1024 + f8s_stages(nb) * (16384 + nb * 128); }

static __device__ int g_f8s_error = 0;

struct F8sArgs {
  const __nv_bfloat16* x;    // 16 columns
  int64_t ldx;
  const float* sx;           // 32 and 64 columns: [blocks of K, M], beside x's codes in map_x
  const float* sw;           // [ceil(N / 128), blocks of K]
  const __nv_bfloat16* bias;
  void* y;
  int M, N, K, S, gated, y_f32;
};

__device__ inline float f8s_ld_peer(const float* mine, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(mine, rank)) : "memory");
  return v;
}

template <int NB>
__global__ void __launch_bounds__(f8s_threads(NB), 2)
fp8_skinny_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8sArgs a) {
  constexpr int STAGES = f8s_stages(NB), XW = f8s_xwarps(NB), THREADS = f8s_threads(NB);
  constexpr int ACCS = 4;                                   // accumulators in turn: the way round one is longer than a tile takes to come
  constexpr bool ROUNDS_X = NB == 16;                       // x comes in bfloat16 and is rounded here
  constexpr uint32_t W_BYTES = 16384, X_BYTES = NB * 128;
  static_assert(STAGES * W_BYTES >= NB * 128 * 4, "the sums take the place of the weight tiles");
  static_assert(STAGES + ACCS + 1 <= F8S_SLOTS, "scales of the rounding warps live until their accumulator has been added up: they follow the tiles' ring");
  extern __shared__ unsigned char f8s_raw[];
  unsigned char* base = f8s_raw + ((1024u - (smem_u32(f8s_raw) & 1023u)) & 1023u);
  unsigned char* sW = base;
  unsigned char* sX = base + STAGES * W_BYTES;
  __shared__ uint64_t wfull[STAGES], xfull[STAGES], empty[STAGES], acc_full[ACCS], acc_empty[ACCS], sfull[F8S_SLOTS], sempty[F8S_SLOTS];
  __shared__ __align__(16) float s_sx[F8S_SLOTS][NB];
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.S > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / a.S, n0 = tile * 128, m0 = blockIdx.y * NB;
  const int kblocks = (a.K + fp8::KB - 1) / fp8::KB;
  const int kb0 = (int)((int64_t)kblocks * rank / a.S), kb1 = (int)((int64_t)kblocks * (rank + 1) / a.S), n_kb = kb1 - kb0;
  constexpr int TM_COLS = ACCS * NB;
  if (threadIdx.x == 0) {
    prefetch_map(&map_w);
    if (!ROUNDS_X) prefetch_map(&map_x);
    for (int s = 0; s < STAGES; ++s) { mbar_init(wfull + s, 1); mbar_init(xfull + s, XW); mbar_init(empty + s, 1); }
    for (int b = 0; b < ACCS; ++b) { mbar_init(acc_full + b, 1); mbar_init(acc_empty + b, 4); }
    for (int s = 0; s < F8S_SLOTS; ++s) { mbar_init(sfull + s, XW); mbar_init(sempty + s, 4); }
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc<TM_COLS>(&tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_trigger();
  bool ok = true;

  if (warp == 0) {
    // ---- weights: no kernel writes them, so the first tiles are asked for before the kernel ahead has ended; x's codes are its work --------
    // (one thread from end to end, as in fp8_wide.cu)
    if (lane == 0) {
      const int early = n_kb < STAGES ? n_kb : STAGES;
      for (int i = 0; i < early; ++i) {
        mbar_expect_tx(wfull + i, W_BYTES + (ROUNDS_X ? 0 : X_BYTES));
        tma_load_2d(sW + i * W_BYTES, &map_w, wfull + i, (kb0 + i) * fp8::KB, n0);
      }
      if (!ROUNDS_X) {
        pdl_wait();
        for (int i = 0; i < early; ++i) tma_load_2d(sX + i * X_BYTES, &map_x, wfull + i, (kb0 + i) * fp8::KB, m0);
      }
      uint32_t asked = early;
      for (int i = early; i < n_kb && ok; ++i) {
        const int s = i % STAGES;
        ok = fp8::wait(empty + s, ((i / STAGES) & 1) ^ 1);
        if (!ok) break;
        mbar_expect_tx(wfull + s, W_BYTES + (ROUNDS_X ? 0 : X_BYTES));
        tma_load_2d(sW + s * W_BYTES, &map_w, wfull + s, (kb0 + i) * fp8::KB, n0);
        if (!ROUNDS_X) tma_load_2d(sX + s * X_BYTES, &map_x, wfull + s, (kb0 + i) * fp8::KB, m0);
        ++asked;
      }
      if (!ok) {
        atomicExch(&g_f8s_error, 1);
        for (uint32_t back = 1; back <= (uint32_t)STAGES && back <= asked; ++back) fp8::wait(wfull + (asked - back) % STAGES, ((asked - back) / STAGES) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      pdl_wait();                                           // (not on a barrier, whose wait is bounded)
      for (int i = 0; i < n_kb && ok; ++i) {
        const int s = i % STAGES, buf = i % ACCS;
        ok = fp8::wait(acc_empty + buf, ((i / ACCS) & 1) ^ 1) && fp8::wait(wfull + s, (i / STAGES) & 1) &&
             (!ROUNDS_X || fp8::wait(xfull + s, (i / STAGES) & 1));
        if (!ok) break;
        fence_after();
        const uint64_t da = smem_desc_k128(smem_u32(sW + s * W_BYTES)), db = smem_desc_k128(smem_u32(sX + s * X_BYTES));
#pragma unroll
        for (int k = 0; k < 4; ++k) fp8::mma_ss(tmem + buf * NB, da + 2 * k, db + 2 * k, fp8::idesc_e4m3(128, NB), k > 0);
        mma_commit(acc_full + buf);
        mma_commit(empty + s);
      }
      if (!ok) atomicExch(&g_f8s_error, 2);
    }
    __syncwarp();
  } else if (warp < 6) {
    // ---- accumulators: lane = feature of this warp's 32, registers over the columns ----------------------------------
    pdl_wait();
    const int q = warp & 3;
    float2 acc[NB / 2];
#pragma unroll
    for (int c = 0; c < NB / 2; ++c) acc[c] = make_float2(0.0f, 0.0f);
    const float* sw = a.sw + (int64_t)tile * kblocks + kb0;
    const uint32_t at = tmem + ((uint32_t)(q * 32) << 16);
    uint32_t d[2][16];
    float w0 = 0.0f, w1 = 0.0f;
    if (ROUNDS_X && n_kb > 0) { w0 = __ldg(sw); w1 = __ldg(sw + min(1, n_kb - 1)); }
    auto open = [&](int i, uint32_t (&r)[16]) -> bool {    // the first 16 columns of step i's accumulator
      if (!__all_sync(0xffffffffu, fp8::wait(acc_full + i % ACCS, (i / ACCS) & 1))) return false;
      fence_after();
      fp8::ld16_issue(at + i % ACCS * NB, r);
      return true;
    };
    constexpr int P = NB / 16;
    auto step = [&](int i, int first) -> bool {            // d[first] is on its way; leaves the next step's in d[first ^ (P & 1)]
      const int slot = i % F8S_SLOTS;
      float w = 1.0f;                                       // (else the scales come with it)
      if (ROUNDS_X) {                                       // asked for two steps ahead
        w = w0;
        w0 = w1;
        w1 = __ldg(sw + min(i + 2, n_kb - 1));
      }
      if (!__all_sync(0xffffffffu, fp8::wait(sfull + slot, (i / F8S_SLOTS) & 1))) return false;
      bool good = true;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        uint32_t (&now)[16] = d[(first + p) & 1];
        uint32_t (&next)[16] = d[(first + p + 1) & 1];
        fp8::ld16_wait(now);
        if (p + 1 < P) {
          fp8::ld16_issue(at + i % ACCS * NB + (p + 1) * 16, next);
        } else {                                           // the accumulator is free, its last part in registers
          fence_before();
          __syncwarp();
          fp8::arrive_first(acc_empty + i % ACCS, lane);
          if (i + 1 < n_kb) good = open(i + 1, next);
        }
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
          float4 sx = *reinterpret_cast<const float4*>(&s_sx[slot][p * 16 + c]);
          if (ROUNDS_X) { sx.x *= w; sx.y *= w; sx.z *= w; sx.w *= w; }
          fp8::fma2(acc[(p * 16 + c) / 2], now[c], now[c + 1], sx.x, sx.y);
          fp8::fma2(acc[(p * 16 + c) / 2 + 1], now[c + 2], now[c + 3], sx.z, sx.w);
        }
      }
      if (!ROUNDS_X) {
        __syncwarp();
        fp8::arrive_first(sempty + slot, lane);
      }
      return good;
    };
    if (n_kb > 0) ok = open(0, d[0]);
    for (int i = 0; i < n_kb && ok; i += 2) {
      ok = step(i, 0);
      if (ok && i + 1 < n_kb) ok = step(i + 1, P & 1);
    }
    if (!ok && lane == 0) atomicExch(&g_f8s_error, 3);
    // (after a failed wait copies may still be landing in the tiles' place: the sums are not to be trusted, nor written there)
    if (ok) {
      float* part = reinterpret_cast<float*>(sW);
#pragma unroll
      for (int c = 0; c < NB; ++c) part[c * 128 + q * 32 + lane] = c & 1 ? acc[c / 2].y : acc[c / 2].x;
    }
  } else if constexpr (!ROUNDS_X) {
    // ---- scales of x, a block of K after the other ----------------------------------------------------------------------
    pdl_wait();
    constexpr int PER = NB / 32;
    constexpr int AHEAD = 4;                                // steps; multiplied only when they are put down (a product at the load would wait for it)
    float x[AHEAD][PER], w[AHEAD];
    auto fetch = [&](int i, float (&v)[PER], float& ws) {
      if (i >= n_kb) return;
      ws = __ldg(a.sw + (int64_t)tile * kblocks + kb0 + i);
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int row = m0 + u * 32 + lane;
        v[u] = row < a.M ? __ldcg(a.sx + (int64_t)(kb0 + i) * a.M + row) : 0.0f;
      }
    };
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) fetch(d, x[d], w[d]);
    for (int i0 = 0; i0 < n_kb && ok; i0 += AHEAD) {
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        const int i = i0 + d;
        if (i >= n_kb) break;
        // the slots are a ring of their own: the tiles' barriers may be two phases on when this warp looks, since the MMAs do not wait for it
        const int slot = i % F8S_SLOTS;
        ok = __all_sync(0xffffffffu, fp8::wait(sempty + slot, ((i / F8S_SLOTS) & 1) ^ 1));
        if (!ok) break;
#pragma unroll
        for (int u = 0; u < PER; ++u) s_sx[slot][u * 32 + lane] = x[d][u] * w[d];
        __syncwarp();
        fp8::arrive_first(sfull + slot, lane);
        fetch(i + AHEAD, x[d], w[d]);
      }
    }
    if (!ok && lane == 0) atomicExch(&g_f8s_error, 5);
  } else {
    // ---- x to codes: four rows a warp at a time, eight lanes a row, 16 features a lane --------------------------------
    pdl_wait();
    const int j = lane & 7, r = (warp - 6) * 4 + (lane >> 3);
    auto fetch = [&](int i, uint4 (&v)[2]) {
      const int row = m0 + r, k = (kb0 + i) * fp8::KB + j * 16;
      v[0] = v[1] = make_uint4(0, 0, 0, 0);
      if (i < n_kb && row < a.M && k < a.K) {
        const uint4* p = reinterpret_cast<const uint4*>(a.x + (int64_t)row * a.ldx + k);
        v[0] = __ldcg(p);
        v[1] = __ldcg(p + 1);
      }
    };
    // two blocks of K ahead of the one that is rounded
    uint4 v[3][2];
    fetch(0, v[0]);
    fetch(1, v[1]);
    auto round = [&](int i, uint4 (&cur)[2], uint4 (&far)[2]) -> bool {
      const int s = i % STAGES, slot = i % F8S_SLOTS;
      fetch(i + 2, far);
      float f[16];
      fp8::widen16(cur[0], cur[1], f);
      float top = fp8::amax16(f);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // one division a lane: even lanes the multiplier, odd lanes the scale
      top = fmaxf(top, fp8::TINY);
      const float quot = __fdiv_rn((j & 1) ? top : fp8::TOP, (j & 1) ? fp8::TOP : top);
      const uint4 codes = fp8::codes16(f, __shfl_sync(0xffffffffu, quot, lane & 24));
      if (!__all_sync(0xffffffffu, fp8::wait(empty + s, ((i / STAGES) & 1) ^ 1))) return false;
      *reinterpret_cast<uint4*>(sX + s * X_BYTES + r * 128 + ((j ^ (r & 7)) << 4)) = codes;
      if (j == 1) s_sx[slot][r] = quot;
      fence_smem_to_tma();                                 // the codes are read through the async proxy
      __syncwarp();
      fp8::arrive_first(xfull + s, lane);
      fp8::arrive_first(sfull + slot, lane);
      return true;
    };
    for (int i = 0; i < n_kb && ok; i += 3) {
      ok = round(i, v[0], v[2]);
      if (ok && i + 1 < n_kb) ok = round(i + 1, v[1], v[0]);
      if (ok && i + 2 < n_kb) ok = round(i + 2, v[2], v[1]);
    }
    if (!ok && lane == 0) atomicExch(&g_f8s_error, 4);
  }

  // ---- the cluster's sums ---------------------------------------------------------------------------------------------
  pdl_wait();                                              // (y may be what an earlier kernel still reads)
  if (a.S > 1) cluster_sync_all(); else __syncthreads();
  {
    const float* part = reinterpret_cast<const float*>(sW);
    const int per = a.gated ? 64 : 128, n_out = a.gated ? a.N / 2 : a.N, o0 = a.gated ? n0 / 2 : n0;
    const int rows = min(NB, a.M - m0), mine = rows > rank ? (rows - rank + a.S - 1) / a.S : 0;
    for (int i = threadIdx.x; i < mine * per; i += THREADS) {
      const int c = rank + i / per * a.S, f = i % per;
      auto total = [&](int feature) {
        if (a.S == 1) return part[c * 128 + feature];
        float v[F8S_MAX_SPLIT];
#pragma unroll
        for (int b = 0; b < F8S_MAX_SPLIT; ++b) v[b] = b < a.S ? f8s_ld_peer(part + c * 128 + feature, b) : 0.0f;
        float sum = v[0];
#pragma unroll
        for (int b = 1; b < F8S_MAX_SPLIT; ++b) if (b < a.S) sum += v[b];
        return sum;
      };
      float out;
      if (o0 + f >= n_out) continue;
      if (a.gated) {
        const float gate = total(f / 8 * 16 + f % 8), up = total(f / 8 * 16 + 8 + f % 8);
        out = __fdividef(gate, 1.0f + __expf(-gate)) * up;
      } else {
        out = total(f) + (a.bias ? __bfloat162float(a.bias[n0 + f]) : 0.0f);
      }
      const int64_t at = (int64_t)(m0 + c) * n_out + o0 + f;
      if (a.y_f32) static_cast<float*>(a.y)[at] = out;
      else static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(out);
    }
  }
  fence_before();
  if (a.S > 1) cluster_sync_all(); else __syncthreads();   // nobody reads a block's shared memory after it has gone
  fence_after();
  if (warp == 1) tmem_free<TM_COLS>(tmem);
}

// Never launched: a block of this kernel's shape for the driver's count of clusters, which for a kernel that allocates tensor memory says one block
// an SM, while two run (as gemm_skinny.cu found by timing).
__global__ void __launch_bounds__(f8s_threads(16)) f8s_block_shape_kernel() {}

// Clusters of s blocks that run at once, two blocks an SM.
static int f8s_max_clusters(int s) {
  static int count[F8S_MAX_SPLIT + 1] = {};
  if (count[s]) return count[s];
  const int smem = (int)f8s_smem(32) + 5 * 1024;
  int n = 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(1024 * s);
  cfg.blockDim = dim3(f8s_threads(16));
  cfg.dynamicSmemBytes = smem;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = s;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(f8s_block_shape_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, f8s_block_shape_kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = 1;
  }
  count[s] = n;
  return n;
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_fp8_skinny_status() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_f8s_error, sizeof(int));
  if (v) { int z = 0; cudaMemcpyToSymbol(g_f8s_error, &z, sizeof(int)); }
  return v;
}

// x: bfloat16 [M, K] up to 16 rows; else its codes [M, K] with sx [blocks, M] as exl3_fp8_quantize leaves them with `transposed` (ldx is not used).
extern "C" int exl3_fp8_skinny(const void* x, int64_t ldx, const float* sx, const void* w, const float* sw, const void* bias, void* y, int out_dtype,
                               int M, int N, int K, int gated, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  if (M < 0 || N < 0 || K < 16 || K % 16 || (out_dtype != DT_F32 && out_dtype != DT_BF16) || (gated && (N % 16 || bias)) || !x || !w || !sw || !y ||
      (M > 16 && !sx)) {
    set_error("fp8_skinny: needs K a multiple of 16, N of 16 and no bias where gated, a bfloat16 or float32 result and its arrays, got M=%d N=%d K=%d", M, N, K);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(x) || !aligned16(w) || (M <= 16 && ldx % 8)) { set_error("fp8_skinny: x, its rows and w must be 16-byte aligned"); return ERR_ALIGNMENT; }
  const int nb = M <= 16 ? 16 : M <= 32 ? 32 : 64, groups = ceil_div(M, nb), tiles = ceil_div(N, 128), kblocks = ceil_div(K, 128);
  if (groups > 65535) { set_error("fp8_skinny: %d rows are too many", M); return ERR_UNSUPPORTED; }
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(fp8_skinny_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)f8s_smem(16));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fp8_skinny_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)f8s_smem(32));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fp8_skinny_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)f8s_smem(64));
    if (e != cudaSuccess) { set_error("fp8_skinny: cannot get its shared memory: %s", cudaGetErrorString(e)); return (int)e; }
    configured = true;
  }
  // As many cuts of K as still let all clusters run at once, with two blocks of K a block at least.  From N and K only, so that a row's result
  // does not depend on the rows beside it.
  int S = F8S_MAX_SPLIT;
  while (S > 1 && (kblocks / S < 2 || tiles > f8s_max_clusters(S))) --S;
  CUtensorMap map_w, map_x;
  int rc = fp8::make_map(&map_w, w, N, K, 128, "fp8_skinny");
  if (rc) return rc;
  map_x = map_w;
  if (nb > 16) {
    rc = fp8::make_map(&map_x, x, M, K, nb, "fp8_skinny");
    if (rc) return rc;
  }
  F8sArgs a = {};
  a.x = static_cast<const __nv_bfloat16*>(x); a.ldx = ldx; a.sx = sx; a.sw = sw; a.bias = static_cast<const __nv_bfloat16*>(bias); a.y = y;
  a.M = M; a.N = N; a.K = K; a.S = S; a.gated = gated; a.y_f32 = out_dtype == DT_F32;
  auto go = [&](auto kernel) {
    launch_pdl_clusters(kernel, dim3(tiles * S, groups), dim3(f8s_threads(nb)), S, f8s_smem(nb), stream, map_w, map_x, a);
  };
  if (nb == 16) go(fp8_skinny_kernel<16>); else if (nb == 32) go(fp8_skinny_kernel<32>); else go(fp8_skinny_kernel<64>);
  return launch_status("fp8_skinny");
}
