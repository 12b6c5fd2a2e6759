// 8-bit floating point (e4m3) with a scale for each row and 128 features of the activations and for each block of 128 x 128 of the
// weights.  A block of 128 activations with a = max |x| (at least 1e-30) has the scale a / 448 and the codes e4m3(x * (448 / a)), every
// operation in float32 and rounded once.  A block with a value that is not finite has a NaN in it, so its row's results are NaN.
#pragma once

#include "tcgen05.cuh"

namespace exl3 {
namespace fp8 {

constexpr int KB = 128;                                   // features of a block: one 128-byte line of codes
constexpr float TINY = 1e-30f, TOP = 448.0f;

__device__ inline uint32_t pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)hi << 16 | lo;
}
// 16 bfloat16 (two vectors of 16 bytes) as floats.
__device__ inline void widen16(const uint4& a, const uint4& b, float (&v)[16]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// A NaN among the values has to reach the codes, and an infinite value makes one: max() drops NaN, and inf * (448 / inf) is NaN.
__device__ inline float amax16(const float (&v)[16]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
  return m;
}
__device__ inline uint4 codes16(const float (&v)[16], float mul) {
  uint4 r;
  r.x = pack4(__fmul_rn(v[0], mul), __fmul_rn(v[1], mul), __fmul_rn(v[2], mul), __fmul_rn(v[3], mul));
  r.y = pack4(__fmul_rn(v[4], mul), __fmul_rn(v[5], mul), __fmul_rn(v[6], mul), __fmul_rn(v[7], mul));
  r.z = pack4(__fmul_rn(v[8], mul), __fmul_rn(v[9], mul), __fmul_rn(v[10], mul), __fmul_rn(v[11], mul));
  r.w = pack4(__fmul_rn(v[12], mul), __fmul_rn(v[13], mul), __fmul_rn(v[14], mul), __fmul_rn(v[15], mul));
  return r;
}

// kind::f8f6f4 instruction descriptor: D float32, A and B e4m3, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ inline void mma_ss(uint32_t d_tmem, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d_tmem), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
// A bounded wait that suspends the thread for up to a microsecond at a time: polls without a pause hold up what they wait for.
__device__ inline bool wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = tc5::smem_u32(bar);
  for (uint32_t i = 0; i < (1u << 20); ++i) {
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
// One arrival a warp, by its first lane: a predicated instruction, not a branch that the warp has to come together after.
__device__ inline void arrive_first(uint64_t* bar, int lane) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(tc5::smem_u32(bar)), "r"(lane) : "memory");
}
// 16 columns of tensor memory, the registers valid after ld16_wait.
__device__ inline void ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ inline void ld16_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}
// acc += (d0, d1) * (f0, f1)
__device__ inline void fma2(float2& acc, uint32_t d0, uint32_t d1, float f0, float f1) {
  uint64_t c, d, f;
  asm("mov.b64 %0, {%1, %2};" : "=l"(c) : "f"(acc.x), "f"(acc.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(d0), "r"(d1));
  asm("mov.b64 %0, {%1, %2};" : "=l"(f) : "f"(f0), "f"(f1));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(d), "l"(f));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(acc.x), "=f"(acc.y) : "l"(c));
}

// A [rows, K] row-major matrix of codes in boxes of box_rows x 128 bytes, 128B swizzle, zeros outside.  K a multiple of 16.
inline int make_map(CUtensorMap* map, const void* ptr, int64_t rows, int K, int box_rows, const char* who) {
  tc5::EncodeTiledFn fn = tc5::encode_fn();
  if (!fn) { set_error("%s: the driver has no cuTensorMapEncodeTiled", who); return ERR_UNSUPPORTED; }
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)K};
  const cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { set_error("%s: cuTensorMapEncodeTiled failed with %d", who, (int)r); return ERR_BAD_ARGUMENT; }
  return 0;
}

}  // namespace fp8
}  // namespace exl3
