// Attention over the pages that the rows of a group share, on the 5th-generation tensor cores (bfloat16, heads of 64 or 128, pages of 64 keys): the keys of a page
// are read once for up to PS_TILE queries (token of the group, query head of the key/value head), whatever rows they belong to.
//
//   m = max_j s_j,  l = sum_j 2^(s_j - m),  y = sum_j 2^(s_j - m) V[j]    over the part's pages, s_j = (q . K[j]) * scale * log2 e
//
// A part's (m, l, y) of every query goes to a record in float32; attention_pages.cu joins the records of a query with its own pages' part.
//
// Two sets of 128 queries stand side by side in a block, each with four softmax warps (thread = query = row of tensor memory), and take turns with
// the tensor core: S = Q K^T into one of two buffers of 64 columns, P over the columns of its own S, O += P V.  The maximum that the exponentials are
// taken against moves only when a row's true maximum has grown by more than 2^8, so that O is rescaled rarely.  Blocks are persistent, one an SM,
// and take equal shares of the list of pages (attention_pages.cuh), whatever the groups' sizes.
//
// Every wait is bounded: a kernel that gives up leaves a code (exl3_attn_shared_status), frees its tensor memory and ends.
#include "api.h"
#include "attention_pages.cuh"
#include "tcgen05.cuh"

#include <math.h>

namespace exl3 {

using namespace tc5;

constexpr int PS_STAGES = 4, PS_THREADS = 352;
constexpr float PS_RESCALE_STEP = 8.0f;        // base-2 units
constexpr uint32_t PS_BOX = PG_PAGE * 128;     // bytes of 64 features of a page
static __device__ int g_ps_error = 0;

__host__ __device__ constexpr uint32_t ps_q_bytes(int hd) { return 128 * hd * 2; }
__host__ __device__ constexpr uint32_t ps_page_bytes(int hd) { return PG_PAGE * hd * 2; }
__host__ __device__ constexpr uint32_t ps_smem(int hd) { return 2 * ps_q_bytes(hd) + 2 * PS_STAGES * ps_page_bytes(hd) + 256 + (uint32_t)sizeof(PsPlan) + 1024; }

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
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(db), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
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
  for (uint32_t i = 0; i < WAIT_LIMIT && !there; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(there) : "r"(addr), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, there);
}
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

// warps 0-3, 4-7: softmax of the first and the second 128 queries; warp 8: S; warp 9: O; warp 10: copies of pages.
template <int HD>
__global__ void __launch_bounds__(PS_THREADS, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PsArgs a) {
  constexpr uint32_t QB = ps_q_bytes(HD), KVB = ps_page_bytes(HD);
  constexpr int BOXES = HD / 64;
  extern __shared__ unsigned char ps_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ps_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sQ = base;                    // [2 sets][boxes][128][64]
  unsigned char* sK = sQ + 2 * QB;             // [stages][boxes][64][64]
  unsigned char* sV = sK + PS_STAGES * KVB;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + PS_STAGES * KVB);
  uint64_t* q_full = bars;                     // [2 sets] Q is there
  uint64_t* kv_full = q_full + 2;              // [stages] a page's keys and values are there
  uint64_t* kv_free = kv_full + PS_STAGES;     // [stages] the products that read it are done
  uint64_t* s_full = kv_free + PS_STAGES;      // [2 sets][2] scores
  uint64_t* p_full = s_full + 4;               // [2 sets][2] probabilities, by four warps
  uint64_t* pv_done = p_full + 4;              // [2 sets][2] O += P V
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 4);
  PsPlan& plan = *reinterpret_cast<PsPlan*>(reinterpret_cast<unsigned char*>(bars) + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(q_full + i, 4);
    for (int i = 0; i < PS_STAGES; ++i) { mbar_init(kv_full + i, 1); mbar_init(kv_free + i, 1); }
    for (int i = 0; i < 4; ++i) { mbar_init(s_full + i, 1); mbar_init(p_full + i, 4); mbar_init(pv_done + i, 1); }
    mbar_init_fence();
  }
  if (warp == 8) tmem_alloc<512>(tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  // The kernel that walks the rows' own pages may start when all that it reads beside the records is there: after this.
  pdl_wait();
  pdl_trigger();
  ps_plan(plan, a.groups, a.n_groups, a.row_start, a.rows, a.T, a.G, a.nkv, a.bt_width, gridDim.x);
  if (blockIdx.x == 0)                         // (for the join)
    for (int i = threadIdx.x; i < (int)(sizeof(PsPlan) / 4); i += PS_THREADS) reinterpret_cast<int*>(a.plan)[i] = reinterpret_cast<const int*>(&plan)[i];
  const uint32_t tmem = *tmem_slot;            // columns: scores of set s at 128 s, O at 256 + 128 s
  const int64_t lo = (int)blockIdx.x < plan.blocks ? plan.begin(blockIdx.x) : 0, hi = (int)blockIdx.x < plan.blocks ? plan.begin(blockIdx.x + 1) : 0;
  // Tiles of more than 128 queries: both sets take every page, 128 queries each.  Smaller ones: the sets take the pages in turn, with the same queries.
  auto both = [&](const PsPart& t) { return plan.queries[t.j] - t.tile * PS_TILE > 128; };
  bool ok = true;

  if (warp == 10) {
    // ---- copies; page numbers come 32 at a time -------------------------------------------------------------------------
    int c = 0;
    for (int64_t x = lo; x < hi && ok;) {
      const PsPart t = ps_part(plan, a.nkv, x, hi);
      const int* bt = a.block_table + (int64_t)plan.row[t.j] * a.bt_stride;
      for (int p = t.p0; p < t.p1 && ok; p += 32) {
        int page = p + lane < t.p1 ? __ldcg(bt + p + lane) : 0;
        if (page < 0 || page > a.n_pages) page = a.n_pages;            // beyond the pool: zeros, hidden by the softmax
        for (int i = 0; i < min(32, t.p1 - p); ++i, ++c) {
          const int st = c % PS_STAGES, y = (__shfl_sync(0xffffffffu, page, i) * a.nkv + t.g) * PG_PAGE;
          if (c >= PS_STAGES && !ps_wait(kv_free + st, (c / PS_STAGES - 1) & 1)) { ok = false; break; }
          if (lane == 0) {
            mbar_expect_tx(kv_full + st, 2 * KVB);
#pragma unroll
            for (int b = 0; b < BOXES; ++b) {
              tma_load_2d(sK + st * KVB + b * PS_BOX, &map_k, kv_full + st, 64 * b, y);
              tma_load_2d(sV + st * KVB + b * PS_BOX, &map_v, kv_full + st, 64 * b, y);
            }
          }
          __syncwarp();
        }
      }
      x += t.p1 - t.p0;
    }
    // what was asked for must land before the block's shared memory goes away
    if (!ok && lane == 0) atomicExch(&g_ps_error, 1);
    for (int u = max(0, c - PS_STAGES); u < c; ++u) ps_wait(kv_full + u % PS_STAGES, (u / PS_STAGES) & 1);
  } else if (warp == 8) {
    // ---- S = Q K^T, up to two pages ahead of the softmax -------------------------------------------------------------------
    int c = 0, f[2] = {0, 0}, k[2] = {0, 0};   // pages, pages of a set, parts of a set so far
    for (int64_t x = lo; x < hi && ok;) {
      const PsPart t = ps_part(plan, a.nkv, x, hi);
      const bool two = both(t);
      for (int p = t.p0; p < t.p1 && ok; ++p, ++c) {
        const int st = c % PS_STAGES;
        if (!ps_wait(kv_full + st, (c / PS_STAGES) & 1)) { ok = false; break; }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!two && ((p - t.p0) & 1) != s) continue;
          const int sb = f[s] & 1;
          if (p == t.p0 + (two ? 0 : s) && !ps_wait(q_full + s, k[s] & 1)) { ok = false; break; }
          if (f[s] >= 2 && !ps_wait(pv_done + 2 * s + sb, ((f[s] >> 1) - 1) & 1)) { ok = false; break; }
          fence_after();
          if (lane == 0) {
#pragma unroll
            for (int b = 0; b < BOXES; ++b) {
              const uint64_t da = smem_desc_k128(smem_u32(sQ + s * QB + b * 128 * 128)), db = smem_desc_k128(smem_u32(sK + st * KVB + b * PS_BOX));
#pragma unroll
              for (int i = 0; i < 4; ++i) mma_ss(tmem + 128 * s + 64 * sb, da + 2 * i, db + 2 * i, PS_IDESC_S, (b | i) > 0);
            }
            mma_commit(s_full + 2 * s + sb);
          }
          __syncwarp();
          ++f[s];
        }
      }
      ++k[0];
      k[1] += two || t.p1 - t.p0 > 1;          // (a set without a page asks for no queries)
      x += t.p1 - t.p0;
    }
    if (!ok && lane == 0) atomicExch(&g_ps_error, 2);
  } else if (warp == 9) {
    // ---- O += P V ----------------------------------------------------------------------------------------------------------------
    int c = 0, f[2] = {0, 0};
    for (int64_t x = lo; x < hi && ok;) {
      const PsPart t = ps_part(plan, a.nkv, x, hi);
      const bool two = both(t);
      for (int p = t.p0; p < t.p1 && ok; ++p, ++c) {
        const int st = c % PS_STAGES;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!two && ((p - t.p0) & 1) != s) continue;
          const int sb = f[s] & 1;
          if (!ps_wait(p_full + 2 * s + sb, (f[s] >> 1) & 1)) { ok = false; break; }
          fence_after();
          if (lane == 0) {
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
      }
      x += t.p1 - t.p0;
    }
    if (!ok && lane == 0) atomicExch(&g_ps_error, 3);
  } else {
    // ---- softmax ---------------------------------------------------------------------------------------------------------------
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + 128 * s, to = tmem + lanes + 256 + 128 * s;
    int f = 0;
    for (int64_t x = lo; x < hi && ok;) {
      const PsPart t = ps_part(plan, a.nkv, x, hi);
      x += t.p1 - t.p0;
      const bool two = both(t);
      const int step = two ? 1 : 2, first = t.p0 + (two ? 0 : s), qr = s * 128 + r;
      const int query = t.tile * PS_TILE + (two ? qr : r);
      float* rec = a.records + ps_slot(plan, a.nkv, t.j, t.g, t.tile, blockIdx.x) * ps_record(HD);
      if (first >= t.p1) {                     // no page for this set
        rec[qr] = -INFINITY;
        rec[PS_TILE + qr] = 0.0f;
        continue;
      }
      const bool in = query < plan.queries[t.j];
      const int tok = plan.tok0[t.j] + (in ? query / a.G : 0), head = t.g * a.G + (in ? query % a.G : 0);
      // Q: this thread's row, into the operand's layout (the last S that read the place before is done)
      {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (int64_t)tok * a.q_stride + (int64_t)head * HD);
        uint4 w[HD / 8];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) w[i] = in ? __ldcg(src + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
          *reinterpret_cast<uint4*>(sQ + s * QB + (i >> 3) * 128 * 128 + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = w[i];
        fence_smem_to_tma();
        ps_arrive_warp(q_full + s);
      }
      // the first key that this query does not see, and whether some page of the part is not there
      int row_lo = plan.row[t.j], row_hi = plan.row[t.j] + plan.rows[t.j] - 1;
      while (row_lo < row_hi) { const int mid = (row_lo + row_hi + 1) >> 1; if (__ldcg(a.row_start + mid) <= tok) row_lo = mid; else row_hi = mid - 1; }
      const int pos = min(__ldcg(a.row_pos0 + row_lo), a.bt_width * PG_PAGE) + tok - __ldcg(a.row_start + row_lo);
      const int* bt = a.block_table + (int64_t)plan.row[t.j] * a.bt_stride;
      bool odd = false;
      for (int p = t.p0 + lane; p < t.p1; p += 32) { const int page = __ldcg(bt + p); odd |= page < 0 || page >= a.n_pages; }
      odd = __any_sync(0xffffffffu, odd);
      const int sees = __reduce_min_sync(0xffffffffu, pos);              // all of the warp's queries see keys up to here
      float m_used = -INFINITY, l = 0.0f;
      uint32_t s0[32], s1[32];
      auto ask = [&](int f) {                  // the scores of the set's page f: on their way
        if (!ps_wait(s_full + 2 * s + (f & 1), (f >> 1) & 1)) return false;
        fence_after();
        tmem_ld32_issue(ts + 64 * (f & 1), s0);
        tmem_ld32_issue(ts + 64 * (f & 1) + 32, s1);
        return true;
      };
      ok = ask(f);
      for (int p = first; p < t.p1 && ok; p += step, ++f) {
        const int sb = f & 1;
        tmem_ld_wait(s0);
        tmem_ld_wait(s1);
        const int key0 = p * PG_PAGE;
        if (key0 + PG_PAGE - 1 > sees || odd) {
          int last = pos;
          if (odd) { const int page = __ldcg(bt + p); if (page < 0 || page >= a.n_pages) last = -1; }
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
      ok = ps_wait(pv_done + 2 * s + ((f - 1) & 1), ((f - 1) >> 1) & 1);
      if (!ok) break;
      fence_after();
      if (in) { rec[qr] = m_used; rec[PS_TILE + qr] = l; }
#pragma unroll
      for (int h = 0; h < HD / 32; ++h) {
        __syncwarp();
        tmem_ld32(to + 32 * h, s0);
        if (in) {
#pragma unroll
          for (int c = 0; c < 32; c += 8) ps_store8(rec + 2 * PS_TILE + (int64_t)qr * HD + 32 * h + c, s0 + c);
        }
      }
      __syncwarp();
      fence_before();                          // O is read: the next part's first product may write it
    }
    if (!ok) asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");         // a row of scores may still be on its way
    if (!ok && lane == 0) atomicExch(&g_ps_error, 4);
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 8) tmem_free<512>(tmem);
}

// Joins the parts of a query: a warp for each (token, head).  The parts of the shared pages are in the order of the pages, the own pages' part is the last, so
// a result does not depend on which block was the first to end.
constexpr int PJ_WARPS = 4, PJ_PARTS = 512;               // two for every SM, at most
template <int HD>
__global__ void __launch_bounds__(PJ_WARPS * 32)
attn_shared_join_kernel(const PsPlan* __restrict__ plan, const float* __restrict__ records, const float* __restrict__ own, __nv_bfloat16* __restrict__ out, int T, int nh, int nkv) {
  constexpr int V = HD / 32;                   // features a lane
  __shared__ float s_w[PJ_WARPS][PJ_PARTS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t th = (int64_t)blockIdx.x * PJ_WARPS + warp;
  pdl_trigger();
  pdl_wait();
  if (th >= (int64_t)T * nh) return;
  const int tok = (int)(th / nh), head = (int)(th - (int64_t)tok * nh), G = nh / nkv, g = head / G;
  // the token's group: the last that begins at or before it; lanes side by side, all of a group's numbers at once
  const int n_groups = __ldcg(&plan->n), blocks_per = (int)min(__ldcg(&plan->per), (int64_t)INT32_MAX);
  const int64_t rem = __ldcg(&plan->rem), per = blocks_per;
  int tok0 = -1, queries = 0, pages = 0, tiles_before = 0;
  int64_t work_before = 0;
  for (int j0 = 0; j0 < n_groups; j0 += 32) {
    const int j = min(j0 + lane, n_groups - 1);
    const int t0 = __ldcg(&plan->tok0[j]), q0 = __ldcg(&plan->queries[j]), p0 = __ldcg(&plan->pages[j]), b0 = __ldcg(&plan->tiles_before[j]);
    const int64_t w0 = __ldcg(&plan->work_before[j]);
    const unsigned here = __ballot_sync(0xffffffffu, j0 + lane < n_groups && t0 <= tok && q0 > 0);
    if (here) {
      const int src = 31 - __clz(here);
      tok0 = __shfl_sync(0xffffffffu, t0, src);
      queries = __shfl_sync(0xffffffffu, q0, src);
      pages = __shfl_sync(0xffffffffu, p0, src);
      tiles_before = __shfl_sync(0xffffffffu, b0, src);
      work_before = __shfl_sync(0xffffffffu, w0, src);
    }
  }
  const int query = (tok - tok0) * G + head - g * G;
  if (tok0 < 0 || query >= queries || pages == 0) return;              // in no group: its own pages' part was all
  const int tile = query / PS_TILE, tiles = (queries + PS_TILE - 1) / PS_TILE;
  const int64_t first = work_before * nkv + ((int64_t)g * tiles + tile) * pages, longer = rem * (per + 1);
  auto block_of = [&](int64_t x) { return x < longer ? (int)(x / (per + 1)) : (int)(rem + (x - longer) / per); };
  const int b0 = block_of(first), halves = queries - tile * PS_TILE > 128 ? 1 : 2;
  const int n = (block_of(first + pages - 1) - b0 + 1) * halves;       // parts: at most two for every SM
  const float* rec0 = records + (tiles_before * nkv + g * tiles + tile + b0) * ps_record(HD);
  const int qr = query - tile * PS_TILE;
  auto rec = [&](int i) { return rec0 + (i / halves) * ps_record(HD); };
  auto row = [&](int i) { return qr + (halves == 2 ? (i & 1) * 128 : 0); };
  const float* mine = own + (int64_t)T * nh * HD + 2 * th;
  float mm = -INFINITY;
  for (int i = lane; i <= n; i += 32) mm = fmaxf(mm, i < n ? __ldcg(rec(i) + row(i)) : __ldcg(mine));
  mm = warp_max(mm);
  const float safe = mm == -INFINITY ? 0.0f : mm;
  float l = 0.0f;
  for (int i = lane; i <= n; i += 32) {
    const float f = ps_exp2((i < n ? __ldcg(rec(i) + row(i)) : __ldcg(mine)) - safe);
    s_w[warp][i] = f;
    l = fmaf(f, i < n ? __ldcg(rec(i) + PS_TILE + row(i)) : __ldcg(mine + 1), l);
  }
  l = warp_sum(l);
  __syncwarp();
  float y[V] = {};
  auto add = [&](const float* p, float f) {
    if (f == 0.0f) return;                     // (a part without a key leaves no sums)
    if (V == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
      y[0] = fmaf(f, v.x, y[0]); y[1] = fmaf(f, v.y, y[1]); y[V - 2] = fmaf(f, v.z, y[V - 2]); y[V - 1] = fmaf(f, v.w, y[V - 1]);
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(p));
      y[0] = fmaf(f, v.x, y[0]); y[1] = fmaf(f, v.y, y[1]);
    }
  };
#pragma unroll 8
  for (int i = 0; i < n; ++i) add(rec(i) + 2 * PS_TILE + (int64_t)row(i) * HD + lane * V, s_w[warp][i]);
  add(own + th * HD + lane * V, s_w[warp][n]);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint32_t w[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) w[i] = ps_pack(y[2 * i] * inv, y[2 * i + 1] * inv);
  if (V == 4) *reinterpret_cast<uint2*>(out + th * HD + lane * V) = make_uint2(w[0], w[V / 2 - 1]);
  else *reinterpret_cast<uint32_t*>(out + th * HD + lane * V) = w[0];
}

int attn_shared_join(const PsPlan* plan, const float* records, const float* own, __nv_bfloat16* out, int T, int nh, int nkv, int hd, cudaStream_t stream) {
  const dim3 grid((unsigned)(((int64_t)T * nh + PJ_WARPS - 1) / PJ_WARPS)), block(PJ_WARPS * 32);
  if (hd == 64) launch_pdl(attn_shared_join_kernel<64>, grid, block, 0, stream, plan, records, own, out, T, nh, nkv);
  else launch_pdl(attn_shared_join_kernel<128>, grid, block, 0, stream, plan, records, own, out, T, nh, nkv);
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
