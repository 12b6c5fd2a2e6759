// Prompts over the 4-bit cache: the rows' pages come out of it in fp16 (cache4.cu), and the prompt attention of
// attention_prefill_tc.cuh, compiled for fp16, runs over them.
//
// Why fp16: it is what tcgen05.mma takes at this rate beside bfloat16, and its 11 bits hold mn + sc * code to 2^-12, where bfloat16's 8
// moved the scores so far that results were 0.005 off (relative to 64 bits; fp16 0.0017, the bfloat16 result's own rounding).  A query row is
// scaled by a power of two into fp16's range, and its factor travels with it; a row's keys of a head are scaled by one of their own, which joins the
// scores' factor, and so are its values, whose factor is taken back from the result.  What is 2^28 below the largest that the row sees loses bits.  The second
// product multiplies hidden values by zero, so a token with a NaN among its values is given as a NaN key and values of zero: who sees it gets NaN (in
// all features), who does not is not touched.
//
// Three kernels a pass: the plan (where a row's copies go, which tiles are whose, the largest keys and values; once), the copies (and, once, the
// queries), the attention.  Copies are made of the pages that a row's queries see and of nothing else, and of no more at a time than the caller gives room for.
//
// Measured: 3,900 new tokens behind 1,200, 32 heads of 128 on 8: 253 us of the GPU in a short run, 270 in a long one (201 GFLOP of causal work, 0.79 and
// 0.74 PFLOP/s): 5 the plan, 30 the copies and the queries, the rest the attention, which is bound as it is for bfloat16, by the softmax's exponentials beside the
// products.  One prompt of 200 tokens 14.9 us, 3 of them the plan.
#define EXL3_PREFILL_F16
#include "attention_prefill_tc.cuh"

extern "C" int exl3_kv4_prompt_status() { return fa_status(); }

static long long kv4_up16(long long n) { return (n + 15) / 16 * 16; }

// Bytes of scratch: copies of `slots` pages, the queries, their factors, the plan (rows, passes, slots of all passes, tiles), the sizes of the rows' keys
// and values by parts, and what undoes their factors.
extern "C" long long exl3_kv4_prompt_scratch(int T, int rows, int row_pages, int total, int slots, int passes, int n_tiles, int nh, int nkv, int hd) {
  return 2 * (long long)slots * nkv * 64 * hd * 2 + kv4_up16((long long)T * nh * hd * 2) + kv4_up16((long long)T * nh * 4) + 16ll * rows +
         16ll * passes + 16ll * total + kv4_up16(4ll * rows) + 16ll * n_tiles + kv4_up16(8ll * rows * nkv) +
         kv4_up16(8ll * rows * nkv * c4_prompt_parts(row_pages));
}

extern "C" int exl3_kv4_prompt(const void* q, int64_t q_stride, int T, void* out, const void* pool, int64_t n_pages, const int* block_table,
                               int bt_stride, int rows, int width, const int* row_start, const int* row_pos0, const int* tile_seq, const int* tile_q0,
                               int n_tiles, int nh, int nkv, int hd, int window, float scale, int few, int row_pages, int total, int slots, int stride,
                               int passes, void* scratch, long long scratch_bytes, cudaStream_t stream) {
  if (T == 0 || n_tiles == 0) return 0;
  if (T < 0 || rows < 1 || width < 1 || nkv < 1 || nh < 1 || nh % nkv || !fa_supported(hd, 64) || n_tiles < 0 || window < 0 || few < 0 || n_pages < 1 ||
      n_pages > INT32_MAX || row_pages < 1 || total < 1 || stride < 1 || passes < 1 || (total - 1) / stride >= passes ||
      slots < (passes == 1 ? total : stride - 1 + row_pages) || !q || !out || !pool || !block_table || !row_start || !row_pos0 || !tile_seq || !tile_q0 ||
      !scratch) {
    set_error("kv4_prompt: needs heads of 64 or 128, passes that hold their rows' pages and all of its arrays, got T=%d rows=%d heads=%d kv_heads=%d "
              "head_dim=%d pages=%d of %d slots=%d stride=%d passes=%d", T, rows, nh, nkv, hd, row_pages, total, slots, stride, passes);
    return ERR_BAD_ARGUMENT;
  }
  if (!aligned16(pool) || !aligned16(q) || q_stride % 8) { set_error("kv4_prompt: q, its rows and the pool must be 16-byte aligned"); return ERR_ALIGNMENT; }
  const long long need = exl3_kv4_prompt_scratch(T, rows, row_pages, total, slots, passes, n_tiles, nh, nkv, hd);
  if (!aligned16(scratch) || scratch_bytes < need) {
    set_error("kv4_prompt: %lld bytes of scratch wanted, 16-byte aligned", need);
    return ERR_SCRATCH;
  }
  if (!isfinite(scale)) { set_error("kv4_prompt: the scale must be finite, got %g", (double)scale); return ERR_BAD_ARGUMENT; }
  unsigned char* at = static_cast<unsigned char*>(scratch);
  auto take = [&](long long bytes) { unsigned char* p = at; at += kv4_up16(bytes); return p; };
  C4Prompt a = {};
  a.pool = static_cast<const unsigned char*>(pool); a.n_pages = (int)n_pages; a.nkv = nkv;
  a.block_table = block_table; a.bt_stride = bt_stride; a.width = width; a.rows = rows;
  a.row_start = row_start; a.row_pos0 = row_pos0; a.window = window; a.few = few; a.parts = c4_prompt_parts(row_pages);
  a.tile_seq = tile_seq; a.tile_q0 = tile_q0; a.n_tiles = n_tiles; a.tile_queries = FA_BQ;
  a.row_pages = row_pages; a.total = total; a.stride = stride; a.passes = passes;
  a.q = static_cast<const __nv_bfloat16*>(q); a.q_stride = q_stride; a.T = T; a.nh = nh;
  a.q_sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;        // (the attention takes positive scales)
  a.k_out = reinterpret_cast<__half*>(take((long long)slots * nkv * 64 * hd * 2));
  a.v_out = reinterpret_cast<__half*>(take((long long)slots * nkv * 64 * hd * 2));
  a.q_out = reinterpret_cast<__half*>(take((long long)T * nh * hd * 2));
  a.q_scale = reinterpret_cast<float*>(take((long long)T * nh * 4));
  a.own = reinterpret_cast<FaRow*>(take(16ll * rows));
  a.pass = reinterpret_cast<PromptPass*>(take(16ll * passes));
  a.slot = reinterpret_cast<int4*>(take(16ll * total));
  a.pass_of = reinterpret_cast<int*>(take(4ll * rows));
  a.tile = reinterpret_cast<PromptTile*>(take(16ll * n_tiles));
  a.undo = reinterpret_cast<float2*>(take(8ll * rows * nkv));
  a.tops = reinterpret_cast<float2*>(at);
  int rc = c4_prompt_plan(a, hd, stream);
  for (int p = 0; p < passes && !rc; ++p) {
    rc = c4_prompt_copies(a, hd, p, slots, stream);
    if (!rc)
      rc = fa_run(a.q_out, (int64_t)nh * hd, T, out, a.k_out, a.v_out, (int64_t)slots * nkv * 64, block_table, bt_stride, row_start, row_pos0, tile_seq,
                  tile_q0, n_tiles, nh, nkv, hd, 64, window, 0, 0, scale != 0.0f ? fabsf(scale) : 1.0f, 0, 0, 0.0f, nullptr, nullptr, 0, nullptr,
                  FaCopies{a.q_scale, a.undo, a.own, a.pass + p, a.tile, passes == 1, (int)n_pages}, stream);
  }
  return rc;
}
