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
// Measured: 3,900 new tokens behind 1,200, 32 heads of 128 on 8: 258 us (201 GFLOP of causal work, 0.78 PFLOP/s), 27 of them the pages and the
// queries.  The attention is bound as it is for bfloat16: by the softmax's exponentials beside the products.
#define EXL3_PREFILL_F16
#include "attention_prefill_tc.cuh"

extern "C" int exl3_kv4_prompt_status() { return fa_status(); }

static long long kv4_up16(long long n) { return (n + 15) / 16 * 16; }

// Bytes of scratch: the pages' keys and values, the queries, their factors, where each row's pages are, the
// sizes of its keys and values by parts, and what undoes their factors.
extern "C" long long exl3_kv4_prompt_scratch(int T, int rows, int width, int nh, int nkv, int hd) {
  return 2 * (long long)rows * width * nkv * 64 * hd * 2 + kv4_up16((long long)T * nh * hd * 2) + kv4_up16((long long)T * nh * 4) + 16ll * rows +
         8ll * rows * nkv * (exl3_kv4_prompt_parts(width) + 1);
}

extern "C" int exl3_kv4_prompt(const void* q, int64_t q_stride, int T, void* out, const void* pool, int64_t n_pages, const int* block_table,
                               int bt_stride, int rows, int width, const int* row_start, const int* row_pos0, const int* tile_seq, const int* tile_q0,
                               int n_tiles, int nh, int nkv, int hd, int window, float scale, void* scratch, long long scratch_bytes,
                               cudaStream_t stream) {
  if (T == 0 || n_tiles == 0) return 0;
  if (T < 0 || rows < 1 || width < 1 || nkv < 1 || nh < 1 || nh % nkv || !fa_supported(hd, 64) || (int64_t)rows * width > INT32_MAX || !q || !out ||
      !pool || !block_table || !row_start || !row_pos0 || !tile_seq || !tile_q0 || !scratch) {
    set_error("kv4_prompt: needs heads of 64 or 128 and all of its arrays, got T=%d rows=%d heads=%d kv_heads=%d head_dim=%d", T, rows, nh, nkv, hd);
    return ERR_BAD_ARGUMENT;
  }
  const int pages = rows * width;
  if (!aligned16(scratch) || scratch_bytes < exl3_kv4_prompt_scratch(T, rows, width, nh, nkv, hd)) {
    set_error("kv4_prompt: %lld bytes of scratch wanted, 16-byte aligned", exl3_kv4_prompt_scratch(T, rows, width, nh, nkv, hd));
    return ERR_SCRATCH;
  }
  unsigned char* k = static_cast<unsigned char*>(scratch);
  unsigned char* v = k + (long long)pages * nkv * 64 * hd * 2;
  unsigned char* q16 = v + (long long)pages * nkv * 64 * hd * 2;
  float* q_scale = reinterpret_cast<float*>(q16 + kv4_up16((long long)T * nh * hd * 2));
  FaRow* own = reinterpret_cast<FaRow*>(reinterpret_cast<unsigned char*>(q_scale) + kv4_up16((long long)T * nh * 4));
  float2* undo = reinterpret_cast<float2*>(own + rows);
  float2* tops = undo + (int64_t)rows * nkv;
  const int rc = exl3_kv4_unpack16(pool, n_pages, block_table, bt_stride, rows, width, row_start, row_pos0, window, nkv, hd, k, v, own, tops, undo, q, q_stride,
                                   T, nh, q16, q_scale, stream);
  if (rc) return rc;
  return fa_run(q16, (int64_t)nh * hd, T, out, k, v, (int64_t)pages * nkv * 64, block_table, bt_stride, row_start, row_pos0, tile_seq, tile_q0, n_tiles,
                nh, nkv, hd, 64, window, 0, 0, scale, 0, 0, 0.0f, nullptr, nullptr, 0, nullptr, q_scale, undo, own, (int)n_pages, stream);
}
