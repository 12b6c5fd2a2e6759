// Prompt attention in bfloat16: the kernels are in attention_prefill_tc.cuh.
#include "attention_prefill_tc.cuh"

extern "C" int exl3_attn_prefill_tc_supported(int dtype, int hd, int page) { return dtype == DT_BF16 && fa_supported(hd, page); }
extern "C" int exl3_attn_prefill_tc_status() { return fa_status(); }

extern "C" int exl3_attn_prefill_tc_opt(const void* q, int64_t q_row_stride, int T, void* out, const void* k_pool,
                                        const void* v_pool, int64_t n_pool_rows, const int* block_table, int bt_stride,
                                        const int* row_start, const int* row_pos0, const int* tile_seq,
                                        const int* tile_q0, int n_tiles, int nh, int nkv, int hd, int page, int window,
                                        int chunk, int sink, float scale, int variant, int keep_first, float softcap,
                                        const float* sink_vals, const float* dist, int dist_len, const float* gate,
                                        cudaStream_t stream) {
  return fa_run(q, q_row_stride, T, out, k_pool, v_pool, n_pool_rows, block_table, bt_stride, row_start, row_pos0, tile_seq, tile_q0,
                n_tiles, nh, nkv, hd, page, window, chunk, sink, scale, variant, keep_first, softcap, sink_vals, dist, dist_len, gate,
                FaCopies{}, stream);
}

extern "C" int exl3_attn_prefill_tc(const void* q, int64_t q_row_stride, int T, void* out, const void* k_pool,
                                    const void* v_pool, int64_t n_pool_rows, const int* block_table, int bt_stride,
                                    const int* row_start, const int* row_pos0, const int* tile_seq,
                                    const int* tile_q0, int n_tiles, int nh, int nkv, int hd, int page, int window,
                                    int chunk, int sink, float scale, int variant, cudaStream_t stream) {
  return exl3_attn_prefill_tc_opt(q, q_row_stride, T, out, k_pool, v_pool, n_pool_rows, block_table, bt_stride, row_start,
                                  row_pos0, tile_seq, tile_q0, n_tiles, nh, nkv, hd, page, window, chunk, sink, scale,
                                  variant, 0, 0.0f, nullptr, nullptr, 0, nullptr, stream);
}
