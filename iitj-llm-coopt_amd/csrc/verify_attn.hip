// Entry points of the paged verification attention; the kernels are in paged_attn.h.
#include "paged_attn.h"

extern "C" size_t coopt_verify_attention_workspace(int B, int Hq, int Hkv, int D, int max_seqlen_q,
                                                   int max_seqlen_k) {
  return attn_workspace(B, Hq, Hkv, D, max_seqlen_q, max_seqlen_k);
}

extern "C" int coopt_verify_attention(int kv_dtype, const void* q, int64_t q_tok_stride,
                                      int64_t q_head_stride, const void* k_cache,
                                      const void* v_cache, int64_t c_blk_stride,
                                      int64_t c_tok_stride, int64_t c_head_stride,
                                      const void* k_scale, const void* v_scale,
                                      int64_t s_blk_stride, int64_t s_tok_stride,
                                      int64_t s_head_stride, const int32_t* block_table,
                                      int64_t bt_stride, const int32_t* cu_seqlens_q,
                                      const int32_t* seq_lens, int B, int Hq, int Hkv, int D,
                                      int block_size, int64_t num_blocks, int max_seqlen_q,
                                      int max_seqlen_k, float softmax_scale, void* out,
                                      int64_t o_tok_stride, int64_t o_head_stride,
                                      void* workspace, size_t workspace_bytes,
                                      coopt_stream_t stream) {
  return attention_impl<false>("coopt_verify_attention", nullptr, 0, 0, kv_dtype, q, q_tok_stride,
                               q_head_stride, k_cache, v_cache, c_blk_stride, c_tok_stride,
                               c_head_stride, k_scale, v_scale, s_blk_stride, s_tok_stride,
                               s_head_stride, block_table, bt_stride, cu_seqlens_q, seq_lens, B,
                               Hq, Hkv, D, block_size, num_blocks, max_seqlen_q, max_seqlen_k,
                               0, softmax_scale, out, o_tok_stride, o_head_stride, workspace,
                               workspace_bytes, stream);
}

extern "C" int coopt_verify_attention_rows(int kv_dtype, const void* q, int64_t q_tok_stride,
                                           int64_t q_head_stride, const void* k_cache,
                                           const void* v_cache, int64_t c_blk_stride,
                                           int64_t c_tok_stride, int64_t c_head_stride,
                                           const void* k_scale, const void* v_scale,
                                           int64_t s_blk_stride, int64_t s_tok_stride,
                                           int64_t s_head_stride, const int32_t* block_table,
                                           int64_t bt_stride, const int32_t* cu_seqlens_q,
                                           const int32_t* seq_lens, int B, int Hq, int Hkv, int D,
                                           int block_size, int64_t num_blocks, int max_seqlen_q,
                                           int max_seqlen_k, int64_t total_q, float softmax_scale,
                                           void* out,
                                           int64_t o_tok_stride, int64_t o_head_stride,
                                           void* workspace, size_t workspace_bytes,
                                           coopt_stream_t stream) {
  return attention_impl<false>("coopt_verify_attention", nullptr, 0, 0, kv_dtype, q, q_tok_stride,
                               q_head_stride, k_cache, v_cache, c_blk_stride, c_tok_stride,
                               c_head_stride, k_scale, v_scale, s_blk_stride, s_tok_stride,
                               s_head_stride, block_table, bt_stride, cu_seqlens_q, seq_lens, B,
                               Hq, Hkv, D, block_size, num_blocks, max_seqlen_q, max_seqlen_k,
                               total_q, softmax_scale, out, o_tok_stride, o_head_stride, workspace,
                               workspace_bytes, stream);
}

extern "C" int coopt_verify_attention_window_rows(int kv_dtype, int B, int Hq, int Hkv, int D,
                                                 int max_seqlen_q, int max_seqlen_k, int64_t total_q) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > kMaxRows || max_seqlen_q <= 0 ||
      max_seqlen_k <= 0)
    return 0;
  const AttnShape s = attn_shape(B, Hq / Hkv, Hkv, D, max_seqlen_q, max_seqlen_k, total_q, kv_dtype == COOPT_DT_I8);
  return s.nwin == 0 ? 0 : s.prefill ? kPrefillRows : kMaxRows;
}

extern "C" int coopt_verify_attention_qkv_supported(int kv_dtype, int B, int Hq, int Hkv, int D,
                                                    int max_seqlen_q, int max_seqlen_k) {
  if (kv_dtype != COOPT_DT_BF16 && kv_dtype != COOPT_DT_I8) return 0;
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || max_seqlen_q <= 0 || max_seqlen_k <= 0) return 0;
  if (D != 64 && D != 128) return 0;
  const int G = Hq / Hkv;
  if (static_cast<int64_t>(G) * max_seqlen_q > kMaxRows) return 0;
  if (!fused_ok(D, kv_dtype == COOPT_DT_I8, (G * max_seqlen_q + 15) / 16)) return 0;
  return attn_shape(B, G, Hkv, D, max_seqlen_q, max_seqlen_k, 0, false).max_splits == 1 ? 1 : 0;
}

extern "C" int coopt_verify_attention_qkv(
    int kv_dtype, const void* qkv, int64_t qkv_tok_stride, const float* part, int ks,
    int64_t slice_stride, const int64_t* positions, const void* cos, const void* sin,
    int64_t table_stride, int max_pos, const int64_t* slot_mapping, void* k_cache, void* v_cache,
    int64_t c_blk_stride, int64_t c_tok_stride, int64_t c_head_stride, void* k_scale,
    void* v_scale, int64_t s_blk_stride, int64_t s_tok_stride, int64_t s_head_stride,
    const int32_t* block_table, int64_t bt_stride, const int32_t* cu_seqlens_q,
    const int32_t* seq_lens, int B, int Hq, int Hkv, int D, int block_size, int64_t num_blocks,
    int max_seqlen_q, int max_seqlen_k, float softmax_scale, void* out, int64_t o_tok_stride,
    int64_t o_head_stride, void* workspace, size_t workspace_bytes, coopt_stream_t stream) {
  const FusedQkv fz{qkv, qkv_tok_stride, part, ks, slice_stride, positions, cos, sin,
                    table_stride, max_pos, slot_mapping};
  return attention_impl<false>("coopt_verify_attention_qkv", &fz, 0, 0, kv_dtype, nullptr, 0, 0,
                               k_cache, v_cache, c_blk_stride, c_tok_stride, c_head_stride,
                               k_scale, v_scale, s_blk_stride, s_tok_stride, s_head_stride,
                               block_table, bt_stride, cu_seqlens_q, seq_lens, B, Hq, Hkv, D,
                               block_size, num_blocks, max_seqlen_q, max_seqlen_k, 0, softmax_scale,
                               out, o_tok_stride, o_head_stride, workspace, workspace_bytes,
                               stream);
}
