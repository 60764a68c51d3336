// Entry points of paged attention with a sliding window and first tokens that stay visible, and over
// INT4 caches; the kernels are the WIN forms of those in paged_attn.h.
#include "paged_attn.h"

namespace {

// A window of max_seqlen_k keys (0: no window) holds every key of every row, and first tokens past
// max_seqlen_k do not exist.
int clamp_window(int window, int max_seqlen_k) { return window == 0 || window > max_seqlen_k ? max_seqlen_k : window; }
int clamp_sinks(int sinks, int max_seqlen_k) { return sinks < max_seqlen_k ? sinks : max_seqlen_k; }

}  // namespace

extern "C" size_t coopt_window_attention_workspace(int B, int Hq, int Hkv, int D, int max_seqlen_q,
                                                   int max_seqlen_k, int window, int sink_tokens) {
  if ((D != 64 && D != 128) || max_seqlen_q <= 0 || max_seqlen_k <= 0 || sink_tokens < 0 || window < 0) return 0;
  return attn_workspace(B, Hq, Hkv, D, max_seqlen_q,
                        visible_keys(max_seqlen_q, max_seqlen_k, clamp_window(window, max_seqlen_k),
                                     clamp_sinks(sink_tokens, max_seqlen_k)));
}

extern "C" int coopt_window_attention(
    int kv_dtype, const void* q, int64_t q_tok_stride, int64_t q_head_stride, const void* k_cache,
    const void* v_cache, int64_t c_blk_stride, int64_t c_tok_stride, int64_t c_head_stride,
    const void* k_scale, const void* v_scale, int64_t s_blk_stride, int64_t s_tok_stride,
    int64_t s_head_stride, const int32_t* block_table, int64_t bt_stride, const int32_t* cu_seqlens_q,
    const int32_t* seq_lens, int B, int Hq, int Hkv, int D, int block_size, int64_t num_blocks,
    int max_seqlen_q, int max_seqlen_k, int64_t total_q, int window, int sink_tokens,
    float softmax_scale, void* out, int64_t o_tok_stride, int64_t o_head_stride, void* workspace,
    size_t workspace_bytes, coopt_stream_t stream) {
  coopt::clear_error();
  COOPT_REQUIRE(window >= 0 && sink_tokens >= 0, "window and sink_tokens must not be negative");
  COOPT_REQUIRE(window > 0 || sink_tokens == 0, "sink_tokens needs a window");
  COOPT_REQUIRE(softmax_scale >= 0.0f && softmax_scale < 1e30f, "softmax_scale must be finite and not negative");
  // positions, windows and tile ends stay inside 32 bits
  COOPT_REQUIRE(max_seqlen_q < (1 << 29) && max_seqlen_k < (1 << 30), "max_seqlen_q/k out of range");
  return attention_impl<true>("coopt_window_attention", nullptr, clamp_window(window, max_seqlen_k),
                              clamp_sinks(sink_tokens, max_seqlen_k), kv_dtype, q, q_tok_stride,
                              q_head_stride, k_cache, v_cache, c_blk_stride, c_tok_stride, c_head_stride,
                              k_scale, v_scale, s_blk_stride, s_tok_stride, s_head_stride, block_table,
                              bt_stride, cu_seqlens_q, seq_lens, B, Hq, Hkv, D, block_size, num_blocks,
                              max_seqlen_q, max_seqlen_k, total_q, softmax_scale, out, o_tok_stride,
                              o_head_stride, workspace, workspace_bytes, stream);
}
