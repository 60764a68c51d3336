// Paged GQA attention with a sliding window and first tokens that stay visible, over bf16, INT8
// and INT4 caches.  Query row j of a sequence of n rows and L keys stands at p = L - n + j and sees
//   key k  iff  k <= p  and  (k > p - window  or  k < sinks)
// and out = sum_k softmax_k(scale * q . K[k]) V[k] over those keys; a row that sees none is 0.
#include <math.h>

#include "common.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const void* kc;
  const void* vc;
  int64_t c_bs, c_ts, c_hs;
  const uint16_t* ks;
  const uint16_t* vs;
  int64_t s_bs, s_ts, s_hs;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* cu;
  const int32_t* seq_lens;
  int Hq, Hkv, bs_shift, max_seqlen_k;
  int64_t num_blocks;
  int window, sinks;
  float scale_log2;
  uint16_t* out;
  int64_t o_ts, o_hs;
};

// One wave per (query row, query head), lane l the elements l * E .. l * E + E of a vector: a plain
// walk over the visible keys.
template <int D, int KV>
__global__ __launch_bounds__(64) void row_kernel(Args a) {
  constexpr int E = D / 64;
  const int b = blockIdx.z, h = blockIdx.y, j = blockIdx.x, lane = threadIdx.x;
  const int q0 = a.cu[b], n = a.cu[b + 1] - q0;
  if (j >= n) return;
  const int L = min(a.seq_lens[b], a.max_seqlen_k), p = L - n + j;
  const int hkv = h / (a.Hq / a.Hkv);
  const int32_t* table = a.bt + b * a.bt_stride;
  float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = bf16_to_f32(a.q[(q0 + j) * a.q_ts + h * a.q_hs + lane * E + e]);
    o[e] = 0.0f;
  }
  auto value = [&](const void* cache, const uint16_t* scales, int64_t blk, int off, int e) {
    const int64_t at = blk * a.c_bs + off * a.c_ts + hkv * a.c_hs;
    const int d = lane * E + e;
    if constexpr (KV == kBf16) return bf16_to_f32(static_cast<const uint16_t*>(cache)[at + d]);
    const float s = f16_to_f32(scales[blk * a.s_bs + off * a.s_ts + hkv * a.s_hs]);
    if constexpr (KV == kI8) return bf16_to_f32(f32_to_bf16(static_cast<const int8_t*>(cache)[at + d] * s));
    const int byte = static_cast<const uint8_t*>(cache)[at + d / 2];
    return static_cast<float>((d & 1 ? byte >> 4 : byte & 15) - 8) * s;
  };
  const int low = max(0, p - a.window + 1);
  for (int k = 0; k <= p; ++k) {
    if (k >= a.sinks && k < low) k = low;
    int64_t blk = table[k >> a.bs_shift];
    blk = blk < 0 ? 0 : (blk >= a.num_blocks ? a.num_blocks - 1 : blk);
    const int off = k & ((1 << a.bs_shift) - 1);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], value(a.kc, a.ks, blk, off, e), s);
    s = wave_sum_f32(s) * a.scale_log2;
    const float m_new = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.0f : exp2f(m - m_new), w = exp2f(s - m_new);
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * value(a.vc, a.vs, blk, off, e);
    m = m_new;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.out[(q0 + j) * a.o_ts + h * a.o_hs + lane * E + e] = f32_to_bf16(p >= 0 ? o[e] / l : 0.0f);
}

template <int D>
void launch(int kv_dtype, const Args& a, dim3 grid, hipStream_t s) {
  if (kv_dtype == COOPT_DT_BF16) hipLaunchKernelGGL((row_kernel<D, kBf16>), grid, dim3(64), 0, s, a);
  else if (kv_dtype == COOPT_DT_I8) hipLaunchKernelGGL((row_kernel<D, kI8>), grid, dim3(64), 0, s, a);
  else hipLaunchKernelGGL((row_kernel<D, kI4>), grid, dim3(64), 0, s, a);
}

}  // namespace

extern "C" size_t coopt_window_attention_workspace(int B, int Hq, int Hkv, int D, int max_seqlen_q,
                                                   int max_seqlen_k, int window, int sink_tokens) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 64 || (D != 64 && D != 128) || max_seqlen_q <= 0 ||
      max_seqlen_k <= 0 || sink_tokens < 0 || window < 0)
    return 0;
  return 256;
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
  COOPT_REQUIRE(kv_dtype == COOPT_DT_BF16 || kv_dtype == COOPT_DT_I8 || kv_dtype == COOPT_DT_I4,
                "kv_dtype must be COOPT_DT_BF16, COOPT_DT_I8 or COOPT_DT_I4");
  COOPT_REQUIRE(B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "Hq must be a multiple of Hkv");
  COOPT_REQUIRE(D == 64 || D == 128, "head_dim must be 64 or 128");
  COOPT_REQUIRE(block_size >= 16 && (block_size & (block_size - 1)) == 0, "block_size must be a power of two >= 16");
  COOPT_REQUIRE(max_seqlen_q > 0 && max_seqlen_k > 0, "max_seqlen_q/k must be positive");
  COOPT_REQUIRE(window >= 0 && sink_tokens >= 0, "window and sink_tokens must not be negative");
  COOPT_REQUIRE(window > 0 || sink_tokens == 0, "sink_tokens needs a window");
  const int G = Hq / Hkv;
  COOPT_REQUIRE(G <= 64, "Hq/Hkv must be <= 64");
  COOPT_REQUIRE(bt_stride >= (static_cast<int64_t>(max_seqlen_k) + block_size - 1) / block_size,
                "block_table narrower than ceil(max_seqlen_k / block_size)");
  COOPT_REQUIRE(B <= 65535, "batch must be <= 65535 sequences");
  if (B == 0) return COOPT_OK;
  COOPT_REQUIRE(q && k_cache && v_cache && block_table && cu_seqlens_q && seq_lens && out, "null pointer");
  COOPT_REQUIRE(coopt::aligned16(q) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0 && coopt::aligned16(out) &&
                    o_tok_stride % 8 == 0 && o_head_stride % 8 == 0,
                "q/out rows must be 16-byte aligned");
  const int64_t step = kv_dtype == COOPT_DT_BF16 ? 8 : 16;  // elements (INT4: bytes) in 16 bytes
  COOPT_REQUIRE(coopt::aligned16(k_cache) && coopt::aligned16(v_cache) && c_blk_stride % step == 0 &&
                    c_tok_stride % step == 0 && c_head_stride % step == 0,
                "cache rows must be 16-byte aligned");
  if (kv_dtype != COOPT_DT_BF16)
    COOPT_REQUIRE(k_scale && v_scale && ((reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) & 1u) == 0,
                  "INT8 and INT4 caches need 2-byte aligned k_scale and v_scale");
  COOPT_REQUIRE(num_blocks > 0, "num_blocks must be positive");
  const size_t need = coopt_window_attention_workspace(B, Hq, Hkv, D, max_seqlen_q, max_seqlen_k, window, sink_tokens);
  if (workspace_bytes < need || workspace == nullptr) {
    coopt::set_error(std::string(__func__) + ": workspace too small");
    return COOPT_EWORKSPACE;
  }
  (void)total_q;
  Args a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_ts = q_tok_stride;
  a.q_hs = q_head_stride;
  a.kc = k_cache;
  a.vc = v_cache;
  a.c_bs = c_blk_stride;
  a.c_ts = c_tok_stride;
  a.c_hs = c_head_stride;
  a.ks = static_cast<const uint16_t*>(k_scale);
  a.vs = static_cast<const uint16_t*>(v_scale);
  a.s_bs = s_blk_stride;
  a.s_ts = s_tok_stride;
  a.s_hs = s_head_stride;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.cu = cu_seqlens_q;
  a.seq_lens = seq_lens;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.bs_shift = __builtin_ctz(block_size);
  a.max_seqlen_k = max_seqlen_k;
  a.num_blocks = num_blocks;
  // a window of max_seqlen_k keys holds every key of every row, and a first token past
  // max_seqlen_k does not exist
  a.window = window == 0 || window > max_seqlen_k ? max_seqlen_k : window;
  a.sinks = sink_tokens < max_seqlen_k ? sink_tokens : max_seqlen_k;
  a.scale_log2 = softmax_scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.o_ts = o_tok_stride;
  a.o_hs = o_head_stride;
  COOPT_REQUIRE(max_seqlen_q < (1 << 24) && Hq <= 65535, "too many rows for one launch");
  const dim3 grid(max_seqlen_q, Hq, B);
  auto s = static_cast<hipStream_t>(stream);
  if (D == 64) launch<64>(kv_dtype, a, grid, s);
  else launch<128>(kv_dtype, a, grid, s);
  return coopt::check_launch("coopt_window_attention");
}
