// Norms of the query and key heads, the rotation and the KV write of a qkv projection's output in
// one pass: for every token t and every query or key head x = qkv[t, head, :]
//   y = x * rsqrt(mean(x^2) + eps) * w        w: the query heads' or the key heads' weight [D]
//   z = (y1 cos - y2 sin, y2 cos + y1 sin)    the halves of y, cos / sin of the token's position
// in fp32, rounded to bf16 once.  q goes to q_out, k to the cache; v goes to the cache unchanged.
// An INT8 or INT4 cache holds the codes of the rounded k and v, as coopt_kv_write makes them.
//
// What bounds it: the loads in flight at many rows (4093 rows of 32/8 heads of 64, 50.9 MB: 11.5 us, 4.4 TB/s;
// a copy of the bytes 8.1): a lane has one 16-byte load of its row out, beside 48 bytes of cos, sin and weight
// that every head reads again from the caches.  At few rows the call's host time (one row: 9.5 us, the
// kernel 2.8).  4093 rows of 128: 21.4 us into bf16, 20.7 into INT8, 20.8 into INT4 caches (101.7, 93.5 and
// 89.3 MB); of 64 12.4, 13.9 and 14.2; 160 rows of 128 3.7 to 4.2, from four slices of partial sums 5.4 to 6.0.
// A vector
// stays in its lanes' registers: the sum of squares goes round the group by DPP, and so does the
// other half that a rotation needs (through LDS shuffles, 8 a lane, the same rows took 14.1 us).  Token and
// slot are uniform in a block: their page arithmetic is one shift, and cos, sin and the slot load beside
// the row.  Partial sums have a form of their own: their 32 loads in flight cost 75 registers, 31 without.
#include "common.h"
#include "kv_store.h"

namespace {

struct QkNormArgs {
  const uint16_t* qkv;
  int64_t qkv_ts;
  const float* part;
  int ks;
  int64_t slice;
  const uint16_t* qw;
  const uint16_t* kw;
  float eps;
  const int64_t* pos;
  const uint16_t* cos;
  const uint16_t* sin;
  int64_t tab_stride;
  int max_pos;
  uint16_t* q_out;
  int64_t q_ts, q_hs;
  void* kc;
  void* vc;
  int64_t c_bs, c_ts, c_hs;
  uint16_t* k_scale;
  uint16_t* v_scale;
  int64_t s_bs, s_ts, s_hs;
  const int64_t* slot_mapping;
  int Hq, Hkv, block_size, bs_shift;  // bs_shift: log2(block_size) of a power of two, else -1
  int64_t num_slots;
};

// A token's vectors fill as few blocks as hold them, evenly: 384 lanes at 32/8 heads of 64, 2 x 384 of 128.
constexpr int kMaxThreads = 512;

// A G-lane group (G = D/8) takes one (token, head) vector, lane c its elements [8c, 8c + 8).
template <int G, int KV, bool PART>
__global__ __launch_bounds__(kMaxThreads) void qk_norm_kernel(QkNormArgs a) {
  constexpr int D = 8 * G;
  const int t = static_cast<int>(blockIdx.x);
  const int lid = static_cast<int>(blockIdx.y * blockDim.x + threadIdx.x);
  const int h = lid / G, c = lid % G;
  if (h >= a.Hq + 2 * a.Hkv) return;  // whole groups leave together
  const int width = (a.Hq + 2 * a.Hkv) * D;
  const int64_t slot = a.slot_mapping[t], pos = a.pos[t];
  uint4 xr;
  if constexpr (PART) {
    const float* p = a.part + static_cast<int64_t>(t) * width + lid * 8;
    const float4 lo = sum_partials4(p, a.ks, a.slice), hi = sum_partials4(p + 4, a.ks, a.slice);
    xr = make_uint4(pack2_bf16(lo.x, lo.y), pack2_bf16(lo.z, lo.w), pack2_bf16(hi.x, hi.y), pack2_bf16(hi.z, hi.w));
  } else {
    xr = *reinterpret_cast<const uint4*>(a.qkv + t * a.qkv_ts + lid * 8);
  }
  uint4 yr = xr;
  if (h < a.Hq + a.Hkv) {
    const RopeTab tab = rope_tab<G>(a.cos, a.sin, a.tab_stride, pos, a.max_pos, c);
    const uint4 wr = *reinterpret_cast<const uint4*>((h < a.Hq ? a.qw : a.kw) + 8 * c);
    const uint32_t xw[4] = {xr.x, xr.y, xr.z, xr.w}, ww[4] = {wr.x, wr.y, wr.z, wr.w};
    const uint32_t cw[4] = {tab.cos.x, tab.cos.y, tab.cos.z, tab.cos.w};
    const uint32_t sw[4] = {tab.sin.x, tab.sin.y, tab.sin.z, tab.sin.w};
    auto half = [](const uint32_t (&w)[4], int e) { return bf16_to_f32(static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)))); };
    float y[8], ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = half(xw, e);
      ss = fmaf(y[e], y[e], ss);
    }
    const float r = rsqrtf(group_sum_f32<G>(ss) * (1.0f / D) + a.eps);
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] * r * half(ww, e);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = group_other_half<G>(y[e]);  // element i +- D/2
      const float turn = other * half(sw, e);
      z[e] = fmaf(y[e], half(cw, e), c < G / 2 ? -turn : turn);
    }
    yr = make_uint4(pack2_bf16(z[0], z[1]), pack2_bf16(z[2], z[3]), pack2_bf16(z[4], z[5]), pack2_bf16(z[6], z[7]));
    if (h < a.Hq) {
      *reinterpret_cast<uint4*>(a.q_out + t * a.q_ts + static_cast<int64_t>(h) * static_cast<int32_t>(a.q_hs) + c * 8) = yr;
      return;
    }
  }
  if (slot < 0 || slot >= a.num_slots) return;  // padding rows write nothing
  const int64_t blk = a.bs_shift >= 0 ? slot >> a.bs_shift : slot / a.block_size;
  const int64_t off = slot - blk * a.block_size;
  const bool is_k = h < a.Hq + a.Hkv;
  const int64_t hk = is_k ? h - a.Hq : h - a.Hq - a.Hkv;
  store_chunk<G, KV>(yr, is_k ? a.kc : a.vc,
                     blk * a.c_bs + off * a.c_ts + hk * static_cast<int32_t>(a.c_hs) + c * chunk_step<KV>(),
                     is_k ? a.k_scale : a.v_scale,
                     blk * a.s_bs + off * a.s_ts + hk * static_cast<int32_t>(a.s_hs), c);
}

template <int G, int KV>
void launch_kv(const QkNormArgs& a, dim3 grid, dim3 block, hipStream_t s) {
  if (a.part) hipLaunchKernelGGL((qk_norm_kernel<G, KV, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((qk_norm_kernel<G, KV, false>), grid, block, 0, s, a);
}

template <int G>
void launch(int cache_dtype, const QkNormArgs& a, dim3 grid, dim3 block, hipStream_t s) {
  if (cache_dtype == COOPT_DT_BF16) launch_kv<G, kBf16>(a, grid, block, s);
  else if (cache_dtype == COOPT_DT_I8) launch_kv<G, kI8>(a, grid, block, s);
  else launch_kv<G, kI4>(a, grid, block, s);
}

}  // namespace

extern "C" int coopt_qkv_norm_epilogue(
    int cache_dtype, const void* qkv, int64_t qkv_tok_stride, const float* part, int ks,
    int64_t slice_stride, const void* q_weight, const void* k_weight, float eps,
    const int64_t* positions, const void* cos, const void* sin, int64_t table_stride, int max_pos,
    void* q_out, int64_t q_tok_stride, int64_t q_head_stride, void* k_cache, void* v_cache,
    int64_t c_blk_stride, int64_t c_tok_stride, int64_t c_head_stride, void* k_scale, void* v_scale,
    int64_t s_blk_stride, int64_t s_tok_stride, int64_t s_head_stride, const int64_t* slot_mapping,
    int T, int Hq, int Hkv, int D, int block_size, int64_t num_blocks, coopt_stream_t stream) {
  coopt::clear_error();
  COOPT_REQUIRE(cache_dtype == COOPT_DT_BF16 || cache_dtype == COOPT_DT_I8 || cache_dtype == COOPT_DT_I4,
                "cache_dtype must be COOPT_DT_BF16, COOPT_DT_I8 or COOPT_DT_I4");
  COOPT_REQUIRE(T >= 0 && Hq > 0 && Hkv > 0 && block_size > 0 && num_blocks > 0 && max_pos > 0, "bad sizes");
  COOPT_REQUIRE(D == 64 || D == 128 || D == 256, "D must be 64, 128 or 256");
  COOPT_REQUIRE(eps >= 0.0f && eps < 1e30f, "eps must be finite and not negative");
  if (T == 0) return COOPT_OK;
  COOPT_REQUIRE((qkv != nullptr) != (part != nullptr), "give exactly one of qkv and part");
  COOPT_REQUIRE(q_weight && k_weight && positions && cos && sin && q_out && k_cache && v_cache && slot_mapping,
                "null pointer");
  const int64_t width = (static_cast<int64_t>(Hq) + 2 * static_cast<int64_t>(Hkv)) * D;
  COOPT_REQUIRE(width < (int64_t{1} << 27), "(Hq + 2 Hkv) * D must stay below 2^27");
  if (part) {
    COOPT_REQUIRE(ks >= 1 && ks <= 16, "1 to 16 partial slices");
    COOPT_REQUIRE(coopt::aligned16(part) && slice_stride % 4 == 0 && slice_stride >= T * width,
                  "partials must be 16-byte aligned [ks, >= T, (Hq + 2 Hkv) D] fp32");
  } else {
    COOPT_REQUIRE(coopt::aligned16(qkv) && qkv_tok_stride % 8 == 0 && qkv_tok_stride >= width,
                  "qkv rows must be 16-byte aligned, at least (Hq + 2 Hkv) D wide");
  }
  COOPT_REQUIRE(coopt::aligned16(q_weight) && coopt::aligned16(k_weight), "norm weights must be 16-byte aligned");
  COOPT_REQUIRE(coopt::aligned16(cos) && coopt::aligned16(sin) && table_stride % 8 == 0 && table_stride >= D / 2,
                "cos/sin rows must be 16-byte aligned with at least D/2 entries");
  COOPT_REQUIRE(coopt::aligned16(q_out) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0,
                "q_out rows must be 16-byte aligned");
  if (const char* bad = coopt::cache_write_error(cache_dtype, k_cache, v_cache, c_blk_stride, c_tok_stride,
                                                 c_head_stride, k_scale, v_scale)) {
    coopt::set_error(std::string(__func__) + ": " + bad);
    return COOPT_EINVAL;
  }
  COOPT_REQUIRE(coopt::narrow_strides({q_head_stride, c_head_stride, s_head_stride}),
                "head strides must stay below 2^31");
  const int lanes = static_cast<int>(width / 8);
  const int blocks = (lanes + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((lanes + blocks - 1) / blocks + COOPT_WAVE - 1) / COOPT_WAVE * COOPT_WAVE;
  COOPT_REQUIRE(static_cast<int64_t>(T) * blocks < (int64_t{1} << 22) && blocks < 65536, "too many rows for one launch");
  QkNormArgs a{static_cast<const uint16_t*>(qkv), qkv_tok_stride, part, ks, slice_stride,
               static_cast<const uint16_t*>(q_weight), static_cast<const uint16_t*>(k_weight), eps,
               positions, static_cast<const uint16_t*>(cos), static_cast<const uint16_t*>(sin),
               table_stride, max_pos, static_cast<uint16_t*>(q_out), q_tok_stride, q_head_stride,
               k_cache, v_cache, c_blk_stride, c_tok_stride, c_head_stride,
               static_cast<uint16_t*>(k_scale), static_cast<uint16_t*>(v_scale), s_blk_stride,
               s_tok_stride, s_head_stride, slot_mapping, Hq, Hkv, block_size,
               (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1, num_blocks * block_size};
  const dim3 grid(static_cast<unsigned>(T), static_cast<unsigned>(blocks)), block(static_cast<unsigned>(threads));
  auto s = static_cast<hipStream_t>(stream);
  if (D == 64) launch<8>(cache_dtype, a, grid, block, s);
  else if (D == 128) launch<16>(cache_dtype, a, grid, block, s);
  else launch<32>(cache_dtype, a, grid, block, s);
  return coopt::check_launch("coopt_qkv_norm_epilogue");
}
