// Microscaled 4-bit rows: quantisation, the values back, and packing for the products of
// mxfp4_linear.hip.  Format and packed layout: mxfp4.h.
#include "mxfp4.h"

namespace {

constexpr int kThreads = 256;

// Eight elements a thread, four neighbouring lanes a block: one 16-byte load (bf16, fp16; two for fp32),
// the block's largest magnitude by two lane exchanges, one 4-byte store of codes.  Rows are contiguous and K
// is a multiple of 32, so blocks do not know rows.  A stream of 2 + 17/32 bytes an element, bound by memory:
// 28672 x 4096 bf16 53 to 58 us (5.1 to 5.6 TB/s); 160 x 4096 2.1, launch and one round trip.
template <int DT>
__global__ __launch_bounds__(kThreads) void mxfp4_quantize_kernel(const void* __restrict__ x, int64_t eighths,
                                                                  uint32_t* __restrict__ codes,
                                                                  uint8_t* __restrict__ scales) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= eighths) return;   // whole groups of four lanes: a block has four eighths
  uint32_t code, s;
  if constexpr (DT == COOPT_DT_BF16) {
    const mxfp4::u32x4_t v[1] = {reinterpret_cast<const mxfp4::u32x4_t*>(x)[i]};
    s = mxfp4::scale_byte(group_max_u32<4>(mxfp4::amax_bits(v)));
    code = mxfp4::codes_of(v[0], s);
  } else {
    float f[8];
    if constexpr (DT == COOPT_DT_F16) {
      const mxfp4::u32x4_t v = reinterpret_cast<const mxfp4::u32x4_t*>(x)[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f16_to_f32(static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1))));
    } else {
      const float4 a = reinterpret_cast<const float4*>(x)[2 * i], b = reinterpret_cast<const float4*>(x)[2 * i + 1];
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t a = __float_as_uint(f[e]) & 0x7fffffffu;
      m = m > a ? m : a;
    }
    s = mxfp4::scale_byte(group_max_u32<4>(m));
    code = mxfp4::codes_of(f, s);
  }
  codes[i] = code;
  if ((i & 3) == 0) scales[i >> 2] = static_cast<uint8_t>(s);
}

// Eight elements a thread: a 4-byte load and one 16-byte store (two for fp32).  The same stream the other way:
// 28672 x 4096 to bf16 53 us (5.6 TB/s).
template <int DT>
__global__ __launch_bounds__(kThreads) void mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ scales,
                                                                    int64_t eighths, void* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= eighths) return;
  const uint32_t s = scales[i >> 2];
  const mxfp4::u32x4_t b = mxfp4::bf16_of(codes[i], mxfp4::scale_operand(s));
  if constexpr (DT == COOPT_DT_BF16) {
    reinterpret_cast<mxfp4::u32x4_t*>(out)[i] = b;
  } else {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = bf16_to_f32(static_cast<uint16_t>(b[e / 2] >> (16 * (e & 1))));
    if constexpr (DT == COOPT_DT_F32) {
      reinterpret_cast<float4*>(out)[2 * i] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(out)[2 * i + 1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {   // rounded to nearest, values past fp16's range to infinity
      uint4 h;
      h.x = f32_to_f16(f[0]) | (static_cast<uint32_t>(f32_to_f16(f[1])) << 16);
      h.y = f32_to_f16(f[2]) | (static_cast<uint32_t>(f32_to_f16(f[3])) << 16);
      h.z = f32_to_f16(f[4]) | (static_cast<uint32_t>(f32_to_f16(f[5])) << 16);
      h.w = f32_to_f16(f[6]) | (static_cast<uint32_t>(f32_to_f16(f[7])) << 16);
      reinterpret_cast<uint4*>(out)[i] = h;
    }
  }
}

// A weight's rows into tiles, once when a model is loaded.  Thread (tu, l): chunk l of tile tu, and with
// u % 4 = 0 the dword of four scales.
__global__ __launch_bounds__(kThreads) void mxfp4_pack_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales, int N, int K,
                                                              int kquads, int64_t chunks,
                                                              uint4* __restrict__ tiles, uint32_t* __restrict__ packed_scales) {
  const int64_t o = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (o >= chunks) return;
  const int l = static_cast<int>(o & 63);
  const int64_t tu = o >> 6, t = tu / (4 * kquads);
  const int u = static_cast<int>(tu - t * 4 * kquads);
  const int64_t row = mxfp4::weight_row(t, l & 15);
  const int block = 4 * u + (l >> 4), blocks = K / mxfp4::kBlock;
  uint4 c = make_uint4(0, 0, 0, 0);
  if (row < N && block < blocks)
    c = *reinterpret_cast<const uint4*>(codes + (row * blocks + block) * (mxfp4::kBlock / 2));
  tiles[o] = c;
  if ((u & 3) == 0) {
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = block + 4 * i;
      s |= (row < N && b < blocks ? static_cast<uint32_t>(scales[row * blocks + b]) : 127u) << (8 * i);
    }
    packed_scales[(t * kquads + u / 4) * 64 + l] = s;
  }
}

// A grid counts its threads in 32 bits.
bool blocks_fit(int64_t threads) { return threads <= 0xffffffffll - kThreads; }

dim3 grid_for(int64_t threads) { return dim3(static_cast<unsigned>((threads + kThreads - 1) / kThreads)); }

}  // namespace

extern "C" int coopt_mxfp4_quantize(int in_dtype, const void* x, int64_t rows, int K, void* codes, void* scales,
                                    coopt_stream_t stream) {
  coopt::clear_error();
  COOPT_REQUIRE(in_dtype == COOPT_DT_BF16 || in_dtype == COOPT_DT_F16 || in_dtype == COOPT_DT_F32,
                "in_dtype must be bf16, fp16 or fp32");
  COOPT_REQUIRE(rows >= 0 && K >= 0 && K % mxfp4::kBlock == 0, "K must be a multiple of 32");
  if (rows == 0 || K == 0) return COOPT_OK;
  COOPT_REQUIRE(x && codes && scales, "null pointer");
  COOPT_REQUIRE(coopt::aligned16(x) && (reinterpret_cast<uintptr_t>(codes) & 3) == 0,
                "x must be 16-byte and codes 4-byte aligned");
  COOPT_REQUIRE(rows <= (int64_t(1) << 40) / K && blocks_fit(rows * (K / 8)), "x too large");
  const int64_t n = rows * (K / 8);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  uint32_t* c = static_cast<uint32_t*>(codes);
  uint8_t* sc = static_cast<uint8_t*>(scales);
  if (in_dtype == COOPT_DT_BF16)
    hipLaunchKernelGGL(mxfp4_quantize_kernel<COOPT_DT_BF16>, grid_for(n), dim3(kThreads), 0, s, x, n, c, sc);
  else if (in_dtype == COOPT_DT_F16)
    hipLaunchKernelGGL(mxfp4_quantize_kernel<COOPT_DT_F16>, grid_for(n), dim3(kThreads), 0, s, x, n, c, sc);
  else
    hipLaunchKernelGGL(mxfp4_quantize_kernel<COOPT_DT_F32>, grid_for(n), dim3(kThreads), 0, s, x, n, c, sc);
  return coopt::check_launch("coopt_mxfp4_quantize");
}

extern "C" int coopt_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int K, int out_dtype,
                                      void* out, coopt_stream_t stream) {
  coopt::clear_error();
  COOPT_REQUIRE(out_dtype == COOPT_DT_BF16 || out_dtype == COOPT_DT_F16 || out_dtype == COOPT_DT_F32,
                "out_dtype must be bf16, fp16 or fp32");
  COOPT_REQUIRE(rows >= 0 && K >= 0 && K % mxfp4::kBlock == 0, "K must be a multiple of 32");
  if (rows == 0 || K == 0) return COOPT_OK;
  COOPT_REQUIRE(codes && scales && out, "null pointer");
  COOPT_REQUIRE(coopt::aligned16(out) && (reinterpret_cast<uintptr_t>(codes) & 3) == 0,
                "out must be 16-byte and codes 4-byte aligned");
  COOPT_REQUIRE(rows <= (int64_t(1) << 40) / K && blocks_fit(rows * (K / 8)), "out too large");
  const int64_t n = rows * (K / 8);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const uint32_t* c = static_cast<const uint32_t*>(codes);
  const uint8_t* sc = static_cast<const uint8_t*>(scales);
  if (out_dtype == COOPT_DT_BF16)
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<COOPT_DT_BF16>, grid_for(n), dim3(kThreads), 0, s, c, sc, n, out);
  else if (out_dtype == COOPT_DT_F16)
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<COOPT_DT_F16>, grid_for(n), dim3(kThreads), 0, s, c, sc, n, out);
  else
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<COOPT_DT_F32>, grid_for(n), dim3(kThreads), 0, s, c, sc, n, out);
  return coopt::check_launch("coopt_mxfp4_dequantize");
}

extern "C" size_t coopt_mxfp4_packed_bytes(int N, int K) {
  if (N <= 0 || K <= 0 || K % mxfp4::kBlock) return 0;
  return static_cast<size_t>(mxfp4::packed_bytes(mxfp4::weight_tiles(N), K));
}

extern "C" int coopt_mxfp4_pack_weight(const void* codes, const void* scales, int N, int K, void* out,
                                       coopt_stream_t stream) {
  coopt::clear_error();
  COOPT_REQUIRE(N >= 0 && K >= 0 && K % mxfp4::kBlock == 0, "K must be a multiple of 32");
  if (N == 0 || K == 0) return COOPT_OK;
  COOPT_REQUIRE(codes && scales && out, "null pointer");
  COOPT_REQUIRE(coopt::aligned16(codes) && coopt::aligned16(out), "codes and out must be 16-byte aligned");
  const int64_t chunks = mxfp4::tile_bytes(mxfp4::weight_tiles(N), K) / 16;
  COOPT_REQUIRE(blocks_fit(chunks), "weight too large");
  hipLaunchKernelGGL(mxfp4_pack_kernel, grid_for(chunks), dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), N, K,
                     static_cast<int>(mxfp4::quads(K)), chunks,
                     static_cast<uint4*>(out),
                     reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out) + mxfp4::tile_bytes(mxfp4::weight_tiles(N), K)));
  return coopt::check_launch("coopt_mxfp4_pack_weight");
}
