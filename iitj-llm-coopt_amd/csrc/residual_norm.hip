// The norm behind a block, the block's gate and scale, the residual sum and the norm before the next
// block, in one pass over a row:
//   b   = x, or x * rsqrt(mean(x^2) + eps) * post_weight
//   b  *= gate                                   (a vector, or a row of its own)
//   r   = residual_scale * residual + branch_scale * b
//   out = r * rsqrt(mean(r^2) + eps) * weight
// Everything between the loads and the two stores is fp32: the residual (bf16) and out are rounded once
// each, and the second norm is that of the unrounded r.  A row stays in its block's registers, so it is read
// once and each result written once: 8 bytes an element (10 with a gate of rows).  All loads of a row are issued before
// its first sum, as many waves a row as leave a chunk a thread: 8191 rows of 4096 with a gate of rows 57 to 59 us
// (5.7 to 5.9 TB/s, above the 5.1 of a large copy), one row 2.7, two sums through the block and one round trip.
#include "common.h"

namespace {

struct Row {
  const uint16_t* x;       // null: part
  const float* part;       // ks slices of fp32 partial sums; x = bf16(their sum in order)
  int ks;
  int64_t slice;
  const uint16_t* residual;
  uint16_t* residual_out;  // may be residual
  const uint16_t* post;    // null: no norm behind the block
  const uint16_t* gate;    // null: none
  int64_t gate_stride;     // 0: one vector for every row
  const uint16_t* weight;
  uint16_t* out;
  int H;
  float eps, branch_scale, residual_scale;
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = __uint_as_float(w[e] << 16);
    f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = f32_to_bf16(f[2 * e]) | (static_cast<uint32_t>(f32_to_bf16(f[2 * e + 1])) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sum over the block, every thread the same bits; `sh` is used by no other call.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = group_sum_f32<64>(v);
  if constexpr (WAVES == 1) return v;
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s += sh[w];
  return s;
}

// One block of 64 * WAVES threads a row, CPT chunks of eight elements a thread.  KS: a bound of the slices of partial sums,
// known to the compiler, so that all of them are loaded at once (0: x, or any number of slices).  Four slices of 160 rows
// of 4096 4.2 us for 4.6, of 32 rows of 2048 3.2 for 3.7.
template <int WAVES, int CPT, int KS>
__global__ __launch_bounds__(64 * WAVES) void residual_norm_kernel(const Row a) {
  constexpr int kThreads = 64 * WAVES;
  __shared__ float sh[2][WAVES];
  const int64_t row = blockIdx.x;
  const int H = a.H;
  float b[CPT][8];
  uint4 res[CPT], wv[CPT], pv[CPT], gv[CPT];
  Partials4<(KS > 0 ? KS : 1)> plo[CPT], phi[CPT];
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * kThreads + threadIdx.x) * 8;
    const int il = i < H ? i : H - 8;   // chunks past the row load its last one and are not counted
    if constexpr (KS > 0) {
      const float* p = a.part + row * H + il;
      plo[c].load(p, a.ks, a.slice);
      phi[c].load(p + 4, a.ks, a.slice);
    } else if (a.part) {
      const float* p = a.part + row * H + il;
      const float4 lo = sum_partials4(p, a.ks, a.slice), hi = sum_partials4(p + 4, a.ks, a.slice);
      const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      unpack8(pack8(f), b[c]);
    } else {
      unpack8(*reinterpret_cast<const uint4*>(a.x + row * H + il), b[c]);
    }
    res[c] = *reinterpret_cast<const uint4*>(a.residual + row * H + il);
    wv[c] = *reinterpret_cast<const uint4*>(a.weight + il);
    if (a.post) pv[c] = *reinterpret_cast<const uint4*>(a.post + il);
    if (a.gate) gv[c] = *reinterpret_cast<const uint4*>(a.gate + row * a.gate_stride + il);
  }
  if constexpr (KS > 0) {
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const float4 lo = plo[c].sum(a.ks), hi = phi[c].sum(a.ks);
      const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      unpack8(pack8(f), b[c]);
    }
  }
  if (a.post) {
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if ((c * kThreads + static_cast<int>(threadIdx.x)) * 8 < H)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += b[c][e] * b[c][e];
    const float rs = rsqrtf(block_sum<WAVES>(ss, sh[0]) / static_cast<float>(H) + a.eps);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      float p[8];
      unpack8(pv[c], p);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[c][e] = b[c][e] * rs * p[e];
    }
  }
  ss = 0.0f;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * kThreads + threadIdx.x) * 8;
    if (a.gate) {
      float g[8];
      unpack8(gv[c], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[c][e] *= g[e];
    }
    float r[8];
    unpack8(res[c], r);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[c][e] = a.residual_scale * r[e] + a.branch_scale * b[c][e];
    if (i < H) {
      *reinterpret_cast<uint4*>(a.residual_out + row * H + i) = pack8(b[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += b[c][e] * b[c][e];
    }
  }
  const float rs = rsqrtf(block_sum<WAVES>(ss, sh[1]) / static_cast<float>(H) + a.eps);
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * kThreads + threadIdx.x) * 8;
    if (i >= H) continue;
    float w[8];
    unpack8(wv[c], w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] *= b[c][e] * rs;
    *reinterpret_cast<uint4*>(a.out + row * H + i) = pack8(w);
  }
}

// A grid counts its threads in 32 bits: more rows than these go in several launches.
constexpr int64_t kLaunchRows = 1 << 21;

template <int WAVES, int CPT, int KS>
void launch_slices(Row a, int64_t rows, hipStream_t s) {
  for (; rows > 0; rows -= kLaunchRows) {
    const int64_t n = rows < kLaunchRows ? rows : kLaunchRows, past = n * a.H;
    hipLaunchKernelGGL((residual_norm_kernel<WAVES, CPT, KS>), dim3(static_cast<unsigned>(n)), dim3(64 * WAVES), 0, s, a);
    if (a.x) a.x += past;
    if (a.part) a.part += past;
    if (a.gate) a.gate += n * a.gate_stride;
    a.residual += past;
    a.residual_out += past;
    a.out += past;
  }
}

template <int WAVES, int CPT>
void launch(const Row& a, int64_t rows, hipStream_t s) {
  if constexpr (CPT == 1) {   // (eight slices of two chunks do not fit the registers of 16 waves)
    if (a.part && a.ks <= 4) return launch_slices<WAVES, CPT, 4>(a, rows, s);
    if (a.part && a.ks <= 8) return launch_slices<WAVES, CPT, 8>(a, rows, s);
  }
  launch_slices<WAVES, CPT, 0>(a, rows, s);
}

constexpr int kMaxHidden = 16384;

}  // namespace

extern "C" int coopt_residual_norm(const void* x, const float* part, int ks, int64_t slice_stride, const void* residual,
                                   void* residual_out, const void* post_weight, const void* gate,
                                   int64_t gate_stride, const void* weight, void* out, int64_t rows, int hidden,
                                   float eps, float branch_scale, float residual_scale, coopt_stream_t stream) {
  coopt::clear_error();
  COOPT_REQUIRE(rows >= 0 && rows <= (int64_t(1) << 40) && hidden > 0 && hidden % 8 == 0 && hidden <= kMaxHidden,
                "hidden must be a multiple of 8, at most 16384");
  COOPT_REQUIRE(eps >= 0.0f && eps <= 3.0e38f, "eps must be finite and not negative");
  if (rows == 0) return COOPT_OK;
  COOPT_REQUIRE((x != nullptr) != (part != nullptr), "exactly one of x and part is needed");
  COOPT_REQUIRE(part == nullptr || (ks >= 1 && ks <= 16 && slice_stride >= rows * hidden && slice_stride % 4 == 0),
                "1 to 16 partial slices of rows * hidden floats");
  COOPT_REQUIRE(residual && residual_out && weight && out, "null pointer");
  COOPT_REQUIRE(gate_stride == 0 || (gate_stride >= hidden && gate_stride % 8 == 0),
                "gate rows must be 16-byte aligned and at least hidden apart");
  for (const void* p : {x, static_cast<const void*>(part), residual, static_cast<const void*>(residual_out), post_weight,
                        gate, weight, static_cast<const void*>(out)})
    COOPT_REQUIRE(coopt::aligned16(p), "rows must be 16-byte aligned");
  const Row a{static_cast<const uint16_t*>(x), part, ks, slice_stride, static_cast<const uint16_t*>(residual),
              static_cast<uint16_t*>(residual_out), static_cast<const uint16_t*>(post_weight),
              static_cast<const uint16_t*>(gate), gate_stride, static_cast<const uint16_t*>(weight),
              static_cast<uint16_t*>(out), hidden, eps, branch_scale, residual_scale};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int chunks = hidden / 8;
  if (chunks <= 64) launch<1, 1>(a, rows, s);
  else if (chunks <= 256) launch<4, 1>(a, rows, s);
  else if (chunks <= 512) launch<8, 1>(a, rows, s);
  else if (chunks <= 1024) launch<16, 1>(a, rows, s);
  else launch<16, 2>(a, rows, s);
  return coopt::check_launch("coopt_residual_norm");
}
