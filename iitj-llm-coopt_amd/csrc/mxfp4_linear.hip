// Products with microscaled 4-bit weights: Y[M, N] = X[M, K] W[N, K]^T, bf16 out, fp32 accumulation.
// W is packed (mxfp4.h); X is bf16 (A4 = false) or quantised in the call to the same 4-bit format (A4 = true).
//
// A4 = false.  A weight is a bf16 number, so the product is exactly that of the bf16 matrix instructions
// on code * 2^e: a lane's 16 bytes of a tile are 32 elements of one row and one block, four operands of
// v_mfma_f32_16x16x32_bf16 after 16 v_cvt_scalef32_pk_bf16_fp4 (two elements each, scale applied).  The K
// order inside a step is any that both operands share: operand j of lane (row, g) holds elements
// 32 g + 8 j .. + 7 of the step.
// A4 = true.  A lane's 16 bytes are its operand of v_mfma_scale_f32_16x16x128_f8f6f4 as they are, with
// their scale bytes: products and sums of a step are formed by the matrix core.
// In both the weight is the A operand, so a lane ends with four consecutive outputs of one row.
#include "mxfp4.h"

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

using mxfp4::kStep;
using mxfp4::kTile;

struct Args {
  const uint16_t* x;           // A4 = false
  int64_t ldx;
  const uint8_t* xt;           // A4 = true: packed activations and their scales
  const uint32_t* xs;
  const uint8_t* w;            // packed weight and its scales
  const uint32_t* ws;
  int M, N, K;
  int ksteps, kquads;
  int slice_quads;             // K quads (512 elements) of a K slice
  uint16_t* y;                 // part == nullptr: the outputs
  int64_t ldy;
  float* part;                 // else slices [part_rows, pitch] of fp32 sums
  int64_t part_slice;
  int pitch;
};

__device__ __forceinline__ f32x4_t mfma_bf16(const uint4& a, const uint4& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                 c, 0, 0, 0);
}

template <int J>
__device__ __forceinline__ f32x4_t mfma_fp4(const uint4& a, uint32_t sa, const uint4& b, uint32_t sb, f32x4_t c) {
  const i32x8_t av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
  const i32x8_t bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, J, static_cast<int>(sa), J,
                                                          static_cast<int>(sb));
}

template <int J>
__device__ __forceinline__ float step_scale(uint32_t quad) {
  return mxfp4::scale_operand((quad >> (8 * J)) & 255u);
}

__device__ __forceinline__ uint32_t dword(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Four consecutive outputs n .. n + 3 of row m.
__device__ __forceinline__ void store4(const Args& a, int m, int n, f32x4_t v) {
  if (m >= a.M || n >= a.N) return;
  if (a.part) {
    float* p = a.part + blockIdx.y * a.part_slice + static_cast<int64_t>(m) * a.pitch + n;
    *reinterpret_cast<f32x4_t*>(p) = v;   // pitch is a multiple of 16
    return;
  }
  uint16_t* o = a.y + static_cast<int64_t>(m) * a.ldy + n;
  const uint32_t lo = f32_to_bf16(v[0]) | (static_cast<uint32_t>(f32_to_bf16(v[1])) << 16);
  const uint32_t hi = f32_to_bf16(v[2]) | (static_cast<uint32_t>(f32_to_bf16(v[3])) << 16);
  if (n + 3 < a.N && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
    *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
  } else {
    const uint16_t e[4] = {static_cast<uint16_t>(lo), static_cast<uint16_t>(lo >> 16), static_cast<uint16_t>(hi),
                           static_cast<uint16_t>(hi >> 16)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = e[i];
  }
}

// Few rows: every wave of a block has the same NT column tiles and its own K quads, reads X where it lies
// (caches serve it to the blocks) and the block adds the waves' sums in LDS, in order.  No barrier before that.
template <bool A4, bool TAIL, int MT, int NT, int KW>
__global__ __launch_bounds__(64 * KW) void mxfp4_stream_kernel(const Args a) {
  __shared__ f32x4_t red[KW][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (NT * 16), m0 = blockIdx.z * (MT * 16);
  const int ntiles = (a.N + 15) / 16, mtiles = (a.M + 15) / 16;
  const int qbeg = blockIdx.y * a.slice_quads;
  const int qend = qbeg + a.slice_quads < a.kquads ? qbeg + a.slice_quads : a.kquads;

  const uint8_t* wt[NT];
  const uint32_t* wsc[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    int t = n0 / 16 + nt;
    t = t < ntiles ? t : ntiles - 1;   // tiles past the weight: computed, not stored
    wt[nt] = a.w + static_cast<int64_t>(t) * a.ksteps * kTile + lane * 16;
    wsc[nt] = a.ws + static_cast<int64_t>(t) * a.kquads * 64 + lane;
  }
  const uint16_t* xr[MT];
  const uint8_t* xt[MT];
  const uint32_t* xsc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if constexpr (A4) {
      int t = m0 / 16 + mt;
      t = t < mtiles ? t : mtiles - 1;
      xt[mt] = a.xt + static_cast<int64_t>(t) * a.ksteps * kTile + lane * 16;
      xsc[mt] = a.xs + static_cast<int64_t>(t) * a.kquads * 64 + lane;
    } else {
      int m = m0 + mt * 16 + l16;
      m = m < a.M ? m : a.M - 1;
      xr[mt] = a.x + static_cast<int64_t>(m) * a.ldx;
    }
  }
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (int q = qbeg + wave; q < qend; q += KW) {
    uint4 w[4][NT];
    uint32_t sw[NT], sx[MT];
    const int left = a.ksteps - 4 * q;   // steps from this quad's first on
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sw[nt] = wsc[nt][q * 64];
    if constexpr (A4) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sx[mt] = xsc[mt][q * 64];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int u = 4 * q + (j < left ? j : left - 1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) w[j][nt] = *reinterpret_cast<const uint4*>(wt[nt] + static_cast<int64_t>(u) * kTile);
    }
    auto step = [&](auto J) {
      constexpr int j = J.value;
      if (j >= left) return;
      const int u = 4 * q + j;
      if constexpr (A4) {
        uint4 xv[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) xv[mt] = *reinterpret_cast<const uint4*>(xt[mt] + static_cast<int64_t>(u) * kTile);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = mfma_fp4<j>(w[j][nt], sw[nt], xv[mt], sx[mt], acc[mt][nt]);
      } else {
        const int k = u * kStep + 32 * g;
        const bool live = !TAIL || k < a.K;
        uint4 xv[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            xv[mt][i] = *reinterpret_cast<const uint4*>(xr[mt] + (live ? k : 0) + 8 * i);
            if (TAIL && !live) xv[mt][i] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float s = step_scale<j>(sw[nt]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 b = mxfp4::bf16_of(dword(w[j][nt], i), s);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = mfma_bf16(b, xv[mt][i], acc[mt][nt]);
          }
        }
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  }

#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) red[wave][mt * NT + nt][lane] = acc[mt][nt];
  __syncthreads();
  for (int t = wave; t < MT * NT; t += KW) {
    f32x4_t s = red[0][t][lane];
#pragma unroll
    for (int k = 1; k < KW; ++k) s += red[k][t][lane];
    store4(a, m0 + (t / NT) * 16 + l16, n0 + (t % NT) * 16 + 4 * g, s);
  }
}

// Rows of X to packed 4-bit tiles.  A block is a tile, a wave its block g of 32 elements, four lanes a row of it.
__global__ __launch_bounds__(256) void mxfp4_pack_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx, int M, int K,
                                                              int ksteps, int kquads, uint32_t* __restrict__ tiles,
                                                              uint8_t* __restrict__ scales) {
  const int u = blockIdx.x, t = blockIdx.y, g = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane >> 2, q = lane & 3;
  const int row = 16 * t + r;
  if (row >= M) return;
  const int k = u * kStep + 32 * g + 8 * q;
  uint32_t code = 0, s = 127;
  if (k < K) {   // the same for a block's four lanes
    const uint4 v = *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(row) * ldx + k);
    s = mxfp4::scale_byte(group_max_u32<4>(mxfp4::amax_bits(v)));
    code = mxfp4::codes_of(v, s);
  }
  const int l = 16 * g + r;
  tiles[((static_cast<int64_t>(t) * ksteps + u) * 64 + l) * 4 + q] = code;
  if (q == 0) scales[((static_cast<int64_t>(t) * kquads + u / 4) * 64 + l) * 4 + (u & 3)] = static_cast<uint8_t>(s);
}

// y[m, n] = bf16(sum over slices in order), four columns a thread.
__global__ __launch_bounds__(256) void mxfp4_reduce_kernel(const float* __restrict__ part, int ks, int64_t slice,
                                                           int pitch, int M, int N, uint16_t* __restrict__ y,
                                                           int64_t ldy) {
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int per_row = pitch / 4;
  const int64_t m = gid / per_row;
  const int n = static_cast<int>(gid - m * per_row) * 4;
  if (m >= M || n >= N) return;
  const float4 s = sum_partials4(part + m * pitch + n, ks, slice);
  Args a{};
  a.M = M; a.N = N; a.y = y; a.ldy = ldy;
  store4(a, static_cast<int>(m), n, f32x4_t{s.x, s.y, s.z, s.w});
}

struct Plan {
  int mt, nt, kw;
  int ks, slice_quads;
  int rows_padded, pitch;
};

Plan plan_for(int M, int N, int K, bool a4) {
  Plan p{};
  const int mtiles = static_cast<int>(mxfp4::row_tiles(M)), quads = static_cast<int>(mxfp4::quads(K));
  p.mt = mtiles <= 1 ? 1 : mtiles <= 2 ? 2 : 4;
  p.nt = 2;
  p.kw = 4;
  p.ks = 1;
  p.slice_quads = (quads + p.ks - 1) / p.ks;
  p.rows_padded = mtiles * 16;
  p.pitch = static_cast<int>(mxfp4::row_tiles(N)) * 16;
  return p;
}

int64_t part_bytes(const Plan& p, bool partials) {
  return p.ks > 1 || partials ? int64_t{4} * p.ks * p.rows_padded * p.pitch : 0;
}

template <bool A4, bool TAIL>
void launch_product(const Plan& p, const Args& a, hipStream_t s) {
  const dim3 grid((a.N + 16 * p.nt - 1) / (16 * p.nt), p.ks, (a.M + 16 * p.mt - 1) / (16 * p.mt));
  switch (p.mt) {
    case 1: hipLaunchKernelGGL((mxfp4_stream_kernel<A4, TAIL, 1, 2, 4>), grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL((mxfp4_stream_kernel<A4, TAIL, 2, 2, 4>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((mxfp4_stream_kernel<A4, TAIL, 4, 2, 4>), grid, dim3(256), 0, s, a); break;
  }
}

constexpr int kMaxRows = 1 << 19;   // the grids count row tiles in a dimension of 65535

const char* shape_error(int M, int N, int K) {
  if (M < 0 || N < 0 || K < 0) return "negative size";
  if (K % mxfp4::kBlock || (K == 0 && M && N)) return "K must be a positive multiple of 32";
  if (M > kMaxRows) return "M must be at most 2^19";
  if (N > (1 << 24) || K > (1 << 24)) return "N and K must be at most 2^24";
  return nullptr;
}

// The product; with `partials` every slice (also a single one) stays in the workspace as fp32.
int run(const void* x, int64_t ldx, const void* w, int M, int N, int K, int act4, void* y, int64_t ldy, void* workspace,
        size_t workspace_bytes, bool partials, coopt_stream_t stream, const char* who) {
  const char* bad = shape_error(M, N, K);
  if (!bad && M && N) {
    if (!x || !w || (!y && !partials)) bad = "null pointer";
    else if (!coopt::aligned16(x) || !coopt::aligned16(w)) bad = "x and w must be 16-byte aligned";
    else if (ldx < K || ldx % 8) bad = "row stride of x must be >= K and a multiple of 8";
    else if (!partials && (ldy < N || (reinterpret_cast<uintptr_t>(y) & 1))) bad = "row stride of y must be >= N";
    else if (partials && N % 16) bad = "partial sums need N a multiple of 16";
  }
  if (bad) {
    coopt::set_error(std::string(who) + ": " + bad);
    return COOPT_EINVAL;
  }
  if (M == 0 || N == 0) return COOPT_OK;
  const Plan p = plan_for(M, N, K, act4 != 0);
  const int64_t pb = part_bytes(p, partials), need = pb + (act4 ? mxfp4::packed_bytes(M, K) : 0);
  if (need && (static_cast<int64_t>(workspace_bytes) < need || !workspace || !coopt::aligned16(workspace))) {
    coopt::set_error(std::string(who) + ": workspace smaller than required (or misaligned)");
    return COOPT_EWORKSPACE;
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.w = static_cast<const uint8_t*>(w);
  a.ws = reinterpret_cast<const uint32_t*>(a.w + mxfp4::tile_bytes(N, K));
  a.M = M; a.N = N; a.K = K;
  a.ksteps = static_cast<int>(mxfp4::steps(K));
  a.kquads = static_cast<int>(mxfp4::quads(K));
  a.slice_quads = p.slice_quads;
  a.y = static_cast<uint16_t*>(y);
  a.ldy = ldy;
  a.part = pb ? static_cast<float*>(workspace) : nullptr;
  a.part_slice = static_cast<int64_t>(p.rows_padded) * p.pitch;
  a.pitch = p.pitch;
  if (act4) {
    uint8_t* tiles = static_cast<uint8_t*>(workspace) + pb;
    uint8_t* scales = tiles + mxfp4::tile_bytes(M, K);
    a.xt = tiles;
    a.xs = reinterpret_cast<const uint32_t*>(scales);
    hipLaunchKernelGGL(mxfp4_pack_rows_kernel, dim3(a.ksteps, static_cast<unsigned>(mxfp4::row_tiles(M))), dim3(256), 0, s,
                       a.x, ldx, M, K, a.ksteps, a.kquads, reinterpret_cast<uint32_t*>(tiles), scales);
    launch_product<true, false>(p, a, s);
  } else if (K % kStep) {
    launch_product<false, true>(p, a, s);
  } else {
    launch_product<false, false>(p, a, s);
  }
  if (pb && !partials) {
    const int64_t n = static_cast<int64_t>(M) * (p.pitch / 4);
    hipLaunchKernelGGL(mxfp4_reduce_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s, a.part, p.ks,
                       a.part_slice, p.pitch, M, N, a.y, ldy);
  }
  return coopt::check_launch(who);
}

}  // namespace

extern "C" size_t coopt_mxfp4_linear_workspace(int M, int N, int K, int act4, int partials) {
  if (shape_error(M, N, K) || M == 0 || N == 0) return 0;
  const Plan p = plan_for(M, N, K, act4 != 0);
  return static_cast<size_t>(part_bytes(p, partials != 0) + (act4 ? mxfp4::packed_bytes(M, K) : 0));
}

extern "C" int coopt_mxfp4_linear_split(int M, int N, int K, int act4, int* ks, int* rows_padded) {
  coopt::clear_error();
  COOPT_REQUIRE(ks && rows_padded, "null output pointer");
  COOPT_REQUIRE(!shape_error(M, N, K) && M > 0 && N > 0, "unsupported shape");
  const Plan p = plan_for(M, N, K, act4 != 0);
  *ks = p.ks;
  *rows_padded = p.rows_padded;
  return COOPT_OK;
}

extern "C" int coopt_mxfp4_linear(const void* x, int64_t ldx, const void* w_packed, int M, int N, int K, int act4, void* y,
                                  int64_t ldy, void* workspace, size_t workspace_bytes, coopt_stream_t stream) {
  coopt::clear_error();
  return run(x, ldx, w_packed, M, N, K, act4, y, ldy, workspace, workspace_bytes, false, stream, "coopt_mxfp4_linear");
}

extern "C" int coopt_mxfp4_linear_partials(const void* x, int64_t ldx, const void* w_packed, int M, int N, int K, int act4,
                                           void* workspace, size_t workspace_bytes, coopt_stream_t stream) {
  coopt::clear_error();
  return run(x, ldx, w_packed, M, N, K, act4, nullptr, 0, workspace, workspace_bytes, true, stream,
             "coopt_mxfp4_linear_partials");
}
