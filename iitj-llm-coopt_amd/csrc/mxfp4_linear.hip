// Products with microscaled 4-bit weights: Y[M, N] = X[M, K] W[N, K]^T, bf16 out, fp32 accumulation.
// W is packed (mxfp4.h); X is bf16 (A4 = false) or quantised in the call to the same 4-bit format (A4 = true).
//
// A4 = false.  A weight is a bf16 number (scale bytes up to 252, mxfp4.h), so the product is exactly that of the bf16
// matrix instructions on code * 2^e: a lane's 16 bytes of a tile are 32 elements of one row and one block, four
// operands of v_mfma_f32_16x16x32_bf16 after 16 v_cvt_scalef32_pk_bf16_fp4 (two elements each, scale applied).  The K
// order inside a step is any that both operands share: operand j of lane (row, g) holds elements 32 g + 8 j .. + 7 of
// the step.
// A4 = true.  A lane's 16 bytes are its operand of v_mfma_scale_f32_16x16x128_f8f6f4 as they are, with
// their scale bytes: products and sums of a step are formed by the matrix core.
// In both the weight is the A operand, so a lane ends with four consecutive outputs of one row.
#include <algorithm>

#include "mxfp4.h"

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

using mxfp4::kQuad;
using mxfp4::kStep;
using mxfp4::u32x4_t;
using mxfp4::kTile;

struct Args {
  const uint16_t* x;           // A4 = false
  int64_t ldx;
  const uint8_t* xt;           // A4 = true: packed activations and their scales
  const uint32_t* xs;
  const uint8_t* w;            // packed weight and its scales
  const uint32_t* ws;
  int M, N, K;
  int kquads;                  // K in quads of 512 elements
  int slice_quads;             // K quads (512 elements) of a K slice
  uint16_t* y;                 // part == nullptr: the outputs
  int64_t ldy;
  float* part;                 // else slices [part_rows, pitch] of fp32 sums
  int64_t part_slice;
  int pitch;
};

__device__ __forceinline__ f32x4_t mfma_bf16(const u32x4_t& a, const u32x4_t& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                 c, 0, 0, 0);
}

// J, JX: the bytes of sa and sb that are the operands' scales.
template <int J, int JX = J>
__device__ __forceinline__ f32x4_t mfma_fp4(const u32x4_t& a, uint32_t sa, const u32x4_t& b, uint32_t sb, f32x4_t c) {
  const i32x8_t av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
  const i32x8_t bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, J, static_cast<int>(sa), JX,
                                                          static_cast<int>(sb));
}

// Two fp32 -> packed bf16, round to nearest even (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo, hi}), mxfp4::bf16x2_t));
}

// A wave-uniform offset that stays in a scalar register: otherwise the compiler turns base + offset + lane into
// a running address a lane of each tile, in vector registers that the products need.
__device__ __forceinline__ uint32_t scalar(uint32_t off) {
  off = __builtin_amdgcn_readfirstlane(off);
  asm("" : "+s"(off));
  return off;
}

template <int J>
__device__ __forceinline__ float step_scale(uint32_t quad) {
  return mxfp4::scale_operand((quad >> (8 * J)) & 255u);
}

// C consecutive outputs n .. of row m (C = 4 or 8: a lane's of one weight tile, or of a pair).
template <int C>
__device__ __forceinline__ void store(const Args& a, int m, int n, const float (&v)[C]) {
  if (m >= a.M || n >= a.N) return;
  if (a.part) {
    float* p = a.part + blockIdx.y * a.part_slice + static_cast<int64_t>(m) * a.pitch + n;   // pitch: whole tiles
#pragma unroll
    for (int i = 0; i < C; i += 4) *reinterpret_cast<f32x4_t*>(p + i) = f32x4_t{v[i], v[i + 1], v[i + 2], v[i + 3]};
    return;
  }
  uint16_t* o = a.y + static_cast<int64_t>(m) * a.ldy + n;
  uint32_t w[C / 2];
#pragma unroll
  for (int i = 0; i < C / 2; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  if (n + C <= a.N && (reinterpret_cast<uintptr_t>(o) & (2 * C - 1)) == 0) {
    if constexpr (C == 8) *reinterpret_cast<u32x4_t*>(o) = u32x4_t{w[0], w[1], w[2], w[3]};
    else *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (n + i < a.N) o[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
  }
}

// The outputs of a wave's tiles (column tiles from t0 on, rows from m on), lane (g, l16).
template <int NT>
__device__ __forceinline__ void store_row(const Args& a, int m, int t0, int g, const f32x4_t (&acc)[NT]) {
#pragma unroll
  for (int nt = 0; nt < NT; nt += 2) {
    if constexpr (NT % 2 == 0) {
      const f32x4_t lo = acc[nt], hi = acc[nt + 1];
      const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      store<8>(a, m, static_cast<int>(mxfp4::weight_row(t0 + nt, 4 * g)), v);
    } else {
      const float v[4] = {acc[0][0], acc[0][1], acc[0][2], acc[0][3]};
      store<4>(a, m, static_cast<int>(mxfp4::weight_row(t0, 4 * g)), v);
    }
  }
}

// Block `id` of a grid of mblocks x nblocks.  Consecutive ids go to the eight XCDs in turn, each with an L2 of its
// own: an XCD gets a run of blocks that lie next to one another, eight blocks of rows by as many of columns
// as it has, so that they share rows and weights there.
__device__ __forceinline__ void block_of(int id, int mblocks, int nblocks, int& mb, int& nb) {
  const int total = mblocks * nblocks;
  const int per = total / 8, extra = total % 8;
  const int xcd = id % 8, at = id / 8;
  const int t = xcd * per + (xcd < extra ? xcd : extra) + at;
  constexpr int kRun = 8;
  const int band = t / (kRun * nblocks);
  const int rows = mblocks - band * kRun < kRun ? mblocks - band * kRun : kRun;
  const int in = t - band * kRun * nblocks;
  mb = __builtin_amdgcn_readfirstlane(band * kRun + in % rows);   // divisions leave their results in vector registers
  nb = __builtin_amdgcn_readfirstlane(in / rows);
}

// X of the stream kernel: bf16 rows multiplied as they are, packed 4-bit rows, or bf16 rows quantised as they are read.
enum { kRows, kPacked, kQuantize };

// Few rows: every wave of a block has the same NT column tiles and its own K quads, reads X where it lies
// (caches serve it to the blocks) and the block adds the waves' sums in LDS, in order.  No barrier before that.
// kQuantize: a lane's 32 elements of a step are one block of the format, so that it finds their scale and codes by
// itself, some 55 instructions a step and row tile in every block, where that takes less than the launch that packs
// them (in_kernel).
template <int X, bool TAIL, int MT, int NT, int KW>
__global__ __launch_bounds__(64 * KW) void mxfp4_stream_kernel(const Args a) {
  __shared__ f32x4_t red[KW][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.x * NT, m0 = blockIdx.z * (MT * 16);
  const int ntiles = (a.N + 31) / 32 * 2, mtiles = (a.M + 15) / 16;
  const int qbeg = blockIdx.y * a.slice_quads;
  const int qend = qbeg + a.slice_quads < a.kquads ? qbeg + a.slice_quads : a.kquads;

  const uint8_t* wt[NT];
  const uint32_t* wsc[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    int t = t0 + nt;
    t = t < ntiles ? t : ntiles - 1;   // tiles past the weight: computed, not stored
    wt[nt] = a.w + static_cast<int64_t>(t) * a.kquads * (4 * kTile) + lane * 16;
    wsc[nt] = a.ws + static_cast<int64_t>(t) * a.kquads * 64 + lane;
  }
  const uint16_t* xr[MT];
  const uint8_t* xt[MT];
  const uint32_t* xsc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if constexpr (X == kPacked) {
      int t = m0 / 16 + mt;
      t = t < mtiles ? t : mtiles - 1;
      xt[mt] = a.xt + static_cast<int64_t>(t) * a.kquads * (4 * kTile) + lane * 16;
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
    u32x4_t w[4][NT];
    uint32_t sw[NT], sx[MT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sw[nt] = wsc[nt][q * 64];
    if constexpr (X == kPacked) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sx[mt] = xsc[mt][q * 64];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        w[j][nt] = *reinterpret_cast<const u32x4_t*>(wt[nt] + (static_cast<int64_t>(4 * q + j)) * kTile);
    // X of the whole quad too before anything waits: step by step, each would wait for the caches' latency.
    u32x4_t xv[4][MT][X == kPacked ? 1 : 4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (X == kPacked) {
          xv[j][mt][0] = *reinterpret_cast<const u32x4_t*>(xt[mt] + (static_cast<int64_t>(4 * q + j)) * kTile);
        } else {
          const int k = q * kQuad + j * kStep + 32 * g;
          const bool live = !TAIL || k < a.K;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            xv[j][mt][i] = *reinterpret_cast<const u32x4_t*>(xr[mt] + (live ? k : 0) + 8 * i);
            if (TAIL && !live) xv[j][mt][i] = u32x4_t{0, 0, 0, 0};
          }
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    auto step = [&](auto J) {
      constexpr int j = J.value;
      if constexpr (X == kRows) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float s = step_scale<j>(sw[nt]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const u32x4_t b = mxfp4::bf16_of(w[j][nt][i], s);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = mfma_bf16(b, xv[j][mt][i], acc[mt][nt]);
          }
        }
        return;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if constexpr (X == kPacked) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = mfma_fp4<j>(w[j][nt], sw[nt], xv[j][mt][0], sx[mt], acc[mt][nt]);
        } else {
          const uint32_t s = mxfp4::scale_byte(mxfp4::amax_bits(xv[j][mt]));
          const u32x4_t c = {mxfp4::codes_of<false>(xv[j][mt][0], s), mxfp4::codes_of<false>(xv[j][mt][1], s),
                             mxfp4::codes_of<false>(xv[j][mt][2], s), mxfp4::codes_of<false>(xv[j][mt][3], s)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = mfma_fp4<j, 0>(w[j][nt], sw[nt], c, s, acc[mt][nt]);
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
  constexpr int kSide = NT % 2 == 0 ? 2 : 1;   // tiles side by side that a wave adds and stores
  for (int p = wave; p < MT * NT / kSide; p += KW) {
    const int mt = p / (NT / kSide), nt = p % (NT / kSide) * kSide;
    f32x4_t s[kSide];
#pragma unroll
    for (int i = 0; i < kSide; ++i) {
      s[i] = red[0][mt * NT + nt + i][lane];
#pragma unroll
      for (int k = 1; k < KW; ++k) s[i] += red[k][mt * NT + nt + i][lane];
    }
    store_row<kSide>(a, m0 + mt * 16 + l16, t0 + nt, g, s);
  }
}

// Between two scheduling barriers: MFMAS products with VALUS conversions, READS and WRITES of LDS and LOADS of global
// memory spread among them, reads with the first products (they are needed first), the rest with the last.
template <int MFMAS, int VALUS, int READS, int WRITES, int LOADS>
__device__ __forceinline__ void spread() {
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    auto share = [&](int n) { return (i + 1) * n / MFMAS - i * n / MFMAS; };
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i < READS) __builtin_amdgcn_sched_group_barrier(0x100, (READS + MFMAS - 1) / MFMAS, 0);
    if (VALUS) __builtin_amdgcn_sched_group_barrier(0x002, (VALUS + MFMAS - 1) / MFMAS, 0);
    if (share(WRITES)) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
    if (share(LOADS)) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// 16-byte reads of a wave go to the 64 LDS banks in four groups of lanes, of which the first is 0-3, 12-15 and
// 20-27: with this key the operand reads (16 rows, one chunk of each of four blocks) touch each bank once a group, as
// consecutive lanes' reads do (5.5 cycles a read; keys of r alone, r % 8 or r % 4: 9.1, no key: 33).  A store of
// a row's 16 chunks touches each bank once with any key.
__device__ __forceinline__ int chunk_key(int r) { return (r >> 2) ^ ((r & 3) << 2); }

constexpr int kMostTiles = 10;   // row tiles of a block of 4-bit rows, at most

// Many rows: a block has WM x WN waves, a wave MT x NT tiles of 16 x 16.  gridDim.y blocks split K.
//
// K goes in stages: 128 elements of bf16 rows, a quad of 512 of 4-bit ones, 4 KB of LDS a row tile in both, and four
// operands (of 32 or 128 elements) a stage.  X goes through LDS, three stages' buffers: in stage s, behind its
// barrier, stage s + 2 is stored (loaded from global memory since stage s - 2) and s + 1 is complete, so
// that the first operand of s + 1 is read before the next barrier and the matrix cores have work on both sides of
// it.  Every wave loads its weight tiles straight into registers, 512 elements ahead, and with bf16 rows converts
// an operand while the one before it is multiplied.  LDS reads and stores, loads and conversions lie among the
// products (spread): with those of X together behind the barrier, no wave multiplied meanwhile, 41 us for 38.7 at
// 160 x 28672 x 4096, 165 for 162 at 2000 x 4096 x 14336 (a call of that takes 166, 1.41 PFLOP/s).
//
// With 4-bit rows a block takes the tiles blockIdx.x, blockIdx.x + gridDim.x, ... .  Loads run into the next tile (its
// first stages behind this one's last), so that between tiles nothing waits but the stores: 4093 x 28672 x 4096, 14
// tiles a CU, took 304 us for 347 with a block for each tile, and takes 285 now (3.4 PFLOP/s).  The launch gives a block
// more than one only where stages come in pairs, four or more.  (bf16 rows: the addresses of a next tile do not fit
// beside the operands of the widest tile.)
//   LDS: bf16 rows of 256 bytes, 16-byte chunk c of row r at place c ^ chunk_key(r % 16); 4-bit tiles as they are.
// Two waves a SIMD at least: above 256 registers a CU holds one four-wave block, 394 us there for 327.
//
// Scalar addresses: the tiles of a wave, or of a block's X, lie one row of tiles apart, so that a load costs two scalar
// additions (ten operations where each tile had its own bound: 294 us for 285 on the same).  The packed rows are
// therefore followed by room for what the last block reads past them.
template <bool A4, bool TAIL, int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void mxfp4_tile_kernel(const Args a) {
  constexpr int kThreads = 64 * WM * WN;
  constexpr int kTiles = MT * WM;                      // row tiles of the block
  constexpr int kChunks = kTiles * 256;                // 16-byte chunks of X in a stage
  constexpr int kRounds = (kChunks + kThreads - 1) / kThreads;
  static_assert(WM * WN % 4 == 0, "a wave's chunks of 4-bit rows lie in one tile");
  static_assert(!A4 || (kChunks % kThreads == 0 && kTiles <= kMostTiles),
                "4-bit rows are read in whole tiles, up to the padding");
  constexpr int kBuf = kRounds * kThreads;
  __shared__ u32x4_t xs[3 * kBuf];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int l16 = lane & 15, g = lane >> 4;
  const int mblocks = (a.M + 16 * kTiles - 1) / (16 * kTiles), nblocks = (a.N + 16 * NT * WN - 1) / (16 * NT * WN);
  const int total = mblocks * nblocks;
  int id = blockIdx.x, mb, nb;
  block_of(id, mblocks, nblocks, mb, nb);
  const int ntiles = (a.N + 31) / 32 * 2;
  const int qbeg = blockIdx.y * a.slice_quads;
  const int qend = qbeg + a.slice_quads < a.kquads ? qbeg + a.slice_quads : a.kquads;
  const int ksteps = (a.K + kStep - 1) / kStep;
  const int nsteps = (4 * qend < ksteps ? 4 * qend : ksteps) - 4 * qbeg;
  const int last = (A4 ? qend - qbeg : nsteps) - 1;
  // Whole quads, zeros behind the last step: stages that may be skipped are waited for as if they had been (widest
  // tile 716 us for 669 at 4093 x 28672 x 4096).  With the zeros' own test the widest tile spills, and skips.
  constexpr bool kWhole = !A4 && (!TAIL || MT * NT <= 10);
  const int nst = kWhole ? 4 * (qend - qbeg) : last + 1;

  // Where the loads are, at the first of the tiles; each of these moves to the next tile as its own run ahead passes
  // this tile's last stage.
  const uint8_t *w_at, *sw_at, *sx_at, *x_at;
  const uint32_t row_bytes = a.kquads * (4 * kTile), scale_bytes = a.kquads * 256;   // from a tile to the next
  const uint16_t* x_base;                  // bf16: the tile's first row; the thread's chunks of X (round r, chunk id
  uint32_t x_off[kRounds];                 // r * kThreads + threadIdx.x) in bytes behind it: at most 160 rows of 2^22
  const int xk = (threadIdx.x & 15) * 8;   // and their first element within a step
  static_assert(NT <= 2 && (NT == 2 || !A4), "a wave's weight tiles are all of the weight or none");
  auto first_tile = [&](int nb) {          // tiles past the weight: the last ones instead, computed and not stored
    const int t = (nb * WN + wn) * NT;
    return t < ntiles ? t : ntiles - NT;
  };
  auto weights_of = [&](int nb) { w_at = a.w + (static_cast<int64_t>(first_tile(nb)) * a.kquads + qbeg) * (4 * kTile); };
  auto scales_of = [&](int mb, int nb) {
    sw_at = reinterpret_cast<const uint8_t*>(a.ws) + (static_cast<int64_t>(first_tile(nb)) * a.kquads + qbeg) * 256;
    if constexpr (A4)
      sx_at = reinterpret_cast<const uint8_t*>(a.xs) + (static_cast<int64_t>((mb * WM + wm) * MT) * a.kquads + qbeg) * 256;
  };
  auto rows_of = [&](int mb) {
    if constexpr (A4) {                    // a wave's chunks of a round lie in one tile
      x_at = a.xt + (static_cast<int64_t>(mb * kTiles + wave / 4) * a.kquads + qbeg) * (4 * kTile);
    } else {
      const int m0 = mb * kTiles * 16;
      x_base = a.x + static_cast<int64_t>(m0) * a.ldx + qbeg * kQuad;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int c = r * kThreads + threadIdx.x;
        int m = c / 16;
        m = m < a.M - m0 ? m : a.M - m0 - 1;   // rows past the last repeat it, and are not stored
        x_off[r] = 2 * (static_cast<uint32_t>(m) * static_cast<uint32_t>(a.ldx) + xk);
      }
    }
  };
  rows_of(mb);
  weights_of(nb);
  scales_of(mb, nb);
  // TAIL: the bytes by which the last step's chunks lie past the row's end and are moved back, to be stored as zeros.
  const uint32_t past = TAIL && qbeg * kQuad + last * kStep + xk >= a.K ? 2 * xk : 0;
  u32x4_t xq[2][kRounds];
  auto load_x = [&](int s, u32x4_t (&v)[kRounds]) {
    s = s < last ? s : last;               // stages past the last repeat it, so that no load is conditional
    if constexpr (A4) {
      const uint8_t* at = x_at + scalar(s * (4 * kTile));
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        v[r] = reinterpret_cast<const u32x4_t*>(at)[threadIdx.x & 255];
        at += WM * WN / 4 * row_bytes;
      }
    } else {
      const uint8_t* at = reinterpret_cast<const uint8_t*>(x_base) + scalar(2 * s * kStep);
      const uint32_t back = TAIL && s == last ? past : 0;   // of the chunk's own 2 * xk
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        asm volatile("" : "+v"(x_off[r]));   // 32 bits beside a scalar base: extended outside the loop it would be 64
        v[r] = *reinterpret_cast<const u32x4_t*>(at + (x_off[r] - back));
      }
    }
  };
  static_assert(kThreads % 256 == 0, "a thread's chunks have one key");
  const int place = A4 ? threadIdx.x : (threadIdx.x & ~15) | ((threadIdx.x & 15) ^ chunk_key((threadIdx.x >> 4) & 15));
  auto store_x = [&](int s, int buf, const u32x4_t (&v)[kRounds]) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      u32x4_t t = v[r];
      if (TAIL && (s > last || (s == last && past))) t = u32x4_t{0, 0, 0, 0};
      xs[buf + r * kThreads + place] = t;
    }
  };
  const int key = chunk_key(l16);
  auto frag = [&](int buf, int i, u32x4_t (&f)[MT]) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      f[mt] = xs[buf + (A4 ? ((wm * MT + mt) * 4 + i) * 64 + lane : ((wm * MT + mt) * 16 + l16) * 16 + ((4 * g + i) ^ key))];
  };
  u32x4_t w[4][NT];                        // bf16: stages s .. s + 3; 4-bit: the stage's four steps
  auto load_w = [&](int u, u32x4_t (&v)[NT]) {
    const uint8_t* at = w_at + scalar(u * kTile);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      v[nt] = reinterpret_cast<const u32x4_t*>(at)[lane];
      at += row_bytes;
    }
  };
  // Scales of even and odd quads: a register that is copied waits for its load, and that for all loads before it.
  uint32_t sw[2][NT], sx[2][MT];
  const int lastq = qend - qbeg - 1;
  auto load_scales = [&](auto P, int q) {
    const uint32_t off = scalar((q < lastq ? q : lastq) * 256);
    const uint8_t* at = sw_at + off;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sw[P.value][nt] = reinterpret_cast<const uint32_t*>(at)[lane];
      at += scale_bytes;
    }
    if constexpr (A4) {
      at = sx_at + off;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        sx[P.value][mt] = reinterpret_cast<const uint32_t*>(at)[lane];
        at += scale_bytes;
      }
    }
  };
  constexpr std::integral_constant<int, 0> kEven{};
  constexpr std::integral_constant<int, 1> kOdd{};

  f32x4_t acc[MT][NT];
  {
    u32x4_t xa[kRounds], xb[kRounds];       // everything in flight before the first wait
    load_x(0, xa);
    load_scales(kEven, 0);
    load_w(0, w[0]);
    load_x(1, xb);
#pragma unroll
    for (int j = 1; j < 4; ++j) load_w(j, w[j]);
    load_x(2, xq[0]);
    load_x(3, xq[1]);
    __builtin_amdgcn_sched_barrier(0);
    store_x(0, 0, xa);
    store_x(1, kBuf, xb);
  }
  __syncthreads();
  u32x4_t f0[MT], f1[MT];
  frag(0, 0, f0);
  int cur = 0, nxt = kBuf, far = 2 * kBuf;   // buffers of stages s, s + 1, s + 2
  auto rotate = [&]() {
    const int t = cur;
    cur = nxt;
    nxt = far;
    far = t;
  };
  int mb_next, nb_next;               // the next tile, if there is one
  bool more = false;
  // X of stage s + 4, of this tile or the next (stages come in pairs where there is one).
  auto rows_ahead = [&](auto P, int s) {   // P: s % 2
    if (A4 && P.value == 0 && s + 4 == nst) rows_of(mb_next);
    load_x(s + 4 < nst || !more ? s + 4 : s + 4 - nst, xq[P.value]);
  };
  u32x4_t b0[NT], b1[NT];
  auto weights = [&](auto J, const uint32_t (&sc)[NT], int i, u32x4_t (&b)[NT]) {
    constexpr int j = J.value;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) b[nt] = mxfp4::bf16_of(w[j][nt][i], step_scale<j>(sc[nt]));
  };
  if constexpr (!A4) weights(std::integral_constant<int, 0>{}, sw[0], 0, b0);
  for (;;) {
    int id_next = id;
    if constexpr (A4) {
      id_next = id + static_cast<int>(gridDim.x) < total ? id + static_cast<int>(gridDim.x) : id;
      block_of(id_next, mblocks, nblocks, mb_next, nb_next);
      more = id_next != id;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if constexpr (A4) {
      auto products = [&](auto P, auto J, const u32x4_t (&f)[MT]) {
        constexpr int j = J.value, p = P.value;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = mfma_fp4<j>(w[j][nt], sw[p][nt], f[mt], sx[p][mt], acc[mt][nt]);
      };
      auto stage = [&](auto P, int s) {
        constexpr int p = P.value;
        constexpr std::integral_constant<int, p ^ 1> kOther{};
        const int un = s < last ? 4 * (s + 1) : more ? 0 : 4 * last;
        __syncthreads();
        if (s == last) scales_of(mb_next, nb_next);
        frag(cur, 1, f1);
        load_scales(kOther, s < last || !more ? s + 1 : 0);
        products(P, std::integral_constant<int, 0>{}, f0);
        spread<MT * NT, 0, MT, 0, MT + NT>();
        if (s == last) weights_of(nb_next);
        frag(cur, 2, f0);
        store_x(s + 2, far, xq[p]);
        load_w(un, w[0]);
        products(P, std::integral_constant<int, 1>{}, f1);
        spread<MT * NT, 0, MT, kRounds, NT>();
        frag(cur, 3, f1);
        rows_ahead(P, s);
        load_w(un + 1, w[1]);
        products(P, std::integral_constant<int, 2>{}, f0);
        spread<MT * NT, 0, MT, 0, kRounds + NT>();
        frag(nxt, 0, f0);
        load_w(un + 2, w[2]);
        products(P, std::integral_constant<int, 3>{}, f1);
        load_w(un + 3, w[3]);
        spread<MT * NT, 0, MT, 0, 2 * NT>();
        rotate();
      };
      for (int s = 0;;) {   // left at each stage's end: were stages skipped one by one, loads would be waited for
        stage(kEven, s);    // as if any of them had been
        if (++s >= nst) break;
        stage(kOdd, s);
        if (++s >= nst) break;
      }
    } else {
      // Products of one operand, the conversion of the next among them.
      auto products = [&](const u32x4_t (&f)[MT], const u32x4_t (&b)[NT]) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = mfma_bf16(b[nt], f[mt], acc[mt][nt]);
      };
      constexpr int kCvts = 4 * NT + 1;
      auto stage = [&](auto P, auto J, int s) {   // P: the quad's parity, J: the stage in it
        constexpr int j = J.value, p = P.value;
        constexpr std::integral_constant<int, j & 1> kSet{};
        __syncthreads();
        frag(cur, 1, f1);
        if constexpr (j == 0) load_scales(std::integral_constant<int, p ^ 1>{}, s / 4 + 1);
        weights(J, sw[p], 1, b1);
        products(f0, b0);
        spread<MT * NT, kCvts, MT, 0, j == 0 ? NT : 0>();
        frag(cur, 2, f0);
        store_x(s + 2, far, xq[kSet.value]);
        weights(J, sw[p], 2, b0);
        products(f1, b1);
        spread<MT * NT, kCvts, MT, kRounds, 0>();
        frag(cur, 3, f1);
        rows_ahead(kSet, s);
        weights(J, sw[p], 3, b1);
        products(f0, b0);
        spread<MT * NT, kCvts, MT, 0, kRounds>();
        frag(nxt, 0, f0);
        load_w(s - j < 4 * lastq ? s + 4 : 4 * lastq + j, w[j]);   // the next quad's: K is padded to whole ones
        if constexpr (j < 3) weights(std::integral_constant<int, (j + 1) & 3>{}, sw[p], 0, b0);
        else weights(std::integral_constant<int, 0>{}, sw[p ^ 1], 0, b0);
        products(f1, b1);
        spread<MT * NT, kCvts, MT, 0, NT>();
        rotate();
      };
      auto quad = [&](auto P, int s) {
        stage(P, std::integral_constant<int, 0>{}, s);
        if (kWhole || s + 1 < nst) stage(P, std::integral_constant<int, 1>{}, s + 1);
        if (kWhole || s + 2 < nst) stage(P, std::integral_constant<int, 2>{}, s + 2);
        if (kWhole || s + 3 < nst) stage(P, std::integral_constant<int, 3>{}, s + 3);
      };
      for (int s = 0;;) {
        quad(kEven, s);
        if ((s += 4) >= nst) break;
        quad(kOdd, s);
        if ((s += 4) >= nst) break;
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      store_row<NT>(a, ((mb * WM + wm) * MT + mt) * 16 + l16, (nb * WN + wn) * NT, g, acc[mt]);
    if (!more) return;
    id = id_next;
    mb = mb_next;
    nb = nb_next;
  }
}

// Rows of X to packed 4-bit tiles.  A block is a tile, a wave its block g of 32 elements, four lanes a row of it.
__global__ __launch_bounds__(256) void mxfp4_pack_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx, int M, int K,
                                                              int kquads, uint32_t* __restrict__ tiles,
                                                              uint8_t* __restrict__ scales) {
  const int u = blockIdx.x, t = blockIdx.y, g = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane >> 2, q = lane & 3;
  const int row = 16 * t + r;
  if (row >= M) return;
  const int k = u * kStep + 32 * g + 8 * q;
  uint32_t code = 0, s = 127;
  if (k < K) {   // the same for a block's four lanes
    const u32x4_t v[1] = {*reinterpret_cast<const u32x4_t*>(x + static_cast<int64_t>(row) * ldx + k)};
    s = mxfp4::scale_byte(group_max_u32<4>(mxfp4::amax_bits(v)));
    code = mxfp4::codes_of(v[0], s);
  }
  const int l = 16 * g + r;
  tiles[((static_cast<int64_t>(t) * 4 * kquads + u) * 64 + l) * 4 + q] = code;
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
  const float v[4] = {s.x, s.y, s.z, s.w};
  store<4>(a, static_cast<int>(m), n, v);
}

// ---- which kernel ------------------------------------------------------------------------------
// Tile kernels, smallest first: MT, NT, WM, WN; us before the first and behind the last product; us a stage with a
// block on every CU (bf16 rows; a stage of 512 elements of 4-bit ones).  Every tile and split of 20 to 4093 rows of
// seven sizes from 2048 x 2048 to 28672 x 4096 was timed in a graph, with the launch that adds slices.  bf16 rows: in
// 93 of 98 products the choice takes at most 8 % more than the best measured, at worst 26.9 us for 21.7 (512 x 2048 x
// 8192).  4-bit rows: in 35 of 77, the median 11 % more, at worst 19.5 us for 14.1 (the same size): the four-wave
// tile of 80 rows is rated too dear, 11.1 us chosen for its 9.4 at 160 x 4096 x 4096.
struct TileConfig {
  int mt, nt, wm, wn;
  float start, us, us4;
  int rows() const { return 16 * mt * wm; }
  int cols() const { return 16 * nt * wn; }
};
constexpr TileConfig kTile2x1{2, 1, 1, 4, 2.7f, 0.27f, 0.f}, kTile2x2{2, 2, 1, 4, 3.7f, 0.33f, 0.f},
    kTile4{4, 2, 1, 4, 4.4f, 0.50f, 0.f}, kTile5{5, 2, 1, 4, 4.8f, 0.68f, 1.30f}, kTile6{3, 2, 2, 4, 4.8f, 0.76f, 1.10f},
    kTile8{4, 2, 2, 4, 5.0f, 0.80f, 1.30f}, kTile10{5, 2, 2, 4, 7.0f, 1.08f, 1.65f},
    kTileWide{8, 2, 1, 8, 5.5f, 1.40f, 2.20f};
constexpr TileConfig kTiles[] = {kTile2x1, kTile2x2, kTile4, kTile5, kTile6, kTile8, kTile10, kTileWide};
constexpr int kFirstTile4 = 3;   // 4-bit rows: up to 64 go to the stream kernel

struct Plan {
  bool stream;
  int x;             // stream: kRows, kPacked, kQuantize
  int tile;          // else index in kTiles
  int mt, nt, kw;    // stream
  int ks, slice_quads;
  int rows_padded, pitch;
};

void split_k(Plan& p, int quads, int ks) {
  p.slice_quads = (quads + ks - 1) / ks;
  p.ks = (quads + p.slice_quads - 1) / p.slice_quads;
}

// Whether the stream kernel quantises X itself.  us in a graph, it / with the launch that packs (3 us more of the host's
// time where there is no graph): one row of 4096 x 4096 4.7 / 6.0, of 16384 x 2048 6.5 / 7.9, of 4096 x 14336
// 10.9 / 10.3, of 28672 x 4096 17.6 / 15.1, of 128256 x 4096 61 / 46; 8 rows 5.8 / 5.8, 7.0 / 7.4, 13.6 / 10.4,
// 16.2 / 15.3, 52 / 49; 16 rows of 2048 x 2048 4.7 / 4.9, of 4096 x 4096 7.1 / 5.9, of 4096 x 14336 18.5 / 10.7, of
// 28672 x 4096 18.6 / 15.6; for a consumer that adds slices, 16 of 2048 x 8192 5.2 / 3.5 and the launch's 2.  Each block of
// columns quantises the rows again, so that the widest and longest weights lose by the rule for up to eight rows,
// which does not look at them.
bool in_kernel(int M, int ntiles, int quads, bool partials) {
  return M <= 8 || (M <= 16 && ntiles <= 1024 && quads <= (partials ? 16 : 8));
}

// 4-bit rows: one block a CU, two of four waves, where a block's loads may run from one tile into the next.
bool persistent(bool a4, int ks, int quads) { return a4 && ks == 1 && quads % 2 == 0 && quads >= 4; }

// The plan for a product.  `partials`: a consumer adds the K slices.
Plan plan_for(int M, int N, int K, bool a4, bool partials) {
  Plan p{};
  const int mtiles = static_cast<int>(mxfp4::row_tiles(M)), quads = static_cast<int>(mxfp4::quads(K));
  const int ntiles = static_cast<int>(mxfp4::weight_tiles(N));
  p.rows_padded = mtiles * 16;
  p.pitch = ntiles * 16;
  if (mtiles <= (a4 ? 4 : 1)) {
    // Stream kernel.  Blocks enough for every CU first, then column tiles, for which X is read once.  us in a graph,
    // NT = 1, 2, 4: 16 bf16 rows of 4096 x 4096 6.6, 7.2, 8.6, of 6144 x 4096 10.4, 7.8, 9.0, of 28672 x 4096 32,
    // 25.5, 19.7; 5 rows of that 19.3, 18.5, 16.2; one 17.4, 17.1, 15.3, of 128256 x 4096 64, 57, 48 (up to four rows
    // take NT = 2 there).  Packed: 16 rows of 4096 x 4096 3.9, 4.3, 32 of 16384 x 2048 6.6, 6.2, 64 of 28672 x 4096
    // 24.5, 19.2, 17.0.  Eight waves where each has a quad.
    p.stream = true;
    p.x = !a4 ? kRows : in_kernel(M, ntiles, quads, partials) ? kQuantize : kPacked;
    p.mt = mtiles <= 2 ? mtiles : 4;
    if (p.x != kPacked) p.nt = ntiles >= 1024 && M > 4 ? 4 : ntiles >= 384 ? 2 : 1;
    else if (p.mt == 4) p.nt = ntiles >= 1408 ? 4 : ntiles >= 192 ? 2 : 1;
    else p.nt = ntiles >= 1024 ? 2 : 1;
    p.kw = p.nt == 4 || quads < 8 ? 4 : 8;
    int ks = 1;
    auto blocks = [&]() { return (ntiles + p.nt - 1) / p.nt; };
    if (p.x == kPacked) {
      if (partials)
        while (ks < 4 && ks * 2 * p.kw <= quads && 2 * ks * blocks() <= 512) ks *= 2;
    } else if (partials || (M > 8 && quads >= 16 && ntiles < 1024)) {
      // Slices instead of waves, and the tiles that leave blocks enough.  us for a consumer, against one slice: one
      // row of 4096 x 4096 4.5 / 4.3, of 2048 x 8192 4.3 / 5.1, 5 rows of 4096 x 14336 9.8 / 11.1, of 6144 x 4096 5.4
      // / 5.8, 16 of 4096 x 4096 5.4 / 6.8, of 2048 x 8192 5.7 / 10.3, of 4096 x 14336 11.9 / 17.6 (for these two a
      // launch that adds them pays as well: 7.7, 14.0).
      p.nt = M > 8 ? (ntiles >= 256 ? 4 : ntiles >= 128 ? 2 : 1) : ntiles >= 192 ? 2 : 1;
      p.kw = 4;
      while (ks < 4 && ks * 4 <= quads && ks * blocks() < (M > 8 ? 256 : 512)) ks *= 2;
    }
    split_k(p, quads, ks);
    return p;
  }
  // Tile kernels: the cheapest of all tiles and K splits by this estimate.  A round is a block on each of the 256 CUs; with
  // two four-wave blocks on a CU two rounds take the time of 1.45, and a stage takes less where CUs are free.  A
  // reduction costs a launch where no consumer does it, and its bytes either way.
  float best = 1e30f;
  for (int t = a4 ? kFirstTile4 : 0; t < static_cast<int>(sizeof(kTiles) / sizeof(kTiles[0])); ++t) {
    const TileConfig& c = kTiles[t];
    const int64_t blocks = static_cast<int64_t>((M + c.rows() - 1) / c.rows()) * ((ntiles * 16 + c.cols() - 1) / c.cols());
    for (int ks = 1; ks <= 16 && ks <= quads; ++ks) {
      Plan q = p;
      split_k(q, quads, ks);
      if (q.ks != ks) continue;
      const int64_t grid = blocks * ks, rounds = (grid + 255) / 256;
      if (ks > 1 && grid > 512) break;   // enough for every CU
      const float stages = a4 ? static_cast<float>(q.slice_quads) : 4.0f * q.slice_quads;
      const float share = grid < 256 ? static_cast<float>(grid) / 256.0f : 1.0f;
      const float block = c.start + stages * (a4 ? c.us4 * (0.4f + 0.6f * share) : c.us * (0.65f + 0.35f * share));
      float us = rounds * block;
      if (c.wm * c.wn == 4 && rounds > 1) us = (rounds + 1) / 2 * block * 1.45f;
      if (persistent(a4, ks, quads)) us -= c.start * (us / block - 1.0f);   // loads run into the next tile
      if (ks > 1) us += (partials ? 0.8f : 2.2f) + 0.7e-6f * ks * M * static_cast<float>(p.pitch);
      if (us < best) {
        best = us;
        p.tile = t;
        p.ks = q.ks;
        p.slice_quads = q.slice_quads;
      }
    }
  }
  return p;
}

// Row tiles of the packed X: what a tile kernel's last block reads past them is in the workspace, and not stored.
int64_t x_tiles(const Plan& p) { return p.rows_padded / 16 + (p.stream ? 0 : kMostTiles - 1); }

int64_t part_bytes(const Plan& p, bool partials) {
  return p.ks > 1 || partials ? int64_t{4} * p.ks * p.rows_padded * p.pitch : 0;
}

template <int X, bool TAIL, int MT, int NT>
void launch_stream(const Plan& p, const Args& a, hipStream_t s) {
  const dim3 grid((static_cast<int>(mxfp4::weight_tiles(a.N)) + NT - 1) / NT, p.ks, (a.M + 16 * MT - 1) / (16 * MT));
  if constexpr (NT < 4) {
    if (p.kw == 8) {
      hipLaunchKernelGGL((mxfp4_stream_kernel<X, TAIL, MT, NT, 8>), grid, dim3(512), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((mxfp4_stream_kernel<X, TAIL, MT, NT, 4>), grid, dim3(256), 0, s, a);
}

template <int X, bool TAIL, int MT>
void launch_stream_rows(const Plan& p, const Args& a, hipStream_t s) {
  if constexpr (X != kPacked || MT == 4) {
    if (p.nt == 4) return launch_stream<X, TAIL, MT, 4>(p, a, s);
  }
  if (p.nt == 2) launch_stream<X, TAIL, MT, 2>(p, a, s);
  else launch_stream<X, TAIL, MT, 1>(p, a, s);
}

unsigned tiles_of(const TileConfig& c, int M, int N) {
  return static_cast<unsigned>((M + c.rows() - 1) / c.rows()) * ((N + c.cols() - 1) / c.cols());
}

// Blocks along x of a tile kernel's grid.
unsigned tile_blocks(const TileConfig& c, const Plan& p, bool a4, int M, int N, int quads) {
  const unsigned tiles = tiles_of(c, M, N), slots = c.wm * c.wn == 4 ? 512 : 256;
  return persistent(a4, p.ks, quads) && tiles > slots ? slots : tiles;
}

template <bool A4, bool TAIL, int T>
void launch_tile(const Plan& p, const Args& a, hipStream_t s) {
  constexpr TileConfig c = kTiles[T];
  const unsigned grid = tile_blocks(c, p, A4, a.M, a.N, a.kquads);
  hipLaunchKernelGGL((mxfp4_tile_kernel<A4, TAIL, c.mt, c.nt, c.wm, c.wn>), dim3(grid, p.ks), dim3(64 * c.wm * c.wn), 0, s, a);
}

template <bool A4, bool TAIL>   // TAIL: K is not whole quads
void launch_tiles(const Plan& p, const Args& a, hipStream_t s) {
  switch (p.tile) {
    case 3: return launch_tile<A4, TAIL, 3>(p, a, s);
    case 4: return launch_tile<A4, TAIL, 4>(p, a, s);
    case 5: return launch_tile<A4, TAIL, 5>(p, a, s);
    case 6: return launch_tile<A4, TAIL, 6>(p, a, s);
    case 7: return launch_tile<A4, TAIL, 7>(p, a, s);
  }
  if constexpr (!A4) {
    if (p.tile == 0) return launch_tile<A4, TAIL, 0>(p, a, s);
    if (p.tile == 1) return launch_tile<A4, TAIL, 1>(p, a, s);
    return launch_tile<A4, TAIL, 2>(p, a, s);
  }
}

void launch_product(const Plan& p, const Args& a, bool a4, hipStream_t s) {
  if (p.stream) {
    const bool tail = a.K % kQuad != 0;
    if (p.x == kPacked) {
      if (p.mt == 1) launch_stream_rows<kPacked, false, 1>(p, a, s);
      else if (p.mt == 2) launch_stream_rows<kPacked, false, 2>(p, a, s);
      else launch_stream_rows<kPacked, false, 4>(p, a, s);
    } else if (p.x == kQuantize) {
      if (tail) launch_stream_rows<kQuantize, true, 1>(p, a, s);
      else launch_stream_rows<kQuantize, false, 1>(p, a, s);
    } else {
      if (tail) launch_stream_rows<kRows, true, 1>(p, a, s);
      else launch_stream_rows<kRows, false, 1>(p, a, s);
    }
  } else {
    if (a4) launch_tiles<true, false>(p, a, s);
    else if (a.K % kQuad) launch_tiles<false, true>(p, a, s);
    else launch_tiles<false, false>(p, a, s);
  }
}

constexpr int kMaxRow = 1 << 22;    // elements from one row of X to the next: 160 rows' bytes are counted in 32 bits
constexpr int kMaxRows = 1 << 19;   // the grids count row tiles in a dimension of 65535

const char* shape_error(int M, int N, int K) {
  if (M < 0 || N < 0 || K < 0) return "negative size";
  if (K % mxfp4::kBlock || (K == 0 && M && N)) return "K must be a positive multiple of 32";
  if (M > kMaxRows) return "M must be at most 2^19";
  if (N > (1 << 24) || K > kMaxRow) return "N must be at most 2^24 and K at most 2^22";
  return nullptr;
}

// The product; with `partials` every slice (also a single one) stays in the workspace as fp32.
int run(const void* x, int64_t ldx, const void* w, int M, int N, int K, int act4, void* y, int64_t ldy, void* workspace,
        size_t workspace_bytes, bool partials, coopt_stream_t stream, const char* who) {
  const char* bad = shape_error(M, N, K);
  if (!bad && M && N) {
    if (!x || !w || (!y && !partials)) bad = "null pointer";
    else if (!coopt::aligned16(x) || !coopt::aligned16(w)) bad = "x and w must be 16-byte aligned";
    else if (ldx < K || ldx % 8 || ldx > kMaxRow) bad = "row stride of x must be >= K, a multiple of 8, at most 2^22";
    else if (!partials && (ldy < N || (reinterpret_cast<uintptr_t>(y) & 1))) bad = "row stride of y must be >= N";
    else if (partials && N % 32) bad = "partial sums need N a multiple of 32";
  }
  if (bad) {
    coopt::set_error(std::string(who) + ": " + bad);
    return COOPT_EINVAL;
  }
  if (M == 0 || N == 0) return COOPT_OK;
  const Plan p = plan_for(M, N, K, act4 != 0, partials);
  const bool pack = act4 && p.x != kQuantize;
  const int64_t pb = part_bytes(p, partials), need = pb + (pack ? mxfp4::packed_bytes(x_tiles(p), K) : 0);
  if (need && (static_cast<int64_t>(workspace_bytes) < need || !workspace || !coopt::aligned16(workspace))) {
    coopt::set_error(std::string(who) + ": workspace smaller than required (or misaligned)");
    return COOPT_EWORKSPACE;
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.w = static_cast<const uint8_t*>(w);
  a.ws = reinterpret_cast<const uint32_t*>(a.w + mxfp4::tile_bytes(mxfp4::weight_tiles(N), K));
  a.M = M; a.N = N; a.K = K;
  a.kquads = static_cast<int>(mxfp4::quads(K));
  a.slice_quads = p.slice_quads;
  a.y = static_cast<uint16_t*>(y);
  a.ldy = ldy;
  a.part = pb ? static_cast<float*>(workspace) : nullptr;
  a.part_slice = static_cast<int64_t>(p.rows_padded) * p.pitch;
  a.pitch = p.pitch;
  if (pack) {
    uint8_t* tiles = static_cast<uint8_t*>(workspace) + pb;
    uint8_t* scales = tiles + mxfp4::tile_bytes(x_tiles(p), K);
    a.xt = tiles;
    a.xs = reinterpret_cast<const uint32_t*>(scales);
    hipLaunchKernelGGL(mxfp4_pack_rows_kernel, dim3(4 * a.kquads, static_cast<unsigned>(mxfp4::row_tiles(M))), dim3(256), 0, s,
                       a.x, ldx, M, K, a.kquads, reinterpret_cast<uint32_t*>(tiles), scales);
  }
  launch_product(p, a, act4 != 0, s);
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
  const Plan p = plan_for(M, N, K, act4 != 0, partials != 0);
  return static_cast<size_t>(part_bytes(p, partials != 0) +
                             (act4 && p.x != kQuantize ? mxfp4::packed_bytes(x_tiles(p), K) : 0));
}

extern "C" int coopt_mxfp4_linear_split(int M, int N, int K, int act4, int* ks, int* rows_padded) {
  coopt::clear_error();
  COOPT_REQUIRE(ks && rows_padded, "null output pointer");
  COOPT_REQUIRE(!shape_error(M, N, K) && M > 0 && N > 0, "unsupported shape");
  const Plan p = plan_for(M, N, K, act4 != 0, true);
  *ks = p.ks;
  *rows_padded = p.rows_padded;
  return COOPT_OK;
}

extern "C" int coopt_mxfp4_linear_plan(int M, int N, int K, int act4, int partials, int* plan) {
  coopt::clear_error();
  COOPT_REQUIRE(plan, "null output pointer");
  COOPT_REQUIRE(!shape_error(M, N, K) && M > 0 && N > 0, "unsupported shape");
  const Plan p = plan_for(M, N, K, act4 != 0, partials != 0);
  if (p.stream) {
    const int v[8] = {0, p.x, p.mt, p.nt, 1, p.kw, p.ks, 1};
    std::copy(v, v + 8, plan);
  } else {
    const TileConfig& c = kTiles[p.tile];
    const unsigned tiles = tiles_of(c, M, N);
    const unsigned grid = tile_blocks(c, p, act4 != 0, M, N, static_cast<int>(mxfp4::quads(K)));
    const int v[8] = {1, act4 ? kPacked : kRows, c.mt, c.nt, c.wm, c.wn, p.ks, static_cast<int>((tiles + grid - 1) / grid)};
    std::copy(v, v + 8, plan);
  }
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
