// Large exact products with an epilogue, on CTA pairs.
//
// Arithmetic: f16 has TF32's 11 significant bits at twice its rate, but few
// exponents. Every 128 of K of an operand's row are scaled by a power of two that
// brings the largest of them to [2^14, 2^15) (exact), then x 2^e = hi + lo with
// hi = f16(x 2^e), lo = f16(x 2^e - hi): 22 bits of x, or 2^-39 of the chunk's
// largest entry where lo leaves f16's range. C = Al Bh + Ah Bl + Ah Bh; Al Bl
// (2^-22) is left out. (The splitting into halves with scaling is that of H.
// Ootomo and R. Yokota, "Recovering single precision accuracy from Tensor Cores
// while surpassing the FP32 theoretical peak performance", IJHPCA 2022.) The
// chunk is also what one TMEM accumulation covers: 24 UMMAs, few enough that the
// tensor core's truncating sums stay below f32's own error, and the epilogue
// warps undo both scales as they add the chunk to the running sum in registers,
// so the scales cost one multiplication per value and no pass over the data.
//
// The copies are made by one pass over 128 x 128 tiles (split_kernel), from a
// matrix or straight from what would have been written for it (dz from dc and z), by
// rows, transposed, or both, so that every product reads K-major operands; the
// loss's logits leave their product as a copy. The passes are bound by HBM: 4 bytes
// read per value (8 for dz), 4 written per copy (8192 x 5632 and 5632 x 2048 in one
// launch 77 us, 6.0 TB/s; dz of 8192 x 5632 by rows and transposed with the column sums
// 148 us, 5.0 TB/s).
//
// Measured, copies aside: 8192 x 2048 x 5632 366 us by itself at 1.5 GHz (516 TFLOP/s of
// the product, 1,550 of f16 executed; the 3xTF32 products of gemm.cu take 730 us), 429 us
// in a loop of backward calls, where the power cap leaves 1.40 GHz (1,322 executed, 93% of
// what the library's bf16 product sustains under the cap); 8192 x 1024 -> 2816 with GELU
// and z kept 124 us by itself, 129 in a loop. The tensor pipe is busy 88 to 96% of the
// cycles of a long product, 69% of the loss's logits of 1024 of K, whose epilogue is the
// longest. The one-pass TF32 form (Tf32Feed) 8192 x 2048 x 5632 273 us by itself, 282 to
// 290 in a loop.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <type_traits>

#include "device.h"
#include "gemm.h"
#include "linear.h"
#include "linear_epi.cuh"
#include "ptx.cuh"
#include "tma.h"

namespace mm {
namespace {

// ------------------------------------------------------------------ split
constexpr int kTile = 128;
constexpr int kSplitWarps = 16;
constexpr int kSplitSums = kSplitWarps * kTile * 4;  // the warps' column sums
constexpr int kSplitSmem = kSplitSums + kTile * kTile * 4;

// The power of two for a chunk whose largest magnitude has the bits m: [2^14, 2^15)
// after scaling; 1 for infinities and NaN, and clamped so that its inverse is a
// normal number.
__device__ __forceinline__ float chunk_scale(uint32_t m, float* inv) {
  const int ex = static_cast<int>(m >> 23);
  int se = ex == 255 ? 127 : 268 - max(ex, 1);
  se = min(se, 253);
  *inv = __uint_as_float(static_cast<uint32_t>(254 - se) << 23);
  return __uint_as_float(static_cast<uint32_t>(se) << 23);
}

// Magnitudes compare as their bits do (a NaN above everything).
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// hi and lo of a pair of scaled values
__device__ __forceinline__ void halves(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Sources: begin once, then load of a row's four columns.
struct MatrixSource {
  SplitMatrix a;
  __device__ __forceinline__ void begin() {}
  __device__ __forceinline__ float4 load(long long row, int col, int cols) const {
    const float4 v = load_quad(a.x + row * a.ld, col, cols);
    if (a.targets) {
      const int t = a.targets[row];
      if (t < 0 || t >= a.vocab) return make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return v;
  }
};
struct BackwardSource {
  SplitBackward a;
  uint64_t seed, offset;
  __device__ __forceinline__ void begin() {
    seed = a.drop.rng ? a.drop.rng[0] : 0;
    offset = a.drop.rng ? a.drop.rng[1] : 0;
  }
  __device__ __forceinline__ float4 load(long long row, int col, int cols) const {
    float4 g = load_quad(a.dc + row * a.lddc, col, cols);
    if (a.drop.rng) g = dropout_quad(g, a.drop, seed, offset, row, col >> 2);
    if (a.act != kActNone) {
      const float4 v = load_quad(a.z + row * a.ldz, col, cols);
      g.x *= activate_slope(v.x, a.act); g.y *= activate_slope(v.y, a.act);
      g.z *= activate_slope(v.z, a.act); g.w *= activate_slope(v.w, a.act);
    }
    return g;
  }
};
struct CopySource {  // a copy's values again, scale and all
  SplitCopy a;
  __device__ __forceinline__ void begin() {}
  __device__ __forceinline__ float4 load(long long row, int col, int) const {  // zeros past k, as the copy has
    const uint16_t* p = a.data + row * a.row_halves() + (col >> 7) * 256 + ((col >> 6) & 1) * 128 + (col & 63);
    const uint2 hi = *reinterpret_cast<const uint2*>(p), lo = *reinterpret_cast<const uint2*>(p + 64);
    const float inv = a.inv[(col >> 7) * a.inv_ld() + row];
    auto sum = [&](uint32_t h, uint32_t l) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
      const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&l));
      return make_float2((x.x + y.x) * inv, (x.y + y.y) * inv);
    };
    const float2 v = sum(hi.x, lo.x), w = sum(hi.y, lo.y);
    return make_float4(v.x, v.y, w.x, w.y);
  }
};

// The columns of a tile of 128 rows x W in shared memory, quad q of row r at quad
// r W / 4 + (q ^ (r / 8 & 7)): a warp takes a quad of columns, lane (c, j) column c and
// rows 8 j.. of each 64 (eight j in eight different bank groups, so neither side has
// conflicts), which are the 16 bytes of hi and of lo that it stores.
template <int W, int WARPS>
__device__ __forceinline__ void split_columns(const float* tile, int cols, const SplitCopy& by_cols, int tile_r,
                                              int c0) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, c = lane & 3, j = lane >> 2;
#pragma unroll 1
  for (int q = warp; q < W / 4 && c0 + 4 * q < cols; q += WARPS) {
    const float* t = tile + 4 * (q ^ j) + c;
    float v[16];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // row 64 (i / 8) + 8 j + i % 8: r / 8 & 7 is j
      v[i] = t[(64 * (i / 8) + 8 * j + i % 8) * W];
      m = max(m, magnitude(v[i]));
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    float inv;
    const float s = chunk_scale(m, &inv);
    const int mine = c0 + 4 * q + c;
    if (mine >= cols) continue;
    uint16_t* out = by_cols.data + mine * by_cols.row_halves() + tile_r * 256ll + 8 * j;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) halves(v[8 * h + 2 * i] * s, v[8 * h + 2 * i + 1] * s, hi[i], lo[i]);
      *reinterpret_cast<uint4*>(out + 128 * h) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(out + 128 * h + 64) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (j == 0) by_cols.inv[tile_r * by_cols.inv_ld() + mine] = inv;
  }
}

// One 128 x 128 tile per block. By rows: a warp per row (8 each), a lane four columns. By
// columns: through shared memory. Two blocks of 16 warps on an SM keep more loads in
// flight than three of eight (8192 x 5632 with 5632 x 2048 by columns 77 us against 83, dz
// by rows and columns 148 against 158; by rows alone 36.5 against 35.2).
template <class Source>
__device__ __forceinline__ void split_tile(Source& src, int rows, int cols, const SplitCopy& by_rows,
                                           const SplitCopy& by_cols, float* part, int tile_r, int tile_c) {
  extern __shared__ __align__(16) float split_smem[];
  float* sums = split_smem;  // [warps][128]
  float4* tile = reinterpret_cast<float4*>(split_smem + kSplitWarps * kTile);  // where the columns are wanted
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int r0 = tile_r * kTile, c0 = tile_c * kTile;
  const int col = c0 + 4 * lane;
  src.begin();
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int U = 4;  // rows of a warp in flight
#pragma unroll 1
  for (int i0 = 0; i0 < kTile / kSplitWarps; i0 += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = r0 + kSplitWarps * (i0 + u) + warp;
      v[u] = row < rows && col < cols ? src.load(row, col, cols) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = kSplitWarps * (i0 + u) + warp;
      const long long row = r0 + r;
      if (by_cols.data) tile[r * 32 + (lane ^ ((r >> 3) & 7))] = v[u];
      if (part) {
        sum.x += v[u].x; sum.y += v[u].y; sum.z += v[u].z; sum.w += v[u].w;
      }
      if (by_rows.data) {
        const uint32_t m = __reduce_max_sync(
            0xffffffffu, max(max(magnitude(v[u].x), magnitude(v[u].y)), max(magnitude(v[u].z), magnitude(v[u].w))));
        if (row < rows) {
          float inv;
          const float s = chunk_scale(m, &inv);
          uint2 hi, lo;
          halves(v[u].x * s, v[u].y * s, hi.x, lo.x);
          halves(v[u].z * s, v[u].w * s, hi.y, lo.y);
          uint16_t* out =
              by_rows.data + row * by_rows.row_halves() + tile_c * 256ll + (lane / 16) * 128 + (lane % 16) * 4;
          *reinterpret_cast<uint2*>(out) = hi;
          *reinterpret_cast<uint2*>(out + 64) = lo;
          if (lane == 0) by_rows.inv[tile_c * by_rows.inv_ld() + row] = inv;
        }
      }
    }
  }
  if (part) {  // column sums over the tile's rows, warps in order
    reinterpret_cast<float4*>(sums + warp * kTile)[lane] = sum;
    __syncthreads();
    if (threadIdx.x < kTile && c0 + static_cast<int>(threadIdx.x) < cols) {
      float s = 0.0f;
      for (int k = 0; k < kSplitWarps; ++k) s += sums[k * kTile + threadIdx.x];
      part[static_cast<long long>(tile_r) * cols + c0 + threadIdx.x] = s;
    }
  }
  if (!by_cols.data) return;
  __syncthreads();
  split_columns<kTile, kSplitWarps>(split_smem + kSplitWarps * kTile, cols, by_cols, tile_r, c0);
}

template <class Source>
__global__ void __launch_bounds__(32 * kSplitWarps, 2) split_kernel(Source src, int rows, int cols, SplitCopy by_rows,
                                                       SplitCopy by_cols, float* part) {
  after_previous();
  let_next();
  const int tc = (cols + kTile - 1) / kTile, t = static_cast<int>(blockIdx.x);
  split_tile(src, rows, cols, by_rows, by_cols, part, t / tc, t % tc);
}

// The transposed copy alone: 128 x 64 tiles, whose half of the shared memory lets six
// blocks share an SM (a block loads, then converts, so it takes several to keep loads in
// flight). 2816 x 32000 of the loss's gradient, 8 bytes a value: 148 us, 4.9 TB/s (157
// with five blocks, 200 with three and 128 x 128 tiles).
constexpr int kHalf = 64;
template <class Source>
__global__ void __launch_bounds__(256, 6) split_transposed_kernel(Source src, int rows, int cols, SplitCopy by_cols) {
  after_previous();
  let_next();
  __shared__ __align__(16) float4 tile[kTile * kHalf / 4];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int tc = (cols + kHalf - 1) / kHalf, tile_r = static_cast<int>(blockIdx.x) / tc;
  const int c0 = (static_cast<int>(blockIdx.x) - tile_r * tc) * kHalf;
  const int q = lane % 16, col = c0 + 4 * q;
  src.begin();
#pragma unroll 1
  for (int i0 = 0; i0 < kTile / 16; i0 += 4) {
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // two rows a warp
      const long long row = static_cast<long long>(tile_r) * kTile + 16 * (i0 + u) + 2 * warp + lane / 16;
      v[u] = row < rows && col < cols ? src.load(row, col, cols) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 16 * (i0 + u) + 2 * warp + lane / 16;
      tile[r * (kHalf / 4) + (q ^ ((r >> 3) & 7))] = v[u];
    }
  }
  __syncthreads();
  split_columns<kHalf, 8>(reinterpret_cast<const float*>(tile), cols, by_cols, tile_r, c0);
}

// Two matrices in one launch (a product's operands): the first's tiles, then the second's.
struct MatrixJob {
  MatrixSource src;
  int rows, cols;
  SplitCopy by_rows, by_cols;
};
__global__ void __launch_bounds__(32 * kSplitWarps, 2) split_two_kernel(MatrixJob x, MatrixJob y) {
  after_previous();
  let_next();
  const int tiles_x = ((x.rows + kTile - 1) / kTile) * ((x.cols + kTile - 1) / kTile);
  const bool first = static_cast<int>(blockIdx.x) < tiles_x;
  MatrixJob& job = first ? x : y;
  const int t = static_cast<int>(blockIdx.x) - (first ? 0 : tiles_x);
  const int tc = (job.cols + kTile - 1) / kTile;
  split_tile(job.src, job.rows, job.cols, job.by_rows, job.by_cols, nullptr, t / tc, t % tc);
}

template <class Source>
void launch_transposed(const Source& src, int rows, int cols, const SplitCopy& by_cols, cudaStream_t s) {
  if (rows <= 0 || cols <= 0) return;
  const long long tiles = ((rows + kTile - 1ll) / kTile) * ((cols + kHalf - 1ll) / kHalf);
  if (tiles > INT32_MAX) throw std::invalid_argument("a matrix is too large");
  launch_next("split", split_transposed_kernel<Source>, dim3(static_cast<unsigned>(tiles)), 256, 0, 1, s, src, rows,
              cols, by_cols);
}

template <class Source>
void launch_split(const Source& src, int rows, int cols, const SplitCopy* by_rows, const SplitCopy* by_cols,
                  float* part, cudaStream_t s) {
  if (rows <= 0 || cols <= 0) return;
  if (by_cols && !by_rows && !part) return launch_transposed(src, rows, cols, *by_cols, s);
  auto kern = split_kernel<Source>;
  static thread_local int configured_device = -1;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (configured_device != dev) {
    check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSplitSmem), "shared memory");
    configured_device = dev;
  }
  const long long tiles = ((rows + kTile - 1ll) / kTile) * ((cols + kTile - 1ll) / kTile);
  if (tiles > INT32_MAX) throw std::invalid_argument("a matrix is too large");
  const SplitCopy none{};
  launch_next("split", kern, dim3(static_cast<unsigned>(tiles)), 32 * kSplitWarps, by_cols ? kSplitSmem : kSplitSums, 1,
              s, src, rows, cols, by_rows ? *by_rows : none, by_cols ? *by_cols : none, part);
}

// ------------------------------------------------------------------ products
// 256 x 256 tiles on CTA pairs (cta_group::2): CTA r of a pair holds rows 128 r..
// of the tile's A and of its B; a stage is 64 of K: Ah, Al, Bh, Bl, 16 KB each, a
// chunk two stages. Per stage a CTA takes in 64 KB and its tensor core reads 3 x
// 48 KB in 1,536 cycles: 135 bytes a cycle of shared memory, which feeds the tensor
// pipe through a long sum (96% busy at 32,000 of K). Warp 0 TMA, warp 1 UMMA (the leader's), warps 4..11 the
// running sums (TMEM lanes 32 (w % 4).., columns 128 ((w - 4) / 4)..) and the
// epilogue; the chunks' two TMEM accumulators let the next tile's first two chunks
// run beside it.
constexpr int BM = 128, PN = 256;
constexpr int P_THREADS = 384;
constexpr int P_SUM_WARP = 4;  // the first of the eight warps that sum and write
// Registers: a launch of 384 threads has 168 a thread; warps 0..3 (TMA, UMMA, two
// idle) give up all but 40, and the summing warps take 232 (40 + 2 x 232 = 3 x 168),
// which holds 128 sums, the residuals and the epilogue (of the 28 instances seven spill 16
// bytes a thread).
constexpr int P_REGS = 168, P_REGS_FEW = 40, P_REGS_SUM = 232;
static_assert(P_REGS_FEW + 2 * P_REGS_SUM <= 3 * P_REGS, "setmaxnreg draws on the launch's registers");
constexpr int P_RING = 196608;  // the stages' bytes
constexpr int P_TILE = 16384;   // 128 rows of 128 bytes
constexpr int P_SMEM = P_RING + 1024 + 256 + 8 * 32 * 32 * 4;
static_assert(P_SMEM <= 232448, "shared memory of a CTA");

// Work unit u. Tiles [0, full) are whole units; each of the rest (the last, partial
// wave) is cut into `splits` parts of its chunks, whose sums go to workspace tiles
// that reduce_kernel adds, in part order, before the epilogue.
struct PairWork {
  int full = 0, splits = 1;
  float* ws = nullptr;  // [(tiles - full) * splits][256][256]
};
struct PairUnit {
  int tile, cb, ce, slot;
};
__device__ __forceinline__ PairUnit unit_of(int u, const PairWork& w, int steps) {
  if (u < w.full) return {u, 0, steps, -1};
  const int v = u - w.full, part = v % w.splits;
  return {w.full + v / w.splits, steps * part / w.splits, steps * (part + 1) / w.splits, v};
}

__device__ __forceinline__ void stage_rows(const float* v, float4* stage_tile, int lane);

// How operands reach the UMMAs. A work step is what a unit's K range counts: `LOADS`
// stages. An accumulation covers CHUNK work steps, then the summing warps add it to the
// sums in registers (SCALED: with both operands' scales undone): the tensor core truncates
// at every UMMA, always toward zero, so what one accumulation loses grows with its length.
struct ExactFeed {  // split copies: hi and lo of A and B, 64 of K a stage, a chunk two
  static constexpr int STAGE = 4 * P_TILE, LOADS = 2, CHUNK = 1;
  static constexpr bool SCALED = true;
  static constexpr uint32_t IDESC = idesc_f16(2 * BM, PN);
  static __device__ __forceinline__ void load(uint32_t st, const CUtensorMap* a, const CUtensorMap* b, uint32_t bar,
                                              int i, int m0, int n0, int) {
    tma_load_3d_pair(st, a, bar, 0, m0, 2 * i);
    tma_load_3d_pair(st + 2 * P_TILE, b, bar, 0, n0, 2 * i);
  }
  // the terms, small ones first: Al Bh, Ah Bl, Ah Bh; 16 f16 = 32 bytes along the swizzled row
  static __device__ __forceinline__ void multiply(uint32_t acc, uint32_t st, bool first) {
#pragma unroll
    for (int term = 0; term < 3; ++term) {
      const uint32_t a = st + (term == 0 ? P_TILE : 0), b = st + (term == 1 ? 3 * P_TILE : 2 * P_TILE);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        umma_f16_pair(acc, smem_desc(a + k * 32, 16, 1024, kLayoutSw128), smem_desc(b + k * 32, 16, 1024, kLayoutSw128),
                      IDESC, (!first || term != 0 || k != 0) ? 1u : 0u);
    }
  }
};
// The f32 operands themselves, one TF32 pass: 32 of K a stage, 2048 an accumulation (256
// UMMAs; sums of one sign come out 1.4e-5 low whatever their length, 2.4e-4 for 32768 of K
// and 9.7e-4 for 131072 in one accumulation. 8192 x 5632 -> 2048: 327 us, 326 in one
// accumulation, 341 in steps of 1024, which the direct kernel has for half the error). Bits
// 1 and 2 of `boxes`: an MN-major A, B loads its stage in one 3-D box, else in 32-wide ones.
template <bool A_MN, bool B_MN>
struct Tf32Feed {
  static constexpr int STAGE = 2 * P_TILE, LOADS = 1, CHUNK = 64;
  static constexpr bool SCALED = false;
  static constexpr uint32_t IDESC = idesc_tf32(2 * BM, PN, A_MN, B_MN);
  template <bool MN>
  static __device__ __forceinline__ void side(uint32_t at, const CUtensorMap* map, uint32_t bar, int k0, int mn0,
                                              bool box3d) {
    if (!MN) {
      tma_load_2d_pair(at, map, bar, k0, mn0);
    } else if (box3d) {
      tma_load_3d_pair(at, map, bar, 0, k0, mn0 / 32);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) tma_load_2d_pair(at + j * 4096, map, bar, mn0 + 32 * j, k0);
    }
  }
  static __device__ __forceinline__ void load(uint32_t st, const CUtensorMap* a, const CUtensorMap* b, uint32_t bar,
                                              int i, int m0, int n0, int boxes) {
    side<A_MN>(st, a, bar, 32 * i, m0, boxes & 1);
    side<B_MN>(st + P_TILE, b, bar, 32 * i, n0, boxes & 2);
  }
  template <bool MN>
  static __device__ __forceinline__ uint64_t desc(uint32_t at, int k) {  // 8 of K: 32 bytes, or 8 rows of 128
    return MN ? smem_desc(at + k * 1024, 4096, 512, kLayoutSw128Base32) : smem_desc(at + k * 32, 16, 1024, kLayoutSw128);
  }
  static __device__ __forceinline__ void multiply(uint32_t acc, uint32_t st, bool first) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      umma_tf32_pair(acc, desc<A_MN>(st, k), desc<B_MN>(st + P_TILE, k), IDESC, (!first || k != 0) ? 1u : 0u);
  }
};

// sum += an accumulation's 32 rows x 128 columns with both scales undone: `ia` is this
// lane's row's inverse (of the loss's gradient it has grad_scale's sign), `ib` the columns'
// (the same for every lane). A chunk's sum is at
// most 2^37 (128 products of entries up to 2^15), so times a row's inverse it stays below
// 2^128 up to kSafeInverse, entries of 2^104. WIDE, where a row of the warp has larger
// ones: the smaller inverse first, so that nothing overflows which the other would bring
// back (two more instructions a value; the test for it costs up to 0.8% of a call, 333 x
// 50001 x 516 with gradients 400 -> 402 us). What the first factor loses to f32's smallest
// numbers is at most 2^-24 of a scaled unit, far below the copies' own 2^-25 of one in
// every entry times the other operand's 2^14.
constexpr float kSafeInverse = 0x1p90f;
template <bool WIDE>
__device__ __forceinline__ void add_chunk(float (&sum)[128], uint32_t acc, float ia, const float4* ib) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t r[32];
    tmem_ld_32x32b_x32(acc + q * 32, r);
    auto add = [&](int e, float b) {
      const float v = __uint_as_float(r[e]);
      float& o = sum[q * 32 + e];
      const bool first = !WIDE || fabsf(ia) < b;
      o = fmaf(v * (first ? ia : b), first ? b : ia, o);
    };
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float4 b = ib[q * 8 + e];
      add(4 * e, b.x);
      add(4 * e + 1, b.y);
      add(4 * e + 2, b.z);
      add(4 * e + 3, b.w);
    }
  }
}

template <class Feed, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const float* inv_a,
                long long ld_ia, const float* inv_b, long long ld_ib, const Epi epi, int M, int N, int steps, int boxes,
                int units, const PairWork work, int* err) {
  constexpr int P_STAGE = Feed::STAGE, P_STAGES = P_RING / P_STAGE;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(blockIdx.x) / 2, npairs = static_cast<int>(gridDim.x) / 2;
  const int tm = (M + 2 * BM - 1) / (2 * BM), tn = (N + PN - 1) / PN;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);
  const uint32_t bar_base = base + P_STAGES * P_STAGE;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (P_STAGES + s); };
  auto acc_full = [&](int b) { return bar_base + 8u * (2 * P_STAGES + b); };
  auto acc_empty = [&](int b) { return bar_base + 8u * (2 * P_STAGES + 2 + b); };
  constexpr int kBars = 2 * P_STAGES + 4;
  const uint32_t tmem_slot = bar_base + 8u * kBars;
  uint8_t* tail = smem + P_STAGES * P_STAGE + 8 * kBars;
  int* loads_issued = reinterpret_cast<int*>(tail + 8);
  int* loads_consumed = loads_issued + 1;
  static_assert(8 * kBars + 16 <= 256, "barriers and counters fit their 256 bytes");

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < P_STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 16);  // eight epilogue warps in each CTA
    }
    *loads_issued = 0;
    *loads_consumed = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * PN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const bool late = epi.late();
  if (!late) after_previous();
  let_next();
  const uint32_t tmem_base = *reinterpret_cast<uint32_t*>(tail);

  if (warp < P_SUM_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P_REGS_FEW));
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer (both CTAs); completions land on the leader's barriers
      int it = 0;
      bool ok = true;
      for (int u = pair; u < units && ok; u += npairs) {
        const PairUnit w = unit_of(u, work, steps);
        int mt, nt;
        tile_mn(w.tile, tm, tn, mt, nt);
        const int my_m0 = mt * 2 * BM + static_cast<int>(rank) * BM;
        const int my_n0 = nt * PN + static_cast<int>(rank) * (PN / 2);
        for (int i = Feed::LOADS * w.cb; i < Feed::LOADS * w.ce; ++i, ++it) {
          const int s = it % P_STAGES, round = it / P_STAGES;
          if (round > 0 && !mbar_wait(empty_bar(s), (round - 1) & 1, err, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(full_bar(s), 2 * P_STAGE);
          Feed::load(base + s * P_STAGE, &tmA, &tmB, mapa_shared(full_bar(s), 0), i, my_m0, my_n0, boxes);
          *loads_issued = it + 1;
        }
      }
    } else if (warp == 1 && lane == 0 && leader) {
      // ---------------- UMMA issuer (leader only), M = 256 across the pair
      int it = 0, j = 0;
      bool ok = true;
      for (int u = pair; u < units && ok; u += npairs) {
        const PairUnit w = unit_of(u, work, steps);
        for (int c = w.cb; c < w.ce && ok; c += Feed::CHUNK) {
          const int buf = j & 1;
          if (j >= 2 && !mbar_wait(acc_empty(buf), ((j >> 1) - 1) & 1, err, kErrWaitAccum)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int loads = Feed::LOADS * min(Feed::CHUNK, w.ce - c);
          for (int h = 0; h < loads; ++h, ++it) {
            const int s = it % P_STAGES, round = it / P_STAGES;
            if (!mbar_wait(full_bar(s), round & 1, err, kErrWaitFull)) {
              ok = false;
              break;
            }
            tc_fence_after();
            *loads_consumed = it + 1;
            Feed::multiply(tmem_base + buf * PN, base + s * P_STAGE, h == 0);
            umma_commit_pair(empty_bar(s), 0x3);
          }
          if (!ok) break;
          umma_commit_pair(acc_full(buf), 0x3);
          ++j;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P_REGS_SUM));
    // ---------------- running sums and epilogue (both CTAs): 32 rows x 128 columns per warp
    const int quarter = warp & 3, half = (warp - P_SUM_WARP) >> 2;
    float4* stage_tile = reinterpret_cast<float4*>(smem + P_STAGES * P_STAGE + 256) + (warp - P_SUM_WARP) * 256;
    int j = 0;
    bool ok = true;
    for (int u = pair; u < units && ok; u += npairs) {
      const PairUnit w = unit_of(u, work, steps);
      int mt, nt;
      tile_mn(w.tile, tm, tn, mt, nt);
      const int wrow0 = mt * 2 * BM + static_cast<int>(rank) * BM + quarter * 32, wcol0 = nt * PN + half * 128;
      float sum[128];
#pragma unroll
      for (int e = 0; e < 128; ++e) sum[e] = 0.0f;
      if (w.slot < 0) epi.prefetch(wrow0, wcol0, M, N, lane);
      // The accumulation's columns [32 q, 32 q + 32) of this warp; `release` hands it back.
      auto wait_acc = [&](uint32_t* acc) {
        const int buf = j & 1;
        if (!mbar_wait(acc_full(buf), (j >> 1) & 1, err, kErrWaitAccum)) return false;
        tc_fence_after();
        *acc = tmem_base + buf * PN + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
        return true;
      };
      auto release_acc = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(acc_empty(j & 1), 0));
        ++j;
      };
      uint32_t acc = 0;
      if (!Feed::SCALED) {
        // the first accumulation on its own: its values are the sums, with nothing added
        auto take = [&](auto first) {
          ok = wait_acc(&acc);
          if (!ok) return;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(acc + q * 32, r);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float v = __uint_as_float(r[e]);
              sum[q * 32 + e] = first ? v : sum[q * 32 + e] + v;
            }
          }
          release_acc();
        };
        take(std::true_type{});
        for (int c = w.cb + Feed::CHUNK; c < w.ce && ok; c += Feed::CHUNK) take(std::false_type{});
      } else {
        // The chunks' inverse scales, one chunk ahead: this lane's row's in a register,
        // the columns' through the staging tile (idle until the epilogue).
        const float* pa = inv_a + w.cb * ld_ia + wrow0 + lane;
        const float4* pb = reinterpret_cast<const float4*>(inv_b + w.cb * ld_ib + wcol0) + lane;
        float ia = *pa;
        stage_tile[lane] = *pb;
        __syncwarp();
        for (int c = w.cb; c < w.ce; ++c) {
          const float4* ib = stage_tile + 32 * ((c - w.cb) & 1);
          const bool more = c + 1 < w.ce;
          pa += ld_ia;
          pb += ld_ib / 4;
          const float ia_next = more ? *pa : 0.0f;
          const float4 ib_next = more ? *pb : make_float4(0.f, 0.f, 0.f, 0.f);
          const bool wide = __any_sync(0xffffffffu, fabsf(ia) > kSafeInverse);
          ok = wait_acc(&acc);
          if (!ok) break;
          if (wide)
            add_chunk<true>(sum, acc, ia, ib);
          else
            add_chunk<false>(sum, acc, ia, ib);
          release_acc();
          ia = ia_next;
          stage_tile[32 * ((c + 1 - w.cb) & 1) + lane] = ib_next;
          __syncwarp();
        }
      }
      if (!ok) break;
      if (w.slot < 0) {
        epi.tile(sum, stage_tile, wrow0, wcol0, M, N, lane);
      } else {  // a part: its sums as they are
        float* out = work.ws + (static_cast<long long>(w.slot) * 2 * BM + rank * BM + quarter * 32) * PN + half * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          stage_rows(sum + 32 * c, stage_tile, lane);
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < 8; ++i) {
            const int rr = i * 4 + (lane >> 3);
            *reinterpret_cast<float4*>(out + rr * PN + 32 * c + 4 * (lane & 7)) =
                stage_tile[rr * 8 + ((lane & 7) ^ (rr & 7))];
          }
          __syncwarp();
        }
      }
    }
  }

  tc_fence_before();
  cluster_sync();  // both CTAs are done with their TMEM and with each other's barriers
  if (leader && threadIdx.x == 0) {
    // after a timed-out wait, let the pair's copies in flight land (bounded)
    for (int i = *loads_consumed; i < *loads_issued; ++i)
      if (!mbar_wait(full_bar(i % P_STAGES), (i / P_STAGES) & 1, err, kErrWaitDrain, 1000000000ull)) break;
  }
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * PN);
  }
  if (late) after_previous();
}

// A warp's 32 rows (lane = row) x 32 columns through its staging tile: 8 lanes per
// row then hold its 32 columns, so loads and stores cover whole 128-byte segments.
__device__ __forceinline__ void stage_rows(const float* v, float4* stage_tile, int lane) {
#pragma unroll
  for (int g = 0; g < 8; ++g)
    stage_tile[lane * 8 + (g ^ (lane & 7))] = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
}

template <int ACT, bool DROP>
struct LinearPair {
  LinearEpilogue e;
  __device__ __forceinline__ bool late() const { return e.late; }
  // The residual's rows into L2 while the sums form (a row's 128 columns: four lines).
  __device__ __forceinline__ void prefetch(int wrow0, int n0, int M, int N, int lane) const {
    if (!e.R || wrow0 + lane >= M) return;
    const float* row = e.R + (wrow0 + lane) * e.ldr;
#pragma unroll
    for (int c = 0; c < 128; c += 32)
      if (n0 + c < N) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + n0 + c));
  }
  // A rolled loop over slices of 32 columns (the unrolled one outgrows the instruction
  // cache): the first slice goes through the staging tile, the rest move down.
  template <bool FULL>
  __device__ __forceinline__ void slices(float (&sum)[128], float4* stage_tile, int wrow0, int n0, int M, int N,
                                         int lane) const {
    const int sub = lane & 7, rsub = lane >> 3;
    uint64_t seed = 0, offset = 0;
    if (DROP) {
      seed = e.drop.rng[0];
      offset = e.drop.rng[1];
    }
    const long long row0 = wrow0 + rsub;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      stage_rows(sum, stage_tile, lane);
#pragma unroll
      for (int i = 0; i < 96; ++i) sum[i] = sum[i + 32];
      const int col = n0 + 32 * c + 4 * sub;
      const float4 bias = bias_quad(e, col, N);
      float4 r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!e.R) continue;
        const float* p = e.R + (row0 + 4 * i) * e.ldr;
        if (FULL)
          r[i] = *reinterpret_cast<const float4*>(p + col);
        else if (row0 + 4 * i < M && col < N)
          r[i] = load_quad(p, col, N);
      }
      __syncwarp();
      if (FULL) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = 4 * i + rsub;
          const float4 v = stage_tile[rr * 8 + (sub ^ (rr & 7))];
          linear_quad<true>(e, ACT, DROP, seed, offset, row0 + 4 * i, col, N, v, bias, r[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = 4 * i + rsub;
          const float4 v = stage_tile[rr * 8 + (sub ^ (rr & 7))];
          if (row0 + 4 * i < M && col < N)
            linear_quad(e, ACT, DROP, seed, offset, row0 + 4 * i, col, N, v, bias, r[i]);
        }
      }
      __syncwarp();  // before the next slice overwrites the staging tile
    }
  }
  __device__ __forceinline__ void tile(float (&sum)[128], float4* stage_tile, int wrow0, int n0, int M, int N,
                                       int lane) const {
    if (wrow0 + 32 <= M && n0 + 128 <= N)
      slices<true>(sum, stage_tile, wrow0, n0, M, N, lane);
    else
      slices<false>(sum, stage_tile, wrow0, n0, M, N, lane);
  }
};

// The split tiles: parts summed in order, then the epilogue. Four rows of a tile per block.
__global__ void __launch_bounds__(256) reduce_kernel(const PairWork work, const LinearEpilogue e, int M, int N) {
  after_previous();
  let_next();
  const int tm = (M + 2 * BM - 1) / (2 * BM), tn = (N + PN - 1) / PN;
  int mt, nt;
  tile_mn(work.full + static_cast<int>(blockIdx.x), tm, tn, mt, nt);
  const int r = blockIdx.y * 4 + threadIdx.x / 64, c = (threadIdx.x % 64) * 4;
  const long long row = mt * 2 * BM + r;
  const int col = nt * PN + c;
  if (row >= M || col >= N) return;
  const float* p = work.ws + (static_cast<long long>(blockIdx.x) * work.splits * 2 * BM + r) * PN + c;
  float4 v = *reinterpret_cast<const float4*>(p);
  for (int i = 1; i < work.splits; ++i) {
    p += 2 * BM * PN;
    const float4 o = *reinterpret_cast<const float4*>(p);
    v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
  }
  const float4 res = e.R ? load_quad(e.R + row * e.ldr, col, N) : make_float4(0.f, 0.f, 0.f, 0.f);
  const bool drop = e.drop.rng != nullptr;
  linear_quad(e, e.act, drop, drop ? e.drop.rng[0] : 0, drop ? e.drop.rng[1] : 0, row, col, N, v, bias_quad(e, col, N),
              res);
}

struct LossPair {
  LossEpilogue e;
  __device__ __forceinline__ bool late() const { return false; }
  __device__ __forceinline__ void prefetch(int, int, int, int, int) const {}
  __device__ __forceinline__ void tile(float (&sum)[128], float4* stage_tile, int wrow0, int n0, int M, int N,
                                       int lane) const {
    if (n0 >= N) return;  // uniform over the warp
    const long long my_row = wrow0 + lane;
    const int live = min(128, N - n0);
    const int t = my_row < M ? e.targets[my_row] - n0 : -1;
    if (t >= 0 && t < live) {
      float zt = 0.0f;
#pragma unroll
      for (int i = 0; i < 128; ++i) zt = i == t ? sum[i] : zt;
      e.zt[my_row] = zt;
    }
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, all[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 128; ++i) top[i % 4] = live == 128 || i < live ? fmaxf(top[i % 4], sum[i]) : top[i % 4];
    const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    if (e.copy) {
      if (live == 128 && wrow0 + 32 <= M)
        copy_slices<true>(sum, all, m, live, stage_tile, wrow0, n0, M, lane);
      else
        copy_slices<false>(sum, all, m, live, stage_tile, wrow0, n0, M, lane);
    } else {
#pragma unroll
      for (int i = 0; i < 128; ++i) all[i % 4] += live == 128 || i < live ? loss_exp(sum[i] - m) : 0.0f;
    }
    if (my_row < M) e.part[my_row * e.tiles + n0 / 128] = make_float2(m, (all[0] + all[1]) + (all[2] + all[3]));
    if (e.copy) return;
    if (!e.Z) return;
    if (wrow0 + 32 <= M && n0 + 128 <= N)
      store<true>(sum, stage_tile, wrow0, n0, M, N, lane);
    else
      store<false>(sum, stage_tile, wrow0, n0, M, N, lane);
  }
  // The chunk's exponentials, in (0, 1], added up and times 2^14 as hi and lo: the copy that
  // dx's product reads once its scales (2^-14 exp(m - row maximum) grad_scale / row sum) are
  // known. A rolled loop over slices of 32 columns, as in LinearPair.
  template <bool FULL>
  __device__ __forceinline__ void copy_slices(float (&sum)[128], float (&all)[4], float m, int live, float4* stage_tile,
                                              int wrow0, int n0, int M, int lane) const {
    const int sub = lane & 7, rsub = lane >> 3;
    uint16_t* row = e.copy + (wrow0 + rsub) * e.copy_ld + (n0 / 128) * 256ll + 4 * sub;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        sum[i] = FULL || 32 * c + i < live ? loss_exp(sum[i] - m) : 0.0f;
        all[i % 4] += sum[i];
      }
      stage_rows(sum, stage_tile, lane);
#pragma unroll
      for (int i = 0; i < 96; ++i) sum[i] = sum[i + 32];
      __syncwarp();
      uint16_t* out = row + (c / 2) * 128 + (c % 2) * 32;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int rr = 4 * i + rsub;
        const float4 v = stage_tile[rr * 8 + (sub ^ (rr & 7))];
        uint2 hi, lo;
        halves(v.x * 16384.0f, v.y * 16384.0f, hi.x, lo.x);
        halves(v.z * 16384.0f, v.w * 16384.0f, hi.y, lo.y);
        if (FULL || wrow0 + rr < M) {
          *reinterpret_cast<uint2*>(out + 4 * i * e.copy_ld) = hi;
          *reinterpret_cast<uint2*>(out + 4 * i * e.copy_ld + 64) = lo;
        }
      }
      __syncwarp();  // before the next slice overwrites the staging tile
    }
  }
  template <bool FULL>
  __device__ __forceinline__ void store(const float (&sum)[128], float4* stage_tile, int wrow0, int n0, int M, int N,
                                        int lane) const {
    const int sub = lane & 7, rsub = lane >> 3;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      stage_rows(sum + 32 * c, stage_tile, lane);
      __syncwarp();
      const int col = n0 + 32 * c + 4 * sub;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int rr = 4 * i + rsub;
        const long long row = wrow0 + rr;
        const float4 v = stage_tile[rr * 8 + (sub ^ (rr & 7))];
        if (FULL || (row < M && col < N)) put_quad<FULL>(e.Z + row * e.ldz, col, N, v);
      }
      __syncwarp();  // before the next slice overwrites the staging tile
    }
  }
};

// G from the exponentials' copy: every chunk's scale becomes 2^-14 exp(its maximum - the
// row's) grad_scale / the row's sum (0 for a row without a target), which the products
// apply as they apply any scale, and the target's chunk is written anew with grad_scale
// taken off. A warp per row.
__global__ void __launch_bounds__(256) loss_scales_kernel(SplitCopy g, const float2* part, const float2* stat,
                                                          const int32_t* targets, int vocab, float grad_scale) {
  after_previous();
  let_next();
  const int row = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (row >= g.rows) return;
  const int chunks = static_cast<int>(g.chunks());
  const int t = targets[row];
  const bool live = t >= 0 && t < vocab;
  const float2 st = stat[row];
  const float2* mine = part + static_cast<long long>(row) * chunks;
  float* inv = g.inv + row;
  const float unit = st.y * 6.103515625e-05f;  // 2^-14 grad_scale / sum
#pragma unroll 8
  for (int c = lane; c < chunks; c += 32) inv[c * g.inv_ld()] = live ? loss_exp(mine[c].x - st.x) * unit : 0.0f;
  if (!live) return;
  const int c = t >> 7;
  const float f = loss_exp(mine[c].x - st.x) * unit;
  uint16_t* p = g.data + row * g.row_halves() + c * 256ll + (lane / 16) * 128 + (lane % 16) * 4;  // columns 4 lane..
  uint2 hi = *reinterpret_cast<const uint2*>(p), lo = *reinterpret_cast<const uint2*>(p + 64);
  const uint32_t h[2] = {hi.x, hi.y}, l[2] = {lo.x, lo.y};
  float v[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&l[i]));
    v[2 * i] = (a.x + b.x) * f;
    v[2 * i + 1] = (a.y + b.y) * f;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((t & 127) == 4 * lane + i) v[i] -= grad_scale;
    m = max(m, magnitude(v[i]));
  }
  float back;
  const float scale = chunk_scale(__reduce_max_sync(0xffffffffu, m), &back);
  halves(v[0] * scale, v[1] * scale, hi.x, lo.x);
  halves(v[2] * scale, v[3] * scale, hi.y, lo.y);
  *reinterpret_cast<uint2*>(p) = hi;
  *reinterpret_cast<uint2*>(p + 64) = lo;
  __syncwarp();  // the loop above wrote this chunk's scale too
  if (lane == 0) inv[c * g.inv_ld()] = back;
}

// (64 halves, rows, segments): one box of {64, 128, 2} is a stage's hi and lo tile.
int copy_map(CUtensorMap* map, const SplitCopy& c) {
  const long long dims[3] = {64, c.rows, 4 * c.chunks()}, strides[2] = {c.row_halves(), 64};
  const int box[3] = {64, 128, 2};
  return encode_tensor_map_f16(map, c.data, 3, dims, strides, box) ? kGemmTensorMap : 0;
}

// The last wave's tiles are cut into parts when that saves at least `worth` work steps
// of its length: writing, reading and summing the parts takes about 8 us, a chunk of
// the exact mode 2 us, a TF32 step 0.45 us. The grid is that of the full part: 74 pairs.
constexpr int kPairs = 74;
constexpr int kWorthExact = 8, kWorthTf32 = 28;
PairWork work_of(long long tiles, int steps, int worth) {
  PairWork w;
  w.full = static_cast<int>(tiles);
  const int tail = static_cast<int>(tiles % kPairs);
  if (tail == 0) return w;
  const int s = std::min(kPairs / tail, steps);
  if (s < 2 || steps - (steps + s - 1) / s < worth) return w;
  w.full = static_cast<int>(tiles - tail);
  w.splits = s;
  return w;
}

long long tiles_of(int M, int N) { return static_cast<long long>((M + 255) / 256) * ((N + 255) / 256); }

// One launch's operands: tensor maps, and the copies' scales or the box flags.
struct PairInput {
  CUtensorMap a{}, b{};
  const float *inv_a = nullptr, *inv_b = nullptr;
  long long ld_ia = 0, ld_ib = 0;
  int M, N, steps, boxes = 0;
};

template <class Feed, class Epi>
int launch_pair(const PairInput& in, const Epi& epi, const PairWork& work, int* d_err, cudaStream_t s) {
  auto kern = pair_kernel<Feed, Epi>;
  static thread_local int configured_device = -1;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (configured_device != dev) {
    check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM), "shared memory");
    // fewer registers at launch than the kernel's setmaxnreg hands out would make it wait
    cudaFuncAttributes fa{};
    check_cuda(cudaFuncGetAttributes(&fa, kern), "kernel attributes");
    if (fa.numRegs != P_REGS) throw std::runtime_error("linear: the pair kernel's registers do not match its split");
    configured_device = dev;
  }
  const long long tiles = tiles_of(in.M, in.N), units = work.full + (tiles - work.full) * work.splits;
  const int grid = 2 * static_cast<int>(std::min<long long>(units, std::min(kPairs, sm_count() / 2)));
  launch_next("linear", kern, dim3(grid), P_THREADS, P_SMEM, 1, s, in.a, in.b, in.inv_a, in.ld_ia, in.inv_b, in.ld_ib,
              epi, in.M, in.N, in.steps, in.boxes, static_cast<int>(units), work, d_err);
  return 0;
}

template <class Feed, int ACT>
int launch_act(const PairInput& in, const LinearEpilogue& e, const PairWork& work, int* d_err, cudaStream_t s) {
  return e.drop.rng ? launch_pair<Feed>(in, LinearPair<ACT, true>{e}, work, d_err, s)
                    : launch_pair<Feed>(in, LinearPair<ACT, false>{e}, work, d_err, s);
}
template <class Feed>
int launch_linear(const PairInput& in, const LinearEpilogue& e, const PairWork& work, int* d_err, cudaStream_t s) {
  switch (e.act) {
    case kActRelu: return launch_act<Feed, kActRelu>(in, e, work, d_err, s);
    case kActGelu: return launch_act<Feed, kActGelu>(in, e, work, d_err, s);
    case kActSilu: return launch_act<Feed, kActSilu>(in, e, work, d_err, s);
    default: return launch_act<Feed, kActNone>(in, e, work, d_err, s);
  }
}

int exact_input(const SplitCopy& A, const SplitCopy& B, PairInput* in) {
  if (A.k != B.k || A.k <= 0 || tiles_of(A.rows, B.rows) > (1 << 26)) return kGemmBadArgument;
  int rc = copy_map(&in->a, A);
  if (!rc) rc = copy_map(&in->b, B);
  in->inv_a = A.inv;
  in->ld_ia = A.inv_ld();
  in->inv_b = B.inv;
  in->ld_ib = B.inv_ld();
  in->M = A.rows;
  in->N = B.rows;
  in->steps = static_cast<int>(A.chunks());
  return rc;
}

int tf32_input(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, PairInput* in) {
  if (K <= 0 || tiles_of(M, N) > (1 << 26)) return kGemmBadArgument;
  bool a3 = false, b3 = false;
  int rc = operand_map(&in->a, A, M, K, 128, &a3);
  if (!rc) rc = operand_map(&in->b, B, N, K, 128, &b3);
  in->M = M;
  in->N = N;
  in->steps = (K + 31) / 32;
  in->boxes = (a3 ? 1 : 0) | (b3 ? 2 : 0);
  return rc;
}

long long parts_bytes(int M, int N, int steps, int worth) {
  const PairWork w = work_of(tiles_of(M, N), steps, worth);
  return (tiles_of(M, N) - w.full) * w.splits * (2ll * BM * PN * 4);
}

// Whether a product is better on pairs than direct: its units keep half of the pairs
// busy, its tiles are mostly full, and it is long enough (`least` GFLOP, 2.9 where both
// sides have two tiles) or has so many tiles that direct ones, which do not overlap
// their starts and ends, would take three waves. Both sides, device time (us, direct /
// pair with its copies; exact, then TF32): 1024 x 1024 x 1024 21 / 28, 13 / 18; 256 x 2048 x
// 5632 49 / 49, 29 / 21; 512 x 1024 x 2816 32 / 30, 18 / 19; 2048 x 512 x 1408 37 / 22,
// 23 / 14; 1024 x 128 x 8192 37 / 21, 30 / 14; 4096 x 2048 x 5632 525 / 225, 250 / 133; 128 x
// 2048 x 5632 26 / 47, 15 / 19.
bool suits(int M, int N, int K, int steps, int worth, double least) {
  const int side = std::min(M, N);
  const double gflop = 2e-9 * M * N * K;
  const long long direct_tiles = ((M + 127ll) / 128) * ((N + 127ll) / 128);
  if (side < 192 || !(gflop >= least || (side >= 512 && gflop >= 2.9) || direct_tiles >= 3 * 148)) return false;
  const PairWork w = work_of(tiles_of(M, N), steps, worth);
  return 2 * (w.full + (tiles_of(M, N) - w.full) * w.splits) >= kPairs;
}

void reduce_parts(const PairInput& in, const PairWork& work, const LinearEpilogue& e, cudaStream_t s) {
  const long long tail = tiles_of(in.M, in.N) - work.full;
  if (!tail) return;
  launch_next("linear", reduce_kernel, dim3(static_cast<unsigned>(tail), 2 * BM / 4), 256, 0, 1, s, work, e, in.M, in.N);
}

long long copy_data_bytes(int rows, int k) { return rows * ((k + 127ll) / 128) * 512; }

}  // namespace

long long split_copy_bytes(int rows, int k) {
  return copy_data_bytes(rows, k) + ((k + 127ll) / 128) * ((rows + 255ll) / 256 * 256) * 4;
}

SplitCopy split_copy_at(void* ptr, int rows, int k) {
  SplitCopy c;
  c.data = static_cast<uint16_t*>(ptr);
  c.inv = reinterpret_cast<float*>(static_cast<uint8_t*>(ptr) + copy_data_bytes(rows, k));
  c.rows = rows;
  c.k = k;
  return c;
}

void split(const SplitMatrix& src, int rows, int cols, const SplitCopy* by_rows, const SplitCopy* by_cols,
           cudaStream_t s) {
  launch_split(MatrixSource{src}, rows, cols, by_rows, by_cols, nullptr, s);
}
void split(const SplitBackward& src, int rows, int cols, const SplitCopy* by_rows, const SplitCopy* by_cols,
           float* part, cudaStream_t s) {
  launch_split(BackwardSource{src, 0, 0}, rows, cols, by_rows, by_cols, part, s);
}
void loss_scales(const SplitCopy& g, const float2* part, const float2* stat, const int32_t* targets, int vocab,
                 float grad_scale, cudaStream_t s) {
  if (g.rows <= 0) return;
  launch_next("loss gradient", loss_scales_kernel, dim3((g.rows + 7) / 8), 256, 0, 1, s, g, part, stat, targets, vocab,
              grad_scale);
}

void split_transposed(const SplitCopy& src, const SplitCopy& by_cols, cudaStream_t s) {
  launch_transposed(CopySource{src}, src.rows, src.k, by_cols, s);
}

void split_two(const SplitMatrix& x, int x_rows, int x_cols, const SplitCopy* x_by_rows, const SplitCopy* x_by_cols,
               const SplitMatrix& y, int y_rows, int y_cols, const SplitCopy* y_by_rows, const SplitCopy* y_by_cols,
               cudaStream_t s) {
  auto job = [](const SplitMatrix& m, int rows, int cols, const SplitCopy* r, const SplitCopy* c) {
    return MatrixJob{{m}, rows, cols, r ? *r : SplitCopy{}, c ? *c : SplitCopy{}};
  };
  auto tiles = [](int rows, int cols) { return ((rows + 127ll) / 128) * ((cols + 127ll) / 128); };
  const int smem = x_by_cols || y_by_cols ? kSplitSmem : kSplitSums;
  static thread_local int configured_device = -1;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (configured_device != dev) {
    check_cuda(cudaFuncSetAttribute(split_two_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSplitSmem),
               "shared memory");
    configured_device = dev;
  }
  const long long n = tiles(x_rows, x_cols) + tiles(y_rows, y_cols);
  if (n > INT32_MAX) throw std::invalid_argument("a matrix is too large");
  launch_next("split", split_two_kernel, dim3(static_cast<unsigned>(n)), 32 * kSplitWarps, smem, 1, s,
              job(x, x_rows, x_cols, x_by_rows, x_by_cols), job(y, y_rows, y_cols, y_by_rows, y_by_cols));
}

long long pair_ws_bytes(int M, int N, int K) { return parts_bytes(M, N, (K + 127) / 128, kWorthExact); }

int pair_product(const SplitCopy& A, const SplitCopy& B, const LinearEpilogue& e, void* ws, int* d_err,
                 cudaStream_t s) {
  if (A.rows <= 0 || B.rows <= 0) return 0;
  PairInput in;
  int rc = exact_input(A, B, &in);
  if (rc) return rc;
  PairWork work = work_of(tiles_of(in.M, in.N), in.steps, kWorthExact);
  work.ws = static_cast<float*>(ws);
  rc = launch_linear<ExactFeed>(in, e, work, d_err, s);
  if (!rc) reduce_parts(in, work, e, s);
  return rc;
}

int pair_loss_product(const SplitCopy& A, const SplitCopy& B, const LossEpilogue& e, int* d_err, cudaStream_t s) {
  if (A.rows <= 0 || B.rows <= 0) return 0;
  PairInput in;
  const int rc = exact_input(A, B, &in);
  if (rc) return rc;
  PairWork work;  // the epilogue needs a tile's whole sums: no parts
  work.full = static_cast<int>(tiles_of(in.M, in.N));
  return launch_pair<ExactFeed>(in, LossPair{e}, work, d_err, s);
}

bool pair_product_suits(int M, int N, int K) { return K >= 128 && suits(M, N, K, (K + 127) / 128, kWorthExact, 6.0); }

double pair_us(int M, int N, int K, bool parts) {
  const int chunks = (K + 127) / 128;
  const long long tiles = tiles_of(M, N);
  PairWork w = work_of(tiles, chunks, kWorthExact);
  if (!parts) {
    w.full = static_cast<int>(tiles);
    w.splits = 1;
  }
  const double whole = 2.05 * chunks + 2.5;
  const long long waves = (w.full + kPairs - 1) / kPairs;
  return waves * whole + (w.full < tiles ? 2.05 * ((chunks + w.splits - 1) / w.splits) + 10.0 : 0.0);
}

long long tf32_pair_ws_bytes(int M, int N, int K) { return parts_bytes(M, N, (K + 31) / 32, kWorthTf32); }

int tf32_pair_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LinearEpilogue& e,
                      void* ws, int* d_err, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  PairInput in;
  int rc = tf32_input(M, N, K, A, B, &in);
  if (rc) return rc;
  PairWork work = work_of(tiles_of(M, N), in.steps, kWorthTf32);
  work.ws = static_cast<float*>(ws);
  if (!A.mn_major)
    rc = B.mn_major ? launch_linear<Tf32Feed<false, true>>(in, e, work, d_err, s)
                    : launch_linear<Tf32Feed<false, false>>(in, e, work, d_err, s);
  else if (B.mn_major && e.act == kActNone && !e.drop.rng)  // a weight's gradient
    rc = launch_pair<Tf32Feed<true, true>>(in, LinearPair<kActNone, false>{e}, work, d_err, s);
  else
    return kGemmBadArgument;
  if (!rc) reduce_parts(in, work, e, s);
  return rc;
}

int tf32_pair_loss_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LossEpilogue& e,
                           int* d_err, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  if (A.mn_major) return kGemmBadArgument;
  PairInput in;
  const int rc = tf32_input(M, N, K, A, B, &in);
  if (rc) return rc;
  PairWork work;
  work.full = static_cast<int>(tiles_of(M, N));
  return B.mn_major ? launch_pair<Tf32Feed<false, true>>(in, LossPair{e}, work, d_err, s)
                    : launch_pair<Tf32Feed<false, false>>(in, LossPair{e}, work, d_err, s);
}

bool tf32_pair_suits(int M, int N, int K) { return suits(M, N, K, (K + 31) / 32, kWorthTf32, 5.0); }

}  // namespace mm
