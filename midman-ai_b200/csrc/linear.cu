// Products with an epilogue for sm_100a:
//
//   z = A B^T (+ bias),  c = r + dropout(act(z))         (LinearEpilogue)
//   z = A B^T, per row and 128 columns max z and sum exp(z - max)  (LossEpilogue)
//
// Exact mode: A B = (Ah + Al)(Bh + Bl) ~ Al Bh + Ah Bl + Ah Bh, hi the bits the
// tensor core reads of an f32 (11 significant bits), lo what they leave out
// rounded to as many: the dropped Al Bl is 2^-22 of the product. The tensor
// core's f32 accumulation loses a little on every UMMA, always in the same
// direction, so every 64 of K start a fresh TMEM accumulation and the chunks are
// summed in f32 registers.
//
// direct_kernel: one 128 x 128 tile per cluster of `splits` CTAs, each CTA a part
// of K (and where few tiles share a long K, clusters for its slices, whose sums go to
// the workspace and join_kernel). TMA brings the f32 operands. Their lo parts are made
// on the way, which saves the passes and the workspace of copies made beforehand (short
// products are bound by latency and one reading of the operands): four warps take A's
// rows to tensor memory, hi and lo, where the UMMAs read them; two write B's lo part
// beside it in shared memory (elementwise, so the swizzled layout is kept). What bounds
// a K step of 32 of a 128 x 128 tile is shared memory: 32 KB in by TMA, 48 KB through
// the converters, 48 KB read by the UMMAs, 1,024 cycles at 128 bytes each; 1,140
// measured, 0.58 us at 1.965 GHz (with A's parts in shared memory too 1,536 and 1,600;
// with four warps on B's lo part instead of two nothing changed). Where all SMs bring
// tiles that no other takes, the L2 bounds it: 148 tiles of 128 rows 0.74 us a step, 6.5
// TB/s; one TF32 term 0.28 to 0.32. The parts' sums meet in shared memory over
// the cluster (each CTA sums 128 / splits rows of all parts, in part order:
// bit-identical run to run) and go through the epilogue in whole rows.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <stdexcept>

#include "device.h"
#include "gemm.h"
#include "linear.h"
#include "linear_epi.cuh"
#include "ptx.cuh"
#include "tma.h"

namespace mm {
namespace {

constexpr int BM = 128, BN = 128;
constexpr int BK = 32;  // 32 f32 = 128 bytes = one swizzle row
constexpr uint32_t MN_BLOCK_BYTES = BK * 128;
constexpr int kEpiWarps = 8;

// ------------------------------------------------------------------ direct kernel
// A stage: A, then B, then (three terms) B's lo part. Three terms: warps 2, 3 write
// B's lo, 4..7 take A to tensor memory (the lanes of warp w are rows 32 (w % 4)..),
// 8..15 sum; one term: warps 2..9 sum.
template <int TERMS>
struct DirectTile {
  static constexpr int A_BYTES = BM * BK * 4;
  static constexpr int B_BYTES = BN * BK * 4;
  static constexpr int IN_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGE = IN_BYTES + (TERMS == 3 ? B_BYTES : 0);
  static constexpr int TMEM_STAGE = 2 * BK;  // columns of A's hi and lo
  static constexpr int FIT = 196608 / STAGE > 8 ? 8 : 196608 / STAGE;
  static constexpr int TMEM_FIT = (512 - 2 * BN) / TMEM_STAGE;
  static constexpr int STAGES = TERMS == 3 && TMEM_FIT < FIT ? TMEM_FIT : FIT;
  static constexpr int TMEM_COLS = TERMS == 3 ? 512 : 2 * BN;
  static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
  static constexpr int SUM_WARP = TERMS == 3 ? 8 : 2;
  static constexpr int THREADS = 32 * (SUM_WARP + kEpiWarps);
  static constexpr int CHUNK = TERMS == 3 ? 2 : 32;  // K steps per TMEM accumulation (24 or 128 UMMAs)
  static_assert(BM * BN * 4 + 2 * BM * 8 <= STAGES * STAGE, "the partial tile and its halves reuse the stages");
};

__device__ __forceinline__ float4 ld_cluster_quad(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The sum over the cluster's parts, in part order, of quad q of tile row r.
__device__ __forceinline__ float4 sum_quad(uint32_t tile, int r, int q, int splits) {
  const uint32_t at = tile + 16u * static_cast<uint32_t>(r * (BN / 4) + (q ^ (r & 7)));
  float4 v;
  if (splits == 1) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
  }
  v = ld_cluster_quad(mapa_shared(at, 0));
  if (splits == 2) {
    const float4 w = ld_cluster_quad(mapa_shared(at, 1));
    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    return v;
  }
  for (int p = 1; p < splits; p += 3) {  // at most three loads in flight
    float4 w[3];
#pragma unroll
    for (int i = 0; i < 3; ++i)
      w[i] = p + i < splits ? ld_cluster_quad(mapa_shared(at, p + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      v.x += w[i].x; v.y += w[i].y; v.z += w[i].z; v.w += w[i].w;
    }
  }
  return v;
}

__device__ __forceinline__ float lo_part(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x - __uint_as_float(__float_as_uint(x) & 0xffffe000u)));
  return __uint_as_float(r);
}

template <int TERMS, bool A_MN, bool B_MN, class Epi>
__global__ void __launch_bounds__(DirectTile<TERMS>::THREADS, 1)
    direct_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Epi epi,
                  int M, int N, int K, int splits, int slices, long long slice_stride, int mn3d, int* err) {
  using TL = DirectTile<TERMS>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);
  const uint32_t bar_base = base + TL::STAGES * TL::STAGE;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (TL::STAGES + s); };
  auto lo_bar = [&](int s) { return bar_base + 8u * (2 * TL::STAGES + s); };
  auto acc_full = [&](int b) { return bar_base + 8u * (3 * TL::STAGES + b); };
  auto acc_empty = [&](int b) { return bar_base + 8u * (3 * TL::STAGES + 2 + b); };
  constexpr int kBars = 3 * TL::STAGES + 4;
  static_assert(8 * kBars + 16 <= 256, "barriers and counters fit their 256 bytes");
  uint8_t* tail = smem + TL::STAGES * TL::STAGE + 8 * kBars;
  const uint32_t tmem_slot = bar_base + 8u * kBars;
  int* loads_issued = reinterpret_cast<int*>(tail + 8);
  int* loads_consumed = loads_issued + 1;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int part = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
  const int cluster = static_cast<int>(blockIdx.x) / splits, slice = cluster / (tm * tn);
  int mt, nt;
  tile_mn(cluster - slice * (tm * tn), tm, tn, mt, nt);
  const int m0 = mt * BM, n0 = nt * BN;
  const int n_k = (K + BK - 1) / BK;
  const long long kpart = static_cast<long long>(slice) * splits + part;
  const long long kparts = static_cast<long long>(slices) * splits;
  const int kb = static_cast<int>(n_k * kpart / kparts), ke = static_cast<int>(n_k * (kpart + 1) / kparts);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < TL::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
      mbar_init(lo_bar(s), 6);  // the converter warps
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), kEpiWarps);
    }
    *loads_issued = 0;
    *loads_consumed = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TL::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const bool late = epi.late();
  if (!late) after_previous();
  let_next();
  const uint32_t tmem_base = *reinterpret_cast<uint32_t*>(tail);
  const uint32_t tmem_a = tmem_base + 2 * BN;  // three terms: A's stages
  float2* halves = reinterpret_cast<float2*>(smem + BM * BN * 4);  // behind the partial tile

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer
      for (int i = kb; i < ke; ++i) {
        const int it = i - kb, s = it % TL::STAGES, round = it / TL::STAGES;
        if (round > 0 && !mbar_wait(empty_bar(s), (round - 1) & 1, err, kErrWaitEmpty)) break;
        const uint32_t sa = base + s * TL::STAGE, sb = sa + TL::A_BYTES;
        mbar_arrive_expect_tx(full_bar(s), TL::IN_BYTES);
        const int k0 = i * BK;
        if (!A_MN) {
          tma_load_2d(sa, &tmA, full_bar(s), k0, m0);
        } else if (mn3d & 1) {
          tma_load_3d(sa, &tmA, full_bar(s), 0, k0, m0 / 32);
        } else {
#pragma unroll
          for (int j = 0; j < BM / 32; ++j) tma_load_2d(sa + j * MN_BLOCK_BYTES, &tmA, full_bar(s), m0 + 32 * j, k0);
        }
        if (!B_MN) {
          tma_load_2d(sb, &tmB, full_bar(s), k0, n0);
        } else if (mn3d & 2) {
          tma_load_3d(sb, &tmB, full_bar(s), 0, k0, n0 / 32);
        } else {
#pragma unroll
          for (int j = 0; j < BN / 32; ++j) tma_load_2d(sb + j * MN_BLOCK_BYTES, &tmB, full_bar(s), n0 + 32 * j, k0);
        }
        *loads_issued = it + 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- UMMA issuer
      constexpr uint32_t idesc = idesc_tf32(BM, BN, TERMS == 1 && A_MN, B_MN);
      int j = 0;
      bool ok = true;
      for (int cb = kb; cb < ke && ok; cb += TL::CHUNK, ++j) {
        const int ce = min(ke, cb + TL::CHUNK), buf = j & 1;
        if (j >= 2 && !mbar_wait(acc_empty(buf), ((j >> 1) - 1) & 1, err, kErrWaitAccum)) break;
        tc_fence_after();
        const uint32_t acc = tmem_base + buf * BN;
        for (int i = cb; i < ce; ++i) {
          const int it = i - kb, s = it % TL::STAGES, round = it / TL::STAGES;
          if (!mbar_wait(full_bar(s), round & 1, err, kErrWaitFull) ||
              (TERMS == 3 && !mbar_wait(lo_bar(s), round & 1, err, kErrWaitFull))) {
            ok = false;
            break;
          }
          tc_fence_after();
          *loads_consumed = it + 1;
          const uint32_t sa = base + s * TL::STAGE, sb = sa + TL::A_BYTES;
          // the terms, small ones first: Al Bh, Ah Bl, Ah Bh (or Ah Bh alone)
#pragma unroll
          for (int term = 0; term < TERMS; ++term) {
            const uint32_t ta = tmem_a + s * TL::TMEM_STAGE + (term == 0 ? BK : 0);
            const uint32_t bt = sb + (TERMS == 3 && term == 1 ? TL::B_BYTES : 0);
#pragma unroll
            for (int k = 0; k < BK / 8; ++k) {
              const uint64_t bdesc = B_MN ? smem_desc(bt + k * 1024, MN_BLOCK_BYTES, 512, kLayoutSw128Base32)
                                          : smem_desc(bt + k * 32, 16, 1024, kLayoutSw128);
              const uint32_t more = (i != cb || term != 0 || k != 0) ? 1u : 0u;
              if (TERMS == 3) {
                umma_tf32_ts(acc, ta + 8 * k, bdesc, idesc, more);
              } else {
                const uint64_t adesc = A_MN ? smem_desc(sa + k * 1024, MN_BLOCK_BYTES, 512, kLayoutSw128Base32)
                                            : smem_desc(sa + k * 32, 16, 1024, kLayoutSw128);
                umma_tf32(acc, adesc, bdesc, idesc, more);
              }
            }
          }
          umma_commit(empty_bar(s));
        }
        if (ok) umma_commit(acc_full(buf));
      }
    }
  } else if (warp >= TL::SUM_WARP) {
    // ---------------- chunk sums: 32 rows x BN / 2 columns per warp, then the partial tile
    constexpr int NC = BN / 2;
    const int quarter = warp & 3, half = (warp - TL::SUM_WARP) >> 2;
    float sum[NC];
#pragma unroll
    for (int e = 0; e < NC; ++e) sum[e] = 0.0f;
    int j = 0;
    bool ok = true;
    for (int cb = kb; cb < ke; cb += TL::CHUNK, ++j) {
      const int buf = j & 1;
      if (!mbar_wait(acc_full(buf), (j >> 1) & 1, err, kErrWaitAccum)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem_base + buf * BN + (static_cast<uint32_t>(quarter * 32) << 16) + half * NC;
#pragma unroll
      for (int c = 0; c < NC / 16; ++c) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(acc + c * 16, r);
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[c * 16 + e] += __uint_as_float(r[e]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(buf));
    }
    if (ok) {
      // Every UMMA of the tile is done, so every stage has landed and been read:
      // the partial tile takes their place, row r's quad q at r BN/4 + (q ^ (r & 7))
      // (eight rows of one quad lie in different banks).
      float4* tile = reinterpret_cast<float4*>(smem);
      const int row = quarter * 32 + lane;
#pragma unroll
      for (int q = 0; q < NC / 4; ++q)
        tile[row * (BN / 4) + ((half * (NC / 4) + q) ^ (row & 7))] =
            make_float4(sum[4 * q], sum[4 * q + 1], sum[4 * q + 2], sum[4 * q + 3]);
      if constexpr (Epi::kOwnSums)
        if (splits == 1) epi.own(sum, m0 + row, n0 + half * NC, M, N, halves + half * BM + row);
    }
  } else if (TERMS == 3 && warp < 4) {
    // ---------------- B's lo part, in the stage's own layout
    for (int i = kb; i < ke; ++i) {
      const int it = i - kb, s = it % TL::STAGES, round = it / TL::STAGES;
      if (!mbar_wait(full_bar(s), round & 1, err, kErrWaitFull)) break;
      const float4* hi = reinterpret_cast<const float4*>(smem + s * TL::STAGE + TL::A_BYTES);
      float4* lo = reinterpret_cast<float4*>(smem + s * TL::STAGE + TL::IN_BYTES);
#pragma unroll 8
      for (int e = threadIdx.x - 64; e < TL::B_BYTES / 16; e += 64) {
        const float4 v = hi[e];
        lo[e] = make_float4(lo_part(v.x), lo_part(v.y), lo_part(v.z), lo_part(v.w));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(lo_bar(s));
    }
  } else if (TERMS == 3) {
    // ---------------- A's rows to tensor memory: lane = row, hi in 32 columns, lo in the next 32
    const int row = 32 * (warp & 3) + lane;
    for (int i = kb; i < ke; ++i) {
      const int it = i - kb, s = it % TL::STAGES, round = it / TL::STAGES;
      if (!mbar_wait(full_bar(s), round & 1, err, kErrWaitFull)) break;
      tc_fence_after();  // the UMMAs that read this stage's columns before are done
      const uint8_t* a = smem + s * TL::STAGE;
      uint32_t hi[32], lo[32];
      if (!A_MN) {  // 16-byte chunk c of row r at chunk c ^ (r & 7)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 v = *reinterpret_cast<const uint4*>(a + row * 128 + ((c ^ (row & 7)) << 4));
          hi[4 * c] = v.x; hi[4 * c + 1] = v.y; hi[4 * c + 2] = v.z; hi[4 * c + 3] = v.w;
        }
      } else {  // 32-wide blocks of 32 K rows; 32-byte chunk c of K row k at chunk c ^ (k & 3)
        const uint8_t* block = a + (warp & 3) * MN_BLOCK_BYTES + (lane & 7) * 4;
#pragma unroll
        for (int k = 0; k < 32; ++k)
          hi[k] = *reinterpret_cast<const uint32_t*>(block + k * 128 + (((lane >> 3) ^ (k & 3)) << 5));
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) lo[e] = __float_as_uint(lo_part(__uint_as_float(hi[e])));
      const uint32_t at = tmem_a + s * TL::TMEM_STAGE + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      tmem_st_32x32b_x32(at, hi);
      tmem_st_32x32b_x32(at + BK, lo);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(lo_bar(s));
    }
  }

  // ---------------- the parts' sums and the epilogue, 128 / splits rows per CTA
  tc_fence_before();
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  const int r0 = BM * part / splits;
  epi.slice(slice * slice_stride)
      .rows(base, halves, m0, n0, r0, BM * (part + 1) / splits - r0, splits, M, N, warp, lane, TL::THREADS / 32);
  if (splits > 1)
    cluster_sync();  // a peer may still be reading this CTA's part
  else
    __syncthreads();
  if (threadIdx.x == 0) {
    // only after a timed-out wait can a stage still be in flight: let it land (bounded)
    for (int i = *loads_consumed; i < *loads_issued; ++i)
      if (!mbar_wait(full_bar(i % TL::STAGES), (i / TL::STAGES) & 1, err, kErrWaitDrain, 1000000000ull)) break;
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TL::TMEM_COLS);
  }
  __syncthreads();
  if (late) after_previous();
}

struct LinearDirect {
  LinearEpilogue e;
  static constexpr bool kOwnSums = false;
  __device__ __forceinline__ bool late() const { return e.late; }
  __device__ __forceinline__ LinearDirect slice(long long offset) const {
    LinearDirect d = *this;
    d.e.C += offset;
    return d;
  }
  // Rows [r0, r0 + nr) of the tile; a warp per row, four rows of a warp at a time
  // so that their loads are in flight together. The tile inside the matrix
  // (FULL) runs without bounds checks: the loop is bound by its instructions.
  template <bool FULL>
  __device__ __forceinline__ void run(uint32_t tile, int m0, int n0, int r0, int nr, int splits, int M, int N,
                                      int warp, int warps, int lane) const {
    const int col = n0 + 4 * lane;
    uint64_t seed = 0, offset = 0;
    const bool drop = e.drop.rng != nullptr;
    if (drop) {
      seed = e.drop.rng[0];
      offset = e.drop.rng[1];
    }
    const float4 bias = bias_quad(e, col, N);
    constexpr int U = 4;
    for (int i = warp; i < nr; i += U * warps) {
      float4 v[U], r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = i + u * warps;
        const long long row = m0 + r0 + j;
        const bool live = j < nr && (FULL || (row < M && col < N));
        v[u] = live ? sum_quad(tile, r0 + j, lane, splits) : make_float4(0.f, 0.f, 0.f, 0.f);
        r[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live && e.R)
          r[u] = FULL ? *reinterpret_cast<const float4*>(e.R + row * e.ldr + col)
                      : load_quad(e.R + row * e.ldr, col, N);
      }
      // Part by part over the batch, so that the path through the code is short and
      // straight: a CTA runs it once, and what it costs is fetching it.
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u].x += bias.x; v[u].y += bias.y; v[u].z += bias.z; v[u].w += bias.w;
      }
      auto put = [&](float* base, long long ld) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = i + u * warps;
          const long long row = m0 + r0 + j;
          if (j < nr && (FULL || (row < M && col < N))) put_quad<FULL>(base + row * ld, col, N, v[u]);
        }
      };
      if (e.Z) put(e.Z, e.ldz);
      activate_quads<U>(v, e.act);
      if (drop)
#pragma unroll
        for (int u = 0; u < U; ++u)
          v[u] = dropout_quad(v[u], e.drop, seed, offset, m0 + r0 + i + u * warps, col >> 2);
      if (e.R)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          v[u].x += r[u].x; v[u].y += r[u].y; v[u].z += r[u].z; v[u].w += r[u].w;
        }
      put(e.C, e.ldc);
    }
  }
  __device__ __forceinline__ void rows(uint32_t tile, const float2*, int m0, int n0, int r0, int nr, int splits, int M,
                                       int N, int warp, int lane, int warps) const {
    if (m0 + r0 + nr <= M && n0 + BN <= N)
      run<true>(tile, m0, n0, r0, nr, splits, M, N, warp, warps, lane);
    else
      run<false>(tile, m0, n0, r0, nr, splits, M, N, warp, warps, lane);
  }
};

struct LossDirect {
  LossEpilogue e;
  static constexpr bool kOwnSums = true;
  __device__ __forceinline__ bool late() const { return false; }
  __device__ __forceinline__ LossDirect slice(long long) const { return *this; }
  // One part: the summing warps hold the row already, half of it each (lane = row): their
  // maximum and sum in registers, the halves joined through shared memory.
  template <int NC>
  __device__ __forceinline__ void own(const float (&sum)[NC], int row, int n0, int M, int N, float2* half_of) const {
    const int live = min(NC, N - n0);
    float m = -INFINITY, s = 0.0f;
    if (live == NC) {
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, all[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NC; ++i) top[i % 4] = fmaxf(top[i % 4], sum[i]);
      m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
#pragma unroll
      for (int i = 0; i < NC; ++i) all[i % 4] += loss_exp(sum[i] - m);
      s = (all[0] + all[1]) + (all[2] + all[3]);
    } else {
#pragma unroll
      for (int i = 0; i < NC; ++i) m = i < live ? fmaxf(m, sum[i]) : m;
#pragma unroll
      for (int i = 0; i < NC; ++i) s += i < live ? loss_exp(sum[i] - m) : 0.0f;
    }
    *half_of = make_float2(m, s);
    if (row < M) {
      const int t = e.targets[row] - n0;
      if (t >= 0 && t < live) {
        float zt = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) zt = i == t ? sum[i] : zt;
        e.zt[row] = zt;
      }
    }
  }
  __device__ __forceinline__ void join(float2 a, float2 b, long long row, int n0) const {
    const float m = fmaxf(a.x, b.x);  // the first half has a column, so b = (-inf, 0) adds nothing
    e.part[row * e.tiles + n0 / 128] = make_float2(m, a.y * loss_exp(a.x - m) + b.y * loss_exp(b.x - m));
  }
  // and the logits, where they are wanted
  __device__ __forceinline__ void store(uint32_t tile, int m0, int n0, int M, int N, int warp, int lane,
                                        int warps) const {
    const int col = n0 + 4 * lane;
    const bool full = col + 3 < N;
#pragma unroll 4
    for (int r = warp; r < BM; r += warps) {
      if (m0 + r >= M) break;  // uniform over the warp
      const float4 v = sum_quad(tile, r, lane, 1);
      float* row = e.Z + static_cast<long long>(m0 + r) * e.ldz;
      if (full)
        *reinterpret_cast<float4*>(row + col) = v;
      else
        store_quad(row, col, N, v);
    }
  }
  // Several parts: a warp per joined row, its 128 columns' maximum and sum by shuffles;
  // three rows at a time.
  __device__ __forceinline__ void rows(uint32_t tile, const float2* halves, int m0, int n0, int r0, int nr, int splits,
                                       int M, int N, int warp, int lane, int warps) const {
    if (splits == 1) {
      const int r = warp * 32 + lane;
      if (r < BM && m0 + r < M) join(halves[r], halves[BM + r], m0 + r, n0);
      if (e.Z) store(tile, m0, n0, M, N, warp, lane, warps);
      return;
    }
    const int col = n0 + 4 * lane;
    constexpr int U = 3;
    for (int i = warp; i < nr && m0 + r0 + i < M; i += U * warps) {  // uniform over the warp
      float4 v[U];
      float m[U], s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = min(i + u * warps, nr - 1);
        v[u] = sum_quad(tile, r0 + j, lane, splits);
        m[u] = col < N ? quad_max(v[u], col, N) : -INFINITY;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) m[u] = fmaxf(m[u], __shfl_xor_sync(0xffffffffu, m[u], o));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = 0.0f;
        if (col < N) s[u] += loss_exp(v[u].x - m[u]);
        if (col + 1 < N) s[u] += loss_exp(v[u].y - m[u]);
        if (col + 2 < N) s[u] += loss_exp(v[u].z - m[u]);
        if (col + 3 < N) s[u] += loss_exp(v[u].w - m[u]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = i + u * warps;
        const long long row = m0 + r0 + j;
        if (j >= nr || row >= M) break;
        if (lane == 0) e.part[row * e.tiles + n0 / 128] = make_float2(m[u], s[u]);
        const int t = e.targets[row] - col;
        if (t >= 0 && t < 4 && col + t < N) e.zt[row] = t == 0 ? v[u].x : t == 1 ? v[u].y : t == 2 ? v[u].z : v[u].w;
        if (e.Z && col < N) store_quad(e.Z + row * e.ldz, col, N, v[u]);
      }
    }
  }
};

// ------------------------------------------------------------------ few rows
// Up to eight rows: bound by one reading of B, so the products are plain f32
// multiply-adds on B as it streams by (a 128-row tensor-core tile would convert and
// multiply 120 rows of nothing: one row of 2048 x 5632 took 30 us in it). A CTA
// takes 32 columns and a part of K, a cluster's parts meet in shared memory, in part
// order. B [k, n]: eight lanes hold the 32 columns of a k, a warp four k at a time,
// eight loads in flight; B [n, k]: a warp takes four columns, its lanes lie along k.
// A's values of 512 k at a time are kept in shared memory. One row of 2048 x 5632 11.2 us
// with twelve such weights in rotation (4.1 TB/s of B from HBM), 7.7 us with one, which
// stays in the L2; 4096 x 11264, larger than the L2, 36 us (5.1). What the small one lacks
// is loads in flight: a CTA's run dry at the end of each piece of 512.
constexpr int kFewRows = 8;
constexpr int kFewPiece = 512;
constexpr int kFewCols = 32;

// v[0 .. n) summed over the warp's lanes; value i ends in the lanes whose top bits
// (log2 n of them) spell i, in v[0]. Half of the values change hands at each step.
template <int N_VALUES>
__device__ __forceinline__ void warp_sums(float (&v)[N_VALUES], int lane) {
  int o = 16;
#pragma unroll
  for (int n = N_VALUES; n > 1; n >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float give = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
}

constexpr int few_blocks(int mt) { return mt <= 4 ? 4 : 3; }  // CTAs of an SM, by registers

template <int MT, bool B_MN>
__global__ void __launch_bounds__(256, few_blocks(MT))
    few_rows_kernel(const float* a, long long lda, const float* b, long long ldb, LinearEpilogue e, int M, int N, int K,
                    int splits, int slices, long long slice_stride) {
  if (!e.late) after_previous();
  let_next();
  __shared__ __align__(16) float as[kFewPiece * MT];
  __shared__ __align__(16) float sums[(B_MN ? 8 : 1) * MT * kFewCols];  // [warps][MT][32], then [MT][32]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int part = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tiles = (N + kFewCols - 1) / kFewCols, cluster = static_cast<int>(blockIdx.x) / splits;
  const int slice = cluster / tiles, n0 = (cluster - slice * tiles) * kFewCols;
  e.C += slice * slice_stride;
  const int units = (K + 31) / 32;  // parts are cut at multiples of 32
  const long long kpart = static_cast<long long>(slice) * splits + part;
  const long long kparts = static_cast<long long>(slices) * splits;
  const int kb = static_cast<int>(units * kpart / kparts) * 32;
  const int ke = min(K, static_cast<int>(units * (kpart + 1) / kparts) * 32);
  float acc[4 * MT];  // [MT][4 columns]
#pragma unroll
  for (int i = 0; i < 4 * MT; ++i) acc[i] = 0.0f;

  for (int k0 = kb; k0 < ke; k0 += kFewPiece) {
    const int kn = min(kFewPiece, ke - k0);
    if (k0 > kb) __syncthreads();
    // B [k, n]: the rows of one k side by side; B [n, k]: k side by side
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < kFewPiece / 256; ++h) {
        const int k = threadIdx.x + 256 * h;
        as[B_MN ? k * MT + m : m * kFewPiece + k] = m < M && k < kn ? a[m * lda + k0 + k] : 0.0f;
      }
    __syncthreads();
    if (B_MN) {
      const int col = n0 + 4 * (lane & 7), kl = 4 * warp + (lane >> 3);
      auto add = [&](int k, float4 w) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float x = as[k * MT + m];
          acc[4 * m] = fmaf(x, w.x, acc[4 * m]);
          acc[4 * m + 1] = fmaf(x, w.y, acc[4 * m + 1]);
          acc[4 * m + 2] = fmaf(x, w.z, acc[4 * m + 2]);
          acc[4 * m + 3] = fmaf(x, w.w, acc[4 * m + 3]);
        }
      };
      if (n0 + kFewCols <= N) {
        for (int k = kl; k < kn; k += 256) {
          float4 w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)  // past the piece: any row of it, not added
            w[i] = *reinterpret_cast<const float4*>(b + (k0 + min(k + 32 * i, kn - 1)) * ldb + col);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (k + 32 * i < kn) add(k + 32 * i, w[i]);
        }
      } else if (col < N) {
        for (int k = kl; k < kn; k += 32) add(k, load_quad(b + (k0 + k) * ldb, col, N));
      }
    } else {
      const int c0 = n0 + 4 * warp;
      const bool whole = c0 + 4 <= N && kn % 128 == 0;
      const float* col = b + c0 * ldb + k0;
#pragma unroll 2
      for (int k = 4 * lane; k < kn; k += 128) {
        float4 w[4];
        if (whole) {
#pragma unroll
          for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const float4*>(col + c * ldb + k);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            w[c] = c0 + c < N ? load_quad(col + c * ldb, k, kn) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float4 x = *reinterpret_cast<const float4*>(as + m * kFewPiece + k);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float& o = acc[4 * m + c];
            o = fmaf(x.x, w[c].x, o);
            o = fmaf(x.y, w[c].y, o);
            o = fmaf(x.z, w[c].z, o);
            o = fmaf(x.w, w[c].w, o);
          }
        }
      }
    }
  }
  if (B_MN) {
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i) {  // the warp's four k
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 8);
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 16);
    }
    if (lane < 8)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        reinterpret_cast<float4*>(sums)[(warp * MT + m) * 8 + lane] =
            make_float4(acc[4 * m], acc[4 * m + 1], acc[4 * m + 2], acc[4 * m + 3]);
    __syncthreads();
    for (int i = threadIdx.x; i < MT * kFewCols; i += 256) {
      float s = sums[i];
      for (int w = 1; w < 8; ++w) s += sums[w * MT * kFewCols + i];
      sums[i] = s;
    }
  } else {
    warp_sums(acc, lane);
    constexpr int SAME = 32 / (4 * MT);  // lanes that hold the same value
    const int i = lane / SAME;
    if (lane % SAME == 0) sums[(i / 4) * kFewCols + 4 * warp + i % 4] = acc[0];
  }
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  const bool drop = e.drop.rng != nullptr;
  for (int i = threadIdx.x * splits + part; i < MT * (kFewCols / 4); i += 256 * splits) {
    const int row = i / (kFewCols / 4), q = i % (kFewCols / 4), col = n0 + 4 * q;
    if (row >= M || col >= N) continue;
    const float4 r = e.R ? load_quad(e.R + row * e.ldr, col, N) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 bias = bias_quad(e, col, N);
    float4 v = reinterpret_cast<const float4*>(sums)[i];
    if (splits > 1) {
      const uint32_t at = smem_u32(sums) + 16u * i;
      float4 w[8];
#pragma unroll
      for (int p = 0; p < 8; ++p)
        w[p] = p < splits ? ld_cluster_quad(mapa_shared(at, p)) : make_float4(0.f, 0.f, 0.f, 0.f);
      v = w[0];
#pragma unroll
      for (int p = 1; p < 8; ++p) {
        v.x += w[p].x; v.y += w[p].y; v.z += w[p].z; v.w += w[p].w;
      }
    }
    linear_quad(e, e.act, drop, drop ? e.drop.rng[0] : 0, drop ? e.drop.rng[1] : 0, row, col, N, v, bias, r);
  }
  if (splits > 1) cluster_sync();  // a peer may still be reading this CTA's part
  if (e.late) after_previous();
}

// ------------------------------------------------------------------ K slices
// The slices' sums [slices][M, ld], in slice order, and the epilogue: a thread per quad.
__global__ void __launch_bounds__(256) join_kernel(const float* parts, int slices, long long slice_stride,
                                                   long long ld, const LinearEpilogue e, int M, int N) {
  after_previous();
  let_next();
  const int quads = (N + 3) / 4;
  const long long i = blockIdx.x * 256ll + threadIdx.x, row = i / quads;
  const int col = 4 * static_cast<int>(i - row * quads);
  if (row >= M) return;
  const float* p = parts + row * ld + col;
  float4 v = *reinterpret_cast<const float4*>(p);  // ld is N rounded up to 4
#pragma unroll 4
  for (int k = 1; k < slices; ++k) {
    const float4 o = *reinterpret_cast<const float4*>(p + k * slice_stride);
    v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
  }
  const bool drop = e.drop.rng != nullptr;
  const float4 r = e.R ? load_quad(e.R + row * e.ldr, col, N) : make_float4(0.f, 0.f, 0.f, 0.f);
  linear_quad(e, e.act, drop, drop ? e.drop.rng[0] : 0, drop ? e.drop.rng[1] : 0, row, col, N, v, bias_quad(e, col, N),
              r);
}

// ------------------------------------------------------------------ backward of the epilogue
// dz and the column sums' partials: 64 rows (16 of a small matrix, for enough blocks) x
// 128 columns per block, a warp per row, so every access covers 512 contiguous bytes.
// Bound by HBM: 4 (dc) + 4 (z) + 4 (dz) bytes an element.
int act_rows(int rows, int cols) {
  return ((rows + 63ll) / 64) * ((cols + 127ll) / 128) >= 2 * 148 ? 64 : 16;
}

__global__ void __launch_bounds__(256) act_backward_kernel(const float* dc, long long lddc, const float* z,
                                                           long long ldz, int act, DropoutArgs drop, int rows,
                                                           int cols, int block_rows, float* dz, long long lddz,
                                                           float* part) {
  after_previous();
  let_next();
  __shared__ float4 sums[8][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int across = (cols + 127) / 128, band = static_cast<int>(blockIdx.x) / across;
  const int col = ((static_cast<int>(blockIdx.x) - band * across) * 32 + lane) * 4;
  const int row0 = band * block_rows;
  uint64_t seed = 0, offset = 0;
  if (drop.rng) {
    seed = drop.rng[0];
    offset = drop.rng[1];
  }
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < cols) {
#pragma unroll 4
    for (int i = warp; i < block_rows; i += 8) {
      const long long row = row0 + i;
      if (row >= rows) break;
      float4 g = load_quad(dc + row * lddc, col, cols);
      if (drop.rng) g = dropout_quad(g, drop, seed, offset, row, col >> 2);
      if (act != kActNone) {
        const float4 v = load_quad(z + row * ldz, col, cols);
        g.x *= activate_slope(v.x, act); g.y *= activate_slope(v.y, act);
        g.z *= activate_slope(v.z, act); g.w *= activate_slope(v.w, act);
      }
      if (dz) store_quad(dz + row * lddz, col, cols, g);
      sum.x += g.x; sum.y += g.y; sum.z += g.z; sum.w += g.w;
    }
  }
  if (!part) return;  // uniform
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && col < cols) {
    for (int w = 1; w < 8; ++w) {
      const float4 o = sums[w][lane];
      sum.x += o.x; sum.y += o.y; sum.z += o.z; sum.w += o.w;
    }
    float* p = part + static_cast<long long>(band) * cols;  // rows of `cols`: any alignment
    p[col] = sum.x;
    if (col + 1 < cols) p[col + 1] = sum.y;
    if (col + 2 < cols) p[col + 2] = sum.z;
    if (col + 3 < cols) p[col + 3] = sum.w;
  }
}

// 32 columns per block, eight rows of partials at a time, joined in a fixed order.
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* part, int parts, int cols, float* out,
                                                        int accumulate) {
  after_previous();
  let_next();
  __shared__ double sums[8][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, col = blockIdx.x * 32 + lane;
  double s = 0.0;
  if (col < cols)
    for (int p = warp; p < parts; p += 8) s += part[static_cast<long long>(p) * cols + col];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < cols) {
    for (int w = 1; w < 8; ++w) s += sums[w][lane];
    out[col] = static_cast<float>(accumulate ? out[col] + s : s);
  }
}

// ------------------------------------------------------------------ dropout
// y = r + dropout(x): a thread takes quads, U in flight. Bound by HBM (8 bytes an
// element, 12 with r: 8192 x 2048 with r 35.5 us, 5.7 TB/s; 31.3 without the mask) and,
// without r, by the generator's twenty 32 x 32 -> 64 multiplications for four elements
// (8192 x 5632: 78 us, 61 without the mask). A 64-bit division by the row's quads would
// cost as much again, so numbers that fit are divided in 32 bits. Four in flight where
// that leaves threads enough (1024 x 1024 with r 3.7 us with one, 5.7 with four; 8192 x
// 5632 without the mask 74 us with two, 61 with four).
template <bool VEC, int U, class Index>
__global__ void __launch_bounds__(256) dropout_kernel(const float* x, long long ldx, const float* r, long long ldr,
                                                      float* y, long long ldy, Index quads, int cols,
                                                      DropoutArgs drop) {
  after_previous();
  let_next();
  const uint64_t seed = drop.rng ? drop.rng[0] : 0, offset = drop.rng ? drop.rng[1] : 0;
  const Index step = static_cast<Index>(gridDim.x) * 256;
  for (long long first = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; first < quads; first += U * step) {
    long long row[U];
    int quad[U];
    float4 v[U], a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long at = first + u * static_cast<long long>(step);
      const Index i = static_cast<Index>(at < quads ? at : first);
      const Index q = i / drop.blocks;
      row[u] = static_cast<long long>(q);
      quad[u] = static_cast<int>(i - q * drop.blocks);
      const float *xp = x + row[u] * ldx, *rp = r + row[u] * ldr;
      v[u] = VEC ? load_quad(xp, 4 * quad[u], cols) : load_each(xp, 4 * quad[u], cols);
      a[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r) a[u] = VEC ? load_quad(rp, 4 * quad[u], cols) : load_each(rp, 4 * quad[u], cols);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u > 0 && first + u * static_cast<long long>(step) >= quads) break;
      if (drop.rng) v[u] = dropout_quad(v[u], drop, seed, offset, row[u], quad[u]);
      v[u].x += a[u].x; v[u].y += a[u].y; v[u].z += a[u].z; v[u].w += a[u].w;
      float* yp = y + row[u] * ldy;
      if (VEC)
        store_quad(yp, 4 * quad[u], cols, v[u]);
      else
        store_each(yp, 4 * quad[u], cols, v[u]);
    }
  }
}

// ------------------------------------------------------------------ host side
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// How K is cut: into parts (a cluster's CTAs) and slices (clusters), by the shortest
// time from waves of clusters, steps of a part and a tile's fixed cost. A cluster lies
// in one GPC, so fewer CTAs run at once in larger ones (the occupancy query's counts for
// this kernel on a B200; a device with other GPCs runs the same plan in other waves). A
// step takes 0.66 us (a fit over whole calls, between the loop's own 0.58 and the 0.74 of
// tiles that share nothing), a tile's start and end 5.5, the parts' join 0.5, the slices' launch
// and their sums 3, some of it the host's (2048 x 4096 -> 128 in six parts takes 24.7 us, in
// nine slices 21.4, in four parts of two slices 22.0; 128 x 2048 -> 2048 16.8, 16.0 and 16.1;
// 4096 x 2048 -> 128 in four parts 20.0, in four slices 21.6; 64 x 32000 -> 512 in eight
// parts alone 80, in four of eight slices 34). (128 x 64 tiles, tried for more CTAs, took
// 0.69 us a step: a UMMA of half the width is no shorter.)
struct Cut {
  int splits = 1, slices = 1;
};
Cut direct_cut(int M, int N, int K, bool sliced) {
  constexpr int kFit[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
  const long long tiles = static_cast<long long>((M + BM - 1) / BM) * ((N + 127) / 128);
  const int n_k = (K + BK - 1) / BK;
  Cut best;
  double best_us = 1e30;
  for (int s = 1; s <= 8 && (s == 1 || n_k >= 4 * s); ++s)
    for (int l = 1; l <= (sliced ? 32 : 1) && (l == 1 || (n_k >= 8 * s * l && tiles * l <= kFit[s])); ++l) {
      const double waves = static_cast<double>((tiles * l + kFit[s] - 1) / kFit[s]);
      const double us = waves * ((n_k + s * l - 1) / (s * l) * 0.66 + 5.5 + (s > 1 ? 0.5 : 0.0)) + (l > 1 ? 3.0 : 0.0);
      if (us < best_us) {
        best = {s, l};
        best_us = us;
      }
    }
  return best;
}

// Few rows: parts that all run at once, each at least 128 of K, then slices while one
// has more than 2048 of it. Parts by powers of two, which leave whole pieces of K (2048 ->
// 5632 by [n, k], four rows: two parts 12.6 us, three 13.5), but six where five to eight
// rows leave no room for eight (8 x 5632 -> 2048 16.6 us, 21.8 in four; 8 x 2048 -> 2048 9.7
// and 10.2).
Cut few_cut(int M, int N, int K) {
  const int fit = few_blocks(M <= 4 ? 4 : 8) * 148;
  const long long tiles = (N + kFewCols - 1) / kFewCols;
  Cut c;
  while (c.splits < 8 && tiles * c.splits * 2 <= fit && K / (2 * c.splits) >= 128) c.splits *= 2;
  if (M > 4 && c.splits == 4 && tiles * 6 <= fit && K / 6 >= 256) c.splits = 6;
  while (tiles * c.splits * c.slices * 2 <= fit && K / (c.splits * c.slices * 2) >= 1024) c.slices *= 2;
  return c;
}

Cut cut_of(int M, int N, int K, bool a_mn_major) {
  return M <= kFewRows && !a_mn_major ? few_cut(M, N, K) : direct_cut(M, N, K, true);
}

long long slice_floats(int M, int N) { return M * ((N + 3ll) & ~3ll); }

template <int TERMS, bool A_MN, bool B_MN, class Epi>
int launch_direct(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const Epi& epi, Cut cut,
                  int* d_err, cudaStream_t s) {
  using TL = DirectTile<TERMS>;
  CUtensorMap ta{}, tb{};
  bool a3 = false, b3 = false;
  int rc = operand_map(&ta, A, M, K, BM, &a3);
  if (!rc) rc = operand_map(&tb, B, N, K, BN, &b3);
  if (rc) return rc;
  auto kern = direct_kernel<TERMS, A_MN, B_MN, Epi>;
  static thread_local int configured_device = -1;
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (configured_device != dev) {
    check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TL::SMEM), "shared memory");
    configured_device = dev;
  }
  const long long tiles = static_cast<long long>((M + BM - 1) / BM) * ((N + BN - 1) / BN);
  if (tiles * cut.splits * cut.slices > 0x7fffffffll) return kGemmBadArgument;
  launch_next("linear", kern, dim3(static_cast<unsigned>(tiles * cut.slices * cut.splits)), TL::THREADS, TL::SMEM,
              cut.splits, s, ta, tb, epi, M, N, K, cut.splits, cut.slices, slice_floats(M, N),
              (a3 ? 1 : 0) | (b3 ? 2 : 0), d_err);
  return 0;
}

template <int MT>
void launch_few(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LinearEpilogue& e, Cut cut,
                cudaStream_t s) {
  const long long clusters = (N + kFewCols - 1) / kFewCols * static_cast<long long>(cut.slices);
  auto kern = B.mn_major ? few_rows_kernel<MT, true> : few_rows_kernel<MT, false>;
  launch_next("linear", kern, dim3(static_cast<unsigned>(clusters * cut.splits)), 256, 0, cut.splits, s, A.ptr, A.ld,
              B.ptr, B.ld, e, M, N, K, cut.splits, cut.slices, slice_floats(M, N));
}

template <int TERMS, class Epi>
int direct_majors(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const Epi& epi, Cut cut,
                  int* d_err, cudaStream_t s) {
  if (!A.mn_major && !B.mn_major) return launch_direct<TERMS, false, false>(M, N, K, A, B, epi, cut, d_err, s);
  if (!A.mn_major) return launch_direct<TERMS, false, true>(M, N, K, A, B, epi, cut, d_err, s);
  if (B.mn_major) return launch_direct<TERMS, true, true>(M, N, K, A, B, epi, cut, d_err, s);
  return kGemmBadArgument;  // no caller has an MN-major A with a K-major B
}

}  // namespace

int operand_map(CUtensorMap* map, const GemmOperand& o, int mn, int k, int box, bool* box3d) {
  if ((o.ld & 3) || !aligned16(o.ptr)) return kGemmMisaligned;
  *box3d = false;
  int rc;
  if (!o.mn_major) {
    const long long dims[2] = {k, mn}, strides[1] = {o.ld};
    const int b[2] = {BK, box};
    rc = encode_tensor_map(map, o.ptr, 2, dims, strides, b, false);
  } else if (mn % 32 == 0) {
    const long long dims[3] = {32, k, mn / 32}, strides[2] = {o.ld, 32};
    const int b[3] = {32, BK, box / 32};
    *box3d = true;
    rc = encode_tensor_map(map, o.ptr, 3, dims, strides, b, true);
  } else {
    const long long dims[2] = {mn, k}, strides[1] = {o.ld};
    const int b[2] = {32, BK};
    rc = encode_tensor_map(map, o.ptr, 2, dims, strides, b, true);
  }
  return rc ? kGemmTensorMap : 0;
}

DropoutArgs dropout_args(double p, const uint64_t* rng, int cols) {
  DropoutArgs d;
  d.blocks = static_cast<uint32_t>((static_cast<long long>(cols) + 3) / 4);
  if (p > 0.0) {
    d.rng = rng;
    d.threshold = static_cast<uint32_t>(p * 4294967296.0);
    d.scale = static_cast<float>(1.0 / (1.0 - p));
  }
  return d;
}

long long direct_ws_bytes(int M, int N, int K, bool a_mn_major) {
  if (M <= 0 || N <= 0) return 0;
  const Cut c = cut_of(M, N, K, a_mn_major);
  return c.slices > 1 ? c.slices * slice_floats(M, N) * 4 : 0;
}

int direct_product(int M, int N, int K, GemmOperand A, GemmOperand B, const LinearEpilogue& e, bool exact, void* ws,
                   int* d_err, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  const Cut cut = cut_of(M, N, K, A.mn_major);
  LinearEpilogue raw;  // a slice's sums as they are
  raw.C = static_cast<float*>(ws);
  raw.ldc = (N + 3ll) & ~3ll;
  raw.late = e.late;
  const LinearEpilogue& out = cut.slices > 1 ? raw : e;
  if (M <= kFewRows && !A.mn_major) {
    if (M == 1) launch_few<1>(M, N, K, A, B, out, cut, s);
    else if (M == 2) launch_few<2>(M, N, K, A, B, out, cut, s);
    else if (M <= 4) launch_few<4>(M, N, K, A, B, out, cut, s);
    else launch_few<8>(M, N, K, A, B, out, cut, s);
  } else {
    const int rc = exact ? direct_majors<3>(M, N, K, A, B, LinearDirect{out}, cut, d_err, s)
                         : direct_majors<1>(M, N, K, A, B, LinearDirect{out}, cut, d_err, s);
    if (rc) return rc;
  }
  if (cut.slices > 1) {
    const long long quads = M * ((N + 3ll) / 4);
    launch_next("linear", join_kernel, dim3(static_cast<unsigned>((quads + 255) / 256)), 256, 0, 1, s, raw.C, cut.slices,
                slice_floats(M, N), raw.ldc, e, M, N);
  }
  return 0;
}

int direct_loss_product(int M, int N, int K, GemmOperand A, GemmOperand B, const LossEpilogue& e, bool exact,
                        int* d_err, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  if (A.mn_major) return kGemmBadArgument;
  const LossDirect epi{e};
  const Cut cut = direct_cut(M, N, K, false);
  if (exact)
    return B.mn_major ? launch_direct<3, false, true>(M, N, K, A, B, epi, cut, d_err, s)
                      : launch_direct<3, false, false>(M, N, K, A, B, epi, cut, d_err, s);
  return B.mn_major ? launch_direct<1, false, true>(M, N, K, A, B, epi, cut, d_err, s)
                    : launch_direct<1, false, false>(M, N, K, A, B, epi, cut, d_err, s);
}

int act_backward_parts(int rows, int cols) {
  const int r = act_rows(rows, cols);
  return (rows + r - 1) / r;
}

void act_backward(const float* dc, long long lddc, const float* z, long long ldz, int act, const DropoutArgs& d,
                  int rows, int cols, float* dz, long long lddz, float* part, cudaStream_t s) {
  if (rows <= 0 || cols <= 0) return;
  const long long blocks = (cols + 127ll) / 128 * act_backward_parts(rows, cols);
  if (blocks > INT32_MAX) throw std::invalid_argument("a matrix is too large");
  launch_next("linear backward", act_backward_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, 1, s, dc, lddc, z, ldz,
              act, d, rows, cols, act_rows(rows, cols), dz, lddz, part);
}

void sum_parts(const float* part, int parts, int cols, float* out, bool accumulate, cudaStream_t s) {
  if (cols <= 0) return;
  launch_next("bias gradient", sum_parts_kernel, dim3((cols + 31) / 32), 256, 0, 1, s, part, parts, cols, out,
              accumulate ? 1 : 0);
}

void dropout(const float* x, long long ldx, const float* r, long long ldr, float* y, long long ldy, long long rows,
             int cols, const DropoutArgs& d, cudaStream_t s) {
  const long long quads = rows * d.blocks;
  if (quads <= 0) return;
  const bool vec = !((ldx | ldy | (r ? ldr : 0)) & 3) && aligned16(x) && aligned16(y) && (!r || aligned16(r));
  const int blocks = static_cast<int>(std::min((quads + 255) / 256, 148ll * 16));
  auto run = [&](auto kernel, auto n) {
    launch_next("dropout", kernel, dim3(blocks), 256, 0, 1, s, x, ldx, r, ldr, y, ldy, n, cols, d);
  };
  if (quads > INT32_MAX)
    vec ? run(dropout_kernel<true, 4, long long>, quads) : run(dropout_kernel<false, 4, long long>, quads);
  else if (quads >= 1 << 21)
    vec ? run(dropout_kernel<true, 4, uint32_t>, static_cast<uint32_t>(quads))
        : run(dropout_kernel<false, 4, uint32_t>, static_cast<uint32_t>(quads));
  else
    vec ? run(dropout_kernel<true, 1, uint32_t>, static_cast<uint32_t>(quads))
        : run(dropout_kernel<false, 1, uint32_t>, static_cast<uint32_t>(quads));
}

}  // namespace mm
