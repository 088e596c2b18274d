// Device code shared by the kernels of linear.cu and linear_pair.cu: overlapping launches,
// activations and their slopes, the order of tiles, four-column loads and stores, and the
// linear epilogue.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "dropout.cuh"
#include "device.h"
#include "linear.h"
#include "ptx.cuh"

namespace mm {

// Launches one after another on a stream: a kernel may start while the one before it
// ends, so that its launch and its prologue are hidden (1 to 2 us a launch, of calls that
// make four to eight short ones). Every thread of every kernel here waits for the one
// before it to be complete and visible (`after_previous`) before it touches global
// memory, then lets the next start (`let_next`); kernels launched in any other way wait
// for everything before them as ever. So completion passes along the chain, and when a
// kernel starts, everything before its predecessor is complete. (Nothing is loaded as
// read-only for the kernel's lifetime, which begins before the one that wrote it ends.)
//
// A product that needs nothing of its predecessor, only of what came before that, may run
// beside it (`late`): it lets the next start at once and waits at its end, when it holds
// no tensor memory, so that its completion still means that of everything before it.
// Several in a row may need what came before the last kernel that waits at its start.
// Which kernels those are must not change between a call's launches, so calls with late
// products are enqueued one at a time (`launch_order`): another thread's late product on
// the same stream, put between a kernel and the one that counts on its end, would break it.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... Params, class... Args>
void launch_next(const char* what, void (*kernel)(Params...), dim3 grid, int threads, int smem, int cluster,
                 cudaStream_t s, const Args&... args) {
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

// The normal distribution function and its density, branch-free (the epilogue runs on
// few warps, so a divergent erff costs both of its paths): C. Hastings' rational
// approximation of erfc (Abramowitz and Stegun, 7.1.26), at most 0.75e-7 off in exact
// arithmetic and 3.4e-7 in this one, taken on the side where nothing cancels. GELU's own
// relative error is 7e-7 down to z = -1, and grows in the tail: 3e-6 at -2, 5e-5 at -3.
__device__ __forceinline__ float normal_cdf(float z, float* density) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f));
  const float e = ex2_approx(z * z * -0.72134752044448170f);  // exp(-z^2 / 2)
  const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f),
                              0.254829592f);
  const float tail = 0.5f * poly * e;
  *density = 0.39894228040143268f * e;
  return z >= 0.0f ? 1.0f - tail : tail;
}
__device__ __forceinline__ float logistic(float z) {
  return __fdividef(1.0f, 1.0f + ex2_approx(z * -1.4426950408889634f));  // 0 where the exponential overflows
}

__device__ __forceinline__ float activate(float z, int act) {
  float density;
  switch (act) {
    case kActRelu: return z < 0.0f ? 0.0f : z;  // a NaN stays
    case kActGelu: return z * normal_cdf(z, &density);
    case kActSilu: return z * logistic(z);
    default: return z;
  }
}

// d act / dz
__device__ __forceinline__ float activate_slope(float z, int act) {
  float density;
  switch (act) {
    case kActRelu: return z <= 0.0f ? 0.0f : 1.0f;
    case kActGelu: {
      const float cdf = normal_cdf(z, &density);
      return fmaf(z, density, cdf);
    }
    case kActSilu: {
      const float s = logistic(z);
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
  }
}

// The activation of U quads, one branch for all of them.
template <int U>
__device__ __forceinline__ void activate_quads(float4 (&v)[U], int act) {
  auto each = [&](auto f) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].x = f(v[u].x); v[u].y = f(v[u].y); v[u].z = f(v[u].z); v[u].w = f(v[u].w);
    }
  };
  switch (act) {
    case kActRelu: each([](float z) { return activate(z, kActRelu); }); break;
    case kActGelu: each([](float z) { return activate(z, kActGelu); }); break;
    case kActSilu: each([](float z) { return activate(z, kActSilu); }); break;
    default: break;
  }
}

// Tiles in groups of 8 row blocks, the row block fastest inside a group: the tiles at
// work at one time then share rows of A and columns of B in L2.
__device__ __forceinline__ void tile_mn(int t, int tm, int tn, int& mt, int& nt) {
  const int per_group = 8 * tn;
  const int g = t / per_group, r = t - g * per_group;
  const int rows = min(8, tm - g * 8);
  mt = g * 8 + r % rows;
  nt = r / rows;
}

// Four columns of a row; those at n and past it are not touched.
__device__ __forceinline__ float4 load_quad(const float* row, int col, int n) {
  if (col + 3 < n) return *reinterpret_cast<const float4*>(row + col);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < n) v.x = row[col];
  if (col + 1 < n) v.y = row[col + 1];
  if (col + 2 < n) v.z = row[col + 2];
  return v;
}
__device__ __forceinline__ void store_quad(float* row, int col, int n, float4 v) {
  if (col + 3 < n) {
    *reinterpret_cast<float4*>(row + col) = v;
    return;
  }
  if (col < n) row[col] = v.x;
  if (col + 1 < n) row[col + 1] = v.y;
  if (col + 2 < n) row[col + 2] = v.z;
}
__device__ __forceinline__ float4 load_each(const float* row, int col, int n) {  // any alignment
  return make_float4(col < n ? row[col] : 0.f, col + 1 < n ? row[col + 1] : 0.f, col + 2 < n ? row[col + 2] : 0.f,
                     col + 3 < n ? row[col + 3] : 0.f);
}
__device__ __forceinline__ void store_each(float* row, int col, int n, float4 v) {
  if (col < n) row[col] = v.x;
  if (col + 1 < n) row[col + 1] = v.y;
  if (col + 2 < n) row[col + 2] = v.z;
  if (col + 3 < n) row[col + 3] = v.w;
}
// v: the product's four columns; bias and r: the bias's and the residual's (r loaded by
// the caller before anything of the batch is stored, so that it may be c). FULL: all
// four columns lie inside, which leaves the unrolled loops one block of straight code.
template <bool FULL>
__device__ __forceinline__ void put_quad(float* row, int col, int n, float4 v) {
  if (FULL)
    *reinterpret_cast<float4*>(row + col) = v;
  else
    store_quad(row, col, n, v);
}
template <bool FULL = false>
__device__ __forceinline__ void linear_quad(const LinearEpilogue& e, int act, bool drop, uint64_t seed,
                                            uint64_t offset, long long row, int col, int n, float4 v, float4 bias,
                                            float4 r) {
  v.x += bias.x; v.y += bias.y; v.z += bias.z; v.w += bias.w;
  if (e.Z) put_quad<FULL>(e.Z + row * e.ldz, col, n, v);
  if (act != kActNone) {
    v.x = activate(v.x, act); v.y = activate(v.y, act); v.z = activate(v.z, act); v.w = activate(v.w, act);
  }
  if (drop) v = dropout_quad(v, e.drop, seed, offset, row, col >> 2);
  v.x += r.x; v.y += r.y; v.z += r.z; v.w += r.w;
  put_quad<FULL>(e.C + row * e.ldc, col, n, v);
}
__device__ __forceinline__ float4 bias_quad(const LinearEpilogue& e, int col, int n) {
  return e.bias ? load_each(e.bias, col, n) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// e^x for the softmax, x <= 0: 2^(x log2 e) on the special-function unit. Relative error
// 2^-22 and, as the product is rounded, |x| 2^-24: 2^-18 for what counts e^-60.
__device__ __forceinline__ float loss_exp(float x) { return ex2_approx(x * 1.4426950408889634f); }

__device__ __forceinline__ float quad_max(float4 v, int col, int n) {  // col < n
  float m = v.x;
  if (col + 1 < n) m = fmaxf(m, v.y);
  if (col + 2 < n) m = fmaxf(m, v.z);
  if (col + 3 < n) m = fmaxf(m, v.w);
  return m;
}

}  // namespace mm
