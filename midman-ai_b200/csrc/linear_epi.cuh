// Device code shared by the kernels of linear.cu and linear_pair.cu: activations
// and their slopes, four-column loads and stores, and the linear epilogue.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "dropout.cuh"
#include "linear.h"
#include "ptx.cuh"

namespace mm {

__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case kActRelu: return fmaxf(z, 0.0f);
    case kActGelu: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case kActSilu: return z / (1.0f + expf(-z));
    default: return z;
  }
}

// d act / dz
__device__ __forceinline__ float activate_slope(float z, int act) {
  switch (act) {
    case kActRelu: return z > 0.0f ? 1.0f : 0.0f;
    case kActGelu:
      return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    case kActSilu: {
      const float s = 1.0f / (1.0f + expf(-z));
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
  }
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
// v: the product's four columns; r: the residual's (loaded by the caller before
// anything of the batch is stored, so that r may be c).
__device__ __forceinline__ void linear_quad(const LinearEpilogue& e, uint64_t seed, uint64_t offset, long long row,
                                            int col, int n, float4 v, float4 r) {
  if (e.bias) {
    const float4 b = load_each(e.bias, col, n);
    v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
  }
  if (e.Z) store_quad(e.Z + row * e.ldz, col, n, v);
  if (e.act != kActNone) {
    v.x = activate(v.x, e.act); v.y = activate(v.y, e.act); v.z = activate(v.z, e.act); v.w = activate(v.w, e.act);
  }
  if (e.drop.rng) v = dropout_quad(v, e.drop, seed, offset, row, col >> 2);
  v.x += r.x; v.y += r.y; v.z += r.z; v.w += r.w;
  store_quad(e.C + row * e.ldc, col, n, v);
}

// e^x for the softmax: 2^(x log2 e) on the special-function unit, 2^-22 relative.
__device__ __forceinline__ float loss_exp(float x) { return ex2_approx(x * 1.4426950408889634f); }

__device__ __forceinline__ float quad_max(float4 v, int col, int n) {  // col < n
  float m = v.x;
  if (col + 1 < n) m = fmaxf(m, v.y);
  if (col + 2 < n) m = fmaxf(m, v.z);
  if (col + 3 < n) m = fmaxf(m, v.w);
  return m;
}

}  // namespace mm
