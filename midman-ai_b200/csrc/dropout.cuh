// Dropout from a counter-based generator: the mask is a function of (seed,
// offset, row, column) and is formed again wherever it is needed, never stored.
//
// Generator: Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011), 128-bit counter and
// 64-bit key. Word j % 4 of the block with counter (row * ceil(cols / 4) + j / 4,
// offset) and key seed decides element (row, j): dropped where the word is below
// floor(p * 2^32). A row starts a new block, so four neighbouring columns share
// one block whatever the row stride is.
#pragma once
#include <cstdint>

namespace mm {

// What a kernel needs to form the mask; rng == nullptr: no dropout.
struct DropoutArgs {
  const uint64_t* rng = nullptr;  // device: {seed, offset}
  uint32_t threshold = 0;         // floor(p * 2^32)
  float scale = 1.0f;             // 1 / (1 - p)
  uint32_t blocks = 0;            // ceil(cols / 4)
};

__device__ __forceinline__ uint4 philox4x32_10(uint64_t counter, uint64_t offset, uint64_t seed) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c1 = static_cast<uint32_t>(p1);
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Four neighbouring columns (quad = column / 4) of a row, times 0 or 1 / (1 - p).
__device__ __forceinline__ float4 dropout_quad(float4 v, const DropoutArgs& d, uint64_t seed, uint64_t offset,
                                               long long row, int quad) {
  const uint4 w = philox4x32_10(static_cast<uint64_t>(row) * d.blocks + static_cast<uint32_t>(quad), offset, seed);
  v.x = w.x >= d.threshold ? v.x * d.scale : 0.0f;
  v.y = w.y >= d.threshold ? v.y * d.scale : 0.0f;
  v.z = w.z >= d.threshold ? v.z * d.scale : 0.0f;
  v.w = w.w >= d.threshold ? v.w * d.scale : 0.0f;
  return v;
}

}  // namespace mm
