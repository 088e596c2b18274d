// Softmax cross-entropy of z = x w^T over a vocabulary, without the [rows, vocab]
// logits: loss_i = lse_i - z_i,t, and on request dx = G w, dw = G^T x with
// G = grad_scale (softmax(z) - onehot(t)). Rows with target -1 are left out: loss
// 0, dx 0, no share in dw whatever their x holds.
//
// The loss alone: the product's epilogue reduces each row's 128 columns to their
// maximum and sum of exponentials, so the logits never leave the chip; a warp per
// row joins the vocab / 128 pairs. With gradients the rows go in blocks whose
// logits fit a fixed part of the workspace: the product (6 N V D operations in
// all, as with the logits kept; pieces of the vocabulary would have to form each
// logit twice, 8 N V D), then z -> G in place, dx = G w, dw += G^T x. Large exact blocks
// never hold z: the epilogue writes exp(z - its chunk's maximum) as the split copy that
// dx's product reads, and what softmax still lacks, exp(that maximum - the row's)
// grad_scale / the row's sum, is one number per row and chunk, which that product
// multiplies by anyhow as the chunk's scale. So only dw needs a pass over the block, to
// transpose (8 bytes a logit; forming both copies from z took 12).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "device.h"
#include "linear.h"
#include "linear_epi.cuh"
#include "ptx.cuh"

namespace mm {
namespace {

constexpr long long kLogitBytes = 384ll << 20;  // a block's logits, or half as much as w if that is more
constexpr long long kPartBytes = 64ll << 20;    // a block's (max, sum) pairs, the loss alone

long long round_up(long long n, long long to) { return (n + to - 1) / to * to; }

struct Plan {
  bool pair;        // pair products on copies, or direct ones
  bool pair_logits; // direct ones, but for the logits
  int tiles, rows;  // (max, sum) pairs per row; rows of a block
  long long ldz, ldx;
  float2* part;
  float2* stat;
  float* zt;
  float* z;
  float* x;                                  // direct: the live rows of x
  SplitCopy w, wt, xr, xt, g, gt;            // pair: [vocab, dim], [dim, vocab], and of a block [n, dim], [dim, n],
  void *xr_at, *xt_at, *g_at, *gt_at;        // [n, vocab], [vocab, n] (a block may be shorter)
  void *parts_dx, *parts_dw;                 // of the gradients' products, which may run side by side
  long long bytes;
};

// Of `least` blocks and a few more, the count whose products take the shortest time: dx
// has few tiles (2048 rows of the large preset's 64, for 74 pairs; 2816 have 88, the 14
// past a wave cut into parts).
long long best_blocks(long long n, long long least, int vocab, int dim) {
  long long best = least;
  double best_us = 1e30;
  for (long long b = least; b <= 2 * least + 1; ++b) {
    const long long rows = round_up((n + b - 1) / b, 256), last = n - rows * (b - 1);
    if (last <= 0) break;
    auto block_us = [&](long long r) {
      const int m = static_cast<int>(r);
      return pair_us(m, vocab, dim, false) + pair_us(m, dim, vocab, true) + pair_us(vocab, dim, m, true);
    };
    const double us = (b - 1) * block_us(rows) + block_us(last);
    if (us < best_us) {
      best_us = us;
      best = b;
    }
  }
  return best;
}

Plan plan_of(int rows, int vocab, int dim, bool dx, bool dw, bool exact, void* ws) {
  Plan p{};
  const bool grad = dx || dw;
  Arena at{static_cast<uint8_t*>(ws)};
  p.tiles = (vocab + 127) / 128;
  p.ldz = round_up(vocab, 4);
  p.ldx = round_up(dim, 4);
  const long long logits = std::max(kLogitBytes, 2ll * vocab * dim);
  const long long most = std::max(256ll, (grad ? logits / (p.ldz * 4) : kPartBytes / (p.tiles * 8ll)) / 256 * 256);
  const long long n = std::max(rows, 1);
  long long blocks = (n + most - 1) / most;
  if (grad && exact && blocks > 1) blocks = best_blocks(n, blocks, vocab, dim);
  p.rows = static_cast<int>(std::min(n, round_up((n + blocks - 1) / blocks, 256)));  // even blocks of whole tiles
  p.pair = exact && pair_product_suits(p.rows, vocab, dim) &&
           (!grad || (pair_product_suits(p.rows, dim, vocab) && pair_product_suits(vocab, dim, p.rows)));
  p.pair_logits = exact && !p.pair && pair_product_suits(p.rows, vocab, dim);
  p.part = static_cast<float2*>(at.take(static_cast<long long>(p.rows) * p.tiles * 8));
  p.zt = static_cast<float*>(at.take(p.rows * 4ll));
  p.stat = static_cast<float2*>(at.take(p.rows * 8ll));
  if (p.pair || p.pair_logits) {
    p.w = at.copy(vocab, dim);
    p.xr_at = at.take(split_copy_bytes(p.rows, dim));
  }
  if (p.pair) {
    if (grad) p.g_at = at.take(split_copy_bytes(p.rows, vocab));
    if (dx) p.wt = at.copy(dim, vocab);
    if (dw) {
      p.xt_at = at.take(split_copy_bytes(dim, p.rows));
      p.gt_at = at.take(split_copy_bytes(vocab, p.rows));
    }
  } else {
    if (grad) p.z = static_cast<float*>(at.take(p.rows * p.ldz * 4));
    if (dw) p.x = static_cast<float*>(at.take(p.rows * p.ldx * 4));
  }
  // the last block may be shorter: its products may be cut into parts that the others are not
  const int last = static_cast<int>(n - (blocks - 1) * p.rows);
  auto parts = [&](int M, int N, int K, bool a_mn_major) {
    return p.pair ? pair_ws_bytes(M, N, K) : plain_ws_bytes(M, N, K, a_mn_major, exact);
  };
  long long most_dx = 0, most_dw = 0;
  for (const int r : {p.rows, std::max(last, 1)}) {
    if (dx) most_dx = std::max(most_dx, parts(r, dim, vocab, false));
    if (dw) most_dw = std::max({most_dw, parts(vocab, dim, r, true), parts(dim, vocab, r, true)});
  }
  p.parts_dx = at.take(most_dx);
  p.parts_dw = at.take(most_dw);
  p.bytes = at.at;
  return p;
}

struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s};  // both empty (sums 0), or NaN logits: the NaN stays
  return {m, a.s * expf(a.m - m) + b.s * expf(b.m - m)};
}
__device__ __forceinline__ MaxSum warp_join(MaxSum a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = join(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
  return a;
}

// The row's loss; a target that is neither -1 nor a class sets the error flag.
__device__ __forceinline__ float loss_of(MaxSum a, int t, int vocab, const float* zt, int* err) {
  if (t >= 0 && t < vocab) return a.m + logf(a.s) - *zt;
  if (t == -1) return 0.0f;
  if (err) atomicCAS(err, 0, kErrIndex);
  return NAN;
}

__global__ void __launch_bounds__(256) row_loss_kernel(const float2* part, int tiles, const float* zt,
                                                       const int32_t* targets, int rows, int vocab,
                                                       float grad_scale, float* row_loss, float2* stat, int* err) {
  after_previous();
  let_next();
  const int r = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (r >= rows) return;
  MaxSum a{-INFINITY, 0.0f};
  const float2* mine = part + static_cast<long long>(r) * tiles;
  for (int i = lane; i < tiles; i += 256) {  // eight loads in flight
    float2 p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) p[u] = i + 32 * u < tiles ? mine[i + 32 * u] : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int u = 0; u < 8; ++u) a = join(a, {p[u].x, p[u].y});
  }
  a = warp_join(a);
  if (lane == 0) {
    row_loss[r] = loss_of(a, targets[r], vocab, zt + r, err);
    if (stat) stat[r] = make_float2(a.m, grad_scale / a.s);
  }
}

// One row's kSegment logits -> gradients, in place; every block of a row joins
// the row's pairs itself (vocab / 128 of them, from L2), the first writes the loss and,
// where dw is wanted, copies the row of x (zeros for a row without a target: dw sums
// over all rows, and 0 times what such a row holds may be NaN). A
// vocabulary may have more segments than a grid's y: those past it lie along z (and what
// the last z has beyond the last segment finds nothing to write).
constexpr int kSegment = 4096;
constexpr long long kGridY = 65535;

__global__ void __launch_bounds__(256) loss_grad_kernel(float* z, long long ldz, const float2* part, int tiles,
                                                        const float* zt, const int32_t* targets, int vocab,
                                                        float grad_scale, float* row_loss, const float* x,
                                                        long long ldx, int dim, float* live_x, long long ldl,
                                                        int* err) {
  after_previous();
  let_next();
  __shared__ MaxSum warps[8];
  const int r = blockIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int segment = static_cast<int>(blockIdx.y + gridDim.y * blockIdx.z);
  const int t = targets[r];
  const bool live = t >= 0 && t < vocab;
  float4* row = reinterpret_cast<float4*>(z + r * ldz);
  const int q_end = static_cast<int>(ldz / 4), q0 = segment * (kSegment / 4) + threadIdx.x;
  float4 v[kSegment / 1024];  // on their way while the row's pairs are joined
#pragma unroll
  for (int u = 0; u < kSegment / 1024; ++u)
    v[u] = q0 + 256 * u < q_end ? row[q0 + 256 * u] : make_float4(0.f, 0.f, 0.f, 0.f);
  MaxSum a{-INFINITY, 0.0f};
  for (int i = threadIdx.x; i < tiles; i += 256) {
    const float2 p = part[static_cast<long long>(r) * tiles + i];
    a = join(a, {p.x, p.y});
  }
  a = warp_join(a);
  if (lane == 0) warps[warp] = a;
  __syncthreads();
  a = warps[0];
  for (int w = 1; w < 8; ++w) a = join(a, warps[w]);
  if (segment == 0 && threadIdx.x == 0) row_loss[r] = loss_of(a, t, vocab, zt + r, err);
  if (segment == 0 && live_x)
    for (unsigned c = 4 * threadIdx.x; c < static_cast<unsigned>(dim); c += 1024)  // ldl is dim rounded up to 4
      *reinterpret_cast<float4*>(live_x + r * ldl + c) =
          live ? load_quad(x + r * ldx, static_cast<int>(c), dim) : make_float4(0.f, 0.f, 0.f, 0.f);
  const float coef = grad_scale / a.s;
#pragma unroll
  for (int u = 0; u < kSegment / 1024; ++u) {
    const int q = q0 + 256 * u;
    if (q >= q_end) break;
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
      g = make_float4(loss_exp(v[u].x - a.m) * coef, loss_exp(v[u].y - a.m) * coef, loss_exp(v[u].z - a.m) * coef,
                      loss_exp(v[u].w - a.m) * coef);
      if ((t >> 2) == q) {
        if ((t & 3) == 0) g.x -= grad_scale;
        if ((t & 3) == 1) g.y -= grad_scale;
        if ((t & 3) == 2) g.z -= grad_scale;
        if ((t & 3) == 3) g.w -= grad_scale;
      }
    }
    row[q] = g;
  }
}

// The mean over the rows that have a target (0 when none has), in f64.
__global__ void __launch_bounds__(1024) mean_live_kernel(const float* row_loss, const int32_t* targets, int rows,
                                                         float* mean) {
  after_previous();
  let_next();
  __shared__ double sums[32];
  __shared__ int counts[32];
  double s = 0.0;
  int n = 0;
  for (unsigned r = threadIdx.x; r < static_cast<unsigned>(rows); r += 1024) {  // its last step may pass 31 bits
    const int t = targets[r];
    const float loss = row_loss[r];  // beside the target's load
    if (t != -1) {
      s += loss;
      ++n;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (threadIdx.x % 32 == 0) {
    sums[threadIdx.x / 32] = s;
    counts[threadIdx.x / 32] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) {
      s += sums[w];
      n += counts[w];
    }
    *mean = static_cast<float>(n ? s / n : 0.0);
  }
}

}  // namespace

long long linear_loss_ws_bytes(int rows, int vocab, int dim, bool grad, bool exact) {
  return plan_of(rows, vocab, dim, grad, grad, exact, nullptr).bytes;
}

namespace {

// The copies of a block's rows of x, transposed too where xt is given, and with the first
// block's those of w. With `targets` rows without one count as zeros.
void copy_operands(const LinearLoss& a, const Plan& p, long long r0, int n, const int32_t* targets, const SplitCopy* wt,
                   const SplitCopy* xt, cudaStream_t s) {
  const SplitMatrix x{a.x + r0 * a.ldx, a.ldx, targets, a.vocab}, w{a.w, a.ldw};
  if (r0 > 0)
    split(x, n, a.dim, &p.xr, xt, s);
  else if (a.w_mn_major)  // [dim, vocab]
    split_two(w, a.dim, a.vocab, wt, &p.w, x, n, a.dim, &p.xr, xt, s);
  else
    split_two(w, a.vocab, a.dim, &p.w, wt, x, n, a.dim, &p.xr, xt, s);
}

void mean_loss(const LinearLoss& a, cudaStream_t s) {
  launch_next("mean loss", mean_live_kernel, dim3(1), 1024, 0, 1, s, a.row_loss, a.targets, a.rows, a.mean_loss);
}

// One block of rows on copies. The mean, once the last block's losses are there, and the
// gradients' products need one another's results neither, so they run side by side.
int pair_block(const LinearLoss& a, Plan& p, long long r0, int n, bool mean, int* d_err, cudaStream_t s) {
  const int32_t* t = a.targets + r0;
  // For gradients x's rows without a target count as zeros: their logits are not used, but
  // their exponentials are multiplied by 0 for dx, and dw sums over all rows, and 0 times
  // what such a row holds may be NaN
  p.xr = split_copy_at(p.xr_at, n, a.dim);
  if (a.dw) p.xt = split_copy_at(p.xt_at, a.dim, n);
  const bool grad = a.dx || a.dw;
  copy_operands(a, p, r0, n, grad ? t : nullptr, a.dx ? &p.wt : nullptr, a.dw ? &p.xt : nullptr, s);
  LossEpilogue e;
  e.part = p.part;
  e.tiles = p.tiles;
  e.targets = t;
  e.zt = p.zt;
  if (grad) {
    p.g = split_copy_at(p.g_at, n, a.vocab);
    e.copy = p.g.data;
    e.copy_ld = p.g.row_halves();
  }
  int rc = pair_loss_product(p.xr, p.w, e, d_err, s);
  if (rc) return rc;
  launch_next("row loss", row_loss_kernel, dim3((n + 7) / 8), 256, 0, 1, s, p.part, p.tiles, p.zt, t, n, a.vocab,
              a.grad_scale, a.row_loss + r0, p.stat, d_err);
  if (!grad) return 0;
  loss_scales(p.g, p.part, p.stat, t, a.vocab, a.grad_scale, s);
  if (a.dw) {
    p.gt = split_copy_at(p.gt_at, a.vocab, n);
    split_transposed(p.g, p.gt, s);
  }
  if (mean) mean_loss(a, s);
  if (a.dx) {
    LinearEpilogue o;
    o.C = a.dx + r0 * a.lddx;
    o.R = a.accumulate ? o.C : nullptr;
    o.ldc = o.ldr = a.lddx;
    o.late = mean;
    rc = pair_product(p.g, p.wt, o, p.parts_dx, d_err, s);
    if (rc) return rc;
  }
  if (a.dw) {
    LinearEpilogue o;
    o.C = a.dw;
    o.R = a.accumulate || r0 > 0 ? a.dw : nullptr;
    o.ldc = o.ldr = a.lddw;
    o.late = mean || a.dx;
    rc = a.w_mn_major ? pair_product(p.xt, p.gt, o, p.parts_dw, d_err, s)
                      : pair_product(p.gt, p.xt, o, p.parts_dw, d_err, s);
  }
  return rc;
}

// One block of rows on direct products: G takes the logits' place. Where rows and classes
// are many but the rows short, the logits have the tiles for a pair product and the
// gradients do not.
int direct_block(const LinearLoss& a, Plan& p, long long r0, int n, bool mean, int* d_err, cudaStream_t s) {
  const float* x = a.x + r0 * a.ldx;
  const int32_t* t = a.targets + r0;
  const LossEpilogue e{p.z, p.ldz, p.part, p.tiles, t, p.zt, nullptr, 0};
  int rc;
  if (p.pair_logits) {
    p.xr = split_copy_at(p.xr_at, n, a.dim);
    copy_operands(a, p, r0, n, nullptr, nullptr, nullptr, s);
    rc = pair_loss_product(p.xr, p.w, e, d_err, s);
  } else {
    rc = plain_loss_product(n, a.vocab, a.dim, {x, a.ldx, false}, {a.w, a.ldw, a.w_mn_major}, e, a.exact, d_err, s);
  }
  if (rc) return rc;
  if (!a.dx && !a.dw) {
    launch_next("row loss", row_loss_kernel, dim3((n + 7) / 8), 256, 0, 1, s, p.part, p.tiles, p.zt, t, n, a.vocab, 0.0f,
                a.row_loss + r0, nullptr, d_err);
    return 0;
  }
  const long long segments = (p.ldz + kSegment - 1) / kSegment;
  const dim3 grid(n, static_cast<unsigned>(std::min(segments, kGridY)),
                  static_cast<unsigned>((segments + kGridY - 1) / kGridY));
  launch_next("loss gradient", loss_grad_kernel, grid, 256, 0, 1, s, p.z, p.ldz, p.part, p.tiles, p.zt, t, a.vocab,
              a.grad_scale, a.row_loss + r0, x, a.ldx, a.dim, a.dw ? p.x : nullptr, p.ldx, d_err);
  if (mean) mean_loss(a, s);
  if (a.dw) {
    LinearEpilogue o;
    o.C = a.dw;
    o.R = a.accumulate || r0 > 0 ? a.dw : nullptr;
    o.ldc = o.ldr = a.lddw;
    o.late = mean;
    const GemmOperand g{p.z, p.ldz, true}, xo{p.x, p.ldx, true};
    rc = a.w_mn_major ? plain_product(a.dim, a.vocab, n, xo, g, o, a.exact, p.parts_dw, d_err, s)
                      : plain_product(a.vocab, a.dim, n, g, xo, o, a.exact, p.parts_dw, d_err, s);
    if (rc) return rc;
  }
  if (a.dx) {
    LinearEpilogue o;
    o.C = a.dx + r0 * a.lddx;
    o.R = a.accumulate ? o.C : nullptr;
    o.ldc = o.ldr = a.lddx;
    o.late = mean || a.dw;
    rc = plain_product(n, a.dim, a.vocab, {p.z, p.ldz, false}, {a.w, a.ldw, !a.w_mn_major}, o, a.exact, p.parts_dx,
                       d_err, s);
  }
  return rc;
}

}  // namespace

int linear_loss(const LinearLoss& a, void* ws, int* d_err, cudaStream_t s) {
  const bool grad = a.dx || a.dw;
  Plan p = plan_of(a.rows, a.vocab, a.dim, grad, grad, a.exact, ws);
  const std::lock_guard<std::mutex> lock(launch_order());
  for (long long r0 = 0; r0 < a.rows; r0 += p.rows) {
    const int n = static_cast<int>(std::min<long long>(p.rows, a.rows - r0));
    const bool mean = a.mean_loss && grad && r0 + n == a.rows;
    const int rc = p.pair ? pair_block(a, p, r0, n, mean, d_err, s) : direct_block(a, p, r0, n, mean, d_err, s);
    if (rc) return rc;
  }
  if (a.mean_loss && !grad) mean_loss(a, s);
  return 0;
}

}  // namespace mm
