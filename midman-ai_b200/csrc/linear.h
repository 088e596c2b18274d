// Host interface of the products with an epilogue (linear.cu), of dropout and of
// the linear cross-entropy (linear_loss.cu). All calls are asynchronous on
// `stream`; every temporary lives in the caller's workspace.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "dropout.cuh"
#include "gemm.h"

namespace mm {

enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3, kActivations = 4 };

// c = r + dropout(act(z)), z = product + bias; z is written where wanted.
struct LinearEpilogue {
  const float* bias = nullptr;
  int act = kActNone;
  DropoutArgs drop;
  const float* R = nullptr;  // may be C
  long long ldr = 0;
  float* Z = nullptr;
  long long ldz = 0;
  float* C = nullptr;
  long long ldc = 0;
};

// One 128-column tile's share of a row's softmax: the maximum of its logits and
// the sum of exp(logit - maximum).
struct LossEpilogue {
  float* Z = nullptr;  // the logits, where the gradient needs them
  long long ldz = 0;
  float2* part = nullptr;  // [rows, tiles]
  int tiles = 0;
  const int32_t* targets = nullptr;
  float* zt = nullptr;  // [rows]: the target's logit
};

DropoutArgs dropout_args(double p, const uint64_t* rng, int cols);

// y = r + dropout(x) over [rows, cols]; r may be null, y may be x or r.
void dropout(const float* x, long long ldx, const float* r, long long ldr, float* y, long long ldy, long long rows,
             int cols, const DropoutArgs& d, cudaStream_t s);

// C = epilogue(sum_k A(m, k) B(n, k)); operands as in gemm.h, precision exact or
// one TF32 pass. Returns a GemmStatus.
int linear_product(int M, int N, int K, GemmOperand A, GemmOperand B, const LinearEpilogue& e, bool exact, int* d_err,
                   cudaStream_t s);
// The same product with the loss's epilogue.
int loss_product(int M, int N, int K, GemmOperand A, GemmOperand B, const LossEpilogue& e, bool exact, int* d_err,
                 cudaStream_t s);

// dz = mask / (1 - p) * dc * act'(z) (dz null: only the column sums), and the
// column sums' partials for dbias where part is not null: part must hold
// act_backward_parts(rows) * cols floats.
void act_backward(const float* dc, long long lddc, const float* z, long long ldz, int act, const DropoutArgs& d,
                  int rows, int cols, float* dz, long long lddz, float* part, cudaStream_t s);
int act_backward_parts(int rows);
// out[c] (+)= sum over p of part[p, c], in f64 and in a fixed order.
void sum_parts(const float* part, int parts, int cols, float* out, bool accumulate, cudaStream_t s);

struct LinearLoss {
  int rows, vocab, dim;
  const float* x;
  long long ldx;
  const float* w;
  long long ldw;
  bool w_mn_major;  // w is [dim, vocab]
  const int32_t* targets;
  float grad_scale;
  float* row_loss;
  float* mean_loss;  // may be null
  float* dx;         // may be null
  long long lddx;
  float* dw;  // may be null
  long long lddw;
  bool accumulate;
  bool exact;
};
long long linear_loss_ws_bytes(int rows, int vocab, int dim, bool grad, bool exact);
int linear_loss(const LinearLoss& a, void* ws, int* d_err, cudaStream_t s);

}  // namespace mm
