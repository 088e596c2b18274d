// Host interface of the products with an epilogue (linear.cu), of dropout and of
// the linear cross-entropy (linear_loss.cu). All calls are asynchronous on
// `stream`; every temporary lives in the caller's workspace.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "dropout.cuh"
#include "gemm.h"

namespace mm {

// The longest dimension: indices of the tile that holds the last row stay inside 32 bits.
constexpr long long kLongest = 0x7fffffffll - 511;

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
  bool late = false;  // needs nothing of the launch before it: may run beside it (linear_epi.cuh)
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
  // Instead of the logits (pair_loss_product): each row's 128 columns' exp(logit -
  // maximum) 2^14 as a split copy's halves, rows of copy_ld.
  uint16_t* copy = nullptr;
  long long copy_ld = 0;
};

// The operand's tensor map: `mn` rows (or columns) of the product, `box` of them
// per tile. MN-major operands of a width that is a multiple of 32 load a stage in
// one 3-D box (32 wide, 32 K rows, box / 32 blocks), others in 32-wide 2-D boxes.
int operand_map(CUtensorMap* map, const GemmOperand& o, int mn, int k, int box, bool* box3d);

// ---- Large exact products (linear_pair.cu): f16 halves of operands scaled block
// by block, three terms on CTA pairs.
//
// A copy of a [rows, k] operand, K-major: per row and chunk of 128 of k, 256 f16
// values [hi 0..63, lo 0..63, hi 64..127, lo 64..127] (zeros past k), and per
// chunk and row the inverse of the power of two that the chunk was scaled by.
struct SplitCopy {
  uint16_t* data = nullptr;
  float* inv = nullptr;  // [chunks, inv_ld], whole 256-row tiles (what lies past rows is never used)
  int rows = 0, k = 0;
  __host__ __device__ long long chunks() const { return (k + 127) / 128; }
  __host__ __device__ long long row_halves() const { return chunks() * 256; }
  __host__ __device__ long long inv_ld() const { return (rows + 255ll) / 256 * 256; }
};
long long split_copy_bytes(int rows, int k);
SplitCopy split_copy_at(void* ptr, int rows, int k);  // ptr 256-byte aligned

// Lays a workspace out front to back, in 256-byte steps; with a null base it only counts.
struct Arena {
  uint8_t* base;
  long long at = 0;
  void* take(long long bytes) {
    void* p = base ? base + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
  SplitCopy copy(int rows, int k) { return split_copy_at(take(split_copy_bytes(rows, k)), rows, k); }
};

// What a split reads: a matrix, or the epilogue's backward (dz of act_backward).
struct SplitMatrix {
  const float* x;
  long long ld;
  const int32_t* targets = nullptr;  // rows without a class as target count as zeros
  int vocab = 0;
};
struct SplitBackward {
  const float* dc;
  long long lddc;
  const float* z;
  long long ldz;
  int act;
  DropoutArgs drop;
};
// [rows, cols] -> its copy by rows (K = cols), its transpose's copy (K = rows), and
// the column sums' partials [split_parts(rows), cols]; each may be absent.
void split(const SplitMatrix& src, int rows, int cols, const SplitCopy* by_rows, const SplitCopy* by_cols,
           cudaStream_t s);
void split(const SplitBackward& src, int rows, int cols, const SplitCopy* by_rows, const SplitCopy* by_cols,
           float* part, cudaStream_t s);
// src [rows, k] -> its transpose's copy [k, rows].
void split_transposed(const SplitCopy& src, const SplitCopy& by_cols, cudaStream_t s);
// The copy that LossEpilogue wrote -> the loss's gradient: part as the epilogue left it,
// stat per row its maximum and grad_scale / its sum.
void loss_scales(const SplitCopy& g, const float2* part, const float2* stat, const int32_t* targets, int vocab,
                 float grad_scale, cudaStream_t s);
// Two matrices in one launch.
void split_two(const SplitMatrix& x, int x_rows, int x_cols, const SplitCopy* x_by_rows, const SplitCopy* x_by_cols,
               const SplitMatrix& y, int y_rows, int y_cols, const SplitCopy* y_by_rows, const SplitCopy* y_by_cols,
               cudaStream_t s);
inline int split_parts(int rows) { return (rows + 127) / 128; }

// ws: pair_ws_bytes(A.rows, B.rows, A.k) bytes (a partial last wave's K parts).
long long pair_ws_bytes(int M, int N, int K);
int pair_product(const SplitCopy& A, const SplitCopy& B, const LinearEpilogue& e, void* ws, int* d_err,
                 cudaStream_t s);
int pair_loss_product(const SplitCopy& A, const SplitCopy& B, const LossEpilogue& e, int* d_err, cudaStream_t s);
// Whether an exact product of this size is worth the copies.
bool pair_product_suits(int M, int N, int K);
// About how long it takes, copies aside; parts: whether its last wave may be cut.
double pair_us(int M, int N, int K, bool parts);

// Large TF32 products on the operands themselves (linear_pair.cu). An MN-major A
// only with an MN-major B and no activation or dropout. ws: tf32_pair_ws_bytes bytes.
long long tf32_pair_ws_bytes(int M, int N, int K);
int tf32_pair_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LinearEpilogue& e,
                      void* ws, int* d_err, cudaStream_t s);
int tf32_pair_loss_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LossEpilogue& e,
                           int* d_err, cudaStream_t s);
bool tf32_pair_suits(int M, int N, int K);

DropoutArgs dropout_args(double p, const uint64_t* rng, int cols);

// y = r + dropout(x) over [rows, cols]; r may be null, y may be x or r.
void dropout(const float* x, long long ldx, const float* r, long long ldr, float* y, long long ldy, long long rows,
             int cols, const DropoutArgs& d, cudaStream_t s);

// C = epilogue(sum_k A(m, k) B(n, k)) on single CTAs; operands as in gemm.h,
// precision exact or one TF32 pass. Returns a GemmStatus.
// ws: direct_ws_bytes bytes (the sums of a long K's slices).
long long direct_ws_bytes(int M, int N, int K, bool a_mn_major);
int direct_product(int M, int N, int K, GemmOperand A, GemmOperand B, const LinearEpilogue& e, bool exact, void* ws,
                   int* d_err, cudaStream_t s);
// The same product with the loss's epilogue.
int direct_loss_product(int M, int N, int K, GemmOperand A, GemmOperand B, const LossEpilogue& e, bool exact,
                        int* d_err, cudaStream_t s);

// dz = mask / (1 - p) * dc * act'(z) (dz null: only the column sums), and the
// column sums' partials for dbias where part is not null: part must hold
// act_backward_parts(rows, cols) * cols floats.
void act_backward(const float* dc, long long lddc, const float* z, long long ldz, int act, const DropoutArgs& d,
                  int rows, int cols, float* dz, long long lddz, float* part, cudaStream_t s);
int act_backward_parts(int rows, int cols);
// out[c] (+)= sum over p of part[p, c], in f64 and in a fixed order.
void sum_parts(const float* part, int parts, int cols, float* out, bool accumulate, cudaStream_t s);

// ---- The operators (linear_ops.cu): direct or pair products by size; workspaces
// are 256-byte aligned.
// A product on the operands themselves: TF32 on pairs where that suits, else direct.
long long plain_ws_bytes(int M, int N, int K, bool a_mn_major, bool exact);
int plain_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LinearEpilogue& e, bool exact,
                  void* ws, int* d_err, cudaStream_t s);
int plain_loss_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LossEpilogue& e,
                       bool exact, int* d_err, cudaStream_t s);

// Held while a call with late products is enqueued (linear_epi.cuh).
std::mutex& launch_order();

struct LinearForward {
  int m, n, k;
  const float* a;
  long long lda;
  const float* b;
  long long ldb;
  bool b_mn_major;
  LinearEpilogue e;
  bool exact;
};
long long linear_forward_ws_bytes(int m, int n, int k, bool exact);
int linear_forward(const LinearForward& f, void* ws, int* d_err, cudaStream_t s);

struct LinearBackward {
  int m, n, k;
  const float* a;
  long long lda;
  const float* b;
  long long ldb;
  bool b_mn_major;
  int act;
  DropoutArgs drop;
  const float* z;  // may be null without an activation
  long long ldz;
  const float* dc;
  long long lddc;
  float* da;  // each may be null
  long long ldda;
  float* db;
  long long lddb;
  float* dbias;
  bool accumulate;
  bool exact;
};
long long linear_backward_ws_bytes(int m, int n, int k, bool exact);
int linear_backward(const LinearBackward& f, void* ws, int* d_err, cudaStream_t s);

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
