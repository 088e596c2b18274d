// Kernel-level C ABI of the products with an epilogue, dropout and the linear
// cross-entropy (include/midman_gpu.h): argument checks, then the launchers.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/midman_gpu.h"
#include "device.h"
#include "linear.h"

namespace {

thread_local std::string g_linear_error;

int32_t fail(int32_t code, const std::string& msg) {
  g_linear_error = msg;
  return code;
}

// Runs `body`; C++ exceptions become MM_GPU_ERR_DEVICE with their message.
template <class R, class F>
R guarded(const char* what, F&& body) {
  R rc;
  try {
    g_linear_error.clear();
    rc = body();
  } catch (const std::exception& e) {
    rc = fail(MM_GPU_ERR_DEVICE, std::string(what) + ": " + e.what());
  } catch (...) {
    rc = fail(MM_GPU_ERR_DEVICE, std::string(what) + ": unknown C++ exception");
  }
  mm::set_last_error(rc < 0 ? g_linear_error : std::string());
  return rc;
}

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// A row-major operand that the vector loads and TMA read: 16-byte aligned rows.
int32_t check_matrix(const char* what, const void* p, int64_t ld, int64_t width) {
  if (!p) return fail(MM_GPU_ERR_ARGUMENT, std::string(what) + ": null pointer");
  if (ld < width || ld % 4)
    return fail(MM_GPU_ERR_SHAPE, std::string(what) + ": the row stride must be a multiple of 4 that holds the row");
  if (!aligned(p, 16)) return fail(MM_GPU_ERR_ARGUMENT, std::string(what) + ": must be 16-byte aligned");
  return MM_GPU_OK;
}

int32_t check_lengths(const char* what, int64_t a, int64_t b, int64_t c) {
  if (a > mm::kLongest || b > mm::kLongest || c > mm::kLongest)
    return fail(MM_GPU_ERR_SHAPE, std::string(what) + ": a dimension is longer than " + std::to_string(mm::kLongest));
  return MM_GPU_OK;
}

int32_t check_precision(int32_t precision) {
  if (precision != MM_GPU_TF32 && precision != MM_GPU_3XTF32)
    return fail(MM_GPU_ERR_ARGUMENT, "precision must be MM_GPU_TF32 or MM_GPU_3XTF32");
  return MM_GPU_OK;
}

int32_t check_dropout(double p, const uint64_t* rng) {
  if (!(p >= 0.0 && p < 1.0)) return fail(MM_GPU_ERR_ARGUMENT, "dropout: p must lie in [0, 1)");
  if (p > 0.0 && (!rng || !aligned(rng, 8)))
    return fail(MM_GPU_ERR_ARGUMENT, "dropout: rng must point to {seed, offset} on the device, 8-byte aligned");
  return MM_GPU_OK;
}

int32_t check_activation(int32_t activation) {
  if (activation < 0 || activation >= mm::kActivations)
    return fail(MM_GPU_ERR_ARGUMENT, "activation must be one of MM_GPU_ACT_*");
  return MM_GPU_OK;
}

// An output that is an input, or another output, would be read after it is written.
// Compared by where they start: rows of two matrices may lie between one another's.
int32_t check_distinct(const char* what, std::initializer_list<const void*> outputs,
                       std::initializer_list<const void*> inputs) {
  for (auto o = outputs.begin(); o != outputs.end(); ++o) {
    if (!*o) continue;
    if (std::find(o + 1, outputs.end(), *o) != outputs.end() ||
        std::find(inputs.begin(), inputs.end(), *o) != inputs.end())
      return fail(MM_GPU_ERR_ARGUMENT, std::string(what) + ": an output must have a buffer of its own");
  }
  return MM_GPU_OK;
}

int32_t check_workspace(const void* ws, int64_t bytes, int64_t need) {
  if (need > 0 && (!ws || bytes < need || !aligned(ws, 256)))
    return fail(MM_GPU_ERR_ARGUMENT, "workspace: needs " + std::to_string(need) + " bytes, 256-byte aligned");
  return MM_GPU_OK;
}

int32_t product_status(int rc) {
  if (!rc) return MM_GPU_OK;
  return fail(rc == mm::kGemmLaunch ? MM_GPU_ERR_DEVICE : MM_GPU_ERR_ARGUMENT, mm::gemm_status_string(rc));
}

}  // namespace

#define MM_TRY(x)               \
  do {                          \
    if (int32_t rc_ = (x)) return rc_; \
  } while (0)

extern "C" {

int32_t mm_gpu_dropout(int64_t rows, int32_t cols, const float* x, int64_t ldx, const float* r, int64_t ldr, float* y,
                       int64_t ldy, double p, const uint64_t* rng, void* stream) {
  return guarded<int32_t>("dropout", [&]() -> int32_t {
    if (rows < 0 || cols <= 0) return fail(MM_GPU_ERR_SHAPE, "dropout: need rows >= 0 and cols > 0");
    MM_TRY(check_lengths("dropout", 0, cols, 0));
    if (rows > 0 && (!x || !y)) return fail(MM_GPU_ERR_ARGUMENT, "dropout: null pointer");
    if (ldx < cols || ldy < cols || (r && ldr < cols))
      return fail(MM_GPU_ERR_SHAPE, "dropout: a row stride is smaller than the row");
    if (rows - 1 > INT64_MAX / 4 / std::max({ldx, ldy, r ? ldr : 0}))  // the last row's address, and the count of quads
      return fail(MM_GPU_ERR_SHAPE, "dropout: more rows than there are addresses");
    if (rows > 0 && ((y == x && ldy != ldx) || (y == r && ldy != ldr)))
      return fail(MM_GPU_ERR_SHAPE, "dropout: y may be x or r only with its row stride");
    MM_TRY(check_dropout(p, rng));
    mm::dropout(x, ldx, r, ldr, y, ldy, rows, cols, mm::dropout_args(p, rng, cols), as_stream(stream));
    return MM_GPU_OK;
  });
}

int64_t mm_gpu_linear_workspace(int32_t m, int32_t n, int32_t k, int32_t backward, int32_t precision) {
  return guarded<int64_t>("linear", [&]() -> int64_t {
    if (m < 0 || n <= 0 || k <= 0) return fail(MM_GPU_ERR_SHAPE, "linear: need m >= 0, n > 0 and k > 0");
    MM_TRY(check_lengths("linear", m, n, k));
    MM_TRY(check_precision(precision));
    const bool exact = precision == MM_GPU_3XTF32;
    return backward ? mm::linear_backward_ws_bytes(m, n, k, exact) : mm::linear_forward_ws_bytes(m, n, k, exact);
  });
}

int32_t mm_gpu_linear_forward(int32_t m, int32_t n, int32_t k, const float* a, int64_t lda, const float* b,
                              int64_t ldb, int32_t b_mn_major, const float* bias, int32_t activation, double p,
                              const uint64_t* rng, const float* r, int64_t ldr, float* z, int64_t ldz, float* c,
                              int64_t ldc, int32_t precision, void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded<int32_t>("linear", [&]() -> int32_t {
    if (m < 0 || n <= 0 || k <= 0) return fail(MM_GPU_ERR_SHAPE, "linear: need m >= 0, n > 0 and k > 0");
    MM_TRY(check_lengths("linear", m, n, k));
    MM_TRY(check_precision(precision));
    MM_TRY(check_activation(activation));
    MM_TRY(check_dropout(p, rng));
    if (m == 0) return MM_GPU_OK;  // an empty batch has no addresses
    MM_TRY(check_matrix("linear: a", a, lda, k));
    MM_TRY(check_matrix("linear: b", b, ldb, b_mn_major ? n : k));
    MM_TRY(check_matrix("linear: c", c, ldc, n));
    if (r) MM_TRY(check_matrix("linear: r", r, ldr, n));
    if (z) MM_TRY(check_matrix("linear: z", z, ldz, n));
    if (r == c && ldr != ldc) return fail(MM_GPU_ERR_SHAPE, "linear: r may be c only with c's row stride");
    MM_TRY(check_distinct("linear", {c, z}, {a, b, bias}));
    if (z && z == r) return fail(MM_GPU_ERR_ARGUMENT, "linear: z must have a buffer of its own");
    const bool exact = precision == MM_GPU_3XTF32;
    MM_TRY(check_workspace(workspace, workspace_bytes, mm::linear_forward_ws_bytes(m, n, k, exact)));
    mm::LinearForward f{m, n, k, a, lda, b, ldb, b_mn_major != 0, {}, exact};
    f.e.bias = bias;
    f.e.act = activation;
    f.e.drop = mm::dropout_args(p, rng, n);
    f.e.R = r;
    f.e.ldr = ldr;
    f.e.Z = z;
    f.e.ldz = ldz;
    f.e.C = c;
    f.e.ldc = ldc;
    return product_status(mm::linear_forward(f, workspace, mm::device_context().d_err, as_stream(stream)));
  });
}

int32_t mm_gpu_linear_backward(int32_t m, int32_t n, int32_t k, const float* a, int64_t lda, const float* b,
                               int64_t ldb, int32_t b_mn_major, int32_t activation, double p, const uint64_t* rng,
                               const float* z, int64_t ldz, const float* dc, int64_t lddc, float* da, int64_t ldda,
                               float* db, int64_t lddb, float* dbias, int32_t accumulate, int32_t precision,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded<int32_t>("linear backward", [&]() -> int32_t {
    if (m < 0 || n <= 0 || k <= 0) return fail(MM_GPU_ERR_SHAPE, "linear backward: need m >= 0, n > 0 and k > 0");
    MM_TRY(check_lengths("linear backward", m, n, k));
    MM_TRY(check_precision(precision));
    MM_TRY(check_activation(activation));
    MM_TRY(check_dropout(p, rng));
    if (m > 0) MM_TRY(check_matrix("linear backward: dc", dc, lddc, n));
    if (m > 0 && activation != MM_GPU_ACT_NONE) MM_TRY(check_matrix("linear backward: z", z, ldz, n));
    if (da && m > 0) {
      MM_TRY(check_matrix("linear backward: b", b, ldb, b_mn_major ? n : k));
      MM_TRY(check_matrix("linear backward: da", da, ldda, k));
    }
    if (db) {
      if (m > 0) MM_TRY(check_matrix("linear backward: a", a, lda, k));
      MM_TRY(check_matrix("linear backward: db", db, lddb, b_mn_major ? n : k));
    }
    const cudaStream_t st = as_stream(stream);
    if (m == 0) {  // sums over no rows
      if (accumulate) return MM_GPU_OK;
      if (db)
        mm::check_cuda(cudaMemset2DAsync(db, lddb * 4, 0, (b_mn_major ? n : k) * 4ull, b_mn_major ? k : n, st), "db");
      if (dbias) mm::check_cuda(cudaMemsetAsync(dbias, 0, n * 4ull, st), "dbias");
      return MM_GPU_OK;
    }
    const bool exact = precision == MM_GPU_3XTF32;
    MM_TRY(check_workspace(workspace, workspace_bytes, mm::linear_backward_ws_bytes(m, n, k, exact)));
    MM_TRY(check_distinct("linear backward", {da, db, dbias}, {a, b, z, dc}));
    const mm::LinearBackward f{m,     n,    k,  a,    lda,        b,   ldb,  b_mn_major != 0,
                               activation, mm::dropout_args(p, rng, n), z, ldz, dc, lddc,
                               da,    ldda, db, lddb, dbias,      accumulate != 0, exact};
    return product_status(mm::linear_backward(f, workspace, mm::device_context().d_err, st));
  });
}

int64_t mm_gpu_linear_cross_entropy_workspace(int32_t rows, int32_t vocab, int32_t dim, int32_t gradients,
                                              int32_t precision) {
  return guarded<int64_t>("linear_cross_entropy", [&]() -> int64_t {
    if (rows < 0 || vocab <= 0 || dim <= 0)
      return fail(MM_GPU_ERR_SHAPE, "linear_cross_entropy: need rows >= 0, vocab > 0 and dim > 0");
    MM_TRY(check_lengths("linear_cross_entropy", rows, vocab, dim));
    MM_TRY(check_precision(precision));
    return mm::linear_loss_ws_bytes(rows, vocab, dim, gradients != 0, precision == MM_GPU_3XTF32);
  });
}

int32_t mm_gpu_linear_cross_entropy(int32_t rows, int32_t vocab, int32_t dim, const float* x, int64_t ldx,
                                    const float* w, int64_t ldw, int32_t w_mn_major, const int32_t* targets,
                                    float grad_scale, float* row_loss, float* mean_loss, float* dx, int64_t lddx,
                                    float* dw, int64_t lddw, int32_t accumulate, int32_t precision, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  return guarded<int32_t>("linear_cross_entropy", [&]() -> int32_t {
    if (rows < 0 || vocab <= 0 || dim <= 0)
      return fail(MM_GPU_ERR_SHAPE, "linear_cross_entropy: need rows >= 0, vocab > 0 and dim > 0");
    MM_TRY(check_lengths("linear_cross_entropy", rows, vocab, dim));
    MM_TRY(check_precision(precision));
    if (!std::isfinite(grad_scale)) return fail(MM_GPU_ERR_ARGUMENT, "linear_cross_entropy: grad_scale must be finite");
    if (rows > 0) {
      if (!targets || !row_loss) return fail(MM_GPU_ERR_ARGUMENT, "linear_cross_entropy: null pointer");
      MM_TRY(check_matrix("linear_cross_entropy: x", x, ldx, dim));
      MM_TRY(check_matrix("linear_cross_entropy: w", w, ldw, w_mn_major ? vocab : dim));
      if (dx) MM_TRY(check_matrix("linear_cross_entropy: dx", dx, lddx, dim));
    }
    if (dw) MM_TRY(check_matrix("linear_cross_entropy: dw", dw, lddw, w_mn_major ? vocab : dim));
    const cudaStream_t st = as_stream(stream);
    if (rows == 0) {
      if (mean_loss) mm::check_cuda(cudaMemsetAsync(mean_loss, 0, 4, st), "mean loss");
      if (dw && !accumulate)
        mm::check_cuda(cudaMemset2DAsync(dw, lddw * 4, 0, (w_mn_major ? vocab : dim) * 4ull, w_mn_major ? dim : vocab,
                                         st),
                       "dw");
      return MM_GPU_OK;
    }
    const bool exact = precision == MM_GPU_3XTF32;
    MM_TRY(check_workspace(workspace, workspace_bytes, mm::linear_loss_ws_bytes(rows, vocab, dim, dx || dw, exact)));
    MM_TRY(check_distinct("linear_cross_entropy", {dx, dw, row_loss, mean_loss}, {x, w, targets}));
    const mm::LinearLoss a{rows, vocab,     dim, x,    ldx, w,    ldw,  w_mn_major != 0,  targets,
                           grad_scale, row_loss, mean_loss, dx, lddx, dw, lddw, accumulate != 0, exact};
    return product_status(mm::linear_loss(a, workspace, mm::device_context().d_err, st));
  });
}

}  // extern "C"
