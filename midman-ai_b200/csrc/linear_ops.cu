// The linear operators: which kernels a call runs, and its workspace.
#include <cuda_runtime.h>

#include <algorithm>

#include "device.h"
#include "linear.h"

namespace mm {
namespace {

long long round4(long long n) { return (n + 3) & ~3ll; }

struct ForwardPlan {
  bool pair;
  SplitCopy a, b;
  void* parts;
  long long bytes;
};
ForwardPlan forward_plan(int m, int n, int k, bool exact, void* ws) {
  ForwardPlan p{};
  Arena at{static_cast<uint8_t*>(ws)};
  p.pair = exact && m > 0 && pair_product_suits(m, n, k);
  if (p.pair) {
    p.a = at.copy(m, k);
    p.b = at.copy(n, k);
    p.parts = at.take(pair_ws_bytes(m, n, k));
  } else {
    p.parts = at.take(plain_ws_bytes(m, n, k, false, exact));
  }
  p.bytes = at.at;
  return p;
}

struct BackwardPlan {
  bool pair;
  SplitCopy dz, dzt, at, b;  // [m, n], [n, m], [k, m], [k, n]
  void *parts_da, *parts_db;  // of the products, which may run side by side
  float* dz_f32;
  float* sums;
  long long bytes;
};
BackwardPlan backward_plan(int m, int n, int k, bool exact, void* ws) {
  BackwardPlan p{};
  Arena at{static_cast<uint8_t*>(ws)};
  p.pair = exact && m > 0 && pair_product_suits(m, k, n) && pair_product_suits(k, n, m);
  if (p.pair) {
    p.dz = at.copy(m, n);
    p.dzt = at.copy(n, m);
    p.at = at.copy(k, m);
    p.b = at.copy(k, n);
    p.parts_da = at.take(pair_ws_bytes(m, k, n));
    p.parts_db = at.take(std::max(pair_ws_bytes(k, n, m), pair_ws_bytes(n, k, m)));
  } else {
    p.dz_f32 = static_cast<float*>(at.take(m * round4(n) * 4));
    p.parts_da = at.take(plain_ws_bytes(m, k, n, false, exact));
    p.parts_db = at.take(std::max(plain_ws_bytes(k, n, m, true, exact), plain_ws_bytes(n, k, m, true, exact)));
  }
  const long long parts = std::max(act_backward_parts(m, n), split_parts(m));
  p.sums = static_cast<float*>(at.take(parts * n * 4));
  p.bytes = at.at;
  return p;
}

}  // namespace

std::mutex& launch_order() {
  static std::mutex m;
  return m;
}

long long plain_ws_bytes(int M, int N, int K, bool a_mn_major, bool exact) {
  return !exact && tf32_pair_suits(M, N, K) ? tf32_pair_ws_bytes(M, N, K) : direct_ws_bytes(M, N, K, a_mn_major);
}
int plain_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LinearEpilogue& e, bool exact,
                  void* ws, int* d_err, cudaStream_t s) {
  if (!exact && tf32_pair_suits(M, N, K)) return tf32_pair_product(M, N, K, A, B, e, ws, d_err, s);
  return direct_product(M, N, K, A, B, e, exact, ws, d_err, s);
}
int plain_loss_product(int M, int N, int K, const GemmOperand& A, const GemmOperand& B, const LossEpilogue& e,
                       bool exact, int* d_err, cudaStream_t s) {
  if (!exact && tf32_pair_suits(M, N, K)) return tf32_pair_loss_product(M, N, K, A, B, e, d_err, s);
  return direct_loss_product(M, N, K, A, B, e, exact, d_err, s);
}

long long linear_forward_ws_bytes(int m, int n, int k, bool exact) {
  return forward_plan(m, n, k, exact, nullptr).bytes;
}

int linear_forward(const LinearForward& f, void* ws, int* d_err, cudaStream_t s) {
  if (f.m <= 0) return 0;
  const ForwardPlan p = forward_plan(f.m, f.n, f.k, f.exact, ws);
  if (!p.pair)
    return plain_product(f.m, f.n, f.k, {f.a, f.lda, false}, {f.b, f.ldb, f.b_mn_major}, f.e, f.exact, p.parts, d_err,
                         s);
  split_two({f.a, f.lda}, f.m, f.k, &p.a, nullptr, {f.b, f.ldb}, f.b_mn_major ? f.k : f.n, f.b_mn_major ? f.n : f.k,
            f.b_mn_major ? nullptr : &p.b, f.b_mn_major ? &p.b : nullptr, s);
  return pair_product(p.a, p.b, f.e, p.parts, d_err, s);
}

long long linear_backward_ws_bytes(int m, int n, int k, bool exact) {
  return backward_plan(m, n, k, exact, nullptr).bytes;
}

int linear_backward(const LinearBackward& f, void* ws, int* d_err, cudaStream_t s) {
  if (f.m <= 0 || !(f.da || f.db || f.dbias)) return 0;
  const BackwardPlan p = backward_plan(f.m, f.n, f.k, f.exact, ws);
  // A tensor that is both input and weight has one gradient buffer: then db's product reads
  // what da's wrote, and waits for it.
  const bool one_buffer = f.da == f.db;
  const std::lock_guard<std::mutex> lock(launch_order());
  LinearEpilogue da, db;
  da.C = f.da;
  da.R = f.accumulate ? f.da : nullptr;
  da.ldc = da.ldr = f.ldda;
  db.C = f.db;
  db.R = f.accumulate ? f.db : nullptr;
  db.ldc = db.ldr = f.lddb;
  int rc = 0;
  if (p.pair) {
    // dz goes from dc and z straight into its copies
    split(SplitBackward{f.dc, f.lddc, f.z, f.ldz, f.act, f.drop}, f.m, f.n, f.da ? &p.dz : nullptr,
          f.db ? &p.dzt : nullptr, f.dbias ? p.sums : nullptr, s);
    if (f.dbias) sum_parts(p.sums, split_parts(f.m), f.n, f.dbias, f.accumulate, s);
    // b [k, n] by rows, or [n, k] by columns, for da; a by columns for db
    const SplitMatrix a{f.a, f.lda}, b{f.b, f.ldb};
    const int br = f.b_mn_major ? f.k : f.n, bc = f.b_mn_major ? f.n : f.k;
    const SplitCopy *b_rows = f.b_mn_major ? &p.b : nullptr, *b_cols = f.b_mn_major ? nullptr : &p.b;
    if (f.da && f.db)
      split_two(b, br, bc, b_rows, b_cols, a, f.m, f.k, nullptr, &p.at, s);
    else if (f.da)
      split(b, br, bc, b_rows, b_cols, s);
    else if (f.db)
      split(a, f.m, f.k, nullptr, &p.at, s);
    db.late = f.da && !one_buffer;
    if (f.da) rc = pair_product(p.dz, p.b, da, p.parts_da, d_err, s);
    if (f.db && !rc)
      rc = f.b_mn_major ? pair_product(p.at, p.dzt, db, p.parts_db, d_err, s)
                        : pair_product(p.dzt, p.at, db, p.parts_db, d_err, s);
    return rc;
  }
  const bool plain = f.act == kActNone && !f.drop.rng;  // dz is dc
  const bool own_dz = !plain && (f.da || f.db);          // the products read it
  const long long ldz = round4(f.n);
  if (own_dz || f.dbias)
    act_backward(f.dc, f.lddc, f.z, f.ldz, f.act, f.drop, f.m, f.n, own_dz ? p.dz_f32 : nullptr, ldz,
                 f.dbias ? p.sums : nullptr, s);
  if (f.dbias) sum_parts(p.sums, act_backward_parts(f.m, f.n), f.n, f.dbias, f.accumulate, s);
  // da beside the bias gradient's sums, db beside da
  da.late = f.dbias != nullptr;
  db.late = (da.late || f.da) && !one_buffer;
  const float* g = plain ? f.dc : p.dz_f32;
  const long long ldg = plain ? f.lddc : ldz;
  if (f.da)
    rc = plain_product(f.m, f.k, f.n, {g, ldg, false}, {f.b, f.ldb, !f.b_mn_major}, da, f.exact, p.parts_da, d_err, s);
  if (f.db && !rc) {
    const GemmOperand ao{f.a, f.lda, true}, go{g, ldg, true};
    rc = f.b_mn_major ? plain_product(f.k, f.n, f.m, ao, go, db, f.exact, p.parts_db, d_err, s)
                      : plain_product(f.n, f.k, f.m, go, ao, db, f.exact, p.parts_db, d_err, s);
  }
  return rc;
}

}  // namespace mm
