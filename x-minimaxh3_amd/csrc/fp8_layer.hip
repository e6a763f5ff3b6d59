// The 8-bit layer's forward and backward passes as one call each: the kernels of the other fp8 sources in sequence, with
// the intermediate codes, parts and sums in one workspace of the caller's. A layer of a few hundred rows is several
// kernels of 5 to 20 us; a call and an allocation per kernel took the host longer than that.
#include "fp8_common.h"

using namespace mxq;

namespace {

struct Pair {  // codes and scales of [rows, cols]
  uint8_t *q, *s;
  int64_t ldq, lds;
};
Pair take_pair(Carve& c, int64_t rows, int64_t cols) {
  const int64_t kb = up(cols, 128) / 128;
  Pair p;
  p.ldq = kb * 128;
  p.lds = up(kb, 4);
  p.q = c.take<uint8_t>(rows * p.ldq);
  p.s = c.take<uint8_t>(rows * p.lds);
  return p;
}

struct ForwardSpace {
  Pair x;
  void* gemm;
  int64_t gemm_bytes, total;
};
int forward_space(uint8_t* base, int64_t M, int64_t N, int64_t K, ForwardSpace& f) {
  f = {};
  if (M <= kFp8FusedRows) return MXQ_OK;
  Carve c{base};
  f.x = take_pair(c, M, K);
  if (const int rc = mxq_fp8_gemm_workspace(M, N, K, &f.gemm_bytes)) return rc;
  f.gemm = c.take<void>(f.gemm_bytes);
  f.total = c.used;
  return MXQ_OK;
}

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && N >= 1 && K >= 1 && M <= (1ll << 31) - 1024 && N <= (1ll << 22) && K <= (1ll << 22);
}

struct BackwardSpace {
  Pair dy, x;
  void* parts;
  float* sums;
  void *gemm, *wgrad;
  int64_t ldp, strips, gemm_bytes, wgrad_bytes, total;
  int n_parts;
};
int backward_space(uint8_t* base, int64_t M, int64_t N, int64_t K, int dy_dtype, int direct, int readable, int needs,
                   BackwardSpace& s) {
  s = {};
  Carve c{base};
  const int most = dy_dtype == MXQ_DTYPE_BF16 ? 1 : dy_dtype == MXQ_DTYPE_F16 ? 2 : 3;
  if (needs & 1) {
    s.dy = take_pair(c, M, N);
    if (const int rc = mxq_fp8_gemm_workspace(M, K, N, &s.gemm_bytes)) return rc;
    s.gemm = c.take<void>(s.gemm_bytes);
  }
  if (needs & 2) {
    s.n_parts = direct || M == 0 ? 0 : most;
    s.ldp = up(N, 128);
    s.parts = c.take<void>(s.n_parts * M * s.ldp * 2);
    if (const int rc = mxq_fp8_wgrad_workspace(M, N, K, direct ? 1 : most, &s.wgrad_bytes)) return rc;
    s.wgrad = c.take<void>(s.wgrad_bytes);
    if (!readable) {
      s.x.ldq = up(K, 128);
      s.x.q = c.take<uint8_t>(M * s.x.ldq);
    }
  }
  if (needs & 4) {
    if (const int rc = mxq_fp8_grad_strips(M, N, &s.strips)) return rc;
    s.sums = c.take<float>(s.strips * N * 4);
  }
  s.total = c.used;
  return MXQ_OK;
}

}  // namespace

extern "C" int mxq_fp8_linear_workspace(int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (!sizes_ok(M, N, K) || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  ForwardSpace f;
  if (const int rc = forward_space(nullptr, M, N, K, f)) return rc;
  *bytes = f.total;
  return MXQ_OK;
}

extern "C" int mxq_fp8_linear(const void* x, int x_dtype, int64_t ldx, const uint8_t* b, int64_t ldb, const uint8_t* sb,
                              int64_t ldsb, const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N,
                              int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!sizes_ok(M, N, K))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (M == 0) return MXQ_OK;
  if (!float_dtype(x_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported input dtype code %d", x_dtype);
  if (M <= kFp8FusedRows)
    return fp8_linear_rows(x, x_dtype, ldx, nullptr, 0, b, ldb, sb, ldsb, bias, d, ldd, out_dtype, M, N, K, stream);
  ForwardSpace f;
  if (const int rc = forward_space((uint8_t*)workspace, M, N, K, f)) return rc;
  if (!workspace || workspace_bytes < f.total || reinterpret_cast<uintptr_t>(workspace) % 16)
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)f.total);
  // (every refusal is ahead of the first launch)
  if (const int rc = fp8_gemm_check(f.x.q, f.x.ldq, f.x.s, f.x.lds, b, ldb, sb, ldsb, d, ldd, out_dtype, M, N, K)) return rc;
  if (const int rc = mxq_fp8_quantize_rows(x, x_dtype, ldx, f.x.q, f.x.ldq, f.x.s, f.x.lds, M, K, stream)) return rc;
  return mxq_fp8_gemm(f.x.q, f.x.ldq, f.x.s, f.x.lds, b, ldb, sb, ldsb, bias, d, ldd, out_dtype, M, N, K, f.gemm, f.gemm_bytes, stream);
}

extern "C" int mxq_fp8_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int dy_dtype, int direct, int readable,
                                                 int needs, int64_t* bytes) {
  dy_dtype &= ~MXQ_FP8_FULL_SUMS;
  if (!sizes_ok(M, N, K) || !float_dtype(dy_dtype) || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  BackwardSpace s;
  if (const int rc = backward_space(nullptr, M, N, K, dy_dtype, direct, readable, needs, s)) return rc;
  *bytes = s.total;
  return MXQ_OK;
}

extern "C" int mxq_fp8_linear_backward(const void* dy, int dy_dtype, int64_t ldy, int direct, const uint8_t* q, int64_t ldq,
                                       const uint8_t* scale, int64_t lds, int readable, const uint8_t* bt, int64_t ldbt,
                                       const uint8_t* sbt, int64_t ldsbt, void* dx, void* dw, void* db, int grad_dtype, int64_t M,
                                       int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  const int dx_dtype = dy_dtype;  // (with MXQ_FP8_FULL_SUMS or without)
  dy_dtype &= ~MXQ_FP8_FULL_SUMS;
  if (!sizes_ok(M, N, K))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (!float_dtype(dy_dtype) || !float_dtype(grad_dtype))
    return mxq_set_error(MXQ_ERR_INVALID, "unsupported dtype codes %d, %d", dy_dtype, grad_dtype);
  if (direct && (dy_dtype != MXQ_DTYPE_BF16 || N % 16 || ldy % 8 || reinterpret_cast<uintptr_t>(dy) % 16))
    return mxq_set_error(MXQ_ERR_INVALID, "the weight's gradient cannot read this dy directly");
  const int needs = (dx ? 1 : 0) | (dw ? 2 : 0) | (db ? 4 : 0);
  BackwardSpace s;
  if (const int rc = backward_space((uint8_t*)workspace, M, N, K, dy_dtype, direct, readable, needs, s)) return rc;
  if (s.total > 0 && (!workspace || workspace_bytes < s.total || reinterpret_cast<uintptr_t>(workspace) % 16))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)s.total);
  // What the last step reads of the input: its own rows, or copies of them. (Every refusal is ahead of the first launch.)
  const void* wy = s.n_parts ? s.parts : dy;
  const int64_t ldwy = s.n_parts || M == 0 ? s.ldp : ldy;
  const bool copied = M > 0 && !readable;
  const uint8_t* wq = copied ? s.x.q : q;
  const int64_t ldwq = M == 0 ? up(K, 16) : copied ? s.x.ldq : ldq, ldws = M == 0 ? up(K, 128) / 128 : lds;
  if (M > 0 && (!dy || ldy < N)) return mxq_set_error(MXQ_ERR_INVALID, "null gradient or bad row stride %lld", (long long)ldy);
  if (dx && M > 0) {
    if (const int rc = fp8_gemm_check(s.dy.q, s.dy.ldq, s.dy.s, s.dy.lds, bt, ldbt, sbt, ldsbt, dx, K, dx_dtype, M, K, N)) return rc;
  }
  if (dw) {
    if (copied && (!q || ldq < K)) return mxq_set_error(MXQ_ERR_INVALID, "null codes or bad row stride %lld", (long long)ldq);
    if (const int rc = fp8_wgrad_check(wy, s.n_parts ? s.n_parts : 1, ldwy, wq, ldwq, scale, ldws, dw, grad_dtype, M, N, K)) return rc;
  }
  if (M > 0 && (dx || db || s.n_parts)) {
    if (const int rc = mxq_fp8_grad_pass(dy, dy_dtype, ldy, dx ? s.dy.q : nullptr, s.dy.ldq, s.dy.s, s.dy.lds,
                                         s.n_parts ? s.parts : nullptr, s.n_parts, s.ldp, db ? s.sums : nullptr, s.strips, M, N,
                                         stream))
      return rc;
  }
  SliceJob join_x = {}, join_w = {};
  if (dx && M > 0) {
    if (const int rc = fp8_gemm(s.dy.q, s.dy.ldq, s.dy.s, s.dy.lds, bt, ldbt, sbt, ldsbt, nullptr, dx, K, dx_dtype, M, K, N, s.gemm,
                                s.gemm_bytes, &join_x, stream))
      return rc;
  }
  if (dw) {
    if (copied) {
      if (const int rc = mxq_pad_rows(q, ldq, K, s.x.q, s.x.ldq, M, stream)) return rc;
    }
    if (const int rc = fp8_wgrad(wy, s.n_parts ? s.n_parts : 1, ldwy, wq, ldwq, scale, ldws, dw, grad_dtype, M, N, K, s.wgrad,
                                 s.wgrad_bytes, &join_w, stream))
      return rc;
  }
  return fp8_join(join_x, join_w, {s.sums, db, s.strips, N, grad_dtype}, stream);
}
