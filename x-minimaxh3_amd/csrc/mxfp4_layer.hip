// The 4-bit layer's forward and backward passes as one call each: the kernels of the other mxfp4 sources in sequence, with the
// intermediate codes, parts and sums in one workspace of the caller's.
#include "mxfp4_common.h"

using namespace mxq;

namespace {

struct Forward {
  uint8_t *q, *s;
  void* gemm;
  int64_t ldq, gemm_bytes, total;
};
// codes: the call makes its own copy of the codes.
int forward_space(uint8_t* base, int64_t M, int64_t N, int64_t K, bool pair, bool codes, Forward& f) {
  f = {};
  if (fp4_few_rows(M, N, K, pair)) return MXQ_OK;
  Carve c{base};
  f.ldq = fp4_row_bytes(K);
  f.q = c.take<uint8_t>(codes ? M * f.ldq : 0);
  f.s = c.take<uint8_t>(fp4_scale_bytes(M, K));
  if (const int rc = mxq_mxfp4_gemm_workspace(M, N, K, &f.gemm_bytes)) return rc;
  f.gemm = c.take<void>(f.gemm_bytes);
  f.total = c.used;
  return MXQ_OK;
}

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && N >= 1 && K >= 1 && M <= (1ll << 31) - 1024 && N <= (1ll << 22) && K <= (1ll << 22);
}

int parts_of(int dtype) { return dtype == MXQ_DTYPE_BF16 ? 1 : dtype == MXQ_DTYPE_F16 ? 2 : 3; }

struct Backward {
  void* parts;
  float* sums;
  void* dgrad;
  int64_t ldp, strips, total;
  int n_parts;
};
int backward_space(uint8_t* base, int64_t M, int64_t N, int64_t K, int dy_dtype, int direct, int needs, Backward& s) {
  s = {};
  Carve c{base};
  if (needs & 1) {
    s.n_parts = direct || M == 0 ? 0 : parts_of(dy_dtype);
    s.ldp = (N + 127) / 128 * 128;
    s.parts = c.take<void>(s.n_parts * M * s.ldp * 2);
    s.dgrad = c.take<void>(fp4_dgrad_workspace(M, N, K, direct ? 1 : parts_of(dy_dtype)));
  }
  if (needs & 2) {
    if (const int rc = mxq_fp8_grad_strips(M, N, &s.strips)) return rc;
    s.sums = c.take<float>(s.strips * N * 4);
  }
  s.total = c.used;
  return MXQ_OK;
}

int check_workspace(const void* workspace, int64_t have, int64_t need) {
  if (need > 0 && (!workspace || have < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)have, (long long)need);
  return MXQ_OK;
}

}  // namespace

extern "C" int mxq_mxfp4_linear_workspace(int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (!sizes_ok(M, N, K) || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  Forward f;
  if (const int rc = forward_space(nullptr, M, N, K, false, true, f)) return rc;
  *bytes = f.total;
  return MXQ_OK;
}

extern "C" int mxq_mxfp4_linear(const void* x, int x_dtype, int64_t ldx, const uint8_t* b, int64_t ldb, const uint8_t* sb,
                                const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  if (!sizes_ok(M, N, K))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (M == 0) return MXQ_OK;
  if (!float_dtype(x_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported input dtype code %d", x_dtype);
  if (!x || ldx < K) return mxq_set_error(MXQ_ERR_INVALID, "null activations or bad row strides of the activations for K=%lld", (long long)K);
  if (fp4_few_rows(M, N, K, false))
    return fp4_linear_rows(x, x_dtype, ldx, nullptr, 0, b, ldb, sb, bias, d, ldd, out_dtype, M, N, K, stream);
  Forward f;
  if (const int rc = forward_space((uint8_t*)workspace, M, N, K, false, true, f)) return rc;
  if (const int rc = check_workspace(workspace, workspace_bytes, f.total)) return rc;
  // (every refusal is ahead of the first launch)
  if (const int rc = fp4_gemm_check(f.q, f.ldq, f.s, b, ldb, sb, d, ldd, out_dtype, M, N, K)) return rc;
  if (const int rc = mxq_mxfp4_quantize_rows(x, x_dtype, ldx, f.q, f.ldq, f.s, 0, M, K, stream)) return rc;
  return mxq_mxfp4_gemm(f.q, f.ldq, f.s, b, ldb, sb, bias, d, ldd, out_dtype, M, N, K, f.gemm, f.gemm_bytes, stream);
}

extern "C" int mxq_mxfp4_linear_prequantized_workspace(int64_t M, int64_t N, int64_t K, int direct, int64_t* bytes) {
  if (!sizes_ok(M, N, K) || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  Forward f;
  if (const int rc = forward_space(nullptr, M, N, K, true, !direct, f)) return rc;
  *bytes = f.total;
  return MXQ_OK;
}

extern "C" int mxq_mxfp4_linear_prequantized(const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, int direct,
                                             const uint8_t* b, int64_t ldb, const uint8_t* sb, const void* bias, void* d, int64_t ldd,
                                             int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                                             void* stream) {
  if (!sizes_ok(M, N, K))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (ldq < (K + 1) / 2 || lds < (K + 31) / 32)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the activations for K=%lld", (long long)K);
  if (direct && (K % 256 || ldq % 16 || ldq > (1ll << 22) || reinterpret_cast<uintptr_t>(q) % 16))
    return mxq_set_error(MXQ_ERR_INVALID, "the product cannot read these codes directly");
  if (M == 0) return MXQ_OK;
  if (!q || !scale) return mxq_set_error(MXQ_ERR_INVALID, "null activations");
  if (fp4_few_rows(M, N, K, true))
    return fp4_linear_rows(q, MXQ_DTYPE_E2M1, ldq, scale, lds, b, ldb, sb, bias, d, ldd, out_dtype, M, N, K, stream);
  Forward f;
  if (const int rc = forward_space((uint8_t*)workspace, M, N, K, true, !direct, f)) return rc;
  if (const int rc = check_workspace(workspace, workspace_bytes, f.total)) return rc;
  const uint8_t* a = direct ? q : f.q;
  const int64_t lda = direct ? ldq : f.ldq;
  if (const int rc = fp4_gemm_check(a, lda, f.s, b, ldb, sb, d, ldd, out_dtype, M, N, K)) return rc;
  if (const int rc = mxq_mxfp4_layout(q, ldq, scale, lds, direct ? nullptr : f.q, f.ldq, f.s, M, K, stream)) return rc;
  return mxq_mxfp4_gemm(a, lda, f.s, b, ldb, sb, bias, d, ldd, out_dtype, M, N, K, f.gemm, f.gemm_bytes, stream);
}

extern "C" int mxq_mxfp4_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int dy_dtype, int direct, int needs, int64_t* bytes) {
  if (!sizes_ok(M, N, K) || !float_dtype(dy_dtype) || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  Backward s;
  if (const int rc = backward_space(nullptr, M, N, K, dy_dtype, direct, needs, s)) return rc;
  *bytes = s.total;
  return MXQ_OK;
}

extern "C" int mxq_mxfp4_linear_backward(const void* dy, int dy_dtype, int64_t ldy, int direct, const uint8_t* b, int64_t ldb,
                                         const uint8_t* sb, void* dx, void* db, int grad_dtype, int64_t M, int64_t N, int64_t K,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
  if (!sizes_ok(M, N, K))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (!float_dtype(dy_dtype) || !float_dtype(grad_dtype))
    return mxq_set_error(MXQ_ERR_INVALID, "unsupported dtype codes %d, %d", dy_dtype, grad_dtype);
  if (direct && (dy_dtype != MXQ_DTYPE_BF16 || N % 8 || ldy % 8 || ldy >= (1 << 24) || reinterpret_cast<uintptr_t>(dy) % 16))
    return mxq_set_error(MXQ_ERR_INVALID, "the input's gradient cannot read this dy directly");
  if (M > 0 && (!dy || ldy < N)) return mxq_set_error(MXQ_ERR_INVALID, "null gradient or bad row stride %lld", (long long)ldy);
  const int needs = (dx && M ? 1 : 0) | (db ? 2 : 0);
  Backward s;
  if (const int rc = backward_space((uint8_t*)workspace, M, N, K, dy_dtype, direct, needs, s)) return rc;
  if (const int rc = check_workspace(workspace, workspace_bytes, s.total)) return rc;
  const void* wy = s.n_parts ? s.parts : dy;
  const int64_t ldwy = s.n_parts ? s.ldp : ldy;
  if (needs & 1) {
    if (const int rc = fp4_dgrad_check(wy, ldwy, b, ldb, sb, dx, dy_dtype, M, N, K)) return rc;
  }
  if (M > 0 && (db || s.n_parts)) {
    if (const int rc = mxq_fp8_grad_pass(dy, dy_dtype, ldy, nullptr, 0, nullptr, 0, s.n_parts ? s.parts : nullptr, s.n_parts, s.ldp,
                                         db ? s.sums : nullptr, s.strips, M, N, stream))
      return rc;
  }
  SliceJob join = {};
  if (needs & 1) {
    if (const int rc = fp4_dgrad(wy, s.n_parts ? s.n_parts : 1, ldwy, b, ldb, sb, dx, dy_dtype, M, N, K, s.dgrad, &join, stream)) return rc;
  }
  return fp8_join(join, {}, {s.sums, db, s.strips, N, grad_dtype}, stream);
}

extern "C" int mxq_mxfp4_linear_plan(int64_t M, int64_t N, int64_t K, int pair, int64_t* plan) {
  if (!sizes_ok(M, N, K) || M == 0 || !plan) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  const bool few = fp4_few_rows(M, N, K, pair != 0);
  const Fp4RowsForm r = few ? fp4_rows_form(M, N, K) : Fp4RowsForm{0, 0};
  const Fp4TileForm t = few ? Fp4TileForm{0, 0, 0} : fp4_gemm_form(M, N, K);
  plan[0] = r.rows;
  plan[1] = r.waves;
  plan[2] = t.rows;
  plan[3] = t.cols;
  plan[4] = t.slices;
  return MXQ_OK;
}

extern "C" int mxq_mxfp4_linear_backward_plan(int64_t M, int64_t N, int64_t K, int dy_dtype, int64_t* plan) {
  if (!sizes_ok(M, N, K) || M == 0 || !float_dtype(dy_dtype) || !plan) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  const Fp4TileForm t = fp4_dgrad_form(M, N, K, parts_of(dy_dtype));
  plan[0] = t.rows;
  plan[1] = t.cols;
  plan[2] = t.slices;
  return MXQ_OK;
}
