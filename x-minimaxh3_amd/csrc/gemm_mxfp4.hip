// Matrix product of MXFP4 operands (mxfp4_common.h) on gfx950 matrix cores:
//
//   D[m, n] = out( sum_b 2^(ea[m, b] + eb[n, b]) * sum_{k in block b} A[m, k] * B[n, k]  +  bias[n] )
//
// A [M, K] activations, B [N, K] a weight, both with one scale per row and 32 columns, sums in float32. The simplest form: a
// wave per 32 x 32 block of D, fragments straight from memory.

#include "mxfp4_common.h"

namespace mxq {

struct Fp4Gemm {
  const uint8_t *a, *b, *sa, *sb;
  const void* bias;
  void* d;
  int64_t M, N, lda, ldb, ldd;
  int groups, stages;
};

template <int kOut>
__global__ __launch_bounds__(64) void gemm_mxfp4_kernel(Fp4Gemm p) {
  const int lane = threadIdx.x, lr = lane & 31, h = lane >> 5;
  const int64_t m0 = (int64_t)blockIdx.x * 32, n0 = (int64_t)blockIdx.y * 32;
  const uint8_t* a = p.a + min(m0 + lr, p.M - 1) * p.lda;
  const uint8_t* b = p.b + min(n0 + lr, p.N - 1) * p.ldb;
  const uint8_t* sa = p.sa + (int64_t)blockIdx.x * p.groups * kFp4ScaleTile + lane * 8;
  const uint8_t* sb = p.sb + (int64_t)blockIdx.y * p.groups * kFp4ScaleTile + lane * 8;
  v16f acc = {};
  for (int s = 0; s < p.stages; ++s) {
    const uint32_t wa = *reinterpret_cast<const uint32_t*>(sa + (s >> 1) * kFp4ScaleTile + (s & 1) * 4);
    const uint32_t wb = *reinterpret_cast<const uint32_t*>(sb + (s >> 1) * kFp4ScaleTile + (s & 1) * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const v4i fa = *reinterpret_cast<const v4i*>(a + s * kFp4Stage + (4 * h + j) * 16);
      const v4i fb = *reinterpret_cast<const v4i*>(b + s * kFp4Stage + (4 * h + j) * 16);
      acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i{fb[0], fb[1], fb[2], fb[3], 0, 0, 0, 0},
                                                            v8i{fa[0], fa[1], fa[2], fa[3], 0, 0, 0, 0}, acc, 4, 4, 0,
                                                            (int)(wb >> (8 * j)), 0, (int)(wa >> (8 * j)));
    }
  }
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  if (m0 + lr >= p.M) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int col = (int)n0 + q * 8 + h * 4;
    if (col >= p.N) continue;
    const v4f bias = bias_run<kOut>(p.bias, col, (int)p.N);
    const float y[4] = {acc[4 * q] + bias[0], acc[4 * q + 1] + bias[1], acc[4 * q + 2] + bias[2], acc[4 * q + 3] + bias[3]};
    store_run4<kOut>(reinterpret_cast<char*>(p.d) + (m0 + lr) * p.ldd * kElem, col, (int)p.N - col, y);
  }
}

}  // namespace mxq

using namespace mxq;

static bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int mxq::fp4_gemm_check(const uint8_t* a, int64_t lda, const uint8_t* sa, const uint8_t* b, int64_t ldb, const uint8_t* sb,
                        const void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 1 || K < 1 || M > (1ll << 31) - 1024 || N > (1ll << 22) || K > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  const int64_t bytes = fp4_row_bytes(K);
  if (ldb < bytes || ldb % 16 || ldb > (1ll << 22) || ldd < N)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the weight or the output for N=%lld K=%lld", (long long)N, (long long)K);
  if (lda < bytes || lda % 16 || lda > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the activations for K=%lld", (long long)K);
  if (M == 0) return MXQ_OK;
  if (!a || !sa || !b || !sb || !d || !aligned(a, 16) || !aligned(b, 16) || !aligned(sa, 16) || !aligned(sb, 16))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  return MXQ_OK;
}

extern "C" int mxq_mxfp4_gemm_workspace(int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (M < 0 || N < 1 || K < 1 || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  *bytes = 0;
  return MXQ_OK;
}

extern "C" int mxq_mxfp4_gemm(const uint8_t* a, int64_t lda, const uint8_t* sa, const uint8_t* b, int64_t ldb, const uint8_t* sb,
                              const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K, void*, int64_t,
                              void* stream) {
  if (const int rc = fp4_gemm_check(a, lda, sa, b, ldb, sb, d, ldd, out_dtype, M, N, K)) return rc;
  if (M == 0) return MXQ_OK;
  const Fp4Gemm p = {a, b, sa, sb, bias, d, M, N, lda, ldb, ldd, (int)fp4_groups(K), (int)(fp4_row_bytes(K) / kFp4Stage)};
  const dim3 grid((unsigned)((M + 31) / 32), (unsigned)((N + 31) / 32));
  with_dtype(out_dtype, [&](auto O) {
    hipLaunchKernelGGL((gemm_mxfp4_kernel<decltype(O)::value>), grid, dim3(64), 0, (hipStream_t)stream, p);
  });
  return mxq_check_launch("gemm_mxfp4_kernel");
}
