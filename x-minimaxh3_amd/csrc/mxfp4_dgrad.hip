// Input gradient through a weight held in 4 bits (mxfp4_common.h):
//
//   dX[m, k] = sum_n dY[m, n] * W[n, k],   W[n, k] = code[n, k] * 2^(b[n, k / 32] - 127)
//
// dY is bfloat16 (float16 and float32 gradients come as two and three bfloat16 parts whose products are summed) and W is
// decoded to bfloat16, which is exact: the only roundings are those of the float32 sums. The simplest form: a wave per
// 32 x 32 block of dX, operands straight from memory.
#include "mxfp4_common.h"

namespace mxq {

struct Dgrad {
  const uint16_t* dy;  // part p at dy + p * part_stride
  const uint8_t *b, *sb;
  void* d;
  int64_t M, N, K, ldy, part_stride, ldb;
  int parts, groups;
};

template <int kOut>
__global__ __launch_bounds__(64) void mxfp4_dgrad_kernel(Dgrad p) {
  const int lane = threadIdx.x, lr = lane & 31, h = lane >> 5;
  const int64_t m0 = (int64_t)blockIdx.x * 32, k0 = (int64_t)blockIdx.y * 32, k = k0 + lr;
  const int block = (int)(k0 >> 5);
  v16f acc = {};
  for (int part = 0; part < p.parts; ++part) {
    const uint16_t* y = p.dy + part * p.part_stride + min(m0 + lr, p.M - 1) * p.ldy;
    for (int64_t n0 = 0; n0 < p.N; n0 += 16) {
      typedef short v8s __attribute__((ext_vector_type(8)));
      v8s fy, fw;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t n = n0 + 8 * h + i, at = min(n, p.N - 1);
        const uint32_t c = p.b[at * p.ldb + min(k, p.K - 1) / 2] >> (4 * (k & 1));
        const uint32_t s = p.sb[((at >> 5) * p.groups + (block >> 4)) * kFp4ScaleTile + fp4_scale_at((int)(at & 31), block & 15)];
        const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c & 15u, fp8_scale_f32(s), 0));
        fy[i] = n < p.N ? (short)y[n] : (short)0;
        fw[i] = n < p.N ? (short)(w & 0xFFFFu) : (short)0;
      }
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, fw), __builtin_bit_cast(v8bf, fy), acc, 0, 0, 0);
    }
  }
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  if (m0 + lr >= p.M) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int col = (int)k0 + q * 8 + h * 4;
    if (col >= p.K) continue;
    const float v[4] = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    store_run4<kOut>(reinterpret_cast<char*>(p.d) + (m0 + lr) * p.K * kElem, col, (int)p.K - col, v);
  }
}

int64_t fp4_dgrad_workspace(int64_t, int64_t, int64_t, int) { return 0; }

int fp4_dgrad_check(const void* dy, int64_t ldy, const uint8_t* b, int64_t ldb, const uint8_t* sb, const void* dx, int out_dtype,
                    int64_t M, int64_t N, int64_t K) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 1 || K < 1 || M > (1ll << 31) - 1024 || N > (1ll << 22) || K > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (ldy < N || ldb < fp4_row_bytes(K) || ldb % 16 || ldb > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldy=%lld ldb=%lld for N=%lld K=%lld", (long long)ldy, (long long)ldb,
                         (long long)N, (long long)K);
  if (M > 0 && (!dy || !b || !sb || !dx || reinterpret_cast<uintptr_t>(dy) % 2 || reinterpret_cast<uintptr_t>(b) % 16 ||
                reinterpret_cast<uintptr_t>(sb) % 16))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  return MXQ_OK;
}

int fp4_dgrad(const void* dy, int parts, int64_t ldy, const uint8_t* b, int64_t ldb, const uint8_t* sb, void* dx, int out_dtype,
              int64_t M, int64_t N, int64_t K, void*, SliceJob*, void* stream) {
  if (const int rc = fp4_dgrad_check(dy, ldy, b, ldb, sb, dx, out_dtype, M, N, K)) return rc;
  const Dgrad p = {(const uint16_t*)dy, b, sb, dx, M, N, K, ldy, M * ldy, ldb, parts, (int)fp4_groups(K)};
  const dim3 grid((unsigned)((M + 31) / 32), (unsigned)((K + 31) / 32));
  with_dtype(out_dtype, [&](auto O) {
    hipLaunchKernelGGL((mxfp4_dgrad_kernel<decltype(O)::value>), grid, dim3(64), 0, (hipStream_t)stream, p);
  });
  return mxq_check_launch("mxfp4_dgrad_kernel");
}

}  // namespace mxq
