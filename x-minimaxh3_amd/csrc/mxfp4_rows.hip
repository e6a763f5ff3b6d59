// The 4-bit layer of few rows (mxfp4_common.h). The simplest form: the quantizer's rows in LDS, a wave per 16 weight rows.
#include "mxfp4_common.h"

namespace mxq {

struct Fp4Rows {
  const void* x;
  const uint8_t *b, *sb;
  const void* bias;
  void* d;
  int64_t M, N, K, ldx, ldb, ldd;
  int x_code, groups, stages;
};

// One stage (256 columns) of all rows quantized into LDS: 16 rows of 128 bytes of codes, then 8 scale bytes each.
template <int kIn>
MXQ_DEVICE void quantize_stage(const Fp4Rows& p, uint8_t* lds, int stage, int lane) {
  constexpr int kElem = kIn == MXQ_DTYPE_F32 ? 4 : 2;
  for (int it = lane; it < 256; it += 64) {
    const int row = it >> 4, piece = it & 15, col = stage * 256 + piece * 16;
    const int n = row < p.M ? (int)p.K - col : 0;
    const Piece<kIn> t = piece_load<kIn>(reinterpret_cast<const char*>(p.x) + (n > 0 ? row * p.ldx + col : 0) * kElem, n);
    uint32_t m = piece_absmax(t);
    m = max(m, dpp_lane<kDppQuadXor1>(m));
    const uint32_t byte = fp4_scale_byte(m);
    v2u c = fp4_encode(t, fp8_scale_f32(byte));
    if (byte == 255u) c = v2u{0, 0};
    *reinterpret_cast<v2u*>(lds + row * 128 + piece * 8) = c;
    if ((piece & 1) == 0) lds[2048 + row * 8 + (piece >> 1)] = (uint8_t)byte;
  }
  wave_lds_fence();
}

template <int kOut>
__global__ __launch_bounds__(64) void mxfp4_rows_kernel(Fp4Rows p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2048 + 128];
  const int lane = threadIdx.x, lr = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, row = min(n0 + lr, p.N - 1);
  v4f acc = {};
  for (int s = 0; s < p.stages; ++s) {
    if (p.x_code == MXQ_DTYPE_BF16) quantize_stage<MXQ_DTYPE_BF16>(p, lds, s, lane);
    else if (p.x_code == MXQ_DTYPE_F16) quantize_stage<MXQ_DTYPE_F16>(p, lds, s, lane);
    else quantize_stage<MXQ_DTYPE_F32>(p, lds, s, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int block = 4 * j + g;
      const v4i w = *reinterpret_cast<const v4i*>(p.b + row * p.ldb + s * kFp4Stage + block * 16);
      const v4i x = *reinterpret_cast<const v4i*>(lds + lr * 128 + block * 16);
      const uint32_t sw = p.sb[((row >> 5) * p.groups + (s >> 1)) * kFp4ScaleTile + fp4_scale_at((int)(row & 31), (s & 1) * 8 + block)];
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v8i{w[0], w[1], w[2], w[3], 0, 0, 0, 0}, v8i{x[0], x[1], x[2], x[3], 0, 0, 0, 0},
                                                             acc, 4, 4, 0, (int)sw, 0, (int)lds[2048 + lr * 8 + block]);
    }
    wave_lds_fence();
  }
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  const int col = (int)n0 + g * 4;
  if (lr < p.M && col < p.N) {
    const v4f y = acc + bias_run<kOut>(p.bias, col, (int)p.N);
    const float v[4] = {y[0], y[1], y[2], y[3]};
    store_run4<kOut>(reinterpret_cast<char*>(p.d) + lr * p.ldd * kElem, col, (int)p.N - col, v);
  }
}

int fp4_linear_rows(const void* x, int x_dtype, int64_t ldx, const uint8_t* b, int64_t ldb, const uint8_t* sb, const void* bias, void* d,
                    int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K, void* stream) {
  if (const int rc = fp4_gemm_check(b, ldb, sb, b, ldb, sb, d, ldd, out_dtype, M, N, K)) return rc;
  const Fp4Rows p = {x, b, sb, bias, d, M, N, K, ldx, ldb, ldd, x_dtype, (int)fp4_groups(K), (int)(fp4_row_bytes(K) / kFp4Stage)};
  with_dtype(out_dtype, [&](auto O) {
    hipLaunchKernelGGL((mxfp4_rows_kernel<decltype(O)::value>), dim3((unsigned)((N + 15) / 16)), dim3(64), 0, (hipStream_t)stream, p);
  });
  return mxq_check_launch("mxfp4_rows_kernel");
}

}  // namespace mxq
