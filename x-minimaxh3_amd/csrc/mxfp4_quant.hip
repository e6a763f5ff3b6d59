// Quantizer of the 4-bit format (mxfp4_common.h), the way back, and pairs laid out as the products read them.
#include "mxfp4_common.h"

namespace mxq {

// ---- rows: one scale per 1 x 32 block ----
// Two lanes hold a block, 16 elements each; the four blocks of eight lanes store one word of scale bytes. kTiled: scales in
// the products' tiles, every byte of a row's tiles written; else [M, lds]. Bound by HBM: 75600 x 5120 bf16 in 170 us, 5.8 TB/s.
template <int kCode, bool kTiled>
__global__ __launch_bounds__(256) void mxfp4_quant_kernel(const char* x, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* s,
                                                          int64_t lds, uint32_t M, uint32_t K, uint32_t units) {
  constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : 2;
  const uint32_t unit = blockIdx.x * 32 + (threadIdx.x >> 3), piece = threadIdx.x & 7;  // a unit: 128 columns of a row
  const uint32_t row = min(unit, M * units - 1) / units, u = min(unit, M * units - 1) - row * units, col = u * 128 + piece * 16;
  const int n = (int)K - (int)col;
  const Piece<kCode> p = piece_load<kCode>(x + ((int64_t)row * ldx + (n > 0 ? col : 0)) * kElem, n);
  uint32_t m = piece_absmax(p);
  m = max(m, dpp_lane<kDppQuadXor1>(m));
  const uint32_t byte = fp4_scale_byte(m);
  v2u codes = fp4_encode(p, fp8_scale_f32(byte));
  if (byte == 255u) codes = v2u{0, 0};
  uint32_t word = byte << (8 * (piece >> 1));
  word |= dpp_lane<kDppQuadXor2>(word);
  word |= lane_xor4(word);
  if (unit >= M * units) return;
  if ((int64_t)(col / 2) < ldq) *reinterpret_cast<v2u*>(q + (int64_t)row * ldq + col / 2) = codes;
  if (piece == 0) {
    uint8_t* d = kTiled ? s + ((int64_t)(row >> 5) * (units >> 2) + (u >> 2)) * kFp4ScaleTile + fp4_scale_at(row & 31, (u & 3) * 4)
                        : s + (int64_t)row * lds + u * 4;
    *reinterpret_cast<uint32_t*>(d) = word;
  }
}

// ---- the way back ----
// A lane takes eight codes (four of float32 outputs), so that a wave's stores are whole lines. Bound by HBM: 75600 x 5376 to bf16 in
// 165 us, 6.2 TB/s.
constexpr int kDequant4Unroll = 4;

template <int kCode>
__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const uint8_t* q, int64_t ldq, const uint8_t* s, int64_t lds, char* out,
                                                            uint32_t M, uint32_t K, uint32_t pieces) {
  constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : 2, kCodes = 16 / kElem;
  const uint32_t total = M * pieces;
  uint32_t c[kDequant4Unroll], row[kDequant4Unroll], col[kDequant4Unroll], sc[kDequant4Unroll];
#pragma unroll
  for (int u = 0; u < kDequant4Unroll; ++u) {
    const uint32_t g = min(blockIdx.x * (256 * kDequant4Unroll) + u * 256 + threadIdx.x, total - 1);
    row[u] = g / pieces;
    col[u] = (g - row[u] * pieces) * kCodes;
    const int bytes = min((int)(K - col[u] + 1) / 2, kCodes / 2);
    const uint8_t* src = q + (int64_t)row[u] * ldq + col[u] / 2;
    sc[u] = s[(int64_t)row[u] * lds + (col[u] >> 5)];
    c[u] = 0;
    if (bytes == kCodes / 2) {
      __builtin_memcpy(&c[u], src, kCodes / 2);
    } else {
#pragma unroll
      for (int i = 0; i < kCodes / 2; ++i) {
        const uint32_t v = src[min(i, bytes - 1)];
        c[u] |= (i < bytes ? v : 0u) << (8 * i);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kDequant4Unroll; ++u) {
    if (blockIdx.x * (256 * kDequant4Unroll) + u * 256 + threadIdx.x >= total) return;
    char* dst = out + ((int64_t)row[u] * K + col[u]) * kElem;
    const int n = (int)(K - col[u]);
    const float scale = fp8_scale_f32(sc[u]);
    if constexpr (kCodes == 4) {
      const v2f a = fp4x2_to_f32<0>(c[u], scale), b = fp4x2_to_f32<1>(c[u], scale);
      const float y[4] = {a[0], a[1], b[0], b[1]};
      store_run4<kCode>(dst, 0, n, y);
    } else {
      const v2f v[4] = {fp4x2_to_f32<0>(c[u], scale), fp4x2_to_f32<1>(c[u], scale), fp4x2_to_f32<2>(c[u], scale),
                        fp4x2_to_f32<3>(c[u], scale)};
      v4u o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = kCode == MXQ_DTYPE_F16 ? f32_to_f16_bits(v[i][0]) | (f32_to_f16_bits(v[i][1]) << 16) : pack_bf16x2(v[i][0], v[i][1]);
      if (n >= 8) {
        *reinterpret_cast<v4u_any*>(dst) = o;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) reinterpret_cast<uint16_t*>(dst)[i] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// ---- pairs of any making as the products read them ----
// A thread takes 16 bytes of a row's codes (nothing is read behind column K; its odd neighbour's code is cleared) and, every
// fourth, the word of scale bytes of those 128 columns (127 behind the row's last block).
__global__ __launch_bounds__(256) void mxfp4_layout_kernel(const uint8_t* q, int64_t ldq, const uint8_t* s, int64_t lds, uint8_t* qo,
                                                           int64_t ldqo, uint8_t* so, int64_t K, int64_t groups, int64_t total) {
  const int64_t pieces = groups * 16, kb = (K + 31) / 32, width = (K + 1) / 2;
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < total; g += (int64_t)gridDim.x * 256) {
    const int64_t row = g / pieces, p = g - row * pieces, byte0 = p * 16;
    if (qo && byte0 < ldqo) {
      const int64_t n = width - byte0;
      v4u v = bytes_load(q + row * ldq + (n > 0 ? byte0 : 0), (int)(n < 16 ? n : 16));
      if ((K & 1) && n >= 1 && n <= 16) {
        const int last = (int)n - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i == last >> 2) v[i] &= ~(0xF0u << (8 * (last & 3)));
      }
      *reinterpret_cast<v4u*>(qo + row * ldqo + byte0) = v;
    }
    if ((p & 3) == 0) {
      const int64_t b0 = p;  // (16 bytes of codes are one block)
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= (b0 + i < kb ? (uint32_t)s[row * lds + b0 + i] : 127u) << (8 * i);
      *reinterpret_cast<uint32_t*>(so + ((row >> 5) * groups + (b0 >> 4)) * kFp4ScaleTile + fp4_scale_at((int)(row & 31), (int)(b0 & 15))) = w;
    }
  }
}

}  // namespace mxq

using namespace mxq;

static bool aligned_to(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

extern "C" int mxq_mxfp4_quantize_rows(const void* x, int x_dtype, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds,
                                       int64_t M, int64_t K, void* stream) {
  if (!float_dtype(x_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported input dtype code %d", x_dtype);
  if (M < 0 || K < 1) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld K=%lld", (long long)M, (long long)K);
  const bool tiled = lds == 0;
  const int64_t least = tiled ? fp4_row_bytes(K) : (K + 31) / 32 * 16;
  if (K >= (1ll << 30) || ldx < K || ldq < least || ldq % 16 || (!tiled && (lds < (K + 127) / 128 * 4 || lds % 4)))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldx=%lld ldq=%lld lds=%lld for K=%lld", (long long)ldx, (long long)ldq,
                         (long long)lds, (long long)K);
  if (M == 0) return MXQ_OK;
  if (!x || !q || !scale || !aligned_to(q, 16) || !aligned_to(scale, 4)) return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  const int64_t units = tiled ? fp4_groups(K) * 4 : (K + 127) / 128;
  // (units are counted in 32 bits, eight lanes each: more of them are several launches, of whole scale tiles)
  const int64_t most = ((1ll << 29) / units - 32) / 32 * 32;
  if (most < 32) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "rows of more than 2^30 elements");
  for (int64_t row = 0; row < M; row += most) {
    const int64_t rows = M - row < most ? M - row : most;
    const unsigned grid = (unsigned)((rows * units + 31) / 32);
    with_dtype(x_dtype, [&](auto C) {
      constexpr int kCode = decltype(C)::value;
      const char* from = (const char*)x + row * ldx * dtype_bytes(kCode);
      if (tiled)
        hipLaunchKernelGGL((mxfp4_quant_kernel<kCode, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, from, ldx, q + row * ldq,
                           ldq, scale + row / 32 * (units / 4) * kFp4ScaleTile, 0, (uint32_t)rows, (uint32_t)K, (uint32_t)units);
      else
        hipLaunchKernelGGL((mxfp4_quant_kernel<kCode, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, from, ldx, q + row * ldq,
                           ldq, scale + row * lds, lds, (uint32_t)rows, (uint32_t)K, (uint32_t)units);
    });
  }
  return mxq_check_launch("mxfp4_quant_kernel");
}

extern "C" int mxq_mxfp4_dequantize_rows(const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, void* out, int out_dtype,
                                         int64_t M, int64_t K, void* stream) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || K < 1) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld K=%lld", (long long)M, (long long)K);
  if (K >= (1ll << 30) || ldq < (K + 1) / 2 || lds < (K + 31) / 32)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldq=%lld lds=%lld for K=%lld", (long long)ldq, (long long)lds, (long long)K);
  if (M == 0) return MXQ_OK;
  if (!q || !scale || !out) return mxq_set_error(MXQ_ERR_INVALID, "null pointer");
  const int codes = 16 / dtype_bytes(out_dtype);
  const int64_t pieces = (K + codes - 1) / codes;
  // (pieces are counted in 32 bits, so more of them are several launches)
  const int64_t most = (1ll << 31) / pieces - 65536 / pieces - 1;
  for (int64_t row = 0; row < M; row += most) {
    const int64_t rows = M - row < most ? M - row : most;
    const unsigned grid = (unsigned)((rows * pieces + 256 * kDequant4Unroll - 1) / (256 * kDequant4Unroll));
    with_dtype(out_dtype, [&](auto C) {
      hipLaunchKernelGGL((mxfp4_dequant_kernel<decltype(C)::value>), dim3(grid), dim3(256), 0, (hipStream_t)stream, q + row * ldq, ldq,
                         scale + row * lds, lds, (char*)out + row * K * dtype_bytes(out_dtype), (uint32_t)rows, (uint32_t)K,
                         (uint32_t)pieces);
    });
  }
  return mxq_check_launch("mxfp4_dequant_kernel");
}

extern "C" int mxq_mxfp4_layout(const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, uint8_t* q_out, int64_t ldqo,
                                uint8_t* scale_out, int64_t rows, int64_t K, void* stream) {
  if (rows < 0 || K < 1 || K >= (1ll << 30)) return mxq_set_error(MXQ_ERR_INVALID, "bad size rows=%lld K=%lld", (long long)rows, (long long)K);
  if (ldq < (K + 1) / 2 || lds < (K + 31) / 32 || (q_out && (ldqo < fp4_row_bytes(K) || ldqo % 16)))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides for K=%lld", (long long)K);
  if (rows == 0) return MXQ_OK;
  if (!scale || !scale_out || !aligned_to(scale_out, 4) || (q_out && (!q || !aligned_to(q_out, 16))))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  if (rows >= (1ll << 31)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "too many rows");
  const int64_t groups = fp4_groups(K), total = rows * groups * 16, blocks = (total + 255) / 256;
  hipLaunchKernelGGL(mxfp4_layout_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, (hipStream_t)stream, q,
                     ldq, scale, lds, q_out, ldqo, scale_out, K, groups, total);
  return mxq_check_launch("mxfp4_layout_kernel");
}
