// Quantizers of the block-128 e4m3 format (fp8_common.h), the way back, and the pass over an output's gradient.
#include "fp8_common.h"

namespace mxq {

// ---- rows: one scale per 1 x 128 block ----
// Eight lanes hold a block, 16 elements each, so a wave's loads cover whole lines, a block's maximum stays inside
// eight lanes and every lane stores 16 codes. HBM-bound: 75600 x 5120 bf16 in 190 us (6.1 TB/s), 8192 x 20480 in 102.
// One piece per lane: two to four in flight per lane took longer at every size (720p 197 and 201 us, 333 x 5000 fp16 4.4 and
// 5.2 us against 4.4), the waves of a CU keep enough loads under way.
template <int kCode>
__global__ __launch_bounds__(256) void fp8_rows_quant_kernel(const char* x, int64_t ldx, uint8_t* q, int64_t ldq,
                                                             uint8_t* s, int64_t lds, uint32_t M, uint32_t K, uint32_t kb) {
  constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : 2;
  const uint32_t block = blockIdx.x * 32 + (threadIdx.x >> 3), piece = threadIdx.x & 7;
  const uint32_t row = min(block, M * kb - 1) / kb, b = min(block, M * kb - 1) - row * kb, col = b * 128 + piece * 16;
  const Piece<kCode> p = piece_load<kCode>(x + ((int64_t)row * ldx + col) * kElem, (int)K - (int)col);
  const uint32_t byte = block_scale_byte(p);
  const v4u codes = piece_encode(p, fp8_scale_f32(byte));
  if (block < M * kb) {
    *reinterpret_cast<v4u*>(q + (int64_t)row * ldq + col) = codes;
    if (piece == 0) s[(int64_t)row * lds + b] = (uint8_t)byte;
  }
}

// ---- the way back ----
// A lane takes the codes whose values fill one 16-byte store, so that a wave's stores are whole lines. 8192 x 20480 to bf16
// in 77 us.
constexpr int kDequantUnroll = 4;  // (8192 x 20480: 76 us, with one 83)

template <int kCode>
__global__ __launch_bounds__(256) void fp8_rows_dequant_kernel(const uint8_t* q, int64_t ldq, const uint8_t* s, int64_t lds,
                                                               char* out, uint32_t M, uint32_t K, uint32_t pieces) {
  constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : 2, kCodes = 16 / kElem;
  const uint32_t total = M * pieces;
  uint32_t c[kDequantUnroll][2], row[kDequantUnroll], col[kDequantUnroll], sc[kDequantUnroll];
#pragma unroll
  for (int u = 0; u < kDequantUnroll; ++u) {
    const uint32_t g = min(blockIdx.x * (256 * kDequantUnroll) + u * 256 + threadIdx.x, total - 1);
    row[u] = g / pieces;
    col[u] = (g - row[u] * pieces) * kCodes;
    const int n = (int)(K - col[u]);
    const uint8_t* src = q + (int64_t)row[u] * ldq + col[u];
    sc[u] = s[(int64_t)row[u] * lds + (col[u] >> 7)];
    c[u][0] = c[u][1] = 0;
    if (n >= kCodes) {
      if constexpr (kCodes == 8) {
        const v2u v = *reinterpret_cast<const v2u_any*>(src);
        c[u][0] = v[0];
        c[u][1] = v[1];
      } else {
        __builtin_memcpy(&c[u][0], src, 4);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCodes; ++i) {
        const uint32_t v = src[min(i, n - 1)];
        c[u][i >> 2] |= (i < n ? v : 0u) << (8 * (i & 3));
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kDequantUnroll; ++u) {
    if (blockIdx.x * (256 * kDequantUnroll) + u * 256 + threadIdx.x >= total) return;
    char* dst = out + ((int64_t)row[u] * K + col[u]) * kElem;
    const int n = (int)(K - col[u]);
    const float scale = fp8_scale_f32(sc[u]);
    if constexpr (kCodes == 4) {
      const v4f v = fp8x4_to_f32(c[u][0], scale);
      const float y[4] = {v[0], v[1], v[2], v[3]};
      store_run4<kCode>(dst, 0, n, y);
    } else {
      const v4f v = fp8x4_to_f32(c[u][0], scale), w = fp8x4_to_f32(c[u][1], scale);
      auto pair = [](float a, float b) {
        return kCode == MXQ_DTYPE_F16 ? f32_to_f16_bits(a) | (f32_to_f16_bits(b) << 16) : pack_bf16x2(a, b);
      };
      const v4u o = {pair(v[0], v[1]), pair(v[2], v[3]), pair(w[0], w[1]), pair(w[2], w[3])};
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

// `n` of 16 bytes from s, zeros behind them (n <= 0: nothing is read).
MXQ_DEVICE v4u bytes_load(const uint8_t* s, int n) {
  v4u v = {0, 0, 0, 0};
  if (n >= 16) {
    v = *reinterpret_cast<const v4u_any*>(s);
  } else if (n > 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t b = s[min(i, n - 1)];
      v[i >> 2] |= (i < n ? b : 0u) << (8 * (i & 3));
    }
  }
  return v;
}

// ---- weights: one scale per 128 x 128 tile, and the transposed codes that the input's gradient reads ----
// One workgroup per tile: row t / 8 + 32 i, piece t % 8. The transposed copy goes through a 16 KB byte tile in LDS.
// HBM-bound: 21504 x 5376 bf16 in 90 us (5.1 TB/s) with the transposed copy, 65 without.
// Writes a tile's codes (c[i]: row t / 8 + 32 i, piece t % 8) and scale byte, and those of the transposed copy.
struct TileOut {
  uint8_t *q, *s, *qt, *st;
  int64_t ldq, lds, ldqt, ldst, N, K;
};
MXQ_DEVICE void store_tile(const TileOut& o, uint8_t* tile, const v4u (&c)[4], uint32_t byte) {
  const int t = threadIdx.x, piece = t & 7;
  const int64_t n0 = (int64_t)blockIdx.y * 128, k0 = (int64_t)blockIdx.x * 128, col = k0 + piece * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (t >> 3) + 32 * i;
    if (n0 + r < o.N) *reinterpret_cast<v4u*>(o.q + (n0 + r) * o.ldq + col) = c[i];
    if (o.qt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(tile + r * 132 + piece * 16 + 4 * j) = c[i][j];
    }
  }
  if (t == 0) o.s[blockIdx.y * o.lds + blockIdx.x] = (uint8_t)byte;
  if (!o.qt) return;
  if (t == 0) o.st[blockIdx.x * o.ldst + blockIdx.y] = (uint8_t)byte;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = (t >> 3) + 32 * i;  // row of the transposed tile
    if (k0 + k < o.K) {
      v4u v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t u = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) u |= (uint32_t)tile[(piece * 16 + 4 * j + e) * 132 + k] << (8 * e);
        v[j] = u;
      }
      *reinterpret_cast<v4u*>(o.qt + (k0 + k) * o.ldqt + n0 + piece * 16) = v;
    }
  }
}

template <int kCode>
__global__ __launch_bounds__(256) void fp8_tiles_quant_kernel(const char* w, int64_t ldw, TileOut o) {
  constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : 2;
  __shared__ uint32_t wave_max[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 132];  // rows of 132: a column's bytes spread over the banks
  const int t = threadIdx.x, piece = t & 7;
  const int64_t n0 = (int64_t)blockIdx.y * 128, col = (int64_t)blockIdx.x * 128 + piece * 16;
  Piece<kCode> p[4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = n0 + (t >> 3) + 32 * i;
    p[i] = piece_load<kCode>(w + (min(row, o.N - 1) * ldw + col) * kElem, row < o.N ? (int)(o.K - col) : 0);
    m = max(m, piece_absmax(p[i]));
  }
  m = wave_max_u32(m);
  if ((t & 63) == 0) wave_max[t >> 6] = m;
  __syncthreads();
  m = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
  if (m >= 0x7F800000u) {  // (the whole workgroup)
    m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, piece_absmax_finite(p[i]));
    m = wave_max_u32(m);
    __syncthreads();
    if ((t & 63) == 0) wave_max[t >> 6] = m;
    __syncthreads();
    m = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
  }
  const uint32_t byte = fp8_scale_byte(m);
  const float scale = fp8_scale_f32(byte);
  v4u c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = piece_encode(p[i], scale);
  store_tile(o, tile, c, byte);
}

// The same of codes that are there already, with their scales [ceil(N / 128), ldws]: 21504 x 5376 in 65 us (5.3 TB/s).
__global__ __launch_bounds__(256) void fp8_tiles_copy_kernel(const uint8_t* w, int64_t ldw, const uint8_t* ws, int64_t ldws,
                                                             TileOut o) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 132];
  const int t = threadIdx.x;
  const int64_t n0 = (int64_t)blockIdx.y * 128, col = (int64_t)blockIdx.x * 128 + (t & 7) * 16;
  v4u c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = n0 + (t >> 3) + 32 * i;
    c[i] = bytes_load(w + min(row, o.N - 1) * ldw + col, row < o.N ? (int)(o.K - col) : 0);
  }
  store_tile(o, tile, c, ws[blockIdx.y * ldws + blockIdx.x]);
}

// ---- the pass over an output's gradient dY [M, N] ----
// One read of dY makes all that the three gradients need of it: its e4m3 rows (the input's gradient), bfloat16 parts
// of it where the weight's gradient cannot read dY itself (kParts: bf16 rows that are not 16-byte aligned 1, float16
// 2, float32 3: parts p0 = bf16(x), p1 = bf16(x - p0), p2 = bf16(x - p0 - p1), whose sum is x to 16 and 24 bits), and
// the column sums (the bias's gradient) of a strip of rows, in float32.
// A workgroup takes 512 columns x `strip` rows: 32 lanes across, 8 rows at a time. 8192 x 5376 bf16 (codes and sums) in
// 25 us (5.3 TB/s), 1501 x 3001 fp16 with two parts in 9.8 us.
template <int kCode, int kParts>
__global__ __launch_bounds__(256) void fp8_grad_pass_kernel(const char* x, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* s,
                                                            int64_t lds, uint16_t* parts, int64_t ldp, float* sums,
                                                            int64_t M, int64_t N, int64_t nb, int64_t strip) {
  constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : 2;
  __shared__ float part_sum[8][512];
  const int t = threadIdx.x, lane = t & 31, r = t >> 5;
  const int64_t col = (int64_t)blockIdx.x * 512 + lane * 16, block = col >> 7;
  const bool in = block < nb;  // (the same for the eight lanes of a block)
  const int64_t first = (int64_t)blockIdx.y * strip, last = min(first + strip, M);
  float acc[16] = {};
  for (int64_t row = first + r; row < last; row += 8) {
    const int n = in ? (int)(N - col) : 0;
    const Piece<kCode> p = piece_load<kCode>(x + (row * ldx + (n > 0 ? col : 0)) * kElem, n);
    if (sums) {
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] += piece_at(p, i);
    }
    if (q) {
      const uint32_t byte = block_scale_byte(p);
      const v4u c = piece_encode(p, fp8_scale_f32(byte));
      if (in) {
        *reinterpret_cast<v4u*>(q + row * ldq + col) = c;
        if ((lane & 7) == 0) s[row * lds + block] = (uint8_t)byte;
      }
    }
    if constexpr (kParts > 0) {
      if (in) {
        uint32_t w[kParts][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float a = piece_at(p, 2 * i), b = piece_at(p, 2 * i + 1);
#pragma unroll
          for (int k = 0; k < kParts; ++k) {
            w[k][i] = pack_bf16x2(a, b);
            // (NaN, an infinity, and a value that bfloat16 rounds to one leave no remainder)
            const float ra = a - bf16_lo(w[k][i]), rb = b - bf16_hi(w[k][i]);
            a = __builtin_fabsf(ra) < __builtin_inff() ? ra : 0.0f;
            b = __builtin_fabsf(rb) < __builtin_inff() ? rb : 0.0f;
          }
        }
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
          uint16_t* d = parts + ((int64_t)k * M + row) * ldp + col;
          *reinterpret_cast<v4u*>(d) = v4u{w[k][0], w[k][1], w[k][2], w[k][3]};
          *reinterpret_cast<v4u*>(d + 8) = v4u{w[k][4], w[k][5], w[k][6], w[k][7]};
        }
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) part_sum[r][lane * 16 + i] = acc[i];
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = t + 256 * h;
    const int64_t g = (int64_t)blockIdx.x * 512 + c;
    if (g < N) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v += part_sum[k][c];
      sums[blockIdx.y * N + g] = v;
    }
  }
}

// Rows of bytes copied to 16-byte rows `ldd` apart, zeros behind their `width`: codes and scales whose own rows are not.
__global__ __launch_bounds__(256) void pad_rows_kernel(const uint8_t* src, int64_t lds, int width, uint8_t* dst, int ldd,
                                                       int64_t total) {
  const int pieces = ldd / 16;
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < total; g += (int64_t)gridDim.x * 256) {
    const int64_t row = g / pieces;
    const int col = (int)(g - row * pieces) * 16, n = width - col;
    const uint8_t* s = src + row * lds + col;
    *reinterpret_cast<v4u*>(dst + row * ldd + col) = bytes_load(s, n);
  }
}

}  // namespace mxq

using namespace mxq;

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

extern "C" int mxq_fp8_quantize_rows(const void* x, int x_dtype, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* scale,
                                     int64_t lds, int64_t M, int64_t K, void* stream) {
  if (!float_dtype(x_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported input dtype code %d", x_dtype);
  if (M < 0 || K < 1) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld K=%lld", (long long)M, (long long)K);
  const int64_t kb = (K + 127) / 128;
  if (K >= (1ll << 30) || ldx < K || ldq < kb * 128 || ldq % 16 || lds < kb)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldx=%lld ldq=%lld lds=%lld for K=%lld", (long long)ldx,
                         (long long)ldq, (long long)lds, (long long)K);
  if (M == 0) return MXQ_OK;
  if (!x || !q || !scale || !aligned16(q)) return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  if (M > (1ll << 29) / kb - 32) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 2^29 blocks");  // (eight lanes each)
  const unsigned grid = (unsigned)((M * kb + 31) / 32);
  with_dtype(x_dtype, [&](auto C) {
    hipLaunchKernelGGL((fp8_rows_quant_kernel<decltype(C)::value>), dim3(grid), dim3(256), 0, (hipStream_t)stream,
                       (const char*)x, ldx, q, ldq, scale, lds, (uint32_t)M, (uint32_t)K, (uint32_t)kb);
  });
  return mxq_check_launch("fp8_rows_quant_kernel");
}

extern "C" int mxq_fp8_dequantize_rows(const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, void* out,
                                       int out_dtype, int64_t M, int64_t K, void* stream) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || K < 1) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld K=%lld", (long long)M, (long long)K);
  if (K >= (1ll << 30) || ldq < K || lds < (K + 127) / 128)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldq=%lld lds=%lld for K=%lld", (long long)ldq, (long long)lds,
                         (long long)K);
  if (M == 0) return MXQ_OK;
  if (!q || !scale || !out) return mxq_set_error(MXQ_ERR_INVALID, "null pointer");
  const int codes = 16 / dtype_bytes(out_dtype);
  const int64_t pieces = (K + codes - 1) / codes;
  // (pieces are counted in 32 bits, so more of them are several launches)
  const int64_t most = (1ll << 31) / pieces - 65536 / pieces - 1;
  for (int64_t row = 0; row < M; row += most) {
    const int64_t rows = M - row < most ? M - row : most;
    const unsigned grid = (unsigned)((rows * pieces + 256 * kDequantUnroll - 1) / (256 * kDequantUnroll));
    with_dtype(out_dtype, [&](auto C) {
      hipLaunchKernelGGL((fp8_rows_dequant_kernel<decltype(C)::value>), dim3(grid), dim3(256), 0, (hipStream_t)stream,
                         q + row * ldq, ldq, scale + row * lds, lds, (char*)out + row * K * dtype_bytes(out_dtype), (uint32_t)rows,
                         (uint32_t)K, (uint32_t)pieces);
    });
  }
  return mxq_check_launch("fp8_rows_dequant_kernel");
}

static int check_tiles(const TileOut& o, const void* w, int64_t ldw) {
  const int64_t kb = (o.K + 127) / 128, nb = (o.N + 127) / 128;
  if (o.N < 1 || o.K < 1) return mxq_set_error(MXQ_ERR_INVALID, "bad size N=%lld K=%lld", (long long)o.N, (long long)o.K);
  if (ldw < o.K || o.ldq < kb * 128 || o.ldq % 16 || o.lds < kb || (o.qt && (o.ldqt < nb * 128 || o.ldqt % 16 || o.ldst < nb)))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides for N=%lld K=%lld", (long long)o.N, (long long)o.K);
  if (!w || !o.q || !o.s || !aligned16(o.q) || (o.qt && (!o.st || !aligned16(o.qt))))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  if (nb > 65535 || kb >= (1ll << 23)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 65535 tile rows or 2^23 columns");
  return MXQ_OK;
}

extern "C" int mxq_fp8_quantize_tiles(const void* w, int w_dtype, int64_t ldw, uint8_t* q, int64_t ldq, uint8_t* scale,
                                      int64_t lds, uint8_t* qt, int64_t ldqt, uint8_t* scale_t, int64_t ldst, int64_t N,
                                      int64_t K, void* stream) {
  if (!float_dtype(w_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported weight dtype code %d", w_dtype);
  const TileOut o = {q, scale, qt, scale_t, ldq, lds, ldqt, ldst, N, K};
  if (const int rc = check_tiles(o, w, ldw)) return rc;
  with_dtype(w_dtype, [&](auto C) {
    hipLaunchKernelGGL((fp8_tiles_quant_kernel<decltype(C)::value>), dim3((unsigned)((K + 127) / 128), (unsigned)((N + 127) / 128)),
                       dim3(256), 0, (hipStream_t)stream, (const char*)w, ldw, o);
  });
  return mxq_check_launch("fp8_tiles_quant_kernel");
}

extern "C" int mxq_fp8_prepare_tiles(const uint8_t* w, int64_t ldw, const uint8_t* w_scale, int64_t ldws, uint8_t* q, int64_t ldq,
                                     uint8_t* scale, int64_t lds, uint8_t* qt, int64_t ldqt, uint8_t* scale_t, int64_t ldst,
                                     int64_t N, int64_t K, void* stream) {
  const TileOut o = {q, scale, qt, scale_t, ldq, lds, ldqt, ldst, N, K};
  if (const int rc = check_tiles(o, w, ldw)) return rc;
  if (!w_scale || ldws < (K + 127) / 128) return mxq_set_error(MXQ_ERR_INVALID, "null scale or bad row stride");
  hipLaunchKernelGGL(fp8_tiles_copy_kernel, dim3((unsigned)((K + 127) / 128), (unsigned)((N + 127) / 128)), dim3(256), 0,
                     (hipStream_t)stream, w, ldw, w_scale, ldws, o);
  return mxq_check_launch("fp8_tiles_copy_kernel");
}

// Rows per strip of the gradient pass: whole eights, about four workgroups per CU in all, at least 16 rows (1501 x 3001 fp16
// 9.8 us, at least 32: 12.0; at least 8 gave no more and doubles the sums to join).
static int64_t grad_strip(int64_t M, int64_t N) {
  const int64_t panels = (N + 511) / 512;
  const int64_t want = panels >= 4 * mxq_cu_count() ? 1 : 4 * mxq_cu_count() / panels;
  int64_t strip = ((M + want - 1) / want + 7) / 8 * 8;
  if (strip < 16) strip = 16;
  const int64_t least = ((M + 65534) / 65535 + 7) / 8 * 8;  // grid.y
  return strip < least ? least : strip;
}

extern "C" int mxq_fp8_grad_strips(int64_t M, int64_t N, int64_t* strips) {
  if (M < 0 || N < 1 || !strips) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld", (long long)M, (long long)N);
  const int64_t strip = grad_strip(M, N);
  *strips = M == 0 ? 0 : (M + strip - 1) / strip;
  return MXQ_OK;
}

extern "C" int mxq_fp8_grad_pass(const void* dy, int dy_dtype, int64_t ldy, uint8_t* q, int64_t ldq, uint8_t* scale,
                                 int64_t lds, void* parts, int n_parts, int64_t ldp, float* sums, int64_t strips,
                                 int64_t M, int64_t N, void* stream) {
  if (!float_dtype(dy_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported gradient dtype code %d", dy_dtype);
  if (M < 0 || N < 1) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld", (long long)M, (long long)N);
  const int64_t nb = (N + 127) / 128, strip = grad_strip(M, N);
  const int most = dy_dtype == MXQ_DTYPE_BF16 ? 1 : dy_dtype == MXQ_DTYPE_F16 ? 2 : 3;
  if (ldy < N || (q && (ldq < nb * 128 || ldq % 16 || lds < nb)) ||
      (n_parts != 0 && (n_parts != most || ldp < nb * 128 || ldp % 8)))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides or parts for N=%lld", (long long)N);
  if (M == 0) return MXQ_OK;
  if (!dy || (q && (!scale || !aligned16(q))) || (n_parts && (!parts || !aligned16(parts))))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  if (sums && strips != (M + strip - 1) / strip)
    return mxq_set_error(MXQ_ERR_INVALID, "room for %lld strips, %lld needed", (long long)strips,
                         (long long)((M + strip - 1) / strip));
  const dim3 grid((unsigned)((N + 511) / 512), (unsigned)((M + strip - 1) / strip));
  with_dtype(dy_dtype, [&](auto C) {
    constexpr int kCode = decltype(C)::value;
    constexpr int kMost = kCode == MXQ_DTYPE_BF16 ? 1 : kCode == MXQ_DTYPE_F16 ? 2 : 3;
    if (n_parts)
      hipLaunchKernelGGL((fp8_grad_pass_kernel<kCode, kMost>), grid, dim3(256), 0, (hipStream_t)stream, (const char*)dy, ldy,
                         q, ldq, scale, lds, (uint16_t*)parts, ldp, sums, M, N, nb, strip);
    else
      hipLaunchKernelGGL((fp8_grad_pass_kernel<kCode, 0>), grid, dim3(256), 0, (hipStream_t)stream, (const char*)dy, ldy, q,
                         ldq, scale, lds, (uint16_t*)nullptr, (int64_t)0, sums, M, N, nb, strip);
  });
  return mxq_check_launch("fp8_grad_pass_kernel");
}

extern "C" int mxq_pad_rows(const uint8_t* src, int64_t lds, int64_t width, uint8_t* dst, int64_t ldd, int64_t rows,
                            void* stream) {
  if (rows < 0 || width < 1 || lds < width || ldd < width || ldd % 16 || ldd >= (1ll << 31))
    return mxq_set_error(MXQ_ERR_INVALID, "bad rows of %lld bytes, strides %lld and %lld", (long long)width, (long long)lds,
                         (long long)ldd);
  if (rows == 0) return MXQ_OK;
  if (!src || !dst || !aligned16(dst)) return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  if (rows >= (1ll << 40)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "too many rows");
  const int64_t total = rows * (ldd / 16), blocks = (total + 255) / 256;
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, (hipStream_t)stream, src, lds,
                     (int)width, dst, (int)ldd, total);
  return mxq_check_launch("pad_rows_kernel");
}
