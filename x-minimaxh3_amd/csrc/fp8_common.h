// 8-bit floating point in blocks of 128: the number format that the fp8 kernels share.
//
// A block (1 x 128 of an activation or a gradient, 128 x 128 of a weight) holds e4m3 codes q and one E8M0 byte b:
// the values are q * 2^(b - 127). The exponent e = b - 127 is the smallest one with absmax <= 448 * 2^e (448 is
// e4m3's largest value), so x / 2^e is exact in float32 and the only rounding of the quantizer is the one to e4m3
// (to nearest, ties to even). A power of two is what the matrix instructions of gfx950 apply by themselves, and a
// value q * 2^e is exact in bfloat16 and float32: e is at least -117, so that the smallest one, 2^-9 * 2^e, is not
// subnormal there. A block of zeros has b = 127. NaN and infinities become e4m3's NaN code in their own place, and
// absmax is that of the finite elements.
#pragma once

#include "mxq_common.h"

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v2s __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

// 16 and 8 bytes from any address: one access, gfx950 splits it where it crosses a boundary. Rows of odd widths are read and
// written through these: element by element they cost an access and a wait for each.
typedef unsigned int v4u_any __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned int v2u_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(1)));

namespace mxq {

// The few-row product (gemm_fp8.hip): rows that it takes as codes, and those it quantizes itself; whether it is the form to
// take; and the product (M within those bounds, arguments as mxq_fp8_gemm's, x of x_dtype where it is not MXQ_DTYPE_E4M3).
constexpr int64_t kFp8FewRows = 32, kFp8FusedRows = 16;
bool fp8_rows_pays(int64_t M, int64_t N, int64_t K);
int fp8_linear_rows(const void* x, int x_dtype, int64_t ldx, const uint8_t* sx, int64_t ldsx, const uint8_t* b, int64_t ldb,
                    const uint8_t* sb, int64_t ldsb, const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N,
                    int64_t K, void* stream);

// Sums to be joined (fp8_join.hip): d [rows, cols] (row stride ldd, of dtype `code`) = slices [splits, rows, ldp] + bias, and
// out [n] = the columns of in [parts, n]. No slices, no out: nothing to do.
struct SliceJob {
  const float* part;
  const void* bias;
  void* d;
  int64_t rows, ldp, ldd;
  int cols, splits, code;
};
struct ColumnJob {
  const float* in;
  void* out;
  int64_t parts, n;
  int code;
};
int fp8_join(const SliceJob& a, const SliceJob& b, const ColumnJob& c, void* stream);

// Microseconds that `s` slices of `n` sums cost a product: the join's launch, and the sums written and read, less where the
// eight L2s (32 MB) hold them: 3 slices of 100 x 21504 (26 MB) took 3.8 beside the launch, 2 of 1024 x 4096 (34 MB) 13.6.
inline double slices_cost(int64_t s, int64_t n) {
  return s > 1 ? 4.0 + (double)n * (double)(s + 1) / (s * n * 4 <= 28000000 ? 2.3e6 : 0.95e6) : 0.0;
}

// mxq_fp8_gemm and mxq_fp8_wgrad, with the join of their slices, if there is one, left to the caller (`later` not NULL).
int fp8_gemm(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t ldsa, const uint8_t* b, int64_t ldb, const uint8_t* sb,
             int64_t ldsb, const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
             int64_t workspace_bytes, SliceJob* later, void* stream);
int fp8_wgrad(const void* dy, int parts, int64_t ldy, const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, void* dw,
              int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, SliceJob* later,
              void* stream);

// Their refusals other than the workspace's, for passes that launch other steps ahead of them.
int fp8_gemm_check(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t ldsa, const uint8_t* b, int64_t ldb, const uint8_t* sb,
                   int64_t ldsb, const void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K);
int fp8_wgrad_check(const void* dy, int parts, int64_t ldy, const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds,
                    const void* dw, int out_dtype, int64_t M, int64_t N, int64_t K);

constexpr int kFp8MinByte = 10;  // 2^-117

// The scale byte of a block from the bits of its (finite) absmax: 448 = 1.75 * 2^8, so a significand above 1.75
// takes the next exponent.
MXQ_DEVICE uint32_t fp8_scale_byte(uint32_t amax_bits) {
  const int b = (int)((amax_bits + 0x1FFFFFu) >> 23) - 8;
  return amax_bits == 0 ? 127u : (uint32_t)max(b, kFp8MinByte);
}

MXQ_DEVICE float fp8_scale_f32(uint32_t byte) { return __uint_as_float(byte << 23); }

// ---- 16 consecutive elements of one row, as loaded: 8 words of 16-bit types, 16 of float32 ----
template <int kCode> struct Piece {
  static constexpr int kWords = kCode == MXQ_DTYPE_F32 ? 16 : 8;
  static constexpr int kBytes = kWords * 4;
  uint32_t w[kWords];
};

template <int kCode>
MXQ_DEVICE Piece<kCode> piece_load_vec(const void* p) {
  Piece<kCode> r;
#pragma unroll
  for (int i = 0; i < Piece<kCode>::kWords / 4; ++i) {
    const v4u v = *reinterpret_cast<const v4u_any*>(reinterpret_cast<const char*>(p) + 16 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
  }
  return r;
}

// The first `n` elements (1 to 15), zeros behind them: each load made, of the last element where there is none.
template <int kCode>
MXQ_DEVICE Piece<kCode> piece_load_some(const void* p, int n) {
  Piece<kCode> r;
  if constexpr (kCode == MXQ_DTYPE_F32) {
    const uint32_t* s = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 16; ++i) r.w[i] = s[min(i, n - 1)];
#pragma unroll
    for (int i = 0; i < 16; ++i) r.w[i] = i < n ? r.w[i] : 0u;
  } else {
    const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
    uint32_t h[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) h[i] = s[min(i, n - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = (2 * i < n ? h[2 * i] : 0u) | ((2 * i + 1 < n ? h[2 * i + 1] : 0u) << 16);
  }
  return r;
}

// `n` of 16 elements from p (n <= 0: zeros, nothing is read).
template <int kCode>
MXQ_DEVICE Piece<kCode> piece_load(const void* p, int n) {
  if (n >= 16) return piece_load_vec<kCode>(p);
  if (n > 0) return piece_load_some<kCode>(p, n);
  return Piece<kCode>{};
}

template <int kCode>
MXQ_DEVICE float piece_at(const Piece<kCode>& r, int i) {  // i is a constant once unrolled
  if constexpr (kCode == MXQ_DTYPE_F32) return __uint_as_float(r.w[i]);
  const uint32_t h = (i & 1) ? r.w[i >> 1] >> 16 : r.w[i >> 1] & 0xFFFFu;
  return kCode == MXQ_DTYPE_F16 ? f16_to_f32(h) : bf16_to_f32(h);
}

// Bits of the float32 absmax of 16 elements, NaN and infinities above every finite value.
template <int kCode>
MXQ_DEVICE uint32_t piece_absmax(const Piece<kCode>& r) {
  if constexpr (kCode == MXQ_DTYPE_F32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, r.w[i] & 0x7FFFFFFFu);
    return m;
  } else {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = absmax_acc_bf16x2(a, r.w[i]);  // (16-bit magnitudes order as integers in both types)
    const uint32_t h = max(a & 0xFFFFu, a >> 16);
    return kCode == MXQ_DTYPE_F16 ? __float_as_uint(f16_to_f32(h)) & 0x7FFFFFFFu : h << 16;
  }
}

// The same over the finite elements only.
template <int kCode>
MXQ_DEVICE uint32_t piece_absmax_finite(const Piece<kCode>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t b = abs_bits(piece_at(r, i));
    m = max(m, b < 0x7F800000u ? b : 0u);
  }
  return m;
}

// 16 elements divided by `scale` (a power of two) and rounded once to e4m3: v_cvt_scalef32_pk_fp8_* divides by the
// scale's power of two, rounds to nearest even and gives the NaN code beyond 448, which only NaN and infinities are.
template <int kCode>
MXQ_DEVICE v4u piece_encode(const Piece<kCode>& r, float scale) {
  v4u o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v2s h = {0, 0};
    if constexpr (kCode == MXQ_DTYPE_F32) {
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, __uint_as_float(r.w[4 * j]), __uint_as_float(r.w[4 * j + 1]), scale,
                                                   false);
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, __uint_as_float(r.w[4 * j + 2]), __uint_as_float(r.w[4 * j + 3]),
                                                   scale, true);
    } else if constexpr (kCode == MXQ_DTYPE_F16) {
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(h, __builtin_bit_cast(v2h, r.w[2 * j]), scale, false);
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(h, __builtin_bit_cast(v2h, r.w[2 * j + 1]), scale, true);
    } else {
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(v2bf, r.w[2 * j]), scale, false);
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(v2bf, r.w[2 * j + 1]), scale, true);
    }
    o[j] = __builtin_bit_cast(uint32_t, h);
  }
  return o;
}

// Four codes times a power of two as two bfloat16 pairs (exact).
MXQ_DEVICE v2u fp8x4_to_bf16(uint32_t q, float scale) {
  v2u o;
  o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, scale, false));
  o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, scale, true));
  return o;
}
MXQ_DEVICE v8bf fp8x8_to_bf16(uint32_t q0, uint32_t q1, float scale) {
  const v2u a = fp8x4_to_bf16(q0, scale), b = fp8x4_to_bf16(q1, scale);
  return __builtin_bit_cast(v8bf, v4u{a[0], a[1], b[0], b[1]});
}
// ... and as four float32 (exact).
MXQ_DEVICE v4f fp8x4_to_f32(uint32_t q, float scale) {
  const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q, scale, false);
  const v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q, scale, true);
  return v4f{a[0], a[1], b[0], b[1]};
}

// max over lanes i, i ^ 1, 2, 4 (eight lanes hold a row's block, 16 elements each)
MXQ_DEVICE uint32_t max8(uint32_t v) {
  v = max(v, dpp_lane<kDppQuadXor1>(v));
  v = max(v, dpp_lane<kDppQuadXor2>(v));
  return max(v, lane_xor4(v));
}

// The scale byte of a block held by eight lanes.
template <int kCode>
MXQ_DEVICE uint32_t block_scale_byte(const Piece<kCode>& p) {
  uint32_t m = max8(piece_absmax(p));
  if (m >= 0x7F800000u) m = max8(piece_absmax_finite(p));  // (the same for the eight lanes of a block)
  return fp8_scale_byte(m);
}

// Bias of the four columns from col on (behind the last: the last one's).
template <int kOut>
MXQ_DEVICE v4f bias_run(const void* bias, int col, int N) {
  v4f b = {0.0f, 0.0f, 0.0f, 0.0f};
  if (!bias) return b;
  const typename OutT<kOut>::T* p = reinterpret_cast<const typename OutT<kOut>::T*>(bias);
  if (col + 4 > N) {
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = OutT<kOut>::load(p + min(col + e, N - 1));
  } else if constexpr (kOut == MXQ_DTYPE_F32) {
    b = *reinterpret_cast<const v4f_any*>(p + col);
  } else {
    const v2u w = *reinterpret_cast<const v2u_any*>(p + col);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
      b[e] = kOut == MXQ_DTYPE_F16 ? f16_to_f32(h) : bf16_to_f32(h);
    }
  }
  return b;
}

// Orders a wave's LDS accesses: what its lanes wrote, its lanes read.
MXQ_DEVICE void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The sum of `n` vectors, `stride` apart, eight in flight at a time and added in pairs.
MXQ_DEVICE v4f sum_slices(const v4f* p, int n, int64_t stride) {
  v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < n; s += 8) {
    v4f t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = s + i < n ? p[(s + i) * stride] : v4f{0.0f, 0.0f, 0.0f, 0.0f};
    y += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
  }
  return y;
}

// Stores 4 float values from column `col` on, as kCode; `n` of them are inside the row.
template <int kCode>
MXQ_DEVICE void store_run4(void* row, int64_t col, int n, const float* y) {
  if constexpr (kCode == MXQ_DTYPE_F32) {
    float* p = reinterpret_cast<float*>(row) + col;
    if (n >= 4) {
      *reinterpret_cast<v4f_any*>(p) = v4f{y[0], y[1], y[2], y[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) p[e] = y[e];
    }
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(row) + col;
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = kCode == MXQ_DTYPE_F16 ? f32_to_f16_bits(y[e]) : f32_to_bf16_bits(y[e]);
    if (n >= 4) {
      *reinterpret_cast<v2u_any*>(p) = v2u{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) p[e] = (uint16_t)h[e];
    }
  }
}

inline int dtype_bytes(int code) { return code == MXQ_DTYPE_F32 ? 4 : 2; }
inline bool float_dtype(int code) { return code == MXQ_DTYPE_F32 || code == MXQ_DTYPE_F16 || code == MXQ_DTYPE_BF16; }

// f.operator()<code>() for the run-time dtype code.
template <class F>
inline auto with_dtype(int code, F&& f) {
  if (code == MXQ_DTYPE_F32) return f(std::integral_constant<int, MXQ_DTYPE_F32>{});
  if (code == MXQ_DTYPE_F16) return f(std::integral_constant<int, MXQ_DTYPE_F16>{});
  return f(std::integral_constant<int, MXQ_DTYPE_BF16>{});
}

}  // namespace mxq
