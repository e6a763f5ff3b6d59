// 4-bit floating point in blocks of 32 (MXFP4): the number format that the mxfp4 kernels share.
//
// A block (1 x 32 of an activation's or a weight's row) holds e2m1 codes and one E8M0 byte b: the values are
// code * 2^(b - 127), codes being 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives (bit 3), two in a byte, the even column's
// in the low four bits. The exponent e = b - 127 is the smallest one >= -125 with absmax <= 6 * 2^e, so no value is cut
// off, x / 2^e is exact in float32 and the only rounding is the one to e2m1 (to nearest, ties to the even code); the
// smallest value, 2^-1 * 2^-125, is not subnormal in bfloat16 and float32, where every value is exact. A block of zeros has
// b = 127. e2m1 has no NaN: a block with a NaN or an infinity has b = 255, which makes all its values NaN (its codes are 0).
//
// The matrix products read scales from tiles: the bytes of 32 rows x 16 blocks (512 columns) are 512 consecutive bytes, in
// the order in which the lanes of a wave take them (fp4_scale_at); tiles of one row of tiles follow each other.
#pragma once

#include "fp8_common.h"

namespace mxq {

constexpr int kFp4MinByte = 2;  // 2^-125
constexpr int64_t kFp4Stage = 128;        // bytes of codes (256 columns) that an activation's rows are padded to; a weight's to two
constexpr int64_t kFp4ScaleTile = 512;    // bytes of a scale tile: 32 rows x 16 blocks
__host__ MXQ_DEVICE int64_t fp4_groups(int64_t K) { return (K + 511) / 512; }  // scale tiles along K
inline int64_t fp4_row_bytes(int64_t K) { return (K + 255) / 256 * kFp4Stage; }
inline int64_t fp4_weight_bytes(int64_t K) { return (K + 511) / 512 * 2 * kFp4Stage; }
inline int64_t fp4_scale_bytes(int64_t rows, int64_t K) { return (rows + 31) / 32 * fp4_groups(K) * kFp4ScaleTile; }

// The place of a row's block in its tile (both counted within the tile). A stage of the product is 256 columns, half h of
// a wave's lanes takes its blocks 4 h .. 4 h + 3, and a lane's eight bytes are those of two stages.
__host__ MXQ_DEVICE int fp4_scale_at(int row, int block) {
  return ((block >> 2) & 1) * 256 + row * 8 + ((block >> 3) & 1) * 4 + (block & 3);
}

// The scale byte of a block from the bits of its absmax: 6 = 1.5 * 2^2, so a significand above 1.5 takes the next exponent.
MXQ_DEVICE uint32_t fp4_scale_byte(uint32_t amax_bits) {
  const int b = (int)((amax_bits + 0x3FFFFFu) >> 23) - 2;
  return amax_bits == 0 ? 127u : amax_bits >= 0x7F800000u ? 255u : (uint32_t)max(b, kFp4MinByte);
}

// v_cvt_scalef32_pk_fp4_* divides by the scale's power of two and rounds to nearest even; byte kByte of `old` is replaced.
template <int kByte>
MXQ_DEVICE uint32_t fp4_pair(uint32_t old, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, scale, kByte);
}

// 16 elements divided by `scale` and rounded once to e2m1.
template <int kCode>
MXQ_DEVICE v2u fp4_encode(const Piece<kCode>& r, float scale) {
  uint32_t o[2] = {0, 0};
  static_for<8>([&](auto I) {
    constexpr int i = decltype(I)::value, kByte = i & 3;
    uint32_t& w = o[i >> 2];
    if constexpr (kCode == MXQ_DTYPE_F32)
      w = fp4_pair<kByte>(w, __uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]), scale);
    else if constexpr (kCode == MXQ_DTYPE_F16)
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2h, r.w[i]), scale, kByte);
    else
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2bf, r.w[i]), scale, kByte);
  });
  return v2u{o[0], o[1]};
}

// Eight codes (a word) times a power of two as eight bfloat16 (exact).
MXQ_DEVICE v8bf fp4x8_to_bf16(uint32_t q, float scale) {
  const v4u o = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3))};
  return __builtin_bit_cast(v8bf, o);
}

// mxq_mxfp4_gemm's and the input gradient's refusals other than the workspace's, for passes that launch other steps ahead of
// them; the gradient leaves the join of its slices, if there are any, to the caller.
int fp4_gemm_check(const uint8_t* a, int64_t lda, const uint8_t* sa, const uint8_t* b, int64_t ldb, const uint8_t* sb, const void* d,
                   int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K);
int fp4_dgrad_check(const void* dy, int64_t ldy, const uint8_t* b, int64_t ldb, const uint8_t* sb, const void* dx, int out_dtype,
                    int64_t M, int64_t N, int64_t K);
int64_t fp4_dgrad_workspace(int64_t M, int64_t N, int64_t K, int parts);
int fp4_dgrad(const void* dy, int parts, int64_t ldy, const uint8_t* b, int64_t ldb, const uint8_t* sb, void* dx, int out_dtype,
              int64_t M, int64_t N, int64_t K, void* workspace, SliceJob* later, void* stream);

// The few-row product (mxfp4_rows.hip): up to kFp4FusedRows rows of x_dtype, which it quantizes itself, or of codes
// (MXQ_DTYPE_E2M1) with scales sx, of any strides and alignment.
constexpr int64_t kFp4FusedRows = 16;
// Where a layer's call takes it. Every workgroup brings all of x, M K elements, while the weight, N K, streams; tiles of 128 rows
// cost a launch, a join and idle rows instead, about the same for one row and sixteen. Measured, few-row kernel / tiles in us, x
// in bf16: K 5120, N 5120, 16 rows 11.4 / 12.4; K 20480, N 5120, 6 rows 20.0 / 22.8, 8 22.6 / 22.9, 16 28.6 / 23.1; K 14336, N 5376,
// 8 rows 17.8 / 18.5, 16 23.1 / 18.7; K 20480, N 20480, 16 rows 54.2 / 56.9; K 40960, N 1024, 2 rows 17.7 / 15.7, 16 42.7 / 16.5.
// Pairs, which need no quantizing: K 20480, N 5120, 12 rows 20.8 / 23.4, 16 22.9 / 23.3; K 40960, N 1024, 16 rows 29.2 / 16.8.
inline bool fp4_few_rows(int64_t M, int64_t N, int64_t K, bool pair) {
  return M <= kFp4FusedRows && M * K <= (pair ? 2 : 1) * (90000 + 12 * N);
}
int fp4_linear_rows(const void* x, int x_dtype, int64_t ldx, const uint8_t* sx, int64_t ldsx, const uint8_t* b, int64_t ldb,
                    const uint8_t* sb, const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K,
                    void* stream);

// What the passes choose on the current device: weight rows and waves of the few-row kernel's workgroups; rows and columns of a
// product's or a gradient's tile and the slices of the summed index.
struct Fp4RowsForm {
  int rows, waves;
};
struct Fp4TileForm {
  int rows, cols, slices;
};
Fp4RowsForm fp4_rows_form(int64_t M, int64_t N, int64_t K);
Fp4TileForm fp4_gemm_form(int64_t M, int64_t N, int64_t K);
Fp4TileForm fp4_dgrad_form(int64_t M, int64_t N, int64_t K, int parts);

// Two codes (byte kByte of a word) as float32 (exact).
template <int kByte>
MXQ_DEVICE v2f fp4x2_to_f32(uint32_t q, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, kByte);
}

}  // namespace mxq
