// What the norms of rows share: eight consecutive elements of a row as words and as float32, sums over a row's waves, and the
// number of waves and chunks of 512 elements that hold a row.
#pragma once

#include "fp8_common.h"

namespace mxq {

constexpr int kCodeFp8 = MXQ_DTYPE_E4M3;

// Eight consecutive elements.
template <int kCode> struct Eight {
  static constexpr int kWords = kCode == MXQ_DTYPE_F32 ? 8 : kCode == kCodeFp8 ? 2 : 4;
  static constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : kCode == kCodeFp8 ? 1 : 2;
  uint32_t w[kWords];
};

template <int kCode>
MXQ_DEVICE void to_f32(const Eight<kCode>& r, float scale, float (&v)[8]) {
  if constexpr (kCode == MXQ_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
  } else if constexpr (kCode == kCodeFp8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v4f q = fp8x4_to_f32(r.w[h], scale);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = q[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = kCode == MXQ_DTYPE_F16 ? f16_to_f32(r.w[i] & 0xFFFFu) : bf16_lo(r.w[i]);
      v[2 * i + 1] = kCode == MXQ_DTYPE_F16 ? f16_to_f32(r.w[i] >> 16) : bf16_hi(r.w[i]);
    }
  }
}

MXQ_DEVICE float lane_value(float v, int lane) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
// v + v[i ^ 8], then ^ 4, 2, 1: the sum of sixteen lanes.
MXQ_DEVICE float sum16(float v) {
  v += __uint_as_float(dpp_lane<kDppRowRor8>(__float_as_uint(v)));
  v += __uint_as_float(lane_xor4(__float_as_uint(v)));
  v += __uint_as_float(dpp_lane<kDppQuadXor2>(__float_as_uint(v)));
  return v + __uint_as_float(dpp_lane<kDppQuadXor1>(__float_as_uint(v)));
}

// Sums over the row's waves of two values at once: one exchange puts a's halves added up in lanes 0-31 and b's in lanes
// 32-63, so the rest of the tree serves both. kOne: the row is one wave's. `red`: 2 x 16 floats of the row's workgroup,
// others for every other call.
template <bool kOne>
MXQ_DEVICE void row_sum(float& a, float& b, float (&red)[2][16], int wave, int waves, int lane) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  float v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = sum16(__uint_as_float(q[0]) + __uint_as_float(q[1]));
  if constexpr (!kOne) {
    if ((lane & 31) == 0) red[lane >> 5][wave] = v;
    __syncthreads();
    v = red[lane >> 5][lane & 15];
    v = sum16((lane & 15) < waves ? v : 0.0f);  // (lanes 16-31 the same as 0-15)
  }
  a = lane_value(v, 0);
  b = lane_value(v, 32);
}

// p, the power of two in r, and q = r^2 / p, for the backward passes' term x r^2 c = (x p) (q c): r^2 by itself leaves float32's
// range for rows whose magnitude is beyond 2^63 or below 2^-64, where dx does not (a row of 10^24: r^2 = 0, and the whole term
// was lost). Scaling by powers of two is exact, so rows whose r^2 is in range have the bits of r g - x (r r c). kUniform: into
// scalar registers (r is the workgroup's one row's).
struct RowFactors {
  float p, q;
};
template <bool kUniform>
MXQ_DEVICE RowFactors row_factors(float r) {
  const int e = __builtin_amdgcn_frexp_expf(r);  // (0 for infinities and NaN, which q keeps)
  const float p = __builtin_ldexpf(0.5f, e), q = r * __builtin_ldexpf(r, 1 - e);
  if constexpr (kUniform) return {lane_value(p, 0), lane_value(q, 0)};
  return {p, q};
}

// Chunks per lane and waves per row of the backward pass: up to 512 elements one wave, up to 8192 a chunk per lane of as
// many waves as it takes (hidden 5120: ten waves, every lane at work), beyond that two and three chunks of up to sixteen.
template <class F>
static void with_bool(bool v, F&& f) {
  if (v)
    f(std::true_type{});
  else
    f(std::false_type{});
}

constexpr int kNormMaxD = 24576;
template <class F>
static void with_shape(int D, F&& f) {
  using std::integral_constant;
  const int n = (D + 511) / 512;
  if (n <= 1) f(integral_constant<int, 1>{}, integral_constant<int, 256>{}, 256);
  else if (n <= 16) f(integral_constant<int, 1>{}, integral_constant<int, 1024>{}, n * 64);
  else if (n <= 32) f(integral_constant<int, 2>{}, integral_constant<int, 1024>{}, (n + 1) / 2 * 64);
  else f(integral_constant<int, 3>{}, integral_constant<int, 1024>{}, (n + 2) / 3 * 64);
}

}  // namespace mxq
