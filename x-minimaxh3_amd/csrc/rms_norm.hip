// Root-mean-square norm of rows behind a residual addition, and its gradients:
//
//   s = x + r, rounded to the rows' type (s = x without a residual)
//   y = (s * rstd) * w                                  rstd = 1 / sqrt(E[s^2] + eps)
//   dx = rstd * (g - xh * E[g * xh]) + ds,  g = dy * w, xh = s * rstd        dw = sum over rows of dy * xh
//
// y leaves in the rows' type, or quantized as the 8-bit layer (fp8_common.h, 1 x 128) or the 4-bit layer (mxfp4_common.h,
// 1 x 32) reads it, straight from the registers that hold the row. eps is a float32; E[s^2] is summed in float64 and rstd rounded
// once from there, then s * rstd and the product with w are one float32 rounding each: with eps rounded to float32 first, y is
// the same to the last bit in an implementation of the formula in float64 (but for an rstd closer to a border of float32 than float64's
// own rounding), and so are the codes made of it, where a last bit decides at the border of two.
//
// A row is held in registers by one or more waves, eight elements per lane and chunk of 512, so x and r are read once. The
// backward pass also keeps its lanes' columns of dw in registers over all the rows a workgroup takes, and fp8_join_kernel
// adds the workgroups' sums in a fixed order: no atomics, the same bits on every run.
//
// Both passes are bound by HBM. Forward with a residual and 4-bit codes, 75600 x 5376 bf16: 478 us, 5.6 TB/s. Backward, 75600 x 5120
// bf16, of an input kept in 8 bits and with a gradient added: 509 us, 5.3 TB/s. (One chunk a lane keeps the row's values behind its
// sum; forming them anew from the words, as two and three do to save registers, took 165 us for 126 at 19531 x 5120, and a second
// row requested ahead another 16.)

#include "mxfp4_common.h"
#include "norm_common.h"

namespace mxq {

constexpr int kOutSame = 0, kOutFp8 = 1, kOutFp4 = 2;

// Eight elements moved down by s (0 to 7) of them, zeros behind.
template <int kCode>
MXQ_DEVICE void shift_down(Eight<kCode>& r, int s) {
  constexpr int kWords = Eight<kCode>::kWords, kBits = 32 * kWords / 8;  // bits of an element
#pragma unroll
  for (int b = 4; b >= 1; b /= 2) {
    const bool on = s & b;
    const int words = b * kBits / 32, bits = b * kBits % 32;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t lo = i + words < kWords ? r.w[i + words] : 0u, hi = i + words + 1 < kWords ? r.w[i + words + 1] : 0u;
      const uint32_t v = bits ? __builtin_amdgcn_alignbit(hi, lo, bits) : lo;
      r.w[i] = on ? v : r.w[i];
    }
  }
}

// A lane's eight columns from `col` on of a row of D, `n` = D - col of them inside it (none: zeros). kVec: n is 8 or more, or none.
// Else every lane makes the same one access, the row's last eight elements where fewer are left, moved into place (a branch
// for the lane with some of them made a wave wait once per operand, and its seven loads spilled: 20000 x 5001 bf16 backward
// 284 us, 178 now). A row below eight elements goes element by element.
template <int kCode, bool kVec>
MXQ_DEVICE Eight<kCode> load_run8(const char* row, int col, int n) {
  constexpr int kWords = Eight<kCode>::kWords, kElem = Eight<kCode>::kElem;
  Eight<kCode> r = {};
  const int D = col + n;
  if (!kVec && D < 8) {
    for (int e = col == 0 ? D - 1 : -1; e >= 0; --e) {
#pragma unroll
      for (int i = kWords - 1; i >= 0; --i) {
        const uint32_t below = i ? r.w[i - 1] : 0u;
        r.w[i] = kElem == 4 ? below : (r.w[i] << (8 * (kElem & 3))) | (below >> (32 - 8 * (kElem & 3)));
      }
      if constexpr (kElem == 4) r.w[0] = reinterpret_cast<const uint32_t*>(row)[e];
      else if constexpr (kElem == 1) r.w[0] |= reinterpret_cast<const uint8_t*>(row)[e];
      else r.w[0] |= reinterpret_cast<const uint16_t*>(row)[e];
    }
    return r;
  }
  if (kVec && n <= 0) return r;
  const int start = kVec ? col : n > 0 ? min(col, D - 8) : 0;
  const char* p = row + (int64_t)start * kElem;
  if constexpr (kWords == 2) {
    const v2u v = *reinterpret_cast<const v2u_any*>(p);
    r.w[0] = v[0];
    r.w[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const v4u v = *reinterpret_cast<const v4u_any*>(p + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
    }
  }
  if constexpr (!kVec) {
    shift_down(r, n > 0 ? col - start : 0);
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.w[i] = n > 0 ? r.w[i] : 0u;
  }
  return r;
}

template <int kCode>
MXQ_DEVICE Eight<kCode> from_f32(const float (&v)[8]) {
  Eight<kCode> r;
  if constexpr (kCode == MXQ_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.w[i] = kCode == MXQ_DTYPE_F16 ? f32_to_f16_bits(v[2 * i]) | (f32_to_f16_bits(v[2 * i + 1]) << 16)
                                      : pack_bf16x2(v[2 * i], v[2 * i + 1]);
  }
  return r;
}

template <int kCode, bool kVec>
MXQ_DEVICE void store_run8(char* row, int col, int n, const Eight<kCode>& r) {
  constexpr int kElem = Eight<kCode>::kElem;
  char* p = row + (int64_t)col * kElem;
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < Eight<kCode>::kWords / 4; ++i)
      *reinterpret_cast<v4u_any*>(p + 16 * i) = v4u{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]};
  } else if (!kVec && n > 0) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) {
        if constexpr (kElem == 4) reinterpret_cast<uint32_t*>(p)[i] = r.w[i];
        else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(r.w[i >> 1] >> (16 * (i & 1)));
      }
  }
}

// The run's values of a weight vector of a run-time type (1 where there is none).
template <bool kVec>
MXQ_DEVICE void weight8(const char* p, int code, int col, int n, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 1.0f;
  } else if (code == MXQ_DTYPE_F32) {
    to_f32(load_run8<MXQ_DTYPE_F32, kVec>(p, col, n), 1.0f, v);
  } else if (code == MXQ_DTYPE_F16) {
    to_f32(load_run8<MXQ_DTYPE_F16, kVec>(p, col, n), 1.0f, v);
  } else {
    to_f32(load_run8<MXQ_DTYPE_BF16, kVec>(p, col, n), 1.0f, v);
  }
}

// 1 / sqrt(a) for a >= 0, rounded once: the hardware's estimate (about 2^-24) and two steps of Newton's method.
MXQ_DEVICE float rsqrt_once(double a) {
  double y = __builtin_amdgcn_rsq(a);
  if (a > 0.0 && a < __builtin_inf()) {
#pragma unroll
    for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-a * y, y, 1.0), y);
  }
  return (float)y;
}

struct Rms {
  const char *x, *r, *w;
  char *sum, *y;  // y: the rows' type [M, D], or codes
  uint8_t* scale;
  float* rstd;
  int64_t M, ldx, ldr, ldq, lds;
  int D, wcode;
  double inv, eps;  // 1 / D
};

// Eight values of a row as codes; `m`, the lanes' absmax bits. All lanes of a wave take part.
MXQ_DEVICE uint32_t absmax8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, abs_bits(v[e]));
  return m;
}
MXQ_DEVICE void store_fp8(const Rms& p, int64_t row, int col, int lane, const float (&v)[8]) {
  uint32_t m = row16_max_u32(absmax8(v));  // (sixteen lanes hold a block)
  if (m >= 0x7F800000u) {
    m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, abs_bits(v[e]) < 0x7F800000u ? abs_bits(v[e]) : 0u);
    m = row16_max_u32(m);
  }
  const uint32_t byte = fp8_scale_byte(m);
  const float scale = fp8_scale_f32(byte);
  v2u o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v2s c = {0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[4 * h], v[4 * h + 1], scale, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[4 * h + 2], v[4 * h + 3], scale, true);
    o[h] = __builtin_bit_cast(uint32_t, c);
  }
  if (col < (p.D + 127) / 128 * 128) {
    *reinterpret_cast<v2u*>(p.y + row * p.ldq + col) = o;
    if ((lane & 15) == 0) p.scale[row * p.lds + (col >> 7)] = (uint8_t)byte;
  }
}
MXQ_DEVICE void store_fp4(const Rms& p, int64_t row, int col, int lane, const float (&v)[8]) {
  uint32_t m = absmax8(v);  // (four lanes hold a block)
  m = max(m, dpp_lane<kDppQuadXor1>(m));
  m = max(m, dpp_lane<kDppQuadXor2>(m));
  const uint32_t byte = fp4_scale_byte(m);
  const float scale = fp8_scale_f32(byte);
  uint32_t o = 0;
  o = fp4_pair<0>(o, v[0], v[1], scale);
  o = fp4_pair<1>(o, v[2], v[3], scale);
  o = fp4_pair<2>(o, v[4], v[5], scale);
  o = fp4_pair<3>(o, v[6], v[7], scale);
  if (byte == 255u) o = 0;
  uint32_t word = byte << (8 * ((lane >> 2) & 3));
  word |= lane_xor4(word);
  word |= dpp_lane<kDppRowRor8>(word);
  if (col < (p.D + 127) / 128 * 128) {
    *reinterpret_cast<uint32_t*>(p.y + row * p.ldq + col / 2) = o;
    if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(p.scale + row * p.lds + (col >> 7) * 4) = word;
  }
}

// The sum of a row's lanes, where they are part of one wave: 16, 32 or 64 of them.
template <int kLanes>
MXQ_DEVICE double lanes_sum_f64(double v) {
  if constexpr (kLanes == 64) return wave_sum_f64(v);
  v = row16_sum_f64(v);
  if constexpr (kLanes == 32) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    v = __builtin_bit_cast(double, (uint64_t)lo[0] | ((uint64_t)hi[0] << 32)) +
        __builtin_bit_cast(double, (uint64_t)lo[1] | ((uint64_t)hi[1] << 32));
  }
  return v;
}
template <int kLanes>
MXQ_DEVICE float lanes_sum(float v) {
  v = sum16(v);
  if constexpr (kLanes == 32) {
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(q[0]) + __uint_as_float(q[1]);
  }
  return v;
}

// kLanes: what holds a row, 16, 32 or 64 lanes of a workgroup of 256 threads (781250 x 128 bf16, a head's columns: 71 us, 5.6
// TB/s; 199 us with a wave per row), or 0, a workgroup.
template <int kCode, int kOut, int kChunks, int kLanes, bool kVec>
__global__ __launch_bounds__(kLanes ? 256 : 1024) void rms_norm_kernel(Rms p) {
  constexpr bool kOne = kLanes != 0;
  constexpr int kGroup = kOne ? kLanes : 64, kRows = 256 / kGroup;
  constexpr int kElem = Eight<kCode>::kElem;
  __shared__ double red[16];
  const int waves = kOne ? 1 : blockDim.x >> 6, wave = kOne ? 0 : threadIdx.x >> 6, lane = threadIdx.x & (kGroup - 1);
  const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, row = kOne ? block * kRows + threadIdx.x / kGroup : block;
  if (row >= p.M) return;  // (all lanes of a row, which alone exchange values)
  auto col = [&](int i) { return ((i * waves + wave) * 64 + lane) * 8; };
  const char* x = p.x + row * p.ldx * kElem;
  Eight<kCode> s[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) s[i] = load_run8<kCode, kVec>(x, col(i), p.D - col(i));
  if (p.r) {
    const char* r = p.r + row * p.ldr * kElem;
    Eight<kCode> t[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) t[i] = load_run8<kCode, kVec>(r, col(i), p.D - col(i));
    char* sum = p.sum + row * p.D * kElem;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float a[8], b[8];
      to_f32(s[i], 1.0f, a);
      to_f32(t[i], 1.0f, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] += b[e];
      s[i] = from_f32<kCode>(a);
      store_run8<kCode, kVec>(sum, col(i), p.D - col(i), s[i]);
    }
  }
  double q = 0.0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float v[8];
    to_f32(s[i], 1.0f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) q = fma((double)v[e], (double)v[e], q);
  }
  q = lanes_sum_f64<kGroup>(q);
  if constexpr (!kOne) {
    if (lane == 0) red[wave] = q;
    __syncthreads();
    q = 0.0;
    for (int w = 0; w < waves; ++w) q += red[w];
  }
  const float rstd = rsqrt_once(fma(q, p.inv, p.eps));
  if (p.rstd && wave == 0 && lane == 0) p.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float v[8], w[8];
    to_f32(s[i], 1.0f, v);
    weight8<kVec>(p.w, p.wcode, col(i), p.D - col(i), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * rstd * w[e];
    if constexpr (kOut == kOutSame)
      store_run8<kCode, kVec>(p.y + row * p.D * kElem, col(i), p.D - col(i), from_f32<kCode>(v));
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = col(i) + e < p.D ? v[e] : 0.0f;  // (0 * infinity behind the row's end)
      if constexpr (kOut == kOutFp8)
        store_fp8(p, row, col(i), lane, v);
      else
        store_fp4(p, row, col(i), lane, v);
    }
  }
}

struct RmsGrad {
  const char *dy, *x, *w, *ds;
  const uint8_t* xs;
  const float* rstd;
  char* dx;
  float* sums;  // [grid][D]: dw of the workgroup's rows
  int64_t M, ldy, ldx, ldxs, ldds;
  int D, wcode;
};

// kLanes: as the forward pass.
template <int kCode, int kX, int kChunks, int kLanes, bool kVec>
__global__ __launch_bounds__(kLanes ? 256 : 1024) void rms_norm_grad_kernel(RmsGrad p) {
  constexpr bool kOne = kLanes != 0;
  constexpr int kGroup = kOne ? kLanes : 64;
  constexpr int kElem = Eight<kCode>::kElem, kElemX = Eight<kX>::kElem, kRows = kOne ? 256 / kGroup : 1;
  __shared__ float red[2][2][16];
  const int waves = kOne ? 1 : blockDim.x >> 6, wave = kOne ? 0 : threadIdx.x >> 6, lane = threadIdx.x & (kGroup - 1);
  const int sub = kOne ? threadIdx.x / kGroup : 0;
  const float inv = 1.0f / (float)p.D;
  // Three chunks leave no registers for a row: it is read again behind its sum, from L2 (4882 x 20480 bf16: 155 us, 221 spilled).
  constexpr bool kTwice = kChunks > 2;
  float dw[kChunks][8] = {};
  auto col = [&](int i) {
    int c = ((i * waves + wave) * 64 + lane) * 8;
    if constexpr (kChunks > 1) __asm__ volatile("" : "+v"(c));  // (else every operand's address is held through the loop)
    return c;
  };
  const int64_t step = (int64_t)gridDim.x * kRows;
  // What a lane keeps of a row is its raw words, from which the values are formed again behind the row's sum.
  Eight<kCode> ty[kChunks], td[kChunks] = {};
  Eight<kX> tx[kChunks];
  uint32_t ts[kChunks];
  auto load = [&](int64_t row, int i, bool ds) {
    const int c = col(i), n = p.D - c;
    ty[i] = load_run8<kCode, kVec>(p.dy + row * p.ldy * kElem, c, n);
    tx[i] = load_run8<kX, kVec>(p.x + row * p.ldx * kElemX, c, n);
    ts[i] = kX == kCodeFp8 ? (uint32_t)p.xs[row * p.ldxs + (n > 0 ? c >> 7 : 0)] : 0u;
    if (ds) td[i] = load_run8<kCode, kVec>(p.ds + row * p.ldds * kElem, c, n);
  };
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + sub; row < p.M; row += step, turn ^= 1) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      if constexpr (!kTwice) load(row, i, p.ds);
    const float r = p.rstd[row];
    float s1 = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if constexpr (kChunks > 1) __builtin_amdgcn_sched_barrier(0);  // one chunk's values at a time
      if constexpr (kTwice) load(row, i, false);
      float y[8], x[8], w[8];
      uint64_t from = (uint64_t)p.w;
      if constexpr (kChunks > 1) __asm__ volatile("" : "+s"(from));
      weight8<kVec>((const char*)from, p.wcode, col(i), p.D - col(i), w);
      to_f32(ty[i], 1.0f, y);
      to_f32(tx[i], fp8_scale_f32(ts[i]), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = x[e] * r;
        s1 = fmaf(y[e] * w[e], xh, s1);
        dw[i][e] = fmaf(y[e], xh, dw[i][e]);
      }
    }
    if constexpr (kGroup < 64)
      s1 = lanes_sum<kGroup>(s1);
    else
      row_sum<kOne>(s1, none, red[turn], wave, waves, lane);
    const RowFactors f = row_factors<!kOne>(r);  // (here: ahead of the sum, the row's loads would be waited for)
    float a = f.q * (s1 * inv);
    int64_t again = row;
    if constexpr (kTwice) __asm__ volatile("" : "+s"(again));
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if constexpr (kChunks > 1) __builtin_amdgcn_sched_barrier(0);
      if constexpr (kTwice) load(again, i, p.ds);
      float v[8], x[8], w[8], d[8] = {};
      // (formed again from the words: the statements keep the compiler from holding the first pass's values instead)
      if constexpr (kChunks > 1) {
#pragma unroll
        for (int k = 0; k < Eight<kCode>::kWords; ++k) __asm__ volatile("" : "+v"(ty[i].w[k]));
#pragma unroll
        for (int k = 0; k < Eight<kX>::kWords; ++k) __asm__ volatile("" : "+v"(tx[i].w[k]));
      }
      uint64_t from = (uint64_t)p.w;
      if constexpr (kChunks > 1) __asm__ volatile("" : "+s"(from));
      weight8<kVec>((const char*)from, p.wcode, col(i), p.D - col(i), w);
      to_f32(ty[i], 1.0f, v);
      to_f32(tx[i], fp8_scale_f32(ts[i]), x);
      if (p.ds) to_f32(td[i], 1.0f, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e] * w[e], r, -(x[e] * f.p * a)) + d[e];
      store_run8<kCode, kVec>(p.dx + row * p.D * kElem, col(i), p.D - col(i), from_f32<kCode>(v));
    }
  }
  if (!p.sums) return;
  float* out = p.sums + (int64_t)blockIdx.x * p.D;
  if constexpr (kOne) {  // the workgroup's rows hold the same columns: their sums in order
    __shared__ float part[kRows][kGroup * 8];
#pragma unroll
    for (int e = 0; e < 8; ++e) part[sub][e * kGroup + lane] = dw[0][e];
    __syncthreads();
    for (int c = threadIdx.x; c < p.D; c += 256) {
      float v = 0.0f;
#pragma unroll
      for (int g = 0; g < kRows; ++g) v += part[g][c % 8 * kGroup + c / 8];
      out[c] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int n = p.D - col(i);
      float* o = out + col(i);
      if (n >= 8) {
        *reinterpret_cast<v4f_any*>(o) = v4f{dw[i][0], dw[i][1], dw[i][2], dw[i][3]};
        *reinterpret_cast<v4f_any*>(o + 4) = v4f{dw[i][4], dw[i][5], dw[i][6], dw[i][7]};
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < n) o[e] = dw[i][e];
      }
    }
  }
}

// Lanes of a row of at most 512 elements.
static int64_t row_lanes(int64_t D) { return D <= 128 ? 16 : D <= 256 ? 32 : 64; }
template <class F>
static void with_lanes(int D, F&& f) {
  using std::integral_constant;
  if (D <= 128) f(integral_constant<int, 16>{});
  else if (D <= 256) f(integral_constant<int, 32>{});
  else f(integral_constant<int, 64>{});
}
// Chunks, lanes (0: a workgroup) and threads of the forward pass.
template <class F>
static void with_rms_shape(int D, F&& f) {
  using std::integral_constant;
  const int n = (D + 511) / 512;
  auto go = [&](auto N) { f(N, integral_constant<int, 0>{}, (n + decltype(N)::value - 1) / decltype(N)::value * 64); };
  if (n <= 1) with_lanes(D, [&](auto L) { f(integral_constant<int, 1>{}, L, 256); });
  else if (n <= 4) go(integral_constant<int, 2>{});
  else if (n <= 12) go(integral_constant<int, 4>{});
  else go(integral_constant<int, 6>{});
}
// And of the backward pass.
template <class F>
static void with_grad_shape(int D, F&& f) {
  with_shape(D, [&](auto N, auto T, int threads) {
    if constexpr (decltype(T)::value == 256) with_lanes(D, [&](auto L) { f(N, L, threads); });
    else f(N, std::integral_constant<int, 0>{}, threads);
  });
}

// Workgroups of the backward pass: about twenty waves per CU, each with an equal share of rows, eight rows at least once every
// CU has a workgroup, since each writes D sums. (Two workgroups of eleven or twelve waves: 18600 x 5376 bf16 in 128 us, 154 with
// one. Four of six instead of three: 33333 x 3000 180 instead of 142.)
static int64_t rms_grad_grid(int64_t M, int64_t D, int cus) {
  const int64_t n = (D + 511) / 512, rows = n <= 1 ? 256 / row_lanes(D) : 1, units = (M + rows - 1) / rows;
  const int64_t most = cus * (n <= 1 ? 5 : n <= 10 ? 20 / n : n <= 12 ? 2 : 1);
  const int64_t few = units < cus ? units : units / 8 > cus ? units / 8 : cus;
  return few < most ? few : most;
}

}  // namespace mxq

using namespace mxq;

// Workgroups across: a launch takes less than 2^32 threads along an axis.
constexpr int64_t kRmsGridX = 1 << 20;

static int check_rms(int64_t M, int64_t D, int dtype, int wcode) {
  if (!float_dtype(dtype) || !float_dtype(wcode)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported dtype codes %d, %d", dtype, wcode);
  if (M < 0 || D < 1 || M >= (1ll << 31)) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld D=%lld", (long long)M, (long long)D);
  if (D > kNormMaxD) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "rows of more than %d elements", kNormMaxD);
  return MXQ_OK;
}

extern "C" int mxq_rms_norm(const void* x, const void* r, int dtype, int64_t ldx, int64_t ldr, const void* w, int param_dtype, float eps,
                            void* sum, void* y, int y_dtype, int64_t ldq, uint8_t* scale, int64_t lds, float* rstd, int64_t M,
                            int64_t D, void* stream) {
  if (const int rc = check_rms(M, D, dtype, param_dtype)) return rc;
  if (ldx < D || (r && ldr < D)) return mxq_set_error(MXQ_ERR_INVALID, "row strides %lld, %lld below %lld columns", (long long)ldx, (long long)ldr, (long long)D);
  if (!(eps >= 0.0f)) return mxq_set_error(MXQ_ERR_INVALID, "eps %g", (double)eps);
  const bool fp8 = y_dtype == MXQ_DTYPE_E4M3, fp4 = y_dtype == MXQ_DTYPE_E2M1;
  if (!fp8 && !fp4 && y_dtype != dtype) return mxq_set_error(MXQ_ERR_INVALID, "output dtype code %d for rows of %d", y_dtype, dtype);
  const int64_t kb = (D + 127) / 128;
  if ((fp8 && (ldq < kb * 128 || ldq % 8 || lds < kb)) || (fp4 && (ldq < kb * 64 || ldq % 4 || lds < kb * 4 || lds % 4)))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldq=%lld lds=%lld for D=%lld", (long long)ldq, (long long)lds, (long long)D);
  if (M == 0) return MXQ_OK;
  if (!x || !y || (r && !sum) || ((fp8 || fp4) && !scale) || (fp8 && reinterpret_cast<uintptr_t>(y) % 8) ||
      (fp4 && (reinterpret_cast<uintptr_t>(y) % 4 || reinterpret_cast<uintptr_t>(scale) % 4)))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  const Rms p = {(const char*)x, (const char*)r, (const char*)w, (char*)sum, (char*)y, scale, rstd, M, ldx, ldr, ldq, lds, (int)D,
                 param_dtype, 1.0 / (double)D, (double)eps};
  with_rms_shape((int)D, [&](auto N, auto L, int threads) {
    constexpr int kChunks = decltype(N)::value, kLanes = decltype(L)::value, kRows = kLanes ? 256 / kLanes : 1;
    const int64_t blocks = (M + kRows - 1) / kRows;
    const unsigned wide = (unsigned)(blocks < kRmsGridX ? blocks : kRmsGridX);
    const dim3 grid(wide, (unsigned)((blocks + wide - 1) / wide));
    with_dtype(dtype, [&](auto C) {
      constexpr int kCode = decltype(C)::value;
      with_bool(D % 8 == 0, [&](auto V) {
        constexpr bool kVec = decltype(V)::value;
        if (fp8)
          hipLaunchKernelGGL((rms_norm_kernel<kCode, kOutFp8, kChunks, kLanes, kVec>), grid, dim3(threads), 0, (hipStream_t)stream, p);
        else if (fp4)
          hipLaunchKernelGGL((rms_norm_kernel<kCode, kOutFp4, kChunks, kLanes, kVec>), grid, dim3(threads), 0, (hipStream_t)stream, p);
        else
          hipLaunchKernelGGL((rms_norm_kernel<kCode, kOutSame, kChunks, kLanes, kVec>), grid, dim3(threads), 0, (hipStream_t)stream, p);
      });
    });
  });
  return mxq_check_launch("rms_norm_kernel");
}

extern "C" int mxq_rms_norm_backward_workspace(int64_t M, int64_t D, int64_t* bytes) {
  if (M < 0 || D < 1 || D > kNormMaxD || !bytes)
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld D=%lld", (long long)M, (long long)D);
  *bytes = rms_grad_grid(M, D, mxq_cu_count()) * D * 4;
  return MXQ_OK;
}

extern "C" int mxq_rms_norm_backward(const void* dy, int dtype, int64_t ldy, const void* x, int x_dtype, int64_t ldx,
                                     const uint8_t* x_scale, int64_t ldxs, const float* rstd, const void* w, int param_dtype,
                                     const void* dsum, int64_t ldds, void* dx, float* dweight, int64_t M, int64_t D, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  if (const int rc = check_rms(M, D, dtype, param_dtype)) return rc;
  const bool kept = x_dtype == MXQ_DTYPE_E4M3;
  if (!kept && x_dtype != dtype) return mxq_set_error(MXQ_ERR_INVALID, "x of dtype code %d for gradients of %d", x_dtype, dtype);
  if (ldy < D || ldx < D || (dsum && ldds < D) || (kept && ldxs < (D + 127) / 128))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides for %lld columns", (long long)D);
  if (M == 0) return dweight ? mxq_column_join(nullptr, 0, D, dweight, MXQ_DTYPE_F32, stream) : MXQ_OK;
  if (!dy || !x || !rstd || !dx || (kept && !x_scale)) return mxq_set_error(MXQ_ERR_INVALID, "null pointer");
  const int64_t grid = rms_grad_grid(M, D, mxq_cu_count()), need = grid * D * 4;
  if (dweight && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  float* sums = dweight ? (float*)workspace : nullptr;
  const RmsGrad p = {(const char*)dy, (const char*)x, (const char*)w, (const char*)dsum, x_scale, rstd, (char*)dx, sums, M, ldy, ldx, ldxs,
                     ldds, (int)D, param_dtype};
  with_grad_shape((int)D, [&](auto N, auto L, int threads) {
    with_dtype(dtype, [&](auto C) {
      constexpr int kCode = decltype(C)::value, kChunks = decltype(N)::value, kLanes = decltype(L)::value;
      with_bool(D % 8 == 0, [&](auto V) {
        with_bool(kept, [&](auto K) {
          constexpr int kX = decltype(K)::value ? kCodeFp8 : kCode;
          hipLaunchKernelGGL((rms_norm_grad_kernel<kCode, kX, kChunks, kLanes, decltype(V)::value>), dim3((unsigned)grid),
                             dim3(threads), 0, (hipStream_t)stream, p);
        });
      });
    });
  });
  if (const int rc = mxq_check_launch("rms_norm_grad_kernel")) return rc;
  return dweight ? mxq_column_join(sums, grid, D, dweight, MXQ_DTYPE_F32, stream) : MXQ_OK;
}
