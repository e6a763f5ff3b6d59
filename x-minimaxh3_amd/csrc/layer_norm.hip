// Layer norm over rows and its gradients, statistics and sums in float32:
//
//   y = (x - mean) * rstd * w + b                       mean = E[x], rstd = 1 / sqrt(E[(x - mean)^2] + eps)
//   dx = rstd * (g - E[g] - xh * E[g * xh]),  g = dy * w, xh = (x - mean) * rstd
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// A row is held in registers by as many waves as it has chunks of 512 elements (up to sixteen), eight elements per lane and
// chunk, so x (and dy) are read once; the variance is that of the centred values, not a difference of large sums.
// HBM-bound: 75600 x 5120 bf16 forward 303 us (5.1 TB/s), backward from the input in 8 bits, with its join, 386 (5.0 TB/s). The
// backward pass also keeps its lanes' columns of dw and db in registers over all the rows a workgroup takes, writes them
// once per workgroup, and fp8_join_kernel adds the workgroups' sums in a fixed order: no atomics, the same bits on
// every run. Its x can be the input as it was kept in 8 bits (fp8_common.h), decoded as it is read.

#include "fp8_common.h"

namespace mxq {

constexpr int kCodeFp8 = MXQ_DTYPE_E4M3;

// Eight consecutive elements.
template <int kCode> struct Eight {
  static constexpr int kWords = kCode == MXQ_DTYPE_F32 ? 8 : kCode == kCodeFp8 ? 2 : 4;
  static constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : kCode == kCodeFp8 ? 1 : 2;
  uint32_t w[kWords];
};

// A lane's eight columns of a row of D: those from `col` on; the last lane with any of a row that is not whole eights takes
// the row's last eight and counts those from `lo` on; a lane behind the row takes the first eight and counts none; of a
// row below eight elements, lane 0 takes and counts them all. kVec: D % 8 == 0.
struct Window {
  int start, lo, hi;
};
template <bool kVec>
MXQ_DEVICE Window window(int col, int D) {
  if constexpr (kVec) return col < D ? Window{col, 0, 8} : Window{0, 8, 8};
  if (D < 8) return col == 0 ? Window{0, 0, D} : Window{0, 8, 8};
  const int n = D - col;
  return n >= 8 ? Window{col, 0, 8} : n > 0 ? Window{D - 8, 8 - n, 8} : Window{0, 8, 8};
}

// The window's elements, from any address (one access each: a branch per element, or per load, would end in a wait).
template <int kCode, bool kVec>
MXQ_DEVICE Eight<kCode> load8(const char* row, const Window& at, int D) {
  constexpr int kWords = Eight<kCode>::kWords;
  Eight<kCode> r;
  const char* p = row + (int64_t)at.start * Eight<kCode>::kElem;
  if (!kVec && D < 8) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < D) {
        if constexpr (kCode == MXQ_DTYPE_F32)
          r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        else if constexpr (kCode == kCodeFp8)
          r.w[i >> 2] |= (uint32_t)reinterpret_cast<const uint8_t*>(p)[i] << (8 * (i & 3));
        else
          r.w[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
      }
  } else if constexpr (kWords == 2) {
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
  return r;
}

// v with the elements that the window does not count at zero.
template <bool kVec>
MXQ_DEVICE void counted(const Window& at, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (kVec ? at.lo == 0 : (e >= at.lo && e < at.hi)) ? v[e] : 0.0f;
}

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

// Eight results at the window (two lanes of a row's end may store the same values twice).
template <int kCode, bool kVec>
MXQ_DEVICE void store8(char* row, const Window& at, int D, const float (&v)[8]) {
  if (at.lo >= 8) return;
  char* p = row + (int64_t)at.start * Eight<kCode>::kElem;
  if (!kVec && D < 8) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < D) store_out<kCode>(reinterpret_cast<typename OutT<kCode>::T*>(p) + i, v[i]);
  } else if constexpr (kCode == MXQ_DTYPE_F32) {
    *reinterpret_cast<v4f_any*>(p) = v4f{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<v4f_any*>(p + 16) = v4f{v[4], v[5], v[6], v[7]};
  } else {
    v4u o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = kCode == MXQ_DTYPE_F16 ? f32_to_f16_bits(v[2 * i]) | (f32_to_f16_bits(v[2 * i + 1]) << 16)
                                    : pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<v4u_any*>(p) = o;
  }
}

// The window's values of a weight or bias vector of a run-time type (`none` where there is none).
template <bool kVec>
MXQ_DEVICE void param8(const char* p, int code, const Window& at, int D, float none, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = none;
  } else if (code == MXQ_DTYPE_F32) {
    to_f32(load8<MXQ_DTYPE_F32, kVec>(p, at, D), 1.0f, v);
  } else if (code == MXQ_DTYPE_F16) {
    to_f32(load8<MXQ_DTYPE_F16, kVec>(p, at, D), 1.0f, v);
  } else {
    to_f32(load8<MXQ_DTYPE_BF16, kVec>(p, at, D), 1.0f, v);
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

struct Norm {
  const char *x, *w, *b;
  char* y;
  float *mean, *rstd;
  int64_t M, ldx;
  int D, wcode;
  float eps;
};

// kOne: a wave per row, four rows per workgroup; else a workgroup per row.
template <int kCode, int kChunks, bool kOne, bool kVec>
__global__ __launch_bounds__(kOne ? 256 : 1024) void layer_norm_kernel(Norm p) {
  constexpr int kElem = Eight<kCode>::kElem;
  __shared__ float red[2][2][16];
  const int waves = kOne ? 1 : blockDim.x >> 6, wave = kOne ? 0 : threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, row = kOne ? block * 4 + (threadIdx.x >> 6) : block;
  if (row >= p.M) return;  // (whole waves; with several per row, whole workgroups)
  const char* x = p.x + row * p.ldx * kElem;
  Eight<kCode> raw[kChunks];
  auto at = [&](int i) { return window<kVec>(((i * waves + wave) * 64 + lane) * 8, p.D); };
#pragma unroll
  for (int i = 0; i < kChunks; ++i) raw[i] = load8<kCode, kVec>(x, at(i), p.D);
  const float inv = 1.0f / (float)p.D;
  float s = 0.0f, none = 0.0f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float v[8];
    to_f32(raw[i], 1.0f, v);
    counted<kVec>(at(i), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[e];
  }
  row_sum<kOne>(s, none, red[0], wave, waves, lane);
  const float mean = s * inv;
  float s2 = 0.0f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float v[8];
    to_f32(raw[i], 1.0f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] -= mean;
    counted<kVec>(at(i), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s2 = fmaf(v[e], v[e], s2);
  }
  none = 0.0f;
  row_sum<kOne>(s2, none, red[1], wave, waves, lane);
  const float rstd = 1.0f / sqrtf(s2 * inv + p.eps);
  if (wave == 0 && lane == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
  char* y = p.y + row * p.D * kElem;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float v[8], w[8], b[8];
    to_f32(raw[i], 1.0f, v);
    param8<kVec>(p.w, p.wcode, at(i), p.D, 1.0f, w);
    param8<kVec>(p.b, p.wcode, at(i), p.D, 0.0f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaf((v[e] - mean) * rstd, w[e], b[e]);
    store8<kCode, kVec>(y, at(i), p.D, v);
  }
}

struct NormGrad {
  const char *dy, *x, *w;
  const uint8_t* xs;
  const float *mean, *rstd;
  char* dx;
  float* sums;  // [grid][2][D]: dw and db of the workgroup's rows
  int64_t M, ldy, ldx, ldxs;
  int D, wcode;
};

template <int kCode, int kX, int kChunks, int kThreads, bool kVec>
__global__ __launch_bounds__(kThreads) void layer_norm_grad_kernel(NormGrad p) {
  constexpr bool kOne = kThreads == 256;  // a wave per row, four rows per workgroup; else a workgroup per row
  constexpr int kElem = Eight<kCode>::kElem, kElemX = Eight<kX>::kElem, kRows = kOne ? 4 : 1;
  constexpr bool kAhead = kChunks == 1;  // (more chunks leave no registers for a second row at 1024 threads)
  __shared__ float red[2][2][16];
  const int waves = kOne ? 1 : blockDim.x >> 6, wave = kOne ? 0 : threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int sub = kOne ? threadIdx.x >> 6 : 0;
  const float inv = 1.0f / (float)p.D;
  // (three chunks' weights beside their sums spill: 2000 x 20480 bf16 148 us; read again for every row 115, what still spills
  // bounds it; six chunks of half as many waves 134)
  constexpr bool kHoldW = kChunks < 3;
  float dw[kChunks][8] = {}, db[kChunks][8] = {}, held[kHoldW ? kChunks : 1][8];
  auto at = [&](int i) { return window<kVec>(((i * waves + wave) * 64 + lane) * 8, p.D); };
  if constexpr (kHoldW) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) param8<kVec>(p.w, p.wcode, at(i), p.D, 1.0f, held[i]);
  }
  auto weight = [&](int i, float (&v)[8]) {
    if constexpr (kHoldW) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = held[i][e];
    } else {
      uint64_t from = (uint64_t)p.w;
      __asm__ volatile("" : "+s"(from));  // (or the compiler reads them ahead of the rows and holds them after all)
      param8<kVec>((const char*)from, p.wcode, at(i), p.D, 1.0f, v);
    }
  };
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + sub;
  // The next row is requested ahead of the present one's arithmetic (kAhead); what a lane keeps of a row is its raw words, from
  // which g and xh are formed again behind the row's sums (kept as float32 they took 60 registers more, a wave per SIMD).
  Eight<kCode> ry[kChunks];
  Eight<kX> rx[kChunks];
  uint32_t rs[kChunks];
  float mean = 0.0f, rstd = 0.0f;
  auto load = [&](int64_t k) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      ry[i] = load8<kCode, kVec>(p.dy + k * p.ldy * kElem, at(i), p.D);
      rx[i] = load8<kX, kVec>(p.x + k * p.ldx * kElemX, at(i), p.D);
      if constexpr (kX == kCodeFp8) {
        const uint8_t* xs = p.xs + k * p.ldxs;
        const Window c = at(i);
        // (a window that was moved to the row's end may reach back into the block before)
        rs[i] = xs[c.start >> 7] | (kVec || p.D < 8 ? 0u : (uint32_t)xs[(c.start + 7) >> 7] << 8);
      }
    }
    mean = p.mean[k];
    rstd = p.rstd[k];
  };
  auto x_values = [&](const Eight<kX>& t, uint32_t scales, int i, float (&v)[8]) {
    to_f32(t, fp8_scale_f32(scales & 0xFFu), v);
    if constexpr (kX == kCodeFp8 && !kVec) {
      if (p.D >= 8) {
        float u[8];
        to_f32(t, fp8_scale_f32(scales >> 8), u);
        const int c = at(i).start & 127;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < 128 ? v[e] : u[e];
      }
    }
  };
  if (kAhead && row < p.M) load(row);
  for (int turn = 0; row < p.M; row += step, turn ^= 1) {
    Eight<kCode> ty[kChunks];
    Eight<kX> tx[kChunks];
    uint32_t ts[kChunks];
    if constexpr (!kAhead) load(row);
    const float m = mean, r = rstd;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      ty[i] = ry[i];
      tx[i] = rx[i];
      ts[i] = rs[i];
    }
    if (kAhead && row + step < p.M) load(row + step);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float y[8], x[8], w[8];
      weight(i, w);
      to_f32(ty[i], 1.0f, y);
      counted<kVec>(at(i), y);  // (y = 0 adds nothing to any sum)
      x_values(tx[i], ts[i], i, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = (x[e] - m) * r, g = y[e] * w[e];
        s1 += g;
        s2 = fmaf(g, xh, s2);
        dw[i][e] = fmaf(y[e], xh, dw[i][e]);
        db[i][e] += y[e];
      }
    }
    row_sum<kOne>(s1, s2, red[turn], wave, waves, lane);
    const float rc1 = r * (s1 * inv), a = r * r * (s2 * inv);  // dx = r g - r c1 - (x - m) r^2 c2
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float v[8], x[8], w[8];
      weight(i, w);
      // (formed again from the words: the statement keeps the compiler from holding the first pass's values instead)
#pragma unroll
      for (int k = 0; k < Eight<kCode>::kWords; ++k) __asm__ volatile("" : "+v"(ty[i].w[k]));
#pragma unroll
      for (int k = 0; k < Eight<kX>::kWords; ++k) __asm__ volatile("" : "+v"(tx[i].w[k]));
      to_f32(ty[i], 1.0f, v);
      x_values(tx[i], ts[i], i, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e] * w[e], r, fmaf(x[e] - m, -a, -rc1));
      store8<kCode, kVec>(p.dx + row * p.D * kElem, at(i), p.D, v);
    }
  }
  if (!p.sums) return;
  float* out = p.sums + (int64_t)blockIdx.x * 2 * p.D;
  if constexpr (kOne) {  // the workgroup's four waves hold the same columns: their sums in order
    __shared__ float part[4][64 * 8];
    const Window c = at(0);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) part[sub][e * 64 + lane] = k ? db[0][e] : dw[0][e];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = sub * 2 + e;
        if (j >= c.lo && j < c.hi)
          out[k * p.D + c.start + j] =
              ((part[0][j * 64 + lane] + part[1][j * 64 + lane]) + part[2][j * 64 + lane]) + part[3][j * 64 + lane];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const Window c = at(i);
      if (c.lo == 0 && c.hi == 8) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float* o = out + k * p.D + c.start;
          const float(&v)[8] = k ? db[i] : dw[i];
          *reinterpret_cast<v4f_any*>(o) = v4f{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<v4f_any*>(o + 4) = v4f{v[4], v[5], v[6], v[7]};
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e >= c.lo && e < c.hi) {
            out[c.start + e] = dw[i][e];
            out[p.D + c.start + e] = db[i][e];
          }
      }
    }
  }
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

// The forward pass holds a row from its loads to its stores, so rows under way per CU count: few waves of many chunks
// (75600 x 5120: two waves of five chunks 297 us, four of three 326, five of two 380, ten of one 458). Other widths, 200 M
// bf16 elements, by one to six chunks: 1024 columns 156 130; 2048 147 132 132 136; 4096 151 133 133 136 135 138; 8192 161
// 134 135 137 137 137; 12288 - 138 136 139 152 140; 16384 - 143 153 140 162 159; 24576 - - 143 144 171 144. Few rows (256)
// take the same 8 us in every form.
template <class F>
static void with_forward_shape(int D, F&& f) {
  using std::integral_constant;
  const int n = (D + 511) / 512;
  auto go = [&](auto N) { f(N, std::false_type{}, (n + decltype(N)::value - 1) / decltype(N)::value * 64); };
  if (n <= 1) f(integral_constant<int, 1>{}, std::true_type{}, 256);
  else if (n <= 4) go(integral_constant<int, 2>{});
  else if (n <= 8) go(integral_constant<int, 4>{});
  else if (n <= 10) go(integral_constant<int, 5>{});
  else if (n <= 24) go(integral_constant<int, 6>{});
  else go(integral_constant<int, 4>{});
}

// Workgroups of the backward pass: about twenty waves per CU (sixteen of the wide forms), each with an equal share of rows; eight rows
// at least once every CU has a workgroup, since each writes 2 D sums (4000 x 2048 bf16, kernel and join: 12.7 + 6.1 us; at
// least four rows 13.4 + 8.2, sixteen 15.1 + 4.3; 777 x 1003 fp32: 256 workgroups 7.1 + 3.4, one per row 7.7 + 6.6).
static int64_t norm_grad_grid(int64_t M, int64_t D, int cus) {
  const int64_t n = (D + 511) / 512, units = n <= 1 ? (M + 3) / 4 : M;
  const int64_t most = cus * (n <= 1 ? 5 : n <= 16 ? (20 / n > 1 ? 20 / n : 1) : 1);
  const int64_t few = units < cus ? units : units / 8 > cus ? units / 8 : cus;
  return few < most ? few : most;
}

}  // namespace mxq

using namespace mxq;

// Workgroups across: a launch takes less than 2^32 threads along an axis.
constexpr int64_t kNormGridX = 1 << 20;

static int check_norm(int64_t M, int64_t D, int dtype, int wcode) {
  if (!float_dtype(dtype) || !float_dtype(wcode)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported dtype codes %d, %d", dtype, wcode);
  if (M < 0 || D < 1 || M >= (1ll << 31)) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld D=%lld", (long long)M, (long long)D);
  if (D > kNormMaxD) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "rows of more than %d elements", kNormMaxD);
  return MXQ_OK;
}

extern "C" int mxq_layer_norm(const void* x, int dtype, int64_t ldx, const void* w, const void* b, int param_dtype, float eps,
                              void* y, float* mean, float* rstd, int64_t M, int64_t D, void* stream) {
  if (const int rc = check_norm(M, D, dtype, param_dtype)) return rc;
  if (ldx < D) return mxq_set_error(MXQ_ERR_INVALID, "row stride %lld below %lld columns", (long long)ldx, (long long)D);
  if (!(eps >= 0.0f)) return mxq_set_error(MXQ_ERR_INVALID, "eps %g", (double)eps);
  if (M == 0) return MXQ_OK;
  if (!x || !y) return mxq_set_error(MXQ_ERR_INVALID, "null pointer");
  const Norm p = {(const char*)x, (const char*)w, (const char*)b, (char*)y, mean, rstd, M, ldx, (int)D, param_dtype, eps};
  with_forward_shape((int)D, [&](auto N, auto One, int threads) {
    with_dtype(dtype, [&](auto C) {
      constexpr bool kOne = decltype(One)::value;
      const int64_t blocks = kOne ? (M + 3) / 4 : M;
      const unsigned wide = (unsigned)(blocks < kNormGridX ? blocks : kNormGridX);
      with_bool(D % 8 == 0, [&](auto V) {
        hipLaunchKernelGGL((layer_norm_kernel<decltype(C)::value, decltype(N)::value, kOne, decltype(V)::value>),
                           dim3(wide, (unsigned)((blocks + wide - 1) / wide)), dim3(threads), 0, (hipStream_t)stream, p);
      });
    });
  });
  return mxq_check_launch("layer_norm_kernel");
}

extern "C" int mxq_layer_norm_backward_workspace(int64_t M, int64_t D, int64_t* bytes) {
  if (M < 0 || D < 1 || D > kNormMaxD || !bytes)
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld D=%lld", (long long)M, (long long)D);
  *bytes = norm_grad_grid(M, D, mxq_cu_count()) * 2 * D * 4;
  return MXQ_OK;
}

extern "C" int mxq_layer_norm_backward(const void* dy, int dtype, int64_t ldy, const void* x, int x_dtype, int64_t ldx,
                                       const uint8_t* x_scale, int64_t ldxs, const float* mean, const float* rstd,
                                       const void* w, int param_dtype, void* dx, float* dparams, int64_t M, int64_t D,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check_norm(M, D, dtype, param_dtype)) return rc;
  const bool kept = x_dtype == MXQ_DTYPE_E4M3;
  if (!kept && x_dtype != dtype) return mxq_set_error(MXQ_ERR_INVALID, "x of dtype code %d for gradients of %d", x_dtype, dtype);
  if (ldy < D || ldx < D || (kept && ldxs < (D + 127) / 128))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides for %lld columns", (long long)D);
  if (M == 0) return dparams ? mxq_column_join(nullptr, 0, 2 * D, dparams, MXQ_DTYPE_F32, stream) : MXQ_OK;
  if (!dy || !x || !mean || !rstd || !dx || (kept && !x_scale)) return mxq_set_error(MXQ_ERR_INVALID, "null pointer");
  const int64_t grid = norm_grad_grid(M, D, mxq_cu_count()), need = grid * 2 * D * 4;
  if (dparams && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  float* sums = dparams ? (float*)workspace : nullptr;
  const NormGrad p = {(const char*)dy, (const char*)x, (const char*)w, x_scale, mean, rstd, (char*)dx, sums, M, ldy, ldx, ldxs,
                      (int)D, param_dtype};
  with_shape((int)D, [&](auto N, auto T, int threads) {
    with_dtype(dtype, [&](auto C) {
      constexpr int kCode = decltype(C)::value, kChunks = decltype(N)::value, kThreads = decltype(T)::value;
      with_bool(D % 8 == 0, [&](auto V) {
        with_bool(kept, [&](auto K) {
          constexpr int kX = decltype(K)::value ? kCodeFp8 : kCode;
          hipLaunchKernelGGL((layer_norm_grad_kernel<kCode, kX, kChunks, kThreads, decltype(V)::value>), dim3((unsigned)grid),
                             dim3(threads), 0, (hipStream_t)stream, p);
        });
      });
    });
  });
  if (const int rc = mxq_check_launch("layer_norm_grad_kernel")) return rc;
  return dparams ? mxq_column_join(sums, grid, 2 * D, dparams, MXQ_DTYPE_F32, stream) : MXQ_OK;
}
