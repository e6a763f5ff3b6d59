// Layer norm over rows and its gradients, statistics and sums in float32:
//
//   y = (x - mean) * rstd * w + b                       mean = E[x], rstd = 1 / sqrt(E[(x - mean)^2] + eps)
//   dx = rstd * (g - E[g] - xh * E[g * xh]),  g = dy * w, xh = (x - mean) * rstd
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// A row is held in registers by kWaves waves, chunks of eight elements per lane, so x (and dy) are read once; the
// variance is that of the centred values, not a difference of large sums. HBM-bound. The backward pass also keeps its
// lanes' columns of dw and db in registers over all the rows a workgroup takes, writes them once per workgroup, and
// column_join_kernel adds the workgroups' sums in a fixed order: no atomics, the same bits on every run. Its x can be
// the input as it was kept in 8 bits (fp8_common.h), decoded as it is read.

#include "fp8_common.h"

namespace mxq {

constexpr int kCodeFp8 = MXQ_DTYPE_E4M3;

// Eight consecutive elements.
template <int kCode> struct Eight {
  static constexpr int kWords = kCode == MXQ_DTYPE_F32 ? 8 : kCode == kCodeFp8 ? 2 : 4;
  static constexpr int kElem = kCode == MXQ_DTYPE_F32 ? 4 : kCode == kCodeFp8 ? 1 : 2;
  uint32_t w[kWords];
};

// `n` of eight elements (n <= 0: none, zeros) from p; `vec`: p is aligned to the eight.
template <int kCode>
MXQ_DEVICE Eight<kCode> load8(const char* p, int n, bool vec) {
  Eight<kCode> r;
  constexpr int kWords = Eight<kCode>::kWords;
#pragma unroll
  for (int i = 0; i < kWords; ++i) r.w[i] = 0;
  if (vec && n >= 8) {
    if constexpr (kWords == 2) {
      const v2u v = *reinterpret_cast<const v2u*>(p);
      r.w[0] = v[0];
      r.w[1] = v[1];
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const v4u v = reinterpret_cast<const v4u*>(p)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
      }
    }
  } else if (n > 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) {
        if constexpr (kCode == MXQ_DTYPE_F32)
          r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        else if constexpr (kCode == kCodeFp8)
          r.w[i >> 2] |= (uint32_t)reinterpret_cast<const uint8_t*>(p)[i] << (8 * (i & 3));
        else
          r.w[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
      }
  }
  return r;
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

template <int kCode>
MXQ_DEVICE void store8(char* p, int n, bool vec, const float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (kCode == MXQ_DTYPE_F32) {
      reinterpret_cast<v4f*>(p)[0] = v4f{v[0], v[1], v[2], v[3]};
      reinterpret_cast<v4f*>(p)[1] = v4f{v[4], v[5], v[6], v[7]};
    } else {
      v4u o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = kCode == MXQ_DTYPE_F16 ? f32_to_f16_bits(v[2 * i]) | (f32_to_f16_bits(v[2 * i + 1]) << 16)
                                      : pack_bf16x2(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<v4u*>(p) = o;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) store_out<kCode>(reinterpret_cast<typename OutT<kCode>::T*>(p) + i, v[i]);
  }
}

// Eight values of a weight or bias vector of a run-time type (`none` where there is none).
MXQ_DEVICE void param8(const char* p, int code, int col, int n, bool vec, float none, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = none;
  } else if (code == MXQ_DTYPE_F32) {
    to_f32(load8<MXQ_DTYPE_F32>(p + (int64_t)col * 4, n, vec), 1.0f, v);
  } else if (code == MXQ_DTYPE_F16) {
    to_f32(load8<MXQ_DTYPE_F16>(p + (int64_t)col * 2, n, vec), 1.0f, v);
  } else {
    to_f32(load8<MXQ_DTYPE_BF16>(p + (int64_t)col * 2, n, vec), 1.0f, v);
  }
}

// Sums over the row's waves of one or two values; every lane gets them. `red`: a slot of kWaves x 2 floats of the row,
// another one for every other call.
template <int kWaves>
MXQ_DEVICE void row_sum(float& a, float& b, float* red, int wave, int lane) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (kWaves > 1) {
    if (lane == 0) {
      red[2 * wave] = a;
      red[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      a += red[2 * i];
      b += red[2 * i + 1];
    }
  }
}

struct Norm {
  const char *x, *w, *b;
  char* y;
  float *mean, *rstd;
  int64_t M, ldx;
  int D, wcode, vec, pvec;
  float eps;
};

template <int kWaves> struct NormBlock {
  static constexpr int kThreads = kWaves == 1 ? 256 : kWaves * 64;
  static constexpr int kRows = kWaves == 1 ? 4 : 1;  // rows a workgroup holds at once
};

template <int kCode, int kChunks, int kWaves>
__global__ __launch_bounds__(NormBlock<kWaves>::kThreads) void layer_norm_kernel(Norm p) {
  constexpr int kElem = Eight<kCode>::kElem;
  __shared__ float red[2][2 * kWaves];
  const int wave = kWaves == 1 ? 0 : threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = kWaves == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= p.M) return;  // (whole waves; with several per row, whole workgroups)
  const char* x = p.x + row * p.ldx * kElem;
  Eight<kCode> raw[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = ((i * kWaves + wave) * 64 + lane) * 8;
    raw[i] = load8<kCode>(x + (int64_t)(col < p.D ? col : 0) * kElem, p.D - col, p.vec);
  }
  const float inv = 1.0f / (float)p.D;
  float s = 0.0f, none = 0.0f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float v[8];
    to_f32(raw[i], 1.0f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[e];
  }
  row_sum<kWaves>(s, none, red[0], wave, lane);
  const float mean = s * inv;
  float s2 = 0.0f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int n = p.D - ((i * kWaves + wave) * 64 + lane) * 8;
    float v[8];
    to_f32(raw[i], 1.0f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = e < n ? v[e] - mean : 0.0f;
      s2 += d * d;
    }
  }
  none = 0.0f;
  row_sum<kWaves>(s2, none, red[1], wave, lane);
  const float rstd = 1.0f / sqrtf(s2 * inv + p.eps);
  if (wave == 0 && lane == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
  char* y = p.y + row * p.D * kElem;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int col = ((i * kWaves + wave) * 64 + lane) * 8, n = p.D - col;
    if (n <= 0) continue;
    float v[8], w[8], b[8];
    to_f32(raw[i], 1.0f, v);
    param8(p.w, p.wcode, col, n, p.pvec, 1.0f, w);
    param8(p.b, p.wcode, col, n, p.pvec, 0.0f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (v[e] - mean) * rstd * w[e] + b[e];
    store8<kCode>(y + (int64_t)col * kElem, n, p.vec, v);
  }
}

struct NormGrad {
  const char *dy, *x, *w;
  const uint8_t* xs;
  const float *mean, *rstd;
  char* dx;
  float* sums;  // [grid][2][D]: dw and db of the workgroup's rows
  int64_t M, ldy, ldx, ldxs;
  int D, wcode, vec_y, vec_x, pvec;
};

template <int kCode, int kX, int kChunks, int kWaves>
__global__ __launch_bounds__(NormBlock<kWaves>::kThreads) void layer_norm_grad_kernel(NormGrad p) {
  constexpr int kElem = Eight<kCode>::kElem, kElemX = Eight<kX>::kElem, kRows = NormBlock<kWaves>::kRows;
  __shared__ float red[2][2 * kWaves];
  const int wave = kWaves == 1 ? 0 : threadIdx.x >> 6, lane = threadIdx.x & 63, sub = kWaves == 1 ? threadIdx.x >> 6 : 0;
  const float inv = 1.0f / (float)p.D;
  float dw[kChunks][8] = {}, db[kChunks][8] = {};
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + sub; row < p.M; row += (int64_t)gridDim.x * kRows) {
    Eight<kCode> ry[kChunks];
    Eight<kX> rx[kChunks];
    float sc[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = ((i * kWaves + wave) * 64 + lane) * 8, n = p.D - col, at = n > 0 ? col : 0;
      ry[i] = load8<kCode>(p.dy + (row * p.ldy + at) * kElem, n, p.vec_y);
      rx[i] = load8<kX>(p.x + (row * p.ldx + at) * kElemX, n, p.vec_x);
      sc[i] = kX == kCodeFp8 ? fp8_scale_f32(p.xs[row * p.ldxs + (at >> 7)]) : 1.0f;
    }
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    float g[kChunks][8], xh[kChunks][8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = ((i * kWaves + wave) * 64 + lane) * 8, n = p.D - col;
      float w[8], y[8];
      to_f32(ry[i], 1.0f, y);
      to_f32(rx[i], sc[i], xh[i]);
      param8(p.w, p.wcode, n > 0 ? col : 0, n, p.pvec, 1.0f, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[i][e] = e < n ? (xh[i][e] - mean) * rstd : 0.0f;
        g[i][e] = y[e] * w[e];
        s1 += g[i][e];
        s2 += g[i][e] * xh[i][e];
        dw[i][e] += y[e] * xh[i][e];
        db[i][e] += y[e];
      }
    }
    row_sum<kWaves>(s1, s2, red[turn], wave, lane);
    turn ^= 1;
    const float c1 = s1 * inv, c2 = s2 * inv;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = ((i * kWaves + wave) * 64 + lane) * 8, n = p.D - col;
      if (n <= 0) continue;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = rstd * (g[i][e] - c1 - xh[i][e] * c2);
      store8<kCode>(p.dx + (row * p.D + col) * kElem, n, p.vec_y && (p.D & 7) == 0, v);
    }
  }
  if (!p.sums) return;
  float* out = p.sums + (int64_t)blockIdx.x * 2 * p.D;
  if constexpr (kWaves == 1) {  // the workgroup's four waves hold the same columns: their sums in order
    __shared__ float part[4][64 * 8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) part[sub][e * 64 + lane] = k ? db[i][e] : dw[i][e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = sub * 2 + e, col = (i * 64 + lane) * 8 + j;
          if (col < p.D)
            out[k * p.D + col] = ((part[0][j * 64 + lane] + part[1][j * 64 + lane]) + part[2][j * 64 + lane]) + part[3][j * 64 + lane];
        }
      }
  } else {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int col = ((i * kWaves + wave) * 64 + lane) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < p.D) {
          out[col + e] = dw[i][e];
          out[p.D + col + e] = db[i][e];
        }
    }
  }
}

// Waves per row and chunks per lane: rows up to 1024 elements by one wave, up to 8192 by four, up to 24576 by sixteen.
constexpr int kNormMaxD = 24576;
template <class F>
static void with_shape(int D, F&& f) {
  using std::integral_constant;
  const int n = (D + 511) / 512;  // chunks of one wave
  if (n <= 1) f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (n <= 2) f(integral_constant<int, 2>{}, integral_constant<int, 1>{});
  else if (n <= 4) f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (n <= 8) f(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  else if (n <= 12) f(integral_constant<int, 3>{}, integral_constant<int, 4>{});
  else if (n <= 16) f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (n <= 32) f(integral_constant<int, 2>{}, integral_constant<int, 16>{});
  else f(integral_constant<int, 3>{}, integral_constant<int, 16>{});
}

// Workgroups of the backward pass: resident ones, each with an equal share of the rows.
static int64_t norm_grad_grid(int64_t M, int64_t D, int cus) {
  const int64_t units = D <= 1024 ? (M + 3) / 4 : M, most = (int64_t)cus * (D <= 8192 ? 3 : 1);
  return units < most ? units : most;
}

}  // namespace mxq

using namespace mxq;

static bool ln_aligned(const void* p, int64_t ld, int elem) {
  return reinterpret_cast<uintptr_t>(p) % (8 * elem < 16 ? 8 * elem : 16) == 0 && ld % 8 == 0;
}

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
  const int elem = dtype_bytes(dtype);
  const Norm p = {(const char*)x, (const char*)w, (const char*)b, (char*)y, mean, rstd, M, ldx, (int)D, param_dtype,
                  ln_aligned(x, ldx, elem) && ln_aligned(y, D, elem), ln_aligned(w, 8, 4) && ln_aligned(b, 8, 4), eps};
  with_shape((int)D, [&](auto N, auto W) {
    with_dtype(dtype, [&](auto C) {
      constexpr int kWaves = decltype(W)::value;
      const unsigned grid = (unsigned)(kWaves == 1 ? (M + 3) / 4 : M);
      hipLaunchKernelGGL((layer_norm_kernel<decltype(C)::value, decltype(N)::value, kWaves>), dim3(grid),
                         dim3(NormBlock<kWaves>::kThreads), 0, (hipStream_t)stream, p);
    });
  });
  return mxq_check_launch("layer_norm_kernel");
}

extern "C" int mxq_layer_norm_backward_strips(int64_t M, int64_t D, int64_t* strips) {
  if (M < 0 || D < 1 || !strips) return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld D=%lld", (long long)M, (long long)D);
  *strips = norm_grad_grid(M, D, mxq_cu_count());
  return MXQ_OK;
}

extern "C" int mxq_layer_norm_backward(const void* dy, int dtype, int64_t ldy, const void* x, int x_dtype, int64_t ldx,
                                       const uint8_t* x_scale, int64_t ldxs, const float* mean, const float* rstd,
                                       const void* w, int param_dtype, void* dx, float* sums, int64_t strips, int64_t M,
                                       int64_t D, void* stream) {
  if (const int rc = check_norm(M, D, dtype, param_dtype)) return rc;
  const bool kept = x_dtype == MXQ_DTYPE_E4M3;
  if (!kept && x_dtype != dtype) return mxq_set_error(MXQ_ERR_INVALID, "x of dtype code %d for gradients of %d", x_dtype, dtype);
  if (ldy < D || ldx < D || (kept && ldxs < (D + 127) / 128))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides for %lld columns", (long long)D);
  if (M == 0) return MXQ_OK;
  if (!dy || !x || !mean || !rstd || !dx || (kept && !x_scale)) return mxq_set_error(MXQ_ERR_INVALID, "null pointer");
  const int64_t grid = norm_grad_grid(M, D, mxq_cu_count());
  if (sums && strips != grid)
    return mxq_set_error(MXQ_ERR_INVALID, "room for %lld strips, %lld needed", (long long)strips, (long long)grid);
  const int elem = dtype_bytes(dtype);
  const NormGrad p = {(const char*)dy, (const char*)x, (const char*)w, x_scale, mean, rstd, (char*)dx, sums, M, ldy, ldx, ldxs,
                      (int)D, param_dtype, ln_aligned(dy, ldy, elem) && ln_aligned(dx, 8, elem),
                      ln_aligned(x, ldx, kept ? 1 : elem), ln_aligned(w, 8, 4)};
  with_shape((int)D, [&](auto N, auto W) {
    with_dtype(dtype, [&](auto C) {
      constexpr int kCode = decltype(C)::value, kWaves = decltype(W)::value, kChunks = decltype(N)::value;
      if (kept)
        hipLaunchKernelGGL((layer_norm_grad_kernel<kCode, kCodeFp8, kChunks, kWaves>), dim3((unsigned)grid),
                           dim3(NormBlock<kWaves>::kThreads), 0, (hipStream_t)stream, p);
      else
        hipLaunchKernelGGL((layer_norm_grad_kernel<kCode, kCode, kChunks, kWaves>), dim3((unsigned)grid),
                           dim3(NormBlock<kWaves>::kThreads), 0, (hipStream_t)stream, p);
    });
  });
  return mxq_check_launch("layer_norm_grad_kernel");
}
