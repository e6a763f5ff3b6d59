// The last additions: float32 sums that a product's slices of the summed index wrote, and column sums that strips of rows
// wrote, added in a fixed order and rounded once. Each is a launch of a few microseconds, most of them the launch itself, so
// all that a backward pass leaves is added by one.
#include "fp8_common.h"

using namespace mxq;

namespace {

constexpr int kThreads = 256, kShares = kThreads / 32;  // (1024: 0.4 us more for small slices, no less for a column's many rows)

// D = out(sum over slices + bias), four columns per thread; the slices' rows are padded to whole fours.
template <int kOut>
MXQ_DEVICE void join_slices(const SliceJob& j, int64_t block) {
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  const int64_t runs = j.ldp / 4, g = block * kThreads + threadIdx.x;
  if (g >= j.rows * runs) return;
  const int64_t row = g / runs;
  const int col = (int)(g - row * runs) * 4;
  v4f y = sum_slices(reinterpret_cast<const v4f*>(j.part + row * j.ldp + col), j.splits, j.rows * runs);
  y += bias_run<kOut>(j.bias, col, j.cols);
  const float v[4] = {y[0], y[1], y[2], y[3]};
  store_run4<kOut>(reinterpret_cast<char*>(j.d) + row * j.ldd * kElem, col, j.cols - col, v);
}

MXQ_DEVICE float sum8(const float (&t)[8]) { return ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7])); }

// out[c] = sum over `parts` rows of a float32 [parts, n] table. 32 columns (a line) and 8 shares of the rows per
// workgroup; a share's loads go out eight at a time and are added in pairs, as the shares are (one after the other, 256
// rows of float32 sums were twice as far off).
static_assert(kShares == 8, "added by sum8");
template <int kOut>
MXQ_DEVICE void join_columns(const ColumnJob& j, int64_t block, float (&sm)[kShares][32]) {
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int64_t col = block * 32 + c;
  float v = 0.0f;
  if (col < j.n) {
    for (int64_t i = r; i < j.parts; i += 8 * kShares) {
      float t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) t[u] = i + u * kShares < j.parts ? j.in[(i + u * kShares) * j.n + col] : 0.0f;
      v += sum8(t);
    }
  }
  sm[r][c] = v;
  __syncthreads();
  if (r == 0 && col < j.n) {
    float t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = sm[k][c];
    store_out<kOut>(reinterpret_cast<typename OutT<kOut>::T*>(j.out) + col, sum8(t));
  }
}

// f with the dtype code as a constant (a workgroup's job has one).
template <class F>
MXQ_DEVICE void of_code(int code, F&& f) {
  if (code == MXQ_DTYPE_F32) f(std::integral_constant<int, MXQ_DTYPE_F32>{});
  else if (code == MXQ_DTYPE_F16) f(std::integral_constant<int, MXQ_DTYPE_F16>{});
  else f(std::integral_constant<int, MXQ_DTYPE_BF16>{});
}

__global__ __launch_bounds__(kThreads) void fp8_join_kernel(SliceJob a, SliceJob b, ColumnJob c, int blocks_c, int blocks_a) {
  __shared__ float sm[kShares][32];
  const int block = blockIdx.x;
  if (block < blocks_c)
    of_code(c.code, [&](auto C) { join_columns<decltype(C)::value>(c, block, sm); });
  else if (block < blocks_c + blocks_a)
    of_code(a.code, [&](auto C) { join_slices<decltype(C)::value>(a, block - blocks_c); });
  else
    of_code(b.code, [&](auto C) { join_slices<decltype(C)::value>(b, block - blocks_c - blocks_a); });
}

int64_t blocks_of(const SliceJob& j) { return j.splits ? (j.rows * (j.ldp / 4) + kThreads - 1) / kThreads : 0; }

}  // namespace

int mxq::fp8_join(const SliceJob& a, const SliceJob& b, const ColumnJob& c, void* stream) {
  const int64_t na = blocks_of(a), nb = blocks_of(b), nc = c.out ? (c.n + 31) / 32 : 0, blocks = na + nb + nc;
  if (blocks == 0) return MXQ_OK;
  if (blocks >= (1 << 24)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "too many sums to join");
  hipLaunchKernelGGL(fp8_join_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, a, b, c, (int)nc, (int)na);
  return mxq_check_launch("fp8_join_kernel");
}

extern "C" int mxq_column_join(const float* in, int64_t parts, int64_t n, void* out, int out_dtype, void* stream) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (parts < 0 || n < 1 || n >= (1ll << 27) || !out || (parts && !in)) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  return fp8_join({}, {}, {in, out, parts, n, out_dtype}, stream);
}
