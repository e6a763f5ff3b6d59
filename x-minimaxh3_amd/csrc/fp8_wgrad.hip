// Weight gradient from an activation kept in 8 bits (fp8_common.h):
//
//   dW[n, k] = sum_m dY[m, n] * X[m, k],   X[m, k] = q[m, k] * 2^(b[m, k / 128] - 127)
//
// dY is bfloat16 [M, N] (float16 and float32 gradients come as two and three bfloat16 parts whose products are summed),
// X is decoded to bfloat16, which is exact, so the only roundings are those of the float32 sums: 16-bit matrix
// instructions (v_mfma_f32_32x32x16_bf16), no second quantization of either operand.
//
// Both operands have the summed index m as their rows, so the fragments (eight consecutive m of one column per lane) are
// read from LDS by ds_read_b64_tr_b16, which hands sixteen lanes the columns of a 4 x 16 patch. A workgroup of eight
// waves owns a 256 (n) x 256 (k) tile, a wave 64 x 128 of it; a stage is 32 rows of m: dY's 32 x 256 bfloat16 (16 KB) and
// X's 32 x 256 codes, decoded on the way from registers to LDS (16 KB). Problems of few tiles split M over workgroups,
// which write float32 sums that wgrad_join_kernel adds in order.

#include "fp8_common.h"

namespace mxq {

constexpr int kWTile = 256, kWRows = 32;
constexpr int kWStage = kWRows * kWTile * 2;  // bytes of one operand's stage in LDS

struct Wgrad {
  const uint16_t* dy;  // part p at dy + p * part_stride
  const uint8_t* q;
  const uint8_t* s;
  void* d;  // split: float32 sums, slice i at i * N * ldd
  int64_t M, N, K, ldy, part_stride, ldq, lds, ldd;
  int parts, tiles_n, tiles_k, splits, split_rows;  // split_rows: a multiple of kWRows
  int vec;  // rows of d aligned to four elements
};

typedef short v4s __attribute__((ext_vector_type(4)));
typedef v4s __attribute__((address_space(3)))* lds_v4s;

// LDS rows are 512 bytes (256 bfloat16): 64-byte piece p of row r sits at piece p ^ (r & 3), so that the sixteen lanes of
// a transposing read (four rows, 32 bytes) and their neighbours cover all banks.
MXQ_DEVICE int wg_at(int r, int byte) { return r * 512 + ((((byte >> 6) ^ (r & 3)) << 6) | (byte & 63)); }

// Column c0 + l % 16.. of rows r0 .. r0 + 3: lane l of a group of sixteen gives the address of row r0 + (l % 16) / 4, columns
// c0 + 4 (l % 4) .. + 3 and receives column c0 + l % 16 of the four rows.
MXQ_DEVICE v4s read_transposed(const char* base, int r0, int c0, int l16) {
  const int r = r0 + (l16 >> 2);
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(base + wg_at(r, (c0 + (l16 & 3) * 4) * 2)));
}

// A fragment: columns c0 + l % 32, rows 8 (l / 32) + {0..7} of the 16 rows from r0 on.
MXQ_DEVICE v8bf read_fragment(const char* base, int r0, int c0, int lane) {
  const int l16 = lane & 15, c = c0 + (lane & 16), r = r0 + (lane >> 5) * 8;
  const v4s a = read_transposed(base, r, c, l16), b = read_transposed(base, r + 4, c, l16);
  typedef short v8s __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(v8bf, v8s{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

template <int kOut, bool kSplit>
__global__ __launch_bounds__(512, 2) void fp8_wgrad_kernel(Wgrad p) {
  __shared__ __attribute__((aligned(1024))) char lds[2][2][kWStage];  // [buffer][dY, X]
  const int tiles = p.tiles_n * p.tiles_k, num = tiles * p.splits, per = num / 8, bid = blockIdx.x;
  int t = bid < per * 8 ? (bid % 8) * per + bid / 8 : bid;  // contiguous ranges over the XCDs
  const int slice = t / tiles;
  t -= slice * tiles;
  const int tn = t / p.tiles_k, tk = t - tn * p.tiles_k;
  const int n0 = tn * kWTile, k0 = tk * kWTile;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wn = (wave & 3) * 64, wk = (wave >> 2) * 128;  // the wave's part of the tile
  const int M = (int)p.M, m_first = slice * p.split_rows, m_last = min(m_first + p.split_rows, M);
  const int stages = (m_last - m_first + kWRows - 1) / kWRows, total = stages * p.parts;

  // a thread's share of a stage: dY row tid / 16 (columns 16 (tid % 16) .. + 15), X the same
  const int r = tid >> 4, c = (tid & 15) * 16;
  const int64_t yn = min<int>(n0 + c, (int)p.ldy - 16 >= 0 ? (int)p.ldy - 16 : 0);
  const bool kin = k0 + c < (int)p.K;
  v4u ya, yb, xq;
  uint32_t xs;
  auto load = [&](int i) {
    const int part = i / stages, m = m_first + (i - part * stages) * kWRows + r;
    ya = yb = xq = v4u{0, 0, 0, 0};
    xs = 127;
    if (m < m_last) {
      // (columns behind N: another column's values, whose sums are not stored)
      const v4u* y = reinterpret_cast<const v4u*>(p.dy + part * p.part_stride + m * p.ldy + yn);
      ya = y[0];
      yb = y[1];
      if (kin) {
        xq = *reinterpret_cast<const v4u*>(p.q + m * p.ldq + k0 + c);
        xs = p.s[m * p.lds + ((k0 + c) >> 7)];
      }
    }
  };
  auto store = [&](int buf) {
    char* y = lds[buf][0];
    char* x = lds[buf][1];
    *reinterpret_cast<v4u*>(y + wg_at(r, c * 2)) = ya;
    *reinterpret_cast<v4u*>(y + wg_at(r, c * 2 + 16)) = yb;
    const float scale = fp8_scale_f32(xs);
    *reinterpret_cast<v4u*>(x + wg_at(r, c * 2)) = __builtin_bit_cast(v4u, fp8x8_to_bf16(xq[0], xq[1], scale));
    *reinterpret_cast<v4u*>(x + wg_at(r, c * 2 + 16)) = __builtin_bit_cast(v4u, fp8x8_to_bf16(xq[2], xq[3], scale));
  };
  v16f acc[2][4] = {};  // [n block][k block]
  if (total > 0) {
    load(0);
    store(0);
  }
  __syncthreads();
  for (int i = 0; i < total; ++i) {
    if (i + 1 < total) load(i + 1);
    const char* y = lds[i & 1][0];
    const char* x = lds[i & 1][1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v8bf fy[2], fx[4];
#pragma unroll
      for (int b = 0; b < 2; ++b) fy[b] = read_fragment(y, h * 16, wn + b * 32, lane);
#pragma unroll
      for (int b = 0; b < 4; ++b) fx[b] = read_fragment(x, h * 16, wk + b * 32, lane);
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fx[b], fy[a], acc[a][b], 0, 0, 0);
    }
    if (i + 1 < total) store((i + 1) & 1);
    __syncthreads();
  }
  // lane l holds row n = l % 32 of a block and, in register e, column (e / 4) * 8 + (l / 32) * 4 + e % 4
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  char* d = reinterpret_cast<char*>(p.d);
  if constexpr (kSplit) d += (int64_t)slice * p.N * p.ldd * 4;
  const int N = (int)p.N, K = (int)p.K;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int n = n0 + wn + a * 32 + (lane & 31);
    if (n >= N) continue;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = k0 + wk + b * 32 + e * 8 + (lane >> 5) * 4;
        const float v[4] = {acc[a][b][4 * e], acc[a][b][4 * e + 1], acc[a][b][4 * e + 2], acc[a][b][4 * e + 3]};
        store_run4<kOut>(d + (int64_t)n * p.ldd * kElem, k, K - k, p.vec, v);
      }
  }
}

// D = out(sum over slices), four columns per thread.
template <int kOut>
__global__ __launch_bounds__(256) void wgrad_join_kernel(const float* part, int splits, int64_t N, int64_t K, int64_t ldp,
                                                         char* d, int vec) {
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  const int64_t runs = ldp / 4, g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (g >= N * runs) return;
  const int64_t row = g / runs;
  const int col = (int)(g - row * runs) * 4;
  v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < splits; ++s) y += *reinterpret_cast<const v4f*>(part + (s * N + row) * ldp + col);
  const float v[4] = {y[0], y[1], y[2], y[3]};
  store_run4<kOut>(d + row * K * kElem, col, (int)K - col, vec, v);
}

struct WgradPlan {
  int splits;
  int64_t rows;
};

// M slices: whole rounds of workgroups, a round costing its stages and a fixed part worth about twelve of them; slices also
// write and read their float32 sums.
static WgradPlan plan_wgrad(int64_t M, int64_t N, int64_t K, int parts, int cus) {
  const int64_t tiles = (N + kWTile - 1) / kWTile * ((K + kWTile - 1) / kWTile);
  WgradPlan best = {1, (M + kWRows - 1) / kWRows * kWRows};
  double best_cost = 1e300;
  for (int64_t s = 1; s <= 64; ++s) {
    const int64_t rows = ((M + s - 1) / s + kWRows - 1) / kWRows * kWRows;
    if (rows == 0 || (M + rows - 1) / rows != s || (s > 1 && tiles * s > 4 * cus)) continue;
    const double rounds = (double)((tiles * s + cus - 1) / cus);
    double cost = rounds * ((double)(rows / kWRows) * parts + 12.0);
    if (s > 1) cost += 12.0 + (double)(N * K) * (double)(s + 1) / 1.5e6;
    if (cost < best_cost) {
      best_cost = cost;
      best = {(int)s, rows};
    }
  }
  return best;
}

static int64_t wgrad_bytes(const WgradPlan& plan, int64_t N, int64_t K) {
  return plan.splits > 1 ? plan.splits * N * ((K + 3) / 4 * 4) * 4 : 0;
}

}  // namespace mxq

using namespace mxq;

static bool wg_aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

extern "C" int mxq_fp8_wgrad_workspace(int64_t M, int64_t N, int64_t K, int parts, int64_t* bytes) {
  if (M < 0 || N < 1 || K < 1 || parts < 1 || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  *bytes = wgrad_bytes(plan_wgrad(M, N, K, parts, mxq_cu_count()), N, K);
  return MXQ_OK;
}

extern "C" int mxq_fp8_wgrad(const void* dy, int parts, int64_t ldy, const uint8_t* q, int64_t ldq, const uint8_t* scale,
                             int64_t lds, void* dw, int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 1 || K < 1 || parts < 1 || parts > 3 || M > (1ll << 31) - 1024 || N > (1 << 30) || K > (1 << 30))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld parts=%d", (long long)M, (long long)N, (long long)K, parts);
  const int64_t kb = (K + 127) / 128;
  // (dY rows of whole sixteens; code rows of whole sixteens, zero behind K)
  if (ldy < (N + 15) / 16 * 16 || ldy % 8 || ldq < (K + 15) / 16 * 16 || ldq % 16 || lds < kb)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldy=%lld ldq=%lld lds=%lld for N=%lld K=%lld", (long long)ldy,
                         (long long)ldq, (long long)lds, (long long)N, (long long)K);
  if (!dw || (M && (!dy || !q || !scale || !wg_aligned(dy, 16) || !wg_aligned(q, 16))))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  const WgradPlan plan = plan_wgrad(M, N, K, parts, mxq_cu_count());
  const int64_t tiles_n = (N + kWTile - 1) / kWTile, tiles_k = (K + kWTile - 1) / kWTile;
  if (tiles_n * tiles_k * plan.splits >= (1ll << 31)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 2^31 tiles");
  const int64_t need = wgrad_bytes(plan, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need || !wg_aligned(workspace, 16)))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  const int run = 4 * dtype_bytes(out_dtype);
  const int vec = wg_aligned(dw, run) && K % 4 == 0;
  Wgrad p = {(const uint16_t*)dy, q, scale, dw, M, N, K, ldy, M * ldy, ldq, lds, K, parts, (int)tiles_n, (int)tiles_k,
             plan.splits, (int)plan.rows, vec};
  const unsigned grid = (unsigned)(tiles_n * tiles_k * plan.splits);
  if (plan.splits > 1) {
    const int64_t ldp = (K + 3) / 4 * 4;
    p.d = workspace;
    p.ldd = ldp;
    p.vec = 1;
    const int64_t blocks = (N * (ldp / 4) + 255) / 256;
    if (blocks >= (1ll << 31)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "gradient too large");
    hipLaunchKernelGGL((fp8_wgrad_kernel<MXQ_DTYPE_F32, true>), dim3(grid), dim3(512), 0, (hipStream_t)stream, p);
    if (const int rc = mxq_check_launch("fp8_wgrad_kernel")) return rc;
    with_dtype(out_dtype, [&](auto O) {
      hipLaunchKernelGGL((wgrad_join_kernel<decltype(O)::value>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                         (const float*)workspace, plan.splits, N, K, ldp, (char*)dw, vec);
    });
    return mxq_check_launch("wgrad_join_kernel");
  }
  with_dtype(out_dtype, [&](auto O) {
    hipLaunchKernelGGL((fp8_wgrad_kernel<decltype(O)::value, false>), dim3(grid), dim3(512), 0, (hipStream_t)stream, p);
  });
  return mxq_check_launch("fp8_wgrad_kernel");
}
