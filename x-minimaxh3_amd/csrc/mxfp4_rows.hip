// The 4-bit layer of few rows (up to 16; mxfp4_common.h): a stream of the weight.
//
// A workgroup's four or eight waves take up to 16 kRT weight rows and share K. Weight fragments go from memory straight to registers (a
// lane: row l % 16, blocks l / 16 and 4 + l / 16 of a stage of 256 columns), a stage ahead of the one at work, and are multiplied by
// v_mfma_scale_f32_16x16x128_f8f6f4 as they are, each lane giving the scale byte of its own block. The activations come in their
// own type or as a pair; each wave brings its own K range of them, a chunk of stages at a time, into its part of LDS, quantizing
// them on the way, which saves the quantizer's launch. How many weight rows a workgroup takes decides (plan_rows): each
// workgroup quantizes all of x again, and what counts is the CU with the most weight rows. Missing rows of a block of sixteen are
// not read.
#include <algorithm>

#include "mxfp4_common.h"

namespace mxq {

struct Fp4Rows {
  const void* x;      // [M, ldx] of the input type, or codes [M, ldx] with scales sx [M, ldsx]
  const uint8_t* sx;
  const uint8_t *b, *sb;
  const void* bias;
  void* d;
  int64_t M, N, K, ldx, ldsx, ldb, ldd;
  int x_code, groups, stages;
  int chunk_log2;  // stages per chunk
  int rows;        // weight rows of a workgroup: a multiple of 4, 16 kRT at most
};

// LDS of a wave's chunk: rows of codes, 16 bytes apart in banks, then eight scale bytes per row and stage.
__host__ MXQ_DEVICE int fp4_chunk_row(int log2) { return (128 << log2) + 16; }
__host__ MXQ_DEVICE int fp4_chunk_bytes(int M, int log2) { return (M * (fp4_chunk_row(log2) + (8 << log2)) + 15) / 16 * 16; }

// Stages `first` .. of all rows quantized into the wave's chunk; stages from `last` on are not read.
template <int kIn>
MXQ_DEVICE void quantize_chunk(const Fp4Rows& p, uint8_t* lds, int first, int last, int lane) {
  constexpr int kElem = kIn == MXQ_DTYPE_F32 ? 4 : 2, kBatch = kIn == MXQ_DTYPE_F32 ? 2 : 4;
  const int M = (int)p.M, log2 = p.chunk_log2, items = M << (log2 + 4), ld = fp4_chunk_row(log2);
  const int end = min(last * 256, (int)p.K);
  uint8_t* sc = lds + M * ld;
  for (int it = lane; it - lane < items; it += 64 * kBatch) {
    Piece<kIn> t[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int item = it + 64 * u, row = item >> (log2 + 4), col = first * 256 + (item & ((16 << log2) - 1)) * 16;
      const int n = row < M ? end - col : 0;
      t[u] = piece_load<kIn>(reinterpret_cast<const char*>(p.x) + (n > 0 ? row * p.ldx + col : 0) * kElem, n);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int item = it + 64 * u, row = item >> (log2 + 4), piece = item & ((16 << log2) - 1);
      uint32_t m = piece_absmax(t[u]);
      m = max(m, dpp_lane<kDppQuadXor1>(m));
      const uint32_t byte = fp4_scale_byte(m);
      v2u c = fp4_encode(t[u], fp8_scale_f32(byte));
      if (byte == 255u) c = v2u{0, 0};
      if (row < M) {
        *reinterpret_cast<v2u*>(lds + row * ld + piece * 8) = c;
        if ((piece & 1) == 0) sc[(row << (log2 + 3)) + (piece >> 1)] = (uint8_t)byte;
      }
    }
  }
  wave_lds_fence();
}

// The same of a pair (nothing is read behind its columns; the code behind an odd row's last is cleared).
MXQ_DEVICE void copy_chunk(const Fp4Rows& p, uint8_t* lds, int first, int last, int lane) {
  const int M = (int)p.M, K = (int)p.K, log2 = p.chunk_log2, items = M << (log2 + 3), ld = fp4_chunk_row(log2);
  uint8_t* sc = lds + M * ld;
  for (int it = lane; it < items; it += 64) {
    const int row = it >> (log2 + 3), block = it & ((8 << log2) - 1), at = first * 8 + block;
    const int n = at < last * 8 ? K - at * 32 : 0;  // columns of the block
    v4u v = bytes_load(reinterpret_cast<const uint8_t*>(p.x) + row * p.ldx + (n > 0 ? at * 16 : 0), (min(n, 32) + 1) / 2);
    if (n > 0 && n < 32 && (n & 1)) {
      const int half = n >> 1;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i == half >> 2) v[i] &= ~(0xF0u << (8 * (half & 3)));
    }
    *reinterpret_cast<v4u*>(lds + row * ld + block * 16) = v;
    sc[(row << (log2 + 3)) + block] = n > 0 ? p.sx[row * p.ldsx + at] : (uint8_t)127;
  }
  wave_lds_fence();
}

MXQ_DEVICE uint32_t rows_load_u32(const void* base, int bytes, uint32_t voff) {
  return __builtin_amdgcn_raw_buffer_load_b32(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, kRawBufferWord3), (int)voff, 0, 0);
}

template <int kRT>
struct Fp4Stage {  // a stage's operands of a wave
  v4u w[kRT][2];
  uint32_t s[kRT][2];
};

template <int kOut, int kRT>
__global__ __launch_bounds__(512) void mxfp4_rows_kernel(Fp4Rows p) {
  const int kW = blockDim.x >> 6;
  extern __shared__ __align__(16) uint8_t rows_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
  const int N = (int)p.N, M = (int)p.M, n0 = blockIdx.x * p.rows;
  const int per = (p.stages + kW - 1) / kW, first = wave * per, last = min(first + per, p.stages);
  const int rows = min(N - n0, p.rows), row_tiles = p.groups * (int)kFp4ScaleTile;
  const uint8_t* wb = p.b + (int64_t)n0 * p.ldb;
  const uint8_t* sb = p.sb + (int64_t)(n0 >> 5) * row_tiles;
  const int wbytes = rows * (int)p.ldb, sbytes = (((n0 & 31) + rows + 31) >> 5) * row_tiles;
  uint32_t woff[kRT], soff[kRT];
#pragma unroll
  for (int r = 0; r < kRT; ++r) {
    const int row = r * 16 + lr, at = (n0 & 31) + row;
    woff[r] = row < rows ? (uint32_t)(row * (int)p.ldb + g * 16) : kBufferOff;
    soff[r] = row < rows ? (uint32_t)((at >> 5) * row_tiles + (at & 31) * 8) : kBufferOff;
  }
  uint8_t* chunk = rows_lds + wave * fp4_chunk_bytes(M, p.chunk_log2);
  const int ld = fp4_chunk_row(p.chunk_log2), chunk_mask = (1 << p.chunk_log2) - 1;
  v4f acc[kRT] = {};
  typedef Fp4Stage<kRT> Stage;
  auto load = [&](Stage& t, int s) {
    const bool in = s < last;
#pragma unroll
    for (int r = 0; r < kRT; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        t.w[r][u] = buffer_load_x4(wb, wbytes, in ? woff[r] + (uint32_t)(s * 128 + u * 64) : kBufferOff);
        t.s[r][u] = rows_load_u32(sb, sbytes, in ? soff[r] + (uint32_t)((s >> 1) * 512 + u * 256 + (s & 1) * 4) : kBufferOff);
      }
  };
  auto compute = [&](const Stage& t, int s) {
    if (s >= last) return;
    const int at = (s - first) & chunk_mask;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      v4i x = {0, 0, 0, 0};
      int byte = 127;
      if (lr < M) {
        x = *reinterpret_cast<const v4i*>(chunk + lr * ld + at * 128 + u * 64 + g * 16);
        byte = chunk[M * ld + (lr << (p.chunk_log2 + 3)) + at * 8 + u * 4 + g];
      }
#pragma unroll
      for (int r = 0; r < kRT; ++r) {
        const v4u w = t.w[r][u];
        acc[r] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            v8i{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0}, v8i{x[0], x[1], x[2], x[3], 0, 0, 0, 0}, acc[r], 4, 4, 0,
            (int)(t.s[r][u] >> (8 * g)), 0, byte);
      }
    }
  };
  Stage t0, t1;
  load(t0, first);
  for (int s = first; s < last; s += 2) {
    load(t1, s + 1);
    if (((s - first) & chunk_mask) == 0) {
      const int end = min(last, s + chunk_mask + 1);
      if (p.x_code == MXQ_DTYPE_BF16) quantize_chunk<MXQ_DTYPE_BF16>(p, chunk, s, end, lane);
      else if (p.x_code == MXQ_DTYPE_F16) quantize_chunk<MXQ_DTYPE_F16>(p, chunk, s, end, lane);
      else if (p.x_code == MXQ_DTYPE_F32) quantize_chunk<MXQ_DTYPE_F32>(p, chunk, s, end, lane);
      else copy_chunk(p, chunk, s, end, lane);
    }
    compute(t0, s);
    load(t0, s + 2);
    compute(t1, s + 1);
  }
  __syncthreads();  // (the sums take the chunks' place)
  v4f* part = reinterpret_cast<v4f*>(rows_lds);
#pragma unroll
  for (int r = 0; r < kRT; ++r) part[(wave * kRT + r) * 64 + lane] = acc[r];
  __syncthreads();
  // the waves' sums in order; blocks of sixteen weight rows are dealt to the waves
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  for (int r = wave; r < kRT; r += kW) {
    const int col = n0 + r * 16 + g * 4;
    v4f y = part[r * 64 + lane];
    for (int k = 1; k < kW; ++k) y += part[(k * kRT + r) * 64 + lane];
    if (lr < M && col < n0 + rows) {
      y += bias_run<kOut>(p.bias, col, N);
      const float v[4] = {y[0], y[1], y[2], y[3]};
      store_run4<kOut>(reinterpret_cast<char*>(p.d) + lr * p.ldd * kElem, col, N - col, v);
    }
  }
}

// Weight rows (a multiple of 4: mostly what gives every CU its share and no more) and waves of a workgroup, by an estimate in
// microseconds: the CU with the most workgroups streams their weight rows, 0.090 (four waves) or 0.079 (eight) per sixteen and stage,
// half of it for a block's missing rows too, and brings x for each workgroup, per row and stage 0.013 (four waves; 0.025 where they
// are alone on their CU) or 0.014 (eight); all CUs together stream at 5.2 TB/s; eight waves take longer to start and to add up. Measured, bf16, weights from
// memory, by rows and waves: one row, K 5120, N 5120: 20/4 6.1, 32/4 6.5, 20/8 6.0, 32/8 6.2, 64/8 9.9; N 20480: 16/4 13.0, 32/4 15.2,
// 80/8 15.6; K 20480, N 5120: 16/4 17.8, 20/4 15.8, 32/4 17.9, 16/8 18.0, 20/8 14.6, 32/8 16.4; K 14336, N 5376: 16/4 12.5, 24/8 11.9,
// 32/8 12.5; four rows, K 20480, N 5120: 20/4 22.1, 20/8 18.4, 32/8 20.4; K 5376, N 21504: 28/4 15.7, 44/4 16.1, 84/8 17.7; 16 rows,
// K 5120, N 20480: 16/4 33.9, 48/4 25.3, 80/8 19.7.
struct RowsPlan4 {
  int rows, waves;
  double cost;
};
static RowsPlan4 plan_rows(int64_t M, int64_t N, int64_t stages, int cus) {
  RowsPlan4 best = {16, 4, 1e300};
  const double stream = (double)(N * stages) * 136.0 / 5.2e6;
  // (more than 96 rows in eight waves spill)
  for (int waves = 4; waves <= 8; waves += 4) {
    for (int rows = 12; rows <= (waves == 4 ? 48 : 96); rows += 4) {
      const int64_t groups = (N + rows - 1) / rows;
      const double turns = (double)((groups + cus - 1) / cus), blocks = (double)((rows + 15) / 16);
      const double units = turns * (double)stages * (rows / 32.0 + blocks / 2.0) * (waves == 4 ? 0.090 : 0.079);
      const double x = turns * (double)(stages * M) * (waves == 8 ? 0.014 : groups <= cus ? 0.025 : 0.013);
      const double cost = (waves == 4 ? 2.5 : 3.0 + 0.35 * blocks) + std::max(units + x, stream);
      if (cost < best.cost) best = {rows, waves, cost};
    }
  }
  return best;
}

Fp4RowsForm fp4_rows_form(int64_t M, int64_t N, int64_t K) {
  const RowsPlan4 plan = plan_rows(M, N, fp4_row_bytes(K) / kFp4Stage, mxq_cu_count());
  return {plan.rows, plan.waves};
}

template <int kOut, int kRT>
static void launch_rows(Fp4Rows p, int waves, void* stream) {
  // chunks of a wave's whole K range where all rows' take up to 36 KB of LDS, down to two stages
  const int per = (p.stages + waves - 1) / waves, M = (int)p.M;
  p.chunk_log2 = 1;
  while (p.chunk_log2 < 6 && (1 << p.chunk_log2) < per && waves * fp4_chunk_bytes(M, p.chunk_log2 + 1) <= 36 * 1024) ++p.chunk_log2;
  const int bytes = std::max(kRT * 1024 * waves, waves * fp4_chunk_bytes(M, p.chunk_log2));
  hipLaunchKernelGGL((mxfp4_rows_kernel<kOut, kRT>), dim3((unsigned)((p.N + p.rows - 1) / p.rows)), dim3(64 * waves), bytes,
                     (hipStream_t)stream, p);
}

int fp4_linear_rows(const void* x, int x_dtype, int64_t ldx, const uint8_t* sx, int64_t ldsx, const uint8_t* b, int64_t ldb,
                    const uint8_t* sb, const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K,
                    void* stream) {
  if (const int rc = fp4_gemm_check(b, ldb, sb, b, ldb, sb, d, ldd, out_dtype, M, N, K)) return rc;
  Fp4Rows p = {x, sx, b, sb, bias, d, M, N, K, ldx, ldsx, ldb, ldd, x_dtype, (int)fp4_groups(K), (int)(fp4_row_bytes(K) / kFp4Stage), 0, 0};
  const RowsPlan4 plan = plan_rows(M, N, p.stages, mxq_cu_count());
  p.rows = plan.rows;
  with_dtype(out_dtype, [&](auto O) {
    constexpr int kOut = decltype(O)::value;
    switch ((plan.rows + 15) / 16) {
      case 1: return launch_rows<kOut, 1>(p, plan.waves, stream);
      case 2: return launch_rows<kOut, 2>(p, plan.waves, stream);
      case 3: return launch_rows<kOut, 3>(p, plan.waves, stream);
      case 4: return launch_rows<kOut, 4>(p, plan.waves, stream);
      case 5: return launch_rows<kOut, 5>(p, plan.waves, stream);
      default: return launch_rows<kOut, 6>(p, plan.waves, stream);
    }
  });
  return mxq_check_launch("mxfp4_rows_kernel");
}

}  // namespace mxq
