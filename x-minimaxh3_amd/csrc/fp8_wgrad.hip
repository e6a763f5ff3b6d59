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
// waves owns a 256 (n) x 256 (k) tile, a wave 64 x 128 of it; a stage is 64 rows of m: dY's 64 x 256 bfloat16 (32 KB) and
// X's 64 x 256 codes, decoded on the way from registers to LDS (32 KB). Problems of few tiles split M over workgroups,
// which write float32 sums that fp8_join_kernel adds in order. 8192 rows, N 5376, K 14336: 1.01 to 1.04 ms, 1.25 PFLOP/s
// at 1.8 GHz, 64 % of the cycles matrix instructions (a library's plain bfloat16 product of row-major operands runs at
// 1.43 on the same card, with a transposed left operand, which this is, at 0.96).

#include "fp8_common.h"

namespace mxq {

constexpr int kWGroup = 4;
constexpr int kWTile = 256, kWRows = 64;
// 32-column blocks of n per wave (a wave: 32 kWNB x 128 of the tile). 2: eight waves, two per SIMD; 4: four waves, which
// read a third less from LDS but leave no second wave to fill a SIMD's gaps: 2.16 M cycles against 1.96 M for
// 5376 x 14336 x 8192 (1.20 M of matrix instructions).
constexpr int kWNB = 2;
constexpr int kWWaves = 16 / kWNB, kWThreads = 64 * kWWaves;
constexpr int kWStage = kWRows * kWTile * 2;  // bytes of one operand's stage in LDS

struct Wgrad {
  const uint16_t* dy;  // part p at dy + p * part_stride
  const uint8_t* q;
  const uint8_t* s;
  void* d;  // split: float32 sums, slice i at i * N * ldd
  int64_t M, N, K, ldy, part_stride, ldq, lds, ldd;
  int parts, tiles_n, tiles_k, splits, split_rows;  // split_rows: a multiple of kWRows
};

typedef short v4s __attribute__((ext_vector_type(4)));
typedef v4s __attribute__((address_space(3)))* lds_v4s;
typedef v4u __attribute__((address_space(3)))* lds_v4u;
typedef char __attribute__((address_space(3)))* lds_ptr;  // (pointer arithmetic: constants become the instructions' offsets)

// LDS rows are 512 bytes (256 bfloat16): 64-byte piece p of row r sits at piece p ^ (r & 3), so that the sixteen lanes of
// a transposing read (four rows, 32 bytes) and their neighbours cover all banks; and in every other 128 bytes of columns the
// two halves of 32 bytes change places, so that the eight lanes a 16-byte write serves at once, 32 bytes apart on 128 bytes
// of banks, do not meet (without it 78 M of 275 M LDS cycles in the product above).
MXQ_DEVICE int wg_at(int r, int byte) { return r * 512 + ((((byte >> 6) ^ (r & 3)) << 6) | ((byte & 63) ^ ((byte >> 3) & 16))); }

// A fragment's eight values: columns c0 + l % 32 (c0 a multiple of 32), rows 8 (l / 32) + {0..7} of the 16 rows from r0 on
// (a multiple of 16), in two transposing reads of four rows. Lane l of a group of sixteen gives the address of row
// (l % 16) / 4, columns 4 (l % 4) .. + 3 of a 4 x 16 patch, and receives its column l % 16. The address is that of
// fragment_base plus a constant: r & 3, which the swizzle uses, is the lane's own.
MXQ_DEVICE uint32_t fragment_base(uint32_t operand, int c0, int lane) {
  const int r = (lane >> 5) * 8 + ((lane & 15) >> 2);
  return operand + (uint32_t)wg_at(r, (c0 + (lane & 16) + (lane & 3) * 4) * 2);
}
template <int kRow>
MXQ_DEVICE v4s read_transposed(uint32_t base) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)((lds_ptr)(uintptr_t)base + kRow * 512));
}
MXQ_DEVICE v8bf join_fragment(const v4s (&f)[2]) {
  typedef short v8s __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(v8bf, v8s{f[0][0], f[0][1], f[0][2], f[0][3], f[1][0], f[1][1], f[1][2], f[1][3]});
}

static_assert(2 * 2 * kWStage / kWWaves >= 32 * 512, "LDS of a wave's block of results");
static_assert(kWRows == 64, "a stage is four half steps, written in two parts");
MXQ_DEVICE uint32_t buffer_load_u8(const void* base, int bytes, uint32_t voff) {
  return __builtin_amdgcn_raw_buffer_load_b8(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, kRawBufferWord3), (int)voff, 0, 0);
}

template <int kOut, bool kSplit>
__global__ __launch_bounds__(kWThreads, 1) void fp8_wgrad_kernel(Wgrad p) {
  __shared__ __attribute__((aligned(131072))) char lds[2 * 2 * kWStage];  // [buffer][dY, X]
  const int tiles = p.tiles_n * p.tiles_k, num = tiles * p.splits, per = num / 8, bid = blockIdx.x;
  int t = bid < per * 8 ? (bid % 8) * per + bid / 8 : bid;  // contiguous ranges over the XCDs
  const int slice = t / tiles;
  t -= slice * tiles;
  // groups of four tile-rows, so that the tiles an XCD runs at once share operand panels in its L2
  const int group = kWGroup * p.tiles_k, g0 = t / group * kWGroup, rows_g = min(p.tiles_n - g0, kWGroup), in_g = t - g0 * p.tiles_k;
  const int tk = in_g / rows_g, tn = g0 + in_g - tk * rows_g;
  const int n0 = tn * kWTile, k0 = tk * kWTile;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wn = (wave % (kWWaves / 2)) * 32 * kWNB, wk = (wave / (kWWaves / 2)) * 128;  // the wave's part of the tile
  const int M = (int)p.M, m_first = slice * p.split_rows, m_last = min(m_first + p.split_rows, M);
  const int stages = (m_last - m_first + kWRows - 1) / kWRows, total = stages * p.parts;

  // A thread's share of a stage: rows tid / 16 + kStep j, columns 16 (tid % 16) .. + 15 of both operands, by buffer loads
  // whose offsets point outside for what lies behind the slice's last row or the last column (they read zeros). Nothing is
  // read behind column N rounded up to 16 of dY or the last scale, where a view's last row may end its storage: the
  // columns behind hold other columns' values, whose sums are not stored.
  constexpr int kStep = kWThreads / 16, kShare = kWRows / kStep;
  const int r = tid >> 4, c = (tid & 15) * 16;
  const int ldy = (int)p.ldy, ldq = (int)p.ldq, lds_ = (int)p.lds;
  const uint32_t oy = (uint32_t)(r * ldy + min(n0 + c, ((int)p.N + 15) / 16 * 16 - 16)) * 2;
  const uint32_t oq = k0 + c < (int)p.K ? (uint32_t)(r * ldq + k0 + c) : kBufferOff;
  const uint32_t os = (uint32_t)(r * lds_ + (min(k0 + c, (int)p.K - 1) >> 7));
  v4u ya[kShare], yb[kShare], xq[kShare];
  uint32_t xs[kShare];
  // (the position of the next load: rows left in the slice and the operands' rows; offsets of lanes with a row stay inside
  // 64 rows, so the resources' size is that)
  int left = m_last - m_first, parts_left = left > 0 ? p.parts : 0;
  const uint16_t* py = p.dy + (int64_t)m_first * ldy;
  const uint8_t* pq = p.q + (int64_t)m_first * ldq;
  const uint8_t* ps = p.s + (int64_t)m_first * lds_;
  auto load = [&](auto JC) {
    constexpr int j = decltype(JC)::value;
    const bool on = r + kStep * j < left;
    const uint32_t vy = on ? oy + (uint32_t)(kStep * j * ldy) * 2 : kBufferOff;
    ya[j] = buffer_load_x4(py, kWRows * 2 * ldy, vy);
    yb[j] = buffer_load_x4(py, kWRows * 2 * ldy, vy + 16);
    xq[j] = buffer_load_x4(pq, kWRows * ldq, on ? oq + (uint32_t)(kStep * j * ldq) : kBufferOff);
    xs[j] = buffer_load_u8(ps, kWRows * lds_, on ? os + (uint32_t)(kStep * j * lds_) : kBufferOff);
    if constexpr (j == kShare - 1) {
      left -= kWRows;
      py += kWRows * ldy;
      pq += kWRows * ldq;
      ps += kWRows * lds_;
      if (left <= 0) {  // (the slice's end: the next part's first rows, or, behind the last part, none: left stays below 1)
        if (--parts_left > 0) {
          left = m_last - m_first;
          py += p.part_stride - (int64_t)stages * kWRows * ldy;
          pq -= (int64_t)stages * kWRows * ldq;
          ps -= (int64_t)stages * kWRows * lds_;
        }
      }
    }
  };
  // (row r + kStep j has r's swizzle)
  const uint32_t at[2] = {lds_addr(lds) + (uint32_t)wg_at(r, c * 2), lds_addr(lds) + (uint32_t)wg_at(r, c * 2 + 16)};
  // Write P (of four) of share j: dY's two halves, X's two halves.
  auto put = [&](uint32_t buf, auto JC, auto PC) {
    constexpr int j = decltype(JC)::value, kP = decltype(PC)::value;
    constexpr int kOff = (kP >= 2 ? kWStage : 0) + j * kStep * 512;
    v4u v = kP == 0 ? ya[j] : yb[j];
    if constexpr (kP >= 2)
      v = __builtin_bit_cast(v4u, fp8x8_to_bf16(xq[j][2 * kP - 4], xq[j][2 * kP - 3], fp8_scale_f32(xs[j])));
    *(lds_v4u)((lds_ptr)(uintptr_t)(at[kP & 1] ^ buf) + kOff) = v;
  };
  v16f acc[kWNB][4] = {};  // [n block][k block]
  // A stage is four half steps of 16 rows, a half step 4 kWNB slots, each one matrix instruction and a part of the other
  // work, in the order written (sched_barrier): fragments are read one half step ahead (a wave that issued its reads in
  // one go would wait for the other waves' reads with its matrix pipe idle: LDS and matrix time then add up, 4760 cycles
  // a stage against 2050 of matrix instructions); the next stage is written to the other buffer, a half each, during half
  // steps 1 and 2, the one behind it requested as the registers get free, and the barrier passed ahead of the last half
  // step, whose instructions cover the next stage's first reads.
  constexpr int kSlots = 4 * kWNB, kReads = 2 * (kWNB + 4), kPuts = 2 * kShare;
  constexpr int kReadSlots = kSlots * 6 / 8;  // the reads end early: the next half step's first instruction waits for them
  v4s fy[2][kWNB][2], fx[2][4][2];
  uint32_t base[kWNB + 4];  // fragment addresses in buffer 0: dY's, X's
#pragma unroll
  for (int b = 0; b < kWNB; ++b) base[b] = fragment_base(lds_addr(lds), wn + b * 32, lane);
#pragma unroll
  for (int b = 0; b < 4; ++b) base[kWNB + b] = fragment_base(lds_addr(lds) + kWStage, wk + b * 32, lane);
  auto read = [&](uint32_t buf, auto RowC, auto SetC, auto IC) {  // transposing read I of a half step
    // (in the order of their use: dY's first block, X's, dY's others)
    constexpr int kSet = decltype(SetC)::value, kI = decltype(IC)::value, kPos = kI / 2;
    constexpr int b = kPos == 0 ? 0 : kPos <= 4 ? kWNB + kPos - 1 : kPos - 4;
    const v4s v = read_transposed<decltype(RowC)::value + (kI & 1) * 4>(base[b] ^ buf);
    if constexpr (b < kWNB)
      fy[kSet][b][kI & 1] = v;
    else
      fx[kSet][b - kWNB][kI & 1] = v;
  };
  auto publish = [&] {
    wait_lgkm<0>();
    __builtin_amdgcn_sched_barrier(0);
    barrier_no_drain();
    __builtin_amdgcn_sched_barrier(0);
  };
  static_assert(2 * kWStage == 0x10000, "the buffers are one address bit apart");
  uint32_t buf = 0;  // byte offset of the stage's buffer
  auto stage = [&] {
    const uint32_t other = buf ^ (2 * kWStage);
    static_for<4>([&](auto H) {
      constexpr int h = decltype(H)::value, kSet = h & 1;
      constexpr bool kPut = h == 1 || h == 2;
      if constexpr (h == 3) publish();
      static_for<kSlots>([&](auto G) {
        constexpr int g = decltype(G)::value, a = g / 4, b = g % 4;
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join_fragment(fx[kSet][b]), join_fragment(fy[kSet][a]), acc[a][b], 0, 0, 0);
        static_for<kReads>([&](auto I) {
          constexpr int i = decltype(I)::value;
          if constexpr (i * kReadSlots / kReads == g)
            read(h < 3 ? buf : other, std::integral_constant<int, h < 3 ? (h + 1) * 16 : 0>{},
                 std::integral_constant<int, kSet ^ 1>{}, I);
        });
        if constexpr (kPut)
          static_for<kPuts>([&](auto P) {
            constexpr int i = decltype(P)::value;
            if constexpr (i * kSlots / kPuts == g)
              put(other, std::integral_constant<int, (h - 1) * (kShare / 2) + i / 4>{}, std::integral_constant<int, i % 4>{});
          });
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (kPut)
        static_for<kShare / 2>([&](auto J) { load(std::integral_constant<int, (h - 1) * (kShare / 2) + decltype(J)::value>{}); });
    });
    buf = other;
  };
  // (one loop for all stages: with the last ones peeled off, the copies of the accumulators between the loops spilled)
  static_for<kShare>(load);
  static_for<kShare>([&](auto J) { static_for<4>([&](auto P) { put(0, J, P); }); });
  static_for<kShare>(load);
  publish();
  static_for<kReads>([&](auto I) { read(0, std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{}, I); });
  for (int i = 0; i < total; ++i) stage();
  // Lane l holds row n = l % 32 of a block and, in register e, column (e / 4) * 8 + (l / 32) * 4 + e % 4. Stored from there, an
  // instruction would touch 32 bytes of 32 rows; through the wave's 16 KB of LDS (no wave reads a stage any more: the last
  // barrier is behind the last half step's reads) 32 lanes store a row's 128 columns. 16-byte piece c of row r sits at
  // piece c ^ r.
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  char* d = reinterpret_cast<char*>(p.d);
  if constexpr (kSplit) d += (int64_t)slice * p.N * p.ldd * 4;
  const int N = (int)p.N, K = (int)p.K;
  char* turn = lds + wave * (2 * 2 * kWStage / kWWaves);
#pragma unroll
  for (int a = 0; a < kWNB; ++a) {
    wave_lds_fence();
    const int r = lane & 31;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<v4f*>(turn + r * 512 + (((b * 8 + e * 2 + (lane >> 5)) ^ r) << 4)) =
            v4f{acc[a][b][4 * e], acc[a][b][4 * e + 1], acc[a][b][4 * e + 2], acc[a][b][4 * e + 3]};
    wave_lds_fence();
    const int k = k0 + wk + (lane & 31) * 4;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const int row = t * 2 + (lane >> 5), n = n0 + wn + a * 32 + row;
      const v4f y = *reinterpret_cast<const v4f*>(turn + row * 512 + (((lane & 31) ^ row) << 4));
      const float v[4] = {y[0], y[1], y[2], y[3]};
      if (n < N) store_run4<kOut>(d + (int64_t)n * p.ldd * kElem, k, K - k, v);
    }
  }
}

struct WgradPlan {
  int splits;
  int64_t rows;
};

// M slices, by an estimate in microseconds: a round of workgroups takes 4.5 and 1.5 per stage and part, slices cost a join.
// Measured: N = K = 1024 over 4096 rows (16 tiles) 23 + 6 us in slices, 101 us whole by the estimate; N = K = 5120 over
// 1024 rows 67 us whole, 400 tiles on 256 CUs.
static WgradPlan plan_wgrad(int64_t M, int64_t N, int64_t K, int parts, int cus) {
  const int64_t tiles = (N + kWTile - 1) / kWTile * ((K + kWTile - 1) / kWTile);
  WgradPlan best = {1, (M + kWRows - 1) / kWRows * kWRows};
  double best_cost = 1e300;
  for (int64_t s = 1; s <= 64; ++s) {
    const int64_t rows = ((M + s - 1) / s + kWRows - 1) / kWRows * kWRows;
    if (rows == 0 || (M + rows - 1) / rows != s || (s > 1 && tiles * s > 4 * cus)) continue;
    const double rounds = (double)((tiles * s + cus - 1) / cus);
    double cost = rounds * ((double)(rows / kWRows) * parts * 1.5 + 4.5);
    cost += slices_cost(s, N * K);
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

int mxq::fp8_wgrad_check(const void* dy, int parts, int64_t ldy, const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds,
                         const void* dw, int out_dtype, int64_t M, int64_t N, int64_t K) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 1 || K < 1 || parts < 1 || parts > 3 || M > (1ll << 31) - 1024 || N > (1 << 30) || K > (1 << 30))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld parts=%d", (long long)M, (long long)N, (long long)K, parts);
  const int64_t kb = (K + 127) / 128;
  // (64 rows are one buffer resource)
  if (ldy >= (1 << 24) || ldq >= (1 << 24) || lds >= (1 << 24) || ldy < (N + 15) / 16 * 16 || ldy % 8 ||
      ldq < (K + 15) / 16 * 16 || ldq % 16 || lds < kb)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldy=%lld ldq=%lld lds=%lld for N=%lld K=%lld", (long long)ldy,
                         (long long)ldq, (long long)lds, (long long)N, (long long)K);
  if (!dw || (M && (!dy || !q || !scale || !wg_aligned(dy, 16) || !wg_aligned(q, 16))))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  if ((N + kWTile - 1) / kWTile * ((K + kWTile - 1) / kWTile) >= (1ll << 23))  // (so many tiles are not split)
    return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 2^23 tiles");
  return MXQ_OK;
}

int mxq::fp8_wgrad(const void* dy, int parts, int64_t ldy, const uint8_t* q, int64_t ldq, const uint8_t* scale,
                             int64_t lds, void* dw, int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                             int64_t workspace_bytes, SliceJob* later, void* stream) {
  if (const int rc = fp8_wgrad_check(dy, parts, ldy, q, ldq, scale, lds, dw, out_dtype, M, N, K)) return rc;
  const WgradPlan plan = plan_wgrad(M, N, K, parts, mxq_cu_count());
  const int64_t tiles_n = (N + kWTile - 1) / kWTile, tiles_k = (K + kWTile - 1) / kWTile;
  const int64_t need = wgrad_bytes(plan, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need || !wg_aligned(workspace, 16)))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  Wgrad p = {(const uint16_t*)dy, q, scale, dw, M, N, K, ldy, M * ldy, ldq, lds, K, parts, (int)tiles_n, (int)tiles_k,
             plan.splits, (int)plan.rows};
  const unsigned grid = (unsigned)(tiles_n * tiles_k * plan.splits);
  if (plan.splits > 1) {
    const int64_t ldp = (K + 3) / 4 * 4;
    p.d = workspace;
    p.ldd = ldp;
    hipLaunchKernelGGL((fp8_wgrad_kernel<MXQ_DTYPE_F32, true>), dim3(grid), dim3(kWThreads), 0, (hipStream_t)stream, p);
    if (const int rc = mxq_check_launch("fp8_wgrad_kernel")) return rc;
    const SliceJob job = {(const float*)workspace, nullptr, dw, N, ldp, K, (int)K, plan.splits, out_dtype};
    if (!later) return fp8_join(job, {}, {}, stream);
    *later = job;
    return MXQ_OK;
  }
  with_dtype(out_dtype, [&](auto O) {
    hipLaunchKernelGGL((fp8_wgrad_kernel<decltype(O)::value, false>), dim3(grid), dim3(kWThreads), 0, (hipStream_t)stream, p);
  });
  return mxq_check_launch("fp8_wgrad_kernel");
}

extern "C" int mxq_fp8_wgrad(const void* dy, int parts, int64_t ldy, const uint8_t* q, int64_t ldq, const uint8_t* scale,
                             int64_t lds, void* dw, int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  return fp8_wgrad(dy, parts, ldy, q, ldq, scale, lds, dw, out_dtype, M, N, K, workspace, workspace_bytes, nullptr, stream);
}
