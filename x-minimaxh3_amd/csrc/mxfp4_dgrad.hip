// Input gradient through a weight held in 4 bits (mxfp4_common.h):
//
//   dX[m, k] = sum_n dY[m, n] * W[n, k],   W[n, k] = code[n, k] * 2^(b[n, k / 32] - 127)
//
// dY is bfloat16 [M, N] (float16 and float32 gradients come as two and three bfloat16 parts whose products are summed; a float32
// value that bfloat16 rounds to an infinity, from (2 - 2^-8) 2^127 on, is one) and W is decoded to bfloat16, which is exact, so the
// only roundings are those of the float32 sums: 16-bit matrix instructions (v_mfma_f32_32x32x16_bf16). The 4-bit instructions cannot take W here: their scales go along the summed index, W's across it.
//
// dY's rows hold the summed index n, so its fragments (eight consecutive n of one row per lane) are plain 16-byte LDS reads; W
// has n as its rows, and its fragments come from transposing reads (ds_read_b64_tr_b16), which hand sixteen lanes the columns
// of a 4 x 16 patch. A workgroup of eight waves owns a 256 (m) x 256 (k) tile, a wave 64 x 128 of it, or, for problems of few
// tiles, four waves one of 128 x 128, or, of up to 64 rows, 64 x 256, a wave 64 x 64 of it; a stage is 64 of n: of the large tile,
// dY's 256 x 64 bfloat16 (32 KB) and W's 64 x 256 codes, decoded on the way from registers to LDS (32 KB). Problems of fewer tiles still split N over workgroups, which write
// float32 sums that fp8_join_kernel adds in order.
//
// 8192 rows, N 14336, K 5376 take 0.963 ms (1.31 PFLOP/s), 16384 rows, N and K 8192 1.65 (1.34): the rate of a library's plain
// bfloat16 product (1.25 to 1.34 for 8192 cubed). The matrix cores are busy 58 % of the time in the first, whose 2.6 rounds of tiles
// run as three. Four waves of 128 x 128, with two thirds of the LDS reads, ran 5 % slower.
#include "mxfp4_common.h"

namespace mxq {

constexpr int kDStage = 64, kDGroup = 4;

// A workgroup's tile: kTM x kTK, waves of 64 x 128 (256 x 256) or 64 x 64.
template <int kTM, int kTK>
struct DgradTile {
  static constexpr int kWavesM = kTM / 64, kMB = 2, kKB = kTM == 256 ? 4 : 2;  // 32-row and 32-column blocks of a wave
  static constexpr int kWaves = kWavesM * (kTK / (kKB * 32)), kThreads = 64 * kWaves;
  static constexpr int kBytesY = kTM * kDStage * 2, kBytesW = kTK * kDStage * 2;  // of an operand's stage in LDS
  static constexpr int kRow = kTK * 2;                                            // of W's rows there
  static constexpr int kRows = kThreads / 8;                                      // rows that the threads' loads take at once
  // a thread's loads of a stage: 16-byte pieces of dY, words of W (kWords in each of its rows), scale words
  static constexpr int kLoadsY = kTM / kRows, kWords = kTK / 64, kLoadsW = kDStage / kRows * kWords, kLoadsS = kLoadsW / 2;
};

struct Dgrad {
  const uint16_t* dy;  // part p at dy + p * part_stride
  const uint8_t *b, *sb;
  void* d;  // split: float32 sums, slice i at i * M * ldd
  int64_t M, N, K, ldy, part_stride, ldb, ldd;
  int parts, groups, tiles_m, tiles_k, splits, split_n;  // split_n: a multiple of kDStage
};

typedef short v4s __attribute__((ext_vector_type(4)));
typedef v4s __attribute__((address_space(3)))* lds_v4s;
typedef v4u __attribute__((address_space(3)))* lds_v4u;
typedef char __attribute__((address_space(3)))* lds_ptr;  // (pointer arithmetic: constants become the instructions' offsets)

// dY in LDS: rows of 128 bytes (64 n), 16-byte piece c of row r at piece c ^ ((r >> 1) & 7), so that the sixteen lanes a 16-byte
// read serves at once (sixteen rows, one piece) touch every bank once.
MXQ_DEVICE int dy_at(int r, int piece) { return r * 128 + ((piece ^ ((r >> 1) & 7)) << 4); }

// W in LDS: rows of kRow bytes (a tile's columns in bfloat16), 64-byte piece p of row r at piece p ^ (r & 3), so that the sixteen
// lanes of a transposing read (four rows, 32 bytes) and their neighbours cover all banks.
template <int kRow>
MXQ_DEVICE int w_at(int r, int byte) { return r * kRow + ((((byte >> 6) ^ (r & 3)) << 6) | (byte & 63)); }

// A fragment of W: columns c0 + l % 32 (c0 a multiple of 32), rows 8 (l / 32) + {0..7} of the 16 rows from r0 on (a multiple of
// 16), in two transposing reads of four rows. Lane l of a group of sixteen gives the address of row (l % 16) / 4, columns
// 4 (l % 4) .. + 3 of a 4 x 16 patch, and receives its column l % 16. The address is that of w_base plus a constant: r & 3, which
// the swizzle uses, is the lane's own.
template <int kRow>
MXQ_DEVICE uint32_t w_base(uint32_t operand, int c0, int lane) {
  const int r = (lane >> 5) * 8 + ((lane & 15) >> 2);
  return operand + (uint32_t)w_at<kRow>(r, (c0 + (lane & 16) + (lane & 3) * 4) * 2);
}
template <int kOff>
MXQ_DEVICE v4s read_transposed(uint32_t base) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)((lds_ptr)(uintptr_t)base + kOff));
}
MXQ_DEVICE v8bf join_fragment(const v4s (&f)[2]) {
  typedef short v8s __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(v8bf, v8s{f[0][0], f[0][1], f[0][2], f[0][3], f[1][0], f[1][1], f[1][2], f[1][3]});
}

MXQ_DEVICE uint32_t dgrad_load_u32(const void* base, int bytes, uint32_t voff) {
  return __builtin_amdgcn_raw_buffer_load_b32(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, kRawBufferWord3), (int)voff, 0, 0);
}

template <int kTM, int kTK, int kOut, bool kSplit>
__global__ __launch_bounds__((DgradTile<kTM, kTK>::kThreads), kTM == 256 ? 1 : 2) void mxfp4_dgrad_kernel(Dgrad p) {
  typedef DgradTile<kTM, kTK> C;
  constexpr int kDMB = C::kMB, kDKB = C::kKB, kBytesY = C::kBytesY, kBytesW = C::kBytesW, kLds = 2 * (kBytesY + kBytesW);
  // W's two buffers, then dY's, an operand's one address bit apart
  static_assert(kBytesY <= kBytesW, "alignment of dY's buffers");
  __shared__ __attribute__((aligned(2 * C::kBytesW))) char lds[kLds];
  const int tiles = p.tiles_m * p.tiles_k, num = tiles * p.splits, per = num / 8, bid = blockIdx.x;
  int t = bid < per * 8 ? (bid % 8) * per + bid / 8 : bid;  // contiguous ranges over the XCDs
  const int slice = t / tiles;
  t -= slice * tiles;
  // groups of four tile-rows, so that the tiles an XCD runs at once share operand panels in its L2
  const int group = kDGroup * p.tiles_k, g0 = t / group * kDGroup, rows_g = min(p.tiles_m - g0, kDGroup), in_g = t - g0 * p.tiles_k;
  const int tk = in_g / rows_g, tm = g0 + in_g - tk * rows_g;
  const int m0 = tm * kTM, k0 = tk * kTK;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = (wave % C::kWavesM) * 64, wk = (wave / C::kWavesM) * 32 * kDKB;  // the wave's part of the tile
  const int M = (int)p.M, K = (int)p.K, n_first = slice * p.split_n, n_last = min(n_first + p.split_n, (int)p.N);
  const int stages = (n_last - n_first + kDStage - 1) / kDStage, total = stages * p.parts;

  // A thread's share of a stage, by buffer loads whose offsets point outside for what lies behind the slice's last n or the last
  // row (they read zeros): of dY the 16-byte piece tid % 8 of rows tid / 8 + kRows j (nothing is read behind column N rounded up to
  // 8); of W the words of eight columns tid % 8 + 8 j of rows tid / 8 (+ kRows), with those rows' scale words, one per 128 columns.
  constexpr int kRows = C::kRows, kWords = C::kWords, kLoadsY = C::kLoadsY, kLoadsW = C::kLoadsW, kLoadsS = C::kLoadsS;
  const int r = tid >> 3, c = tid & 7;
  const int ldy = (int)p.ldy, ldb = (int)p.ldb, row_tiles = p.groups * (int)kFp4ScaleTile;
  const uint32_t oy = (uint32_t)(r * ldy + c * 8) * 2, ow = (uint32_t)(r * ldb + c * 4);
  const uint32_t os = (uint32_t)((r >> 5) * row_tiles + (r & 31) * 8 + ((k0 >> 8) & 1) * 4 + (kTK == 128 ? ((k0 >> 7) & 1) * 256 : 0));
  v4u y[kLoadsY];
  uint32_t w[kLoadsW], ws[kLoadsS];
  // (the position of the next load: n left in the slice and the operands' place)
  int left = n_last - n_first, parts_left = left > 0 ? p.parts : 0;
  const uint16_t* py = p.dy + (int64_t)m0 * ldy + n_first;
  const uint8_t* pw = p.b + (int64_t)n_first * ldb + k0 / 2;
  const uint8_t* ps = p.sb + (int64_t)(n_first >> 5) * row_tiles + (k0 >> 9) * kFp4ScaleTile;
  auto load = [&](auto HC) {  // the first or second half of a share
    constexpr int kH = decltype(HC)::value;
#pragma unroll
    for (int j = kH * kLoadsY / 2; j < (kH + 1) * kLoadsY / 2; ++j)
      y[j] = buffer_load_x4(py + (int64_t)(kRows * j) * ldy, kRows * 2 * ldy, c * 8 < left && m0 + kRows * j + r < M ? oy : kBufferOff);
#pragma unroll
    for (int j = kH * kLoadsW / 2; j < (kH + 1) * kLoadsW / 2; ++j) {
      const int down = j / kWords * kRows;
      w[j] = dgrad_load_u32(pw, kDStage * ldb, r + down < left ? ow + (uint32_t)(down * ldb + 32 * (j % kWords)) : kBufferOff);
    }
#pragma unroll
    for (int j = kH * kLoadsS / 2; j < (kH + 1) * kLoadsS / 2; ++j) {
      const int down = j / (kWords / 2) * kRows;
      ws[j] = dgrad_load_u32(ps, 2 * row_tiles, r + down < left ? os + (uint32_t)((down >> 5) * row_tiles + 256 * (j % (kWords / 2))) : kBufferOff);
    }
    if constexpr (kH == 1) {
      left -= kDStage;
      py += kDStage;
      pw += (int64_t)kDStage * ldb;
      ps += 2 * row_tiles;
      if (left <= 0) {  // (the slice's end: the next part's first n, or, behind the last part, none: left stays below 1)
        if (--parts_left > 0) {
          left = n_last - n_first;
          py += p.part_stride - (int64_t)stages * kDStage;
          pw -= (int64_t)stages * kDStage * ldb;
          ps -= (int64_t)stages * 2 * row_tiles;
        }
      }
    }
  };
  const uint32_t lds_y = lds_addr(lds) + 2 * kBytesW;
  const uint32_t at_y = lds_y + (uint32_t)dy_at(r, c);  // (row r + kRows j has r's swizzle)
  // (words c + 8 j: 128 bytes further on, two 64-byte pieces, whose number the swizzle is exclusive with)
  const uint32_t at_w = lds_addr(lds) + (uint32_t)w_at<C::kRow>(r, c * 16);
  // (odd: the second of an operand's buffers, all bits set, or none)
  auto put_y = [&](uint32_t odd, auto JC) {
    constexpr int j = decltype(JC)::value;
    *(lds_v4u)((lds_ptr)(uintptr_t)(at_y ^ (odd & kBytesY)) + j * kRows * 128) = y[j];
  };
  auto put_w = [&](uint32_t odd, auto JC) {
    constexpr int j = decltype(JC)::value, kWord = j % kWords, kRowOff = j / kWords * kRows * C::kRow;
    const uint32_t byte = (ws[j >> 1] >> (16 * (j & 1) + 8 * (c >> 2))) & 0xFFu;
    *(lds_v4u)((lds_ptr)(uintptr_t)(at_w ^ (odd & kBytesW) ^ (kWord * 128)) + kRowOff) =
        __builtin_bit_cast(v4u, fp4x8_to_bf16(w[j], fp8_scale_f32(byte)));
  };
  v16f acc[kDMB][kDKB] = {};
  // A stage is four steps of 16 n, a step kMB kKB slots, each one matrix instruction and a part of the other work, in the order
  // written (sched_barrier): fragments are read one step ahead; the next stage is written to the other buffer, a half each,
  // during steps 1 and 2, the one behind it requested as the registers get free, and the barrier passed ahead of the last
  // step, whose instructions cover the next stage's first reads.
  constexpr int kSlots = kDMB * kDKB, kReads = kDMB + 2 * kDKB;
  constexpr int kReadSlots = kSlots * 6 / 8;  // the reads end early: the next step's first instruction waits for them
  v4u fy[2][kDMB];
  v4s fw[2][kDKB][2];
  uint32_t base[kDKB];  // of W's fragments in buffer 0
#pragma unroll
  for (int b = 0; b < kDKB; ++b) base[b] = w_base<C::kRow>(lds_addr(lds), wk + b * 32, lane);
  // dY's fragments: row wm + l % 32 (+ 32 a), piece 2 step + l / 32
  uint32_t base_y[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) base_y[h] = lds_y + (uint32_t)dy_at(wm + (lane & 31), 2 * h + (lane >> 5));
  auto read = [&](uint32_t odd, auto StepC, auto SetC, auto IC) {  // read I of a step, in the order of their use
    constexpr int kStep = decltype(StepC)::value, kSet = decltype(SetC)::value, kI = decltype(IC)::value;
    if constexpr (kI == 0 || kI > 2 * kDKB) {
      constexpr int a = kI == 0 ? 0 : kI - 2 * kDKB;
      fy[kSet][a] = *(lds_v4u)((lds_ptr)(uintptr_t)(base_y[kStep] ^ (odd & kBytesY)) + a * 32 * 128);
    } else {
      constexpr int b = (kI - 1) / 2, kPart = (kI - 1) & 1;
      fw[kSet][b][kPart] = read_transposed<(kStep * 16 + kPart * 4) * C::kRow>(base[b] ^ (odd & kBytesW));
    }
  };
  auto publish = [&] {
    wait_lgkm<0>();
    __builtin_amdgcn_sched_barrier(0);
    barrier_no_drain();
    __builtin_amdgcn_sched_barrier(0);
  };
  uint32_t buf = 0;  // the stage's buffers
  auto stage = [&] {
    const uint32_t other = ~buf;
    static_for<4>([&](auto H) {
      constexpr int h = decltype(H)::value, kSet = h & 1;
      constexpr bool kPut = h == 1 || h == 2;
      if constexpr (h == 3) publish();
      static_for<kSlots>([&](auto G) {
        constexpr int g = decltype(G)::value, a = g / kDKB, b = g % kDKB;
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join_fragment(fw[kSet][b]), __builtin_bit_cast(v8bf, fy[kSet][a]), acc[a][b], 0, 0, 0);
        static_for<kReads>([&](auto I) {
          constexpr int i = decltype(I)::value;
          if constexpr (i * kReadSlots / kReads == g)
            read(h < 3 ? buf : other, std::integral_constant<int, h < 3 ? h + 1 : 0>{}, std::integral_constant<int, kSet ^ 1>{}, I);
        });
        if constexpr (kPut) {  // (half of dY's and of W's writes a step)
          constexpr int kPutsY = kLoadsY / 2, kPuts = kPutsY + kLoadsW / 2;
          static_for<kPuts>([&](auto I) {
            constexpr int i = decltype(I)::value;
            if constexpr (i * kSlots / kPuts == g) {
              if constexpr (i % 2 == 0 && i / 2 < kPutsY) put_y(other, std::integral_constant<int, (h - 1) * kPutsY + i / 2>{});
              else put_w(other, std::integral_constant<int, (h - 1) * (kLoadsW / 2) + i - (i / 2 + 1 < kPutsY ? i / 2 + 1 : kPutsY)>{});
            }
          });
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (kPut) load(std::integral_constant<int, h - 1>{});
    });
    buf = other;
  };
  // (one loop for all stages: with the last ones peeled off, copies of the accumulators between the loops would spill)
  static_for<2>(load);
  static_for<kLoadsY>([&](auto J) { put_y(0, J); });
  static_for<kLoadsW>([&](auto J) { put_w(0, J); });
  static_for<2>(load);
  publish();
  static_for<kReads>([&](auto I) { read(0, std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{}, I); });
  for (int i = 0; i < total; ++i) stage();
  // Lane l holds row m = l % 32 of a block and, in register e, column (e / 4) * 8 + (l / 32) * 4 + e % 4. Stored from there, an
  // instruction would touch 32 bytes of 32 rows; through the wave's 16 KB of LDS (no wave reads a stage any more: the last
  // barrier is behind the last step's reads) kLanes lanes store a row of the wave's columns. 16-byte piece c of row r sits at piece
  // c ^ (r % kLanes).
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2, kLanes = kDKB * 8, kTurn = kLanes * 16;
  static_assert(kLds / C::kWaves >= 32 * kTurn, "LDS of a wave's block of results");
  char* d = reinterpret_cast<char*>(p.d);
  if constexpr (kSplit) d += (int64_t)slice * p.M * p.ldd * 4;
  char* turn = lds + wave * (kLds / C::kWaves);
#pragma unroll
  for (int a = 0; a < kDMB; ++a) {
    wave_lds_fence();
    const int row = lane & 31;
#pragma unroll
    for (int b = 0; b < kDKB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<v4f*>(turn + row * kTurn + (((b * 8 + e * 2 + (lane >> 5)) ^ (row & (kLanes - 1))) << 4)) =
            v4f{acc[a][b][4 * e], acc[a][b][4 * e + 1], acc[a][b][4 * e + 2], acc[a][b][4 * e + 3]};
    wave_lds_fence();
    const int l = lane & (kLanes - 1), k = k0 + wk + l * 4;
#pragma unroll
    for (int u = 0; u < kLanes / 2; ++u) {
      const int q = u * (64 / kLanes) + lane / kLanes, m = m0 + wm + a * 32 + q;
      const v4f z = *reinterpret_cast<const v4f*>(turn + q * kTurn + ((l ^ (q & (kLanes - 1))) << 4));
      const float v[4] = {z[0], z[1], z[2], z[3]};
      if (m < M && k < K) store_run4<kOut>(d + (int64_t)m * p.ldd * kElem, k, K - k, v);
    }
  }
}

struct DgradPlan {
  int tile, splits;  // tile: its rows
  int64_t n;
};

static int tile_width(int rows) { return rows == 128 ? 128 : 256; }

// Tile and N slices, by an estimate in microseconds: a round of workgroups takes 5 and, per stage and part, 1.2 (256 x 256), 0.575
// (128 x 128) or 0.8 (64 x 256) where few CUs are at work, 1.58, 0.93 or 1.1 (two workgroups a CU) where all are, slices cost a join.
// Measured, whole and in the best number of slices, 128 / 256: one row, K 5120, N 5120: 52, 15.4 in twelve / 101, 19.8; 700 rows: 54.7,
// 52.8 in two / 105, 53.9 in four; 2048 rows 128 / 109; 700 rows, K 5120, N 20480: 195, 166 in two / 389, 142 in four; 4096 rows, K
// 20480, N 5120: 831 / 657; 2048 rows, K 1000, N 3001: 43.7, 34.9 in two / 74.6, 40.6 in four. In slices, 64 / 128: 40 rows, K 5120,
// N 5120: 17.5 / 17.9; K 5120, N 20480: 29.0 / 35.2, one row 24.4 / 32.4, 64 in fp32 67.4 / 89.7; K 2048, N 2048: 10.8 / 10.3.
static DgradPlan plan_dgrad(int64_t M, int64_t N, int64_t K, int parts, int cus) {
  DgradPlan best = {256, 1, (N + kDStage - 1) / kDStage * kDStage};
  double best_cost = 1e300;
  for (const int tile : {256, 128, 64}) {
    if (tile == 64 && M > 64) break;
    const int64_t tiles = (M + tile - 1) / tile * ((K + tile_width(tile) - 1) / tile_width(tile)), at_once = tile == 256 ? cus : 2 * cus;
    const double alone = tile == 256 ? 1.2 : tile == 128 ? 0.575 : 0.8, all = tile == 256 ? 1.58 : tile == 128 ? 0.93 : 1.1;
    for (int64_t s = 1; s <= 64; ++s) {
      const int64_t n = ((N + s - 1) / s + kDStage - 1) / kDStage * kDStage;
      if ((N + n - 1) / n != s || (s > 1 && tiles * s > 4 * cus)) continue;
      const double units = (double)(n / kDStage * parts), rest = (double)(tiles * s % at_once) / at_once;
      const double cost = (double)(tiles * s / at_once) * (units * all + 5.0) +
                          (rest > 0.0 ? units * (alone + (all - alone) * rest) + 5.0 : 0.0) + slices_cost(s, M * K) + 0.1 * s;
      if (cost < best_cost) {
        best_cost = cost;
        best = {tile, (int)s, n};
      }
    }
  }
  return best;
}

Fp4TileForm fp4_dgrad_form(int64_t M, int64_t N, int64_t K, int parts) {
  const DgradPlan plan = plan_dgrad(M, N, K, parts, mxq_cu_count());
  return {plan.tile, tile_width(plan.tile), plan.splits};
}

static int64_t dgrad_bytes(const DgradPlan& plan, int64_t M, int64_t K) {
  return plan.splits > 1 ? plan.splits * M * ((K + 3) / 4 * 4) * 4 : 0;
}

int64_t fp4_dgrad_workspace(int64_t M, int64_t N, int64_t K, int parts) {
  return M == 0 ? 0 : dgrad_bytes(plan_dgrad(M, N, K, parts, mxq_cu_count()), M, K);
}

int fp4_dgrad_check(const void* dy, int64_t ldy, const uint8_t* b, int64_t ldb, const uint8_t* sb, const void* dx, int out_dtype,
                    int64_t M, int64_t N, int64_t K) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 1 || K < 1 || M > (1ll << 31) - 1024 || N > (1ll << 22) || K > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (ldy < N || ldy % 8 || ldy >= (1 << 24) || ldb < fp4_row_bytes(K) || ldb % 16 || ldb > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides ldy=%lld ldb=%lld for N=%lld K=%lld", (long long)ldy, (long long)ldb,
                         (long long)N, (long long)K);
  if (M > 0 && (!dy || !b || !sb || !dx || reinterpret_cast<uintptr_t>(dy) % 16 || reinterpret_cast<uintptr_t>(b) % 16 ||
                reinterpret_cast<uintptr_t>(sb) % 16))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  if ((M + 127) / 128 * ((K + 127) / 128) >= (1ll << 23))  // (so many tiles are not split)
    return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 2^23 tiles");
  return MXQ_OK;
}

template <int kTM, int kTK, int kOut, bool kSplit>
static void launch_tile(const Dgrad& p, unsigned grid, void* stream) {
  hipLaunchKernelGGL((mxfp4_dgrad_kernel<kTM, kTK, kOut, kSplit>), dim3(grid), dim3(DgradTile<kTM, kTK>::kThreads), 0, (hipStream_t)stream, p);
}
template <int kOut, bool kSplit>
static void launch_dgrad(const Dgrad& p, int tile, unsigned grid, void* stream) {
  if (tile == 256) launch_tile<256, 256, kOut, kSplit>(p, grid, stream);
  else if (tile == 128) launch_tile<128, 128, kOut, kSplit>(p, grid, stream);
  else launch_tile<64, 256, kOut, kSplit>(p, grid, stream);
}

int fp4_dgrad(const void* dy, int parts, int64_t ldy, const uint8_t* b, int64_t ldb, const uint8_t* sb, void* dx, int out_dtype,
              int64_t M, int64_t N, int64_t K, void* workspace, SliceJob* later, void* stream) {
  if (const int rc = fp4_dgrad_check(dy, ldy, b, ldb, sb, dx, out_dtype, M, N, K)) return rc;
  const DgradPlan plan = plan_dgrad(M, N, K, parts, mxq_cu_count());
  const int64_t tiles_m = (M + plan.tile - 1) / plan.tile, tiles_k = (K + tile_width(plan.tile) - 1) / tile_width(plan.tile);
  Dgrad p = {(const uint16_t*)dy, b, sb, dx, M, N, K, ldy, M * ldy, ldb, K, parts, (int)fp4_groups(K), (int)tiles_m, (int)tiles_k,
             plan.splits, (int)plan.n};
  const unsigned grid = (unsigned)(tiles_m * tiles_k * plan.splits);
  if (plan.splits > 1) {
    const int64_t ldp = (K + 3) / 4 * 4;
    p.d = workspace;
    p.ldd = ldp;
    launch_dgrad<MXQ_DTYPE_F32, true>(p, plan.tile, grid, stream);
    *later = {(const float*)workspace, nullptr, dx, M, ldp, K, (int)K, plan.splits, out_dtype};
    return mxq_check_launch("mxfp4_dgrad_kernel");
  }
  with_dtype(out_dtype, [&](auto O) {
    launch_dgrad<decltype(O)::value, false>(p, plan.tile, grid, stream);
  });
  return mxq_check_launch("mxfp4_dgrad_kernel");
}

}  // namespace mxq
