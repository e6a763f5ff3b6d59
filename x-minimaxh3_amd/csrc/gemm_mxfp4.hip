// Matrix product of MXFP4 operands (mxfp4_common.h) on gfx950 matrix cores:
//
//   D[m, n] = out( sum_b 2^(ea[m, b] + eb[n, b]) * sum_{k in block b} A[m, k] * B[n, k]  +  bias[n] )
//
// A [M, K] activations, B [N, K] a weight, both with one scale per row and 32 columns, sums in float32.
//
// A workgroup of four waves, one per SIMD, owns a 256 x 256, 128 x 256 or 128 x 128 tile, a wave a quarter of it: with 128 x 128 a wave
// the fragments of a step are read from LDS once for 16 matrix instructions (eight waves of 128 x 64, which took turns, read a
// third more; power bounds the product, and they ran at 4.5 PFLOP/s where this form runs at 4.8). Operand chunks are fetched by
// direct-to-LDS loads into a ring of five 32 KB slots, one to two stages ahead; one barrier a stage.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes 32 columns of a row from each lane, one block, and the lane's own scale byte for it: of 256
// columns, lanes 0-31 take the blocks 0 .. 3 in turn, lanes 32-63 the blocks 4 .. 7, so that a lane's scales are the four bytes of a
// word, which the instruction picks from. The scale tiles hold these words lane by lane, two of them: one eight-byte load a
// wave (512 consecutive bytes) for 32 rows and 512 columns.
//
// 75600 x 5120 of K 5120 takes 0.94 ms (4.2 PFLOP/s), 16384 cubed 1.83 (4.8), 8192 x 21504 of K 5376 0.44 (4.3); a library's product of
// the same format 3.1 to 3.4 PFLOP/s. The clock falls to 1.55 GHz, power bounds it: without LDS reads, operand loads and scales,
// the matrix instructions alone run at 1.2 times the rate.
//
// Precision of the instruction, measured: a block's 32 products are added exactly (they are whole multiples of one power of
// two), and the blocks' sums and the float32 with what lies below 2^-22 of the largest cut. On a layer's usual data every
// sum up to K 20480 came out exact: the products are multiples of few powers of two. So there is one kernel for all outputs.
//
// Problems of few tiles split K over workgroups, which write float32 sums that fp8_join_kernel adds in order.

#include <algorithm>

#include "gemm_tiles.h"
#include "mxfp4_common.h"

namespace mxq {

struct Fp4Gemm {
  const uint8_t *a, *b, *sa, *sb;
  const void* bias;
  void* d;  // split: float32 sums, slice s at s * M * ldd
  int64_t M, N, lda, ldb, ldd;
  int groups, stages;
  int tiles_m, tiles_n;
  int splits, split_stages;  // K slices of split_stages stages (an even number)
  int vec;                   // rows of d are 16-byte aligned
};

// A workgroup's tile: four waves, each half of its rows and columns.
template <int kTM>
struct Fp4Tile {
  static constexpr int kBM = kTM, kBN = kTileN;
  static constexpr int kBI = kTM / 64, kBJ = kTileN / 64;          // 32-row blocks of a wave
  static constexpr int kLoadsA = kTM / 32, kLoadsB = kTileN / 32;  // 1 KB loads per wave and chunk
  static constexpr int kScales = kBI + kBJ;                        // scale loads per wave and two stages
};

// acc += (b * 2^(sb - 127)) (a * 2^(sa - 127))^T over a block of each half of the lanes; the scales are byte kByte. Written as
// assembly with the sum in place (see gemm_fp8.hip), in the accumulation registers: two wait states between a vector
// instruction's write of an operand and its read (s_nop), and mfma_drain before the sums are read.
template <int kByte>
MXQ_DEVICE void mfma_fp4(v16f& acc, v4i b, v4i a, uint32_t sb, uint32_t sa) {
  if constexpr (kByte == 0)
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else if constexpr (kByte == 1)
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else if constexpr (kByte == 2)
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
}

// A wave's scale words of two stages, its rows' and its columns', as loaded.
template <class C>
struct WordPairs {
  v2u a[C::kBI], b[C::kBJ];
};
template <class C>
struct ScaleSource {
  const uint8_t *a, *b;
  int bytes_a, bytes_b, row_tiles;
  uint32_t off_a, off_b;  // of the wave's first 32 rows; the next ones are row_tiles further on
};
MXQ_DEVICE v2u buffer_load_x2(const void* base, int bytes, uint32_t voff, int soff) {
  return __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(
                                     __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, kRawBufferWord3),
                                     (int)voff, soff, 0));
}
// Scale load t: of the 32-row blocks of A, then of B.
template <class C, int kT>
MXQ_DEVICE void load_scale(const ScaleSource<C>& s, int stage, WordPairs<C>& w) {
  const int at = (stage >> 1) * (int)kFp4ScaleTile;
  if constexpr (kT < C::kBI)
    w.a[kT] = buffer_load_x2(s.a, s.bytes_a, s.off_a, at + kT * s.row_tiles);
  else
    w.b[kT - C::kBI] = buffer_load_x2(s.b, s.bytes_b, s.off_b, at + (kT - C::kBI) * s.row_tiles);
}

// The whole main loop of a wave over stages [0, n). The operand chunks A_0 B_0 A_1 B_1 ... go to slot (chunk index) % 5. A stage is
// four steps, one block of each half of the lanes (pieces 4 (l / 32) + step of a row's 128 bytes); a step is kBI * 4 slots, each
// one matrix instruction and a part of the other work in the order written (sched_barrier): the fragments of the next step, one
// ahead; during steps 0 and 1 the loads of A_s+2 into B_s-1's slot; during step 2 of every other stage the scale words of the next
// two; then, ahead of step 3, whose reads are the next stage's, the wait for that stage and the workgroup's barrier, behind which
// nobody reads this one; and during step 3 the loads of B_s+2 into A_s's slot.
template <class C>
MXQ_DEVICE void main_loop(char* lds, const Chunk<C::kLoadsA>& ca, const Chunk<C::kLoadsB>& cb, const ScaleSource<C>& ss,
                          int n, int wrow, int wcol, int lane, v16f (&acc)[C::kBI][C::kBJ]) {
  constexpr int kSlots = C::kBI * C::kBJ, kReads = C::kBI + C::kBJ;
  constexpr int kReadSlots = kSlots * 3 / 4;  // the reads end early: the next step's first instruction waits for them
  const uint32_t base = lds_addr(lds);
  WordPairs<C> cur, next;
  static_for<C::kScales>([&](auto T) { load_scale<C, decltype(T)::value>(ss, 0, next); });
  __builtin_amdgcn_sched_barrier(0);
  issue_chunk(ca, lds, 0, true);
  issue_chunk(cb, lds + kSlot, 0, true);
  issue_chunk(ca, lds + 2 * kSlot, 1, n > 1);
  issue_chunk(cb, lds + 3 * kSlot, 1, n > 1);
  if (n > 1)
    wait_vmcnt<C::kLoadsA + C::kLoadsB>();
  else
    wait_vmcnt<0>();
  phase_barrier();
  // The 16 bytes of row (l % 32) of a 32-row block that a lane feeds step j.
  uint32_t piece[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) piece[j] = base + (uint32_t)((lane & 31) * kStageK + ((((lane >> 5) * 4 + j) ^ swizzle(lane & 31)) << 4));
  v4i fa[2][C::kBI], fb[2][C::kBJ];
  auto read = [&](auto SetC, auto IC, uint32_t at_a, uint32_t at_b) {  // in the order of their use: A_0, B_0 .., A_1 ..
    constexpr int kSet = decltype(SetC)::value, kI = decltype(IC)::value;
    if constexpr (kI == 0)
      fa[kSet][0] = lds_read_b128<0>(at_a);
    else if constexpr (kI <= C::kBJ)
      fb[kSet][kI - 1] = lds_read_b128<(kI - 1) * 32 * kStageK>(at_b);
    else
      fa[kSet][kI - C::kBJ] = lds_read_b128<(kI - C::kBJ) * 32 * kStageK>(at_a);
  };
  const uint32_t row_a = (uint32_t)(wrow * kStageK), row_b = (uint32_t)(wcol * kStageK);
  static_for<kReads>([&](auto I) { read(std::integral_constant<int, 0>{}, I, piece[0] + row_a, piece[0] + row_b + kSlot); });
  auto take = [&] {  // the words requested two stages ago
#pragma unroll
    for (int i = 0; i < C::kBI; ++i) {
      cur.a[i] = next.a[i];
      __asm__ volatile("" : "+v"(cur.a[i]));
    }
#pragma unroll
    for (int j = 0; j < C::kBJ; ++j) {
      cur.b[j] = next.b[j];
      __asm__ volatile("" : "+v"(cur.b[j]));
    }
  };
  take();

  int sa = 0;  // slot of A_s; B_s is in the next one
  // kSecond: the second of two stages; kSteady: stages s + 1 and s + 2 (and the second's next words) exist
  auto stage = [&](int s, auto SecondC, auto SteadyC) {
    constexpr int kP = decltype(SecondC)::value;
    constexpr bool kSteady = decltype(SteadyC)::value;
    const int sb = sa == kRing - 1 ? 0 : sa + 1;
    const int na = sb == kRing - 1 ? 0 : sb + 1;
    const int nb = na == kRing - 1 ? 0 : na + 1;
    const int pa = sa == 0 ? kRing - 1 : sa - 1;
    const bool more = kSteady || s + 2 < n;
    static_for<4>([&](auto H) {
      constexpr int h = decltype(H)::value, kSet = h & 1;
      if constexpr (h == 3) {
        // stage s + 1 has landed: only A_s+2 and the words (when there are any) were issued after it
        if constexpr (kSteady)
          wait_vmcnt<C::kLoadsA + (kP == 0 ? C::kScales : 0)>();
        else
          wait_vmcnt<0>();
      }
      wait_lgkm<0>();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (h == 3) phase_barrier();
      const uint32_t at = piece[(h + 1) & 3];
      const uint32_t at_a = at + row_a + (uint32_t)((h < 3 ? sa : na) * kSlot), at_b = at + row_b + (uint32_t)((h < 3 ? sb : nb) * kSlot);
      static_for<kSlots>([&](auto G) {
        constexpr int g = decltype(G)::value, i = g / C::kBJ, j = g % C::kBJ;
        mfma_fp4<h>(acc[i][j], fb[kSet][j], fa[kSet][i], cur.b[j][kP], cur.a[i][kP]);
        static_for<kReads>([&](auto I) {
          if constexpr (decltype(I)::value * kReadSlots / kReads == g) read(std::integral_constant<int, kSet ^ 1>{}, I, at_a, at_b);
        });
        if constexpr (h < 2) {
          constexpr int kHalf = C::kLoadsA / 2;
          static_for<kHalf>([&](auto T) {
            if constexpr (decltype(T)::value * kSlots / kHalf == g)
              if (more) issue_load(ca, lds + pa * kSlot, s + 2, h * kHalf + decltype(T)::value);
          });
        } else if constexpr (h == 2 && kP == 0) {
          static_for<C::kScales>([&](auto T) {
            if constexpr (decltype(T)::value * kSlots / C::kScales == g)
              if (more) load_scale<C, decltype(T)::value>(ss, s + 2, next);
          });
        } else if constexpr (h == 3) {
          static_for<C::kLoadsB>([&](auto T) {
            if constexpr (decltype(T)::value * kSlots / C::kLoadsB == g)
              if (more) issue_load(cb, lds + sa * kSlot, s + 2, decltype(T)::value);
          });
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    sa = na;
  };
  const std::integral_constant<int, 0> first{};
  const std::integral_constant<int, 1> second{};
  int s = 0;
  for (; s + 3 < n; s += 2) {
    stage(s, first, std::true_type{});
    stage(s + 1, second, std::true_type{});
    take();
  }
  for (; s < n; s += 2) {
    stage(s, first, std::false_type{});
    if (s + 1 < n) stage(s + 1, second, std::false_type{});
    take();
  }
  wait_lgkm<0>();  // (the last step's reads, of slots nobody uses)
#pragma unroll
  for (int i = 0; i < C::kBI; ++i) __asm__ volatile("" ::"v"(fa[0][i]));
#pragma unroll
  for (int j = 0; j < C::kBJ; ++j) __asm__ volatile("" ::"v"(fb[0][j]));
  mfma_drain();
  phase_barrier();
}

// ---- the tile of 128 x 128 ----
// For problems of few tiles, whose time is that of one workgroup's stages one after the other: four waves of 64 x 64. A stage is 256
// bytes of each row, 512 columns (one scale tile wide), so that the ring of five 32 KB slots reaches as far ahead in time as
// with the larger tiles; chunk rows are 256 bytes, 16-byte piece c of row r at piece c ^ (r & 15). Rows of B are zero-padded to
// whole stages; A's are to half of one, and in place of the half behind them a last stage reads the half before it again:
// every code is a finite number, whose products with B's zeros are zeros.
struct Fp4Small {
  static constexpr int kBM = 128, kBN = 128, kBI = 2, kBJ = 2;
  static constexpr int kRow = 256, kLoads = 8;  // bytes of a chunk's row, 1 KB loads per wave and chunk
  static constexpr int kScales = kBI + kBJ;
};

struct WideChunk {
  const uint8_t* base;
  int bytes;
  uint32_t off[Fp4Small::kLoads], back;  // back: bit t % 4 is set where load t's piece is in the second half of the row
  int wave;
};
MXQ_DEVICE WideChunk make_wide_chunk(const uint8_t* p, int64_t ld, int row0, int rows, int wave, int lane) {
  WideChunk c;
  const int valid = min(rows - row0, 128);
  c.base = p + row0 * ld;
  c.bytes = valid * (int)ld;
  c.wave = wave;
  c.back = 0;
#pragma unroll
  for (int t = 0; t < Fp4Small::kLoads; ++t) {
    const int r = (wave * Fp4Small::kLoads + t) * 4 + (lane >> 4), piece = (lane & 15) ^ (r & 15);
    c.off[t] = (uint32_t)(min(r, valid - 1) * (int)ld + (piece << 4));
    if (t < 4) c.back |= (uint32_t)(piece >> 3) << t;
  }
  return c;
}
MXQ_DEVICE void issue_wide(const WideChunk& c, char* slot, int stage, bool half, int t) {
  const uint32_t off = c.off[t] - (half ? ((c.back >> (t & 3)) & 1u) << 7 : 0u);
  buffer_load_lds16(c.base, c.bytes, (lptr_t)(slot + (c.wave * Fp4Small::kLoads + t) * 1024), off, stage * Fp4Small::kRow);
}

// As main_loop, with steps of two blocks; the scale words are requested two stages ahead, in two sets. half: the last stage of A is
// half of one.
MXQ_DEVICE void main_loop_small(char* lds, const WideChunk& ca, const WideChunk& cb, const ScaleSource<Fp4Small>& ss, int n, bool half,
                                int wrow, int wcol, int lane, v16f (&acc)[2][2]) {
  typedef Fp4Small C;
  constexpr int kSlots = 8, kReads = 8, kReadSlots = 6;
  const uint32_t base = lds_addr(lds);
  WordPairs<C> cur, next[2];
  auto words = [&](int s, WordPairs<C>& w) { static_for<C::kScales>([&](auto T) { load_scale<C, decltype(T)::value>(ss, 2 * s, w); }); };
  auto chunk = [&](const WideChunk& c, char* slot, int s, bool h) {
#pragma unroll
    for (int t = 0; t < C::kLoads; ++t) issue_wide(c, slot, s, h, t);
  };
  words(0, next[0]);
  words(n > 1 ? 1 : 0, next[1]);
  __builtin_amdgcn_sched_barrier(0);
  chunk(ca, lds, 0, half && n == 1);
  chunk(cb, lds + kSlot, 0, false);
  if (n > 1) {
    chunk(ca, lds + 2 * kSlot, 1, half && n == 2);
    chunk(cb, lds + 3 * kSlot, 1, false);
    wait_vmcnt<2 * C::kLoads>();
  } else {
    wait_vmcnt<0>();
  }
  phase_barrier();
  // The 16 bytes of row (l % 32) of a 32-row block that a lane feeds for block b of its eight (word b / 4, byte b % 4).
  uint32_t piece[8];
#pragma unroll
  for (int b = 0; b < 8; ++b)
    piece[b] = base + (uint32_t)((lane & 31) * C::kRow + ((((b >> 2) * 8 + (lane >> 5) * 4 + (b & 3)) ^ (lane & 15)) << 4));
  v4i fa[2][2][2], fb[2][2][2];  // [set][block of the step][32 rows]
  const uint32_t row_a = (uint32_t)(wrow * C::kRow), row_b = (uint32_t)(wcol * C::kRow);
  auto read = [&](auto SetC, auto IC, uint32_t p0, uint32_t p1, uint32_t slot_a, uint32_t slot_b) {
    constexpr int kSet = decltype(SetC)::value, kI = decltype(IC)::value, t = kI >> 2, k = kI & 3;
    const uint32_t at = t ? p1 : p0;
    if constexpr (k == 0)
      fa[kSet][t][0] = lds_read_b128<0>(at + slot_a);
    else if constexpr (k < 3)
      fb[kSet][t][k - 1] = lds_read_b128<(k - 1) * 32 * C::kRow>(at + slot_b);
    else
      fa[kSet][t][1] = lds_read_b128<32 * C::kRow>(at + slot_a);
  };
  static_for<kReads>([&](auto I) { read(std::integral_constant<int, 0>{}, I, piece[0], piece[1], row_a, row_b + kSlot); });

  int sa = 0;  // slot of A_s; B_s is in the next one
  auto stage = [&](int s, auto ParityC, auto SteadyC) {
    constexpr int kParity = decltype(ParityC)::value;
    constexpr bool kSteady = decltype(SteadyC)::value;
    const int sb = sa == kRing - 1 ? 0 : sa + 1;
    const int na = sb == kRing - 1 ? 0 : sb + 1;
    const int nb = na == kRing - 1 ? 0 : na + 1;
    const int pa = sa == 0 ? kRing - 1 : sa - 1;
    const bool more = kSteady || s + 2 < n, cut = half && s + 3 == n;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      cur.a[i] = next[kParity].a[i];
      cur.b[i] = next[kParity].b[i];
      __asm__ volatile("" : "+v"(cur.a[i]), "+v"(cur.b[i]));
    }
    static_for<4>([&](auto H) {
      constexpr int h = decltype(H)::value, kSet = h & 1;
      if constexpr (h == 3) {
        // stage s + 1 has landed: only the words and A_s+2 were issued after it
        if constexpr (kSteady)
          wait_vmcnt<C::kScales + C::kLoads>();
        else
          wait_vmcnt<0>();
      }
      wait_lgkm<0>();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (h == 3) phase_barrier();
      const uint32_t p0 = piece[(2 * h + 2) & 7], p1 = piece[(2 * h + 3) & 7];
      const uint32_t slot_a = row_a + (uint32_t)((h < 3 ? sa : na) * kSlot), slot_b = row_b + (uint32_t)((h < 3 ? sb : nb) * kSlot);
      static_for<kSlots>([&](auto G) {
        constexpr int g = decltype(G)::value, t = g >> 2, i = (g >> 1) & 1, j = g & 1, kBlock = 2 * h + t;
        mfma_fp4<kBlock & 3>(acc[i][j], fb[kSet][t][j], fa[kSet][t][i], cur.b[j][kBlock >> 2], cur.a[i][kBlock >> 2]);
        static_for<kReads>([&](auto I) {
          if constexpr (decltype(I)::value * kReadSlots / kReads == g)
            read(std::integral_constant<int, kSet ^ 1>{}, I, p0, p1, slot_a, slot_b);
        });
        if constexpr (h == 0 && g < C::kScales) {
          if (more) load_scale<C, (g < C::kScales ? g : 0)>(ss, 2 * (s + 2), next[kParity]);
        }
        if constexpr (h < 2 && (g & 1)) {
          if (more) issue_wide(ca, lds + pa * kSlot, s + 2, cut, h * 4 + (g >> 1));
        } else if constexpr (h == 3) {
          if (more) issue_wide(cb, lds + sa * kSlot, s + 2, false, g);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    sa = na;
  };
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> odd{};
  int s = 0;
  for (; s + 3 < n; s += 2) {
    stage(s, even, std::true_type{});
    stage(s + 1, odd, std::true_type{});
  }
  for (; s < n; s += 2) {
    stage(s, even, std::false_type{});
    if (s + 1 < n) stage(s + 1, odd, std::false_type{});
  }
  wait_lgkm<0>();  // (the last step's reads, of slots nobody uses)
#pragma unroll
  for (int i = 0; i < 2; ++i) __asm__ volatile("" ::"v"(fa[0][0][i]), "v"(fa[0][1][i]), "v"(fb[0][0][i]), "v"(fb[0][1][i]));
  mfma_drain();
  phase_barrier();
}

// kTM: rows of the tile, which has 256 columns; 0: the tile of 128 x 128.
template <int kTM, int kOut, bool kSplit>
__global__ __launch_bounds__(256, 1) void gemm_mxfp4_kernel(Fp4Gemm p) {
  typedef std::conditional_t<kTM == 0, Fp4Small, Fp4Tile<kTM == 0 ? 128 : kTM>> C;
  __shared__ __attribute__((aligned(1024))) char lds[kGemmLds];
  int tm, tn, slice;
  tile_of(blockIdx.x, p, tm, tn, slice);
  const int M = (int)p.M, N = (int)p.N, m0 = tm * C::kBM, n0 = tn * C::kBN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wrow = (wave >> 1) * (C::kBM / 2), wcol = (wave & 1) * (C::kBN / 2);
  const int first = slice * p.split_stages, n = min(p.split_stages, p.stages - first);
  const uint8_t *a = p.a + (int64_t)first * kStageK, *b = p.b + (int64_t)first * kStageK;
  // (a row of scale tiles holds 32 rows; behind the operands' last one, reads give zeros)
  ScaleSource<C> ss;
  const int row_tiles = p.groups * (int)kFp4ScaleTile, skip = (first >> 1) * (int)kFp4ScaleTile;
  ss.a = p.sa + (int64_t)(m0 >> 5) * row_tiles + skip;
  ss.b = p.sb + (int64_t)(n0 >> 5) * row_tiles + skip;
  ss.bytes_a = ((min(M - m0, C::kBM) + 31) >> 5) * row_tiles - skip;
  ss.bytes_b = ((min(N - n0, C::kBN) + 31) >> 5) * row_tiles - skip;
  ss.row_tiles = row_tiles;
  ss.off_a = (uint32_t)((wrow >> 5) * row_tiles + lane * 8);
  ss.off_b = (uint32_t)((wcol >> 5) * row_tiles + lane * 8);
  v16f acc[C::kBI][C::kBJ] = {};
  if constexpr (kTM == 0)
    main_loop_small(lds, make_wide_chunk(a, p.lda, m0, M, wave, lane), make_wide_chunk(b, p.ldb, n0, N, wave, lane), ss, (n + 1) >> 1,
                    n & 1, wrow, wcol, lane, acc);
  else
    main_loop<C>(lds, make_chunk<C::kLoadsA, 4>(a, p.lda, m0, M, wave, lane), make_chunk<C::kLoadsB, 4>(b, p.ldb, n0, N, wave, lane), ss, n,
                 wrow, wcol, lane, acc);
  void* d = p.d;
  if constexpr (kSplit) d = reinterpret_cast<float*>(p.d) + slice * p.M * p.ldd;
  epilogue<C, kOut, kSplit>(p, lds, acc, m0, n0, wrow, wcol, wave, lane, d);
}

// ---- host side ----

struct Fp4Plan {
  int tile, splits, split_stages;  // tile: rows, 0 for the tile of 128 x 128
  double cost;
};

static int64_t tile_rows(int tile, int64_t M) { return (M + (tile ? tile : 128) - 1) / (tile ? tile : 128); }
static int64_t tile_cols(int tile, int64_t N) { return (N + (tile ? 256 : 128) - 1) / (tile ? 256 : 128); }
static int64_t tiles_of(int tile, int64_t M, int64_t N) { return tile_rows(tile, M) * tile_cols(tile, N); }

// Tile and K slices, by an estimate in microseconds: a round of workgroups takes 6 (256 x 256) or 4.5 (128 x 256, 128 x 128) for its
// first loads and its epilogue and, per 256 columns of K, 0.94, 0.64 or 0.36 where few CUs are at work, 1.6, 1.0 or 0.47 (power)
// where all are; all rounds take at least the weight's bytes, slices cost a join. Measured, with the layout's launch, whole and in
// the best number of slices, 128 x 128 / 128 x 256 / 256 x 256: 100 rows, K 5120, N 5120: 15.9 / 22.5, 20 / 31; 700 rows: 17.7 / 23.2 /
// 31.9; 1024 rows 28.5 / 23.2 / 31.1; 3000 rows 55 / 47 / 42.5; 8192 rows, K 20480: 463 / 408 / 375; 200 rows, K 20480, N 5120: 38.1,
// 26.0 in three / 60.7, 28.6 in five / 88; 1024 rows, K 5000, N 2049: 20.2 / 26.3 / 39.2.
static Fp4Plan plan_fp4(int64_t M, int64_t N, int64_t stages, int cus) {
  Fp4Plan best = {256, 1, (int)((stages + 1) / 2 * 2), 1e300};
  const double stream = (double)(N * stages) * 136.0 / 4.9e6 + 2.0;
  for (const int tile : {256, 128, 0}) {
    const int64_t tiles = tiles_of(tile, M, N);
    const double alone = tile == 256 ? 0.94 : tile ? 0.64 : 0.36, all = tile == 256 ? 1.6 : tile ? 1.0 : 0.47;
    const double ends = tile == 256 ? 6.0 : 4.5;
    for (int64_t s = 1; s <= 32; ++s) {
      const int64_t per = ((stages + s - 1) / s + 1) / 2 * 2, splits = (stages + per - 1) / per;
      if (splits != s || (s > 1 && tiles * s > 4 * cus)) continue;
      const double n = (double)(per < stages ? per : stages);
      const int64_t full = tiles * s / cus;
      const double rest = (double)(tiles * s % cus) / cus;
      double cost = (double)full * (n * all + ends) + (rest > 0.0 ? n * (alone + (all - alone) * rest) + ends : 0.0);
      if (cost < stream) cost = stream;
      cost += slices_cost(s, M * N);
      if (cost < best.cost) best = {tile, (int)s, (int)per, cost};
    }
  }
  return best;
}

Fp4TileForm fp4_gemm_form(int64_t M, int64_t N, int64_t K) {
  const Fp4Plan plan = plan_fp4(M, N, fp4_row_bytes(K) / kFp4Stage, mxq_cu_count());
  return {plan.tile ? plan.tile : 128, plan.tile ? 256 : 128, plan.splits};
}

}  // namespace mxq

using namespace mxq;

static bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int mxq::fp4_gemm_check(const uint8_t* a, int64_t lda, const uint8_t* sa, const uint8_t* b, int64_t ldb, const uint8_t* sb,
                        const void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K) {
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 1 || K < 1 || M > (1ll << 31) - 1024 || N > (1ll << 22) || K > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  const int64_t bytes = fp4_row_bytes(K);
  if (ldb < fp4_weight_bytes(K) || ldb % 16 || ldb > (1ll << 22) || ldd < N)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the weight or the output for N=%lld K=%lld", (long long)N, (long long)K);
  if (lda < bytes || lda % 16 || lda > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the activations for K=%lld", (long long)K);
  if (M == 0) return MXQ_OK;
  // (counted in tiles of 256 x 256; of the plan's other tiles there are up to four times as many, fewer than 2^24 workgroups of 256
  // threads, and a launch takes less than 2^32 threads. So many tiles are not split.)
  if ((M + 255) / 256 * ((N + kTileN - 1) / kTileN) >= (1ll << 22)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 2^22 tiles");
  if (!a || !sa || !b || !sb || !d || !aligned(a, 16) || !aligned(b, 16) || !aligned(sa, 16) || !aligned(sb, 16))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  return MXQ_OK;
}

template <int kTM, int kOut, bool kSplit>
static int launch_gemm(const Fp4Gemm& p, void* stream) {
  hipLaunchKernelGGL((gemm_mxfp4_kernel<kTM, kOut, kSplit>), dim3((unsigned)(p.tiles_m * p.tiles_n * p.splits)), dim3(256), 0,
                     (hipStream_t)stream, p);
  return mxq_check_launch("gemm_mxfp4_kernel");
}

static int64_t split_bytes(const Fp4Plan& plan, int64_t M, int64_t N) {
  return plan.splits > 1 ? plan.splits * M * ((N + 3) / 4 * 4) * 4 : 0;
}

extern "C" int mxq_mxfp4_gemm_workspace(int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (M < 0 || N < 1 || K < 1 || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  *bytes = M == 0 ? 0 : split_bytes(plan_fp4(M, N, fp4_row_bytes(K) / kFp4Stage, mxq_cu_count()), M, N);
  return MXQ_OK;
}

extern "C" int mxq_mxfp4_gemm(const uint8_t* a, int64_t lda, const uint8_t* sa, const uint8_t* b, int64_t ldb, const uint8_t* sb,
                              const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (const int rc = fp4_gemm_check(a, lda, sa, b, ldb, sb, d, ldd, out_dtype, M, N, K)) return rc;
  if (M == 0) return MXQ_OK;
  const int64_t stages = fp4_row_bytes(K) / kFp4Stage;
  const Fp4Plan plan = plan_fp4(M, N, stages, mxq_cu_count());
  const int64_t tiles_m = tile_rows(plan.tile, M), tiles_n = tile_cols(plan.tile, N);
  const int64_t need = split_bytes(plan, M, N);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  Fp4Gemm p = {a, b, sa, sb, bias, d, M, N, lda, ldb, ldd, (int)fp4_groups(K), (int)stages, (int)tiles_m, (int)tiles_n, plan.splits,
               plan.split_stages, 0};
  if (plan.splits > 1) {
    const int64_t ldp = (N + 3) / 4 * 4;
    p.d = workspace;
    p.ldd = ldp;
    p.vec = 1;
    p.bias = nullptr;
    const int rc = plan.tile == 256 ? launch_gemm<256, 0, true>(p, stream)
                   : plan.tile      ? launch_gemm<128, 0, true>(p, stream)
                                    : launch_gemm<0, 0, true>(p, stream);
    if (rc) return rc;
    return fp8_join({(const float*)workspace, bias, d, M, ldp, ldd, (int)N, plan.splits, out_dtype}, {}, {}, stream);
  }
  p.vec = aligned(d, 16) && ldd * dtype_bytes(out_dtype) % 16 == 0;
  return with_dtype(out_dtype, [&](auto O) {
    constexpr int kOut = decltype(O)::value;
    return plan.tile == 256 ? launch_gemm<256, kOut, false>(p, stream)
           : plan.tile      ? launch_gemm<128, kOut, false>(p, stream)
                            : launch_gemm<0, kOut, false>(p, stream);
  });
}
