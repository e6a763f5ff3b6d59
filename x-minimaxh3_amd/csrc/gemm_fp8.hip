// Matrix product of block-128 e4m3 operands (fp8_common.h) on gfx950 matrix cores:
//
//   D[m, n] = out( sum_b 2^(ea[m, b] + eb[n / 128, b]) * sum_{k in block b} A[m, k] * B[n, k]  +  bias[n] )
//
// A [M, K] activations (or output gradients) with one scale per row and block, B [N, K] a weight (or its transposed
// copy) with one per 128 x 128 tile; both K-contiguous, rows zero-padded to whole blocks. Sums are float32.
//
// Main loop: a workgroup of eight waves (two per SIMD) owns a 256 x 256 (or 128 x 256) output tile, a wave 128 x 64 (or
// 64 x 64) of it. A stage is one block of 128 K-bytes; its A and B chunks are fetched by direct-to-LDS loads into a
// ring of five 32 KB slots, one to two stages ahead. The two waves of a SIMD take turns: one issues the matrix
// instructions of a half stage while the other reads its next fragments and issues loads. v_mfma_scale_f32_32x32x64_
// f8f6f4 applies the scales itself: each lane gives one byte for its row, so a block's scale costs the loop nothing but
// four words per four stages and wave (a byte per stage, shifted out of a word).
//
// Precision of that instruction, measured: within one 64-long product sum, addends are cut below 2^-13 of the largest,
// and the sum is added to a float32. How much that is depends on the data: on the layers' own 5e-5 to 2e-4 of the result's
// root mean square, beside bfloat16's and float16's rounding of 1.7e-3 and 2.1e-4; at worst, one product beside 63 of its
// own sign just under 2^-13 of it, 63 * 2^-13 (0.8 %) of the result. 16-bit results take it for its rate. For float32
// results, and 16-bit ones that are asked for with full sums (kWide), the fragments are converted to bfloat16 with their
// scales, exactly, and the sums run on v_mfma_f32_32x32x16_bf16, which keeps every addend to float32's precision at half
// the rate.
//
// 75600 x 5120 of K 5120 takes 1.57 to 1.63 ms (2.5 PFLOP/s; 2.67 in the loop, from K 5120 against 10240 at 16384 x 4096):
// the clock falls to about 1.85 GHz, power bounds it (a library's product 2.81).
//
// Problems of few tiles split K over workgroups, which write float32 sums that fp8_join_kernel adds in order.

#include <algorithm>
#include <cmath>

#include "gemm_tiles.h"

namespace mxq {

struct Fp8Gemm {
  const uint8_t* a;
  const uint8_t* b;
  const uint8_t* sa;
  const uint8_t* sb;
  const void* bias;
  void* d;  // split: float32 sums, slice s at s * M * N
  int64_t M, N, lda, ldb, ldsa, ldsb, ldd;
  int kb;                  // blocks of K
  int tiles_m, tiles_n;
  int splits, split_kb;    // K slices of split_kb blocks (a multiple of 4)
  int vec;                 // rows of d are 16-byte aligned
};

// The 32 bytes of each of kCount 32-row blocks that a lane feeds the matrix instruction of half stage `half`: row
// l % 32, pieces 4 half + l / 32 and 4 half + 2 + l / 32. (Both operands take the same bytes of K, in any order: a
// block has one scale.)
template <int kCount>
MXQ_DEVICE void read_frags(uint32_t slot, int row, int lane, int half, v8i (&f)[kCount]) {
  const int lr = lane & 31, c = half * 4 + (lane >> 5);
  const uint32_t at = slot + (uint32_t)((row + lr) * kStageK);
  const uint32_t x0 = at + (uint32_t)((c ^ swizzle(lr)) << 4), x1 = at + (uint32_t)(((c + 2) ^ swizzle(lr)) << 4);
  static_for<kCount>([&](auto I) {
    constexpr int i = decltype(I)::value;
    f[i] = join8(lds_read_b128<i * 32 * kStageK>(x0), lds_read_b128<i * 32 * kStageK>(x1));
  });
}

// acc += (b * 2^(sb - 127)) (a * 2^(sa - 127))^T over 64 bytes of K; the scales are the low bytes. Written as assembly
// with the sum in place: the builtin's result may be another register tuple than its addend, and the 256-row tile then
// spilled its accumulators (660 registers). What the compiler would look after is done here: two wait states between a
// vector instruction's write of an operand and its read (s_nop), and mfma_drain before the sums are read.
MXQ_DEVICE void mfma_scaled(v16f& acc, v8i b, v8i a, uint32_t sb, uint32_t sa) {
  __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                   : "+v"(acc)
                   : "v"(b), "v"(a), "v"(sb), "v"(sa));
}
// The matrix instructions of a half stage. They compute D^T blocks (B first): lane l holds row l % 32 of D and, in
// register r, column (r / 4) * 8 + (l / 32) * 4 + r % 4.
template <class C, bool kWide>
MXQ_DEVICE void half_stage(const v8i (&fa)[C::kBI], const v8i (&fb)[C::kBJ], const uint32_t (&sa)[C::kBI], uint32_t sb,
                           v16f (&acc)[C::kBI][C::kBJ]) {
  if constexpr (!kWide) {
#pragma unroll
    for (int i = 0; i < C::kBI; ++i)
#pragma unroll
      for (int j = 0; j < C::kBJ; ++j)
        mfma_scaled(acc[i][j], fb[j], fa[i], sb, sa[i]);
  } else {
    const float fsb = fp8_scale_f32(sb & 0xFFu);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v8bf wb[C::kBJ];
#pragma unroll
      for (int j = 0; j < C::kBJ; ++j) wb[j] = fp8x8_to_bf16((uint32_t)fb[j][2 * q], (uint32_t)fb[j][2 * q + 1], fsb);
#pragma unroll
      for (int i = 0; i < C::kBI; ++i) {
        const v8bf xa = fp8x8_to_bf16((uint32_t)fa[i][2 * q], (uint32_t)fa[i][2 * q + 1], fp8_scale_f32(sa[i] & 0xFFu));
#pragma unroll
        for (int j = 0; j < C::kBJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j], xa, acc[i][j], 0, 0, 0);
      }
    }
  }
}

// A wave's scale words for the four stages from `stage` on (a multiple of 4): its rows' and its columns'.
template <class C>
struct Scales {
  uint32_t a[C::kBI], b;
};
template <class C>
struct ScaleSource {
  const uint8_t *a, *b;
  int bytes_a, bytes_b;
  uint32_t off[C::kBI];
};
MXQ_DEVICE uint32_t buffer_load_x1(const void* base, int bytes, uint32_t voff, int soff) {
  return __builtin_amdgcn_raw_buffer_load_b32(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, kRawBufferWord3), (int)voff, soff, 0);
}
template <class C>
MXQ_DEVICE void load_scales(const ScaleSource<C>& s, int stage, Scales<C>& w) {
#pragma unroll
  for (int i = 0; i < C::kBI; ++i) w.a[i] = buffer_load_x1(s.a, s.bytes_a, s.off[i], stage);
  w.b = buffer_load_x1(s.b, s.bytes_b, 0, stage);
}

// One group's whole main loop over stages [0, n) (kG = 0: waves 0-3, 1: waves 4-7). The operand chunks A_0 B_0 A_1
// B_1 ... go to slot (chunk index) % 5. Iteration kt has four phases, a workgroup barrier behind each; group g computes
// in phases 2 q + g and reads in the others:
//   P0  g0: first half of kt      g1: reads (kt, 0), loads A_kt+2 into B_kt-1's slot
//   P1  g1: first half            g0: reads (kt, 1), loads A_kt+2
//   P2  g0: second half           g1: reads (kt, 1)          both then wait for stage kt+1
//   P3  g1: second half + loads   g0: reads (kt+1, 0), loads B_kt+2 into A_kt's slot
//       of B_kt+2
// The scale words of stages 4 g .. 4 g + 3 are requested with the B loads of iteration 4 g - 2, so the next
// iteration's wait covers them.
template <class C, int kG, bool kWide>
MXQ_DEVICE void main_loop(char* lds, const Chunk<C::kLoadsA>& ca, const Chunk<C::kLoadsB>& cb, const ScaleSource<C>& ss,
                          int n, int wrow, int wcol, int lane, v16f (&acc)[C::kBI][C::kBJ]) {
  const uint32_t base = lds_addr(lds);
  auto slot_addr = [&](int s) { return base + (uint32_t)(s * kSlot); };
  Scales<C> cur, next;
  load_scales(ss, 0, cur);
  __builtin_amdgcn_sched_barrier(0);
  issue_chunk(ca, lds, 0, true);
  issue_chunk(cb, lds + kSlot, 0, true);
  issue_chunk(ca, lds + 2 * kSlot, 1, n > 1);
  issue_chunk(cb, lds + 3 * kSlot, 1, n > 1);
  if (n > 1)
    wait_vmcnt<C::kLoadsA + C::kLoadsB>();
  else
    wait_vmcnt<0>();
#pragma unroll
  for (int i = 0; i < C::kBI; ++i) __asm__ volatile("" : "+v"(cur.a[i]));
  __asm__ volatile("" : "+v"(cur.b));
  next = cur;
  phase_barrier();
  v8i fa[C::kBI], fb[C::kBJ];
  if constexpr (kG == 0) {
    read_frags<C::kBI>(slot_addr(0), wrow, lane, 0, fa);
    read_frags<C::kBJ>(slot_addr(1), wcol, lane, 0, fb);
    wait_lgkm<0>();
  }
  phase_barrier();

  int sa = 0;  // slot of A_kt; B_kt is in the next one
  auto iteration = [&](int kt, auto SteadyC) {
    constexpr bool kSteady = decltype(SteadyC)::value;  // stage kt + 2 exists
    const int sb = sa == kRing - 1 ? 0 : sa + 1;
    const int na = sb == kRing - 1 ? 0 : sb + 1;
    const int nb = na == kRing - 1 ? 0 : na + 1;
    const int pa = sa == 0 ? kRing - 1 : sa - 1;
    const bool more = kSteady || kt + 2 < n;
    char* slot_pa = lds + pa * kSlot;
    char* slot_sa = lds + sa * kSlot;
    auto next_scales = [&] {
      if ((kt & 3) == 2 && more) load_scales(ss, kt + 2, next);
    };
    if constexpr (kG == 0) {
      half_stage<C, kWide>(fa, fb, cur.a, cur.b, acc);  // P0
      phase_barrier();
      read_frags<C::kBI>(slot_addr(sa), wrow, lane, 1, fa);  // P1
      read_frags<C::kBJ>(slot_addr(sb), wcol, lane, 1, fb);
      issue_chunk(ca, slot_pa, kt + 2, more);
      wait_lgkm<0>();
      phase_barrier();
      half_stage<C, kWide>(fa, fb, cur.a, cur.b, acc);  // P2
    } else {
      read_frags<C::kBI>(slot_addr(sa), wrow, lane, 0, fa);  // P0
      read_frags<C::kBJ>(slot_addr(sb), wcol, lane, 0, fb);
      issue_chunk(ca, slot_pa, kt + 2, more);
      wait_lgkm<0>();
      phase_barrier();
      half_stage<C, kWide>(fa, fb, cur.a, cur.b, acc);  // P1
      phase_barrier();
      read_frags<C::kBI>(slot_addr(sa), wrow, lane, 1, fa);  // P2
      read_frags<C::kBJ>(slot_addr(sb), wcol, lane, 1, fb);
      wait_lgkm<0>();
    }
    // stage kt + 1 has landed: only A_kt+2 (when it exists) was issued after it
    if (more)
      wait_vmcnt<C::kLoadsA>();
    else
      wait_vmcnt<0>();
    // The scale words requested an iteration ago have landed with it: the next stage's scales are taken here, ahead of
    // the next request (behind it, the compiler would wait for that one).
    Scales<C> after;
    const bool whole = (kt & 3) == 3;
#pragma unroll
    for (int i = 0; i < C::kBI; ++i) {
      after.a[i] = whole ? next.a[i] : cur.a[i] >> 8;
      __asm__ volatile("" : "+v"(after.a[i]));
    }
    after.b = whole ? next.b : cur.b >> 8;
    __asm__ volatile("" : "+v"(after.b));
    phase_barrier();
    if constexpr (kG == 0) {
      // P3 (at the last stage these reads fetch slots nobody uses)
      read_frags<C::kBI>(slot_addr(na), wrow, lane, 0, fa);
      read_frags<C::kBJ>(slot_addr(nb), wcol, lane, 0, fb);
      next_scales();
      issue_chunk(cb, slot_sa, kt + 2, more);
      wait_lgkm<0>();
    } else {
      next_scales();
      issue_chunk(cb, slot_sa, kt + 2, more);
      half_stage<C, kWide>(fa, fb, cur.a, cur.b, acc);  // P3
    }
    phase_barrier();
    cur = after;
    sa = na;
  };
  int kt = 0;
  for (; kt + 2 < n; ++kt) iteration(kt, std::true_type{});
  do {
    iteration(kt, std::false_type{});
  } while (++kt < n);
  mfma_drain();
}

template <int kTM, int kOut, bool kSplit, bool kWide>
__global__ __launch_bounds__(512, 2) void gemm_fp8_kernel(Fp8Gemm p) {
  typedef Tile<kTM> C;
  __shared__ __attribute__((aligned(1024))) char lds[kGemmLds];
  int tm, tn, slice;
  tile_of(blockIdx.x, p, tm, tn, slice);
  const int M = (int)p.M, N = (int)p.N, m0 = tm * kTM, n0 = tn * kTileN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // waves w and w + 4 share a SIMD: the two 64-column halves of quadrant w % 4
  const int wrow = ((wave & 3) >> 1) * C::kWaveM, wcol = (wave & 1) * 128 + (wave >> 2) * 64;
  const int kb0 = slice * p.split_kb, n = min(p.split_kb, p.kb - kb0);
  const auto ca = make_chunk<C::kLoadsA>(p.a + (int64_t)kb0 * kStageK, p.lda, m0, M, wave, lane);
  const auto cb = make_chunk<C::kLoadsB>(p.b + (int64_t)kb0 * kStageK, p.ldb, n0, N, wave, lane);
  ScaleSource<C> ss;
  const int rows = min(M - m0, kTM);
  ss.a = p.sa + m0 * p.ldsa + kb0;
  ss.bytes_a = rows * (int)p.ldsa - kb0;
#pragma unroll
  for (int i = 0; i < C::kBI; ++i) ss.off[i] = (uint32_t)(min(wrow + i * 32 + (lane & 31), rows - 1) * (int)p.ldsa);
  ss.b = p.sb + min((n0 + wcol) >> 7, (N - 1) >> 7) * p.ldsb + kb0;
  ss.bytes_b = (int)p.ldsb - kb0;
  v16f acc[C::kBI][C::kBJ] = {};
  if (wave < 4)
    main_loop<C, 0, kWide>(lds, ca, cb, ss, n, wrow, wcol, lane, acc);
  else
    main_loop<C, 1, kWide>(lds, ca, cb, ss, n, wrow, wcol, lane, acc);
  void* d = p.d;
  if constexpr (kSplit) d = reinterpret_cast<float*>(p.d) + slice * p.M * p.ldd;
  epilogue<C, kOut, kSplit>(p, lds, acc, m0, n0, wrow, wcol, wave, lane, d);
}

// ---- few rows (up to 32): a stream of the weight ----
// A workgroup's four or eight waves take 16 kRT weight rows and share K. Fragments go from memory straight to registers
// (a lane: row l % 16, bytes 16 (l / 16) + {0..15} and + 64 of a block), a group of kG blocks ahead of the one at work,
// are converted to bfloat16 with their scales, exactly, and multiplied by v_mfma_f32_16x16x32_bf16, so the sums keep
// float32's precision at no cost: the weight's bytes bound this kernel. kFused: the activations come in their own type
// and each wave quantizes its own K range of them, a chunk of blocks at a time, into its part of LDS (up to 16 rows:
// the 16 columns of the instruction), which saves the quantizer's launch. How many weight rows a workgroup takes
// decides (plan_rows): each workgroup quantizes, or reads, all of x again, and what counts is the CU with the most
// weight rows. Measured (bf16 in and out): K 5120, N 20480 (80 weight rows: a workgroup per CU) 1 row 19.6 us (5.4 TB/s),
// 16 rows 23.2; with 32 weight rows a workgroup 20.4 and 32.0.
struct Fp8Rows {
  const void* x;  // kFused: [M, ldx] of the input type; else e4m3 codes [M, ldx]
  const uint8_t* sx;
  const uint8_t* b;
  const uint8_t* sb;
  const void* bias;
  void* d;
  int64_t M, N, K, ldx, ldsx, ldb, ldsb, ldd;
  int kb;
  int chunk_log2, x_code;  // kFused: blocks per chunk, x's type
};

// LDS of a wave's chunk: rows of codes, 16 bytes apart in banks, then a scale byte per row and block.
__host__ MXQ_DEVICE int chunk_row(int chunk_log2) { return (128 << chunk_log2) + 16; }
__host__ MXQ_DEVICE int chunk_bytes(int M, int chunk_log2) { return (M * (chunk_row(chunk_log2) + (1 << chunk_log2)) + 15) / 16 * 16; }

// Blocks kb0 .. of all rows into the wave's chunk; blocks from `last` on are not read.
template <int kIn>
MXQ_DEVICE void quantize_chunk(const Fp8Rows& p, uint8_t* lds, int kb0, int last, int lane) {
  constexpr int kElem = kIn == MXQ_DTYPE_F32 ? 4 : 2, kBatch = kIn == MXQ_DTYPE_F32 ? 2 : 4;
  const int M = (int)p.M, log2 = p.chunk_log2, items = M << (log2 + 3), ld = chunk_row(log2);
  const int end = min(last * 128, (int)p.K);
  uint8_t* sc = lds + M * ld;
  for (int it = lane; it - lane < items; it += 64 * kBatch) {
    Piece<kIn> t[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int item = it + 64 * u, row = item >> (log2 + 3), col = kb0 * 128 + (item & ((8 << log2) - 1)) * 16;
      const int n = row < M ? end - col : 0;
      t[u] = piece_load<kIn>(reinterpret_cast<const char*>(p.x) + (n > 0 ? row * p.ldx + col : 0) * kElem, n);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int item = it + 64 * u, row = item >> (log2 + 3), piece = item & ((8 << log2) - 1);
      const uint32_t byte = block_scale_byte(t[u]);
      const v4u c = piece_encode(t[u], fp8_scale_f32(byte));
      if (row < M) {
        *reinterpret_cast<v4u*>(lds + row * ld + piece * 16) = c;
        if ((piece & 7) == 0) sc[(row << log2) + (piece >> 3)] = (uint8_t)byte;
      }
    }
  }
  wave_lds_fence();
}

// Blocks per group; a chunk holds two groups.
constexpr int rows_group(int mt, int rt) { return mt == 1 && rt <= 2 ? 2 : 1; }

template <int kMT, int kRT, bool kFused>
struct RowsBlock {  // one block's operands of a wave
  v4u w[kRT][2];
  uint32_t ws[2];  // of the weight rows in the first and the second 128-row tile
  v4u x[kFused ? 1 : kMT][2];
  uint32_t xs[kFused ? 1 : kMT];
};

template <int kOut, int kMT, int kRT, bool kFused>
__global__ __launch_bounds__(512) void fp8_rows_kernel(Fp8Rows p) {
  constexpr int kG = rows_group(kMT, kRT);
  const int kW = blockDim.x >> 6;
  extern __shared__ __align__(16) uint8_t rows_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
  const int N = (int)p.N, M = (int)p.M, n0 = blockIdx.x * (16 * kRT);
  const int per = (p.kb + kW - 1) / kW, first = wave * per, last = min(first + per, p.kb);
  const int rows = min(N - n0, 16 * kRT);
  const uint8_t* wb = p.b + n0 * p.ldb;
  const int wbytes = (int)(rows * p.ldb);
  uint32_t woff[kRT];
#pragma unroll
  for (int r = 0; r < kRT; ++r) {
    const int row = r * 16 + lr;
    woff[r] = row < rows ? (uint32_t)(row * (int)p.ldb + g * 16) : kBufferOff;
  }
  const uint8_t* sw = p.sb + (n0 >> 7) * p.ldsb;
  const int64_t sw1 = ((n0 + rows - 1) >> 7) > (n0 >> 7) ? p.ldsb : 0;
  uint8_t* chunk = rows_lds + (kFused ? wave * chunk_bytes(M, p.chunk_log2) : 0);
  const int ld = chunk_row(p.chunk_log2), chunk_mask = (1 << p.chunk_log2) - 1;
  v4f acc[kRT][kMT] = {};
  typedef RowsBlock<kMT, kRT, kFused> Block;
  auto load = [&](Block (&t)[kG], int kb) {
#pragma unroll
    for (int u = 0; u < kG; ++u) {
      const bool in = kb + u < last;
      const int at = in ? kb + u : first;
#pragma unroll
      for (int r = 0; r < kRT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          t[u].w[r][h] = buffer_load_x4(wb, wbytes, in ? woff[r] + (uint32_t)((kb + u) * 128 + h * 64) : kBufferOff);
      t[u].ws[0] = sw[min(at, p.kb - 1)];
      if constexpr (kRT > 2) t[u].ws[1] = sw[sw1 + min(at, p.kb - 1)];
      if constexpr (!kFused) {
#pragma unroll
        for (int m = 0; m < kMT; ++m) {  // (rows behind the last are the last one again; their sums are not stored)
          const int64_t row = min(m * 16 + lr, M - 1);
          const int b = min(at, p.kb - 1);
          const uint8_t* xq = reinterpret_cast<const uint8_t*>(p.x) + row * p.ldx + b * 128 + g * 16;
          t[u].x[m][0] = *reinterpret_cast<const v4u*>(xq);
          t[u].x[m][1] = *reinterpret_cast<const v4u*>(xq + 64);
          t[u].xs[m] = p.sx[row * p.ldsx + b];
        }
      }
    }
  };
  auto compute = [&](const Block (&t)[kG], int kb) {
#pragma unroll
    for (int u = 0; u < kG; ++u) {
      if (kb + u >= last) break;
      v8bf xf[kMT][4];
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        v4u c[2] = {};
        uint32_t byte = 127;
        if constexpr (kFused) {
          const int b = (kb + u - first) & chunk_mask;
          if (lr < M) {
            c[0] = *reinterpret_cast<const v4u*>(chunk + lr * ld + b * 128 + g * 16);
            c[1] = *reinterpret_cast<const v4u*>(chunk + lr * ld + b * 128 + g * 16 + 64);
            byte = chunk[M * ld + (lr << p.chunk_log2) + b];
          }
        } else {
          c[0] = t[u].x[m][0];
          c[1] = t[u].x[m][1];
          byte = t[u].xs[m];
        }
        const float scale = fp8_scale_f32(byte);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          xf[m][2 * h] = fp8x8_to_bf16(c[h][0], c[h][1], scale);
          xf[m][2 * h + 1] = fp8x8_to_bf16(c[h][2], c[h][3], scale);
        }
      }
#pragma unroll
      for (int r = 0; r < kRT; ++r) {
        const float ws = fp8_scale_f32(kRT <= 2 || ((n0 + r * 16) >> 7) == (n0 >> 7) ? t[u].ws[0] : t[u].ws[1]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const v8bf wf = fp8x8_to_bf16(t[u].w[r][q >> 1][2 * (q & 1)], t[u].w[r][q >> 1][2 * (q & 1) + 1], ws);
#pragma unroll
          for (int m = 0; m < kMT; ++m) acc[r][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[m][q], acc[r][m], 0, 0, 0);
        }
      }
    }
  };
  Block t0[kG], t1[kG];
  load(t0, first);
  for (int kb = first; kb < last; kb += 2 * kG) {
    load(t1, kb + kG);
    if constexpr (kFused) {
      if (((kb - first) & chunk_mask) == 0) {
        const int end = min(last, kb + chunk_mask + 1);
        if (p.x_code == MXQ_DTYPE_BF16) quantize_chunk<MXQ_DTYPE_BF16>(p, chunk, kb, end, lane);
        else if (p.x_code == MXQ_DTYPE_F16) quantize_chunk<MXQ_DTYPE_F16>(p, chunk, kb, end, lane);
        else quantize_chunk<MXQ_DTYPE_F32>(p, chunk, kb, end, lane);
      }
    }
    compute(t0, kb);
    load(t0, kb + 2 * kG);
    compute(t1, kb + kG);
  }
  if constexpr (kFused) __syncthreads();  // (the sums take the chunks' place)
  v4f* part = reinterpret_cast<v4f*>(rows_lds);
#pragma unroll
  for (int r = 0; r < kRT; ++r)
#pragma unroll
    for (int m = 0; m < kMT; ++m) part[((wave * kRT + r) * kMT + m) * 64 + lane] = acc[r][m];
  __syncthreads();
  // the waves' sums in order; (r, m) pairs are dealt to the waves
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  for (int t = wave; t < kRT * kMT; t += kW) {
    const int r = t / kMT, m = t - r * kMT;
    const int row = m * 16 + lr, col = n0 + r * 16 + g * 4;
    v4f y = part[t * 64 + lane];
    for (int k = 1; k < kW; ++k) y += part[(k * kRT * kMT + t) * 64 + lane];
    if (row < M && col < N) {
      y += bias_run<kOut>(p.bias, col, N);
      const float v[4] = {y[0], y[1], y[2], y[3]};
      store_run4<kOut>(reinterpret_cast<char*>(p.d) + row * p.ldd * kElem, col, N - col, v);
    }
  }
}

// ---- host side ----

struct Fp8Plan {
  int tile, splits, split_kb;
  double cost;
};

// Tile rows and K slices, by an estimate in microseconds: a round of workgroups takes 5 for its first loads and its
// epilogue and 1.35 (256 rows) or 0.72 (128 rows) per stage, all rounds at least the weight's bytes; slices cost a join.
// Both sides measured: 1501 x 1000 of K 3001 (48 tiles) takes 14.4 + 5.9 us in slices, 21.9 us whole; 100 x 21504 of K 5376
// 28.9 + 6.3 and 38.3; 1024 x 4096 of K 5120 26.9 + 10.1 and 36.2; 1024 x 5120 of K 5120 38 us as 160 tiles of 128 rows,
// 2048 rows 60 us as 160 of 256.
static Fp8Plan plan_fp8(int64_t M, int64_t N, int64_t kb, int cus) {
  Fp8Plan best = {256, 1, (int)((kb + 3) / 4 * 4), 1e300};
  const double stream = (double)(N * kb) * 128.0 / 4.9e6 + 2.0;
  for (int tile = 256; tile >= 128; tile /= 2) {
    const int64_t tiles = (M + tile - 1) / tile * ((N + kTileN - 1) / kTileN);
    for (int64_t s = 1; s <= 32; ++s) {
      const int64_t per = ((kb + s - 1) / s + 3) / 4 * 4, splits = (kb + per - 1) / per;
      if (splits != s || (s > 1 && tiles * s > 4 * cus)) continue;
      const double rounds = (double)((tiles * s + cus - 1) / cus);
      const double stages = (double)(per < kb ? per : kb);
      double cost = rounds * (stages * (tile == 256 ? 1.35 : 0.72) + 5.0);
      if (cost < stream) cost = stream;
      cost += slices_cost(s, M * N);
      if (cost < best.cost) best = {tile, (int)s, (int)per, cost};
    }
  }
  return best;
}

// Weight rows (in sixteens) and waves of a workgroup of the few-row product, by an estimate in microseconds. The CU with
// the most workgroups (rounds) streams its weight rows, 0.086 per sixteen and block with every CU at work (less where some
// are idle), and reads x for each workgroup, 0.0052 per row and block where it quantizes them, 0.0023 from codes.
// Workgroups of four waves share a CU, so that the last round counts half; those of eight take 1 us more to start and end
// and reach more of a lone CU's rate. Measured, bf16, by 16 / 32 / 48 weight rows and four waves, 32 / 64 / 80 / 96 / 128 and
// eight: one row, K 5120, N 5120: 8.1 8.8 11.0, 9.1 12.5 15.7 18.6 23.1; N 32768: 26.5 26.9 27.2, 34.8 27.8 33.8 39.9 28.4;
// K 20480, N 5120: 25.9 24.0 33.2, 22.0 39.0 49.1 58.4 73.5; 16 rows, K 5120, N 15360: 27.6 24.3 26.2, 29.5 18.8 21.3 23.7
// 27.7; N 32768: 49.7 41.8 35.2, 57.6 35.6 41.4 46.4 31.3.
struct RowsPlan {
  int rt, waves;
  double cost;
};
static RowsPlan plan_rows(int64_t M, int64_t N, int64_t kb, int cus, bool fused) {
  RowsPlan best = {1, 4, 1e300};
  for (int waves = 4; waves <= 8; waves += 4) {
    for (const int rt : {1, 2, 3, 4, 5, 6, 8}) {
      if (waves == 4 && rt > 3) break;
      const double groups = (double)((N + 16 * rt - 1) / (16 * rt)), share = groups / cus, rounds = std::ceil(share);
      const double busy = std::min(1.0, std::max(share, waves == 4 ? 0.78 : 0.7));
      const double turns = waves == 4 && rounds > 1.0 ? (rounds + share) / 2 : rounds;
      const double cost = (waves == 4 ? 2.5 : 3.5) + turns * (double)kb * (rt * 0.086 * busy + (double)M * (fused ? 0.0052 : 0.0023));
      if (cost < best.cost) best = {rt, waves, cost};
    }
  }
  return best;
}

// Up to 16 rows always; up to 32 where the tiles would not be split or take longer (32 rows, bf16: K 5120, N 5120 13 us
// against 11.2 + 4.1; K 20480, N 5120 48 against 24 + 4.1).
bool fp8_rows_pays(int64_t M, int64_t N, int64_t K) {
  if (M <= kFp8FusedRows) return true;
  if (M > kFp8FewRows) return false;
  const int64_t kb = (K + 127) / 128;
  const int cus = mxq_cu_count();
  const Fp8Plan tiles = plan_fp8(M, N, kb, cus);
  return tiles.splits == 1 || plan_rows(M, N, kb, cus, false).cost <= tiles.cost;
}

}  // namespace mxq

using namespace mxq;

static bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <int kTM, int kOut, bool kSplit, bool kWide>
static int launch_gemm(const Fp8Gemm& p, void* stream) {
  hipLaunchKernelGGL((gemm_fp8_kernel<kTM, kOut, kSplit, kWide>), dim3((unsigned)(p.tiles_m * p.tiles_n * p.splits)), dim3(512),
                     0, (hipStream_t)stream, p);
  return mxq_check_launch("gemm_fp8_kernel");
}

static int64_t split_bytes(const Fp8Plan& plan, int64_t M, int64_t N) {
  return plan.splits > 1 ? plan.splits * M * ((N + 3) / 4 * 4) * 4 : 0;
}

// (out_dtype may carry MXQ_FP8_FULL_SUMS in what follows)
static int out_code(int out_dtype) { return out_dtype & ~MXQ_FP8_FULL_SUMS; }

static int check_product(int64_t M, int64_t N, int64_t K, int64_t ldb, int64_t ldsb, int64_t ldd, int out_dtype) {
  out_dtype = out_code(out_dtype);
  if (!float_dtype(out_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 1 || K < 1 || M > (1ll << 31) - 1024 || N > (1ll << 27) || K > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad size M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  const int64_t kb = (K + 127) / 128;
  if (ldb < kb * 128 || ldb % 16 || ldb > (1ll << 22) + 4096 || ldsb < (kb + 3) / 4 * 4 || ldsb % 4 || ldsb > (1ll << 20) ||
      ldd < N)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the weight or the output for N=%lld K=%lld", (long long)N,
                         (long long)K);
  return MXQ_OK;
}

extern "C" int mxq_fp8_gemm_workspace(int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (M < 0 || N < 1 || K < 1 || !bytes) return mxq_set_error(MXQ_ERR_INVALID, "bad argument");
  *bytes = M == 0 || fp8_rows_pays(M, N, K) ? 0 : split_bytes(plan_fp8(M, N, (K + 127) / 128, mxq_cu_count()), M, N);
  return MXQ_OK;
}

static int64_t tiles_of(const Fp8Plan& plan, int64_t M, int64_t N) {
  return (M + plan.tile - 1) / plan.tile * ((N + kTileN - 1) / kTileN) * plan.splits;
}

int mxq::fp8_gemm_check(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t ldsa, const uint8_t* b, int64_t ldb,
                        const uint8_t* sb, int64_t ldsb, const void* d, int64_t ldd, int out_dtype, int64_t M, int64_t N, int64_t K) {
  if (const int rc = check_product(M, N, K, ldb, ldsb, ldd, out_dtype)) return rc;
  const int64_t kb = (K + 127) / 128;
  if (lda < kb * 128 || lda % 16 || lda > (1ll << 22) + 4096 || ldsa < (kb + 3) / 4 * 4 || ldsa % 4 || ldsa > (1ll << 20))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the activations for K=%lld", (long long)K);
  if (M == 0) return MXQ_OK;
  if (!a || !sa || !b || !sb || !d || !aligned(a, 16) || !aligned(b, 16) || !aligned(sa, 4) || !aligned(sb, 4))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  // (so many tiles are not split; the plan is asked for only where they may be too many)
  if (tiles_of({128, 1}, M, N) >= (1ll << 23) && tiles_of(plan_fp8(M, N, kb, mxq_cu_count()), M, N) >= (1ll << 23))
    return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 2^23 tiles");
  return MXQ_OK;
}

int mxq::fp8_gemm(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t ldsa, const uint8_t* b, int64_t ldb,
                            const uint8_t* sb, int64_t ldsb, const void* bias, void* d, int64_t ldd, int out_dtype,
                            int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, SliceJob* later, void* stream) {
  if (const int rc = fp8_gemm_check(a, lda, sa, ldsa, b, ldb, sb, ldsb, d, ldd, out_dtype, M, N, K)) return rc;
  if (M == 0) return MXQ_OK;
  const int64_t kb = (K + 127) / 128;
  if (fp8_rows_pays(M, N, K))
    return fp8_linear_rows(a, MXQ_DTYPE_E4M3, lda, sa, ldsa, b, ldb, sb, ldsb, bias, d, ldd, out_dtype, M, N, K, stream);
  const Fp8Plan plan = plan_fp8(M, N, kb, mxq_cu_count());
  const int64_t tiles_m = (M + plan.tile - 1) / plan.tile, tiles_n = (N + kTileN - 1) / kTileN;
  const int64_t need = split_bytes(plan, M, N);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return mxq_set_error(MXQ_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  Fp8Gemm p = {a, b, sa, sb, bias, d, M, N, lda, ldb, ldsa, ldsb, ldd, (int)kb, (int)tiles_m, (int)tiles_n, plan.splits,
               plan.split_kb, 0};
  const bool wide = out_dtype == MXQ_DTYPE_F32 || (out_dtype & MXQ_FP8_FULL_SUMS);
  out_dtype = out_code(out_dtype);
  if (plan.splits > 1) {
    const int64_t ldp = (N + 3) / 4 * 4;
    p.d = workspace;
    p.ldd = ldp;
    p.vec = 1;
    p.bias = nullptr;
    int rc;
    if (plan.tile == 256)
      rc = wide ? launch_gemm<256, 0, true, true>(p, stream) : launch_gemm<256, 0, true, false>(p, stream);
    else
      rc = wide ? launch_gemm<128, 0, true, true>(p, stream) : launch_gemm<128, 0, true, false>(p, stream);
    if (rc) return rc;
    const SliceJob job = {(const float*)workspace, bias, d, M, ldp, ldd, (int)N, plan.splits, out_dtype};
    if (!later) return fp8_join(job, {}, {}, stream);
    *later = job;
    return MXQ_OK;
  }
  p.vec = aligned(d, 16) && ldd * dtype_bytes(out_dtype) % 16 == 0;
  return with_dtype(out_dtype, [&](auto O) {
    constexpr int kOut = decltype(O)::value;
    if constexpr (kOut != MXQ_DTYPE_F32) {
      if (!wide) return plan.tile == 256 ? launch_gemm<256, kOut, false, false>(p, stream) : launch_gemm<128, kOut, false, false>(p, stream);
    }
    return plan.tile == 256 ? launch_gemm<256, kOut, false, true>(p, stream) : launch_gemm<128, kOut, false, true>(p, stream);
  });
}

extern "C" int mxq_fp8_gemm(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t ldsa, const uint8_t* b, int64_t ldb,
                            const uint8_t* sb, int64_t ldsb, const void* bias, void* d, int64_t ldd, int out_dtype,
                            int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  return fp8_gemm(a, lda, sa, ldsa, b, ldb, sb, ldsb, bias, d, ldd, out_dtype, M, N, K, workspace, workspace_bytes, nullptr, stream);
}

template <int kOut, int kMT, int kRT, bool kFused>
static void launch_rows_of(Fp8Rows p, int waves, void* stream) {
  int bytes = kRT * kMT * 1024 * waves;
  if constexpr (kFused) {
    // chunks of a wave's whole K range where all rows' take up to 36 KB of LDS, down to two groups of blocks
    constexpr int kLeast = rows_group(kMT, kRT) == 2 ? 2 : 1;
    const int per = (p.kb + waves - 1) / waves, M = (int)p.M;
    p.chunk_log2 = kLeast;
    while (p.chunk_log2 < 6 && (1 << p.chunk_log2) < per && waves * chunk_bytes(M, p.chunk_log2 + 1) <= 36 * 1024) ++p.chunk_log2;
    bytes = std::max(bytes, waves * chunk_bytes(M, p.chunk_log2));
  }
  hipLaunchKernelGGL((fp8_rows_kernel<kOut, kMT, kRT, kFused>), dim3((unsigned)((p.N + 16 * kRT - 1) / (16 * kRT))),
                     dim3(64 * waves), bytes, (hipStream_t)stream, p);
}

template <int kOut, int kMT, bool kFused>
static void launch_rows(const Fp8Rows& p, void* stream) {
  const RowsPlan plan = plan_rows(p.M, p.N, p.kb, mxq_cu_count(), kFused);
  switch (plan.rt) {
    case 1: return launch_rows_of<kOut, kMT, 1, kFused>(p, plan.waves, stream);
    case 2: return launch_rows_of<kOut, kMT, 2, kFused>(p, plan.waves, stream);
    case 3: return launch_rows_of<kOut, kMT, 3, kFused>(p, plan.waves, stream);
    case 4: return launch_rows_of<kOut, kMT, 4, kFused>(p, plan.waves, stream);
    case 5: return launch_rows_of<kOut, kMT, 5, kFused>(p, plan.waves, stream);
    case 6: return launch_rows_of<kOut, kMT, 6, kFused>(p, plan.waves, stream);
    default: return launch_rows_of<kOut, kMT, 8, kFused>(p, plan.waves, stream);
  }
}

int mxq::fp8_linear_rows(const void* x, int x_dtype, int64_t ldx, const uint8_t* sx, int64_t ldsx, const uint8_t* b, int64_t ldb,
                         const uint8_t* sb, int64_t ldsb, const void* bias, void* d, int64_t ldd, int out_dtype, int64_t M,
                         int64_t N, int64_t K, void* stream) {
  if (const int rc = check_product(M, N, K, ldb, ldsb, ldd, out_dtype)) return rc;
  const bool fused = x_dtype != MXQ_DTYPE_E4M3;
  const int64_t kb = (K + 127) / 128;
  if (fused && !float_dtype(x_dtype)) return mxq_set_error(MXQ_ERR_INVALID, "unsupported input dtype code %d", x_dtype);
  if (fused && ldx < K)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the activations for K=%lld", (long long)K);
  if (!x || !b || !sb || !d || !aligned(b, 16)) return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  const Fp8Rows p = {x, sx, b, sb, bias, d, M, N, K, ldx, ldsx, ldb, ldsb, ldd, (int)kb, 0, x_dtype};
  with_dtype(out_code(out_dtype), [&](auto O) {
    constexpr int kOut = decltype(O)::value;
    if (fused)
      launch_rows<kOut, 1, true>(p, stream);
    else if (M <= 16)
      launch_rows<kOut, 1, false>(p, stream);
    else
      launch_rows<kOut, 2, false>(p, stream);
  });
  return mxq_check_launch("fp8_rows_kernel");
}
