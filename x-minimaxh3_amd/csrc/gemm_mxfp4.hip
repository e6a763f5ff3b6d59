// Matrix product of MXFP4 operands (mxfp4_common.h) on gfx950 matrix cores:
//
//   D[m, n] = out( sum_b 2^(ea[m, b] + eb[n, b]) * sum_{k in block b} A[m, k] * B[n, k]  +  bias[n] )
//
// A [M, K] activations, B [N, K] a weight, both with one scale per row and 32 columns, sums in float32.
//
// Main loop, as that of the 8-bit product (gemm_fp8.hip): a workgroup of eight waves (two per SIMD) owns a 256 x 256 (or 128 x
// 256) output tile, a wave 128 x 64 (or 64 x 64) of it. A stage is 128 bytes of each row, 256 columns; its A and B chunks are
// fetched by direct-to-LDS loads into a ring of five 32 KB slots, one to two stages ahead. The two waves of a SIMD take turns:
// one issues the matrix instructions of a half stage while the other reads its next fragments and issues loads.
// v_mfma_scale_f32_32x32x64_f8f6f4 takes 32 columns of a row from each lane, one block, and the lane's own scale byte for it:
// lanes 0-31 the blocks 0 .. 3 of a stage in turn, lanes 32-63 the blocks 4 .. 7, so that a lane's scales of a stage are the four
// bytes of a word, which the instruction picks from. The scale tiles hold these words lane by lane, for two stages: one
// eight-byte load a wave (512 consecutive bytes) for 32 rows and two stages.
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

// The 16 bytes (a block) of each of kCount 32-row blocks that a lane feeds the matrix instructions of half stage `half`: row
// l % 32, pieces 4 (l / 32) + 2 half and the next.
template <int kCount>
MXQ_DEVICE void read_frags(uint32_t slot, int row, int lane, int half, v4i (&f)[kCount][2]) {
  const int lr = lane & 31, c = (lane >> 5) * 4 + half * 2;
  const uint32_t at = slot + (uint32_t)((row + lr) * kStageK);
  const uint32_t x0 = at + (uint32_t)((c ^ swizzle(lr)) << 4), x1 = at + (uint32_t)(((c + 1) ^ swizzle(lr)) << 4);
  static_for<kCount>([&](auto I) {
    constexpr int i = decltype(I)::value;
    f[i][0] = lds_read_b128<i * 32 * kStageK>(x0);
    f[i][1] = lds_read_b128<i * 32 * kStageK>(x1);
  });
}

// acc += (b * 2^(sb - 127)) (a * 2^(sa - 127))^T over a block of each half of the lanes; the scales are byte kByte. Written as
// assembly with the sum in place (see gemm_fp8.hip): two wait states between a vector instruction's write of an operand and
// its read (s_nop), and mfma_drain before the sums are read.
template <int kByte>
MXQ_DEVICE void mfma_fp4(v16f& acc, v4i b, v4i a, uint32_t sb, uint32_t sa) {
  if constexpr (kByte == 0)
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+v"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else if constexpr (kByte == 1)
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+v"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else if constexpr (kByte == 2)
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                     : "+v"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else
    __asm__ volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                     : "+v"(acc)
                     : "v"(b), "v"(a), "v"(sb), "v"(sa));
}

// A wave's scale words of a stage: its rows' and its columns'.
template <class C>
struct Words {
  uint32_t a[C::kBI], b[C::kBJ];
};
// ... and of two stages, as loaded.
template <class C>
struct WordPairs {
  v2u a[C::kBI], b[C::kBJ];
};

// The matrix instructions of a half stage. They compute D^T blocks (B first): lane l holds row l % 32 of D and, in
// register r, column (r / 4) * 8 + (l / 32) * 4 + r % 4.
template <class C, int kHalf>
MXQ_DEVICE void half_stage(const v4i (&fa)[C::kBI][2], const v4i (&fb)[C::kBJ][2], const Words<C>& s, v16f (&acc)[C::kBI][C::kBJ]) {
  static_for<2>([&](auto T) {
    constexpr int t = decltype(T)::value;
#pragma unroll
    for (int i = 0; i < C::kBI; ++i)
#pragma unroll
      for (int j = 0; j < C::kBJ; ++j) mfma_fp4<kHalf * 2 + t>(acc[i][j], fb[j][t], fa[i][t], s.b[j], s.a[i]);
  });
}

template <class C>
struct ScaleSource {
  const uint8_t *a, *b;
  int bytes_a, bytes_b;
  uint32_t off_a[C::kBI], off_b[C::kBJ];
};
MXQ_DEVICE v2u buffer_load_x2(const void* base, int bytes, uint32_t voff, int soff) {
  return __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(
                                     __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, kRawBufferWord3),
                                     (int)voff, soff, 0));
}
template <class C>
MXQ_DEVICE void load_scales(const ScaleSource<C>& s, int stage, WordPairs<C>& w) {
  const int at = (stage >> 1) * (int)kFp4ScaleTile;
#pragma unroll
  for (int i = 0; i < C::kBI; ++i) w.a[i] = buffer_load_x2(s.a, s.bytes_a, s.off_a[i], at);
#pragma unroll
  for (int j = 0; j < C::kBJ; ++j) w.b[j] = buffer_load_x2(s.b, s.bytes_b, s.off_b[j], at);
}

// One group's whole main loop over stages [0, n) (kG = 0: waves 0-3, 1: waves 4-7). The operand chunks A_0 B_0 A_1
// B_1 ... go to slot (chunk index) % 5. Iteration kt has four phases, a workgroup barrier behind each; group g computes
// in phases 2 q + g and reads in the others:
//   P0  g0: first half of kt      g1: reads (kt, 0), loads A_kt+2 into B_kt-1's slot
//   P1  g1: first half            g0: reads (kt, 1), loads A_kt+2
//   P2  g0: second half           g1: reads (kt, 1)          both then wait for stage kt+1
//   P3  g1: second half + loads   g0: reads (kt+1, 0), loads B_kt+2 into A_kt's slot
//       of B_kt+2
// The scale words of stages 2 g and 2 g + 1 are requested with the B loads of iteration 2 g - 2, so the next iteration's wait
// covers them.
template <class C, int kG>
MXQ_DEVICE void main_loop(char* lds, const Chunk<C::kLoadsA>& ca, const Chunk<C::kLoadsB>& cb, const ScaleSource<C>& ss,
                          int n, int wrow, int wcol, int lane, v16f (&acc)[C::kBI][C::kBJ]) {
  const uint32_t base = lds_addr(lds);
  auto slot_addr = [&](int s) { return base + (uint32_t)(s * kSlot); };
  Words<C> cur;
  WordPairs<C> next;
  load_scales(ss, 0, next);
  __builtin_amdgcn_sched_barrier(0);
  issue_chunk(ca, lds, 0, true);
  issue_chunk(cb, lds + kSlot, 0, true);
  issue_chunk(ca, lds + 2 * kSlot, 1, n > 1);
  issue_chunk(cb, lds + 3 * kSlot, 1, n > 1);
  if (n > 1)
    wait_vmcnt<C::kLoadsA + C::kLoadsB>();
  else
    wait_vmcnt<0>();
  auto take = [&](Words<C>& w, bool second) {
#pragma unroll
    for (int i = 0; i < C::kBI; ++i) {
      w.a[i] = second ? next.a[i][1] : next.a[i][0];
      __asm__ volatile("" : "+v"(w.a[i]));
    }
#pragma unroll
    for (int j = 0; j < C::kBJ; ++j) {
      w.b[j] = second ? next.b[j][1] : next.b[j][0];
      __asm__ volatile("" : "+v"(w.b[j]));
    }
  };
  take(cur, false);
  phase_barrier();
  v4i fa[C::kBI][2], fb[C::kBJ][2];
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
      if ((kt & 1) == 0 && more) load_scales(ss, kt + 2, next);
    };
    if constexpr (kG == 0) {
      half_stage<C, 0>(fa, fb, cur, acc);  // P0
      phase_barrier();
      read_frags<C::kBI>(slot_addr(sa), wrow, lane, 1, fa);  // P1
      read_frags<C::kBJ>(slot_addr(sb), wcol, lane, 1, fb);
      issue_chunk(ca, slot_pa, kt + 2, more);
      wait_lgkm<0>();
      phase_barrier();
      half_stage<C, 1>(fa, fb, cur, acc);  // P2
    } else {
      read_frags<C::kBI>(slot_addr(sa), wrow, lane, 0, fa);  // P0
      read_frags<C::kBJ>(slot_addr(sb), wcol, lane, 0, fb);
      issue_chunk(ca, slot_pa, kt + 2, more);
      wait_lgkm<0>();
      phase_barrier();
      half_stage<C, 0>(fa, fb, cur, acc);  // P1
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
    // The words requested an iteration ago have landed with it: the next stage's are taken here, ahead of the next request
    // (behind it, the compiler would wait for that one).
    Words<C> after;
    take(after, (kt & 1) == 0);
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
      half_stage<C, 1>(fa, fb, cur, acc);  // P3
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

template <int kTM, int kOut, bool kSplit>
__global__ __launch_bounds__(512, 2) void gemm_mxfp4_kernel(Fp4Gemm p) {
  typedef Tile<kTM> C;
  __shared__ __attribute__((aligned(1024))) char lds[kGemmLds];
  int tm, tn, slice;
  tile_of(blockIdx.x, p, tm, tn, slice);
  const int M = (int)p.M, N = (int)p.N, m0 = tm * kTM, n0 = tn * kTileN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // waves w and w + 4 share a SIMD: the two 64-column halves of quadrant w % 4
  const int wrow = ((wave & 3) >> 1) * C::kWaveM, wcol = (wave & 1) * 128 + (wave >> 2) * 64;
  const int first = slice * p.split_stages, n = min(p.split_stages, p.stages - first);
  const auto ca = make_chunk<C::kLoadsA>(p.a + (int64_t)first * kStageK, p.lda, m0, M, wave, lane);
  const auto cb = make_chunk<C::kLoadsB>(p.b + (int64_t)first * kStageK, p.ldb, n0, N, wave, lane);
  // (a row of scale tiles holds 32 rows; behind the operands' last one, reads give zeros)
  ScaleSource<C> ss;
  const int row_tiles = p.groups * (int)kFp4ScaleTile, skip = (first >> 1) * (int)kFp4ScaleTile;
  ss.a = p.sa + (int64_t)(m0 >> 5) * row_tiles + skip;
  ss.b = p.sb + (int64_t)(n0 >> 5) * row_tiles + skip;
  ss.bytes_a = ((min(M - m0, kTM) + 31) >> 5) * row_tiles - skip;
  ss.bytes_b = ((min(N - n0, kTileN) + 31) >> 5) * row_tiles - skip;
#pragma unroll
  for (int i = 0; i < C::kBI; ++i) ss.off_a[i] = (uint32_t)(((wrow >> 5) + i) * row_tiles + lane * 8);
#pragma unroll
  for (int j = 0; j < C::kBJ; ++j) ss.off_b[j] = (uint32_t)(((wcol >> 5) + j) * row_tiles + lane * 8);
  v16f acc[C::kBI][C::kBJ] = {};
  if (wave < 4)
    main_loop<C, 0>(lds, ca, cb, ss, n, wrow, wcol, lane, acc);
  else
    main_loop<C, 1>(lds, ca, cb, ss, n, wrow, wcol, lane, acc);
  void* d = p.d;
  if constexpr (kSplit) d = reinterpret_cast<float*>(p.d) + slice * p.M * p.ldd;
  epilogue<C, kOut, kSplit>(p, lds, acc, m0, n0, wrow, wcol, wave, lane, d);
}

// ---- host side ----

struct Fp4Plan {
  int tile, splits, split_stages;
  double cost;
};

// Tile rows and K slices, by an estimate in microseconds: a round of workgroups takes 5 for its first loads and its epilogue and
// 1.0 (256 rows) or 0.55 (128 rows) per stage, all rounds at least the weight's bytes; slices cost a join.
static Fp4Plan plan_fp4(int64_t M, int64_t N, int64_t stages, int cus) {
  Fp4Plan best = {256, 1, (int)((stages + 1) / 2 * 2), 1e300};
  const double stream = (double)(N * stages) * 136.0 / 4.9e6 + 2.0;
  for (int tile = 256; tile >= 128; tile /= 2) {
    const int64_t tiles = (M + tile - 1) / tile * ((N + kTileN - 1) / kTileN);
    for (int64_t s = 1; s <= 32; ++s) {
      const int64_t per = ((stages + s - 1) / s + 1) / 2 * 2, splits = (stages + per - 1) / per;
      if (splits != s || (s > 1 && tiles * s > 4 * cus)) continue;
      const double rounds = (double)((tiles * s + cus - 1) / cus);
      double cost = rounds * ((double)(per < stages ? per : stages) * (tile == 256 ? 1.0 : 0.55) + 5.0);
      if (cost < stream) cost = stream;
      cost += slices_cost(s, M * N);
      if (cost < best.cost) best = {tile, (int)s, (int)per, cost};
    }
  }
  return best;
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
  if (ldb < bytes || ldb % 16 || ldb > (1ll << 22) || ldd < N)
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the weight or the output for N=%lld K=%lld", (long long)N, (long long)K);
  if (lda < bytes || lda % 16 || lda > (1ll << 22))
    return mxq_set_error(MXQ_ERR_INVALID, "bad row strides of the activations for K=%lld", (long long)K);
  if (M == 0) return MXQ_OK;
  // (so many tiles are not split; of 256 rows, as the plan may take them, there are half as many)
  if ((M + 255) / 256 * ((N + kTileN - 1) / kTileN) >= (1ll << 22)) return mxq_set_error(MXQ_ERR_UNSUPPORTED, "more than 2^22 tiles");
  if (!a || !sa || !b || !sb || !d || !aligned(a, 16) || !aligned(b, 16) || !aligned(sa, 16) || !aligned(sb, 16))
    return mxq_set_error(MXQ_ERR_INVALID, "null or misaligned pointer");
  return MXQ_OK;
}

template <int kTM, int kOut, bool kSplit>
static int launch_gemm(const Fp4Gemm& p, void* stream) {
  hipLaunchKernelGGL((gemm_mxfp4_kernel<kTM, kOut, kSplit>), dim3((unsigned)(p.tiles_m * p.tiles_n * p.splits)), dim3(512), 0,
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
  const int64_t tiles_m = (M + plan.tile - 1) / plan.tile, tiles_n = (N + kTileN - 1) / kTileN;
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
    if (const int rc = plan.tile == 256 ? launch_gemm<256, 0, true>(p, stream) : launch_gemm<128, 0, true>(p, stream)) return rc;
    return fp8_join({(const float*)workspace, bias, d, M, ldp, ldd, (int)N, plan.splits, out_dtype}, {}, {}, stream);
  }
  p.vec = aligned(d, 16) && ldd * dtype_bytes(out_dtype) % 16 == 0;
  return with_dtype(out_dtype, [&](auto O) {
    constexpr int kOut = decltype(O)::value;
    return plan.tile == 256 ? launch_gemm<256, kOut, false>(p, stream) : launch_gemm<128, kOut, false>(p, stream);
  });
}
