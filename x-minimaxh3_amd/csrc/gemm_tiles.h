// What the block-scaled matrix products share, gemm_fp8.hip's workgroups of eight waves (Tile) and gemm_mxfp4.hip's of four: operand
// chunks of 128 bytes a row on their way into a ring of LDS slots, the tile order and the epilogue.
#pragma once

#include "fp8_common.h"

namespace mxq {

constexpr int kTileN = 256, kStageK = 128;
constexpr int kRing = 5, kSlot = 256 * kStageK;
constexpr int kGemmLds = kRing * kSlot;
static_assert(kGemmLds <= 160 * 1024, "LDS of a CU");
constexpr int kGroupRows = 4;  // tile-rows per group of the tile order

template <int kTM>
struct Tile {
  static constexpr int kBM = kTM, kBN = kTileN, kWaveM = kTM / 2, kBI = kWaveM / 32, kBJ = 2;
  static constexpr int kLoadsA = kTM / 64, kLoadsB = 4;  // 1 KB loads per wave and chunk
};

// ---- operand loads ----
// Chunk rows are 128 bytes; 16-byte piece c of row r sits at piece c ^ ((r >> 1) & 7), so that the sixteen lanes a
// ds_read_b128 serves at once (sixteen rows, one piece) touch every bank once. One load fills 1 KB: eight rows.
MXQ_DEVICE int swizzle(int r) { return (r >> 1) & 7; }

template <int kLoads>
struct Chunk {
  const uint8_t* base;  // row 0 of the tile
  int bytes;            // the tile's rows in memory: rows behind the operand's last are the last one again
  uint32_t off[kLoads];
  int wave;
};

// (Rows are counted in 32 bits: a buffer resource has to be in scalar registers, and there is no scalar 64-bit minimum.
// Computed in vector registers, it made every access loop over the lanes' resources.)
template <int kLoads, int kWaves = 8>
MXQ_DEVICE Chunk<kLoads> make_chunk(const uint8_t* p, int64_t ld, int row0, int rows, int wave, int lane) {
  Chunk<kLoads> c;
  const int valid = min(rows - row0, kLoads * 8 * kWaves);
  c.base = p + row0 * ld;
  c.bytes = valid * (int)ld;
  c.wave = wave;
#pragma unroll
  for (int t = 0; t < kLoads; ++t) {
    const int r = (wave * kLoads + t) * 8 + (lane >> 3);
    c.off[t] = (uint32_t)(min(r, valid - 1) * (int)ld + (((lane & 7) ^ swizzle(r)) << 4));
  }
  return c;
}

// Load t of a chunk.
template <int kLoads>
MXQ_DEVICE void issue_load(const Chunk<kLoads>& c, char* slot, int stage, int t) {
  buffer_load_lds16(c.base, c.bytes, (lptr_t)(slot + (c.wave * kLoads + t) * 1024), c.off[t], stage * kStageK);
}

template <int kLoads>
MXQ_DEVICE void issue_chunk(const Chunk<kLoads>& c, char* slot, int stage, bool on) {
  if (on) {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) issue_load(c, slot, stage, t);
  }
}

MXQ_DEVICE v8i join8(v4i a, v4i b) { return v8i{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

// Waits out the 16 passes of the last matrix instruction (19 wait states) before its sums are read.
MXQ_DEVICE void mfma_drain() {
  __builtin_amdgcn_sched_barrier(0);
  __asm__ volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

MXQ_DEVICE void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  barrier_no_drain();
  __builtin_amdgcn_sched_barrier(0);
}

// ---- epilogue ----
// A wave passes its output through 4 KB of LDS in pieces of 32 rows x 128 bytes (32-row block i, one or two column
// blocks), so that eight lanes store a whole line, or, where rows are not 16-byte aligned or the tile is an edge's, 16 bytes
// a lane from any address (lane by lane straight from the sums, 1024 rows x 2049 columns took 8 us longer).
MXQ_DEVICE char* out_stage_at(char* buf, int r, int c) { return buf + r * 128 + ((c ^ ((r >> 1) & 7)) << 4); }

template <int kOut>
MXQ_DEVICE uint32_t out_pair(float a, float b) {  // two 16-bit values
  if constexpr (kOut == MXQ_DTYPE_BF16) return pack_bf16x2(a, b);
  return f32_to_f16_bits(a) | (f32_to_f16_bits(b) << 16);
}

template <class C, int kOut, bool kSplit, class P>
MXQ_DEVICE void epilogue(const P& p, char* lds, const v16f (&acc)[C::kBI][C::kBJ], int m0, int n0, int wrow,
                         int wcol, int wave, int lane, void* d) {
  constexpr int kElem = kOut == MXQ_DTYPE_F32 ? 4 : 2;
  char* buf = lds + wave * 4096;
  const int M = (int)p.M, N = (int)p.N;
  const bool lines = p.vec && M - m0 >= C::kBM && N - n0 >= C::kBN;
  const int lr = lane & 31, lh = lane >> 5;
  char* out = reinterpret_cast<char*>(d);
  v4f bias[kSplit ? 1 : C::kBJ][4];  // (read once, ahead of the first piece's stores)
  if constexpr (!kSplit) {
#pragma unroll
    for (int j = 0; j < C::kBJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) bias[j][q] = bias_run<kOut>(p.bias, n0 + wcol + j * 32 + q * 8 + lh * 4, N);
  }
#pragma unroll
  for (int i = 0; i < C::kBI; ++i) {
    const int row0 = m0 + wrow + i * 32;
#pragma unroll
    for (int j = 0; j < C::kBJ; ++j) {
      const int col0 = n0 + wcol + j * 32;
      if (kElem == 4 || (j & 1) == 0) wave_lds_fence();  // the piece before has been read
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = kSplit ? acc[i][j][q * 4 + e] : acc[i][j][q * 4 + e] + bias[kSplit ? 0 : j][q][e];
        if constexpr (kElem == 4) {
          *reinterpret_cast<v4f*>(out_stage_at(buf, lr, 2 * q + lh)) = v4f{y[0], y[1], y[2], y[3]};
        } else {
          *reinterpret_cast<v2u*>(out_stage_at(buf, lr, (j & 1) * 4 + q) + lh * 8) =
              v2u{out_pair<kOut>(y[0], y[1]), out_pair<kOut>(y[2], y[3])};
        }
      }
      if (kElem == 4 || (j & 1) == 1) {
        wave_lds_fence();
        constexpr int kRun = 16 / kElem;
        const int col = (kElem == 4 ? col0 : col0 - 32) + (lane & 7) * kRun;
        v4u v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = *reinterpret_cast<const v4u*>(out_stage_at(buf, t * 8 + (lane >> 3), lane & 7));
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int row = row0 + t * 8 + (lane >> 3);
          char* to = out + (row * p.ldd + col) * kElem;
          if (lines) {
            __builtin_nontemporal_store(v[t], reinterpret_cast<v4u*>(to));
          } else if (row < M) {
            const int n = N - col;
            if (n >= kRun) {
              *reinterpret_cast<v4u_any*>(to) = v[t];
            } else {
#pragma unroll
              for (int e = 0; e < kRun; ++e)
                if (e < n) {
                  if constexpr (kElem == 4) reinterpret_cast<uint32_t*>(to)[e] = v[t][e];
                  else reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[t][e >> 1] >> (16 * (e & 1)));
                }
            }
          }
        }
      }
    }
  }
}

// Tile order: contiguous ranges over the 8 XCDs (workgroup ids are dealt to them in turn), each walked in groups of
// kGroupRows tile-rows, so that an XCD's workgroups share operand panels in its L2.
template <class P>
MXQ_DEVICE void tile_of(int bid, const P& p, int& tm, int& tn, int& slice) {
  const int tiles = p.tiles_m * p.tiles_n, num = tiles * p.splits, per = num / 8;
  int t = bid < per * 8 ? (bid % 8) * per + bid / 8 : bid;
  slice = t / tiles;
  t -= slice * tiles;
  const int group = kGroupRows * p.tiles_n, g = t / group, first = g * kGroupRows, rows = min(p.tiles_m - first, kGroupRows);
  const int in = t - g * group;
  tn = in / rows;
  tm = first + in - tn * rows;
}

}  // namespace mxq
