// C[i][j] = sum_k A[i][k] * B[j][k] of two K-contiguous operands ("NT") on the matrix cores: the tile
// loop shared by the 8-bit product (int8_gemm.hip) and the Newton-Schulz products (newton_schulz.hip).
//
// A K tile is 64 bytes of every operand row: 64 int8 values or 32 fp16 values, the K extent of one
// v_mfma_i32_16x16x64_i8 / v_mfma_f32_16x16x32_f16, whose operand registers hold 16 bytes per lane of
// row lane & 15, 16-byte chunk lane >> 4.  Both types therefore run the same loop on bytes.
//
// Operands go from memory to LDS with buffer_load ... lds (no registers), NR - 1 K tiles ahead in a
// ring of NR; one barrier per K tile.  Rows and chunks outside an operand are given an offset beyond
// the descriptor's record count, which reads as zero.  LDS rows are 64 bytes, chunk c of row r stored
// at c ^ ((r >> 2) & 3): the 16 rows of a fragment read fall on distinct 16-byte bank slots.  The DMA
// writes lane-linear, so the permutation is applied to the chunk each lane fetches.
//
// fp16 operands come as pairs v = hi + lo (22 significant bits, two planes): a product is
// hi lo + lo hi + hi hi with fp32 accumulation, small terms first.  The dropped lo lo is below 2^-22 of the
// product.  Each plane has its own LDS rows.
#pragma once
#include "../matrix_ops.h"
#include "common.h"

#include <type_traits>

namespace mxr {

typedef _Float16 nt_f16x8 __attribute__((ext_vector_type(8)));
typedef float nt_f32x4 __attribute__((ext_vector_type(4)));
typedef int nt_i32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kNtOob = 0x80000000u;  // past any record count (windows are below 2 GiB)

// rows [0, rows) of an operand from its block's first row on: `base` points there
struct NtOperand {
  const char* base;
  uint32_t ld;    // bytes from row to row (multiple of 16)
  int rows;       // rows that exist (may exceed the tile)
  int64_t plane;  // bytes to the second plane (pairs)
};

// PL planes; BA x BB output tile, WA x WB waves, NR K tiles in the LDS ring
template <int PL_, int BA_, int BB_, int WA_, int WB_, int NR_>
struct NtCfg {
  static constexpr int PL = PL_, BA = BA_, BB = BB_, WA = WA_, WB = WB_, NR = NR_;
  static constexpr int WAVES = WA * WB, THREADS = 64 * WAVES;
  static constexpr int TA = BA / WA / 16, TB = BB / WB / 16;
  static constexpr int ROWS = PL * (BA + BB);         // LDS rows of a K tile: A planes, then B planes
  static constexpr int LPT = ROWS / 16 / WAVES;       // DMA instructions of a wave per K tile
  static constexpr int TILE = ROWS * 64, LDS = NR * TILE;
  using Acc = typename std::conditional<PL == 2, nt_f32x4, nt_i32x4>::type;
  static_assert(ROWS % (16 * WAVES) == 0, "every wave issues the same number of 16-row loads");
  static_assert(BA % (16 * WA) == 0 && BB % (16 * WB) == 0, "whole 16x16 tiles per wave");
};

template <int N>
__device__ __forceinline__ void nt_wait() {
  // the loads of all but the N youngest instructions have landed; this wave's LDS reads are done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t nt_rsrc(const char* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes, 0x00020000);
}
// 16 bytes per lane from byte `voff` + `soff` of the window to 1 KiB of LDS, lane after lane
__device__ __forceinline__ void nt_dma(__amdgpu_buffer_rsrc_t rs, char* lds, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, (int)voff, soff, 0, 0);
}

__device__ __forceinline__ nt_f32x4 nt_mma(const uint4& a, const uint4& b, nt_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(nt_f16x8, a), __builtin_bit_cast(nt_f16x8, b), c, 0,
                                                0, 0);
}
__device__ __forceinline__ nt_i32x4 nt_mma(const uint4& a, const uint4& b, nt_i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(nt_i32x4, a), __builtin_bit_cast(nt_i32x4, b), c, 0, 0,
                                               0);
}

// Fragments of K tile `T` into the accumulators of this wave.
template <class C>
__device__ __forceinline__ void nt_tile_mma(const char* T, int wa, int wb, int lane,
                                            typename C::Acc (&acc)[C::TA][C::TB]) {
  const int r16 = lane & 15, ch = lane >> 4;
  const auto frag = [&](int row) {
    return *reinterpret_cast<const uint4*>(T + row * 64 + ((ch ^ ((row >> 2) & 3)) << 4));
  };
  uint4 b[C::PL][C::TB];
#pragma unroll
  for (int p = 0; p < C::PL; ++p)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) b[p][j] = frag(C::PL * C::BA + p * C::BB + (wb * C::TB + j) * 16 + r16);
#pragma unroll
  for (int i = 0; i < C::TA; ++i) {
    uint4 a[C::PL];
#pragma unroll
    for (int p = 0; p < C::PL; ++p) a[p] = frag(p * C::BA + (wa * C::TA + i) * 16 + r16);
    if constexpr (C::PL == 2) {
#pragma unroll
      for (int j = 0; j < C::TB; ++j) acc[i][j] = nt_mma(a[0], b[1][j], acc[i][j]);
#pragma unroll
      for (int j = 0; j < C::TB; ++j) acc[i][j] = nt_mma(a[1], b[0][j], acc[i][j]);
    }
#pragma unroll
    for (int j = 0; j < C::TB; ++j) acc[i][j] = nt_mma(a[0], b[0][j], acc[i][j]);
  }
}

// The K loop over bytes [k_lo, k_hi) of every row (k_lo a multiple of 64, k_hi of 16).  Lane l of wave
// (wa, wb) ends with C[(wa * TA + i) * 16 + (l >> 4) * 4 + r][(wb * TB + j) * 16 + (l & 15)] in
// acc[i][j][r].  `lds`: C::LDS bytes as a plain pointer (given the __shared__ array itself, the
// compiler waits for every load in flight before each fragment read).
template <class C>
__device__ __forceinline__ void nt_loop_body(char* lds, const char* __restrict__ a_base, const char* __restrict__ b_base,
                                             const NtOperand& A, const NtOperand& B, int k_lo, int k_hi,
                                             typename C::Acc (&acc)[C::TA][C::TB]) {
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wa = wid / C::WB, wb = wid % C::WB;
#pragma unroll
  for (int i = 0; i < C::TA; ++i)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) acc[i][j] = typename C::Acc{0, 0, 0, 0};
  // bytes of an operand's window: up to the end of its last row
  const auto window = [&](const NtOperand& o, int tile) {
    const int rows = min(o.rows, tile);
    return rows > 0 ? (int)((uint32_t)(rows - 1) * o.ld + (uint32_t)k_hi) : 0;
  };
  const int wina = window(A, C::BA), winb = window(B, C::BB);
  const __amdgpu_buffer_rsrc_t ra0 = nt_rsrc(a_base, wina), rb0 = nt_rsrc(b_base, winb);
  const __amdgpu_buffer_rsrc_t ra1 = nt_rsrc(a_base + A.plane, wina), rb1 = nt_rsrc(b_base + B.plane, winb);
  uint32_t off[C::LPT];
  int chunk[C::LPT];
#pragma unroll
  for (int i = 0; i < C::LPT; ++i) {
    const int r = (i * C::WAVES + wid) * 16 + (lane >> 2);  // LDS row
    const bool is_b = r >= C::PL * C::BA;
    const int row = is_b ? (r - C::PL * C::BA) % C::BB : r % C::BA;
    chunk[i] = ((lane & 3) ^ ((r >> 2) & 3)) * 16;
    const uint32_t ld = is_b ? B.ld : A.ld;
    off[i] = row < (is_b ? B.rows : A.rows) ? (uint32_t)row * ld + (uint32_t)chunk[i] : kNtOob;
  }
  const auto issue = [&](int buf, int k) {
    char* base = lds + buf * C::TILE + wid * 1024;
#pragma unroll
    for (int i = 0; i < C::LPT; ++i) {
      const int r0 = (i * C::WAVES + wid) * 16;  // wave-uniform
      const bool is_b = r0 >= C::PL * C::BA;
      const int p = is_b ? (r0 - C::PL * C::BA) / C::BB : r0 / C::BA;
      const uint32_t vo = k + chunk[i] < k_hi ? off[i] : kNtOob;
      char* dst = base + i * C::WAVES * 1024;
      if (is_b) {
        if (p == 0) nt_dma(rb0, dst, vo, k);
        else nt_dma(rb1, dst, vo, k);
      } else {
        if (p == 0) nt_dma(ra0, dst, vo, k);
        else nt_dma(ra1, dst, vo, k);
      }
    }
  };
  const int nk = (k_hi - k_lo + 63) / 64;
  // pairs: the sums of kNtRun K tiles at a time are added up apart.  The matrix core rounds its accumulator to
  // fp32 after every 8 products, so one long sum of positive terms (a diagonal of X X^T) would lose
  // sqrt(3 K / 8) / 2 last places; in runs that is 2 to 3 of them at K = 2048.
  constexpr int kNtRun = 8;
  typename C::Acc sum[C::PL == 2 ? C::TA : 1][C::PL == 2 ? C::TB : 1];
  if constexpr (C::PL == 2) {
#pragma unroll
    for (int i = 0; i < C::TA; ++i)
#pragma unroll
      for (int j = 0; j < C::TB; ++j) sum[i][j] = typename C::Acc{0, 0, 0, 0};
  }
#pragma unroll
  for (int s = 0; s < C::NR - 1; ++s)
    if (s < nk) issue(s, k_lo + s * 64);
  for (int kt = 0; kt < nk; ++kt) {
    // K tile kt has landed for this wave; the younger tiles stay in flight
    const int ahead = min(C::NR - 2, nk - 1 - kt);
    if (C::NR > 3 && ahead >= 2) nt_wait<2 * C::LPT>();
    else if (C::NR > 2 && ahead == 1) nt_wait<C::LPT>();
    else nt_wait<0>();
    __builtin_amdgcn_s_barrier();  // ... for every wave, and tile kt - 1 has been read by all
    asm volatile("" ::: "memory");
    if (kt + C::NR - 1 < nk) issue((kt + C::NR - 1) % C::NR, k_lo + (kt + C::NR - 1) * 64);
    nt_tile_mma<C>(lds + kt % C::NR * C::TILE, wa, wb, lane, acc);
    if constexpr (C::PL == 2) {
      if (kt % kNtRun == kNtRun - 1) {
#pragma unroll
        for (int i = 0; i < C::TA; ++i)
#pragma unroll
          for (int j = 0; j < C::TB; ++j) {
            sum[i][j] += acc[i][j];
            acc[i][j] = typename C::Acc{0, 0, 0, 0};
          }
      }
    }
  }
  if constexpr (C::PL == 2) {
#pragma unroll
    for (int i = 0; i < C::TA; ++i)
#pragma unroll
      for (int j = 0; j < C::TB; ++j) acc[i][j] += sum[i][j];
  }
  static_assert(C::NR >= 2 && C::NR <= 4, "ring depth");
  // the ring may be reused by the epilogue: every wave is past its last read
  nt_wait<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <class C>
__device__ __forceinline__ void nt_loop(char* lds, const NtOperand& A, const NtOperand& B, int k_lo, int k_hi,
                                        typename C::Acc (&acc)[C::TA][C::TB]) {
  nt_loop_body<C>(lds, A.base, B.base, A, B, k_lo, k_hi, acc);
}

// Consecutive workgroups go to the 8 XCDs in turn: give each XCD a contiguous range of work items, so
// that tiles sharing operand rows share an L2.
__device__ __forceinline__ int nt_xcd_item(int bid, int n) {
  const int q = n / 8, r = n % 8, x = bid % 8;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + bid / 8;
}

}  // namespace mxr
