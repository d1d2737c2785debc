// C[i][j] = sum_k A[i][k] * B[j][k] of two K-contiguous operands ("NT") on the matrix cores: the tile
// loop shared by the 8-bit product (int8_gemm.hip) and the Newton-Schulz products (newton_schulz.hip).
//
// A K tile is 128 bytes of every operand row -- one whole cache line, fetched once.  (With 64-byte tiles the other
// half of each line was fetched again one tile later: Newton-Schulz of 4096 x 4096 with tiles of pairs of 256 x 256
// took 5030 instead of 4715 us, of 128 x 128 5540 instead of 4730.)  The 128 bytes are
// eight 16-byte chunks: 128 int8 values, two k steps of v_mfma_i32_16x16x64_i8; or 32 fp16 pairs v = hi + lo
// (22 significant bits), the 32 hi values in chunks 0 - 3 and the 32 lo values in chunks 4 - 7, one k step of
// v_mfma_f32_16x16x32_f16 for each of hi lo + lo hi + hi hi (small terms first, fp32 accumulation; the dropped
// lo lo is below 2^-22 of the product).  The operand registers of both instructions hold 16 bytes per lane: of row
// lane & 15, chunk lane >> 4 of the k step.  So both types run the same loop on bytes.
//
// Operands go from memory to LDS with buffer_load ... lds (no registers), NR - 1 K tiles ahead in a
// ring of NR; one barrier per K tile.  Rows and chunks outside an operand are given an offset beyond
// the descriptor's record count, which reads as zero.  Chunk c of LDS row r is stored at c ^ ((r >> 1) & 7): the
// 16 rows of a fragment read fall on distinct 16-byte bank slots.  The DMA writes lane-linear, so the
// permutation is applied to the chunk each lane fetches.
#pragma once
#include "../matrix_ops.h"
#include "common.h"

#include <type_traits>

namespace mxr {

typedef _Float16 nt_f16x8 __attribute__((ext_vector_type(8)));
typedef float nt_f32x4 __attribute__((ext_vector_type(4)));
typedef int nt_i32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kNtOob = 0x80000000u;  // past any record count (windows are below 2 GiB)

// Rows [0, rows) of an operand from its block's first row on: `base` points there.
// Pairs lie in panels: the 128-byte lines of K tile 0 of all rows, then those of K tile 1, .. -- `step` bytes from one
// K tile to the next.  A block's K tile is then one run of memory.  (Row after row, a K tile of fc6's 4096 x 25088
// touched one line in each of 256 rows 100 KB apart: 3.1 ms for X X^T instead of 1.7.)
// int8 operands are the caller's rows, `ld` bytes apart (a multiple of 16).
// TURN: A lies in panels the other way round, lines of k with 32 of A's rows each: panel after panel (`step` bytes) of
// 32 rows, `rows` a multiple of 32.  A K tile is then 32 lines of each of BA / 32 panels, line k of panel p in LDS row
// 32 p + k, and a fragment's 8 k values of one row come together in ds_read_b64_tr_b16: of a group of 16 lanes, lane
// 4 i + j gives the address of elements 4 j .. 4 j + 3 of line i, and lane r receives element r of the four lines.
struct NtOperand {
  const char* base;
  int rows;  // rows that exist (may exceed the tile)
  uint32_t ld;
  int64_t step;
};

// fp16 pairs or int8; BA x BB output tile; KG groups of WA x WB waves, each with every KG-th K tile (joined at the
// end); NR stages of KG K tiles in the LDS ring; RUN: stages summed apart (0: all); AHEAD: fragments of a stage are
// read while those of the one before are multiplied.  TURN: operand A is read across its lines (NtOperand).
template <bool PAIR_, int BA_, int BB_, int KG_, int WA_, int WB_, int NR_, int RUN_ = 0, bool AHEAD_ = false,
          bool TURN_ = false>
struct NtCfg {
  static constexpr bool PAIR = PAIR_, AHEAD = AHEAD_, TURN = TURN_;
  using Turned = NtCfg<PAIR_, BA_, BB_, KG_, WA_, WB_, NR_, RUN_, AHEAD_, true>;
  static constexpr int BA = BA_, BB = BB_, KG = KG_, WA = WA_, WB = WB_, NR = NR_, RUN = RUN_;
  static constexpr int GROUP = WA * WB, WAVES = KG * GROUP, THREADS = 64 * WAVES;
  static constexpr int TA = BA / WA / 16, TB = BB / WB / 16;
  static constexpr int ROWS = BA + BB;               // LDS rows of a K tile: A, then B
  // DMA instructions (8 rows) of a wave per stage; where they come out uneven (int8 only), the last ones fill rows
  // behind the stage's that nobody reads
  static constexpr int LPT = (KG * ROWS / 8 + WAVES - 1) / WAVES;
  static constexpr int TILE = ROWS * 128, STAGE = LPT * WAVES * 1024, RING = NR * STAGE;
  static constexpr int JOIN = KG > 1 ? WAVES * TA * TB * 1024 : 0;  // accumulators exchanged between groups
  static constexpr int LDS = RING > JOIN + WAVES * 1280 ? RING : JOIN + WAVES * 1280;
  using Acc = typename std::conditional<PAIR, nt_f32x4, nt_i32x4>::type;
  static_assert(!TURN || (PAIR && BA % 32 == 0), "turned operands are panels of pairs");
  static_assert(!PAIR || KG * ROWS % (8 * WAVES) == 0, "pairs: every load has its rows");
  static_assert(BA % (16 * WA) == 0 && BB % (16 * WB) == 0, "whole 16x16 tiles per wave");
  static_assert(NR >= 2 && LDS <= 160 * 1024 && (NR - 1) * LPT < 64, "ring depth (vmcnt counts to 63)");
  // this wave: its group, its place in it; the 16 x 16 tiles that it holds after the join
  static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
  static __device__ __forceinline__ int kg() { return wave() / GROUP; }
  static __device__ __forceinline__ int wa() { return wave() % GROUP / WB; }
  static __device__ __forceinline__ int wb() { return wave() % WB; }
  static __device__ __forceinline__ bool mine(int i, int j) { return KG == 1 || (i * TB + j) % KG == kg(); }
  // 1280 bytes of LDS of this wave alone, free after the loop
  static __device__ __forceinline__ float* scratch(char* lds) {
    return reinterpret_cast<float*>(lds + JOIN + wave() * 1280);
  }
};

template <int N>
__device__ __forceinline__ void nt_wait() {
  // the loads of all but the N youngest instructions have landed; this wave's LDS reads are done.  (As a builtin,
  // so that the compiler counts it; vmcnt in bits 3:0 and 15:14, expcnt 7 and lgkmcnt 0 between.)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t nt_rsrc(const char* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes, 0x00020000);
}
// 16 bytes per lane from byte `voff` + `soff` of the window to 1 KiB of LDS, lane after lane
__device__ __forceinline__ void nt_dma(__amdgpu_buffer_rsrc_t rs, char* lds, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, (int)voff, soff, 0, 0);
}

// the same 16 bytes into registers
typedef uint32_t nt_u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 nt_load(__amdgpu_buffer_rsrc_t rs, uint32_t voff, int soff) {
  return __builtin_bit_cast(uint4, (nt_u32x4)__builtin_amdgcn_raw_buffer_load_b128(rs, (int)voff, soff, 0));
}
__device__ __forceinline__ uint32_t nt_load1(__amdgpu_buffer_rsrc_t rs, uint32_t voff, int soff) {  // 4 bytes
  return __builtin_amdgcn_raw_buffer_load_b32(rs, (int)voff, soff, 0);
}

__device__ __forceinline__ nt_f32x4 nt_mma(const uint4& a, const uint4& b, nt_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(nt_f16x8, a), __builtin_bit_cast(nt_f16x8, b), c, 0,
                                                0, 0);
}
__device__ __forceinline__ nt_i32x4 nt_mma(const uint4& a, const uint4& b, nt_i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(nt_i32x4, a), __builtin_bit_cast(nt_i32x4, b), c, 0, 0,
                                               0);
}

// One fragment: 16 bytes of row `row` of K tile `T`, of its first (0) or second (1) four chunks.
__device__ __forceinline__ uint4 nt_frag(const char* T, int row, int half, int lane) {
  return *reinterpret_cast<const uint4*>(T + row * 128 + (((half * 4 + (lane >> 4)) ^ ((row >> 1) & 7)) << 4));
}

// The same of a turned operand, rows row0 .. row0 + 15 of the K tile (row0 a multiple of 16).  Its lines are swizzled by
// pairs of chunks: the 8 lines that 32 lanes read at once are 4 apart in (k >> 1), in two runs, and take 32 bytes each.
__device__ __forceinline__ int nt_turn_swizzle(int k) { return ((k >> 1) & 1) << 1 | ((k >> 3) & 1) << 2; }
typedef short nt_s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ nt_s16x4 nt_turned_read(const char* at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) nt_s16x4*)at);
}
__device__ __forceinline__ uint4 nt_turned_frag(const char* T, int row0, int half, int lane) {
  uint2 v[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int k = 8 * (lane >> 4) + 4 * t + ((lane & 15) >> 2);
    const int chunk = half * 4 + ((row0 & 16) >> 3) + ((lane & 3) >> 1);
    v[t] = __builtin_bit_cast(uint2, nt_turned_read(T + ((row0 & ~31) + k) * 128 + ((chunk ^ nt_turn_swizzle(k)) << 4) +
                                                    (lane & 1) * 8));
  }
  return make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
}
template <class C>
__device__ __forceinline__ uint4 nt_a_frag(const char* T, int row0, int half, int lane) {
  if constexpr (C::TURN) return nt_turned_frag(T, row0, half, lane);
  else return nt_frag(T, row0 + (lane & 15), half, lane);
}

// The products of one row of fragments with all columns.
template <class C>
__device__ __forceinline__ void nt_row_mma(const uint4 (&a)[2], const uint4 (&b)[2][C::TB],
                                           typename C::Acc (&acc)[C::TB]) {
  if constexpr (C::PAIR) {
#pragma unroll
    for (int j = 0; j < C::TB; ++j) acc[j] = nt_mma(a[0], b[1][j], acc[j]);
#pragma unroll
    for (int j = 0; j < C::TB; ++j) acc[j] = nt_mma(a[1], b[0][j], acc[j]);
  } else {
#pragma unroll
    for (int j = 0; j < C::TB; ++j) acc[j] = nt_mma(a[1], b[1][j], acc[j]);
  }
#pragma unroll
  for (int j = 0; j < C::TB; ++j) acc[j] = nt_mma(a[0], b[0][j], acc[j]);
}

// All fragments of this wave's part of a K tile.
template <class C>
struct NtFrags {
  uint4 a[C::TA][2], b[2][C::TB];
  __device__ __forceinline__ void load(const char* T, int wa, int wb, int lane) {
    const int r16 = lane & 15;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < C::TB; ++j) b[h][j] = nt_frag(T, C::BA + (wb * C::TB + j) * 16 + r16, h, lane);
#pragma unroll
    for (int i = 0; i < C::TA; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) a[i][h] = nt_a_frag<C>(T, (wa * C::TA + i) * 16, h, lane);
  }
  __device__ __forceinline__ void mma(typename C::Acc (&acc)[C::TA][C::TB]) const {
#pragma unroll
    for (int i = 0; i < C::TA; ++i) nt_row_mma<C>(a[i], b, acc[i]);
  }
};

// A K tile read and multiplied, each row of fragments read while the one before it is multiplied.
template <class C>
__device__ __forceinline__ void nt_tile_mma(const char* T, int wa, int wb, int lane,
                                            typename C::Acc (&acc)[C::TA][C::TB]) {
  const int r16 = lane & 15;
  uint4 b[2][C::TB], a[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) b[h][j] = nt_frag(T, C::BA + (wb * C::TB + j) * 16 + r16, h, lane);
#pragma unroll
  for (int h = 0; h < 2; ++h) a[0][h] = nt_a_frag<C>(T, wa * C::TA * 16, h, lane);
#pragma unroll
  for (int i = 0; i < C::TA; ++i) {
    if (i + 1 < C::TA) {
#pragma unroll
      for (int h = 0; h < 2; ++h) a[(i + 1) & 1][h] = nt_a_frag<C>(T, (wa * C::TA + i + 1) * 16, h, lane);
    }
    __builtin_amdgcn_sched_barrier(0);  // (the compiler would sink these reads behind the products)
    nt_row_mma<C>(a[i & 1], b, acc[i]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The K loop over bytes [k_lo, k_hi) of every row (k_lo a multiple of 128, k_hi of 16; pairs: of 128).  Lane l of
// wave (wa, wb) ends with C[(wa * TA + i) * 16 + (l >> 4) * 4 + r][(wb * TB + j) * 16 + (l & 15)] in
// acc[i][j][r] of the tiles that are its own (C::mine).  `lds`: C::LDS bytes as a plain pointer, and the operands' bases
// as __restrict__ parameters: otherwise the compiler waits for every load in flight before each fragment read.
template <class C>
__device__ __forceinline__ void nt_loop_body(char* lds, const char* __restrict__ a_base, const char* __restrict__ b_base,
                                             const NtOperand& A, const NtOperand& B, int k_lo, int k_hi,
                                             typename C::Acc (&acc)[C::TA][C::TB]) {
  const int lane = threadIdx.x & 63, wid = C::wave(), wa = C::wa(), wb = C::wb(), kg = C::kg();
#pragma unroll
  for (int i = 0; i < C::TA; ++i)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) acc[i][j] = typename C::Acc{0, 0, 0, 0};
  const int arows = min(A.rows, C::BA), brows = min(B.rows, C::BB);
  const int nk = (k_hi - k_lo + 128 * C::KG - 1) / (128 * C::KG);  // stages
  // Load i of this wave fills 8 LDS rows of the stage, lane l chunk l & 7 of row l >> 3: the same operand and K tile
  // for the whole wave.
  uint32_t off[C::LPT];
  int chunk[C::LPT];
#pragma unroll
  for (int i = 0; i < C::LPT; ++i) {
    const int lr = (i * C::WAVES + wid) * 8 + (lane >> 3);
    const int r = lr % C::ROWS, g = lr / C::ROWS;
    const bool is_b = r >= C::BA;
    const int row = is_b ? r - C::BA : r;
    chunk[i] = ((lane & 7) ^ ((r >> 1) & 7)) * 16;
    if constexpr (C::PAIR) {
      off[i] = row * 128 + chunk[i];
      if (C::TURN && !is_b)
        off[i] = row < arows ? (uint32_t)(row >> 5) * (uint32_t)A.step + (row & 31) * 128 +
                                   ((lane & 7) ^ nt_turn_swizzle(row & 31)) * 16
                             : kNtOob;
    } else {
      chunk[i] += g * 128;
      off[i] = g < C::KG && row < (is_b ? brows : arows) ? (uint32_t)row * (is_b ? B.ld : A.ld) + (uint32_t)chunk[i]
                                                         : kNtOob;
    }
  }
  // int8: one window per operand, up to the end of its last row
  const __amdgpu_buffer_rsrc_t ra = nt_rsrc(a_base, arows > 0 ? (int)((uint32_t)(arows - 1) * A.ld + (uint32_t)k_hi) : 0);
  const __amdgpu_buffer_rsrc_t rb = nt_rsrc(b_base, brows > 0 ? (int)((uint32_t)(brows - 1) * B.ld + (uint32_t)k_hi) : 0);
  const auto issue = [&](int buf, int kt) {
    char* base = lds + buf * C::STAGE + wid * 1024;
#pragma unroll
    for (int i = 0; i < C::LPT; ++i) {
      char* dst = base + i * C::WAVES * 1024;
      const int r0 = (i * C::WAVES + wid) * 8;  // wave-uniform
      const bool is_b = r0 % C::ROWS >= C::BA;
      if constexpr (C::PAIR) {
        // a window of the operand's rows at this K tile; none past the end
        const int t = kt * C::KG + r0 / C::ROWS;
        const bool in = t * 128 < k_hi;
        const char* at = is_b ? b_base + t * B.step : a_base + (C::TURN ? t * 4096 : t * A.step);
        const int bytes = C::TURN && !is_b ? (arows / 32 - 1) * (int)A.step + 4096 : (is_b ? brows : arows) * 128;
        nt_dma(nt_rsrc(at, in ? bytes : 0), dst, off[i], 0);
      } else {
        const int k = k_lo + kt * 128 * C::KG;
        nt_dma(is_b ? rb : ra, dst, k + chunk[i] < k_hi ? off[i] : kNtOob, k);
      }
    }
  };
  // RUN: the sums of that many K tiles at a time are added up apart.  The matrix core rounds its accumulator to
  // fp32 after every 8 products, so one long sum of positive terms (a diagonal of X X^T) would lose
  // sqrt(3 K / 8) / 2 last places; in runs of 8 that is 2 to 3 of them at K = 2048.
  typename C::Acc sum[C::RUN ? C::TA : 1][C::RUN ? C::TB : 1];
  if constexpr (C::RUN > 0) {
#pragma unroll
    for (int i = 0; i < C::TA; ++i)
#pragma unroll
      for (int j = 0; j < C::TB; ++j) sum[i][j] = typename C::Acc{0, 0, 0, 0};
  }
  const auto end_of_run = [&](int kt) {
    if constexpr (C::RUN > 0) {
      if (kt % C::RUN == C::RUN - 1) {
#pragma unroll
        for (int i = 0; i < C::TA; ++i)
#pragma unroll
          for (int j = 0; j < C::TB; ++j) {
            sum[i][j] += acc[i][j];
            acc[i][j] = typename C::Acc{0, 0, 0, 0};
          }
      }
    }
  };
  // Every iteration issues one K tile, past the end one of zeros, so that the count of loads in flight is a constant.
  constexpr int LEAD = C::AHEAD ? C::NR : C::NR - 1;  // K tiles on their way before the loop
#pragma unroll
  for (int s = 0; s < LEAD; ++s) issue(s, s);
  const auto barrier = [] {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if constexpr (C::AHEAD) {
    // the fragments of K tile kt + 1 are read while those of kt are multiplied
    NtFrags<C> f[2];
    nt_wait<(C::NR - 1) * C::LPT>();
    barrier();
    f[0].load(lds + kg * C::TILE, wa, wb, lane);
    const auto step = [&](int kt, const NtFrags<C>& now, NtFrags<C>& next) {
      // tile kt + 1 has landed and tile kt's fragments have been read, for every wave
      nt_wait<(C::NR - 2) * C::LPT>();
      barrier();
      issue(kt % C::NR, kt + C::NR);
      next.load(lds + (kt + 1) % C::NR * C::STAGE + kg * C::TILE, wa, wb, lane);
      __builtin_amdgcn_sched_barrier(0);
      now.mma(acc);
      __builtin_amdgcn_sched_barrier(0);
      end_of_run(kt);
    };
    for (int kt = 0; kt < nk; kt += 2) {
      step(kt, f[0], f[1]);
      if (kt + 1 < nk) step(kt + 1, f[1], f[0]);
    }
  } else {
    for (int kt = 0; kt < nk; ++kt) {
      // K tile kt has landed and tile kt - 1 has been read, for every wave; the younger tiles stay in flight
      nt_wait<(C::NR - 2) * C::LPT>();
      barrier();
      issue((kt + C::NR - 1) % C::NR, kt + C::NR - 1);
      nt_tile_mma<C>(lds + kt % C::NR * C::STAGE + kg * C::TILE, wa, wb, lane, acc);
      end_of_run(kt);
    }
  }
  if constexpr (C::RUN > 0) {
#pragma unroll
    for (int i = 0; i < C::TA; ++i)
#pragma unroll
      for (int j = 0; j < C::TB; ++j) acc[i][j] += sum[i][j];
  }
  // the ring may be reused by the epilogue: every wave is past its last read
  nt_wait<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if constexpr (C::KG > 1) {
    // each group adds up its share of the tiles: 1 KiB per tile and wave, 16 bytes per lane
    const auto slot = [&](int g, int t) {
      return reinterpret_cast<typename C::Acc*>(lds + ((g * C::GROUP + wid % C::GROUP) * C::TA * C::TB + t) * 1024) +
             lane;
    };
#pragma unroll
    for (int t = 0; t < C::TA * C::TB; ++t) *slot(kg, t) = acc[t / C::TB][t % C::TB];
    nt_wait<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int t = 0; t < C::TA * C::TB; ++t) {
      if (t % C::KG != kg) continue;
#pragma unroll
      for (int g = 1; g < C::KG; ++g) acc[t / C::TB][t % C::TB] += *slot((kg + g) % C::KG, t);
    }
  }
}

template <class C>
__device__ __forceinline__ void nt_loop(char* lds, const NtOperand& A, const NtOperand& B, int k_lo, int k_hi,
                                        typename C::Acc (&acc)[C::TA][C::TB]) {
  nt_loop_body<C>(lds, A.base, B.base, A, B, k_lo, k_hi, acc);
}

// Consecutive workgroups go to the 8 XCDs in turn: give each XCD a contiguous range of work items, so
// that tiles sharing operand rows share an L2.  (Of items of about equal cost: where a launch holds groups of
// different cost, each group is dealt out by itself.)
__device__ __forceinline__ int nt_xcd_item(int bid, int n) {
  const int q = n / 8, r = n % 8, x = bid % 8;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + bid / 8;
}

}  // namespace mxr
