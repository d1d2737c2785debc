// 8-bit integer products with one scale per row of either operand:
//   y[m][n] = relu(xs[m] * ws[n] * sum_k x[m][k] w[n][k] + bias[n])
// The sum is exact in int32 (K <= 131071: 2^14 * K < 2^31 even where a caller's values reach -128), the
// scales and the bias are applied in fp32, and the result is rounded once to its type.  Integer sums do not
// depend on their order, so any split of K gives the same bits.
//
// quantize_rows makes such an operand: scale = max|x| * (1 / 127) in fp32 (at least 2^-126, so that no quotient
// overflows), q = x / scale rounded to the nearest integer, ties to even; a row that holds an infinity or a NaN gets
// the scale NaN and zeros, so that its products are NaN and other rows are not touched.
#include "tile_nt.h"

#include <algorithm>
#include <cmath>

namespace mxr {
namespace {

// a launch has fewer than 2^32 threads: blocks of at most 512, and rows of at most 1024 threads each
constexpr double kInt8Blocks = 1 << 22;
constexpr int64_t kInt8RowsPerLaunch = 1 << 21;

// ---- rows to 8 bits -----------------------------------------------------------------------------
// bits of |v|: as integers these order like the values, with infinities and NaN on top
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float row_scale(uint32_t peak) {
  return peak >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(peak) * (1.f / 127.f), 0x1p-126f);
}
// Eight values as they lie in memory: 8 x fp32 or 8 x 16 bits.
template <int CODE>
struct Raw8 {
  uint32_t w[CODE == 0 ? 8 : 4];
  // from any address, by the compiler's unaligned loads
  __device__ __forceinline__ void load(const void* x, int64_t i) {
    __builtin_memcpy(w, static_cast<const char*>(x) + i * (CODE == 0 ? 4 : 2), sizeof(w));
  }
  __device__ __forceinline__ float get(int e) const {
    if (CODE == 0) return __uint_as_float(w[e]);
    if (CODE == 1) return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    return f16_to_f32((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
  }
};

// Eight quotients v / s rounded to integers, packed.  A quotient is taken as v * (1 / s), which is within
// 127 * 1.5 * 2^-23 of the fp32 quotient (two roundings against one): only where that lies within 127 * 2^-22 of a tie
// can the two round differently, and only there it is divided.  Adding 1.5 * 2^23 rounds to an integer, ties to even,
// and leaves it in the low bits.  (|v| <= 127 s (1 + 2^-22): never past 127.)
template <int CODE>
__device__ __forceinline__ uint2 to_i8x8(const Raw8<CODE>& v, float s, float inv) {
  constexpr float kBig = 12582912.f;
  uint32_t q[8];
  float off = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = v.get(e) * inv, r = t + kBig;
    off = fmaxf(off, fabsf(t - (r - kBig)));
    q[e] = __float_as_uint(r);
  }
  if (off > 0.5f - 127.f * 0x1p-22f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __float_as_uint(v.get(e) / s + kBig);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(q[4 * h + 1], q[4 * h], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(q[4 * h + 3], q[4 * h + 2], 0x0c0c0400u);
    w[h] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// T threads per row (a wave: four rows per block), which hold it in registers while its peak is found -- NV times eight
// values each -- so that x is read once; HELD = false: a row longer than that is read twice, the second time from the
// caches.  Rows have at least eight values: a thread whose eight would pass the end takes the last eight, and writes
// what its neighbour writes.  Rows of q are ldq apart, with zeros behind K.
template <int CODE, int T, int NV, bool HELD>
__global__ void __launch_bounds__(T < 256 ? 256 : T) quantize_kernel(const void* __restrict__ x, int64_t ld_, int64_t rows,
                                                                     int K, int8_t* __restrict__ q, int ldq,
                                                                     float* __restrict__ scale) {
  const int tid = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (T < 256 ? 256 / T : 1) + threadIdx.x / T;
  if (row >= rows) return;  // (whole waves: rows share a block only where a row is a wave)
  const int64_t x0 = row * ld_;
  int8_t* out = q + row * ldq;
  Raw8<CODE> v[HELD ? NV : 1];
  uint32_t peak = 0;
  if constexpr (HELD) {
#pragma unroll
    for (int c = 0; c < NV; ++c) v[c].load(x, x0 + min((c * T + tid) * 8, K - 8));
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) peak = max(peak, abs_bits(v[c].get(e)));
  } else {
    for (int64_t k = tid * 8; k < K; k += T * 8) {  // (64 bits: K reaches 2^31 - 1)
      v[0].load(x, x0 + min(k, (int64_t)K - 8));
#pragma unroll
      for (int e = 0; e < 8; ++e) peak = max(peak, abs_bits(v[0].get(e)));
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) peak = max(peak, (uint32_t)__shfl_xor((int)peak, o, 64));
  if constexpr (T > 64) {
    __shared__ uint32_t red[T / 64];
    if ((tid & 63) == 0) red[tid >> 6] = peak;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; ++w) peak = max(peak, red[w]);
  }
  const float s = row_scale(peak);
  const bool bad = s != s;
  const float inv = 1.f / s;
  if (tid == 0) {
    scale[row] = s;
    for (int k = K; k < ldq; ++k) out[k] = 0;
  }
  const auto put = [&](const Raw8<CODE>& d, int64_t k) {
    const uint2 w = bad ? make_uint2(0, 0) : to_i8x8(d, s, inv);
    __builtin_memcpy(out + min(k, (int64_t)K - 8), &w, 8);
  };
  if constexpr (HELD) {
#pragma unroll
    for (int c = 0; c < NV; ++c)
      if ((c * T + tid) * 8 < K) put(v[c], (c * T + tid) * 8);
  } else {
    for (int64_t k = tid * 8; k < K; k += T * 8) {
      v[0].load(x, x0 + min(k, (int64_t)K - 8));
      put(v[0], k);
    }
  }
}

// Rows of fewer than eight values: a thread each.
__global__ void __launch_bounds__(256) quantize_short_kernel(const void* __restrict__ x, int code, int64_t ld_,
                                                             int64_t rows, int K, int8_t* __restrict__ q, int ldq,
                                                             float* __restrict__ scale) {
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= rows) return;
  uint32_t peak = 0;
  for (int k = 0; k < K; ++k) peak = max(peak, abs_bits(ld(x, row * ld_ + k, code)));
  const float s = row_scale(peak);
  scale[row] = s;
  for (int k = 0; k < ldq; ++k) q[row * ldq + k] = k >= K || s != s ? 0 : (int8_t)rintf(ld(x, row * ld_ + k, code) / s);
}

template <int CODE>
void quantize(const void* x, int64_t rows, int64_t ld, int K, int8_t* q, int ldq, float* scale, hipStream_t st) {
  const auto go = [&](auto kernel, int t) {
    const int per = t < 256 ? 256 / t : 1;
    kernel<<<(unsigned)((rows + per - 1) / per), t < 256 ? 256 : t, 0, st>>>(x, ld, rows, K, q, ldq, scale);
  };
  // bf16 rows (fp32 and fp16 rows follow the same limits, not measured apart), us, one way and the next: 2048 x 512
  // 2.7 / 2.9 (a wave, 8 values a lane / 32), 2048 x 1024 3.5 / 4.2 but 64 x 1024 3.1 / 2.7 (a wave / 256 threads), 2048 x
  // 4096 7.3 / 8.1 (256 / 512), 2048 x 8192 11 / 15.5 (16 values / 64), 2048 x 32768 39 / 50 (held / read twice); 2400 x
  // 25088 with 256 / 512 / 1024 threads per row 36 / 33 / 41 (5.5 TB/s)
  if (K < 8) quantize_short_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(x, CODE, ld, rows, K, q, ldq, scale);
  else if (K <= 512) go(quantize_kernel<CODE, 64, 1, true>, 64);
  else if (K <= 2048 && rows >= 2048) go(quantize_kernel<CODE, 64, 4, true>, 64);
  else if (K <= 4096) go(quantize_kernel<CODE, 256, 2, true>, 256);
  else if (K <= 8192) go(quantize_kernel<CODE, 512, 2, true>, 512);
  else if (K <= 32768) go(quantize_kernel<CODE, 512, 8, true>, 512);
  else go(quantize_kernel<CODE, 1024, 1, false>, 1024);
}

// ---- products -----------------------------------------------------------------------------------
// 16 bytes at any address: the compiler's unaligned load (one instruction on this target)
__device__ __forceinline__ uint4 load16(const int8_t* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// bytes k .. k + 15 of a row of K, zeros behind its end; nothing behind it is read
__device__ __forceinline__ uint4 load16_tail(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return load16(row + k);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int e = 0; e < K - k; ++e) w[e >> 2] |= (uint32_t)(uint8_t)row[k + e] << (8 * (e & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows of x (the first `mx`) and of w to 16-byte-aligned copies, `lda` bytes apart, zeros behind K, one behind the
// other; from row r0 on, a block each.
__global__ void __launch_bounds__(256) pack_rows_kernel(Int8Args p, int64_t mx, int64_t r0, int8_t* __restrict__ y,
                                                        int lda) {
  const int64_t row = r0 + blockIdx.x;
  const int8_t* src = row < mx ? p.x + row * p.ldx : p.w + (row - mx) * p.ldw;
  for (int k = threadIdx.x * 16; k < lda; k += 4096)
    *reinterpret_cast<uint4*>(y + row * lda + k) = load16_tail(src, k, p.K);
}

__device__ __forceinline__ float int8_out(int acc, float xs, float ws, float bias, int relu) {
  const float v = (float)acc * xs * ws + bias;
  return relu && v < 0.f ? 0.f : v;  // (a NaN stays)
}

// Four outputs n .. n + 3 of row m: the result, or with several runs of K the run's int32 sums.
__device__ __forceinline__ void int8_store(const Int8Args& p, int32_t* part, int splits, int sp, int64_t m, int n,
                                           const nt_i32x4& acc) {
  if (m >= p.M || n >= p.N) return;
  const int cnt = min(4, p.N - n);
  const bool vec = cnt == 4 && p.N % 4 == 0;
  if (splits > 1) {
    int32_t* d = part + ((int64_t)sp * p.M + m) * p.N + n;
    if (vec) *reinterpret_cast<int4*>(d) = make_int4(acc[0], acc[1], acc[2], acc[3]);
    else
      for (int e = 0; e < cnt; ++e) d[e] = acc[e];
    return;
  }
  const float xs = p.xs[m];
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = min(n + e, p.N - 1);
    v[e] = int8_out(acc[e], xs, p.ws[c], p.bias != nullptr ? p.bias[c] : 0.f, p.relu);
  }
  const int64_t at = m * p.N + n;
  if (vec) st4c(p.y, at, p.code, 0, v);
  else
    for (int e = 0; e < cnt; ++e) st(p.y, at + e, v[e], p.code);
}

// Few rows of x, or little of everything: each of KG waves reads both operands' fragments of every KG-th K tile
// straight into registers, two K tiles ahead, with no barrier until the sums of the waves are added up in LDS.  A
// block has 16 rows of w, 16 TB rows of x and one run of K.  One row against 4096 x 25088: 19.5 us, 5.3 TB/s.
//
// Rows at any address (ALIGNED = false) need no copy: the 4 or 5 dwords that hold a lane's 16 bytes are loaded and moved
// down when they are used.  (As one unaligned load they take 5 times as long as an aligned one.)  Behind K the bytes of x
// are cleared; those of w then do not matter.  The last, partial step over K is read by single dwords, so that what is
// past the last row's last dword, and only that, is out of the window.
template <int TB, bool ALIGNED>
struct Int8Stream {
  static constexpr int KG = 8, U = 2, STEP = U * KG * 128;
  const Int8Args& p;
  int n0, k_hi, r, ch, kg;
  int64_t m0;
  __amdgpu_buffer_rsrc_t rw, rx;
  uint32_t ow, ox[TB];  // of this lane's first byte; unaligned: of its dword
  int sw, sx[TB];       // unaligned: the byte within the dword

  // K columns from k_lo on, a multiple of STEP
  __device__ __forceinline__ Int8Stream(const Int8Args& a, int n, int64_t m, int k_lo, int k)
      : p(a), n0(n), k_hi(k), r(threadIdx.x & 15), ch((threadIdx.x & 63) >> 4 << 4),
        kg(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), m0(m) {
    const int wr = min(p.N - n0, 16), xr = (int)min(p.M - m0, (int64_t)16 * TB);
    const int ldw = (int)p.ldw, ldx = (int)p.ldx;  // (below 2^22)
    const char* w = reinterpret_cast<const char*>(p.w) + n0 * p.ldw + k_lo;
    const char* x = reinterpret_cast<const char*>(p.x) + m0 * p.ldx + k_lo;
    const int w0 = ALIGNED ? 0 : (int)(reinterpret_cast<uintptr_t>(w) & 3);
    const int x0 = ALIGNED ? 0 : (int)(reinterpret_cast<uintptr_t>(x) & 3);
    rw = nt_rsrc(w - w0, (w0 + (wr - 1) * ldw + k_hi + 3) & ~3);
    rx = nt_rsrc(x - x0, (x0 + (xr - 1) * ldx + k_hi + 3) & ~3);
    const auto place = [](bool in, int at, uint32_t& off, int& by) {
      by = at & 3;
      off = in ? (uint32_t)(at & ~3) : kNtOob;
    };
    place(r < wr, w0 + r * ldw + ch, ow, sw);
#pragma unroll
    for (int j = 0; j < TB; ++j) place(j * 16 + r < xr, x0 + (j * 16 + r) * ldx + ch, ox[j], sx[j]);
  }
  struct Piece {
    uint4 v;
    uint32_t next;  // unaligned: the dword behind them
  };
  struct Frags {
    Piece w[U][2], x[U][2][TB];
  };
  __device__ __forceinline__ int column(int k0, int u, int h) const { return k0 + (u * KG + kg) * 128 + h * 64; }
  template <bool TAIL>
  __device__ __forceinline__ void piece(Piece& d, __amdgpu_buffer_rsrc_t rs, uint32_t off, int k) const {
    if constexpr (ALIGNED) {
      d.v = nt_load(rs, k + ch < k_hi ? off : kNtOob, k);
    } else if constexpr (!TAIL) {
      d.v = nt_load(rs, off, k);
      d.next = nt_load1(rs, off + 16, k);
    } else {
      const uint32_t at = k + ch < k_hi ? off : kNtOob;
      d.v.x = nt_load1(rs, at, k);
      d.v.y = nt_load1(rs, at + 4, k);
      d.v.z = nt_load1(rs, at + 8, k);
      d.v.w = nt_load1(rs, at + 12, k);
      d.next = nt_load1(rs, at + 16, k);
    }
  }
  // the step at k0; `in` (unaligned whole steps): it is not past the last one
  template <bool TAIL>
  __device__ __forceinline__ void load(Frags& d, int k0, bool in = true) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + (u * KG + kg) * 128 + h * 64;
        piece<TAIL>(d.w[u][h], rw, in ? ow : kNtOob, k);
#pragma unroll
        for (int j = 0; j < TB; ++j) piece<TAIL>(d.x[u][h][j], rx, in ? ox[j] : kNtOob, k);
      }
  }
  static __device__ __forceinline__ uint4 bytes(const Piece& d, int by) {
    if constexpr (ALIGNED) return d.v;
    return make_uint4(__builtin_amdgcn_alignbyte(d.v.y, d.v.x, by), __builtin_amdgcn_alignbyte(d.v.z, d.v.y, by),
                      __builtin_amdgcn_alignbyte(d.v.w, d.v.z, by), __builtin_amdgcn_alignbyte(d.next, d.v.w, by));
  }
  static __device__ __forceinline__ uint32_t keep(uint32_t v, int n) {  // its first n bytes
    return n >= 4 ? v : n <= 0 ? 0 : v & ((1u << (8 * n)) - 1);
  }
  template <bool TAIL>
  __device__ __forceinline__ void mma(const Frags& d, int k0, nt_i32x4 (&acc)[TB]) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 w = bytes(d.w[u][h], sw);
        const int n = k_hi - (k0 + (u * KG + kg) * 128 + h * 64 + ch);  // this lane's bytes up to the end
#pragma unroll
        for (int j = 0; j < TB; ++j) {
          uint4 x = bytes(d.x[u][h][j], sx[j]);
          if (!ALIGNED && TAIL) x = make_uint4(keep(x.x, n), keep(x.y, n - 4), keep(x.z, n - 8), keep(x.w, n - 12));
          acc[j] = nt_mma(w, x, acc[j]);
        }
      }
  }
};

template <int TB, bool ALIGNED>
__global__ void __launch_bounds__(512) int8_stream_kernel(Int8Args p, int nt, int mt, int splits, int run,
                                                         int32_t* __restrict__ part) {
  using S = Int8Stream<TB, ALIGNED>;
  __shared__ nt_i32x4 sums[S::KG][TB][64];
  const int id = nt_xcd_item(blockIdx.x, nt * mt * splits), lane = threadIdx.x & 63;
  const int sp = id / (nt * mt), t = id % (nt * mt), K = min(run, p.K - sp * run);
  const S s(p, t / mt * 16, (int64_t)(t % mt) * 16 * TB, sp * run, K);
  constexpr int STEP = S::STEP;
  nt_i32x4 acc[TB];
#pragma unroll
  for (int j = 0; j < TB; ++j) acc[j] = nt_i32x4{0, 0, 0, 0};
  // whole steps (aligned: all; what is past the end is zeros), and an unaligned rest
  const int end = ALIGNED ? K : K / STEP * STEP;
  typename S::Frags f[2], rest;
  if constexpr (!ALIGNED) s.template load<true>(rest, end);
  s.template load<false>(f[0], 0, ALIGNED || 0 < end);
  for (int k = 0; k < end; k += 2 * STEP) {
    s.template load<false>(f[1], k + STEP, ALIGNED || k + STEP < end);
    s.template mma<false>(f[0], k, acc);
    s.template load<false>(f[0], k + 2 * STEP, ALIGNED || k + 2 * STEP < end);
    s.template mma<false>(f[1], k + STEP, acc);
  }
  if constexpr (!ALIGNED) s.template mma<true>(rest, end, acc);
#pragma unroll
  for (int j = 0; j < TB; ++j) sums[s.kg][j][lane] = acc[j];
  __syncthreads();
  if (s.kg >= TB) return;
  nt_i32x4 v = sums[0][s.kg][lane];
#pragma unroll
  for (int g = 1; g < S::KG; ++g) v += sums[g][s.kg][lane];
  int8_store(p, part, splits, sp, s.m0 + s.kg * 16 + s.r, s.n0 + s.ch / 4, v);
}

// One BA (of N) x BB (of M) tile and one run of K per block: the result itself, or with several runs the
// int32 sums of each, added up by int8_join_kernel.
template <class C>
__global__ void __launch_bounds__(C::THREADS) int8_tile_kernel(Int8Args p, int nt, int mt, int splits, int run,
                                                               int32_t* __restrict__ part) {
  __shared__ __attribute__((aligned(1024))) char ring[C::LDS];
  const int id = nt_xcd_item(blockIdx.x, nt * mt * splits);
  const int sp = id / (nt * mt), t = id % (nt * mt);
  const int n0 = t / mt * C::BA;
  const int64_t m0 = (int64_t)(t % mt) * C::BB;
  const NtOperand A = {reinterpret_cast<const char*>(p.w) + n0 * p.ldw, p.N - n0, (uint32_t)p.ldw, 0};
  const NtOperand B = {reinterpret_cast<const char*>(p.x) + m0 * p.ldx, (int)min((int64_t)C::BB, p.M - m0),
                       (uint32_t)p.ldx, 0};
  typename C::Acc acc[C::TA][C::TB];
  const int k0 = sp * run;
  nt_loop<C>(ring, A, B, k0, min(p.K, k0 + run), acc);
  const int lane = threadIdx.x & 63, wa = C::wa(), wb = C::wb();
#pragma unroll
  for (int i = 0; i < C::TA; ++i)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) {
      if (!C::mine(i, j)) continue;
      const int n = n0 + (wa * C::TA + i) * 16 + (lane >> 4) * 4;
      const int64_t m = m0 + (wb * C::TB + j) * 16 + (lane & 15);
      int8_store(p, part, splits, sp, m, n, acc[i][j]);
    }
}

__global__ void __launch_bounds__(256) int8_join_kernel(Int8Args p, int splits, const int32_t* __restrict__ part) {
  const int64_t total = p.M * p.N;
  const bool vec = p.N % 4 == 0;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += (int64_t)gridDim.x * 1024) {
    nt_i32x4 acc = {0, 0, 0, 0};
    if (vec) {
      for (int s = 0; s < splits; ++s) acc += *reinterpret_cast<const nt_i32x4*>(part + s * total + i);
      const int64_t m = i / p.N;
      int8_store(p, nullptr, 1, 0, m, (int)(i - m * p.N), acc);
    } else {
      for (int64_t e = i; e < min(i + 4, total); ++e) {
        int a = 0;
        for (int s = 0; s < splits; ++s) a += part[s * total + e];
        const int64_t m = e / p.N;
        const int n = (int)(e - m * p.N);
        st(p.y, e, int8_out(a, p.xs[m], p.ws[n], p.bias != nullptr ? p.bias[n] : 0.f, p.relu), p.code);
      }
    }
  }
}

// ---- choice of kernel ---------------------------------------------------------------------------
// Tiles and their measured cost: microseconds per K tile of 128 bytes with up to half of the slots (blocks resident on
// the chip) taken and with all, and per round (start, epilogue).  Runs of K summed apart cost a second launch and
// their traffic.  Measured at these rows only, us: 300 x 4096 x 25088 in 4 runs of 128 x 160 tiles 50, in 8 of 256 x 160
// 56, in 5 of 128 x 128 55, in 8 of 256 x 256 60; 2400 x 4096 x 25088 258 with 256 x 160 (1.9 POPS), 264 256 x 256 (3
// runs), 295 128 x 160, 569 64 x 64; 64 x 4096 x 25088 25 in 4 runs of 64 x 64, 28 in 8 of 128 x 160.
using Int8Tile64 = NtCfg<false, 64, 64, 1, 2, 2, 4>;
using Int8Tile128 = NtCfg<false, 128, 160, 1, 4, 2, 4>;  // (a ring of 4 fills the LDS)
using Int8Tile256 = NtCfg<false, 256, 160, 1, 4, 2, 2>;

struct Int8Cand {
  int bn, bm, slots;
  double half, full, round;
};
constexpr Int8Cand kInt8Tiles[3] = {
    {64, 64, 512, 0.35, 0.60, 2.5}, {128, 160, 256, 0.63, 0.80, 4.0}, {256, 160, 256, 1.00, 1.28, 6.0}};

struct Int8Plan {
  int kind;  // 0, 1: stream of 16 / 32 rows of x, 2 ..: tiles
  bool pack;
  int lda, nt, mt, splits, run;
  int64_t pack_bytes, bytes;
  double us;
};

constexpr int kStreamTiles = Int8Stream<1, true>::STEP / 128;
constexpr int64_t kInt8Ld = 1 << 22;  // rows closer than that: 32-bit offsets within a tile's rows
bool int8_aligned(const void* q, int64_t ld) {  // 16-byte loads
  return (reinterpret_cast<uintptr_t>(q) | (uint64_t)ld) % 16 == 0 && ld < kInt8Ld;
}
bool int8_x_aligned(const Int8Args& a) { return (a.K % 16 == 0 || a.x_padded) && int8_aligned(a.x, a.ldx); }
bool int8_w_aligned(const Int8Args& a) { return a.K % 16 == 0 && int8_aligned(a.w, a.ldw); }

Int8Plan int8_plan(const Int8Args& a) {
  Int8Plan best = {};
  best.us = 1e30;
  const bool ax = int8_x_aligned(a), aw = int8_w_aligned(a), aligned = ax && aw;
  const int lda = (a.K + 15) / 16 * 16, nk = std::max(1, div_up(lda, 128));
  const double mn = (double)a.M * a.N, k = a.K;
  const double hbm = ((double)a.N + a.M) * k / 5.2e6;
  const int64_t packed = (ax ? 0 : a.M) + (aw ? 0 : a.N);  // rows to copy
  const double pack_us = packed ? 3 + 2 * packed * k / 5e6 : 0;
  const int64_t pack_bytes = (packed * lda + 255) / 256 * 256;
  // 16 or 32 rows of x; unaligned rows as they are, or copied first (16 x 4096 x 4099: 8.5 / 20 us, 40 x 64 x 20001:
  // 28 / 16); K whole, or in runs of whole steps where there are few tiles (1 x 512 x 25088: 12.6 / 10.1 us, 15 x 64 x
  // 21419: 16.4 / 12.4)
  for (int s = 0; s < 4; ++s) {
    if (s >= 2 && aligned) break;
    if (s < 2 && (a.ldw >= kInt8Ld || a.ldx >= kInt8Ld)) continue;
    for (int splits : {1, 2, 3, 4, 6, 8, 12}) {
      Int8Plan p = {};
      p.kind = s & 1;
      p.pack = s >= 2;
      p.lda = lda;
      p.nt = div_up(a.N, 16);
      p.mt = div_up(a.M, 16 << p.kind);
      const int run = div_up(div_up(nk, splits), kStreamTiles) * kStreamTiles;
      p.run = run * 128;
      p.splits = div_up(nk, run);
      if (p.splits != splits) continue;
      const double blocks = (double)p.nt * p.mt * splits, rows = std::min<double>(a.M, 16 << p.kind);
      p.us = std::max(hbm, std::ceil(blocks / 512) * (run / kStreamTiles * (aligned || p.pack ? 0.9 : 2.2) + 2)) +
             blocks / splits * (rows + (p.mt > 1 ? 16 : 0)) * k / 12e6 + 2;
      if (splits > 1) p.us += 5 + splits * mn * 8 / 6e6;
      if (p.pack) {
        p.us += pack_us;
        p.pack_bytes = pack_bytes;
      }
      p.bytes = p.pack_bytes + (splits > 1 ? splits * a.M * a.N * 4 : 0);
      if (blocks < kInt8Blocks && p.us < best.us) best = p;
    }
  }
  for (int t = 0; t < 3; ++t) {
    const Int8Cand& c = kInt8Tiles[t];
    for (int splits : {1, 2, 3, 4, 6, 8, 12}) {
      Int8Plan p = {};
      p.kind = 2 + t;
      p.pack = !aligned;
      p.lda = lda;
      p.nt = div_up(a.N, c.bn);
      p.mt = div_up(a.M, c.bm);
      const int run = div_up(nk, splits);
      p.run = run * 128;
      p.splits = div_up(nk, run);
      if (p.splits != splits) continue;
      const double blocks = (double)p.nt * p.mt * splits, whole = std::floor(blocks / c.slots);
      const double rest = blocks - whole * c.slots;
      p.us = whole * (run * c.full + c.round) + 2;
      if (rest > 0) p.us += run * (c.half + (c.full - c.half) * std::max(0.0, 2 * rest / c.slots - 1)) + c.round;
      p.us = std::max(p.us, hbm);
      if (splits > 1) p.us += 3 + splits * mn * 8 / 6e6;
      p.us += pack_us;
      p.pack_bytes = pack_bytes;
      p.bytes = pack_bytes + (splits > 1 ? splits * a.M * a.N * 4 : 0);
      if (blocks < kInt8Blocks && p.us < best.us) best = p;
    }
  }
  return best;
}

template <class C>
void int8_tiles(const Int8Args& a, const Int8Plan& p, int32_t* part, hipStream_t st) {
  int8_tile_kernel<C><<<(unsigned)(p.nt * p.mt * p.splits), C::THREADS, 0, st>>>(a, p.nt, p.mt, p.splits, p.run, part);
}

}  // namespace

void quantize_rows(const void* x, int code, int64_t rows, int64_t ld, int K, int8_t* q, int ldq, float* scale,
                   hipStream_t st) {
  for (int64_t at = 0; at < rows; at += kInt8RowsPerLaunch) {
    const int64_t n = std::min(rows - at, kInt8RowsPerLaunch);
    const char* from = static_cast<const char*>(x) + at * ld * (code == 0 ? 4 : 2);
    if (code == 0) quantize<0>(from, n, ld, K, q + at * ldq, ldq, scale + at, st);
    else if (code == 1) quantize<1>(from, n, ld, K, q + at * ldq, ldq, scale + at, st);
    else quantize<2>(from, n, ld, K, q + at * ldq, ldq, scale + at, st);
  }
}

int64_t int8_matmul_ws(const Int8Args& a) { return int8_plan(a).bytes; }

void int8_matmul(const Int8Args& args, void* ws, hipStream_t st) {
  Int8Args a = args;
  const Int8Plan p = int8_plan(a);
  if (p.pack) {
    int8_t* xb = static_cast<int8_t*>(ws);
    const int64_t mx = int8_x_aligned(a) ? 0 : a.M, nw = int8_w_aligned(a) ? 0 : a.N;
    for (int64_t r0 = 0; r0 < mx + nw; r0 += kInt8RowsPerLaunch)
      pack_rows_kernel<<<(unsigned)std::min(mx + nw - r0, kInt8RowsPerLaunch), 256, 0, st>>>(a, mx, r0, xb, p.lda);
    if (mx > 0) {
      a.x = xb;
      a.ldx = p.lda;
    }
    if (nw > 0) {
      a.w = xb + mx * p.lda;
      a.ldw = p.lda;
    }
    a.K = p.lda;
  }
  int32_t* part = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + p.pack_bytes);
  const auto stream = [&](auto kernel) {
    kernel<<<(unsigned)(p.nt * p.mt * p.splits), 512, 0, st>>>(a, p.nt, p.mt, p.splits, p.run, part);
  };
  const bool aligned = int8_x_aligned(a) && int8_w_aligned(a);
  if (p.kind == 0 && aligned) stream(int8_stream_kernel<1, true>);
  else if (p.kind == 0) stream(int8_stream_kernel<1, false>);
  else if (p.kind == 1 && aligned) stream(int8_stream_kernel<2, true>);
  else if (p.kind == 1) stream(int8_stream_kernel<2, false>);
  else if (p.kind == 2) int8_tiles<Int8Tile64>(a, p, part, st);
  else if (p.kind == 3) int8_tiles<Int8Tile128>(a, p, part, st);
  else int8_tiles<Int8Tile256>(a, p, part, st);
  if (p.splits > 1)
    int8_join_kernel<<<(unsigned)std::min<int64_t>(div_up(a.M * a.N, 1024), 4096), 256, 0, st>>>(a, p.splits, part);
}

}  // namespace mxr
