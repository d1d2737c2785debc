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

namespace mxr {
namespace {

// ---- rows to 8 bits -----------------------------------------------------------------------------
// bits of |v|: as integers these order like the values, with infinities and NaN on top
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float row_scale(uint32_t peak) {
  return peak >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(peak) * (1.f / 127.f), 0x1p-126f);
}
__device__ __forceinline__ int to_i8(float v, float s) {
  return (int)rintf(v / s);  // |v| <= 127 s (1 + 2^-22): never past 127
}

// One block per row; the second read of the row comes from the caches.
template <int CODE, bool VEC>
__global__ void __launch_bounds__(256) quantize_kernel(const void* __restrict__ x, int64_t ld_, int K,
                                                       int8_t* __restrict__ q, float* __restrict__ scale) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  uint32_t peak = 0;
  const int64_t x0 = row * ld_, q0 = row * K;
  if (VEC) {
    for (int k = tid * 8; k < K; k += 2048) {
      float v[8];
      ld8c(x, x0 + k, CODE, 0, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) peak = max(peak, abs_bits(v[e]));
    }
  } else {
    for (int k = tid; k < K; k += 256) peak = max(peak, abs_bits(ld(x, x0 + k, CODE)));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) peak = max(peak, (uint32_t)__shfl_xor((int)peak, o, 64));
  __shared__ uint32_t red[4];
  if ((tid & 63) == 0) red[tid >> 6] = peak;
  __syncthreads();
  peak = max(max(red[0], red[1]), max(red[2], red[3]));
  const float s = row_scale(peak);
  if (tid == 0) scale[row] = s;
  const bool bad = s != s;
  if (VEC) {
    for (int k = tid * 8; k < K; k += 2048) {
      float v[8];
      ld8c(x, x0 + k, CODE, 0, v);
      uint32_t w[2] = {0, 0};
      if (!bad) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)(to_i8(v[e], s) & 255) << (8 * (e & 3));
      }
      *reinterpret_cast<uint2*>(q + q0 + k) = make_uint2(w[0], w[1]);
    }
  } else {
    for (int k = tid; k < K; k += 256) q[q0 + k] = bad ? 0 : (int8_t)to_i8(ld(x, x0 + k, CODE), s);
  }
}

// ---- products -----------------------------------------------------------------------------------
// Rows to a 16-byte-aligned copy, `lda` bytes apart, zeros behind K.
__global__ void __launch_bounds__(256) pack_rows_kernel(const int8_t* __restrict__ x, int64_t ld_, int K,
                                                        int8_t* __restrict__ y, int lda) {
  const int8_t* src = x + (int64_t)blockIdx.x * ld_;
  int8_t* dst = y + (int64_t)blockIdx.x * lda;
  for (int k = threadIdx.x * 4; k < lda; k += 1024) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= k + e < K ? (uint32_t)(uint8_t)src[k + e] << (8 * e) : 0u;
    *reinterpret_cast<uint32_t*>(dst + k) = w;
  }
}

__device__ __forceinline__ float int8_out(int acc, float xs, float ws, float bias, int relu) {
  const float v = (float)acc * xs * ws + bias;
  return relu && v < 0.f ? 0.f : v;  // (a NaN stays)
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
      if (m >= p.M || n >= p.N) continue;
      const int cnt = min(4, p.N - n);
      if (splits > 1) {
        int32_t* d = part + ((int64_t)sp * p.M + m) * p.N + n;
        if (cnt == 4 && p.N % 4 == 0) *reinterpret_cast<int4*>(d) = make_int4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        else
          for (int e = 0; e < cnt; ++e) d[e] = acc[i][j][e];
        continue;
      }
      const float xs = p.xs[m];
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = min(n + e, p.N - 1);
        v[e] = int8_out(acc[i][j][e], xs, p.ws[c], p.bias != nullptr ? p.bias[c] : 0.f, p.relu);
      }
      const int64_t at = m * p.N + n;
      if (cnt == 4 && p.N % 4 == 0) st4c(p.y, at, p.code, 0, v);
      else
        for (int e = 0; e < cnt; ++e) st(p.y, at + e, v[e], p.code);
    }
}

__global__ void __launch_bounds__(256) int8_join_kernel(Int8Args p, int splits, const int32_t* __restrict__ part) {
  const int64_t total = p.M * p.N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    int acc = 0;
    for (int s = 0; s < splits; ++s) acc += part[s * total + i];
    const int64_t m = i / p.N;
    const int n = (int)(i - m * p.N);
    st(p.y, i, int8_out(acc, p.xs[m], p.ws[n], p.bias != nullptr ? p.bias[n] : 0.f, p.relu), p.code);
  }
}

using Int8Tile = NtCfg<false, 64, 64, 1, 2, 2, 4>;

struct Int8Plan {
  bool pack;
  int lda, nt, mt, splits, run;
  int64_t pack_bytes, bytes;
};

Int8Plan int8_plan(const Int8Args& a) {
  using C = Int8Tile;
  Int8Plan p;
  // 16-byte loads, and 32-bit offsets within a tile's rows
  const auto aligned = [](const void* q, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(q) | (uint64_t)ld) % 16 == 0 && ld < (1 << 22);
  };
  p.pack = a.K % 16 != 0 || !aligned(a.x, a.ldx) || !aligned(a.w, a.ldw);
  p.lda = (a.K + 15) / 16 * 16;
  p.nt = div_up(a.N, C::BA);
  p.mt = div_up(a.M, C::BB);
  const int nk = div_up(p.lda, 128);
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / ((int64_t)p.nt * p.mt), nk / 8));
  p.run = std::max(1, div_up(nk, p.splits)) * 128;
  p.splits = std::max(1, div_up(nk * 128, p.run));
  p.pack_bytes = p.pack ? ((a.M + a.N) * p.lda + 255) / 256 * 256 : 0;
  p.bytes = p.pack_bytes + (p.splits > 1 ? p.splits * a.M * a.N * 4 : 0);
  return p;
}

}  // namespace

void quantize_rows(const void* x, int code, int64_t rows, int64_t ld, int K, int8_t* q, float* scale, hipStream_t st) {
  const int64_t esize = code == 0 ? 4 : 2;
  const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) | (uint64_t)(ld * esize)) % 16 == 0;
#define MXR_Q(CODE)                                                                                        \
  do {                                                                                                     \
    if (vec) quantize_kernel<CODE, true><<<(unsigned)rows, 256, 0, st>>>(x, ld, K, q, scale);              \
    else quantize_kernel<CODE, false><<<(unsigned)rows, 256, 0, st>>>(x, ld, K, q, scale);                 \
  } while (0)
  if (code == 0) MXR_Q(0);
  else if (code == 1) MXR_Q(1);
  else MXR_Q(2);
#undef MXR_Q
}

int64_t int8_matmul_ws(const Int8Args& a) { return int8_plan(a).bytes; }

void int8_matmul(const Int8Args& args, void* ws, hipStream_t st) {
  using C = Int8Tile;
  Int8Args a = args;
  const Int8Plan p = int8_plan(a);
  if (p.pack) {
    int8_t* xb = static_cast<int8_t*>(ws);
    int8_t* wb = xb + a.M * p.lda;
    pack_rows_kernel<<<(unsigned)a.M, 256, 0, st>>>(a.x, a.ldx, a.K, xb, p.lda);
    pack_rows_kernel<<<(unsigned)a.N, 256, 0, st>>>(a.w, a.ldw, a.K, wb, p.lda);
    a.x = xb;
    a.w = wb;
    a.ldx = a.ldw = a.K = p.lda;
  }
  int32_t* part = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + p.pack_bytes);
  const int64_t grid = (int64_t)p.nt * p.mt * p.splits;
  int8_tile_kernel<C><<<(unsigned)grid, C::THREADS, 0, st>>>(a, p.nt, p.mt, p.splits, p.run, part);
  if (p.splits > 1)
    int8_join_kernel<<<(unsigned)std::min<int64_t>(div_up(a.M * a.N, 256), 4096), 256, 0, st>>>(a, p.splits, part);
}

}  // namespace mxr
