// Newton-Schulz orthogonalisation of weight-shaped matrices, and the Muon update built on it.
//
// For G (r x c), X0 = G / (|G|_F + eps), turned so that X is m x n with m <= n; a step is
//   A = X X^T,  P = a I + b A + c A^2,  X <- P X        (a, b, c) = (3.4445, -4.7750, 2.0315).
// P is a polynomial of A, so consecutive steps stay in the small dimension: X_{k+1} = P_k X_k gives
// A_{k+1} = P_k A_k P_k, and X_k = P_{k-1} .. P_0 X_0 = Q X_0.  All of A, P, Q, P A commute and are
// symmetric, so every m x m product computes the tiles on and above the diagonal and mirrors them.  Steps
// are gathered by twos (5 = 2 + 2 + 1), after which A is formed from X anew: 9 n m^2 + 11 m^3 operations
// for five steps against 15 n m^2 + 5 m^3 step by step.  Longer groups would be cheaper and lose: A holds
// sigma^2, so what rounding does to the smallest directions is magnified by the square of the gain (3.44 per
// step).  Measured on gradient-like matrices (a few strong directions over noise), error against 64 bits over that
// of the plain recurrence in fp32: by twos 0.25 to 1.1 (six of 12 560 random cases 1.5 to 2.1, with a smaller side of 8
// to 15), 3 + 2 up to 10, all five in one up to 30 and more.
//
// Operands are fp16 pairs (22 bits, tile_nt.h).  Single fp16 or bf16 operands were found 1e-3 to 3e-1 off: a
// rounding of X in a small singular direction grows with that direction, up to 485 times.  fp16 holds
// 22 bits in two planes only near the top of its range, so every buffer carries the largest power-of-two
// scale that its spectral norm allows below 65504: X and A 2^15 (|X| <= 1.2025, |A| and |P A| <= 1.446), P and Q
// 2^12 (|Q| <= 3.4445^2 = 11.9).
//
// Every m x m product is made exactly symmetric (its lower half is the mirrored upper half): the commuting of A, P
// and Q is what the gathering rests on, and antisymmetric rounding left in them was found up to 100
// times larger in the result (2 x 3 matrices, 1e-4).
//
// One launch runs a product of every matrix of the call: a block finds its matrix among the groups of
// equal shape that the launch carries by value (no tables in memory, so a call can be captured).  Small matrices, bound
// by launches, take other ways: ns_chain_kernel, and ns_block_kernel for whole matrices.
//
// Times on this card (5 steps): 64 x 576 74 us, 23 of 256 x 2304 300 us, 4096 x 4096 3.7 ms; the update of ResNet-101's
// filters 1.36 ms, of VGG16's 17.0 ms.  4096 x 4096 and VGG16 run at 89 and 85 % of
// the rate of a large fp16 product.
#include "tile_nt.h"

#include <algorithm>
#include <cmath>

namespace mxr {
namespace {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr float kNsX = 32768.f, kNsP = 4096.f;  // scales of X and A, of P and Q

struct NsArgs {
  NsGroup g[kNsMaxGroups];
  int64_t off[kNsMaxMats];  // element offset of each matrix in the flat buffers
  int ng;
  uint16_t* ws;
  double* part;  // partial sums of squares: kNsParts per matrix
};

enum NsSlot { kA, kT, kP0, kP1, kQ, kSlots };

// The group of work item `id` (prefix sums over groups) -> the item's number within the group.
__device__ __forceinline__ int ns_find(const NsArgs& p, int& id, int NsGroup::*start) {
  int k = 0;
  while (k + 1 < p.ng && id >= p.g[k + 1].*start) ++k;
  id -= p.g[k].*start;
  return k;
}

// Buffers hold fp16 pairs in panels (tile_nt.h): for every 32 columns, the lines of all rows, each 32 hi and 32 lo.
__host__ __device__ __forceinline__ int64_t ns_size(int rows, int cols) { return (int64_t)rows * cols * 2; }
__host__ __device__ __forceinline__ int64_t ns_stride(const NsGroup& g) {  // of one matrix, in fp16 elements
  return 2 * ns_size(g.mp, g.np) + kSlots * ns_size(g.mp, g.mp);
}
// matrix mi of group g: X (mp x np) in two versions, m x m slots
__device__ __forceinline__ uint16_t* ns_x(const NsArgs& p, const NsGroup& g, int mi, int ver) {
  return p.ws + g.ws + mi * ns_stride(g) + ver * ns_size(g.mp, g.np);
}
__device__ __forceinline__ uint16_t* ns_sq(const NsArgs& p, const NsGroup& g, int mi, int slot) {
  return ns_x(p, g, mi, 2) + slot * ns_size(g.mp, g.mp);
}

__device__ __forceinline__ void split_f16(float v, uint16_t& hi, uint16_t& lo) {
  hi = f32_to_f16(v);
  lo = f32_to_f16(v - f16_to_f32(hi));
}
// element (row, col) of a pair buffer of `rows` rows: its hi value; the lo value is 32 further
__device__ __forceinline__ int64_t ns_at(int row, int rows, int col) {
  return ((int64_t)(col >> 5) * rows + row) * 64 + (col & 31);
}
__device__ __forceinline__ void st4_pair(uint16_t* d, const float v[4]) {  // 4 columns, the first a multiple of 4
  uint16_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) split_f16(v[e], h[e], l[e]);
  *reinterpret_cast<ushort4*>(d) = make_ushort4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<ushort4*>(d + 32) = make_ushort4(l[0], l[1], l[2], l[3]);
}

// ---- the values that are orthogonalised ---------------------------------------------------------
// u = G, or for the update g' = clip(rescale g), mom' = mu mom + g', u = g' + mu mom' (nesterov) or mom'.
// A NaN passes the clip (fminf / fmaxf would make it -clip and hide it).
__device__ __forceinline__ float ns_clip(const NsUpdate& u, float g) {
  g *= u.rescale;
  if (u.clip > 0.f) g = g < -u.clip ? -u.clip : g > u.clip ? u.clip : g;
  return g;
}

// 1 / (|u| + eps).  Finite also where |u| is zero and eps below 1 / DBL_MAX, so that zeros stay zero: any other |u| of
// fp32 values is at least 2^-149.
__device__ __forceinline__ double ns_inverse(double squares, double eps) {
  const double norm = sqrt(squares) + eps;
  return norm < 1e-300 ? 1e300 : 1.0 / norm;  // (NaN: NaN)
}

__device__ __forceinline__ void ns_ld4(const void* p, int64_t i, int code, bool vec, int n, float v[4]) {
  if (vec) {
    ld4c(p, i, code, 0, v);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = k < n ? ld(p, i + k, code) : 0.f;
}

// Pass 1: momentum, and the partial sums of u^2 (fp64: no overflow, no order dependence worth naming).
// A matrix is cut into kNsParts runs of equal length (a multiple of 1024 elements).
__global__ void __launch_bounds__(256) ns_norm_kernel(NsArgs p, NsUpdate u) {
  int id = blockIdx.x;
  const int k = ns_find(p, id, &NsGroup::ew);
  const NsGroup& g = p.g[k];
  const int mi = id / g.parts, part = id % g.parts;
  const int64_t n = (int64_t)g.rows * g.cols, off = p.off[g.first + mi];
  const int64_t lo = (int64_t)part * g.run, hi = min(n, lo + g.run);
  const bool vec = off % 4 == 0 && u.vec;
  double s = 0.0;
  for (int64_t i = lo + threadIdx.x * 4; i < hi; i += 1024) {
    const int cnt = (int)min((int64_t)4, hi - i);
    float v[4];
    ns_ld4(u.grad, off + i, u.code, vec && cnt == 4, cnt, v);
    if (u.mom != nullptr) {
      float m[4];
      ns_ld4(u.mom, off + i, 0, vec && cnt == 4, cnt, m);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float gv = ns_clip(u, v[e]);
        m[e] = u.mu * m[e] + gv;
        v[e] = u.nesterov ? gv + u.mu * m[e] : m[e];
      }
      if (vec && cnt == 4) *reinterpret_cast<float4*>(u.mom + off + i) = make_float4(m[0], m[1], m[2], m[3]);
      else
        for (int e = 0; e < cnt; ++e) u.mom[off + i + e] = m[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s += e < cnt ? (double)v[e] * (double)v[e] : 0.0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  __shared__ double red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) p.part[(int64_t)(g.first + mi) * kNsParts + part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Pass 2: X = u / (|u| + eps) as scaled fp16 pairs with zeroed padding; 64 x 64 elements per block, those of a tall
// matrix turned in LDS.  Clears the gradient it consumed when asked to.
__global__ void __launch_bounds__(256) ns_init_kernel(NsArgs p, NsUpdate u) {
  int id = blockIdx.x;
  const int k = ns_find(p, id, &NsGroup::init);
  const NsGroup& g = p.g[k];
  const int rt = (g.tall ? g.np : g.mp) / 64, ct = (g.tall ? g.mp : g.np) / 64;
  const int mi = id / (rt * ct), t = id % (rt * ct), r0 = t / ct * 64, c0 = t % ct * 64;
  const int64_t off = p.off[g.first + mi];
  const int tid = threadIdx.x;
  // the norm, from the partial sums in a fixed order
  double s = 0.0;
  const double* part = p.part + (int64_t)(g.first + mi) * kNsParts;
  for (int i = tid; i < g.parts; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  __shared__ double red[4];
  __shared__ float tile[64][65];
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  const double f = ns_inverse((red[0] + red[1]) + (red[2] + red[3]), u.eps) * (double)kNsX;
  const int lr = tid >> 4, lc = (tid & 15) * 4;
  uint16_t* x = ns_x(p, g, mi, 0);
  // elements as they lie in memory: 4 columns of rows lr, lr + 16, ..
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = r0 + lr + 16 * q, c = c0 + lc;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const int cnt = r < g.rows ? max(0, min(4, g.cols - c)) : 0;
    if (cnt > 0) {
      const int64_t i = off + (int64_t)r * g.cols + c;
      const bool vec = u.vec && i % 4 == 0 && cnt == 4;
      ns_ld4(u.grad, i, u.code, vec, cnt, v);
      if (u.mom != nullptr) {
        float m[4];
        ns_ld4(u.mom, i, 0, vec, cnt, m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float gv = ns_clip(u, v[e]);
          v[e] = u.nesterov ? gv + u.mu * m[e] : m[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = e < cnt ? (float)((double)v[e] * f) : 0.f;
      if (u.zero != nullptr)
        for (int e = 0; e < cnt; ++e) st(u.zero, i + e, 0.f, u.zero_code);
    }
    if (!g.tall) {
      st4_pair(x + ns_at(r, g.mp, c), v);
      continue;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[lr + 16 * q][lc + e] = v[e];
  }
  if (!g.tall) return;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int a = lr + 16 * q;
    float t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = tile[lc + e][a];
    st4_pair(x + ns_at(c0 + a, g.mp, r0 + lc), t);
  }
}

// ---- products -----------------------------------------------------------------------------------
__device__ __forceinline__ NtOperand ns_op(const uint16_t* base, int row0, int rows) {
  return {reinterpret_cast<const char*>(base + (int64_t)row0 * 64), rows - row0, 0, (int64_t)rows * 128};
}
// columns col0 .. of a buffer of `rows` x `cols`, as the rows of a turned operand
__device__ __forceinline__ NtOperand ns_op_turned(const uint16_t* base, int rows, int col0, int cols) {
  return {reinterpret_cast<const char*>(base + ns_at(0, rows, col0)), cols - col0, 0, (int64_t)rows * 128};
}

// A 16 x 16 tile turned within the wave: lane l holds rows 4 (l >> 4) .. + 3 of column l & 15, and gets columns
// 4 (l >> 4) .. + 3 of row l & 15.  `s`: 16 x 20 floats of this wave alone (its LDS accesses stay in order).
__device__ __forceinline__ void ns_turn(float* s, int lane, const float v[4], float t[4]) {
  const int g = lane >> 4, r = lane & 15;
#pragma unroll
  for (int e = 0; e < 4; ++e) s[(4 * g + e) * 20 + r] = v[e];
  __builtin_amdgcn_wave_barrier();
  const float4 q = *reinterpret_cast<const float4*>(s + r * 20 + 4 * g);
  __builtin_amdgcn_wave_barrier();
  t[0] = q.x; t[1] = q.y; t[2] = q.z; t[3] = q.w;
}

// upper-triangle tile t (row-major) of nt x nt tiles
__device__ __forceinline__ void ns_tri(int t, int nt, int& ti, int& tj) {
  ti = 0;
  while (t >= nt - ti) {
    t -= nt - ti;
    ++ti;
  }
  tj = ti + t;
}

// Symmetric m x m products.  kGram: A = X X^T; kPoly: P = a I + b A + c A^2; kMul: L R of two slots.
// (ls, rs: the operands' slots, of kGram the version of X; ds: the result's)
enum NsKind { kGram, kPoly, kMul };

template <class C, int KIND>
__global__ void __launch_bounds__(C::THREADS) ns_sym_kernel(NsArgs p, int ls, int rs, int ds) {
  static_assert(C::BA == C::BB, "square tiles");
  __shared__ __attribute__((aligned(1024))) char ring[C::LDS];
  int id = blockIdx.x;
  const int k = ns_find(p, id, KIND == kGram ? &NsGroup::gram : &NsGroup::sym);
  const NsGroup& g = p.g[k];
  const int nt = (g.mp + C::BA - 1) / C::BA, tri = nt * (nt + 1) / 2;
  id = nt_xcd_item(id, g.count * tri);
  const int mi = id / tri;
  int ti, tj;
  ns_tri(id % tri, nt, ti, tj);
  nt_f32x4 acc[C::TA][C::TB];
  const int a0 = tj * C::BA, b0 = ti * C::BB;  // 4 consecutive elements of a lane run along rows of A: columns of C
  if constexpr (KIND == kGram) {
    const uint16_t* x = ns_x(p, g, mi, ls);
    nt_loop<C>(ring, ns_op(x, a0, g.mp), ns_op(x, b0, g.mp), 0, g.np * 4, acc);
  } else {
    const uint16_t *l = ns_sq(p, g, mi, ls), *r = ns_sq(p, g, mi, rs);
    nt_loop<C>(ring, ns_op(l, a0, g.mp), ns_op(r, b0, g.mp), 0, g.mp * 4, acc);
  }
  float* scratch = C::scratch(ring);
  uint16_t* dst = ns_sq(p, g, mi, ds);
  const uint16_t* av = ns_sq(p, g, mi, kA);
  const int lane = threadIdx.x & 63, wa = C::wa(), wb = C::wb();
  const float f = KIND == kGram ? 1.f / kNsX : KIND == kPoly ? 1.f / (kNsX * kNsX) : 1.f / kNsP;
#pragma unroll
  for (int i = 0; i < C::TA; ++i)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) {
      if (!C::mine(i, j)) continue;
      const int ca = a0 + (wa * C::TA + i) * 16 + (lane >> 4) * 4;  // column of C
      const int cb = b0 + (wb * C::TB + j) * 16 + (lane & 15);      // row of C
      if (a0 + (wa * C::TA + i) * 16 >= g.mp || b0 + (wb * C::TB + j) * 16 >= g.mp) continue;  // (wave-uniform)
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * f;
      if constexpr (KIND == kPoly) {
        const uint16_t* q = av + ns_at(cb, g.mp, ca);
        const ushort4 h = *reinterpret_cast<const ushort4*>(q), l = *reinterpret_cast<const ushort4*>(q + 32);
        const float ah[4] = {f16_to_f32(h.x) + f16_to_f32(l.x), f16_to_f32(h.y) + f16_to_f32(l.y),
                             f16_to_f32(h.z) + f16_to_f32(l.z), f16_to_f32(h.w) + f16_to_f32(l.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = kNsP * ((ca + e == cb ? kNsA : 0.f) + kNsB * (ah[e] / kNsX) + kNsC * v[e]);
      }
      // the turned tile: rows ca.., columns cb..; the lower half of a diagonal block comes from the upper half
      float t[4];
      ns_turn(scratch, lane, v, t);
      const int ra = a0 + (wa * C::TA + i) * 16 + (lane & 15), rb = b0 + (wb * C::TB + j) * 16 + (lane >> 4) * 4;
      if (ti != tj) {
        st4_pair(dst + ns_at(cb, g.mp, ca), v);
        st4_pair(dst + ns_at(ra, g.mp, rb), t);
        continue;
      }
      const int tile_a = wa * C::TA + i, tile_b = wb * C::TB + j;
      if (tile_a > tile_b) {
        st4_pair(dst + ns_at(cb, g.mp, ca), v);
        st4_pair(dst + ns_at(ra, g.mp, rb), t);
      } else if (tile_a == tile_b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ca + e >= cb ? v[e] : t[e];
        st4_pair(dst + ns_at(cb, g.mp, ca), v);
      }
    }
}

// A = X X^T of few matrices with long rows: a tile's K is cut into g.splits runs of g.run_k K tiles, whose fp32 sums
// go to the version of X that is not in use (splits <= np / mp), row-major mp x mp each; ns_join_kernel adds them up.
template <class C>
__global__ void __launch_bounds__(C::THREADS) ns_gram_part_kernel(NsArgs p, int ver) {
  __shared__ __attribute__((aligned(1024))) char ring[C::LDS];
  int id = blockIdx.x;
  const int k = ns_find(p, id, &NsGroup::gram);
  const NsGroup& g = p.g[k];
  const int nt = (g.mp + C::BA - 1) / C::BA, tri = nt * (nt + 1) / 2;
  id = nt_xcd_item(id, g.count * tri * g.splits);
  const int mi = id / (tri * g.splits), sp = id / tri % g.splits;
  int ti, tj;
  ns_tri(id % tri, nt, ti, tj);
  const int a0 = tj * C::BA, b0 = ti * C::BB, k0 = sp * g.run_k;
  const uint16_t* x = ns_x(p, g, mi, ver) + (int64_t)k0 * g.mp * 64;
  nt_f32x4 acc[C::TA][C::TB];
  nt_loop<C>(ring, ns_op(x, a0, g.mp), ns_op(x, b0, g.mp), 0, min(g.run_k, g.np / 32 - k0) * 128, acc);
  float* dst = reinterpret_cast<float*>(ns_x(p, g, mi, ver ^ 1)) + (int64_t)sp * g.mp * g.mp;
  const int lane = threadIdx.x & 63, wa = C::wa(), wb = C::wb();
#pragma unroll
  for (int i = 0; i < C::TA; ++i)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) {
      if (!C::mine(i, j)) continue;
      const int ca = a0 + (wa * C::TA + i) * 16 + (lane >> 4) * 4, cb = b0 + (wb * C::TB + j) * 16 + (lane & 15);
      if (ca >= g.mp || cb >= g.mp) continue;
      *reinterpret_cast<nt_f32x4*>(dst + (int64_t)cb * g.mp + ca) = acc[i][j];
    }
}

__global__ void __launch_bounds__(256) ns_join_kernel(NsArgs p, int ver) {
  __shared__ float tile[64][65];
  int id = blockIdx.x;
  const int k = ns_find(p, id, &NsGroup::join);
  const NsGroup& g = p.g[k];
  const int nt = g.mp / 64, tri = nt * (nt + 1) / 2, mi = id / tri;
  int ti, tj;
  ns_tri(id % tri, nt, ti, tj);
  const float* src = reinterpret_cast<const float*>(ns_x(p, g, mi, ver ^ 1));
  uint16_t* dst = ns_sq(p, g, mi, kA);
  const int lr = threadIdx.x >> 4, lc = (threadIdx.x & 15) * 4, r0 = ti * 64, c0 = tj * 64;
  const int64_t mm = (int64_t)g.mp * g.mp;
  nt_f32x4 s[4] = {};
  for (int sp = 0; sp < g.splits; ++sp)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      s[q] += *reinterpret_cast<const nt_f32x4*>(src + sp * mm + (int64_t)(r0 + lr + 16 * q) * g.mp + c0 + lc);
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[lr + 16 * q][lc + e] = s[q][e] * (1.f / kNsX);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int a = lr + 16 * q;
    float v[4], t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = tile[lc + e][a];
      v[e] = ti == tj && lc + e < a ? t[e] : tile[a][lc + e];  // (a diagonal tile: its upper half both ways)
    }
    st4_pair(dst + ns_at(r0 + a, g.mp, c0 + lc), v);
    if (ti != tj) st4_pair(dst + ns_at(c0 + a, g.mp, r0 + lc), t);
  }
}

// The m x m products of a group of steps in one block, for mp <= kNsChain: A (from kA) to P0, or with `two` to Q = P1
// P0, in slot kQ.  Two matrices of LDS, in the layout of a K tile of the products above, K tile after K tile: s0
// holds A, then T = P0 A, A' = T P0 and P1; s1 holds P0.  A product's 16 x 16 tiles on and above the diagonal are
// dealt to the 16 waves, held in registers until every wave has read its operands, and written with their mirror
// images.  Five launches of 5 us or more become one of 8 (64 x 576: 116 -> 74 us in all).  Here the lo lo products
// are taken too: their cost does not show, and small matrices come out 10 to 15 % nearer.
constexpr int kNsChain = 128;

__device__ __forceinline__ int ns_lds_at(int row, int rows, int col) {  // byte of the hi value; the lo value's is ^ 64
  return ((col >> 5) * rows + row) * 128 + ((((col & 31) >> 3) ^ ((row >> 1) & 7)) << 4) + (col & 7) * 2;
}

__global__ void __launch_bounds__(1024) ns_chain_kernel(NsArgs p, int two) {
  constexpr int kTiles = (kNsChain / 16) * (kNsChain / 16 + 1) / 2;
  constexpr int kMine = (kTiles + 15) / 16;  // tiles of a wave, at most
  __shared__ __attribute__((aligned(1024))) char lds[2 * kNsChain * kNsChain * 4 + 16 * 1280];
  char *s0 = lds, *s1 = lds + kNsChain * kNsChain * 4;
  int mi = blockIdx.x;
  const int k = ns_find(p, mi, &NsGroup::chain);
  const NsGroup& g = p.g[k];
  const int mp = g.mp, nt = mp / 16, tri = nt * (nt + 1) / 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float* scratch = reinterpret_cast<float*>(lds + 2 * kNsChain * kNsChain * 4 + wave * 1280);
  const char* a = reinterpret_cast<const char*>(ns_sq(p, g, mi, kA));
  uint16_t* out = ns_sq(p, g, mi, kQ);
  for (int i = threadIdx.x; i < mp * mp / 4; i += 1024) {  // 16 bytes: chunk i & 7 of line i >> 3
    const int row = (i >> 3) % mp;
    *reinterpret_cast<uint4*>(s0 + (i >> 3) * 128 + (((i & 7) ^ ((row >> 1) & 7)) << 4)) =
        reinterpret_cast<const uint4*>(a)[i];
  }
  __syncthreads();
  // dst = a I + b L + c L L (poly) or L R, to LDS or (nullptr) to `out`
  const auto product = [&](const char* L, const char* R, char* dst, bool poly) {
    nt_f32x4 acc[kMine];
    int ti[kMine], tj[kMine];
#pragma unroll
    for (int t = 0; t < kMine; ++t) {
      acc[t] = nt_f32x4{0, 0, 0, 0};
      if (wave + 16 * t >= tri) continue;
      ns_tri(wave + 16 * t, nt, ti[t], tj[t]);
      for (int kt = 0; kt < mp / 32; ++kt) {
        uint4 x[2], y[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x[h] = nt_frag(L + kt * mp * 128, tj[t] * 16 + (lane & 15), h, lane);
          y[h] = nt_frag(R + kt * mp * 128, ti[t] * 16 + (lane & 15), h, lane);
        }
        acc[t] = nt_mma(x[1], y[1], acc[t]);
        acc[t] = nt_mma(x[0], y[1], acc[t]);
        acc[t] = nt_mma(x[1], y[0], acc[t]);
        acc[t] = nt_mma(x[0], y[0], acc[t]);
      }
    }
    __syncthreads();
    const auto put = [&](int row, int col, const float v[4]) {
      if (dst == nullptr) {
        st4_pair(out + ns_at(row, mp, col), v);
        return;
      }
      uint16_t h[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) split_f16(v[e], h[e], l[e]);
      const int at = ns_lds_at(row, mp, col);
      *reinterpret_cast<ushort4*>(dst + at) = make_ushort4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<ushort4*>(dst + (at ^ 64)) = make_ushort4(l[0], l[1], l[2], l[3]);
    };
#pragma unroll
    for (int t = 0; t < kMine; ++t) {
      if (wave + 16 * t >= tri) continue;
      const int row = ti[t] * 16 + (lane & 15), col = tj[t] * 16 + (lane >> 4) * 4;
      float v[4], m[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[t][e] * (poly ? 1.f / (kNsX * kNsX) : 1.f / kNsP);
      if (poly) {
        const int at = ns_lds_at(row, mp, col);
        const ushort4 h = *reinterpret_cast<const ushort4*>(L + at);
        const ushort4 l = *reinterpret_cast<const ushort4*>(L + (at ^ 64));
        const float av[4] = {f16_to_f32(h.x) + f16_to_f32(l.x), f16_to_f32(h.y) + f16_to_f32(l.y),
                             f16_to_f32(h.z) + f16_to_f32(l.z), f16_to_f32(h.w) + f16_to_f32(l.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = kNsP * ((col + e == row ? kNsA : 0.f) + kNsB * (av[e] / kNsX) + kNsC * v[e]);
      }
      ns_turn(scratch, lane, v, m);
      if (ti[t] == tj[t]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = col + e >= row ? v[e] : m[e];
      } else {
        put(tj[t] * 16 + (lane & 15), ti[t] * 16 + (lane >> 4) * 4, m);
      }
      put(row, col, v);
    }
    __syncthreads();
  };
  if (!two) {
    product(s0, s0, nullptr, true);
    return;
  }
  product(s0, s0, s1, true);
  product(s1, s0, s0, false);
  product(s0, s1, s0, false);
  product(s0, s0, s0, true);
  product(s0, s1, nullptr, false);
}

// ---- a matrix in one block -----------------------------------------------------------------------
// Matrices of at most 64 in the small dimension and ns_block_x elements go through all steps in one block's LDS, in
// one launch, in fp32 on the fp32 matrix instructions: X (pm x pn, both padded to 16), A and P.  Launches and their
// latency, not products, are what such matrices cost otherwise; and the steps run one by one, since few and short
// sums leave the plain recurrence in fp32 so exact that gathering them was up to 2.2 times further off (8 x 8, 64 x
// 12). In a block / by launches, us: 8 x 8 10 / 60, 64 x 64 27 / 62, 64 x 256 57 / 68, 64 x 320 68 / 69, 64 x 400 85
// / 71, 48 x 400 58 / 71, 30 x 600 49 / 74, 30 x 1000 74 / 81, 16 x 1200 60 / 81, 100 of 64 x 64 27 / 70.
__host__ __device__ constexpr int ns_block_x(int pm) { return pm > 32 ? 20992 : 28800; }
constexpr int kNsBlockFloats =
    std::max(ns_block_x(64) + 64 * 4 + 2 * 64 * 68, ns_block_x(32) + 32 * 4 + 2 * 32 * 36);
__host__ __device__ __forceinline__ int ns_pad16(int n) { return (n + 15) / 16 * 16; }

__global__ void __launch_bounds__(1024) ns_block_kernel(NsArgs p, NsUpdate u, int steps) {
  __shared__ __attribute__((aligned(16))) float pool[kNsBlockFloats];
  __shared__ double red[16];
  int mi = blockIdx.x;
  const int k = ns_find(p, mi, &NsGroup::chain);
  const NsGroup& g = p.g[k];
  const int pm = ns_pad16(g.m), pn = ns_pad16(g.n), lx = pn + 4, la = pm + 4;  // (16 rows: 16 different banks)
  float *X = pool, *A = X + pm * lx, *P = A + pm * la;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g4 = lane >> 4 << 2;
  const int64_t off = p.off[g.first + mi];
  const int total = g.rows * g.cols;
  for (int i = tid; i < pm * lx; i += 1024) X[i] = 0.f;
  __syncthreads();
  const auto place = [&](int i) {  // of element i of the matrix in memory
    const int r = i / g.cols, c = i - r * g.cols;
    return g.tall ? c * lx + r : r * lx + c;
  };
  double s = 0.0;
  for (int i = tid; i < total; i += 1024) {
    float v = ns_clip(u, ld(u.grad, off + i, u.code));
    if (u.mom != nullptr) {
      const float m = u.mu * u.mom[off + i] + v;
      u.mom[off + i] = m;
      v = u.nesterov ? v + u.mu * m : m;
    }
    if (u.zero != nullptr) st(u.zero, off + i, 0.f, u.zero_code);
    X[place(i)] = v;
    s += (double)v * (double)v;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += red[w];
  const double f = ns_inverse(s, u.eps);
  for (int i = tid; i < pm * lx; i += 1024) X[i] = (float)((double)X[i] * f);
  __syncthreads();

  // Of 16 consecutive k a lane holds the four of its group for its row of either operand: four matrix instructions, each
  // over one k of every group.
  const auto mma4 = [](const float4& a, const float4& b, nt_f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
  };
  // dst (pm x pm) = L L^T over nk columns, or a I + b L + c L L^T: at most 10 tiles on and above the diagonal, a wave
  // each, every value written to both of its places.  Sums in runs of 64 k.
  const int nt = pm / 16;
  const auto product = [&](const float* L, int ld, int nk, float* dst, bool poly) {
    int ti = 0, tj = 0;
    const bool mine = wave < nt * (nt + 1) / 2;
    nt_f32x4 sum = {0, 0, 0, 0};
    if (mine) {
      ns_tri(wave, nt, ti, tj);
      const float *a = L + (tj * 16 + r16) * ld + g4, *b = L + (ti * 16 + r16) * ld + g4;
      int k0 = 0;
      for (; k0 + 64 <= nk; k0 += 64) {
        nt_f32x4 acc = {0, 0, 0, 0};
        float4 x[4], y[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          x[q] = *reinterpret_cast<const float4*>(a + k0 + 16 * q);
          y[q] = *reinterpret_cast<const float4*>(b + k0 + 16 * q);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) acc = mma4(x[q], y[q], acc);
        sum += acc;
      }
      nt_f32x4 acc = {0, 0, 0, 0};
      for (; k0 < nk; k0 += 16)
        acc = mma4(*reinterpret_cast<const float4*>(a + k0), *reinterpret_cast<const float4*>(b + k0), acc);
      sum += acc;
    }
    __syncthreads();
    if (mine) {
      const int row = ti * 16 + r16, col = tj * 16 + g4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (col + e < row) continue;
        const float v = poly ? (col + e == row ? kNsA : 0.f) + kNsB * L[row * la + col + e] + kNsC * sum[e] : sum[e];
        dst[row * la + col + e] = v;
        dst[(col + e) * la + row] = v;
      }
    }
    __syncthreads();
  };
  for (int step = 0; step < steps; ++step) {
    product(X, lx, pn, A, false);
    product(A, la, pm, P, true);
    // X = P X in place: a wave reads and writes whole columns, 16 at a time
    for (int c0 = wave * 16; c0 < pn; c0 += 256) {
      nt_f32x4 acc[4] = {};
      float4 b[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < nt) {
          const float* x = X + (q * 16 + g4) * lx + c0 + r16;
          b[q] = make_float4(x[0], x[lx], x[2 * lx], x[3 * lx]);
        }
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (q < nt && i < nt)
            acc[i] = mma4(*reinterpret_cast<const float4*>(P + (i * 16 + r16) * la + q * 16 + g4), b[q], acc[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) X[(i * 16 + g4 + e) * lx + c0 + r16] = acc[i][e];
        }
    }
    __syncthreads();
  }
  const float lr = u.lr != nullptr ? *u.lr : 0.f;
  for (int i = tid; i < total; i += 1024) {
    float v = X[place(i)];
    if (u.w != nullptr) {
      const float w = u.w[off + i];
      v = w - lr * (g.scale * v + u.wd * w);
    }
    st(u.out, off + i, v, u.out_code);
    if (u.shadow != nullptr) stc(u.shadow, off + i, v, u.shadow_code, u.shadow_plane);
  }
}

// X' = Q X, X read across its lines (TURN), so that it need not be kept both ways: with X^T written beside X, 52 us
// instead of 41 at 23 x 256 x 2304 (and 24 instead of 17 in pass 2).  FINAL: the result leaves as the matrix itself
// (out) or as the weight update; otherwise X' is the other version of X for the next group of steps.
template <class C, bool FINAL>
__global__ void __launch_bounds__(C::THREADS) ns_apply_kernel(NsArgs p, NsUpdate u, int ver) {
  __shared__ __attribute__((aligned(1024))) char ring[C::LDS];
  int id = blockIdx.x;
  const int k = ns_find(p, id, &NsGroup::rect);
  const NsGroup& g = p.g[k];
  const int mt = (g.mp + C::BA - 1) / C::BA, nt = (g.np + C::BA - 1) / C::BA;
  id = nt_xcd_item(id, g.count * mt * nt);
  const int mi = id / (mt * nt), t = id % (mt * nt);
  const int m0 = t % mt * C::BA, n0 = t / mt * C::BA;
  nt_f32x4 acc[C::TA][C::TB];
  nt_loop<C>(ring, ns_op_turned(ns_x(p, g, mi, ver), g.mp, n0, g.np), ns_op(ns_sq(p, g, mi, kQ), m0, g.mp), 0, g.mp * 4,
             acc);
  const int lane = threadIdx.x & 63, wa = C::wa(), wb = C::wb();
  const int64_t off = p.off[g.first + mi];
  const float lr = FINAL && u.lr != nullptr ? *u.lr : 0.f;
  float* scratch = C::scratch(ring);
  uint16_t* dx = ns_x(p, g, mi, ver ^ 1);
#pragma unroll
  for (int i = 0; i < C::TA; ++i)
#pragma unroll
    for (int j = 0; j < C::TB; ++j) {
      if (!C::mine(i, j)) continue;
      // the tile's first n and m (wave-uniform); a lane has n0 + 4 (lane >> 4) .. + 3 of m0 + (lane & 15)
      const int tn = n0 + (wa * C::TA + i) * 16, tm = m0 + (wb * C::TB + j) * 16;
      if (tn >= g.np || tm >= g.mp) continue;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * (FINAL ? 1.f / (kNsP * kNsX) : 1.f / kNsP);
      if constexpr (!FINAL) {
        st4_pair(dx + ns_at(tm + (lane & 15), g.mp, tn + (lane >> 4) * 4), v);
      } else {
        if (g.tall) ns_turn(scratch, lane, v, v);
        const int r = (g.tall ? tn : tm) + (lane & 15), c = (g.tall ? tm : tn) + (lane >> 4) * 4;
        if (r >= g.rows || c >= g.cols) continue;
        const int cnt = min(4, g.cols - c);
        const int64_t at = off + (int64_t)r * g.cols + c;
        const bool vec = u.vec && at % 4 == 0 && cnt == 4;
        if (u.w != nullptr) {
          float w[4];
          ns_ld4(u.w, at, 0, vec, cnt, w);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = w[e] - lr * (g.scale * v[e] + u.wd * w[e]);
        }
        if (vec) {
          st4c(u.out, at, u.out_code, 0, v);
          if (u.shadow != nullptr) st4c(u.shadow, at, u.shadow_code, u.shadow_plane, v);
        } else {
          for (int e = 0; e < cnt; ++e) {
            st(u.out, at + e, v[e], u.out_code);
            if (u.shadow != nullptr) stc(u.shadow, at + e, v[e], u.shadow_code, u.shadow_plane);
          }
        }
      }
    }
}

// Tiles and their measured cost: microseconds per K tile with one block per CU alone and with every slot taken, slots
// (blocks resident on the chip), and microseconds of start and epilogue per round.  Larger tiles read fewer bytes per
// product, smaller ones fill the chip.  Whole runs with one kind of product at 64 / 128 / 192 / 256, us: symmetric m
// x m products of 4096 x 4096 5580 / 4410 / 3930 / -, of ResNet-101's 84 matrices 1500 / 1390 / - / -, of 23 x 256 x
// 2304 300 / 392 / - / -; P X of 4096 x 4096 - / 4060 / 4210 / 3920, of ResNet-101 - / 1390 / 1575 / 1383; X X^T of
// 23 x 256 x 2304 294 / 388 / 514 / 654.  The ring of the 64 x 64 tile holds 4 stages: 2 took 27 instead of 24 us for
// the last.
using Tile64 = NtCfg<true, 64, 64, 2, 2, 2, 4, 4, true>;  // two K groups: short products are bound by latency
using Tile128 = NtCfg<true, 128, 128, 1, 2, 4, 2, 8>;
using Tile192 = NtCfg<true, 192, 192, 1, 2, 4, 3, 8>;
using Tile256 = NtCfg<true, 256, 256, 1, 2, 4, 2>;  // (no registers for sums in runs)

struct NsTile {
  int size, slots;
  double alone, full, round;
};
constexpr NsTile kNsTiles[4] = {
    {64, 256, 0.28, 0.30, 6.0}, {128, 512, 0.75, 1.40, 7.0}, {192, 256, 1.31, 1.68, 9.0}, {256, 256, 1.95, 2.45, 20.0}};

enum NsLaunch { kLaunchGram, kLaunchSym, kLaunchRect };

int ns_tiles(const NsGroup& g, int size, NsLaunch what) {
  const int mt = (g.mp + size - 1) / size, nt = (g.np + size - 1) / size;
  return g.count * (what == kLaunchRect ? mt * nt : mt * (mt + 1) / 2 * (what == kLaunchGram ? g.splits : 1));
}

// Microseconds of one launch: the groups' tiles dealt out in rounds.
double ns_cost(const NsGroup* g, int ng, const NsTile& c, NsLaunch what) {
  double us = 0;
  int filled = 0, k_round = 0;
  for (int i = 0; i < ng; ++i) {
    const int k = what == kLaunchGram ? g[i].run_k : g[i].mp / 32;
    for (int n = ns_tiles(g[i], c.size, what); n > 0;) {
      if (filled == 0) k_round = 0;
      k_round = std::max(k_round, k);
      const int take = std::min(n, c.slots - filled);
      n -= take;
      filled += take;
      if (filled == c.slots) {
        us += k_round * c.full + c.round;
        filled = 0;
        // whole rounds of this group alone
        us += (n / c.slots) * (k * c.full + c.round);
        n %= c.slots;
      }
    }
  }
  if (filled > 0) us += k_round * (c.alone + (c.full - c.alone) * filled / c.slots) + c.round;
  return us;
}

// The 256 tile has no registers for sums in runs, so it takes no sums of squares (X X^T, A A) longer than that many K
// tiles.  With / without them, error against 64 bits and ms: 12288 x 12288 6.5e-6 89 / 3.5e-6 101, 16384 x 16384 8.9e-6
// 221 / 4.0e-6 253 (the plain recurrence in fp32 3.4e-6 and 3.6e-6).
constexpr int kNsLongestSum = 160;

int ns_pick(const NsGroup* g, int ng, NsLaunch what) {
  int longest = 0;
  for (int i = 0; i < ng; ++i) longest = std::max(longest, what == kLaunchGram ? g[i].run_k : g[i].mp / 32);
  int best = 0;
  for (int t = 1; t < (longest > kNsLongestSum && what != kLaunchRect ? 3 : 4); ++t)
    if (ns_cost(g, ng, kNsTiles[t], what) < ns_cost(g, ng, kNsTiles[best], what)) best = t;
  return best;
}

// Cuts X X^T into runs of about `cap` K tiles (as far as the unused version of X holds their sums) -> microseconds
// of the launch that joins them.
double ns_cut(NsGroup* g, int ng, int cap) {
  double bytes = 0;
  bool any = false;
  for (int i = 0; i < ng; ++i) {
    const int nk = g[i].np / 32, s = std::max(1, std::min(g[i].np / g[i].mp, (nk + cap - 1) / cap));
    g[i].run_k = (nk + s - 1) / s;
    g[i].splits = (nk + g[i].run_k - 1) / g[i].run_k;
    any |= g[i].splits > 1;
    bytes += (double)g[i].count * g[i].mp * g[i].mp * 4 * (g[i].splits + 1);  // (written and read: the upper half)
  }
  return any ? 5 + bytes / 4.5e6 : 0;
}

// The tile of X X^T and the runs of its K.  Whole / cut, us in all: 64 x 4608 144 / 90, 512 x 4608 276 / 231, VGG16's
// update 17250 / 16900; for ResNet-101's matrices 126 / 90 + 16 in this launch (uncut, 80 are one tile of 512 x 9216).
int ns_pick_gram(NsGroup* g, int ng, bool& cut) {
  constexpr int kWhole = 1 << 20;
  int tile = 0, runs = kWhole;
  double least = 1e30;
  for (int cap : {kWhole, 128, 64, 32, 16}) {
    const double join = ns_cut(g, ng, cap);
    const int t = ns_pick(g, ng, kLaunchGram);
    const double us = ns_cost(g, ng, kNsTiles[t], kLaunchGram) + join;
    if (us < least) {
      least = us;
      tile = t;
      runs = cap;
    }
  }
  cut = ns_cut(g, ng, runs) > 0;
  return tile;
}

template <class F>
void ns_with_tile(int t, F f) {
  if (t == 0) f(Tile64());
  else if (t == 1) f(Tile128());
  else if (t == 2) f(Tile192());
  else f(Tile256());
}

template <int KIND>
void ns_sym(const NsArgs& p, int tile, int blocks, int ls, int rs, int ds, hipStream_t st) {
  ns_with_tile(tile, [&](auto c) {
    using C = decltype(c);
    ns_sym_kernel<C, KIND><<<blocks, C::THREADS, 0, st>>>(p, ls, rs, ds);
  });
}

}  // namespace

void ns_shape(NsGroup& g) {
  g.tall = g.rows > g.cols;
  g.m = std::min(g.rows, g.cols);
  g.n = std::max(g.rows, g.cols);
  g.mp = (g.m + 63) / 64 * 64;
  g.np = (g.n + 63) / 64 * 64;
  const int64_t n = (int64_t)g.rows * g.cols;
  g.run = (n + kNsParts - 1) / kNsParts;
  g.run = std::max<int64_t>(4096, (g.run + 1023) / 1024 * 1024);
  g.parts = (int)((n + g.run - 1) / g.run);
  g.scale = (float)std::sqrt(std::max(1.0, (double)g.rows / g.cols));
}

int64_t ns_ws_elements(const NsGroup& g) { return g.count * ns_stride(g); }

bool ns_in_blocks(const NsGroup* g, int ng) {
  return std::all_of(g, g + ng, [](const NsGroup& g) {
    const int pm = ns_pad16(g.m), pn = ns_pad16(g.n);
    return g.m <= 64 && (int64_t)pm * pn <= ns_block_x(pm);
  });
}

void ns_run(const NsGroup* groups, int ng, const int64_t* off, int nmats, const NsUpdate& u, int steps, uint16_t* ws,
            double* part, hipStream_t st) {
  NsArgs p = {};
  p.ng = ng;
  p.ws = ws;
  p.part = part;
  std::copy(off, off + nmats, p.off);
  int at = 0;
  for (int k = 0; k < ng; ++k) {
    p.g[k] = groups[k];
    p.g[k].first = at;
    at += groups[k].count;
  }
  if (ns_in_blocks(p.g, ng)) {
    int blocks = 0;
    for (int k = 0; k < ng; ++k) {
      p.g[k].chain = blocks;
      blocks += p.g[k].count;
    }
    ns_block_kernel<<<blocks, 1024, 0, st>>>(p, u, steps);
    return;
  }
  // long products first
  std::stable_sort(p.g, p.g + ng, [](const NsGroup& a, const NsGroup& b) {
    return a.np != b.np ? a.np > b.np : a.mp > b.mp;
  });
  bool cut;
  const int tg = ns_pick_gram(p.g, ng, cut), ts = ns_pick(p.g, ng, kLaunchSym), tr = ns_pick(p.g, ng, kLaunchRect);
  int ew = 0, init = 0, gram = 0, sym = 0, rect = 0, chain = 0, join = 0;
  int64_t wat = 0;
  for (int k = 0; k < ng; ++k) {
    NsGroup& g = p.g[k];
    g.ws = wat;
    g.ew = ew;
    g.init = init;
    g.gram = gram;
    g.sym = sym;
    g.rect = rect;
    g.chain = chain;
    g.join = join;
    chain += g.count;
    join += ns_tiles(g, 64, kLaunchSym);
    wat += ns_ws_elements(g);
    ew += g.count * g.parts;
    init += g.count * (g.mp / 64) * (g.np / 64);
    gram += ns_tiles(g, kNsTiles[tg].size, kLaunchGram);
    sym += ns_tiles(g, kNsTiles[ts].size, kLaunchSym);
    rect += ns_tiles(g, kNsTiles[tr].size, kLaunchRect);
  }
  ns_norm_kernel<<<ew, 256, 0, st>>>(p, u);
  ns_init_kernel<<<init, 256, 0, st>>>(p, u);
  // products that fit one block each are chained in it: 5 launches less for two steps
  const bool chained = std::all_of(p.g, p.g + ng, [](const NsGroup& g) { return g.mp <= kNsChain; });
  int ver = 0;
  for (int done = 0; done < steps; ver ^= 1) {
    const bool two = steps - done >= 2;
    if (cut) {
      ns_with_tile(tg, [&](auto c) {
        using C = decltype(c);
        ns_gram_part_kernel<C><<<gram, C::THREADS, 0, st>>>(p, ver);
      });
      ns_join_kernel<<<join, 256, 0, st>>>(p, ver);
    } else {
      ns_sym<kGram>(p, tg, gram, ver, 0, kA, st);
    }
    if (chained) {
      ns_chain_kernel<<<chain, 1024, 0, st>>>(p, two);
    } else {
      ns_sym<kPoly>(p, ts, sym, kA, kA, two ? kP0 : kQ, st);
      if (two) {
        ns_sym<kMul>(p, ts, sym, kP0, kA, kT, st);
        ns_sym<kMul>(p, ts, sym, kT, kP0, kA, st);
        ns_sym<kPoly>(p, ts, sym, kA, kA, kP1, st);
        ns_sym<kMul>(p, ts, sym, kP1, kP0, kQ, st);
      }
    }
    done += two ? 2 : 1;
    ns_with_tile(tr, [&](auto c) {
      using C = typename decltype(c)::Turned;
      if (done < steps) ns_apply_kernel<C, false><<<rect, C::THREADS, 0, st>>>(p, u, ver);
      else ns_apply_kernel<C, true><<<rect, C::THREADS, 0, st>>>(p, u, ver);
    });
  }
}

}  // namespace mxr
