// Launchers of the weight-matrix operators: Newton-Schulz updates and 8-bit products.
#pragma once
#include <hip/hip_runtime_api.h>
#include <cstdint>

namespace mxr {

// ---- Newton-Schulz orthogonalisation, Muon update (newton_schulz.hip) -------------------------
constexpr int kNsMaxGroups = 16;  // groups of equal shape and matrices per launch (kernel arguments)
constexpr int kNsMaxMats = 128;
constexpr int kNsParts = 512;     // partial sums of squares per matrix, at most

constexpr int kShadowX2 = 3, kShadowX3 = 4;  // storage codes of the 2- and 3-plane shadows

struct NsGroup {
  int count, rows, cols;  // matrices of this shape
  // derived (ns_shape): m = min, n = max, padded to multiples of 64; runs of the norm pass
  int tall, m, n, mp, np, parts;
  int64_t run;
  float scale;  // sqrt(max(1, rows / cols)), the update's
  // filled per launch: first matrix, workspace offset (fp16 elements), first work item of each pass
  int first, ew, init, gram, sym, rect, chain, join;
  int splits, run_k;  // X X^T: runs of K, K tiles of a run
  int64_t ws;
};

struct NsUpdate {
  const void* grad;  // input, at the matrices' element offsets; storage code 0 fp32, 1 bf16, 2 fp16
  int code;
  float* mom;  // momentum (nullptr: grad itself is orthogonalised)
  float mu, rescale, clip;
  int nesterov;
  double eps;
  void* zero;  // cleared after it is read (may be grad)
  int zero_code;
  void* out;  // result, or the updated weights
  int out_code;
  float* w;  // weights to update (nullptr: out receives the orthogonal factor)
  const float* lr;
  float wd;
  void* shadow;  // low-precision planes of the new weights
  int shadow_code;
  int64_t shadow_plane;
  int vec;  // base pointers allow 4-element accesses where the offset does
};

void ns_shape(NsGroup& g);                     // from count / rows / cols
int64_t ns_ws_elements(const NsGroup& g);      // fp16 elements of workspace
bool ns_in_blocks(const NsGroup* g, int ng);   // all of them fit a block each: no workspace
void ns_run(const NsGroup* groups, int ng, const int64_t* off, int nmats, const NsUpdate& u, int steps, uint16_t* ws,
            double* part, hipStream_t st);

// ---- 8-bit rows and products (int8_gemm.hip) -----------------------------------------------------
// rows of q are ldq >= K bytes apart, zeros behind K
void quantize_rows(const void* x, int code, int64_t rows, int64_t ld, int K, int8_t* q, int ldq, float* scale,
                   hipStream_t st);

struct Int8Args {
  const int8_t *x, *w;  // (M, K), (N, K), rows ldx / ldw apart
  int64_t ldx, ldw;
  const float *xs, *ws, *bias;
  void* y;  // (M, N) contiguous, storage code 0 / 1 / 2
  int64_t M;
  int N, K, code, relu;
  int x_padded;  // rows of x hold zeros from K to the next multiple of 16
};
int64_t int8_matmul_ws(const Int8Args& a);  // bytes of workspace
void int8_matmul(const Int8Args& a, void* ws, hipStream_t st);

}  // namespace mxr
