// gemm.cuh -- the matrix product behind the linear layer and the gated feed-forward block:
// C[M][N] = A[M][K] B[N][K]^T, with the operator's elementwise work as its epilogue.
#pragma once

#include <type_traits>

#include "act.cuh"

namespace mhc {

// A matrix operand: [MN][K] rows `ld` apart if k_major, else [K][MN] rows `ld` apart.
struct Operand {
  const void* p = nullptr;
  int64_t ld = 0;
  bool k_major = true;
};

enum EpiKind {
  kEpiLinear = 0,    // y = act(acc + bias) + residual, z = acc + bias
  kEpiGated = 1,     // two products: gate, up; h = act(gate) * up
  kEpiGatedBwd = 2,  // acc = gh; from gate and up: gg, gu and h
};

struct EpiParams {
  int act = MHC_ACT_NONE;
  // kEpiLinear: out = y.  kEpiGated, kEpiGatedBwd: out = h
  void* out = nullptr;
  int64_t ld_out = 0;
  const void* bias = nullptr;
  const void* res = nullptr;
  int64_t ld_res = 0;
  void* z = nullptr;  // packed like out
  // kEpiGated: outputs or null.  kEpiGatedBwd: inputs
  void* gate = nullptr;
  void* up = nullptr;
  int64_t ld_gu = 0;
  // kEpiGatedBwd: outputs
  void* gg = nullptr;
  void* gu = nullptr;
  int64_t ld_g = 0;
  bool vec = false;  // every row above starts on a 16-byte boundary
};

struct Gemm {
  int kind = kEpiLinear;
  int32_t dtype = MHC_BF16;
  int64_t M = 0, N = 0, K = 0;
  Operand a, b;
  Operand b2;         // kEpiGated: the up projection, N and K as b
  Operand a3, b3;     // if K3 > 0: adds a3 b3^T to the product (M, N and orders as a and b)
  int64_t K3 = 0;
  EpiParams epi;
};

// Operands must be aligned (operand_aligned).  ws: gemm_ws_bytes, which goes by the kind and the
// sizes alone (and whether a is K-major).
size_t gemm_ws_bytes(const Gemm& g);
int gemm_run(const Gemm& g, void* ws, cudaStream_t s);
bool gemm_few_form(const Gemm& g);  // it takes the form of gemm_few.cu

// The form with swapped roles (gemm_few.cu): its estimated time, tile and cut, and the run.
double few_estimate(const Gemm& g, int* nt, int* splits);
int few_run(const Gemm& g, int nt, int splits, cudaStream_t s);

// For few tokens: K-major operands of any alignment, kEpiLinear or kEpiGated, no third product.
bool gemv_takes(int64_t M, int64_t N, int64_t K);
int gemv_run(const Gemm& g, cudaStream_t s);

// Base and rows on 16-byte boundaries, as TMA reads them.
bool operand_aligned(const Operand& o);
// Copies (rows, cols) 16-bit elements, rows ls apart, to rows ld apart.
int pack_rows(const void* src, int64_t ls, int64_t rows, int64_t cols, void* dst, int64_t ld,
              cudaStream_t s);

// Whether all rows the epilogue touches start on 16-byte boundaries.
bool epi_vec_ok(const Gemm& g);

// ---------------------------------------------------------------- epilogue
template <typename E, int NC>
__device__ __forceinline__ void row_load(const void* base, int64_t off, int n, bool vec, float* f) {
  const E* p = reinterpret_cast<const E*>(base) + off;
  if (vec && n == NC) {
#pragma unroll
    for (int i = 0; i < NC; i += 8) widen<E>(*reinterpret_cast<const uint4*>(p + i), f + i);
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i) f[i] = i < n ? from_e(p[i]) : 0.f;
  }
}
template <typename E, int NC>
__device__ __forceinline__ void row_store(void* base, int64_t off, int n, bool vec, const float* f) {
  E* p = reinterpret_cast<E*>(base) + off;
  if (vec && n == NC) {
#pragma unroll
    for (int i = 0; i < NC; i += 8) *reinterpret_cast<uint4*>(p + i) = narrow<E>(f + i);
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (i < n) p[i] = to_e<E>(f[i]);
  }
}

// n <= NC valid columns of one row, starting at col (a multiple of 8).  acc: the product;
// acc2: the second product of kEpiGated.
template <typename E, int KIND, int ACT, int NC>
__device__ __forceinline__ void epi_act(const EpiParams& e, int64_t row, int64_t col, int n,
                                        float* acc, const float* acc2) {
  float v[NC];
  if constexpr (KIND == kEpiLinear) {
    if (e.bias) {
      row_load<E, NC>(e.bias, col, n, e.vec, v);
#pragma unroll
      for (int i = 0; i < NC; ++i) acc[i] += v[i];
    }
    if (e.z) row_store<E, NC>(e.z, row * e.ld_out + col, n, e.vec, acc);
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = act_fwd<ACT>(acc[i]);
    if (e.res) {
      row_load<E, NC>(e.res, row * e.ld_res + col, n, e.vec, v);
#pragma unroll
      for (int i = 0; i < NC; ++i) acc[i] += v[i];
    }
    row_store<E, NC>(e.out, row * e.ld_out + col, n, e.vec, acc);
  } else if constexpr (KIND == kEpiGated) {
    if (e.gate) {
      row_store<E, NC>(e.gate, row * e.ld_gu + col, n, e.vec, acc);
      row_store<E, NC>(e.up, row * e.ld_gu + col, n, e.vec, acc2);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i] = act_fwd<ACT>(acc[i]) * acc2[i];
    row_store<E, NC>(e.out, row * e.ld_out + col, n, e.vec, v);
  } else {
    float u[NC];
    row_load<E, NC>(e.gate, row * e.ld_gu + col, n, e.vec, v);
    row_load<E, NC>(e.up, row * e.ld_gu + col, n, e.vec, u);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float a, da;
      act_both<ACT>(v[i], a, da);
      v[i] = acc[i] * u[i] * da;  // gg
      u[i] *= a;                  // h
      acc[i] *= a;                // gu
    }
    row_store<E, NC>(e.gg, row * e.ld_g + col, n, e.vec, v);
    row_store<E, NC>(e.gu, row * e.ld_g + col, n, e.vec, acc);
    row_store<E, NC>(e.out, row * e.ld_out + col, n, e.vec, u);
  }
}
template <typename E, int KIND, int NC>
__device__ __forceinline__ void epi_chunk(const EpiParams& e, int64_t row, int64_t col, int n,
                                          float* acc, const float* acc2) {
  switch (e.act) {  // uniform over the grid
    case MHC_ACT_RELU: return epi_act<E, KIND, MHC_ACT_RELU, NC>(e, row, col, n, acc, acc2);
    case MHC_ACT_GELU: return epi_act<E, KIND, MHC_ACT_GELU, NC>(e, row, col, n, acc, acc2);
    case MHC_ACT_GELU_TANH: return epi_act<E, KIND, MHC_ACT_GELU_TANH, NC>(e, row, col, n, acc, acc2);
    case MHC_ACT_SILU: return epi_act<E, KIND, MHC_ACT_SILU, NC>(e, row, col, n, acc, acc2);
    default: return epi_act<E, KIND, MHC_ACT_NONE, NC>(e, row, col, n, acc, acc2);
  }
}

}  // namespace mhc
