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
  kEpiGatedBwd32 = 3,  // the same, gate and up in fp32 (EpiParams::gu32)
};

struct EpiParams {
  int act = MHC_ACT_NONE;
  // kEpiLinear: out = y.  The others: out = h
  void* out = nullptr;
  int64_t ld_out = 0;
  const void* bias = nullptr;
  const void* res = nullptr;
  int64_t ld_res = 0;
  void* z = nullptr;  // packed like out
  // kEpiGated: outputs or null.  kEpiGatedBwd(32): inputs.  fp32 if gu32, else the operands' type
  void* gate = nullptr;
  void* up = nullptr;
  int64_t ld_gu = 0;
  int gu32 = 0;
  // kEpiGatedBwd(32): outputs
  void* gg = nullptr;
  void* gu = nullptr;
  int64_t ld_g = 0;
  int vec = 0;  // 1: every row above starts on a 16-byte boundary, 2: on a 32-byte one
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
// How a product is cut: mt accumulators of 256 rows to a tile, or 0: the form of gemm_few.cu
// with nt tokens to a tile; `splits` ranges of K.
struct GemmPlan {
  int mt, splits, nt;
};
GemmPlan gemm_plan(const Gemm& g);  // by the kind, the sizes and a.k_major alone

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

// EpiParams::vec
int epi_vec(const EpiParams& e);

// ---------------------------------------------------------------- epilogue
// A thread owns a row here, so every access of a warp touches 32 rows: 32-byte accesses (whole
// sectors) halve the requests where the rows allow them.  E: the type in memory, 16 bits or fp32.
struct alignas(32) Raw32 {
  uint4 a, b;
};
__device__ __forceinline__ Raw32 ld_row32(const void* p) {
  Raw32 v;
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v.a.x), "=r"(v.a.y), "=r"(v.a.z), "=r"(v.a.w), "=r"(v.b.x), "=r"(v.b.y),
                 "=r"(v.b.z), "=r"(v.b.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ void st_row32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y),
               "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}
template <typename E, int NC>
__device__ __forceinline__ void row_load(const void* base, int64_t off, int n, int vec, float* f) {
  constexpr int P = 16 / sizeof(E);
  const E* p = reinterpret_cast<const E*>(base) + off;
  if (NC % (2 * P) == 0 && vec == 2 && n == NC) {
#pragma unroll
    for (int i = 0; i < NC; i += 2 * P) {
      const Raw32 r = ld_row32(p + i);
      widen<E>(r.a, f + i);
      widen<E>(r.b, f + i + P);
    }
  } else if (NC % P == 0 && vec && n == NC) {
#pragma unroll
    for (int i = 0; i < NC; i += P) widen<E>(*reinterpret_cast<const uint4*>(p + i), f + i);
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i) f[i] = i < n ? from_e(p[i]) : 0.f;
  }
}
template <typename E, int NC>
__device__ __forceinline__ void row_store(void* base, int64_t off, int n, int vec, const float* f) {
  constexpr int P = 16 / sizeof(E);
  E* p = reinterpret_cast<E*>(base) + off;
  if (NC % (2 * P) == 0 && vec == 2 && n == NC) {
#pragma unroll
    for (int i = 0; i < NC; i += 2 * P) st_row32(p + i, narrow<E>(f + i), narrow<E>(f + i + P));
  } else if (NC % P == 0 && vec && n == NC) {
#pragma unroll
    for (int i = 0; i < NC; i += P) *reinterpret_cast<uint4*>(p + i) = narrow<E>(f + i);
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (i < n) p[i] = to_e<E>(f[i]);
  }
}

// Where an epilogue's outputs go: which = 0: out, 1: z, gate or gg, 2: up or gu.
struct StoreRows {
  template <typename E, int NC>
  __device__ __forceinline__ void put(int which, void* base, int64_t row, int64_t ld, int64_t col,
                                      int n, int vec, const float* f) const {
    row_store<E, NC>(base, row * ld + col, n, vec, f);
  }
};

// Roundings.  Everything here is fp32; what is stored in 16 bits is stored so because it is an operand
// of the next product, which the tensor cores take in 16 bits (h, gg, gu), or because the caller keeps
// it so from the forward to the backward (z; gate and up on request, which halves the largest tensors
// that a training step keeps; in fp32 otherwise).  The backward's activation is of the kept gate.  Each
// rounding adds an independent half step: where that of the output alone makes 1.66e-3 in the 2-norm
// in bf16, the gated block's output and its gradients are off by 2.35e-3, the gradients by 3.5e-3 with
// gate and up in 16 bits; the linear layer's gradients by 1.45 times the output's.  In fp16 h passes
// the type's range where act(gate) up does.
//
// n <= NC valid columns of one row, starting at col (a multiple of 8).  acc: the product;
// acc2: the second product of kEpiGated; for kEpiGatedBwd gate and up where they were loaded
// ahead, else null.
template <typename E, int KIND, int ACT, int NC, typename Store>
__device__ __forceinline__ void epi_act(const EpiParams& e, int64_t row, int64_t col, int n,
                                        float* acc, const float* acc2, Store& st) {
  float v[NC];
  if constexpr (KIND == kEpiLinear) {
    if (e.bias) {
      row_load<E, NC>(e.bias, col, n, e.vec, v);
#pragma unroll
      for (int i = 0; i < NC; ++i) acc[i] += v[i];
    }
    if (e.z) st.template put<E, NC>(1, e.z, row, e.ld_out, col, n, e.vec, acc);
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = act_fwd<ACT>(acc[i]);
    if (e.res) {
      row_load<E, NC>(e.res, row * e.ld_res + col, n, e.vec, v);
#pragma unroll
      for (int i = 0; i < NC; ++i) acc[i] += v[i];
    }
    st.template put<E, NC>(0, e.out, row, e.ld_out, col, n, e.vec, acc);
  } else if constexpr (KIND == kEpiGated) {
    if (e.gate && e.gu32) {
      st.template put<float, NC>(1, e.gate, row, e.ld_gu, col, n, e.vec, acc);
      st.template put<float, NC>(2, e.up, row, e.ld_gu, col, n, e.vec, acc2);
    } else if (e.gate) {
      st.template put<E, NC>(1, e.gate, row, e.ld_gu, col, n, e.vec, acc);
      st.template put<E, NC>(2, e.up, row, e.ld_gu, col, n, e.vec, acc2);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i] = act_fwd<ACT>(acc[i]) * acc2[i];
    st.template put<E, NC>(0, e.out, row, e.ld_out, col, n, e.vec, v);
  } else {
    using G = std::conditional_t<KIND == kEpiGatedBwd32, float, E>;
    float u[NC];
    if (acc2) {  // loaded ahead: gate in v's place, then up
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = acc2[i], u[i] = acc2[NC + i];
    } else {
      row_load<G, NC>(e.gate, row * e.ld_gu + col, n, e.vec, v);
      row_load<G, NC>(e.up, row * e.ld_gu + col, n, e.vec, u);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float a, da;
      act_both<ACT>(v[i], a, da);
      v[i] = acc[i] * u[i] * da;  // gg
      u[i] *= a;                  // h
      acc[i] *= a;                // gu
    }
    st.template put<E, NC>(1, e.gg, row, e.ld_g, col, n, e.vec, v);
    st.template put<E, NC>(2, e.gu, row, e.ld_g, col, n, e.vec, acc);
    st.template put<E, NC>(0, e.out, row, e.ld_out, col, n, e.vec, u);
  }
}
template <typename E, int KIND, int NC, typename Store>
__device__ __forceinline__ void epi_chunk(const EpiParams& e, int64_t row, int64_t col, int n,
                                          float* acc, const float* acc2, Store& st) {
  switch (e.act) {  // uniform over the grid
    case MHC_ACT_RELU: return epi_act<E, KIND, MHC_ACT_RELU, NC>(e, row, col, n, acc, acc2, st);
    case MHC_ACT_GELU: return epi_act<E, KIND, MHC_ACT_GELU, NC>(e, row, col, n, acc, acc2, st);
    case MHC_ACT_GELU_TANH:
      return epi_act<E, KIND, MHC_ACT_GELU_TANH, NC>(e, row, col, n, acc, acc2, st);
    case MHC_ACT_SILU: return epi_act<E, KIND, MHC_ACT_SILU, NC>(e, row, col, n, acc, acc2, st);
    default: return epi_act<E, KIND, MHC_ACT_NONE, NC>(e, row, col, n, acc, acc2, st);
  }
}
template <typename E, int KIND, int NC>
__device__ __forceinline__ void epi_chunk(const EpiParams& e, int64_t row, int64_t col, int n,
                                          float* acc, const float* acc2) {
  StoreRows st;
  epi_chunk<E, KIND, NC>(e, row, col, n, acc, acc2, st);
}

}  // namespace mhc
