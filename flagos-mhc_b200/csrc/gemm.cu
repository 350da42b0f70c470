// gemm.cu -- matrix product with the operators' epilogues: 64 x 64 tiles in shared memory,
// fp32 multiply-adds, a thread owns one row and 16 columns.
#include "gemm.cuh"

namespace mhc {

static constexpr int kBM = 64, kBN = 64, kBK = 16, kNC = 16;

template <typename E>
__device__ __forceinline__ void load_tile(float (*s)[kBM + 1], const Operand& o, int64_t r0,
                                          int64_t R, int64_t k0, int64_t K) {
  const E* p = (const E*)o.p;
  for (int i = threadIdx.x; i < kBM * kBK; i += 256) {
    const int r = o.k_major ? i / kBK : i % kBM, k = o.k_major ? i % kBK : i / kBM;
    float v = 0.f;
    if (r0 + r < R && k0 + k < K)
      v = from_e(p[o.k_major ? (r0 + r) * o.ld + k0 + k : (k0 + k) * o.ld + r0 + r]);
    s[k][r] = v;
  }
}

template <typename E, int KIND>
__global__ void __launch_bounds__(256) gemm_kernel(Gemm g) {
  pdl_enter();
  constexpr bool dual = KIND == kEpiGated;
  __shared__ float sa[kBK][kBM + 1], sb[kBK][kBN + 1], sb2[dual ? kBK : 1][kBN + 1];
  const int64_t m0 = (int64_t)blockIdx.x * kBM, n0 = (int64_t)blockIdx.y * kBN;
  const int r = threadIdx.x & 63, c = (threadIdx.x >> 6) * kNC;
  float acc[kNC] = {}, acc2[kNC] = {};
  for (int seg = 0; seg < 2; ++seg) {
    const Operand &A = seg ? g.a3 : g.a, &B = seg ? g.b3 : g.b;
    const int64_t K = seg ? g.K3 : g.K;
    for (int64_t k0 = 0; k0 < K; k0 += kBK) {
      load_tile<E>(sa, A, m0, g.M, k0, K);
      load_tile<E>(sb, B, n0, g.N, k0, K);
      if constexpr (dual) load_tile<E>(sb2, g.b2, n0, g.N, k0, K);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kBK; ++k) {
        const float a = sa[k][r];
#pragma unroll
        for (int i = 0; i < kNC; ++i) {
          acc[i] = fmaf(a, sb[k][c + i], acc[i]);
          if constexpr (dual) acc2[i] = fmaf(a, sb2[k][c + i], acc2[i]);
        }
      }
      __syncthreads();
    }
  }
  const int64_t left = g.N - (n0 + c);
  if (m0 + r < g.M && left > 0)
    epi_chunk<E, KIND, kNC>(g.epi, m0 + r, n0 + c, left < kNC ? (int)left : kNC, acc, acc2);
}

bool epi_vec_ok(const Gemm& g) {
  const EpiParams& e = g.epi;
  return aligned16(e.out) && e.ld_out % 8 == 0 && aligned16(e.bias) && aligned16(e.res) &&
         e.ld_res % 8 == 0 && aligned16(e.z) && aligned16(e.gate) && aligned16(e.up) &&
         e.ld_gu % 8 == 0 && aligned16(e.gg) && aligned16(e.gu) && e.ld_g % 8 == 0;
}

template <typename E>
static int gemm_typed(const Gemm& g, cudaStream_t s) {
  const dim3 grid((unsigned)cdiv(g.M, kBM), (unsigned)cdiv(g.N, kBN));
  if (g.kind == kEpiGated)
    launch(gemm_kernel<E, kEpiGated>, grid, 256, 0, s, g);
  else if (g.kind == kEpiGatedBwd)
    launch(gemm_kernel<E, kEpiGatedBwd>, grid, 256, 0, s, g);
  else
    launch(gemm_kernel<E, kEpiLinear>, grid, 256, 0, s, g);
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

int gemm_run(const Gemm& g0, cudaStream_t s) {
  Gemm g = g0;
  g.epi.vec = epi_vec_ok(g);
  return g.dtype == MHC_F16 ? gemm_typed<__half>(g, s) : gemm_typed<__nv_bfloat16>(g, s);
}

}  // namespace mhc
