// gemv.cu -- the products of gemm.cuh for few tokens (M <= 16): the weights are read once, at
// the memory's rate, and nothing else matters.
//
// A block owns 16 rows of the weights and all of K; its 8 warps take 64-element chunks of K in
// turn.  mma.sync.m16n8k16 does the products: A = the weights' rows, B = the tokens.  Since the
// order of K within a contraction is free as long as both operands agree, a lane feeds the MMAs
// from 16 consecutive elements of its row (two 16-byte or one 32-byte load, no shared memory,
// no shuffles): lane (g, t) holds rows g and g+8 and token g at k = 16 t .. 16 t + 15 of the
// chunk, of which MMA j takes elements 4j .. 4j+3.  The warps' 16 x 8 results are added in
// order in shared memory and one thread runs the epilogue of each output element.
//
// Bound by HBM: bytes in flight are what counts, so a warp issues the loads of several chunks
// before the first MMA, and blocks are small enough that all SMs hold several.
#include <algorithm>

#include "gemm.cuh"

namespace mhc {

static constexpr int kGvWarps = 8;

// 16 consecutive elements of a row of length K, zeros past its end.  AL: bytes the row is
// aligned to (32, 16 or 2).
template <int AL>
__device__ __forceinline__ void gv_load(const uint16_t* row, int64_t k, int64_t K, bool live,
                                        uint32_t* r) {
  if constexpr (AL == 32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = 0;
    if (live && k < K) {  // K is a multiple of 16
      asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                     "=r"(r[6]), "=r"(r[7])
                   : "l"(row + k));
    }
  } else if constexpr (AL == 16) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // K is a multiple of 8
      const uint4 v = live && k + 8 * h < K ? *reinterpret_cast<const uint4*>(row + k + 8 * h)
                                            : make_uint4(0, 0, 0, 0);
      r[4 * h] = v.x; r[4 * h + 1] = v.y; r[4 * h + 2] = v.z; r[4 * h + 3] = v.w;
    }
  } else {
    uint16_t e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = live && k + i < K ? row[k + i] : (uint16_t)0;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
  }
}

template <typename E>
__device__ __forceinline__ void gv_mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                       uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<E, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9},"
        " {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9},"
        " {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: tiles of 8 tokens.  W: weight matrices (2 for kEpiGated).  U: chunks loaded together.
template <typename E, int KIND, int NT, int U, int AL>
__global__ void __launch_bounds__(32 * kGvWarps, 2)
    gemv_kernel(const uint16_t* __restrict__ x, int64_t xs, const uint16_t* __restrict__ w0,
                int64_t ws0, const uint16_t* __restrict__ w1, int64_t ws1, int T, int64_t N,
                int64_t K, const __grid_constant__ EpiParams epi) {
  pdl_enter();
  constexpr int W = KIND == kEpiGated ? 2 : 1;
  __shared__ float red[kGvWarps][W][NT][16][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const bool lo = n0 + g < N, hi = n0 + g + 8 < N;
  const uint16_t* wr[W][2];
  wr[0][0] = w0 + (n0 + g) * ws0;
  wr[0][1] = w0 + (n0 + g + 8) * ws0;
  if constexpr (W == 2) {
    wr[1][0] = w1 + (n0 + g) * ws1;
    wr[1][1] = w1 + (n0 + g + 8) * ws1;
  }
  float acc[W][NT][4] = {};
  const int64_t chunks = (K + 63) / 64;
  for (int64_t c = warp; c < chunks; c += kGvWarps * U) {
    uint32_t a[U][W][2][8], b[U][NT][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = (c + u * kGvWarps) * 64 + t * 16;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        gv_load<AL>(wr[i][0], k, K, lo, a[u][i][0]);
        gv_load<AL>(wr[i][1], k, K, hi, a[u][i][1]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = (c + u * kGvWarps) * 64 + t * 16;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        gv_load<AL>(x + (int64_t)(n * 8 + g) * xs, k, K, n * 8 + g < T, b[u][n]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            gv_mma<E>(acc[i][n], a[u][i][0][2 * j], a[u][i][1][2 * j], a[u][i][0][2 * j + 1],
                      a[u][i][1][2 * j + 1], b[u][n][2 * j], b[u][n][2 * j + 1]);
  }
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* d = &red[warp][i][n][0][0];
      d[g * 8 + 2 * t] = acc[i][n][0];
      d[g * 8 + 2 * t + 1] = acc[i][n][1];
      d[(g + 8) * 8 + 2 * t] = acc[i][n][2];
      d[(g + 8) * 8 + 2 * t + 1] = acc[i][n][3];
    }
  __syncthreads();
  for (int o = threadIdx.x; o < NT * 128; o += 32 * kGvWarps) {  // token o / 16, row o % 16
    const int tok = o >> 4, r = o & 15;
    if (tok >= T || n0 + r >= N) continue;
    float s[W] = {};
#pragma unroll
    for (int k = 0; k < kGvWarps; ++k)
#pragma unroll
      for (int i = 0; i < W; ++i) s[i] += red[k][i][tok >> 3][r][tok & 7];
    epi_chunk<E, KIND, 1>(epi, tok, n0 + r, 1, &s[0], &s[W - 1]);
  }
}

static int row_align(const void* p, int64_t ld, int64_t K) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  if (((a | (uintptr_t)(ld * 2)) & 31) == 0 && K % 16 == 0) return 32;
  if (((a | (uintptr_t)(ld * 2)) & 15) == 0 && K % 8 == 0) return 16;
  return 2;
}

template <typename E, int KIND, int NT, int U, int AL>
static int gemv_launch(const Gemm& g, cudaStream_t s) {
  launch(gemv_kernel<E, KIND, NT, U, AL>, (unsigned)cdiv(g.N, 16), 32 * kGvWarps, 0, s,
         (const uint16_t*)g.a.p, g.a.ld, (const uint16_t*)g.b.p, g.b.ld, (const uint16_t*)g.b2.p,
         g.b2.ld, (int)g.M, g.N, g.K, g.epi);
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}
template <typename E, int KIND>
static int gemv_kind(const Gemm& g, cudaStream_t s) {
  constexpr int U = KIND == kEpiGated ? 2 : 4;
  int al = std::min(row_align(g.a.p, g.a.ld, g.K), row_align(g.b.p, g.b.ld, g.K));
  if (KIND == kEpiGated) al = std::min(al, row_align(g.b2.p, g.b2.ld, g.K));
#define MHC_GV(AL)                                                    \
  return g.M <= 8 ? gemv_launch<E, KIND, 1, U, AL>(g, s)              \
                  : gemv_launch<E, KIND, 2, U / 2, AL>(g, s)
  if (al == 32) MHC_GV(32);
  if (al == 16) MHC_GV(16);
  MHC_GV(2);
#undef MHC_GV
}
template <typename E>
static int gemv_typed(const Gemm& g, cudaStream_t s) {
  return g.kind == kEpiGated ? gemv_kind<E, kEpiGated>(g, s) : gemv_kind<E, kEpiLinear>(g, s);
}

// 9 to 16 tokens read a second set of B fragments: the tcgen05 form is faster there from 64 MB of
// weights on (4096 -> 16384 features, T=16: 29.0 us here, 26.4 us there; 4096 -> 4096: 9.5 us here,
// 11.1 us there).
bool gemv_takes(int64_t M, int64_t N, int64_t K) {
  return M <= 8 || (M <= 16 && N * K < (int64_t)1 << 25);
}

int gemv_run(const Gemm& g0, cudaStream_t s) {
  Gemm g = g0;
  g.epi.vec = 0;  // element by element
  return g.dtype == MHC_F16 ? gemv_typed<__half>(g, s) : gemv_typed<__nv_bfloat16>(g, s);
}

}  // namespace mhc
