// gemm_few.cu -- the products of gemm.cuh with tens to hundreds of tokens, on tcgen05.
//
// There the weights' bytes bound the product, and 256-row tiles of tokens leave most SMs
// without work.  So the roles are swapped: a CTA owns 128 output features (the M of its MMAs:
// weights as the A operand) by NT tokens (N = 32 .. 256, the B operand), and a cluster of
// `splits` CTAs shares one such tile, each with a range of K.  The ranges' accumulators meet in
// distributed shared memory: each CTA sums a slice of the tokens over the cluster, in order,
// and runs the epilogue of its slice.  One launch, no partial sums in HBM, nothing atomic.
#include <algorithm>

#include "gemm.cuh"
#include "tc.cuh"

namespace mhc {
namespace fk {
constexpr int BM = 128, BK = 64;
constexpr int A_BYTES = BM * BK * 2;
constexpr int THREADS = 256;
template <int NT, int W> struct Ring {
  static constexpr int STAGE_BYTES = W * A_BYTES + NT * BK * 2;
  // as many stages as fit 200 KB, up to 10; never fewer bytes than the accumulators need
  static constexpr int STAGES = (200 << 10) / STAGE_BYTES > 10 ? 10 : (200 << 10) / STAGE_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024;
  static constexpr int COLS = W * NT < 32 ? 32 : W * NT;  // TMEM columns
  static_assert(W * NT * BM * 4 <= STAGES * STAGE_BYTES, "accumulators reuse the ring");
  static_assert(COLS <= 512, "TMEM");
};
}  // namespace fk

struct FewMaps {
  CUtensorMap a, a2, b, a3, b3;  // a: weights, b: tokens
};
struct FewWalk {
  int64_t M, N;  // tokens, output features
  int32_t tiles_n, tiles_m, nk1, nk, splits;
};

__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
  float4 v;
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

template <typename E, int KIND, int NT, bool AK>
__global__ void __launch_bounds__(fk::THREADS, 1)
    gemm_few_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ FewWalk w,
                    const __grid_constant__ EpiParams epi) {
  using namespace fk;
  constexpr int W = KIND == kEpiGated ? 2 : 1;
  using R = Ring<NT, W>;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                       ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[R::STAGES], empty[R::STAGES], done;
  __shared__ uint32_t tmem_slot, filled;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = w.splits > 1 ? tc::cta_rank() : 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < R::STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&done, 1);
    abort_word = 0;
    tc::fence_barrier_init();
    tc::prefetch_tmap(&maps.a);
    tc::prefetch_tmap(&maps.b);
  }
  if (warp == 1) {
    tc::tmem_alloc(&tmem_slot, R::COLS);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t*)&tmem_slot;
  pdl_enter();

  const int32_t tile = blockIdx.x / w.splits;
  const int32_t nt = tile / w.tiles_m, mt = tile - nt * w.tiles_m;
  const int32_t f0 = nt * BM, t0 = mt * NT;
  const int32_t kb0 = (int32_t)((int64_t)w.nk * rank / w.splits);
  const int32_t kb1 = (int32_t)((int64_t)w.nk * (rank + 1) / w.splits);
  // The two issuing loops are warp-wide and unrolled over the ring: barriers, addresses and
  // descriptors are then constants or uniform registers.  (One lane looping alone, with its
  // addresses computed, took 600 cycles to a K block.)
  if (warp == 0) {
    const bool issue = tc::elect_one();
    int32_t kb = kb0;
    for (uint32_t ph = 1; kb < kb1; ph ^= 1) {
#pragma unroll
      for (int s = 0; s < R::STAGES; ++s) {
        if (kb >= kb1) break;
        if (!tc::mbar_wait_warp(&empty[s], ph, abort_flag)) {
          kb = kb1;
          if (issue) filled = tc::fills_at(s, ph);
          break;
        }
        char* sa = smem + s * R::STAGE_BYTES;
        char* sb = sa + W * A_BYTES;
        const bool second = kb >= w.nk1;
        const int32_t k0 = (second ? kb - w.nk1 : kb) * BK;
        if (issue) {
          tc::mbar_arrive_expect_tx(&full[s], R::STAGE_BYTES);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const CUtensorMap* ma = second ? &maps.a3 : i ? &maps.a2 : &maps.a;
            if constexpr (AK) {
              tc::tma_load_2d(sa + i * A_BYTES, ma, &full[s], k0, f0);
            } else {
              tc::tma_load_2d(sa + i * A_BYTES, ma, &full[s], f0, k0);
              tc::tma_load_2d(sa + i * A_BYTES + A_BYTES / 2, ma, &full[s], f0 + 64, k0);
            }
          }
          // tokens are K-major in every product of this form
          tc::tma_load_2d(sb, second ? &maps.b3 : &maps.b, &full[s], k0, t0);
        }
        __syncwarp();
        if (++kb == kb1 && issue) filled = tc::fills_at(s + 1, ph);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = tc::idesc_16<E>(128, NT, !AK, false);
    // descriptor step of 16 K elements: 32 bytes of a K-major row, or two 8-row atoms
    constexpr uint32_t stepa = AK ? 2 : 128;
    const uint32_t base = tc::smem_u32(smem);
    const uint64_t da0 = tc::smem_desc(base, AK ? 16 : A_BYTES / 2, 1024, tc::kSwizzle128);
    const uint64_t db0 = tc::smem_desc(base + W * A_BYTES, 16, 1024, tc::kSwizzle128);
    const bool issue = tc::elect_one();
    int32_t kb = kb0;
    for (uint32_t ph = 0; kb < kb1; ph ^= 1) {
#pragma unroll
      for (int s = 0; s < R::STAGES; ++s) {
        if (kb >= kb1) break;
        if (!tc::mbar_wait_warp(&full[s], ph, abort_flag)) {
          kb = kb1;
          break;
        }
        tc::tc_fence_after();
        if (issue) {
          const uint64_t da = da0 + s * (R::STAGE_BYTES >> 4), db = db0 + s * (R::STAGE_BYTES >> 4);
#pragma unroll
          for (int i = 0; i < W; ++i)
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              tc::mma_bf16(tmem + i * NT, da + i * (A_BYTES >> 4) + k * stepa, db + k * 2, idesc,
                           (kb != kb0 || k != 0) ? 1u : 0u);
          tc::mma_commit(&empty[s]);
        }
        __syncwarp();
        ++kb;
      }
    }
    if (issue) tc::mma_commit(&done);
  }
  __syncwarp();
  // Accumulators to shared memory, [W][NT tokens][128 features]: the ring has been read by the
  // last MMA, and every load into it has landed before that.
  if (warp >= 4) {
    const int q = warp & 3;
    volatile int never = 0;
    const bool ok = tc::mbar_wait(&done, 0, &never);
    if (!__all_sync(0xffffffffu, ok) && lane == 0) *abort_flag = 1;
    __syncwarp();
    tc::tc_fence_after();
    float* acc = reinterpret_cast<float*>(smem);
    const uint32_t tq = tmem + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
    for (int c = 0; c < W * NT; c += 16) {
      float v[16];
      tc::tmem_ld16(tq + c, v);
      tc::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[(c + i) * BM + q * 32 + lane] = v[i];
    }
  }
  tc::tc_fence_before();
  if (w.splits > 1)
    tc::cluster_sync();
  else
    __syncthreads();
  // each CTA of the cluster: its tokens, 8 features to a thread
  const uint32_t sacc = tc::smem_u32(smem);
  const int tok0 = NT * (int)rank / w.splits, tok1 = NT * ((int)rank + 1) / w.splits;
  for (int i = threadIdx.x; i < (tok1 - tok0) * (BM / 8); i += THREADS) {
    const int tok = tok0 + i / (BM / 8), f = (i % (BM / 8)) * 8;
    const int64_t left = w.N - (f0 + f);
    if (t0 + tok >= w.M || left <= 0) continue;
    float v[W][8];
#pragma unroll
    for (int p = 0; p < W; ++p) {
      const uint32_t off = sacc + (uint32_t)(((p * NT + tok) * BM + f) * 4);
      if (w.splits == 1) {
        *reinterpret_cast<float4*>(&v[p][0]) = *reinterpret_cast<const float4*>(smem + (off - sacc));
        *reinterpret_cast<float4*>(&v[p][4]) =
            *reinterpret_cast<const float4*>(smem + (off - sacc) + 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[p][e] = 0.f;
#pragma unroll 4
        for (int r = 0; r < w.splits; ++r) {
          const float4 a = ld_cluster(off, r), b = ld_cluster(off + 16, r);
          v[p][0] += a.x; v[p][1] += a.y; v[p][2] += a.z; v[p][3] += a.w;
          v[p][4] += b.x; v[p][5] += b.y; v[p][6] += b.z; v[p][7] += b.w;
        }
      }
    }
    epi_chunk<E, KIND, 8>(epi, t0 + tok, f0 + f, left < 8 ? (int)left : 8, v[0],
                          W == 2 ? v[W - 1] : nullptr);
  }
  if (*abort_flag && threadIdx.x == 0) {
    flag_timeout();
    tc::drain(full, R::STAGES, filled);
  }
  if (w.splits > 1)
    tc::cluster_sync();  // the others may still read this CTA's accumulators
  else
    __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, R::COLS);
  }
}

static int few_map(CUtensorMap* m, const Operand& o, int32_t dtype, int64_t mn, int64_t k, int box) {
  const CUtensorMapDataType dt =
      dtype == MHC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return o.k_major ? make_tmap_2d(m, o.p, dt, 2, k, mn, o.ld * 2, fk::BK, box,
                                  CU_TENSOR_MAP_SWIZZLE_128B)
                   : make_tmap_2d(m, o.p, dt, 2, mn, k, o.ld * 2, 64, fk::BK,
                                  CU_TENSOR_MAP_SWIZZLE_128B);
}

// AK: the weights are K-major
template <typename E, int KIND, int NT, bool AK>
static int few_launch(const Gemm& g, int splits, cudaStream_t s) {
  using namespace fk;
  constexpr int W = KIND == kEpiGated ? 2 : 1;
  using R = Ring<NT, W>;
  FewMaps m;
  int st;
  if ((st = few_map(&m.a, g.b, g.dtype, g.N, g.K, BM))) return st;
  if ((st = few_map(&m.b, g.a, g.dtype, g.M, g.K, NT))) return st;
  m.a2 = m.a; m.a3 = m.a; m.b3 = m.b;
  if (W == 2 && (st = few_map(&m.a2, g.b2, g.dtype, g.N, g.K, BM))) return st;
  if (g.K3 > 0) {
    if ((st = few_map(&m.a3, g.b3, g.dtype, g.N, g.K3, BM))) return st;
    if ((st = few_map(&m.b3, g.a3, g.dtype, g.M, g.K3, NT))) return st;
  }
  FewWalk w;
  w.M = g.M; w.N = g.N;
  w.tiles_n = (int32_t)cdiv(g.N, BM);
  w.tiles_m = (int32_t)cdiv(g.M, NT);
  w.nk1 = (int32_t)cdiv(g.K, BK);
  w.nk = w.nk1 + (int32_t)cdiv(g.K3, BK);
  w.splits = splits;
  static bool attr_set[64];
  int dev = 0;
  MHC_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    MHC_CUDA_CHECK(cudaFuncSetAttribute((const void*)gemm_few_kernel<E, KIND, NT, AK>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, R::SMEM));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t blocks = (int64_t)w.tiles_n * w.tiles_m * splits;
  if (blocks > INT32_MAX) return MHC_ERR_INVALID_ARGUMENT;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = R::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = (!pdl_first_launch() && pdl_enabled()) ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, gemm_few_kernel<E, KIND, NT, AK>, m, w, g.epi) != cudaSuccess) {
    (void)cudaGetLastError();
    return MHC_ERR_CUDA;
  }
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

// The tile and the cut in K whose estimated time (us) is least; 0 if this form does not take the
// product.  Measured: 4 us to start and end a launch; to a K block 0.17 us, or its bytes at 130
// GB/s an SM and 14 TB/s in all; at a tile's end 0.6 us and 0.016 us a token, and with a cut in K
// 0.8 us and 0.012 us a token more; the weights at 6.4 TB/s after 6 us.
// (Clusters of 8 CTAs of this size leave SMs empty: 1024 -> 2048 features, T=128: 22 us against
// 9.6 with 2.)
double few_estimate(const Gemm& g, int* nt_best, int* splits) {
  if (!g.a.k_major) return 0.0;
  const int W = g.kind == kEpiGated ? 2 : 1;
  const int64_t nk = cdiv(g.K, fk::BK) + cdiv(g.K3, fk::BK);
  const double hbm = 6.0 + (double)W * g.N * (g.K + g.K3) * 2 / 6.4e6;
  double best = 1e30;
  for (int nt = 32; nt <= (W == 2 ? 128 : 256); nt *= 2) {
    if (nt > 32 && nt >= 2 * g.M) break;
    const int64_t tiles = cdiv(g.N, fk::BM) * cdiv(g.M, nt);
    const double bytes = W * 16384.0 + nt * 128.0;
    for (int sp = 1; sp <= 4; sp *= 2) {
      if (sp > 1 && nk < 2 * sp) break;
      const double waves = (double)cdiv(tiles * sp, sm_count());
      const double active = (double)std::min<int64_t>(tiles * sp, sm_count());
      const double per_k = std::max(0.17 * W, std::max(bytes / 130e3, bytes * active / 14e6));
      double us = 4.0 + (sp > 1 ? 0.8 + 0.012 * W * nt : 0.0) +
                  waves * ((double)cdiv(nk, sp) * per_k + 0.6 + 0.016 * W * nt);
      us = std::max(us, hbm);
      if (us < best) best = us, *nt_best = nt, *splits = sp;
    }
  }
  return best;
}

template <typename E, int KIND, bool AK>
static int few_kind(const Gemm& g, int nt, int splits, cudaStream_t s) {
  switch (nt) {
    case 32: return few_launch<E, KIND, 32, AK>(g, splits, s);
    case 64: return few_launch<E, KIND, 64, AK>(g, splits, s);
    case 128: return few_launch<E, KIND, 128, AK>(g, splits, s);
    default:
      if constexpr (KIND != kEpiGated) return few_launch<E, KIND, 256, AK>(g, splits, s);
      return MHC_ERR_INVALID_ARGUMENT;
  }
}
template <typename E>
static int few_typed(const Gemm& g, int nt, int splits, cudaStream_t s) {
  if (g.kind == kEpiGated) return few_kind<E, kEpiGated, true>(g, nt, splits, s);
  if (g.kind == kEpiGatedBwd) return few_kind<E, kEpiGatedBwd, false>(g, nt, splits, s);
  if (g.kind == kEpiGatedBwd32) return few_kind<E, kEpiGatedBwd32, false>(g, nt, splits, s);
  return g.b.k_major ? few_kind<E, kEpiLinear, true>(g, nt, splits, s)
                     : few_kind<E, kEpiLinear, false>(g, nt, splits, s);
}
int few_run(const Gemm& g, int nt, int splits, cudaStream_t s) {
  return g.dtype == MHC_F16 ? few_typed<__half>(g, nt, splits, s)
                            : few_typed<__nv_bfloat16>(g, nt, splits, s);
}

int gemm_few_device_error() { return read_and_clear_tu_error(); }

}  // namespace mhc
