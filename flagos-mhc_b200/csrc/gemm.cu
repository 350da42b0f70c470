// gemm.cu -- the matrix product of gemm.cuh on tcgen05, with the operators' epilogues.
//
// A cluster of two CTAs owns a tile of 512 or 256 rows and 256 columns (cta_group::2): of a
// 64-deep K block each CTA keeps 128 or 256 rows of A and half of the tile's B rows in shared
// memory (4 stages of 48 KB, or 6 of 32 KB).  Warp 0 loads (TMA), one thread of the leader CTA
// issues the MMAs of both, eight warps run the epilogue.  Bound by the tensor pipe where K is
// long, and before it by what L2 can feed the SMs: 256-row tiles ran at 1150-1200 TFLOP/s
// (8192^3; 1460 with the loads left out), 512-row tiles, which read B half as often, at
// 1400-1580.  Their two accumulators of 128 x 256 fp32 fill TMEM, so a tile's epilogue runs
// alone; with 256 rows there are two sets, and it runs beside the products of the next tile,
// which the long epilogue of the gate's backward needs.  For the gated kind of product the
// leader's B rows are the gate projection's and its peer's the up projection's, so both values
// of one hidden element meet in one thread.
//
// Either operand may be K-major or MN-major (the transposed products of the backward): only
// the TMA box and the shared-memory descriptor differ.  Rows and columns past the edges are
// read as zeros and not stored.
#include <algorithm>

#include "gemm.cuh"
#include "tc.cuh"

namespace mhc {
namespace gk {
constexpr int BM = 128;          // rows of A per CTA (256 per cluster)
constexpr int BNC = 128;         // rows of B per CTA (256 per cluster)
constexpr int BK = 64;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BNC * BK * 2;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int GROUP_ROWS = 2048;  // rows of tiles that walk the column tiles together
constexpr int STORE_BYTES = 2 * 2048;  // two boxes of 32 x 32 outputs per epilogue warp
// MT accumulators of 256 rows to a tile
template <int MT> struct Ring {
  static constexpr int STAGES = MT == 1 ? 6 : 4;
  static constexpr int STAGE_BYTES = MT * A_BYTES + B_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + STORE_BYTES * EPI_WARPS + 1024;  // and room to align
};
}  // namespace gk

struct GemmMaps {
  CUtensorMap a, b, b2, a3, b3;
  CUtensorMap out[3];  // the epilogue's outputs, in StoreRows' order
};
// How one launch walks the problem.
struct GemmWalk {
  int64_t M, N;                       // of the output
  int32_t tiles_m, tiles_n, nk1, nk;  // K blocks of the first segment, of both
  int32_t splits;                     // ranges of K, each a unit of work of its own
  float* part;                        // splits > 1: [splits][planes][M][ldp] partial products
  int64_t ldp;
};

namespace tc2 {
// address of the leader CTA's copy of a shared variable
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tc::smem_u32(p)));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// load into this CTA's shared memory; the bytes are counted on the leader's barrier
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                        int32_t x, int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                    uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrive on this barrier of both CTAs once all MMAs issued so far have completed
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(tc::smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
}  // namespace tc2

// Outputs by TMA: a warp's 32 x 32 chunk goes to one of its two boxes in shared memory (64-byte
// swizzle) and from there to HBM, whole lines at a time; rows and columns past the edges are
// clipped.  A thread owns a row here, so its own stores touch 32 lines to an instruction: with
// those, T=509, D=2048, F=5464 took 76 us for the gated block that keeps gate and up (58 us by TMA)
// and 58 us for the one that does not (54 us).  Large products do not notice, but for gate and up in
// fp32: 2.5% more than in 16 bits at T=4096, 4096/16384, 6% by the threads' stores.
struct StoreTma {
  const CUtensorMap* maps;
  char* box;      // of this warp
  int32_t row0;   // of the warp's chunk
  int lane;
  int next = 0;
  template <typename E, int NC>  // the type in memory; a chunk is one box of 16 bits, two of fp32
  __device__ __forceinline__ void put(int which, void*, int64_t, int64_t, int64_t col, int n, int,
                                      const float* f) {
    static_assert(NC == 32, "a chunk is 32 columns wide");
    constexpr int P = 16 / sizeof(E), PER = 4 * P;
#pragma unroll
    for (int c = 0; c < NC; c += PER) {
      if (c >= n) break;                       // a box that starts past the last column
      if (lane == 0) tc::bulk_wait_read<1>();  // the store before the last has read this box
      __syncwarp();
      char* b = box + next * 2048 + lane * 64;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(b + ((j ^ ((lane >> 1) & 3)) << 4)) = narrow<E>(f + c + P * j);
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        tc::tma_store_2d(&maps[which], box + next * 2048, (int32_t)col + c, row0);
        tc::bulk_commit_group();
      }
      next ^= 1;
    }
  }
};

// Unit u is tile u % tiles of K range u / tiles.  GROUP row tiles walk all column tiles together,
// so that the tiles in flight share their operands in L2.
struct Unit {
  int32_t mt, nt, split, kb0, kb1;
};
template <int MT>
__device__ __forceinline__ Unit unit_at(const GemmWalk& w, int32_t u) {
  Unit r;
  const int32_t tiles = w.tiles_m * w.tiles_n;
  r.split = u / tiles;
  const int32_t i = u - r.split * tiles;
  r.kb0 = (int32_t)((int64_t)w.nk * r.split / w.splits);
  r.kb1 = (int32_t)((int64_t)w.nk * (r.split + 1) / w.splits);
  constexpr int32_t GROUP = gk::GROUP_ROWS / (256 * MT);
  const int32_t per = GROUP * w.tiles_n;
  const int32_t g = i / per, rest = i - g * per;
  const int32_t rows = min(GROUP, w.tiles_m - g * GROUP);
  r.nt = rest / rows;
  r.mt = g * GROUP + rest - r.nt * rows;
  return r;
}

// AK, BKM: the operand is K-major
template <typename E, int KIND, int MT, bool AK, bool BKM>
__global__ void __launch_bounds__(gk::THREADS, 1)
    gemm_kernel(const __grid_constant__ GemmMaps maps, const __grid_constant__ GemmWalk w,
                const __grid_constant__ EpiParams epi) {
  using namespace gk;
  constexpr bool dual = KIND == kEpiGated;
  constexpr int STAGES = Ring<MT>::STAGES, STAGE_BYTES = Ring<MT>::STAGE_BYTES;
  constexpr int ROWS = 256 * MT;  // of a tile
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                       ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], tfull[2], tempty[2], tdone;
  __shared__ uint32_t tmem_slot, filled;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cta_rank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&tfull[i], 1);
      tc::mbar_init(&tempty[i], 2 * EPI_WARPS / MT);
    }
    tc::mbar_init(&tdone, 1);
    abort_word = 0;
    tc::fence_barrier_init();
    tc::prefetch_tmap(&maps.a);
    tc::prefetch_tmap(&maps.b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     tc::smem_u32(&tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();  // both CTAs' barriers are initialised
  tc::tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t*)&tmem_slot;
  pdl_enter();

  const int32_t units = w.tiles_m * w.tiles_n * w.splits;
  const int32_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
  // The two issuing loops are warp-wide and unrolled over the ring: barriers, addresses and
  // descriptors are then constants or uniform registers.
  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    const bool issue = tc::elect_one();
    const uint32_t base = tc::smem_u32(smem), bar0 = tc2::leader_addr(&full[0]);
    int32_t i = first, kb = 0, kb1 = 0, m0 = 0, n0 = 0;
    bool more = true;
    // the next K block of this cluster's units
    auto advance = [&]() {
      if (++kb < kb1) return;
      if (i >= units) {
        more = false;
        return;
      }
      const Unit u = unit_at<MT>(w, i);
      m0 = u.mt * ROWS + (int32_t)rank * BM;
      n0 = dual ? u.nt * BNC : u.nt * 2 * BNC + (int32_t)rank * BNC;
      kb = u.kb0;
      kb1 = u.kb1;
      i += step;
    };
    advance();
    for (uint32_t ph = 1; more; ph ^= 1) {
#pragma unroll
      for (int s = 0; s < STAGES; ++s) {
        if (!more) break;
        if (!tc::mbar_wait_warp(&empty[s], ph, abort_flag)) {
          more = false;
          if (issue) filled = tc::fills_at(s, ph);
          break;
        }
        const uint32_t bar = bar0 + s * 8;
        const uint32_t sa = base + s * STAGE_BYTES, sb = sa + MT * A_BYTES;
        const bool second = kb >= w.nk1;
        const int32_t k0 = (second ? kb - w.nk1 : kb) * BK;
        const CUtensorMap* ma = second ? &maps.a3 : &maps.a;
        const CUtensorMap* mb = second ? &maps.b3 : (dual && rank) ? &maps.b2 : &maps.b;
        if (issue) {
          if (leader) tc::mbar_arrive_expect_tx(&full[s], 2 * STAGE_BYTES);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint32_t dst = sa + m * A_BYTES;
            const int32_t r0 = m0 + m * 256;
            if constexpr (AK) {
              tc2::load_2d(dst, ma, bar, k0, r0);
            } else {
              tc2::load_2d(dst, ma, bar, r0, k0);
              tc2::load_2d(dst + A_BYTES / 2, ma, bar, r0 + 64, k0);
            }
          }
          if constexpr (BKM) {
            tc2::load_2d(sb, mb, bar, k0, n0);
          } else {
            tc2::load_2d(sb, mb, bar, n0, k0);
            tc2::load_2d(sb + B_BYTES / 2, mb, bar, n0 + 64, k0);
          }
        }
        __syncwarp();
        advance();
        if (!more && issue) filled = tc::fills_at(s + 1, ph);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs
    if (leader) {
      constexpr uint32_t idesc = tc::idesc_16<E>(256, 256, !AK, !BKM);
      // descriptor step of 16 K elements: 32 bytes of a K-major row, or two 8-row atoms
      constexpr uint32_t stepa = AK ? 2 : 128, stepb = BKM ? 2 : 128;
      const uint32_t base = tc::smem_u32(smem);
      const uint64_t da0 = tc::smem_desc(base, AK ? 16 : A_BYTES / 2, 1024, tc::kSwizzle128);
      const uint64_t db0 =
          tc::smem_desc(base + MT * A_BYTES, BKM ? 16 : B_BYTES / 2, 1024, tc::kSwizzle128);
      const bool issue = tc::elect_one();
      int32_t i = first, left = 0;  // K blocks left of this unit
      uint32_t j = 0, buf = 0, accum = 0;
      bool more = i < units;
      for (uint32_t ph = 0; more; ph ^= 1) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
          if (left == 0) {  // the next unit
            if (i >= units) {
              more = false;
              break;
            }
            const Unit u = unit_at<MT>(w, i);
            left = u.kb1 - u.kb0;
            i += step;
            accum = 0;
            // MT = 1: units take the two accumulators in turn; MT = 2: each takes both
            buf = MT == 1 ? j & 1 : 0;
            const uint32_t tph = (MT == 1 ? (j >> 1) & 1 : j & 1) ^ 1;
            ++j;
            if (!tc::mbar_wait_warp(&tempty[buf], tph, abort_flag) ||
                (MT == 2 && !tc::mbar_wait_warp(&tempty[1], tph, abort_flag))) {
              more = false;
              break;
            }
            tc::tc_fence_after();
          }
          if (!tc::mbar_wait_warp(&full[s], ph, abort_flag)) {
            more = false;
            break;
          }
          tc::tc_fence_after();
          --left;
          if (issue) {
            const uint64_t da = da0 + s * (STAGE_BYTES >> 4), db = db0 + s * (STAGE_BYTES >> 4);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                tc2::mma(tmem + (buf + m) * 256, da + m * (A_BYTES >> 4) + k * stepa,
                         db + k * stepb, idesc, k != 0 ? 1u : accum);
              if (MT == 2 && left == 0) tc2::commit_both(&tfull[m]);
            }
            tc2::commit_both(&empty[s]);
            if (MT == 1 && left == 0) tc2::commit_both(&tfull[buf]);
          }
          accum = 1;
          __syncwarp();
        }
      }
      if (issue) tc2::commit_both(&tdone);  // every MMA is done before TMEM is freed
    }
    __syncwarp();
    volatile int never = 0;
    tc::mbar_wait(&tdone, 0, &never);
  } else {
    // ---------------------------------------------------------------- epilogue
    // eight warps, four lane quarters: the pair of a quarter splits the columns of the one
    // accumulator, or takes an accumulator each
    constexpr int COLS = (dual ? BNC : 2 * BNC) / (MT == 1 ? 2 : 1);  // output columns per warp
    const int q = warp & 3, pair = (warp - 2) >> 2;
    const int col_off = MT == 1 ? pair * COLS : 0;
    const uint32_t tq = tmem + ((uint32_t)(q * 32) << 16) + col_off;
    StoreTma st{maps.out, smem + STAGES * STAGE_BYTES + (warp - 2) * STORE_BYTES, 0, lane};
    uint32_t j = 0;
    for (int32_t i = first; i < units; i += step, ++j) {
      const Unit u = unit_at<MT>(w, i);
      const uint32_t buf = MT == 1 ? j & 1 : pair, ph = MT == 1 ? (j >> 1) & 1 : j & 1;
      const int64_t row0 = (int64_t)u.mt * ROWS + (MT == 1 ? 0 : pair * 256) + rank * BM + q * 32;
      const int64_t row = row0 + lane, rrow = row < w.M ? row : w.M - 1;
      st.row0 = (int32_t)row0;
      const int64_t col0 = (int64_t)u.nt * (dual ? BNC : 2 * BNC) + col_off;
      // kEpiGatedBwd reads gate and up: a chunk ahead, the first before the products are done.
      // kEpiGatedBwd32, whose chunk would take 64 registers, asks for its lines in L2 instead (T=4096,
      // 4096/16384: 455 us; 492 us with the whole tile's lines at its start, some of which were gone
      // again when they were read).
      constexpr bool ahead = KIND == kEpiGatedBwd;
      Raw32 pre[ahead ? 4 : 1];
      auto fetch = [&](int c) {
        if constexpr (KIND == kEpiGatedBwd32) {
          if (w.splits == 1 && col0 + c < w.N) {  // a chunk's row is 128 bytes
            const int64_t at = rrow * epi.ld_gu + col0 + c;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const float*>(epi.gate) + at));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const float*>(epi.up) + at));
          }
        }
        if constexpr (ahead) {
          if (epi.vec == 2 && w.splits == 1 && col0 + c + 32 <= w.N) {
            const E* pg = reinterpret_cast<const E*>(epi.gate) + rrow * epi.ld_gu + col0 + c;
            const E* pu = reinterpret_cast<const E*>(epi.up) + rrow * epi.ld_gu + col0 + c;
            pre[0] = ld_row32(pg); pre[1] = ld_row32(pg + 16);
            pre[2] = ld_row32(pu); pre[3] = ld_row32(pu + 16);
          }
        }
      };
      fetch(0);
      const bool got = tc::mbar_wait(&tfull[buf], ph, abort_flag);
      if (!__all_sync(0xffffffffu, got)) break;
      tc::tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < COLS; c += 32) {
        __syncwarp();  // rows past M skip the epilogue below
        float acc[32], acc2[dual ? 32 : 1];
        tc2::ld32(tq + buf * 256 + c, acc);
        if constexpr (dual) tc2::ld32(tq + buf * 256 + BNC + c, acc2);
        tc::tmem_ld_wait();
        if (c + 32 == COLS) {  // the accumulators have been read
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc2::arrive_cluster(tc2::leader_addr(&tempty[buf]));
        }
        const int64_t left = w.N - (col0 + c);
        if (left <= 0 || row0 >= w.M) continue;  // the whole warp's chunk
        const int n = left < 32 ? (int)left : 32;
        if (w.splits > 1) {  // ldp is N rounded up to 32
          if (row < w.M) {
            float* d = w.part + ((int64_t)u.split * (dual ? 2 : 1) * w.M + row) * w.ldp + col0 + c;
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              st_row32(d + k, narrow<float>(acc + k), narrow<float>(acc + k + 4));
            if constexpr (dual) {
              d += w.M * w.ldp;
#pragma unroll
              for (int k = 0; k < 32; k += 8)
                st_row32(d + k, narrow<float>(acc2 + k), narrow<float>(acc2 + k + 4));
            }
          }
        } else if (epi.vec) {
          // every lane takes part in the stores; lanes past the last row read that row again
          const float* more = dual ? acc2 : nullptr;
          if constexpr (ahead) {
            if (epi.vec == 2 && n == 32) {
              float gu[64];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                widen<E>(pre[k].a, gu + 16 * k);
                widen<E>(pre[k].b, gu + 16 * k + 8);
              }
              if (c + 32 < COLS) fetch(c + 32);
              epi_chunk<E, KIND, 32>(epi, rrow, col0 + c, n, acc, gu, st);
            } else {
              epi_chunk<E, KIND, 32>(epi, rrow, col0 + c, n, acc, more, st);
            }
          } else {
            if (c + 32 < COLS) fetch(c + 32);
            epi_chunk<E, KIND, 32>(epi, rrow, col0 + c, n, acc, more, st);
          }
        } else if (row < w.M) {
          epi_chunk<E, KIND, 32>(epi, row, col0 + c, n, acc, dual ? acc2 : nullptr);
        }
      }
    }
    if (lane == 0) tc::bulk_wait_all<0>();  // the outputs have landed
  }
  __syncwarp();
  if (*abort_flag && threadIdx.x == 0) flag_timeout();
  tc::tc_fence_before();
  __syncthreads();
  // the loads of both CTAs are counted on the leader's barriers
  if (leader && *abort_flag && threadIdx.x == 0) tc::drain(full, STAGES, filled);
  tc::cluster_sync();  // neither CTA leaves while the other may still signal it
  if (warp == 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Sums the K ranges' partial products in order and runs the epilogue: 8 columns to a thread.
template <typename E, int KIND>
__global__ void __launch_bounds__(256)
    gemm_finish_kernel(const float* __restrict__ part, int splits, int64_t M, int64_t N,
                       int64_t ldp, const __grid_constant__ EpiParams epi) {
  pdl_enter();
  constexpr int PL = KIND == kEpiGated ? 2 : 1;
  const int64_t cols = ldp / 8, n = M * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / cols, col = (i - row * cols) * 8;
    if (col >= N) continue;
    float acc[PL][8] = {};
#pragma unroll
    for (int p = 0; p < PL; ++p) {
      const float* d = part + ((int64_t)p * M + row) * ldp + col;
#pragma unroll 4
      for (int s = 0; s < splits; ++s, d += PL * M * ldp) {
        const float4 a = *reinterpret_cast<const float4*>(d);
        const float4 b = *reinterpret_cast<const float4*>(d + 4);
        acc[p][0] += a.x; acc[p][1] += a.y; acc[p][2] += a.z; acc[p][3] += a.w;
        acc[p][4] += b.x; acc[p][5] += b.y; acc[p][6] += b.z; acc[p][7] += b.w;
      }
    }
    epi_chunk<E, KIND, 8>(epi, row, col, N - col < 8 ? (int)(N - col) : 8, acc[0],
                          PL == 2 ? acc[PL - 1] : nullptr);
  }
}

static int64_t k_blocks(const Gemm& g) { return cdiv(g.K, gk::BK) + cdiv(g.K3, gk::BK); }
static int64_t part_ld(const Gemm& g) { return cdiv(g.N, 32) * 32; }

// The cut whose estimated time (us) is least.  Measured: 7 us to start and end a launch; 0.36 us
// to a K block of a 256-row tile and 0.73 us of a 512-row one in a short run, 0.50 and 0.86 us
// under the power cap (the 512-row tile reads B half as often for its work), and 0.28 and 0.56 us
// with few clusters at work; the constants lie between.  The 512-row tile's
// epilogue, with no accumulators left for the next tile, stands alone: 2 us, 3 us with a gate,
// 20 us with the gate's backward.  A cut in K writes and reads fp32 partials (at 4 TB/s) and
// takes another launch (3 us).
GemmPlan gemm_plan(const Gemm& g) {
  const bool dual = g.kind == kEpiGated;
  const int64_t nk = k_blocks(g), clusters = sm_count() / 2;
  const int64_t tn = cdiv(g.N, dual ? gk::BNC : 2 * gk::BNC);
  const double plane = (double)g.M * (double)part_ld(g) * (dual ? 2 : 1);
  GemmPlan best{0, 1, 0};
  double best_us = few_estimate(g, &best.nt, &best.splits);
  if (best_us == 0.0) best = {1, 1, 0}, best_us = 1e30;
  for (int mt = 1; mt <= 2; ++mt) {
    if (mt == 2 && g.M <= 256) break;
    const int64_t tiles = cdiv(g.M, 256 * mt) * tn;
    const double tail = mt == 1 ? 1.0 : g.kind == kEpiLinear ? 2.0 : dual ? 3.0 : 20.0;
    for (int sp = 1; sp <= 16; ++sp) {
      // (beyond eight waves a cut gains nothing)
      if (sp > 1 && (nk < 4 * sp || plane * sp * 4 > 1e9 || tiles * (sp - 1) > 8 * clusters)) break;
      const double waves = (double)cdiv(tiles * sp, clusters);
      const double busy = std::min(1.0, (double)(tiles * sp) / (double)clusters);
      const double per_k = mt == 1 ? 0.28 + 0.12 * busy : 0.56 + 0.19 * busy;
      double us = 7.0 + waves * ((double)cdiv(nk, sp) * per_k + tail);
      if (sp > 1) us += 3.0 + plane * sp * 8 / 4e6;
      if (us < best_us) best_us = us, best = {mt, sp, 0};
    }
  }
  return best;
}

size_t gemm_ws_bytes(const Gemm& g) {
  const GemmPlan p = gemm_plan(g);
  if (p.splits == 1 || p.mt == 0) return 0;
  return align_up((size_t)p.splits * (g.kind == kEpiGated ? 2 : 1) * g.M * part_ld(g) * 4);
}

int epi_vec(const EpiParams& e) {
  uintptr_t bits = 0;
  for (const void* p : {(const void*)e.out, e.bias, e.res, (const void*)e.z, (const void*)e.gate,
                        (const void*)e.up, (const void*)e.gg, (const void*)e.gu})
    bits |= reinterpret_cast<uintptr_t>(p);
  for (int64_t ld : {e.ld_out, e.ld_res, e.gu32 ? 2 * e.ld_gu : e.ld_gu, e.ld_g})
    bits |= (uintptr_t)ld * 2;
  return (bits & 31) == 0 ? 2 : (bits & 15) == 0 ? 1 : 0;
}

bool operand_aligned(const Operand& o) { return aligned16(o.p) && o.ld % 8 == 0; }

static int operand_map(CUtensorMap* m, const Operand& o, int32_t dtype, int64_t mn, int64_t k) {
  const CUtensorMapDataType dt =
      dtype == MHC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return o.k_major ? make_tmap_2d(m, o.p, dt, 2, k, mn, o.ld * 2, gk::BK, gk::BM,
                                  CU_TENSOR_MAP_SWIZZLE_128B)
                   : make_tmap_2d(m, o.p, dt, 2, mn, k, o.ld * 2, 64, gk::BK,
                                  CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename E, int KIND, int MT, bool AK, bool BKM>
static int gemm_launch(const Gemm& g, int splits, float* part, cudaStream_t s) {
  using namespace gk;
  constexpr bool dual = KIND == kEpiGated;
  GemmMaps m;
  int st = MHC_OK;
  if ((st = operand_map(&m.a, g.a, g.dtype, g.M, g.K))) return st;
  if ((st = operand_map(&m.b, g.b, g.dtype, g.N, g.K))) return st;
  m.b2 = m.b; m.a3 = m.a; m.b3 = m.b;
  if (dual && (st = operand_map(&m.b2, g.b2, g.dtype, g.N, g.K))) return st;
  if (g.K3 > 0) {
    if ((st = operand_map(&m.a3, g.a3, g.dtype, g.M, g.K3))) return st;
    if ((st = operand_map(&m.b3, g.b3, g.dtype, g.N, g.K3))) return st;
  }
  for (CUtensorMap& o : m.out) o = m.a;
  if (splits == 1 && g.epi.vec) {
    const EpiParams& e = g.epi;
    auto out = [&](int i, const void* p, int64_t ld, bool f32 = false) {
      if (!p || st) return;
      const int size = f32 ? 4 : 2;
      st = make_tmap_2d(&m.out[i], p,
                        f32                  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : g.dtype == MHC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                             : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                        size, g.N, g.M, ld * size, 64 / size, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    };
    out(0, e.out, e.ld_out);
    if (KIND == kEpiLinear) out(1, e.z, e.ld_out);
    if (KIND == kEpiGated) out(1, e.gate, e.ld_gu, e.gu32), out(2, e.up, e.ld_gu, e.gu32);
    if (KIND == kEpiGatedBwd || KIND == kEpiGatedBwd32) out(1, e.gg, e.ld_g), out(2, e.gu, e.ld_g);
    if (st) return st;
  }
  GemmWalk w;
  w.M = g.M; w.N = g.N;
  w.tiles_m = (int32_t)cdiv(g.M, 256 * MT);
  w.tiles_n = (int32_t)cdiv(g.N, dual ? BNC : 2 * BNC);
  w.nk1 = (int32_t)cdiv(g.K, BK);
  w.nk = w.nk1 + (int32_t)cdiv(g.K3, BK);
  w.splits = splits;
  w.part = part;
  w.ldp = part_ld(g);
  constexpr int smem = Ring<MT>::SMEM;
  static bool attr_set[64];
  int dev = 0;
  MHC_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    MHC_CUDA_CHECK(cudaFuncSetAttribute((const void*)gemm_kernel<E, KIND, MT, AK, BKM>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t units = (int64_t)w.tiles_m * w.tiles_n * splits;
  if (units > INT32_MAX / 2) return MHC_ERR_INVALID_ARGUMENT;
  const int clusters = (int)std::min<int64_t>(units, sm_count() / 2);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = (!pdl_first_launch() && pdl_enabled()) ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, gemm_kernel<E, KIND, MT, AK, BKM>, m, w, g.epi) != cudaSuccess) {
    (void)cudaGetLastError();
    return MHC_ERR_CUDA;
  }
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

template <typename E, int KIND, bool AK, bool BKM>
static int gemm_kind(const Gemm& g, void* ws, cudaStream_t s) {
  const GemmPlan p = gemm_plan(g);
  if (p.mt == 0) return few_run(g, p.nt, p.splits, s);
  float* part = p.splits > 1 ? (float*)ws : nullptr;
  const int st = p.mt == 2 ? gemm_launch<E, KIND, 2, AK, BKM>(g, p.splits, part, s)
                           : gemm_launch<E, KIND, 1, AK, BKM>(g, p.splits, part, s);
  if (st != MHC_OK || !part) return st;
  const int64_t n = g.M * (part_ld(g) / 8);
  launch(gemm_finish_kernel<E, KIND>, (unsigned)std::min<int64_t>(cdiv(n, 256), 8 * sm_count()),
         256, 0, s, (const float*)part, p.splits, g.M, g.N, part_ld(g), g.epi);
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

template <typename E>
static int gemm_typed(const Gemm& g, void* ws, cudaStream_t s) {
  // the operands' orders that the operators meet
  if (g.kind == kEpiGated) return gemm_kind<E, kEpiGated, true, true>(g, ws, s);
  if (g.kind == kEpiGatedBwd) return gemm_kind<E, kEpiGatedBwd, true, false>(g, ws, s);
  if (g.kind == kEpiGatedBwd32) return gemm_kind<E, kEpiGatedBwd32, true, false>(g, ws, s);
  if (!g.a.k_major) return gemm_kind<E, kEpiLinear, false, false>(g, ws, s);
  return g.b.k_major ? gemm_kind<E, kEpiLinear, true, true>(g, ws, s)
                     : gemm_kind<E, kEpiLinear, true, false>(g, ws, s);
}

int gemm_run(const Gemm& g0, void* ws, cudaStream_t s) {
  Gemm g = g0;
  g.epi.vec = epi_vec(g.epi);
  return g.dtype == MHC_F16 ? gemm_typed<__half>(g, ws, s) : gemm_typed<__nv_bfloat16>(g, ws, s);
}

int gemm_device_error() { return read_and_clear_tu_error(); }

// ---------------------------------------------------------------- packed copies
// Rows of 2-byte elements, copied between matrices whose rows start anywhere.  A thread writes
// one 16-byte chunk of a row, aligned in the destination; its source, shifted against that, comes
// from the two aligned 16-byte words that hold it (a warp's threads share them in L1).  Bound by
// HBM; with an element to a thread the 6704 x 11861 weight took 300 us of a gated block's 430.
// `begin`, `end`: the source matrix, past which no word is read.
template <typename I>  // of the chunks' count
__global__ void __launch_bounds__(256)
    pack_rows_kernel(const char* __restrict__ src, int64_t ls, int64_t rows, int64_t cols,
                     char* __restrict__ dst, int64_t ld, const char* begin, const char* end) {
  pdl_enter();
  const I per = (I)((cols + 7) / 8 + 1), total = (I)rows * per;  // a row may touch one chunk more
  for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += (I)gridDim.x * 256) {
    const I r = i / per;
    const char* sp = src + (int64_t)r * ls;
    char* dp = dst + (int64_t)r * ld;
    const int64_t e0 = (int64_t)(i - r * per) * 8 - (int64_t)((reinterpret_cast<uintptr_t>(dp) & 15) >> 1);
    if (e0 >= cols) continue;
    if (e0 >= 0 && e0 + 8 <= cols) {
      const char* sa = sp + e0 * 2;
      const int sh = (int)((reinterpret_cast<uintptr_t>(sa) & 15) >> 1);  // elements
      const char* a0 = sa - 2 * sh;
      uint32_t w[8];
      if (sh == 0 || (a0 >= begin && a0 + 32 <= end)) {
        const uint4 lo = *reinterpret_cast<const uint4*>(a0);
        const uint4 hi = sh ? *reinterpret_cast<const uint4*>(a0 + 16) : make_uint4(0, 0, 0, 0);
        w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w;
        w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
        if (sh & 4) {
#pragma unroll
          for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
        }
        if (sh & 2) {
#pragma unroll
          for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
        }
        if (sh & 1) {
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
        }
      } else {
        const uint16_t* se = reinterpret_cast<const uint16_t*>(sa);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = se[2 * k] | (uint32_t)se[2 * k + 1] << 16;
      }
      *reinterpret_cast<uint4*>(dp + e0 * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      const int64_t e1 = e0 + 8 < cols ? e0 + 8 : cols;
      for (int64_t e = e0 > 0 ? e0 : 0; e < e1; ++e)
        *reinterpret_cast<uint16_t*>(dp + 2 * e) = *reinterpret_cast<const uint16_t*>(sp + 2 * e);
    }
  }
}

int pack_rows(const void* src, int64_t ls, int64_t rows, int64_t cols, void* dst, int64_t ld,
              cudaStream_t s) {
  const char* begin = (const char*)src;
  const char* end = begin + ((rows - 1) * ls + cols) * 2;
  const int64_t total = rows * ((cols + 7) / 8 + 1);
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(total, 256), 32 * sm_count());
  launch(total < INT32_MAX / 2 ? pack_rows_kernel<uint32_t> : pack_rows_kernel<uint64_t>, grid, 256, 0, s,
         begin, ls * 2, rows, cols, (char*)dst, ld * 2, begin, end);
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

}  // namespace mhc
