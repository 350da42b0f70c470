// layer_norm.cu -- layer norm over the last dimension, forward and backward.
#include <math.h>

#include <algorithm>
#include <utility>

#include "tc.cuh"

namespace mhc {

// Both directions read HBM once and write it once.  A row belongs to WARPS warps, whose
// threads hold EPT of its elements each in registers, so the centred sum of squares costs no
// second read.  Rows are read in 16-byte packs where their addresses allow it, else element
// by element (still whole sectors per warp).  Rows wider than kLnMaxD go to the loop kernels
// below, which read them again from L2 for each sum.
static constexpr int kLnThreads = 256;
static constexpr int kLnMaxStages = 16;

// Sums over the threads of one row; red has two rows of slots per warp, used in turn, so one
// barrier per sum is enough.
template <int WARPS, int NS>
__device__ __forceinline__ void row_sums(float* v, float (*red)[NS][WARPS], int par) {
#pragma unroll
  for (int i = 0; i < NS; ++i) v[i] = warp_sum(v[i]);
  if constexpr (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < NS; ++i) red[par][i][threadIdx.x >> 5] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) s += red[par][i][k];
      v[i] = s;
    }
  }
}

// Two fp32 operations to an instruction; the kernels would be bound by their instructions
// otherwise (a row of 16-bit elements leaves 1.6 cycles of an SM to an element and direction).
__device__ __forceinline__ uint64_t pk(float2 v) {
  return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x);
}
__device__ __forceinline__ float2 unpk(uint64_t v) {
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pk(a)), "l"(pk(b)));
  return unpk(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pk(a)), "l"(pk(b)));
  return unpk(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pk(a)), "l"(pk(b)), "l"(pk(c)));
  return unpk(r);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// One element, or 0 where `in` is false; BYTES: offset from p.  Volatile: the compiler may move
// an asm that only has outputs out of the branch or past the wait that guards the address.
template <int BYTES>
__device__ __forceinline__ uint32_t ld_raw(const float* p, int in) {
  uint32_t r;
  asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; mov.b32 %0, 0; @q ld.global.nc.b32 %0, [%1+%3];}"
      : "=r"(r)
      : "l"(p), "r"(in), "n"(BYTES));
  return r;
}
template <int BYTES, typename E>
__device__ __forceinline__ uint16_t ld_raw(const E* p, int in) {
  uint16_t r;
  asm volatile("{.reg .pred q; setp.ne.b32 q, %2, 0; mov.b16 %0, 0; @q ld.global.nc.b16 %0, [%1+%3];}"
      : "=h"(r)
      : "l"(p), "r"(in), "n"(BYTES));
  return r;
}
template <typename E> __device__ __forceinline__ float widen1(uint16_t v) {
  return from_e(*reinterpret_cast<const E*>(&v));
}
template <typename E> __device__ __forceinline__ float widen1(uint32_t v) {
  return __uint_as_float(v);
}
template <typename E, int GT, int V, int... I>
__device__ __forceinline__ void ld_elems(const E* p, int tid, int D, float* f,
                                         std::integer_sequence<int, I...>) {
  decltype(ld_raw<0>(p, 0)) raw[V] = {
      ld_raw<I * GT * (int)sizeof(E)>(p, I * GT + tid < D)...};  // all in flight together
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = widen1<E>(raw[v]);
}

// A thread's share of a row, widened: V packs of PN elements (16 bytes) or V single ones.  The
// packs of a row go round its GT threads; past the row's end the share is 0.
template <typename E, int PN, int GT, int V>
__device__ __forceinline__ void ld_row(const E* row, int tid, int D, float* f) {
  if constexpr (PN == 1) {
    ld_elems<E, GT, V>(row + tid, tid, D, f, std::make_integer_sequence<int, V>{});
  } else {
    uint4 raw[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      raw[v] = (v * GT + tid) * PN < D ? ld_stream(row + (v * GT + tid) * PN)
                                       : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int v = 0; v < V; ++v) widen<E>(raw[v], f + v * PN);
  }
}
// the same columns of a parameter, or `fill` where there is none
template <int PN, int GT, int V>
__device__ __forceinline__ void ld_params(const float* p, int tid, int D, float fill, float* f) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V * PN; ++i) f[i] = fill;
  } else if constexpr (PN == 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = v * GT + tid < D ? __ldg(p + v * GT + tid) : 0.f;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < PN; i += 4)
        widen<float>((v * GT + tid) * PN < D ? ld_keep(p + (v * GT + tid) * PN + i)
                                             : make_uint4(0, 0, 0, 0),
                     f + v * PN + i);
  }
}
template <typename E, int PN, int GT, int V>
__device__ __forceinline__ void st_row(E* row, int tid, int D, const float* f) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * GT + tid) * PN;
    if (c < D) {
      if constexpr (PN == 1)
        st1<E>(row + c, f[v]);
      else
        st_stream(row + c, narrow<E>(f + v * PN));
    }
  }
}

template <typename E, int PN, int WARPS, int V>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS, WARPS == 1 ? 6 : WARPS == 32 ? 1 : 24 / WARPS)
    ln_fwd_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ w,
                  const float* __restrict__ b, int64_t T, int D, float eps, E* __restrict__ y,
                  float* __restrict__ mean, float* __restrict__ rstd) {
  pdl_enter();
  constexpr int ROWS = WARPS == 1 ? 4 : 1, GT = 32 * WARPS, EPT = V * PN;
  __shared__ float red[2][1][WARPS];
  const int tid = threadIdx.x % GT;
  for (int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / GT; t < T;
       t += (int64_t)gridDim.x * ROWS) {
    float2 f[EPT / 2];
    ld_row<E, PN, GT, V>(x + t * xs, tid, D, reinterpret_cast<float*>(f));
    float2 s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) s2 = add2(s2, f[i]);
    float s = s2.x + s2.y;
    row_sums<WARPS, 1>(&s, red, 0);
    const float m = s / (float)D;
    s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      f[i] = add2(f[i], both(-m));
      // elements past the end are packs (or single elements) as a whole
      const int c0 = ((2 * i / PN) * GT + tid) * PN, c1 = (((2 * i + 1) / PN) * GT + tid) * PN;
      float2 c = f[i];
      if (c0 >= D) c.x = 0.f;
      if (c1 >= D) c.y = 0.f;
      s2 = fma2(c, c, s2);
    }
    s = s2.x + s2.y;
    row_sums<WARPS, 1>(&s, red, 1);
    const float rs = rsqrtf(s / (float)D + eps);
    float2 p[EPT / 2], q[EPT / 2];
    ld_params<PN, GT, V>(w, tid, D, 1.f, reinterpret_cast<float*>(p));
    ld_params<PN, GT, V>(b, tid, D, 0.f, reinterpret_cast<float*>(q));
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) f[i] = fma2(mul2(f[i], both(rs)), p[i], q[i]);
    st_row<E, PN, GT, V>(y + t * D, tid, D, reinterpret_cast<const float*>(f));
    if (tid == 0) {
      if (mean) mean[t] = m;
      if (rstd) rstd[t] = rs;
    }
  }
}

// Wide rows on 16-byte boundaries: persistent blocks, 16 warps of them to an SM, whose rows
// arrive by bulk copies in a ring of shared memory, several rows ahead; weight and bias stay in
// registers.  One barrier a row: each warp centres on its own mean, and the warps' means and
// sums of squares are joined (M2 = sum M2_i + sum n_i (m_i - m)^2).
template <typename E, int WARPS, int V>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS)
    ln_fwd_ring_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ w,
                       const float* __restrict__ b, int64_t T, int D, float eps,
                       E* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                       int stages) {
  constexpr int PN = Pack<E>::n, GT = 32 * WARPS, EPT = V * PN;
  extern __shared__ __align__(16) char ring[];
  __shared__ __align__(8) uint64_t full[kLnMaxStages];
  __shared__ float red[2][2][WARPS], n_of[WARPS];
  __shared__ int abort_word;
  __shared__ uint32_t filled;  // thread 0's: the parity of each stage's last fill
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t row_bytes = (uint32_t)D * sizeof(E);
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
    abort_word = 0;
    filled = ~0u;
    tc::fence_barrier_init();
  }
  __syncthreads();
  pdl_enter();
  auto fetch = [&](int64_t t, int s) {
    filled ^= 1u << s;
    tc::mbar_arrive_expect_tx(&full[s], row_bytes);
    tc::bulk_load(ring + (size_t)s * row_bytes, x + t * xs, row_bytes, &full[s]);
  };
  const int64_t step = gridDim.x;
  if (tid == 0) {
    int64_t t = blockIdx.x;
    for (int s = 0; s < stages && t < T; ++s, t += step) fetch(t, s);
  }
  float2 p[EPT / 2], q[EPT / 2];
  ld_params<PN, GT, V>(w, tid, D, 1.f, reinterpret_cast<float*>(p));
  ld_params<PN, GT, V>(b, tid, D, 0.f, reinterpret_cast<float*>(q));
  // elements of warp k's share: pack v of lane l is pack v GT + 32 k + l of the row
  auto count = [&](int k) {
    int n = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) n += max(0, min(32 * PN, D - (v * GT + 32 * k) * PN));
    return (float)n;
  };
  const float n_own = count(warp), inv_own = n_own > 0.f ? 1.f / n_own : 0.f;
  const float inv_d = 1.f / (float)D;
  if (lane == 0) n_of[warp] = n_own;  // read after the first row's barrier
  int s = 0, par = 0;
  uint32_t ph = 0;
  for (int64_t t = blockIdx.x; t < T; t += step, par ^= 1) {
    if (!tc::mbar_wait(&full[s], ph, &abort_word)) flag_timeout();
    float2 f[EPT / 2], a = both(0.f);
    const uint4* sx = reinterpret_cast<const uint4*>(ring + (size_t)s * row_bytes);
#pragma unroll
    for (int v = 0; v < V; ++v)
      widen<E>((v * GT + tid) * PN < D ? sx[v * GT + tid] : make_uint4(0, 0, 0, 0),
               reinterpret_cast<float*>(f) + v * PN);
    tc::fence_proxy_async();  // these reads before the refill of the stage
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) a = add2(a, f[i]);
    const float mw = warp_sum(a.x + a.y) * inv_own;
    a = both(0.f);
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      if (((2 * i / PN) * GT + tid) * PN < D) {
        const float2 c = add2(f[i], both(-mw));
        a = fma2(c, c, a);
      }
    }
    const float m2w = warp_sum(a.x + a.y);
    if (lane == 0) red[par][0][warp] = mw, red[par][1][warp] = m2w;
    __syncthreads();
    if (tid == 0 && t + step * stages < T) fetch(t + step * stages, s);
    float m = 0.f, m2 = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) m = fmaf(n_of[k], red[par][0][k], m);
    m *= inv_d;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float d = red[par][0][k] - m;
      m2 += fmaf(n_of[k] * d, d, red[par][1][k]);
    }
    const float rs = rsqrtf(m2 * inv_d + eps);
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i)
      f[i] = fma2(mul2(add2(f[i], both(-m)), both(rs)), p[i], q[i]);
    st_row<E, PN, GT, V>(y + t * D, tid, D, reinterpret_cast<const float*>(f));
    if (tid == 0) {
      if (mean) mean[t] = m;
      if (rstd) rstd[t] = rs;
    }
    if (++s == stages) s = 0, ph ^= 1;
  }
  if (tid == 0 && *(volatile int*)&abort_word) tc::drain(full, stages, filled);
}

// The part of the backward that follows the loads: sums over the row, grad_x, and with PARAMS
// this thread's column sums.  f = x, g = grad_y.
template <typename E, int PN, int WARPS, int V, bool PARAMS>
__device__ __forceinline__ void ln_bwd_row(float2* f, float2* g, const float* w, float m, float r,
                                           int tid, int D, float inv_d, float (*red)[2][WARPS],
                                           int par, E* gx, float2* aw, float2* ab) {
  constexpr int GT = 32 * WARPS, EPT = V * PN;
  float2 s0 = both(0.f), s1 = both(0.f);
  {
    float2 p[EPT / 2];
    ld_params<PN, GT, V>(w, tid, D, 1.f, reinterpret_cast<float*>(p));
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {  // past the row's end g is 0: nothing there counts
      f[i] = mul2(add2(f[i], both(-m)), both(r));
      if constexpr (PARAMS) {
        aw[i] = fma2(g[i], f[i], aw[i]);
        ab[i] = add2(ab[i], g[i]);
      }
      g[i] = mul2(g[i], p[i]);
      s0 = add2(s0, g[i]);
      s1 = fma2(g[i], f[i], s1);
    }
  }
  float s[2] = {s0.x + s0.y, s1.x + s1.y};
  row_sums<WARPS, 2>(s, red, par);
  // r (h - c1 - xh c2)
  const float2 c1 = both(-s[0] * inv_d), c2 = both(-s[1] * inv_d);
#pragma unroll
  for (int i = 0; i < EPT / 2; ++i) g[i] = mul2(add2(g[i], fma2(f[i], c2, c1)), both(r));
  st_row<E, PN, GT, V>(gx, tid, D, reinterpret_cast<const float*>(g));
}

template <int PN, int GT, int V>
__device__ __forceinline__ void ln_bwd_partials(float* part, int tid, int D, const float2* aw2,
                                                const float2* ab2) {
  const float *aw = reinterpret_cast<const float*>(aw2), *ab = reinterpret_cast<const float*>(ab2);
  float* pw = part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * GT + tid) * PN;
    if (c < D) {
#pragma unroll
      for (int i = 0; i < PN; ++i) pw[c + i] = aw[v * PN + i], pw[D + c + i] = ab[v * PN + i];
    }
  }
}

// grad_x, and with PARAMS the column sums of this block's rows: part[block][2][D]
template <typename E, int PN, int WARPS, int V, bool PARAMS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS)
    ln_bwd_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ w,
                  const float* __restrict__ mean, const float* __restrict__ rstd,
                  const E* __restrict__ gy, int64_t gs, int64_t T, int D, E* __restrict__ gx,
                  float* __restrict__ part) {
  pdl_enter();
  constexpr int ROWS = WARPS == 1 ? 4 : 1, GT = 32 * WARPS, EPT = V * PN;
  __shared__ float red[2][2][WARPS];
  const int tid = threadIdx.x % GT;
  const float inv_d = 1.f / (float)D;
  float2 aw[PARAMS ? EPT / 2 : 1], ab[PARAMS ? EPT / 2 : 1];
#pragma unroll
  for (int i = 0; i < (PARAMS ? EPT / 2 : 1); ++i) aw[i] = ab[i] = both(0.f);
  int par = 0;
  for (int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / GT; t < T;
       t += (int64_t)gridDim.x * ROWS, par ^= 1) {
    float2 f[EPT / 2], g[EPT / 2];
    const float m = __ldg(mean + t), r = __ldg(rstd + t);
    ld_row<E, PN, GT, V>(x + t * xs, tid, D, reinterpret_cast<float*>(f));
    ld_row<E, PN, GT, V>(gy + t * gs, tid, D, reinterpret_cast<float*>(g));
    ln_bwd_row<E, PN, WARPS, V, PARAMS>(f, g, w, m, r, tid, D, inv_d, red, par, gx + t * D, aw,
                                        ab);
  }
  if constexpr (PARAMS) {
    if constexpr (ROWS > 1) {  // the block's row groups, in order
      __shared__ float2 comb[ROWS - 1][2][EPT / 2][GT];
      const int grp = threadIdx.x / GT;
      if (grp > 0) {
#pragma unroll
        for (int i = 0; i < EPT / 2; ++i)
          comb[grp - 1][0][i][tid] = aw[i], comb[grp - 1][1][i][tid] = ab[i];
      }
      __syncthreads();
      if (grp > 0) return;
#pragma unroll
      for (int k = 0; k < ROWS - 1; ++k)
#pragma unroll
        for (int i = 0; i < EPT / 2; ++i)
          aw[i] = add2(aw[i], comb[k][0][i][tid]), ab[i] = add2(ab[i], comb[k][1][i][tid]);
    }
    ln_bwd_partials<PN, GT, V>(part, tid, D, aw, ab);
  }
}

// The same for wide rows on 16-byte boundaries: persistent blocks, 16 warps of them to an SM,
// whose x and grad_y rows arrive by bulk copies in a ring of shared memory, several rows ahead:
// the accumulators of the column sums leave no registers for that many loads in flight.  The
// sums over the next row are taken beside this row's output, one barrier a row; the row is read
// from shared memory again for it.
template <typename E, int WARPS, int V, bool PARAMS>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS)
    ln_bwd_ring_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ w,
                       const float* __restrict__ mean, const float* __restrict__ rstd,
                       const E* __restrict__ gy, int64_t gs, int64_t T, int D,
                       E* __restrict__ gx, float* __restrict__ part, int stages) {
  constexpr int PN = Pack<E>::n, GT = 32 * WARPS, EPT = V * PN;
  extern __shared__ __align__(16) char ring[];
  __shared__ __align__(8) uint64_t full[kLnMaxStages];
  __shared__ __align__(16) float red[2][2][WARPS];
  __shared__ int abort_word;
  __shared__ uint32_t filled;  // thread 0's: the parity of each stage's last fill
  const int tid = threadIdx.x;
  const uint32_t row_bytes = (uint32_t)D * sizeof(E);
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
    abort_word = 0;
    filled = ~0u;
    tc::fence_barrier_init();
  }
  __syncthreads();
  pdl_enter();
  auto fetch = [&](int64_t t, int s) {
    filled ^= 1u << s;
    char* dst = ring + (size_t)s * 2 * row_bytes;
    tc::mbar_arrive_expect_tx(&full[s], 2 * row_bytes);
    tc::bulk_load(dst, x + t * xs, row_bytes, &full[s]);
    tc::bulk_load(dst + row_bytes, gy + t * gs, row_bytes, &full[s]);
  };
  const int64_t step = gridDim.x;
  if (tid == 0) {
    int64_t t = blockIdx.x;
    for (int s = 0; s < stages && t < T; ++s, t += step) fetch(t, s);
  }
  const float inv_d = 1.f / (float)D;
  const int warp = tid >> 5, lane = tid & 31;
  float2 aw[PARAMS ? EPT / 2 : 1], ab[PARAMS ? EPT / 2 : 1], p[EPT / 2];
#pragma unroll
  for (int i = 0; i < (PARAMS ? EPT / 2 : 1); ++i) aw[i] = ab[i] = both(0.f);
  ld_params<PN, GT, V>(w, tid, D, 1.f, reinterpret_cast<float*>(p));
  auto share = [&](int s, int which, float2* f) {
    const uint4* sx = reinterpret_cast<const uint4*>(ring + (size_t)(2 * s + which) * row_bytes);
#pragma unroll
    for (int v = 0; v < V; ++v)
      widen<E>((v * GT + tid) * PN < D ? sx[v * GT + tid] : make_uint4(0, 0, 0, 0),
               reinterpret_cast<float*>(f) + v * PN);
  };
  // the row's two sums, by warp, and the column sums; past the row's end g is 0
  auto sums = [&](int s, uint32_t ph, int par, float m, float r) {
    if (!tc::mbar_wait(&full[s], ph, &abort_word)) flag_timeout();
    float2 f[EPT / 2], g[EPT / 2], s0 = both(0.f), s1 = both(0.f);
    share(s, 0, f);
    share(s, 1, g);
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      const float2 xh = mul2(add2(f[i], both(-m)), both(r));
      if constexpr (PARAMS) {
        aw[i] = fma2(g[i], xh, aw[i]);
        ab[i] = add2(ab[i], g[i]);
      }
      const float2 h = mul2(g[i], p[i]);
      s0 = add2(s0, h);
      s1 = fma2(h, xh, s1);
    }
    const float a = warp_sum(s0.x + s0.y), c = warp_sum(s1.x + s1.y);
    if (lane == 0) red[par][0][warp] = a, red[par][1][warp] = c;
  };
  float m = 0.f, r = 0.f, m1 = 0.f, r1 = 0.f;  // of this row and the next
  if (blockIdx.x < T) m = __ldg(mean + blockIdx.x), r = __ldg(rstd + blockIdx.x);
  if (blockIdx.x + step < T) m1 = __ldg(mean + blockIdx.x + step), r1 = __ldg(rstd + blockIdx.x + step);
  int s = 0, par = 0;
  uint32_t ph = 0;
  if (blockIdx.x < T) sums(0, 0, 0, m, r);
  __syncthreads();
  for (int64_t t = blockIdx.x; t < T; t += step, par ^= 1) {
    float m2 = 0.f, r2 = 0.f;
    if (t + 2 * step < T) m2 = __ldg(mean + t + 2 * step), r2 = __ldg(rstd + t + 2 * step);
    int s1 = s + 1;
    uint32_t ph1 = ph;
    if (s1 == stages) s1 = 0, ph1 ^= 1;
    if (t + step < T) sums(s1, ph1, par ^ 1, m1, r1);
    // r (h - c1 - xh c2)
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) a += red[par][0][k], c += red[par][1][k];
    const float2 c1 = both(-a * inv_d), c2 = both(-c * inv_d);
    float2 f[EPT / 2], g[EPT / 2];
    share(s, 0, f);
    share(s, 1, g);
#pragma unroll
    for (int i = 0; i < EPT / 2; ++i) {
      const float2 xh = mul2(add2(f[i], both(-m)), both(r));
      g[i] = mul2(fma2(xh, c2, fma2(g[i], p[i], c1)), both(r));
    }
    st_row<E, PN, GT, V>(gx + t * D, tid, D, reinterpret_cast<const float*>(g));
    tc::fence_proxy_async();  // the reads of this row before the refill of its stage
    __syncthreads();
    if (tid == 0 && t + step * stages < T) fetch(t + step * stages, s);
    s = s1;
    ph = ph1;
    m = m1;
    r = r1;
    m1 = m2;
    r1 = r2;
  }
  if constexpr (PARAMS) ln_bwd_partials<PN, GT, V>(part, tid, D, aw, ab);
  if (tid == 0 && *(volatile int*)&abort_word) tc::drain(full, stages, filled);
}

// Sums of the blocks' partials: 32 columns per block, 16 contiguous ranges of partials added
// side by side and then in order.
static constexpr int kLnSegs = 16;
__global__ void __launch_bounds__(32 * kLnSegs)
    ln_bwd_finish_kernel(const float* __restrict__ part, int blocks, int64_t D,
                         float* __restrict__ gw, float* __restrict__ gb) {
  pdl_enter();
  __shared__ float sum[kLnSegs][33];
  const int lane = threadIdx.x & 31, seg = threadIdx.x >> 5;
  const int64_t d = (int64_t)blockIdx.x * 32 + lane;
  KahanInf k;
  if (d < 2 * D) {
    const int i0 = blocks * seg / kLnSegs, i1 = blocks * (seg + 1) / kLnSegs;
    for (int i = i0; i < i1; i += 16) {
      float v[16];  // loads in flight together, past the range 0
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = i + j < i1 ? part[(int64_t)(i + j) * 2 * D + d] : 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) k.add(v[j]);
    }
  }
  sum[seg][lane] = k.value();
  __syncthreads();
  if (seg == 0 && d < 2 * D) {
    KahanInf t;
#pragma unroll
    for (int i = 0; i < kLnSegs; ++i) t.add(sum[i][lane]);
    (d < D ? gw : gb - D)[d] = t.value();
  }
}

// ------------------------------------------------------------------ any width
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kLnThreads / 32; ++i) s += red[i];
  __syncthreads();
  return s;
}

template <typename E>
__global__ void __launch_bounds__(kLnThreads)
    ln_fwd_loop_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ w,
                       const float* __restrict__ b, int64_t T, int64_t D, float eps,
                       E* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  pdl_enter();
  __shared__ float red[kLnThreads / 32];
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const E* xr = x + t * xs;
    float s = 0.f;
    for (int64_t d = threadIdx.x; d < D; d += kLnThreads) s += ld1<E>(xr + d);
    const float m = block_sum(s, red) / (float)D;
    s = 0.f;
    for (int64_t d = threadIdx.x; d < D; d += kLnThreads) {
      const float c = ld1<E>(xr + d) - m;
      s = fmaf(c, c, s);
    }
    const float r = rsqrtf(block_sum(s, red) / (float)D + eps);
    for (int64_t d = threadIdx.x; d < D; d += kLnThreads) {
      const float v = (ld1<E>(xr + d) - m) * r;
      st1<E>(y + t * D + d, fmaf(v, w ? w[d] : 1.f, b ? b[d] : 0.f));
    }
    if (threadIdx.x == 0) {
      if (mean) mean[t] = m;
      if (rstd) rstd[t] = r;
    }
  }
}

template <typename E>
__global__ void __launch_bounds__(kLnThreads)
    ln_bwd_rows_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ w,
                       const float* __restrict__ mean, const float* __restrict__ rstd,
                       const E* __restrict__ gy, int64_t gs, int64_t T, int64_t D,
                       E* __restrict__ gx) {
  pdl_enter();
  __shared__ float red[kLnThreads / 32];
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const E *xr = x + t * xs, *gr = gy + t * gs;
    const float m = mean[t], r = rstd[t];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t d = threadIdx.x; d < D; d += kLnThreads) {
      const float h = ld1<E>(gr + d) * (w ? w[d] : 1.f);
      s1 += h;
      s2 = fmaf(h, (ld1<E>(xr + d) - m) * r, s2);
    }
    s1 = block_sum(s1, red) / (float)D;
    s2 = block_sum(s2, red) / (float)D;
    for (int64_t d = threadIdx.x; d < D; d += kLnThreads) {
      const float h = ld1<E>(gr + d) * (w ? w[d] : 1.f);
      st1<E>(gx + t * D + d, r * (h - s1 - (ld1<E>(xr + d) - m) * r * s2));
    }
  }
}

// one thread a column and range of rows; partials [ranges][2][D]
template <typename E>
__global__ void __launch_bounds__(kLnThreads)
    ln_bwd_cols_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ mean,
                       const float* __restrict__ rstd, const E* __restrict__ gy, int64_t gs,
                       int64_t T, int64_t D, float* __restrict__ part) {
  pdl_enter();
  const int64_t d = (int64_t)blockIdx.x * kLnThreads + threadIdx.x;
  if (d >= D) return;
  const int64_t t0 = T * blockIdx.y / gridDim.y, t1 = T * (blockIdx.y + 1) / gridDim.y;
  float sw = 0.f, sb = 0.f;
  for (int64_t t = t0; t < t1; ++t) {
    const float g = ld1<E>(gy + t * gs + d);
    sb += g;
    sw = fmaf(g, (ld1<E>(x + t * xs + d) - mean[t]) * rstd[t], sw);
  }
  part[(int64_t)blockIdx.y * 2 * D + d] = sw;
  part[(int64_t)blockIdx.y * 2 * D + D + d] = sb;
}

// ------------------------------------------------------------------ launches
static constexpr int64_t kLnMaxD = 16384;
// warps to a row, for `ept` elements to a thread
static int ln_warps(int64_t D, int ept) {
  int w = 1;
  while ((int64_t)w * 32 * ept < D) w *= w == 1 ? 4 : 2;
  return w;
}
// The ring kernels: rows of 16-byte packs, 513 to 8192 elements; `warps` to a row and ept
// elements to a thread (the forward's threads take twice as many: measured at D=7168, bf16,
// T=32768, 152 us against 214; the backward, whose column sums are registers too, 284 us with 16
// and 349 with 32).  16 warps to an SM, whose rings share 200 KB.
struct RingPlan {
  int warps, ept;
};
static bool ln_ring(int64_t D, int elem) {
  return D > 512 && D <= 8192 && (D * elem) % 16 == 0;
}
static RingPlan ln_fwd_plan(int64_t D) {
  return D <= 1024 ? RingPlan{2, 16} : D <= 2048 ? RingPlan{2, 32} : D <= 4096 ? RingPlan{4, 32}
                                                                               : RingPlan{8, 32};
}
static int ln_bwd_warps(int64_t D) { return D <= 1024 ? 2 : D <= 2048 ? 4 : D <= 4096 ? 8 : 16; }
static int ln_ring_stages(int warps, int64_t stage_bytes) {
  const int64_t fit = (200 << 10) / (stage_bytes * (16 / warps));
  return (int)std::max<int64_t>(2, std::min<int64_t>(fit, kLnMaxStages));
}
// Row blocks of the backward, each with a partial: as many as run at once, but no more than
// leave each group of warps a few rows, since the partials are written and read again (two, four
// and sqrt(T / 32) = 7 rows: T=1999, D=1001: 13.0, 10.7, 10.5 us; T=500, D=4096: 17.8 with two,
// 13.7 with four; T=64, D=4096: 10.7, 12.3).
static int ln_bwd_blocks(int64_t T, int64_t D) {
  if (D > kLnMaxD) return (int)(T < 64 * 64 ? cdiv(T, 64) : 64);
  const int warps = D > 512 && D <= 8192 ? ln_bwd_warps(D) : ln_warps(D, 16);
  const int rows = warps == 1 ? 4 : 1;
  const int64_t fit = (int64_t)sm_count() * (warps == 1 ? 5 : warps >= 16 ? 1 : 16 / warps);
  const int64_t per = std::max<int64_t>(T < 128 || rows > 1 ? 2 : 4,
                                        (int64_t)sqrt((double)T / 32.0) / rows);
  return (int)std::max<int64_t>(std::min<int64_t>(cdiv(T, per * rows), fit), T > 0 ? 1 : 0);
}

// V of the direct kernels is for 16 elements to a thread, 8 in rows of up to 256
#define LN_WARPS(W_, CALL)                                  \
  switch (W_) {                                             \
    case 1:                                                 \
      if (D <= 256) {                                       \
        CALL(1, 8 / PN);                                    \
      } else {                                              \
        CALL(1, 16 / PN);                                   \
      }                                                     \
      break;                                                \
    case 4: CALL(4, 16 / PN); break;                        \
    case 8: CALL(8, 16 / PN); break;                        \
    case 16: CALL(16, 16 / PN); break;                      \
    default: CALL(32, 16 / PN); break;                      \
  }

template <typename E, int PN>
static int ln_fwd_rows(const E* x, int64_t xs, const float* w, const float* b, int64_t T, int D,
                       float eps, E* y, float* mean, float* rstd, cudaStream_t s) {
  const int warps = ln_warps(D, 16), rows = warps == 1 ? 4 : 1;
  // narrow rows: blocks that stay, eight to an SM (65536 rows of 256 bf16: 35 us with a block
  // to four rows)
  const unsigned grid = (unsigned)std::min<int64_t>(
      cdiv(T, rows), warps == 1 ? (int64_t)sm_count() * 8 : 1 << 20);
#define LN_FWD(W, V)                                                                           \
  launch(ln_fwd_kernel<E, PN, W, V>, grid, W == 1 ? 128 : 32 * W, 0, s, x, xs, w, b, T, D, eps, \
         y, mean, rstd)
  LN_WARPS(warps, LN_FWD)
#undef LN_FWD
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

template <typename E, int WARPS, int EPT>
static int ln_fwd_ring_launch(const E* x, int64_t xs, const float* w, const float* b, int64_t T,
                              int D, float eps, E* y, float* mean, float* rstd, cudaStream_t s) {
  constexpr int V = EPT / Pack<E>::n;
  static bool attr_set[64];
  int dev = 0;
  MHC_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    MHC_CUDA_CHECK(cudaFuncSetAttribute((const void*)ln_fwd_ring_kernel<E, WARPS, V>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, 200 << 10));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int stages = ln_ring_stages(WARPS, D * sizeof(E));
  const int grid = (int)std::min<int64_t>(T, (int64_t)sm_count() * (16 / WARPS));
  launch(ln_fwd_ring_kernel<E, WARPS, V>, grid, 32 * WARPS, (size_t)stages * D * sizeof(E), s, x,
         xs, w, b, T, D, eps, y, mean, rstd, stages);
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

template <typename E>
static int ln_fwd_run(const void* x, int64_t xs, const float* w, const float* b, int64_t T,
                      int64_t D, float eps, void* y, float* mean, float* rstd, cudaStream_t s) {
  constexpr int PN = Pack<E>::n;
  if (D > kLnMaxD) {
    launch(ln_fwd_loop_kernel<E>, (unsigned)std::min<int64_t>(T, 65535), kLnThreads, 0, s,
           (const E*)x, xs, w, b, T, D, eps, (E*)y, mean, rstd);
    MHC_LAUNCH_CHECK();
    return MHC_OK;
  }
  const bool vec = aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b) && xs % PN == 0 &&
                   D % PN == 0;
  if (vec && ln_ring(D, sizeof(E))) {
    const RingPlan p = ln_fwd_plan(D);
    auto run = p.ept == 16   ? ln_fwd_ring_launch<E, 2, 16>
               : p.warps == 2 ? ln_fwd_ring_launch<E, 2, 32>
               : p.warps == 4 ? ln_fwd_ring_launch<E, 4, 32>
                              : ln_fwd_ring_launch<E, 8, 32>;
    return run((const E*)x, xs, w, b, T, (int)D, eps, (E*)y, mean, rstd, s);
  }
  if (vec)
    return ln_fwd_rows<E, PN>((const E*)x, xs, w, b, T, (int)D, eps, (E*)y, mean, rstd, s);
  return ln_fwd_rows<E, 1>((const E*)x, xs, w, b, T, (int)D, eps, (E*)y, mean, rstd, s);
}

template <typename E, int PN>
static int ln_bwd_rows(const E* x, int64_t xs, const float* w, const float* mean,
                       const float* rstd, const E* gy, int64_t gs, int64_t T, int D, E* gx,
                       float* part, int blocks, cudaStream_t s) {
  const int warps = ln_warps(D, 16);
#define LN_BWD(W, V)                                                                              \
  if (part)                                                                                    \
    launch(ln_bwd_kernel<E, PN, W, V, true>, blocks, W == 1 ? 128 : 32 * W, 0, s, x, xs, w,    \
           mean, rstd, gy, gs, T, D, gx, part);                                                \
  else                                                                                         \
    launch(ln_bwd_kernel<E, PN, W, V, false>, blocks, W == 1 ? 128 : 32 * W, 0, s, x, xs, w,   \
           mean, rstd, gy, gs, T, D, gx, part)
  LN_WARPS(warps, LN_BWD)
#undef LN_BWD
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

template <typename E, int WARPS, bool PARAMS>
static int ln_bwd_ring_launch(const E* x, int64_t xs, const float* w, const float* mean,
                              const float* rstd, const E* gy, int64_t gs, int64_t T, int D, E* gx,
                              float* part, int blocks, cudaStream_t s) {
  constexpr int V = 16 / Pack<E>::n;
  static bool attr_set[64];
  int dev = 0;
  MHC_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    MHC_CUDA_CHECK(cudaFuncSetAttribute((const void*)ln_bwd_ring_kernel<E, WARPS, V, PARAMS>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, 200 << 10));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int stages = ln_ring_stages(WARPS, 2 * D * sizeof(E));
  launch(ln_bwd_ring_kernel<E, WARPS, V, PARAMS>, blocks, 32 * WARPS,
         (size_t)stages * 2 * D * sizeof(E), s, x, xs, w, mean, rstd, gy, gs, T, D, gx, part,
         stages);
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}
template <typename E>
static int ln_bwd_ring(const E* x, int64_t xs, const float* w, const float* mean,
                       const float* rstd, const E* gy, int64_t gs, int64_t T, int D, E* gx,
                       float* part, int blocks, cudaStream_t s) {
  const int warps = ln_bwd_warps(D);
#define LN_RING(W) (part ? ln_bwd_ring_launch<E, W, true> : ln_bwd_ring_launch<E, W, false>)
  auto run = warps == 2 ? LN_RING(2) : warps == 4 ? LN_RING(4) : warps == 8 ? LN_RING(8) : LN_RING(16);
#undef LN_RING
  return run(x, xs, w, mean, rstd, gy, gs, T, D, gx, part, blocks, s);
}

template <typename E>
static int ln_bwd_run(const void* x, int64_t xs, const float* w, const float* mean,
                      const float* rstd, const void* gy, int64_t gs, int64_t T, int64_t D,
                      void* gx, float* gw, float* gb, float* part, cudaStream_t s) {
  constexpr int PN = Pack<E>::n;
  const int blocks = ln_bwd_blocks(T, D);
  float* pt = gw ? part : nullptr;
  if (T > 0 && D > kLnMaxD) {
    launch(ln_bwd_rows_kernel<E>, (unsigned)std::min<int64_t>(T, 65535), kLnThreads, 0, s,
           (const E*)x, xs, w, mean, rstd, (const E*)gy, gs, T, D, (E*)gx);
    MHC_LAUNCH_CHECK();
    if (gw) {
      launch(ln_bwd_cols_kernel<E>, dim3((unsigned)cdiv(D, kLnThreads), blocks), kLnThreads, 0, s,
             (const E*)x, xs, mean, rstd, (const E*)gy, gs, T, D, part);
      MHC_LAUNCH_CHECK();
    }
  } else if (T > 0) {
    const bool vec = aligned16(x) && aligned16(gy) && aligned16(gx) && aligned16(w) && xs % PN == 0 &&
                     gs % PN == 0 && D % PN == 0;
    const int st = vec && ln_ring(D, sizeof(E))
                       ? ln_bwd_ring<E>((const E*)x, xs, w, mean, rstd, (const E*)gy, gs, T, (int)D,
                                        (E*)gx, pt, blocks, s)
                   : vec ? ln_bwd_rows<E, PN>((const E*)x, xs, w, mean, rstd, (const E*)gy, gs, T,
                                            (int)D, (E*)gx, pt, blocks, s)
                       : ln_bwd_rows<E, 1>((const E*)x, xs, w, mean, rstd, (const E*)gy, gs, T,
                                           (int)D, (E*)gx, pt, blocks, s);
    if (st != MHC_OK) return st;
  }
  if (gw) {
    launch(ln_bwd_finish_kernel, (unsigned)cdiv(2 * D, 32), 32 * kLnSegs, 0, s, (const float*)part, blocks,
           D, gw, gb);
    MHC_LAUNCH_CHECK();
  }
  return MHC_OK;
}

int layer_norm_device_error() { return read_and_clear_tu_error(); }

static bool ln_sizes_ok(int64_t T, int64_t D) {
  return T >= 0 && D > 0 && D <= INT32_MAX / 4;
}

}  // namespace mhc

using namespace mhc;

extern "C" {

int mhc_layer_norm_fwd(const void* x, int64_t x_stride, const float* weight, const float* bias,
                       int64_t T, int64_t D, int32_t dtype, float eps, void* y, float* mean,
                       float* rstd, void* stream) {
  if (!ln_sizes_ok(T, D) || x_stride < D || !(eps >= 0.f)) return MHC_ERR_INVALID_ARGUMENT;
  if (dtype != MHC_F32 && dtype != MHC_F16 && dtype != MHC_BF16) return MHC_ERR_UNSUPPORTED_DTYPE;
  if (T == 0) return MHC_OK;
  if (!x || !y) return MHC_ERR_INVALID_ARGUMENT;
  const int st = check_device();
  if (st != MHC_OK) return st;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == MHC_F32)
    return ln_fwd_run<float>(x, x_stride, weight, bias, T, D, eps, y, mean, rstd, s);
  if (dtype == MHC_F16)
    return ln_fwd_run<__half>(x, x_stride, weight, bias, T, D, eps, y, mean, rstd, s);
  return ln_fwd_run<__nv_bfloat16>(x, x_stride, weight, bias, T, D, eps, y, mean, rstd, s);
}

size_t mhc_layer_norm_bwd_workspace_bytes(int64_t T, int64_t D, int32_t dtype) {
  if (!ln_sizes_ok(T, D) || (dtype != MHC_F32 && dtype != MHC_F16 && dtype != MHC_BF16)) return 0;
  return align_up((size_t)ln_bwd_blocks(T, D) * 2 * D * 4);
}

int mhc_layer_norm_bwd(const void* x, int64_t x_stride, const float* weight, const float* mean,
                       const float* rstd, const void* grad_y, int64_t grad_y_stride, int64_t T,
                       int64_t D, int32_t dtype, void* grad_x, float* grad_weight,
                       float* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  if (!ln_sizes_ok(T, D) || x_stride < D || grad_y_stride < D) return MHC_ERR_INVALID_ARGUMENT;
  if (dtype != MHC_F32 && dtype != MHC_F16 && dtype != MHC_BF16) return MHC_ERR_UNSUPPORTED_DTYPE;
  if ((grad_weight == nullptr) != (grad_bias == nullptr)) return MHC_ERR_INVALID_ARGUMENT;
  if (T > 0 && (!x || !mean || !rstd || !grad_y || !grad_x)) return MHC_ERR_INVALID_ARGUMENT;
  if (T == 0 && !grad_weight) return MHC_OK;
  const size_t need = mhc_layer_norm_bwd_workspace_bytes(T, D, dtype);
  if (grad_weight && need > 0 &&
      (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return MHC_ERR_WORKSPACE;
  const int st = check_device();
  if (st != MHC_OK) return st;
  const cudaStream_t s = (cudaStream_t)stream;
  float* part = (float*)workspace;
  if (dtype == MHC_F32)
    return ln_bwd_run<float>(x, x_stride, weight, mean, rstd, grad_y, grad_y_stride, T, D, grad_x,
                             grad_weight, grad_bias, part, s);
  if (dtype == MHC_F16)
    return ln_bwd_run<__half>(x, x_stride, weight, mean, rstd, grad_y, grad_y_stride, T, D,
                              grad_x, grad_weight, grad_bias, part, s);
  return ln_bwd_run<__nv_bfloat16>(x, x_stride, weight, mean, rstd, grad_y, grad_y_stride, T, D,
                                   grad_x, grad_weight, grad_bias, part, s);
}

}  // extern "C"
