// layer_norm.cu -- layer norm over the last dimension, forward and backward.
#include "common.cuh"

namespace mhc {

static constexpr int kLnThreads = 256;

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
    ln_fwd_kernel(const E* __restrict__ x, int64_t xs, const float* __restrict__ w,
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

__global__ void __launch_bounds__(kLnThreads)
    ln_bwd_finish_kernel(const float* __restrict__ part, int ranges, int64_t D,
                         float* __restrict__ gw, float* __restrict__ gb) {
  pdl_enter();
  const int64_t d = (int64_t)blockIdx.x * kLnThreads + threadIdx.x;
  if (d >= 2 * D) return;
  Kahan k;
  for (int i = 0; i < ranges; ++i) k.add(part[(int64_t)i * 2 * D + d]);
  (d < D ? gw : gb - D)[d] = k.s;
}

static int ln_ranges(int64_t T) { return (int)(T < 64 * 64 ? cdiv(T, 64) : 64); }

template <typename E>
static int ln_fwd_run(const void* x, int64_t xs, const float* w, const float* b, int64_t T,
                      int64_t D, float eps, void* y, float* mean, float* rstd, cudaStream_t s) {
  const int grid = (int)(T < 65535 ? T : 65535);
  launch(ln_fwd_kernel<E>, grid, kLnThreads, 0, s, (const E*)x, xs, w, b, T, D, eps, (E*)y, mean,
         rstd);
  MHC_LAUNCH_CHECK();
  return MHC_OK;
}

template <typename E>
static int ln_bwd_run(const void* x, int64_t xs, const float* w, const float* mean,
                      const float* rstd, const void* gy, int64_t gs, int64_t T, int64_t D,
                      void* gx, float* gw, float* gb, float* part, cudaStream_t s) {
  if (T > 0) {
    const int grid = (int)(T < 65535 ? T : 65535);
    launch(ln_bwd_rows_kernel<E>, grid, kLnThreads, 0, s, (const E*)x, xs, w, mean, rstd,
           (const E*)gy, gs, T, D, (E*)gx);
    MHC_LAUNCH_CHECK();
  }
  if (gw) {
    const int ranges = ln_ranges(T);
    if (ranges > 0) {
      launch(ln_bwd_cols_kernel<E>, dim3((unsigned)cdiv(D, kLnThreads), ranges), kLnThreads, 0, s,
             (const E*)x, xs, mean, rstd, (const E*)gy, gs, T, D, part);
      MHC_LAUNCH_CHECK();
    }
    launch(ln_bwd_finish_kernel, (unsigned)cdiv(2 * D, kLnThreads), kLnThreads, 0, s,
           (const float*)part, ranges, D, gw, gb);
    MHC_LAUNCH_CHECK();
  }
  return MHC_OK;
}

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
  return align_up((size_t)ln_ranges(T) * 2 * D * 4);
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
