// sublayer.cu -- entry points of the linear layer and the gated feed-forward block: argument
// checks, workspace layout and the sequence of matrix products (gemm.cuh).
#include <algorithm>
#include <initializer_list>

#include "gemm.cuh"

namespace mhc {

// ------------------------------------------------------------------ gz and grad_bias
// gz = grad_y * act'(z), rounded to dtype as the operand of both products that follow, and, per row
// range, the column sums of the unrounded gz: bound by HBM.  A block takes 256 columns of a row
// range, 8 to a thread (a 16-byte pack where the rows allow it), its warps every eighth row; their
// sums are added in order.
// About 4096 blocks, of at least 32 rows (65536 x 4096, silu: 271 us with 256 ranges, 306 us with
// 64; two or four rows of a warp at once took 380 and 473 us).
static int gz_ranges(int64_t T, int64_t F) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(256, 4096 / cdiv(F, 256)));
  return (int)std::min<int64_t>(cdiv(T, 32), most);
}

template <typename E, int ACT, bool VEC>
__global__ void __launch_bounds__(256)
    act_bwd_kernel(const E* __restrict__ z, int64_t zs, const E* __restrict__ gy, int64_t gs,
                   int64_t T, int64_t F, E* __restrict__ gz, int64_t ld, float* __restrict__ part) {
  pdl_enter();
  __shared__ float red[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = (int64_t)blockIdx.x * 256;
  const int64_t t0 = T * blockIdx.y / gridDim.y, t1 = T * (blockIdx.y + 1) / gridDim.y;
  // element e of this thread is column c0 + 8 lane + e, or c0 + lane + 32 e
  const int64_t c = c0 + (VEC ? 8 * lane : lane);
  constexpr int STEP = VEC ? 1 : 32;
  float s[8] = {};
  const int64_t tn = VEC && c >= F ? t0 : t1;  // F is a multiple of 8 with VEC
  for (int64_t t = t0 + warp; t < tn; t += 8) {
    float v[8], zv[8];
    if constexpr (VEC) {
      widen<E>(ld_stream(gy + t * gs + c), v);
      if constexpr (ACT != MHC_ACT_NONE) widen<E>(ld_stream(z + t * zs + c), zv);
    } else {
      E a[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t k = min(c + 32 * e, F - 1);
        a[e] = gy[t * gs + k];
        if constexpr (ACT != MHC_ACT_NONE) b[e] = z[t * zs + k];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = c + 32 * e < F ? from_e(a[e]) : 0.f;
        if constexpr (ACT != MHC_ACT_NONE) zv[e] = from_e(b[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (ACT != MHC_ACT_NONE) {
        float av, da;
        act_both<ACT>(zv[e], av, da);
        v[e] *= da;
      }
      if (VEC || c + 32 * e < F) s[e] += v[e];
    }
    if (gz) {
      if constexpr (VEC) {
        *reinterpret_cast<uint4*>(gz + t * ld + c) = narrow<E>(v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + 32 * e < F) gz[t * ld + c + 32 * e] = to_e<E>(v[e]);
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[warp][(VEC ? 8 * lane : lane) + STEP * e] = s[e];
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += red[k][threadIdx.x];
  if (c0 + threadIdx.x < F) part[(int64_t)blockIdx.y * F + c0 + threadIdx.x] = sum;
}

// 32 columns per block; eight contiguous ranges of partials side by side, then in order
template <typename E>
__global__ void __launch_bounds__(256)
    bias_finish_kernel(const float* __restrict__ part, int ranges, int64_t F, E* __restrict__ gb) {
  pdl_enter();
  __shared__ float sum[8][33];
  const int lane = threadIdx.x & 31, seg = threadIdx.x >> 5;
  const int64_t f = (int64_t)blockIdx.x * 32 + lane;
  KahanInf k;
  if (f < F) {
    const int i0 = ranges * seg / 8, i1 = ranges * (seg + 1) / 8;
    for (int i = i0; i < i1; i += 8) {
      float v[8];  // loads in flight together, past the range 0
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + j < i1 ? part[(int64_t)(i + j) * F + f] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) k.add(v[j]);
    }
  }
  sum[seg][lane] = k.value();
  __syncthreads();
  if (seg == 0 && f < F) {
    KahanInf t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t.add(sum[i][lane]);
    st1<E>(gb + f, t.value());
  }
}

template <typename E>
static int act_bwd_run(int act, const void* z, int64_t zs, const void* gy, int64_t gs, int64_t T,
                       int64_t F, void* gz, int64_t ld, void* gb, float* part, cudaStream_t s) {
  const int ranges = gz_ranges(T, F);
  const dim3 grid((unsigned)cdiv(F, 256), ranges);
  float* pt = gb ? part : nullptr;
  const bool vec = aligned16(z) && zs % 8 == 0 && aligned16(gy) && gs % 8 == 0 && F % 8 == 0;
#define MHC_GZ(A)                                                                               \
  (launch(vec ? act_bwd_kernel<E, A, true> : act_bwd_kernel<E, A, false>, grid, 256, 0, s,      \
          (const E*)z, zs, (const E*)gy, gs, T, F, (E*)gz, ld, pt),                             \
   MHC_OK)
  auto run = [&]() -> int { MHC_DISPATCH_ACT(act, MHC_GZ) };
#undef MHC_GZ
  const int st = run();
  if (st != MHC_OK) return st;
  MHC_LAUNCH_CHECK();
  if (gb) {
    launch(bias_finish_kernel<E>, (unsigned)cdiv(F, 32), 256, 0, s, (const float*)part, ranges, F,
           (E*)gb);
    MHC_LAUNCH_CHECK();
  }
  return MHC_OK;
}

// ------------------------------------------------------------------ checks and workspace
static int64_t pad16(int64_t n) { return (n + 15) / 16 * 16; }  // rows on 32-byte boundaries

static int sub_check(int64_t T, int64_t D, int64_t F, int32_t dtype, int32_t act) {
  // tile coordinates are 32-bit
  if (T < 0 || D <= 0 || F <= 0 || T > INT32_MAX - 512 || D > INT32_MAX / 8 || F > INT32_MAX / 8)
    return MHC_ERR_INVALID_ARGUMENT;
  if (dtype != MHC_F16 && dtype != MHC_BF16) return MHC_ERR_UNSUPPORTED_DTYPE;
  if (act < MHC_ACT_NONE || act > MHC_ACT_SILU) return MHC_ERR_INVALID_ARGUMENT;
  return MHC_OK;
}

static bool ws_ok(const void* ws, size_t bytes, size_t need) {
  return need == 0 || (ws && bytes >= need && (reinterpret_cast<uintptr_t>(ws) & 255) == 0);
}

// Takes regions of the workspace in order; with a null base only the offsets are counted.
struct Carver {
  char* base;
  size_t off = 0;
  void* take(size_t bytes) {
    void* p = base ? base + off : nullptr;
    off += align_up(bytes);
    return p;
  }
};

// An operand as the matrix product takes it: itself, or a packed copy in the workspace.
static size_t packed_bytes(int64_t rows, int64_t cols) {
  return (size_t)rows * pad16(cols) * 2;
}
static int aligned_operand(Operand* o, int64_t rows, int64_t cols, Carver* c, cudaStream_t s) {
  if (operand_aligned(*o)) return MHC_OK;
  void* dst = c->take(packed_bytes(rows, cols));
  const int st = pack_rows(o->p, o->ld, rows, cols, dst, pad16(cols), s);
  o->p = dst;
  o->ld = pad16(cols);
  return st;
}
// Room for the partial products of the largest of these products (they run one by one).
// a_k: whether a (and a3) is K-major, which the plan goes by too.
static Gemm product(int kind, bool a_k, int64_t M, int64_t N, int64_t K, int64_t K3 = 0) {
  Gemm g;
  g.a.k_major = g.a3.k_major = a_k;
  g.kind = kind;
  g.M = M; g.N = N; g.K = K; g.K3 = K3;
  return g;
}
static size_t gemm_room(std::initializer_list<Gemm> gs) {
  size_t n = 0;
  for (const Gemm& g : gs) n = std::max(n, gemm_ws_bytes(g));
  return n;
}
// dtype with the flag on the kept gate and up taken off
static bool take_gate_up_f32(int32_t* dtype) {
  const bool f32 = (*dtype & MHC_GATE_UP_F32) != 0;
  *dtype &= ~MHC_GATE_UP_F32;
  return f32;
}
// The matrix products of the operators, as enum mhc_product names them.
static Gemm product_of(int32_t which, int64_t T, int64_t D, int64_t F) {
  switch (which) {
    case MHC_PRODUCT_GATE_UP: return product(kEpiGated, true, T, F, D);
    case MHC_PRODUCT_GATED_GRAD_HIDDEN: return product(kEpiGatedBwd, true, T, F, D);
    case MHC_PRODUCT_GATED_GRAD_X: return product(kEpiLinear, true, T, D, F, F);
    case MHC_PRODUCT_GRAD_X: return product(kEpiLinear, true, T, D, F);
    case MHC_PRODUCT_GRAD_WEIGHT: return product(kEpiLinear, false, F, D, T);
    default: return product(kEpiLinear, true, T, F, D);
  }
}
static size_t linear_fwd_room(int64_t T, int64_t D, int64_t F) {
  return T == 0 || gemv_takes(T, F, D) ? 0 : gemm_room({product_of(MHC_PRODUCT_LINEAR, T, D, F)});
}
static size_t linear_bwd_room(int64_t T, int64_t D, int64_t F) {
  return T == 0 ? 0 : gemm_room({product_of(MHC_PRODUCT_GRAD_X, T, D, F),
                                 product_of(MHC_PRODUCT_GRAD_WEIGHT, T, D, F)});
}
static size_t ffn_fwd_room(int64_t T, int64_t D, int64_t F) {
  return T == 0 || gemv_takes(T, F, D) ? 0 : gemm_room({product_of(MHC_PRODUCT_GATE_UP, T, D, F),
                                                        product_of(MHC_PRODUCT_LINEAR, T, F, D)});
}
static size_t ffn_bwd_room(int64_t T, int64_t D, int64_t F) {
  return T == 0 ? 0 : gemm_room({product_of(MHC_PRODUCT_GATED_GRAD_HIDDEN, T, D, F),
                                 product_of(MHC_PRODUCT_GATED_GRAD_X, T, D, F),
                                 product_of(MHC_PRODUCT_GRAD_WEIGHT, T, D, F),
                                 product_of(MHC_PRODUCT_GRAD_WEIGHT, T, F, D)});
}

// Runs a product whose output's rows may be unaligned: then it goes to a packed copy first, for
// the epilogue's row-wise stores (2 bytes to a row at a time: 2503 x 1001 outputs took 50 us, 27
// us by the copy).  The copy's room is taken from the Carver and free again afterwards.
static int run_product(Gemm* g, void* room, Carver c, cudaStream_t s) {
  EpiParams& e = g->epi;
  if (gemm_plan(*g).mt == 0 || operand_aligned({e.out, e.ld_out, true})) return gemm_run(*g, room, s);
  void *out = e.out, *z = e.z;
  const int64_t ld = e.ld_out;
  e.out = c.take(packed_bytes(g->M, g->N));
  if (z) e.z = c.take(packed_bytes(g->M, g->N));
  e.ld_out = pad16(g->N);
  int st = gemm_run(*g, room, s);
  if (st == MHC_OK) st = pack_rows(e.out, e.ld_out, g->M, g->N, out, ld, s);
  if (st == MHC_OK && z) st = pack_rows(e.z, e.ld_out, g->M, g->N, z, ld, s);
  e.out = out; e.z = z; e.ld_out = ld;
  return st;
}

// Matrices that the call does not have (null) do not count, whatever their stride.
static bool any_unaligned(std::initializer_list<Operand> ops) {
  for (const Operand& o : ops)
    if (o.p && !operand_aligned(o)) return true;
  return false;
}

static int zero(void* p, size_t bytes, cudaStream_t s) {
  if (p && bytes) MHC_CUDA_CHECK(cudaMemsetAsync(p, 0, bytes, s));
  return MHC_OK;
}

}  // namespace mhc

using namespace mhc;

#define RETURN_IF(x)               \
  do {                             \
    int _st = (x);                 \
    if (_st != MHC_OK) return _st; \
  } while (0)

extern "C" {

int mhc_sublayer_plan(int32_t which, int64_t T, int64_t D, int64_t F, int32_t* form, int32_t* tile,
                      int32_t* cuts) {
  if (sub_check(T, D, F, MHC_BF16, MHC_ACT_NONE) != MHC_OK || T == 0 || which < MHC_PRODUCT_LINEAR ||
      which > MHC_PRODUCT_GATED_GRAD_X || !form || !tile || !cuts)
    return MHC_ERR_INVALID_ARGUMENT;
  if ((which == MHC_PRODUCT_LINEAR || which == MHC_PRODUCT_GATE_UP) && gemv_takes(T, F, D)) {
    *form = MHC_FORM_STREAM;
    *tile = T <= 8 ? 8 : 16;
    *cuts = 1;
    return MHC_OK;
  }
  const GemmPlan p = gemm_plan(product_of(which, T, D, F));
  *form = p.mt == 0 ? MHC_FORM_CLUSTER : MHC_FORM_PAIR;
  *tile = p.mt == 0 ? p.nt : 256 * p.mt;
  *cuts = p.splits;
  return MHC_OK;
}

size_t mhc_linear_fwd_workspace_bytes(int64_t T, int64_t D, int64_t F, int32_t dtype,
                                      int32_t unaligned) {
  if (sub_check(T, D, F, dtype, 0) != MHC_OK) return 0;
  Carver c{nullptr};
  c.take(linear_fwd_room(T, D, F));
  if (unaligned && !gemv_takes(T, F, D)) {
    c.take(packed_bytes(T, D));  // x
    c.take(packed_bytes(F, D));  // weight
    for (int i = 0; i < 3; ++i) c.take(packed_bytes(T, F));  // residual, y, z
  }
  return c.off;
}

int mhc_linear_fwd(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                   const void* bias, const void* residual, int64_t residual_stride, int64_t T,
                   int64_t D, int64_t F, int32_t dtype, int32_t act, void* y, void* z,
                   void* workspace, size_t workspace_bytes, void* stream) {
  RETURN_IF(sub_check(T, D, F, dtype, act));
  if (x_stride < D || weight_stride < D || (residual && residual_stride < F))
    return MHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return MHC_OK;
  if (!x || !weight || !y) return MHC_ERR_INVALID_ARGUMENT;
  Gemm g;
  g.dtype = dtype;
  g.M = T; g.N = F; g.K = D;
  g.a = {x, x_stride, true};
  g.b = {weight, weight_stride, true};
  if (!ws_ok(workspace, workspace_bytes,
             mhc_linear_fwd_workspace_bytes(
                 T, D, F, dtype,
                 any_unaligned({g.a, g.b, {y, F, true}, {residual, residual_stride, true}}))))
    return MHC_ERR_WORKSPACE;
  RETURN_IF(check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  Carver c{(char*)workspace};
  void* room = c.take(linear_fwd_room(T, D, F));
  g.epi.act = act; g.epi.out = y; g.epi.ld_out = F; g.epi.bias = bias; g.epi.z = z;
  g.epi.res = residual; g.epi.ld_res = residual ? residual_stride : 0;
  if (gemv_takes(T, F, D)) return gemv_run(g, s);
  RETURN_IF(aligned_operand(&g.a, T, D, &c, s));
  RETURN_IF(aligned_operand(&g.b, F, D, &c, s));
  if (residual) {
    Operand r{residual, residual_stride, true};
    RETURN_IF(aligned_operand(&r, T, F, &c, s));
    g.epi.res = r.p; g.epi.ld_res = r.ld;
  }
  return run_product(&g, room, c, s);
}

size_t mhc_linear_bwd_workspace_bytes(int64_t T, int64_t D, int64_t F, int32_t dtype,
                                      int32_t act, int32_t unaligned) {
  if (sub_check(T, D, F, dtype, act) != MHC_OK) return 0;
  Carver c{nullptr};
  if (act != MHC_ACT_NONE || unaligned) c.take(packed_bytes(T, F));  // gz
  c.take((size_t)gz_ranges(T, F) * F * 4);
  c.take(linear_bwd_room(T, D, F));
  if (unaligned) {
    c.take(packed_bytes(T, D));                               // x
    c.take(packed_bytes(F, D));                               // weight
    c.take(std::max(packed_bytes(T, D), packed_bytes(F, D)));  // grad_x, then grad_weight
  }
  return c.off;
}

int mhc_linear_bwd(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                   const void* z, int64_t z_stride, const void* grad_y, int64_t grad_y_stride,
                   int64_t T, int64_t D, int64_t F, int32_t dtype, int32_t act, void* grad_x,
                   void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                   void* stream) {
  RETURN_IF(sub_check(T, D, F, dtype, act));
  if (x_stride < D || weight_stride < D || grad_y_stride < F ||
      (act != MHC_ACT_NONE && z_stride < F))
    return MHC_ERR_INVALID_ARGUMENT;
  const cudaStream_t s = (cudaStream_t)stream;
  if (T > 0 && (!x || !weight || !grad_y || (act != MHC_ACT_NONE && !z)))
    return MHC_ERR_INVALID_ARGUMENT;
  if (!grad_x && !grad_weight && !grad_bias) return MHC_OK;
  Operand ox{x, x_stride, false}, ow{weight, weight_stride, false};
  const bool gy_packed = act == MHC_ACT_NONE && !operand_aligned({grad_y, grad_y_stride, false});
  if (T > 0 && !ws_ok(workspace, workspace_bytes,
                      mhc_linear_bwd_workspace_bytes(T, D, F, dtype, act,
                                                     gy_packed || any_unaligned({ox, ow, {grad_x, D, true}, {grad_weight, D, true}}))))
    return MHC_ERR_WORKSPACE;
  RETURN_IF(check_device());
  if (T == 0) {
    RETURN_IF(zero(grad_weight, (size_t)F * D * 2, s));
    return zero(grad_bias, (size_t)F * 2, s);
  }
  Carver c{(char*)workspace};
  // without an activation gz is grad_y, copied only where its rows are unaligned
  void* gzb = act != MHC_ACT_NONE || gy_packed ? c.take(packed_bytes(T, F)) : nullptr;
  float* part = (float*)c.take((size_t)gz_ranges(T, F) * F * 4);
  void* room = c.take(linear_bwd_room(T, D, F));
  if (gzb || grad_bias) {
    const int64_t ld = pad16(F);
    RETURN_IF(dtype == MHC_F16
                  ? act_bwd_run<__half>(act, z, z_stride, grad_y, grad_y_stride, T, F, gzb, ld,
                                        grad_bias, part, s)
                  : act_bwd_run<__nv_bfloat16>(act, z, z_stride, grad_y, grad_y_stride, T, F, gzb,
                                               ld, grad_bias, part, s));
  }
  const void* gz = gzb ? gzb : grad_y;
  const int64_t gzs = gzb ? pad16(F) : grad_y_stride;
  if (grad_x) RETURN_IF(aligned_operand(&ow, F, D, &c, s));
  if (grad_weight) RETURN_IF(aligned_operand(&ox, T, D, &c, s));
  Gemm g;
  g.dtype = dtype;
  if (grad_x) {
    g.M = T; g.N = D; g.K = F;
    g.a = {gz, gzs, true};
    g.b = ow;
    g.epi.out = grad_x; g.epi.ld_out = D;
    RETURN_IF(run_product(&g, room, c, s));
  }
  if (grad_weight) {
    g.M = F; g.N = D; g.K = T;
    g.a = {gz, gzs, false};
    g.b = ox;
    g.epi.out = grad_weight; g.epi.ld_out = D;
    RETURN_IF(run_product(&g, room, c, s));
  }
  return MHC_OK;
}

size_t mhc_gated_ffn_fwd_workspace_bytes(int64_t T, int64_t D, int64_t F, int32_t dtype,
                                         int32_t unaligned) {
  take_gate_up_f32(&dtype);
  if (sub_check(T, D, F, dtype, 0) != MHC_OK) return 0;
  Carver c{nullptr};
  c.take(packed_bytes(T, F));  // h
  c.take(ffn_fwd_room(T, D, F));
  if (unaligned && !gemv_takes(T, F, D)) {
    c.take(packed_bytes(T, D));                              // x
    for (int i = 0; i < 2; ++i) c.take(packed_bytes(F, D));  // w_gate, w_up
    c.take(packed_bytes(D, F));                              // w_down
    c.take(packed_bytes(T, D));                              // y
  }
  return c.off;
}

int mhc_gated_ffn_fwd(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride,
                      const void* w_up, int64_t w_up_stride, const void* w_down,
                      int64_t w_down_stride, int64_t T, int64_t D, int64_t F, int32_t dtype,
                      int32_t act, void* y, void* gate, void* up, int64_t gate_up_stride,
                      void* workspace, size_t workspace_bytes, void* stream) {
  const bool gate_up_f32 = take_gate_up_f32(&dtype);
  RETURN_IF(sub_check(T, D, F, dtype, act));
  if (x_stride < D || w_gate_stride < D || w_up_stride < D || w_down_stride < F ||
      (gate == nullptr) != (up == nullptr) || (gate && gate_up_stride < F))
    return MHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return MHC_OK;
  if (!x || !w_gate || !w_up || !w_down || !y) return MHC_ERR_INVALID_ARGUMENT;
  Operand ox{x, x_stride, true}, og{w_gate, w_gate_stride, true}, ou{w_up, w_up_stride, true},
      od{w_down, w_down_stride, true};
  if (!ws_ok(workspace, workspace_bytes,
             mhc_gated_ffn_fwd_workspace_bytes(
                 T, D, F, dtype, any_unaligned({ox, og, ou, od, {y, D, true}}))))
    return MHC_ERR_WORKSPACE;
  RETURN_IF(check_device());
  const cudaStream_t s = (cudaStream_t)stream;
  Carver c{(char*)workspace};
  const int64_t ldh = pad16(F);
  void* h = c.take(packed_bytes(T, F));
  void* room = c.take(ffn_fwd_room(T, D, F));
  const bool few = gemv_takes(T, F, D);
  if (!few) {
    RETURN_IF(aligned_operand(&ox, T, D, &c, s));
    RETURN_IF(aligned_operand(&og, F, D, &c, s));
    RETURN_IF(aligned_operand(&ou, F, D, &c, s));
    RETURN_IF(aligned_operand(&od, D, F, &c, s));
  }
  Gemm g;
  g.kind = kEpiGated;
  g.dtype = dtype;
  g.M = T; g.N = F; g.K = D;
  g.a = ox;
  g.b = og;
  g.b2 = ou;
  g.epi.act = act; g.epi.out = h; g.epi.ld_out = ldh;
  g.epi.gate = gate; g.epi.up = up; g.epi.ld_gu = gate ? gate_up_stride : 0;
  g.epi.gu32 = gate_up_f32;
  RETURN_IF(few ? gemv_run(g, s) : gemm_run(g, room, s));
  Gemm d;
  d.dtype = dtype;
  d.M = T; d.N = D; d.K = F;
  d.a = {h, ldh, true};
  d.b = od;
  d.epi.out = y; d.epi.ld_out = D;
  return few ? gemv_run(d, s) : run_product(&d, room, c, s);
}

size_t mhc_gated_ffn_bwd_workspace_bytes(int64_t T, int64_t D, int64_t F, int32_t dtype,
                                         int32_t unaligned) {
  take_gate_up_f32(&dtype);
  if (sub_check(T, D, F, dtype, 0) != MHC_OK) return 0;
  Carver c{nullptr};
  for (int i = 0; i < 3; ++i) c.take(packed_bytes(T, F));  // gg, gu, h
  c.take(ffn_bwd_room(T, D, F));
  if (unaligned) {
    for (int i = 0; i < 2; ++i) c.take(packed_bytes(T, D));  // x, grad_y
    for (int i = 0; i < 2; ++i) c.take(packed_bytes(F, D));  // w_gate, w_up
    c.take(packed_bytes(D, F));                              // w_down
    c.take(std::max(packed_bytes(T, D), std::max(packed_bytes(F, D), packed_bytes(D, F))));
  }
  return c.off;
}

int mhc_gated_ffn_bwd(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride,
                      const void* w_up, int64_t w_up_stride, const void* w_down,
                      int64_t w_down_stride, const void* gate, const void* up,
                      int64_t gate_up_stride, const void* grad_y, int64_t grad_y_stride,
                      int64_t T, int64_t D, int64_t F, int32_t dtype, int32_t act, void* grad_x,
                      void* grad_w_gate, void* grad_w_up, void* grad_w_down, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const bool gate_up_f32 = take_gate_up_f32(&dtype);
  RETURN_IF(sub_check(T, D, F, dtype, act));
  if (x_stride < D || w_gate_stride < D || w_up_stride < D || w_down_stride < F ||
      gate_up_stride < F || grad_y_stride < D)
    return MHC_ERR_INVALID_ARGUMENT;
  const cudaStream_t s = (cudaStream_t)stream;
  if (T > 0 && (!x || !w_gate || !w_up || !w_down || !gate || !up || !grad_y))
    return MHC_ERR_INVALID_ARGUMENT;
  if (!grad_x && !grad_w_gate && !grad_w_up && !grad_w_down) return MHC_OK;
  Operand ox{x, x_stride, false}, oy{grad_y, grad_y_stride, true},
      og{w_gate, w_gate_stride, false}, ou{w_up, w_up_stride, false},
      od{w_down, w_down_stride, false};
  if (T > 0 &&
      !ws_ok(workspace, workspace_bytes,
             mhc_gated_ffn_bwd_workspace_bytes(
                 T, D, F, dtype,
                 any_unaligned({ox, oy, og, ou, od, {grad_x, D, true}, {grad_w_gate, D, true},
                                {grad_w_up, D, true}, {grad_w_down, F, true}}))))
    return MHC_ERR_WORKSPACE;
  RETURN_IF(check_device());
  if (T == 0) {
    RETURN_IF(zero(grad_w_gate, (size_t)F * D * 2, s));
    RETURN_IF(zero(grad_w_up, (size_t)F * D * 2, s));
    return zero(grad_w_down, (size_t)F * D * 2, s);
  }
  Carver c{(char*)workspace};
  const int64_t ld = pad16(F);
  void* gg = c.take(packed_bytes(T, F));
  void* gu = c.take(packed_bytes(T, F));
  void* h = c.take(packed_bytes(T, F));
  void* room = c.take(ffn_bwd_room(T, D, F));
  RETURN_IF(aligned_operand(&oy, T, D, &c, s));
  RETURN_IF(aligned_operand(&od, D, F, &c, s));
  {
    Gemm g;  // gh = grad_y w_down, then gg, gu and h in its epilogue
    g.kind = gate_up_f32 ? kEpiGatedBwd32 : kEpiGatedBwd;
    g.dtype = dtype;
    g.M = T; g.N = F; g.K = D;
    g.a = oy;
    g.b = od;
    g.epi.act = act;
    g.epi.gate = const_cast<void*>(gate); g.epi.up = const_cast<void*>(up);
    g.epi.ld_gu = gate_up_stride;
    g.epi.gu32 = gate_up_f32;
    g.epi.gg = gg; g.epi.gu = gu; g.epi.ld_g = ld;
    g.epi.out = h; g.epi.ld_out = ld;
    RETURN_IF(gemm_run(g, room, s));
  }
  if (grad_x) {
    RETURN_IF(aligned_operand(&og, F, D, &c, s));
    RETURN_IF(aligned_operand(&ou, F, D, &c, s));
  }
  if (grad_w_gate || grad_w_up) RETURN_IF(aligned_operand(&ox, T, D, &c, s));
  Gemm g;
  g.dtype = dtype;
  if (grad_x) {
    g.M = T; g.N = D; g.K = F;
    g.a = {gg, ld, true};
    g.b = og;
    g.a3 = {gu, ld, true};
    g.b3 = ou;
    g.K3 = F;
    g.epi.out = grad_x; g.epi.ld_out = D;
    RETURN_IF(run_product(&g, room, c, s));
    g.K3 = 0;
  }
  g.K = T;
  g.M = F; g.N = D;
  g.b = ox;
  g.epi.ld_out = D;
  if (grad_w_gate) {
    g.a = {gg, ld, false};
    g.epi.out = grad_w_gate;
    RETURN_IF(run_product(&g, room, c, s));
  }
  if (grad_w_up) {
    g.a = {gu, ld, false};
    g.epi.out = grad_w_up;
    RETURN_IF(run_product(&g, room, c, s));
  }
  if (grad_w_down) {
    g.M = D; g.N = F;
    g.a = {oy.p, oy.ld, false};
    g.b = {h, ld, false};
    g.epi.out = grad_w_down; g.epi.ld_out = F;
    RETURN_IF(run_product(&g, room, c, s));
  }
  return MHC_OK;
}

}  // extern "C"
