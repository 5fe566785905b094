// Gated layers: h = act(x Wg^T) * (x Wu^T), both projections, the activation and their product in one kernel, and the gradient.
//
// With g = x Wg^T, u = x Wu^T and a the activation:
//   dg = dh u a'(g)   du = dh a(g)   dx = dg Wg + du Wu   dWg = dg^T x   dWu = du^T x
//   silu: a = g s(g), a' = s (1 + g (1 - s)) with s = 1 / (1 + exp(-g));  gelu: a = g P(g), a' = P(g) + g exp(-g^2 / 2) / sqrt(2 pi)
//   with the normal distribution P(g) = (1 + erf(g / sqrt 2)) / 2;  relu: a = max(0, g), a' = [g > 0].
#include "common.cuh"
#include "vector_io.cuh"

namespace {

enum GatedAct { ACT_SILU = SB_ACT_SILU, ACT_GELU = SB_ACT_GELU, ACT_RELU = SB_ACT_RELU };

__device__ __forceinline__ float gated_sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

template <int ACT>
__device__ __forceinline__ float gated_act(float g) {
  if (ACT == ACT_SILU) return g * gated_sigmoid(g);
  if (ACT == ACT_GELU) return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
  return g > 0.f ? g : (g != g ? g : 0.f);
}
// The activation and its derivative.
template <int ACT>
__device__ __forceinline__ float2 gated_act_grad(float g) {
  if (ACT == ACT_SILU) {
    const float s = gated_sigmoid(g);
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  if (ACT == ACT_GELU) {
    const float p = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    return make_float2(g * p, p + g * __expf(-0.5f * g * g) * 0.39894228040143268f);
  }
  return make_float2(gated_act<ACT_RELU>(g), g > 0.f ? 1.f : 0.f);
}

// Any sizes, pitches and alignments, on the CUDA cores: 64 x 64 outputs per block, 16 of K at a time.
constexpr int GS_TILE = 64, GS_K = 16;

// A matrix by the distances of neighbours in a column and in a row.
struct Strided {
  const void* p;
  long long down, across;
};

template <typename T>
__device__ __forceinline__ float strided_at(const Strided& m, long long i, long long j) {
  return sb_to_f32<T>(reinterpret_cast<const T*>(m.p)[i * m.down + j * m.across]);
}

template <typename T>
__device__ __forceinline__ void simple_tile(float (*to)[GS_TILE + 4], const Strided& m, long long i0, long long k0, long long rows, long long ks, bool rows_first) {
  for (int e = threadIdx.x; e < GS_TILE * GS_K; e += 256) {
    // Neighbouring threads read neighbouring elements.
    const int i = rows_first ? e % GS_TILE : e / GS_K, k = rows_first ? e / GS_TILE : e % GS_K;
    to[k][i] = i0 + i < rows && k0 + k < ks ? strided_at<T>(m, i0 + i, k0 + k) : 0.f;
  }
}

struct GatedArgs {
  const void* x;
  const void* w;
  void* h;
  void* saved;
  long long ldx, ldw, ldh, lds;
  int m, f, k;
};

template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_simple_kernel(GatedArgs p) {
  __shared__ float sx[GS_K][GS_TILE + 4], sg[GS_K][GS_TILE + 4], su[GS_K][GS_TILE + 4];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const long long i0 = (long long)blockIdx.x * GS_TILE, j0 = (long long)blockIdx.y * GS_TILE;
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  const Strided x = {p.x, p.ldx, 1}, g = {p.w, p.ldw, 1}, u = {reinterpret_cast<const T*>(p.w) + (long long)p.f * p.ldw, p.ldw, 1};
  float ag[4][4] = {}, au[4][4] = {};
  for (long long k0 = 0; k0 < p.k; k0 += GS_K) {
    simple_tile<T>(sx, x, i0, k0, p.m, p.k, false);
    simple_tile<T>(sg, g, j0, k0, p.f, p.k, false);
    simple_tile<T>(su, u, j0, k0, p.f, p.k, false);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < GS_K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ag[i][j] = fmaf(sx[k][ti + i], sg[k][tj + j], ag[i][j]);
          au[i][j] = fmaf(sx[k][ti + i], su[k][tj + j], au[i][j]);
        }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const long long r = i0 + ti + i, c = j0 + tj + j;
      if (r >= p.m || c >= p.f) continue;
      reinterpret_cast<T*>(p.h)[r * p.ldh + c] = sb_from_f32<T>(gated_act<ACT>(ag[i][j]) * au[i][j]);
      if (p.saved) {
        reinterpret_cast<T*>(p.saved)[r * p.lds + c] = sb_from_f32<T>(ag[i][j]);
        reinterpret_cast<T*>(p.saved)[r * p.lds + p.f + c] = sb_from_f32<T>(au[i][j]);
      }
    }
}

// c (+)= a b with a [m, k] and b [n, k] by their strides.
template <typename T, typename Out>
__global__ void __launch_bounds__(256) gated_product_simple_kernel(Strided a, Strided b, Out* c, long long ldc, long long m, long long n, long long k, int accumulate) {
  __shared__ float sa[GS_K][GS_TILE + 4], sb[GS_K][GS_TILE + 4];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const long long i0 = (long long)blockIdx.x * GS_TILE, j0 = (long long)blockIdx.y * GS_TILE;
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  float acc[4][4] = {};
  for (long long k0 = 0; k0 < k; k0 += GS_K) {
    simple_tile<T>(sa, a, i0, k0, m, k, a.down == 1);
    simple_tile<T>(sb, b, j0, k0, n, k, b.down == 1);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < GS_K; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[kk][ti + i], sb[kk][tj + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const long long r = i0 + ti + i, q = j0 + tj + j;
      if (r >= m || q >= n) continue;
      Out* o = c + r * ldc + q;
      *o = sb_from_f32<Out>(accumulate ? acc[i][j] + sb_to_f32<Out>(*o) : acc[i][j]);
    }
}

struct GatedGradArgs {
  const void* dh;
  const void* saved;
  void* d;                        // [m, 2 f]: dg, du
  long long lddh, lds, ldd;
  int m, f;
};

template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_act_grad_kernel(GatedGradArgs p) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const long long total = (long long)p.m * p.f;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
    const long long r = e / p.f, c = e - r * p.f;
    const T* saved = reinterpret_cast<const T*>(p.saved) + r * p.lds + c;
    const float dh = sb_to_f32<T>(reinterpret_cast<const T*>(p.dh)[r * p.lddh + c]);
    const float2 a = gated_act_grad<ACT>(sb_to_f32<T>(saved[0]));
    T* d = reinterpret_cast<T*>(p.d) + r * p.ldd + c;
    d[0] = sb_from_f32<T>(dh * sb_to_f32<T>(saved[p.f]) * a.y);
    d[p.f] = sb_from_f32<T>(dh * a.x);
  }
}

bool gated_element_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (size_t)sb_dtype_size(dtype) == 0; }
bool gated_rows16(const void* p, long long ld, int dtype) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * sb_dtype_size(dtype) % 16 == 0; }

int gated_args_ok(const char* who, int m, int f, int k, int dtype, int activation) {
  if (m < 0 || f < 0 || k < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (dtype != SB_BF16 && dtype != SB_F16) return sb_fail(SB_ERR_UNSUPPORTED, "%s: storage types are bf16 and f16 (got %d)", who, dtype);
  if (activation != SB_ACT_SILU && activation != SB_ACT_GELU && activation != SB_ACT_RELU)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: unknown activation %d", who, activation);
  if (f > (1 << 21) || k > (1 << 21)) return sb_fail(SB_ERR_TOO_LARGE, "%s: layers of at most 2^21 columns and inputs", who);
  return SB_OK;
}

template <typename T, int ACT>
int launch_gated(const GatedArgs& p, cudaStream_t s) {
  const dim3 grid((unsigned)((p.m + GS_TILE - 1) / GS_TILE), (unsigned)((p.f + GS_TILE - 1) / GS_TILE));
  SB_CUDA(sb_launch(gated_simple_kernel<T, ACT>, grid, dim3(256), 0, s, 1, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int ACT>
int launch_gated_act_grad(const GatedGradArgs& p, cudaStream_t s) {
  long long blocks = ((long long)p.m * p.f + 255) / 256;
  const long long most = 16LL * sb_sm_count();
  SB_CUDA(sb_launch(gated_act_grad_kernel<T, ACT>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, s, 1, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, typename Out>
int launch_product_simple(const Strided& a, const Strided& b, void* c, long long ldc, long long m, long long n, long long k, int accumulate, cudaStream_t s) {
  const dim3 grid((unsigned)((m + GS_TILE - 1) / GS_TILE), (unsigned)((n + GS_TILE - 1) / GS_TILE));
  SB_CUDA(sb_launch(gated_product_simple_kernel<T, Out>, grid, dim3(256), 0, s, 1, a, b, reinterpret_cast<Out*>(c), ldc, m, n, k, accumulate));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T>
int gated_grad_simple(const GatedGradArgs& g, const void* x, long long ldx, const void* w, long long ldw, void* dx, long long lddx, void* dw,
                      long long lddw, int dw_dtype, int accumulate, int k, cudaStream_t s) {
  int rc = SB_OK;
  const long long f2 = 2LL * g.f;
  if (dx && g.m > 0 && k > 0) rc = launch_product_simple<T, T>({g.d, g.ldd, 1}, {w, 1, ldw}, dx, lddx, g.m, k, f2, 0, s);
  if (rc == SB_OK && dw && f2 > 0 && k > 0) {
    const Strided a = {g.d, 1, g.ldd}, b = {x, 1, ldx};
    rc = dw_dtype == SB_F32 ? launch_product_simple<T, float>(a, b, dw, lddw, f2, k, g.m, accumulate, s)
                            : launch_product_simple<T, T>(a, b, dw, lddw, f2, k, g.m, accumulate, s);
  }
  return rc;
}

}  // namespace

extern "C" {

int sb_gated(const void* x, long long ldx, const void* w, long long ldw, void* h, long long ldh, void* saved, long long lds, int m, int f,
             int k, int dtype, int activation, void* stream) {
  const char* who = "sb_gated";
  int rc = gated_args_ok(who, m, f, k, dtype, activation);
  if (rc != SB_OK || m == 0 || f == 0) return rc;
  if (!h || (k > 0 && (!x || !w))) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ldh < f || (saved && lds < 2LL * f) || (k > 0 && (ldx < k || ldw < k)))
    return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than its rows", who);
  if (!gated_element_aligned(x, dtype) || !gated_element_aligned(w, dtype) || !gated_element_aligned(h, dtype) || !gated_element_aligned(saved, dtype))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  const GatedArgs p = {x, w, h, saved, ldx, ldw, ldh, lds, m, f, k};
  cudaStream_t s = (cudaStream_t)stream;
#define SB_GATED_CALL(ACT) (dtype == SB_BF16 ? launch_gated<__nv_bfloat16, ACT>(p, s) : launch_gated<__half, ACT>(p, s))
  return activation == SB_ACT_SILU ? SB_GATED_CALL(ACT_SILU) : activation == SB_ACT_GELU ? SB_GATED_CALL(ACT_GELU) : SB_GATED_CALL(ACT_RELU);
#undef SB_GATED_CALL
}

int sb_gated_grad_workspace_bytes(int m, int f, int k, size_t* bytes) {
  const char* who = "sb_gated_grad_workspace_bytes";
  if (!bytes) return sb_fail(SB_ERR_BAD_ARG, "%s: null output", who);
  if (m < 0 || f < 0 || k < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  *bytes = (size_t)m * 2 * (size_t)f * 2;
  return SB_OK;
}

int sb_gated_grad(const void* dh, long long lddh, const void* x, long long ldx, const void* w, long long ldw, const void* saved, long long lds,
                  void* dx, long long lddx, void* dw, long long lddw, int dw_dtype, int accumulate, int m, int f, int k, int dtype,
                  int activation, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "sb_gated_grad";
  int rc = gated_args_ok(who, m, f, k, dtype, activation);
  if (rc != SB_OK) return rc;
  if (dw && dw_dtype != dtype && dw_dtype != SB_F32) return sb_fail(SB_ERR_UNSUPPORTED, "%s: dw holds f32 or the storage type (got %d)", who, dw_dtype);
  const bool any = m > 0 && f > 0;
  if (any && (!dh || !saved || !workspace)) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (any && ((dx && k > 0 && !w) || (dw && k > 0 && !x))) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if ((any && (lddh < f || lds < 2LL * f)) || (x && ldx < k) || (w && ldw < k) || (dx && lddx < k) || (dw && lddw < k))
    return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than its rows", who);
  if (!gated_element_aligned(dh, dtype) || !gated_element_aligned(saved, dtype) || !gated_element_aligned(x, dtype) || !gated_element_aligned(w, dtype) ||
      !gated_element_aligned(dx, dtype) || (dw && !gated_element_aligned(dw, dw_dtype)) || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size, or the workspace not to 256 bytes", who);
  size_t need = 0;
  if ((rc = sb_gated_grad_workspace_bytes(m, f, k, &need)) != SB_OK) return rc;
  if (any && workspace_bytes < need) return sb_fail(SB_ERR_BAD_ARG, "%s: the workspace has %zu bytes, %zu are needed", who, workspace_bytes, need);
  if (!dx && !dw) return SB_OK;
  const GatedGradArgs g = {dh, saved, workspace, lddh, lds, 2LL * f, m, f};
  cudaStream_t s = (cudaStream_t)stream;
#define SB_GATED_CALL(ACT) (dtype == SB_BF16 ? launch_gated_act_grad<__nv_bfloat16, ACT>(g, s) : launch_gated_act_grad<__half, ACT>(g, s))
  if (any) rc = activation == SB_ACT_SILU ? SB_GATED_CALL(ACT_SILU) : activation == SB_ACT_GELU ? SB_GATED_CALL(ACT_GELU) : SB_GATED_CALL(ACT_RELU);
#undef SB_GATED_CALL
  if (rc != SB_OK) return rc;
  return dtype == SB_BF16 ? gated_grad_simple<__nv_bfloat16>(g, x, ldx, w, ldw, dx, lddx, dw, lddw, dw_dtype, accumulate, k, s)
                          : gated_grad_simple<__half>(g, x, ldx, w, ldw, dx, lddx, dw, lddw, dw_dtype, accumulate, k, s);
}

}  // extern "C"
