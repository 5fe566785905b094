// Layer normalisation and its gradient.
//
//   mean = sum(x) / n, var = sum((x - mean)^2) / n, rstd = 1 / sqrt(var + eps), xhat = (x - mean) rstd
//   y = xhat w + b
//   with g = dy w:  dx = rstd (g - sum(g) / n - xhat sum(g xhat) / n)
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// Statistics and sums are fp32; the variance is taken about the mean (a second pass over values that are already in
// registers), since the difference of two moments loses all digits of rows with a large offset.
#include "common.cuh"
#include "vector_io.cuh"

namespace {

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;                     // y, or dx
  const float* weight;           // NULL: ones
  const float* bias;             // NULL: zeros
  float* mean;                   // written by the forward pass (may be NULL there), read by the backward pass
  float* rstd;
  float* partial;                // backward: fp32 [blocks][2][cols] partial column sums; NULL: not wanted
  long long rows, ldx, lddy, ldout;
  int cols;
  float eps, inv_cols;
};

__device__ __forceinline__ float ln_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the block; `slot` (32 floats of shared memory) must not be in use by a sum whose readers may still be
// behind: callers alternate between slots, so that one barrier per sum is enough.
__device__ __forceinline__ float ln_block_sum(float v, float* slot) {
  v = ln_warp_sum(v);
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  const float w = (int)(threadIdx.x & 31) < warps ? slot[threadIdx.x & 31] : 0.f;
  return ln_warp_sum(w);
}

// Any row length and alignment: a block per row, the row read three times (the second and third time from L2).
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_wide_kernel(NormArgs a) {
  __shared__ float slots[2][32];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    T* y = (T*)a.out + row * a.ldout;
    float s = 0.f;
    for (int j = threadIdx.x; j < a.cols; j += blockDim.x) s += sb_to_f32<T>(x[j]);
    const float mean = ln_block_sum(s, slots[0]) * a.inv_cols;
    float q = 0.f;
    for (int j = threadIdx.x; j < a.cols; j += blockDim.x) {
      const float d = sb_to_f32<T>(x[j]) - mean;
      q += d * d;
    }
    const float rstd = 1.f / sqrtf(ln_block_sum(q, slots[1]) * a.inv_cols + a.eps);
    for (int j = threadIdx.x; j < a.cols; j += blockDim.x) {
      const float h = (sb_to_f32<T>(x[j]) - mean) * rstd;
      y[j] = sb_from_f32<T>(h * (a.weight ? a.weight[j] : 1.f) + (a.bias ? a.bias[j] : 0.f));
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_grad_wide_kernel(NormArgs a) {
  __shared__ float slots[2][32];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    const T* dy = (const T*)a.dy + row * a.lddy;
    T* dx = (T*)a.out + row * a.ldout;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.f, sgx = 0.f;
    for (int j = threadIdx.x; j < a.cols; j += blockDim.x) {
      const float g = sb_to_f32<T>(dy[j]) * (a.weight ? a.weight[j] : 1.f);
      sg += g;
      sgx += g * ((sb_to_f32<T>(x[j]) - mean) * rstd);
    }
    sg = ln_block_sum(sg, slots[0]) * a.inv_cols;
    sgx = ln_block_sum(sgx, slots[1]) * a.inv_cols;
    for (int j = threadIdx.x; j < a.cols; j += blockDim.x) {
      const float g = sb_to_f32<T>(dy[j]) * (a.weight ? a.weight[j] : 1.f);
      const float h = (sb_to_f32<T>(x[j]) - mean) * rstd;
      dx[j] = sb_from_f32<T>(rstd * (g - sg - h * sgx));
    }
  }
}

// Column sums of dy xhat and dy over this block's rows: a thread per column, coalesced along the row.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(NormArgs a) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= a.cols) return;
  const T* x = (const T*)a.x + j;
  const T* dy = (const T*)a.dy + j;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float d = sb_to_f32<T>(dy[row * a.lddy]);
    dw += d * ((sb_to_f32<T>(x[row * a.ldx]) - a.mean[row]) * a.rstd[row]);
    db += d;
  }
  float* p = a.partial + (long long)blockIdx.y * 2 * a.cols;
  p[j] = dw;
  p[a.cols + j] = db;
}

// Adds the partial column sums of all blocks in their order: 32 columns per block, its warps take every 32nd part,
// and the warps' sums meet in shared memory.
__global__ void __launch_bounds__(1024)
layer_norm_partials_kernel(const float* __restrict__ partial, int parts, int cols, float* __restrict__ dweight,
                           float* __restrict__ dbias, int accumulate) {
  __shared__ float sums[32][33];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;
  float* out = blockIdx.y == 0 ? dweight : dbias;
  if (!out) return;
  float s = 0.f;
  if (j < cols)
    for (int p = warp; p < parts; p += 32) s += partial[((long long)p * 2 + blockIdx.y) * cols + j];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && j < cols) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) total += sums[w][lane];
    out[j] = accumulate ? out[j] + total : total;
  }
}

int ln_columns_blocks(long long rows) {
  const long long want = (rows + 31) / 32, most = 4LL * sb_sm_count();
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

int norm_args_ok(const char* who, long long rows, int cols, int dtype, const void* x, long long ldx) {
  if (rows < 0 || cols < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (dtype != SB_F32 && dtype != SB_BF16 && dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: storage types are f32, bf16 and f16 (got %d)", who, dtype);
  if (rows == 0 || cols == 0) return SB_OK;
  if (!x) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ldx < cols) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch of %lld is shorter than the %d columns", who, ldx, cols);
  return SB_OK;
}

// Misaligned elements fault on the device, so their alignment is checked here.
int norm_element_aligned(const char* who, const void* p, int dtype) {
  if ((reinterpret_cast<uintptr_t>(p) % (size_t)sb_dtype_size(dtype)) != 0)
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  return SB_OK;
}

template <typename T>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t s) {
  const int threads = a.cols >= 1024 ? 1024 : (a.cols + 31) / 32 * 32;
  const long long most = 16LL * sb_sm_count();
  const int grid = (int)(a.rows < most ? a.rows : most);
  return sb_launch(layer_norm_wide_kernel<T>, dim3(grid), dim3(threads), 0, s, 1, a);
}

template <typename T>
cudaError_t launch_norm_grad(const NormArgs& a, cudaStream_t s) {
  const int threads = a.cols >= 1024 ? 1024 : (a.cols + 31) / 32 * 32;
  const long long most = 16LL * sb_sm_count();
  const int grid = (int)(a.rows < most ? a.rows : most);
  return sb_launch(layer_norm_grad_wide_kernel<T>, dim3(grid), dim3(threads), 0, s, 1, a);
}

}  // namespace

extern "C" {

int sb_layer_norm(const void* x, long long ldx, void* y, long long ldy, const float* weight, const float* bias, float eps,
                  float* mean, float* rstd, long long rows, int cols, int dtype, void* stream) {
  int rc = norm_args_ok("sb_layer_norm", rows, cols, dtype, x, ldx);
  if (rc != SB_OK || rows == 0 || cols == 0) return rc;
  if ((rc = norm_args_ok("sb_layer_norm", rows, cols, dtype, y, ldy)) != SB_OK) return rc;
  if ((rc = norm_element_aligned("sb_layer_norm", x, dtype)) != SB_OK) return rc;
  if ((rc = norm_element_aligned("sb_layer_norm", y, dtype)) != SB_OK) return rc;
  for (const void* p : {(const void*)weight, (const void*)bias, (const void*)mean, (const void*)rstd})
    if ((rc = norm_element_aligned("sb_layer_norm", p, SB_F32)) != SB_OK) return rc;
  if (!(eps >= 0.f)) return sb_fail(SB_ERR_BAD_ARG, "sb_layer_norm: eps must not be negative");
  NormArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x; a.out = y; a.weight = weight; a.bias = bias; a.mean = mean; a.rstd = rstd;
  a.rows = rows; a.ldx = ldx; a.ldout = ldy; a.cols = cols; a.eps = eps; a.inv_cols = 1.f / (float)cols;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = dtype == SB_F32 ? launch_norm<float>(a, s)
                                  : dtype == SB_BF16 ? launch_norm<__nv_bfloat16>(a, s) : launch_norm<__half>(a, s);
  SB_COUNT_LAUNCH();
  return sb_check_cuda(e, "sb_layer_norm");
}

int sb_layer_norm_grad_workspace_bytes(long long rows, int cols, size_t* bytes) {
  if (!bytes) return sb_fail(SB_ERR_BAD_ARG, "sb_layer_norm_grad_workspace_bytes: null output");
  if (rows < 0 || cols < 0) return sb_fail(SB_ERR_BAD_ARG, "sb_layer_norm_grad_workspace_bytes: negative size");
  *bytes = (size_t)ln_columns_blocks(rows) * 2 * (size_t)cols * sizeof(float);
  return SB_OK;
}

int sb_layer_norm_grad(const void* dy, long long lddy, const void* x, long long ldx, const float* mean, const float* rstd,
                       const float* weight, void* dx, long long lddx, float* dweight, float* dbias, int accumulate,
                       long long rows, int cols, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "sb_layer_norm_grad";
  int rc = norm_args_ok(who, 0, cols, dtype, nullptr, 0);
  if (rc != SB_OK || cols == 0) return rc;
  if (rows < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {               // no row, no gradient: sums over nothing
    if (!accumulate)
      for (float* p : {dweight, dbias})
        if (p) SB_CUDA(cudaMemsetAsync(p, 0, sizeof(float) * (size_t)cols, s));
    return SB_OK;
  }
  if ((rc = norm_args_ok(who, rows, cols, dtype, dy, lddy)) != SB_OK) return rc;
  if ((rc = norm_args_ok(who, rows, cols, dtype, x, ldx)) != SB_OK) return rc;
  if (dx && (rc = norm_args_ok(who, rows, cols, dtype, dx, lddx)) != SB_OK) return rc;
  if (!mean || !rstd) return sb_fail(SB_ERR_BAD_ARG, "%s: the rows' mean and rstd are needed", who);
  for (const void* p : {dy, x, (const void*)dx})
    if ((rc = norm_element_aligned(who, p, dtype)) != SB_OK) return rc;
  for (const void* p : {(const void*)mean, (const void*)rstd, (const void*)weight, (const void*)dweight, (const void*)dbias,
                        (const void*)workspace})
    if ((rc = norm_element_aligned(who, p, SB_F32)) != SB_OK) return rc;
  const bool columns = dweight || dbias;
  if (columns) {
    size_t need = 0;
    sb_layer_norm_grad_workspace_bytes(rows, cols, &need);
    if (!workspace || workspace_bytes < need)
      return sb_fail(SB_ERR_BAD_ARG, "%s: needs a workspace of %zu bytes (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
  }
  NormArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x; a.dy = dy; a.out = dx; a.weight = weight; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.partial = (float*)workspace; a.rows = rows; a.ldx = ldx; a.lddy = lddy; a.ldout = lddx; a.cols = cols;
  a.inv_cols = 1.f / (float)cols;
  if (dx) {
    cudaError_t e = dtype == SB_F32 ? launch_norm_grad<float>(a, s)
                                    : dtype == SB_BF16 ? launch_norm_grad<__nv_bfloat16>(a, s) : launch_norm_grad<__half>(a, s);
    SB_COUNT_LAUNCH();
    SB_CUDA(e);
  }
  if (columns) {
    const int parts = ln_columns_blocks(rows);
    const dim3 grid((cols + 255) / 256, parts);
    cudaError_t e = dtype == SB_F32 ? sb_launch(layer_norm_columns_kernel<float>, grid, dim3(256), 0, s, 1, a)
                    : dtype == SB_BF16 ? sb_launch(layer_norm_columns_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, 1, a)
                                       : sb_launch(layer_norm_columns_kernel<__half>, grid, dim3(256), 0, s, 1, a);
    SB_COUNT_LAUNCH();
    SB_CUDA(e);
    e = sb_launch(layer_norm_partials_kernel, dim3((cols + 31) / 32, 2), dim3(1024), 0, s, 1, (const float*)workspace, parts, cols,
                  dweight, dbias, accumulate);
    SB_COUNT_LAUNCH();
    SB_CUDA(e);
  }
  return SB_OK;
}

}  // extern "C"
