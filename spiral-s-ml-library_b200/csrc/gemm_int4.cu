// Products with weights in 4 bits and a scale per group of 32, 64 or 128 along a row: w = scale (q - 8), q in 0 .. 15.
//
// Codes [n, ceil(k / 2)] hold two weights in a byte, the even one in the low half; scales are [ceil(k / group), n], so that
// those that a tile of rows needs together are neighbours.  c = a w^T of few rows of `a` reads every weight once, and its
// time is that of their bytes.
#include "common.cuh"
#include "vector_io.cuh"

namespace {

template <typename S>
struct Int4ScaleMax { static constexpr float value = 3.38953139e38f; };
template <>
struct Int4ScaleMax<__half> { static constexpr float value = 65504.f; };

struct QuantInt4Args {
  const void* x;
  uint8_t* codes;
  void* scales;
  long long ldx, ldc, n, groups;
  int k, group;
};

// One warp per group: the largest magnitude becomes 7 steps.
template <typename T, typename S>
__global__ void __launch_bounds__(256) quantize_int4_kernel(QuantInt4Args p) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x & 31;
  for (long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); item < p.n * p.groups; item += (long long)gridDim.x * 8) {
    const long long row = item / p.groups, b = item - row * p.groups;
    const long long k0 = b * p.group;
    const int count = (int)min((long long)p.group, p.k - k0);
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx + k0;
    float largest = 0.f;
    for (int i = lane; i < count; i += 32) largest = fmaxf(largest, fabsf(sb_to_f32<T>(x[i])));
    for (int o = 16; o; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    // (f16: a scale of at most its largest value, whose groups' larger weights are cut off.)
    const S scale = sb_from_f32<S>(sizeof(S) == 2 ? fminf(largest / 7.f, Int4ScaleMax<S>::value) : largest / 7.f);
    const float s = sb_to_f32<S>(scale);
    if (lane == 0) reinterpret_cast<S*>(p.scales)[b * p.n + row] = scale;
    for (int i = 2 * lane; i < count; i += 64) {
      uint32_t byte = 0;
      for (int h = 0; h < 2; ++h) {
        const float v = i + h < count && s > 0.f ? rintf(sb_to_f32<T>(x[i + h]) / s) : 0.f;
        byte |= (uint32_t)(int)(fminf(fmaxf(v, -8.f), 7.f) + 8.f) << (4 * h);
      }
      p.codes[row * p.ldc + (k0 + i) / 2] = (uint8_t)byte;
    }
  }
}

struct Int4Args {
  const void* a;
  const uint8_t* codes;
  const void* scales;
  const float* bias;
  void* c;
  long long lda, ldw, ldc;
  int m, n, k, group, relu, out_dtype;
};

template <typename S, typename Out>
__global__ void __launch_bounds__(256) dequantize_int4_kernel(const uint8_t* codes, long long ldw, const S* scales, Out* out, long long ldo, long long n, int k, int group) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const long long pairs = (k + 1) / 2;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n * pairs; e += (long long)gridDim.x * 256) {
    const long long row = e / pairs, b = e - row * pairs;
    const uint32_t q = codes[row * ldw + b];
    const float s = sb_to_f32<S>(scales[2 * b / group * n + row]);
    Out* o = out + row * ldo + 2 * b;
    o[0] = sb_from_f32<Out>(s * ((float)(q & 15u) - 8.f));
    if (2 * b + 1 < k) o[1] = sb_from_f32<Out>(s * ((float)(q >> 4) - 8.f));
  }
}

__device__ __forceinline__ void int4_store(const Int4Args& p, long long row, int col, float v) {
  if (p.bias) v += p.bias[col];
  if (p.relu) v = fmaxf(v, 0.f);
  const long long at = row * p.ldc + col;
  if (p.out_dtype == SB_F32) reinterpret_cast<float*>(p.c)[at] = v;
  else if (p.out_dtype == SB_BF16) reinterpret_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p.c)[at] = __float2half_rn(v);
}

// Any pitch and alignment: a warp per output, lanes over the bytes of the row.
template <typename T, typename S>
__global__ void __launch_bounds__(256) gemm_int4_simple_kernel(Int4Args p) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x & 31;
  const long long total = (long long)p.m * p.n;
  for (long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); item < total; item += (long long)gridDim.x * 8) {
    const long long row = item / p.n;
    const int col = (int)(item - row * p.n);
    const T* a = reinterpret_cast<const T*>(p.a) + row * p.lda;
    const uint8_t* w = p.codes + (long long)col * p.ldw;
    const S* s = reinterpret_cast<const S*>(p.scales) + col;
    float sum = 0.f;
    for (int b = lane; b < (p.k + 1) / 2; b += 32) {
      const uint32_t q = w[b];
      float v = sb_to_f32<T>(a[2 * b]) * ((float)(q & 15u) - 8.f);
      if (2 * b + 1 < p.k) v = fmaf(sb_to_f32<T>(a[2 * b + 1]), (float)(q >> 4) - 8.f, v);
      sum = fmaf(v, sb_to_f32<S>(s[(long long)(2 * b / p.group) * p.n]), sum);
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) int4_store(p, row, col, sum);
  }
}

int int4_args_ok(const char* who, long long n, int k, int group, int scale_dtype) {
  if (n < 0 || k < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (group != 32 && group != 64 && group != 128) return sb_fail(SB_ERR_UNSUPPORTED, "%s: groups of 32, 64 or 128 (got %d)", who, group);
  if (scale_dtype != SB_F32 && scale_dtype != SB_BF16 && scale_dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: scales are f32, bf16 or f16 (got %d)", who, scale_dtype);
  if (n > (1LL << 30) || k > (1 << 30)) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most 2^30 rows and columns", who);
  return SB_OK;
}

bool int4_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (size_t)sb_dtype_size(dtype) == 0; }

template <typename T, typename S>
int launch_int4_simple(const Int4Args& p, cudaStream_t s) {
  const long long blocks = ((long long)p.m * p.n + 7) / 8, most = 64LL * sb_sm_count();
  SB_CUDA(sb_launch(gemm_int4_simple_kernel<T, S>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, s, 1, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

// Calls FN<.., S> by the type of the scales.
template <typename T>
int launch_int4(const Int4Args& p, int scale_dtype, cudaStream_t s) {
  return scale_dtype == SB_F32 ? launch_int4_simple<T, float>(p, s)
         : scale_dtype == SB_BF16 ? launch_int4_simple<T, __nv_bfloat16>(p, s) : launch_int4_simple<T, __half>(p, s);
}

template <typename T>
int launch_quantize_int4(const QuantInt4Args& p, int scale_dtype, cudaStream_t s) {
  const long long blocks = (p.n * p.groups + 7) / 8, most = 32LL * sb_sm_count();
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (scale_dtype == SB_F32) SB_CUDA(sb_launch(quantize_int4_kernel<T, float>, grid, dim3(256), 0, s, 1, p));
  else if (scale_dtype == SB_BF16) SB_CUDA(sb_launch(quantize_int4_kernel<T, __nv_bfloat16>, grid, dim3(256), 0, s, 1, p));
  else SB_CUDA(sb_launch(quantize_int4_kernel<T, __half>, grid, dim3(256), 0, s, 1, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename S>
int launch_dequantize_int4(const uint8_t* codes, long long ldw, const void* scales, void* out, long long ldo, int out_dtype, long long n, int k, int group, cudaStream_t s) {
  const long long blocks = (n * ((k + 1) / 2) + 255) / 256, most = 32LL * sb_sm_count();
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  const S* sc = reinterpret_cast<const S*>(scales);
  if (out_dtype == SB_F32) SB_CUDA(sb_launch(dequantize_int4_kernel<S, float>, grid, dim3(256), 0, s, 1, codes, ldw, sc, reinterpret_cast<float*>(out), ldo, n, k, group));
  else if (out_dtype == SB_BF16) SB_CUDA(sb_launch(dequantize_int4_kernel<S, __nv_bfloat16>, grid, dim3(256), 0, s, 1, codes, ldw, sc, reinterpret_cast<__nv_bfloat16*>(out), ldo, n, k, group));
  else SB_CUDA(sb_launch(dequantize_int4_kernel<S, __half>, grid, dim3(256), 0, s, 1, codes, ldw, sc, reinterpret_cast<__half*>(out), ldo, n, k, group));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

}  // namespace

extern "C" {

int sb_quantize_int4(const void* x, long long ldx, int dtype, long long n, int k, int group, uint8_t* codes, long long ldc, void* scales,
                     int scale_dtype, void* stream) {
  const char* who = "sb_quantize_int4";
  int rc = int4_args_ok(who, n, k, group, scale_dtype);
  if (rc != SB_OK) return rc;
  if (dtype != SB_F32 && dtype != SB_BF16 && dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: storage types are f32, bf16 and f16 (got %d)", who, dtype);
  if (n == 0 || k == 0) return SB_OK;
  if (!x || !codes || !scales) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ldx < k || ldc < (k + 1) / 2) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than its rows", who);
  if (!int4_aligned(x, dtype) || !int4_aligned(scales, scale_dtype))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  const QuantInt4Args p = {x, codes, scales, ldx, ldc, n, (k + group - 1) / group, k, group};
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_F32 ? launch_quantize_int4<float>(p, scale_dtype, s)
         : dtype == SB_BF16 ? launch_quantize_int4<__nv_bfloat16>(p, scale_dtype, s) : launch_quantize_int4<__half>(p, scale_dtype, s);
}

int sb_dequantize_int4(const uint8_t* codes, long long ldw, const void* scales, int scale_dtype, void* out, long long ldo, int out_dtype,
                       long long n, int k, int group, void* stream) {
  const char* who = "sb_dequantize_int4";
  int rc = int4_args_ok(who, n, k, group, scale_dtype);
  if (rc != SB_OK) return rc;
  if (out_dtype != SB_F32 && out_dtype != SB_BF16 && out_dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: storage types are f32, bf16 and f16 (got %d)", who, out_dtype);
  if (n == 0 || k == 0) return SB_OK;
  if (!codes || !scales || !out) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ldw < (k + 1) / 2 || ldo < k) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than its rows", who);
  if (!int4_aligned(out, out_dtype) || !int4_aligned(scales, scale_dtype))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  cudaStream_t s = (cudaStream_t)stream;
  return scale_dtype == SB_F32 ? launch_dequantize_int4<float>(codes, ldw, scales, out, ldo, out_dtype, n, k, group, s)
         : scale_dtype == SB_BF16 ? launch_dequantize_int4<__nv_bfloat16>(codes, ldw, scales, out, ldo, out_dtype, n, k, group, s)
                                  : launch_dequantize_int4<__half>(codes, ldw, scales, out, ldo, out_dtype, n, k, group, s);
}

int sb_matmul_int4(const void* a, long long lda, int dtype, const uint8_t* codes, long long ldw, const void* scales, int scale_dtype, void* c,
                   long long ldc, int m, int n, int k, int group, int out_dtype, int epilogue, const float* bias, void* stream) {
  const char* who = "sb_matmul_int4";
  int rc = int4_args_ok(who, n, k, group, scale_dtype);
  if (rc != SB_OK) return rc;
  if (m < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (dtype != SB_BF16 && dtype != SB_F16) return sb_fail(SB_ERR_UNSUPPORTED, "%s: a holds bf16 or f16 (got %d)", who, dtype);
  if (out_dtype != SB_F32 && out_dtype != SB_BF16 && out_dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: outputs are f32, bf16 or f16 (got %d)", who, out_dtype);
  if (epilogue & ~(SB_EPI_BIAS | SB_EPI_RELU)) return sb_fail(SB_ERR_UNSUPPORTED, "%s: epilogues are bias and ReLU", who);
  if (m == 0 || n == 0) return SB_OK;
  if (!c || ((epilogue & SB_EPI_BIAS) && !bias) || (k > 0 && (!a || !codes || !scales))) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ldc < n || (k > 0 && (lda < k || ldw < (k + 1) / 2))) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than its rows", who);
  if (!int4_aligned(a, dtype) || !int4_aligned(scales, scale_dtype) || !int4_aligned(c, out_dtype) || !int4_aligned(bias, SB_F32))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  Int4Args p;
  memset(&p, 0, sizeof(p));
  p.a = a; p.codes = codes; p.scales = scales; p.bias = (epilogue & SB_EPI_BIAS) ? bias : nullptr; p.c = c;
  p.lda = lda; p.ldw = ldw; p.ldc = ldc; p.m = m; p.n = n; p.k = k; p.group = group; p.relu = (epilogue & SB_EPI_RELU) ? 1 : 0;
  p.out_dtype = out_dtype;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_BF16 ? launch_int4<__nv_bfloat16>(p, scale_dtype, s) : launch_int4<__half>(p, scale_dtype, s);
}

}  // extern "C"
