// Products in 8-bit floating point (E4M3) with an fp32 scale per block of 128, and the quantisation that makes their
// operands.
//
//   codes = round(x * (448 / a)), scale = a / 448, a = max |x| over a block (1 x 128 or 128 x 128), at least 2^-100
//   C[m, n] = sum over blocks b of K   sa[b, m] * sw[n / 128, b] * sum over k in b of A[m, k] W[n, k]   (+ bias, ReLU)
//
// The sum inside a block and the sum over blocks are fp32.
#include "common.cuh"
#include "vector_io.cuh"

namespace {

constexpr int F8_BLOCK = 128;
constexpr float F8_TOP = 448.f;                              // the largest E4M3 value
constexpr float F8_FLOOR = 7.888609052210118e-31f;           // 2^-100

// Two fp32 values -> two E4M3 codes, lo in the low byte; round to nearest even, a NaN stays one.
__device__ __forceinline__ uint32_t f8_pack2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float2 f8_unpack2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float f8_to_f32(uint8_t c) { return f8_unpack2(c).x; }

struct QuantArgs {
  const void* x;
  uint8_t* codes;
  float* scales;
  long long rows, ldx, ldc;
  int cols;
};

// ------------------------------ quantisation -------------------------------------
// A block of 256 threads per ROWS x 128 tile of x, which stays in registers between the search for its largest magnitude
// and the rounding; L lanes share a row, V neighbouring elements each.  SQUARE: one scale for the tile, else one per row.
template <typename T, int V, int ROWS, bool SQUARE>
__global__ void __launch_bounds__(256) quantize_fp8_kernel(QuantArgs a) {
  constexpr int L = F8_BLOCK / V < 32 ? F8_BLOCK / V : 32;   // lanes per row
  constexpr int STEPS = F8_BLOCK / (V * L);                  // packs per lane and row
  constexpr int AT_ONCE = 256 / L;                           // rows
  constexpr int PASSES = ROWS / AT_ONCE;
  __shared__ uint32_t warp_max[8];
  __shared__ float row_scale[ROWS];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x % L, r0 = threadIdx.x / L;
  const long long row0 = (long long)blockIdx.x * ROWS;
  const int col0 = blockIdx.y * F8_BLOCK;
  SbPack<T, V> in[PASSES][STEPS];
  uint32_t all = 0u;
  uint32_t largest[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const long long row = row0 + p * AT_ONCE + r0;
    uint32_t mx = 0u;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int col = col0 + (s * L + lane) * V;
      in[p][s] = row < a.rows && col < a.cols ? sb_load_pack<T, V>((const T*)a.x + row * a.ldx + col) : sb_zero_pack<T, V>();
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      float v[V];
      sb_unpack<T, V>(in[p][s], v);
#pragma unroll
      for (int k = 0; k < V; ++k) mx = max(mx, __float_as_uint(v[k]) & 0x7fffffffu);   // a NaN is the largest and stays
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    largest[p] = max(mx, __float_as_uint(F8_FLOOR));
    all = max(all, largest[p]);
  }
  if (SQUARE) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = max(all, __shfl_xor_sync(0xffffffffu, all, o));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, warp_max[w]);
    if (threadIdx.x == 0) a.scales[(long long)blockIdx.x * gridDim.y + blockIdx.y] = __fdiv_rn(__uint_as_float(all), F8_TOP);
  }
  const float square_inv = __fdiv_rn(F8_TOP, __uint_as_float(all));
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = p * AT_ONCE + r0;
    const long long row = row0 + r;
    const float inv = SQUARE ? square_inv : __fdiv_rn(F8_TOP, __uint_as_float(largest[p]));
    if (!SQUARE && lane == 0) row_scale[r] = __fdiv_rn(__uint_as_float(largest[p]), F8_TOP);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int col = col0 + (s * L + lane) * V;
      if (row < a.rows && col < a.cols) {
        float v[V];
        sb_unpack<T, V>(in[p][s], v);
        uint8_t* to = a.codes + row * a.ldc + col;
        if constexpr (V == 1) {
          *to = (uint8_t)f8_pack2(v[0] * inv, 0.f);
        } else {
          SbPack<uint16_t, V / 2> c;
#pragma unroll
          for (int k = 0; k < V; k += 2) c.v[k / 2] = (uint16_t)f8_pack2(v[k] * inv, v[k + 1] * inv);
          *reinterpret_cast<SbPack<uint16_t, V / 2>*>(to) = c;
        }
      }
    }
  }
  if (!SQUARE) {
    __syncthreads();
    for (int r = threadIdx.x; r < ROWS; r += 256)
      if (row0 + r < a.rows) a.scales[(long long)blockIdx.y * a.rows + row0 + r] = row_scale[r];
  }
}

template <typename T, int V>
int launch_quantize(const QuantArgs& a, int block_rows, cudaStream_t s) {
  const int across = (a.cols + F8_BLOCK - 1) / F8_BLOCK;
  const int rows = block_rows == 1 ? 64 : 128;
  const dim3 grid((unsigned)((a.rows + rows - 1) / rows), (unsigned)across);
  if (block_rows == 1) SB_CUDA(sb_launch(quantize_fp8_kernel<T, V, 64, false>, grid, dim3(256), 0, s, 1, a));
  else SB_CUDA(sb_launch(quantize_fp8_kernel<T, V, 128, true>, grid, dim3(256), 0, s, 1, a));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T>
int launch_quantize_width(const QuantArgs& a, int block_rows, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(T);
  const int v = sb_vector_width(a.x, a.ldx, a.cols, sizeof(T), MOST);
  if (v == MOST && sb_vector_width(a.codes, a.ldc, a.cols, 1, MOST) == MOST) return launch_quantize<T, MOST>(a, block_rows, s);
  return launch_quantize<T, 1>(a, block_rows, s);
}

// ------------------------------- product -----------------------------------------
struct F8Args {
  const uint8_t* a;
  const uint8_t* w;
  const float* sa;               // [blocks of K][M]
  const float* sw;               // [blocks of N][blocks of K]
  const float* bias;
  void* c;
  long long lda, ldw, ldc;
  int m, n, k, k_blocks;
  int relu, out_dtype;
};

__device__ __forceinline__ void f8_store(const F8Args& g, long long row, int col, float v) {
  if (g.bias) v += g.bias[col];
  if (g.relu) v = fmaxf(v, 0.f);
  const long long at = row * g.ldc + col;
  if (g.out_dtype == SB_F32) ((float*)g.c)[at] = v;
  else if (g.out_dtype == SB_BF16) ((__nv_bfloat16*)g.c)[at] = __float2bfloat16_rn(v);
  else ((__half*)g.c)[at] = __float2half_rn(v);
}

// Any sizes, pitches and alignment: 64 x 64 tiles on the CUDA cores, 4 x 4 values per thread, 16 elements of K at a time.
__global__ void __launch_bounds__(256) gemm_fp8_simple_kernel(F8Args g) {
  __shared__ float ta[16][65], tw[16][65];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const long long row0 = (long long)blockIdx.x * 64;
  const int col0 = blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int b = 0; b < g.k_blocks; ++b) {
    float part[4][4] = {};
    const int k_end = min(g.k, (b + 1) * F8_BLOCK);
    for (int k0 = b * F8_BLOCK; k0 < k_end; k0 += 16) {
      __syncthreads();
      for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int k = i & 15, r = i >> 4;
        ta[k][r] = row0 + r < g.m && k0 + k < k_end ? f8_to_f32(g.a[(row0 + r) * g.lda + k0 + k]) : 0.f;
        tw[k][r] = col0 + r < g.n && k0 + k < k_end ? f8_to_f32(g.w[(long long)(col0 + r) * g.ldw + k0 + k]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] += ta[k][ty + 16 * i] * tw[k][tx + 16 * j];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = row0 + ty + 16 * i;
      const float sa = row < g.m ? g.sa[(long long)b * g.m + row] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = col0 + tx + 16 * j;
        const float sw = col < g.n ? g.sw[(long long)(col / F8_BLOCK) * g.k_blocks + b] : 0.f;
        acc[i][j] += part[i][j] * (sa * sw);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long row = row0 + ty + 16 * i;
      const int col = col0 + tx + 16 * j;
      if (row < g.m && col < g.n) f8_store(g, row, col, acc[i][j]);
    }
}

bool f8_aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

extern "C" {

int sb_quantize_fp8(const void* x, long long ldx, int dtype, long long rows, int cols, int block_rows, uint8_t* codes, long long ldc,
                    float* scales, void* stream) {
  const char* who = "sb_quantize_fp8";
  if (rows < 0 || cols < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (block_rows != 1 && block_rows != F8_BLOCK) return sb_fail(SB_ERR_UNSUPPORTED, "%s: blocks are 1 x 128 or 128 x 128 (got %d rows)", who, block_rows);
  if (dtype != SB_F32 && dtype != SB_BF16 && dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: storage types are f32, bf16 and f16 (got %d)", who, dtype);
  if (rows == 0 || cols == 0) return SB_OK;
  if (!x || !codes || !scales) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ldx < cols || ldc < cols) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than the %d columns", who, cols);
  if ((cols + F8_BLOCK - 1) / F8_BLOCK > 65535 || rows > 0x7fffffffLL)
    return sb_fail(SB_ERR_TOO_LARGE, "%s: at most 2^31 - 1 rows and 65535 blocks across", who);
  if (!f8_aligned(x, sb_dtype_size(dtype)) || !f8_aligned(scales, 4))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  QuantArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x; a.codes = codes; a.scales = scales; a.rows = rows; a.ldx = ldx; a.ldc = ldc; a.cols = cols;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_F32 ? launch_quantize_width<float>(a, block_rows, s)
         : dtype == SB_BF16 ? launch_quantize_width<__nv_bfloat16>(a, block_rows, s) : launch_quantize_width<__half>(a, block_rows, s);
}

int sb_matmul_fp8(const uint8_t* a, long long lda, const float* a_scales, const uint8_t* w, long long ldw, const float* w_scales, void* c,
                  long long ldc, int m, int n, int k, int out_dtype, int epilogue, const float* bias, void* stream) {
  const char* who = "sb_matmul_fp8";
  if (m < 0 || n < 0 || k < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (out_dtype != SB_F32 && out_dtype != SB_BF16 && out_dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: outputs are f32, bf16 or f16 (got %d)", who, out_dtype);
  if (epilogue & ~(SB_EPI_BIAS | SB_EPI_RELU)) return sb_fail(SB_ERR_UNSUPPORTED, "%s: epilogues are bias and ReLU", who);
  if (m == 0 || n == 0) return SB_OK;
  if (!c || ((epilogue & SB_EPI_BIAS) && !bias) || (k > 0 && (!a || !w || !a_scales || !w_scales)))
    return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ldc < n || (k > 0 && (lda < k || ldw < k))) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than its rows", who);
  if ((n + 63) / 64 > 65535) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most %d columns", who, 64 * 65535);
  if (!f8_aligned(c, sb_dtype_size(out_dtype)) || !f8_aligned(a_scales, 4) || !f8_aligned(w_scales, 4) || !f8_aligned(bias, 4))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  F8Args g;
  memset(&g, 0, sizeof(g));
  g.a = a; g.w = w; g.sa = a_scales; g.sw = w_scales; g.bias = (epilogue & SB_EPI_BIAS) ? bias : nullptr; g.c = c;
  g.lda = lda; g.ldw = ldw; g.ldc = ldc; g.m = m; g.n = n; g.k = k; g.k_blocks = (k + F8_BLOCK - 1) / F8_BLOCK;
  g.relu = (epilogue & SB_EPI_RELU) ? 1 : 0; g.out_dtype = out_dtype;
  const dim3 grid((unsigned)((m + 63) / 64), (unsigned)((n + 63) / 64));
  SB_CUDA(sb_launch(gemm_fp8_simple_kernel, grid, dim3(256), 0, (cudaStream_t)stream, 1, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

}  // extern "C"
