// Products with weights in 4 bits and a scale per group of 32, 64 or 128 along a row: w = scale (q - 8), q in 0 .. 15.
//
// Codes [n, ceil(k / 2)] hold two weights in a byte, the even one in the low half; scales are [ceil(k / group), n], so that
// those that a tile of rows needs together are neighbours.  c = a w^T of few rows of `a` reads every weight once, and its
// time is that of their bytes.
#include "common.cuh"
#include "few_rows.cuh"
#include "vector_io.cuh"

#include <type_traits>

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
    const S scale = sb_from_f32<S>(fminf(largest / 7.f, Int4ScaleMax<S>::value));
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

// Eight codes as four pairs of 16-bit numbers q - 8, (0, 4), (1, 5), (2, 6), (3, 7): with the bits of 1024 (f16) or 128 (bf16) above them a
// code is the number 1024 + q or 128 + q, from which 1032 or 136 is taken without rounding.
template <typename T>
__device__ __forceinline__ void int4_pairs(uint32_t w, uint32_t* out) {
  constexpr bool HALF = std::is_same<T, __half>::value;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | (HALF ? 0x64006400u : 0x43004300u);
    if (HALF) {
      const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __floats2half2_rn(1032.f, 1032.f));
      memcpy(&out[i], &r, 4);
    } else {
      const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __floats2bfloat162_rn(136.f, 136.f));
      memcpy(&out[i], &r, 4);
    }
  }
}

constexpr int I4_WARPS = 8;
struct Int4Few {
  int whole_words;               // codes can be read by the words of a lane
  int whole_rows;                // rows of a start on 16 bytes
  int scale_dtype;
  int blocks;                    // of a cluster
};

// A scale from its 16 bits.
__device__ __forceinline__ float int4_scale(SbWords<2> s, int dtype) {
  const float half = __half2float(__ushort_as_half(s.v));
  return dtype == SB_BF16 ? __uint_as_float((uint32_t)s.v << 16) : half;
}

// V words (8 codes each) from column k0 on, byte by byte; what lies beyond k holds anything, since the rows of a are zero there.
template <int V>
__device__ __forceinline__ void int4_bytes(uint32_t* out, const uint8_t* row, int k0, int k) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    uint32_t word = 0u;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int at = k0 + 8 * v + 2 * b;
      if (at < k) word |= (uint32_t)row[at / 2] << (8 * b);
    }
    out[v] = word;
  }
}
// Eight elements of a row of a one by one, zeros beyond k.
template <typename T>
__device__ __forceinline__ uint4 int4_eight(const T* row, int k0, int k) {
  uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k0 + i < k) v[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[k0 + i] << (16 * (i % 2));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A block has 16 RT rows of w and up to 8 NT rows of a; its warps take groups in turn, UNROLL of them on their way at a time, and the blocks
// of a cluster share K.  The codes of a lane (32 / 4 = 8 per word) are of one group in all four lanes of a row, so the products of a word
// are summed as whole numbers times elements of a and scaled as sums.  All partial sums are joined in a fixed order.
template <typename T, int G, int NT, int RT>
__global__ void __launch_bounds__(32 * I4_WARPS, NT <= 4 ? 2 : 1) gemm_int4_kernel(Int4Args p, Int4Few q) {
  constexpr int V = G / 32, UNROLL = RT == 1 ? (V == 1 ? 8 : 4) : V == 1 ? 2 : 1, ROWS = 16 * RT, COLS = 8 * NT, PITCH = COLS + 1;
  extern __shared__ float i4_smem[];
  float* part = i4_smem;                               // [warps][16][PITCH]
  float* sums = i4_smem + I4_WARPS * 16 * PITCH;       // [ROWS][PITCH], this block's
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int blocks = q.blocks, rank = blockIdx.x % blocks;
  const int r0 = blockIdx.x / blocks * ROWS, n0 = blockIdx.y * COLS;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const T* a = reinterpret_cast<const T*>(p.a);
  const bool whole_words = q.whole_words != 0, whole_rows = q.whole_rows != 0;
  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[r][n][j] = 0.f;
  const int groups = (p.k + G - 1) / G;
  for (int b0 = rank + blocks * warp; b0 < groups; b0 += blocks * I4_WARPS * UNROLL) {
    SbWords<4 * V> words[UNROLL][RT][2];
    SbWords<2> raw[UNROLL][RT][2];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int b = b0 + u * blocks * I4_WARPS;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = r0 + 16 * r + g + 8 * h;
          const bool there = b < groups && row < p.n;
          memset(&words[u][r][h], 0, 4 * V);
          sb_load_words(words[u][r][h], p.codes + (long long)(there ? row : 0) * p.ldw + (b * G + 8 * V * t) / 2, there && whole_words && (b + 1) * G <= p.k);
          raw[u][r][h].v = 0;
          sb_load_kept(raw[u][r][h], reinterpret_cast<const uint16_t*>(p.scales) + (there ? (long long)b * p.n + row : 0), there);
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int b = b0 + u * blocks * I4_WARPS;
      if (b >= groups) break;
      const bool whole = (b + 1) * G <= p.k;
      if (!whole_words || !whole) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = r0 + 16 * r + g + 8 * h;
            uint32_t w[V];
            if (row < p.n) {
              int4_bytes<V>(w, p.codes + (long long)row * p.ldw, b * G + 8 * V * t, p.k);
              memcpy(&words[u][r][h], w, 4 * V);
            }
          }
      }
      float scale[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) scale[r][h] = int4_scale(raw[u][r][h], q.scale_dtype);
      // Words of a at a time: all of a group's where there is room for them.
      constexpr int AHEAD = NT * V <= 4 ? V : 1;
#pragma unroll
      for (int v0 = 0; v0 < V; v0 += AHEAD) {
        SbWords<16> x[AHEAD][NT];
        if (whole_rows && whole) {
#pragma unroll
          for (int v = 0; v < AHEAD; ++v)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int row = n0 + 8 * n + g;
              x[v][n].v = make_uint4(0u, 0u, 0u, 0u);
              sb_load_kept(x[v][n], a + (long long)row * p.lda + b * G + 8 * (V * t + v0 + v), row < p.m);
            }
        } else {
#pragma unroll
          for (int v = 0; v < AHEAD; ++v)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int row = n0 + 8 * n + g;
              x[v][n].v = row < p.m ? int4_eight<T>(a + (long long)row * p.lda, b * G + 8 * (V * t + v0 + v), p.k) : make_uint4(0u, 0u, 0u, 0u);
            }
        }
#pragma unroll
        for (int v = 0; v < AHEAD; ++v) {
          uint32_t w[RT][2][4];
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t codes[V];
              memcpy(codes, &words[u][r][h], 4 * V);
              int4_pairs<T>(codes[v0 + v], w[r][h]);
            }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 e = x[v][n].v;
            const uint32_t x04 = __byte_perm(e.x, e.z, 0x5410), x15 = __byte_perm(e.x, e.z, 0x7632), x26 = __byte_perm(e.y, e.w, 0x5410),
                           x37 = __byte_perm(e.y, e.w, 0x7632);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16x8x16<T>(c, w[r][0][0], w[r][1][0], w[r][0][1], w[r][1][1], x04, x15);
              mma_16x8x16<T>(c, w[r][0][2], w[r][1][2], w[r][0][3], w[r][1][3], x26, x37);
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[r][n][j] = fmaf(scale[r][j >> 1], c[j], acc[r][n][j]);
            }
          }
        }
      }
    }
  }
  for (int r = 0; r < RT; ++r) {
#pragma unroll
    for (int s = 0; s < RT; ++s)
      if (s == r) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[(warp * 16 + g + 8 * (j >> 1)) * PITCH + 8 * n + 2 * t + (j & 1)] = acc[s][n][j];
      }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * COLS; e += 32 * I4_WARPS) {
      const int row = e % 16, col = e / 16;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < I4_WARPS; ++w) sum += part[(w * 16 + row) * PITCH + col];
      sums[(16 * r + row) * PITCH + col] = sum;
    }
    __syncthreads();
  }
  if (blocks > 1) cluster_sync_all();
  for (int e = threadIdx.x + 32 * I4_WARPS * rank; e < ROWS * COLS; e += 32 * I4_WARPS * blocks) {
    const int row = e % ROWS, col = e / ROWS;
    if (r0 + row >= p.n || n0 + col >= p.m) continue;
    float sum = 0.f;
    if (blocks == 1) {
      sum = sums[row * PITCH + col];
    } else {
      const uint32_t at = smem_u32(&sums[row * PITCH + col]);
      for (int b = 0; b < blocks; ++b) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(at, (uint32_t)b)) : "memory");
        sum += v;
      }
    }
    int4_store(p, n0 + col, r0 + row, sum);
  }
  __syncwarp();
  if (blocks > 1) cluster_sync_all();                  // no block leaves while another reads its sums
}

int int4_args_ok(const char* who, long long n, int k, int group, int scale_dtype) {
  if (n < 0 || k < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (group != 32 && group != 64 && group != 128) return sb_fail(SB_ERR_UNSUPPORTED, "%s: groups of 32, 64 or 128 (got %d)", who, group);
  if (scale_dtype != SB_BF16 && scale_dtype != SB_F16) return sb_fail(SB_ERR_UNSUPPORTED, "%s: scales are bf16 or f16 (got %d)", who, scale_dtype);
  if (n > (1LL << 30) || k > (1 << 30)) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most 2^30 rows and columns", who);
  return SB_OK;
}

bool int4_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (size_t)sb_dtype_size(dtype) == 0; }

template <typename T, int G, int NT, int RT>
int launch_int4(const Int4Args& p, Int4Few q, cudaStream_t s) {
  constexpr int PITCH = 8 * NT + 1, BYTES = (I4_WARPS * 16 + 16 * RT) * PITCH * 4;
  const long long tiles = ((long long)p.n + 16 * RT - 1) / (16 * RT), down = ((long long)p.m + 8 * NT - 1) / (8 * NT);
  // Blocks that share K until there are three for every two SMs, each warp with a group of its own.
  int blocks = 1;
  while (blocks < 8 && 2 * tiles * down * blocks < 3LL * sb_sm_count() && (p.k + G - 1) / G >= 2 * blocks * I4_WARPS) blocks *= 2;
  static std::atomic<bool> ready[64];
  if (BYTES > 48 * 1024) {
    const int rc = sb_allow_smem(gemm_int4_kernel<T, G, NT, RT>, BYTES, ready);
    if (rc != SB_OK) return rc;
  }
  q.blocks = blocks;
  SB_CUDA(sb_launch(gemm_int4_kernel<T, G, NT, RT>, dim3((unsigned)(tiles * blocks), (unsigned)down), dim3(32 * I4_WARPS), (size_t)BYTES, s, blocks, p, q));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int G>
int launch_int4(const Int4Args& p, const Int4Few& q, cudaStream_t s) {
  if (p.m <= 2) return launch_int4<T, G, 1, 1>(p, q, s);
  if (p.m <= 8) return launch_int4<T, G, 1, 4>(p, q, s);
  if (p.m <= 16) return launch_int4<T, G, 2, 4>(p, q, s);
  if (p.m <= 32) return launch_int4<T, G, 4, 2>(p, q, s);
  return launch_int4<T, G, 8, 2>(p, q, s);
}

template <typename T>
int launch_int4(const Int4Args& p, int scale_dtype, cudaStream_t s) {
  Int4Few q;
  const int lane_bytes = p.group / 8;
  q.whole_words = (reinterpret_cast<uintptr_t>(p.codes) % lane_bytes == 0 && p.ldw % lane_bytes == 0) ? 1 : 0;
  q.whole_rows = (reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && (p.m == 1 || p.lda % 8 == 0)) ? 1 : 0;
  q.scale_dtype = scale_dtype;
  return p.group == 32 ? launch_int4<T, 32>(p, q, s) : p.group == 64 ? launch_int4<T, 64>(p, q, s) : launch_int4<T, 128>(p, q, s);
}

template <typename T>
int launch_quantize_int4(const QuantInt4Args& p, int scale_dtype, cudaStream_t s) {
  const long long blocks = (p.n * p.groups + 7) / 8, most = 32LL * sb_sm_count();
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (scale_dtype == SB_BF16) SB_CUDA(sb_launch(quantize_int4_kernel<T, __nv_bfloat16>, grid, dim3(256), 0, s, 1, p));
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
  return scale_dtype == SB_BF16 ? launch_dequantize_int4<__nv_bfloat16>(codes, ldw, scales, out, ldo, out_dtype, n, k, group, s)
                                : launch_dequantize_int4<__half>(codes, ldw, scales, out, ldo, out_dtype, n, k, group, s);
}

int sb_matmul_int4(const void* a, long long lda, int dtype, const uint8_t* codes, long long ldw, const void* scales, int scale_dtype, void* c,
                   long long ldc, int m, int n, int k, int group, int out_dtype, int epilogue, const float* bias, void* stream) {
  const char* who = "sb_matmul_int4";
  int rc = int4_args_ok(who, n, k, group, scale_dtype);
  if (rc != SB_OK) return rc;
  if (m < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (m > (1 << 22) - 64) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most 2^22 - 64 rows", who);
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
