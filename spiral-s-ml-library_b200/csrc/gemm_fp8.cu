// Products in 8-bit floating point (E4M3) with an fp32 scale per block of 128, and the quantisation that makes their
// operands.
//
//   codes = round(x * (448 / a)), scale = a / 448, a = max |x| over a block (1 x 128 or 128 x 128), at least 2^-100
//   C[m, n] = sum over blocks b of K   sa[b, m] * sw[n / 128, b] * sum over k in b of A[m, k] W[n, k]   (+ bias, ReLU)
//
// The sum inside a block and the sum over blocks are fp32.
#include "common.cuh"
#include "vector_io.cuh"

#include <math.h>

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
  unsigned across;               // blocks of 128 columns
};

// ------------------------------ quantisation -------------------------------------
// The bits of the largest magnitude in a pack: as integers, so that a NaN is the largest and stays; 16-bit types two at a
// time.  fp32 bits come back from `f8_largest_bits`.
template <typename T, int V>
__device__ __forceinline__ uint32_t f8_larger(const SbPack<T, V>& p, uint32_t largest) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    uint32_t w[V / 2];
    memcpy(w, &p, sizeof(w));
#pragma unroll
    for (int k = 0; k < V / 2; ++k) asm("max.u16x2 %0, %0, %1;" : "+r"(largest) : "r"(w[k] & 0x7fff7fffu));
    return largest;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) largest = max(largest, __float_as_uint(sb_to_f32<T>(p.v[k])) & 0x7fffffffu);
    return largest;
  }
}
template <typename T, int V>
__device__ __forceinline__ uint32_t f8_largest_bits(uint32_t largest) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    const uint16_t h = (uint16_t)max(largest & 0xffffu, largest >> 16);
    T v;
    memcpy(&v, &h, sizeof(v));
    return __float_as_uint(sb_to_f32<T>(v));
  } else {
    return largest;
  }
}

// A block of 256 threads per ROWS x 128 tile of x, which stays in registers between the search for its largest magnitude
// and the rounding; L lanes share a row, V neighbouring elements each.  SQUARE: one scale for the tile, else one per row.
// Bound by issue (products, roundings and packing: three quarters of the slots) more than by memory: 16384 x 4096 bf16 40 us,
// 5.0 TB/s, 65536 x 1024 f16 39.5 (42 with the magnitudes one at a time).  One scale per tile, whose rows all wait for the largest
// magnitude: 16384 x 4096 bf16 54 us, 3.7 TB/s; 4096 x 4096 fp32 22, 3.7 TB/s.
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
  // Tiles that are neighbours in a row run at the same time: their pieces of x are neighbours in memory.
  const long long up = blockIdx.x / a.across;
  const int over = (int)(blockIdx.x - up * a.across);
  const long long row0 = up * ROWS;
  const int col0 = over * F8_BLOCK;
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
    for (int s = 0; s < STEPS; ++s) mx = f8_larger<T, V>(in[p][s], mx);
    mx = f8_largest_bits<T, V>(mx);
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
    if (threadIdx.x == 0) a.scales[blockIdx.x] = __fdiv_rn(__uint_as_float(all), F8_TOP);
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
          const unsigned long long inv2 = pack_f32x2(inv, inv);
#pragma unroll
          for (int k = 0; k < V; k += 2) {
            float lo, hi;
            unpack_f32x2(mul_f32x2(pack_f32x2(v[k], v[k + 1]), inv2), lo, hi);
            c.v[k / 2] = (uint16_t)f8_pack2(lo, hi);
          }
          *reinterpret_cast<SbPack<uint16_t, V / 2>*>(to) = c;
        }
      }
    }
  }
  if (!SQUARE) {
    __syncthreads();
    for (int r = threadIdx.x; r < ROWS; r += 256)
      if (row0 + r < a.rows) a.scales[over * a.rows + row0 + r] = row_scale[r];
  }
}

template <typename T, int V>
int launch_quantize(const QuantArgs& a, int block_rows, cudaStream_t s) {
  const int rows = block_rows == 1 ? 64 : 128;
  const long long tiles = (a.rows + rows - 1) / rows * a.across;
  if (tiles > 0x7fffffffLL) return sb_fail(SB_ERR_TOO_LARGE, "sb_quantize_fp8: more than 2^31 - 1 tiles");
  const dim3 grid((unsigned)tiles);
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

// The product of a block's two scales, or, where that is no normal number although both are (1e-20 each are enough), two factors that
// are taken one after the other: values beside which neither step leaves the range unless the result does.  A scale of at most
// 2^-100 / 448 is that of a block of zeros, or of magnitudes of at most 2^-100: what it gives below the normal range may be lost.
struct F8Scale {
  float first, second;
};
__device__ __forceinline__ bool f8_unsafe(float sa, float sw) {
  const float product = sa * sw;
  return (product < 1.17549435e-38f || product == INFINITY) && fminf(sa, sw) > F8_FLOOR / F8_TOP && fmaxf(sa, sw) < INFINITY;
}
// Two instructions and one register of a product of scales: F8_OUTSIDE and more where it is no normal number.
constexpr uint32_t F8_OUTSIDE = 0x7f000000u;
__device__ __forceinline__ uint32_t f8_outside(float product) { return __float_as_uint(product) - 0x00800000u; }
__device__ __forceinline__ F8Scale f8_scale(float sa, float sw) {
  const float product = sa * sw;
  if (!f8_unsafe(sa, sw)) return {1.f, product};
  return (sa >= sw) == (product < 1.f) ? F8Scale{sa, sw} : F8Scale{sw, sa};   // the larger one first where they shrink
}

__device__ __forceinline__ void f8_store(const F8Args& g, long long row, int col, float v) {
  if (g.bias) v += g.bias[col];
  if (g.relu) v = fmaxf(v, 0.f);
  const long long at = row * g.ldc + col;
  if (g.out_dtype == SB_F32) ((float*)g.c)[at] = v;
  else if (g.out_dtype == SB_BF16) ((__nv_bfloat16*)g.c)[at] = __float2bfloat16_rn(v);
  else ((__half*)g.c)[at] = __float2half_rn(v);
}

// Whether a row and a block of columns have such scales in blocks `begin` .. `end` - 1 of K; LOADS of each on their way at a time.
template <int LOADS>
__device__ __forceinline__ bool f8_row_unsafe(const F8Args& g, long long row, int n_block, int begin, int end) {
  bool unsafe = false;
#pragma unroll LOADS
  for (int b = begin; b < end; ++b) unsafe |= f8_unsafe(g.sa[(long long)b * g.m + row], g.sw[(long long)n_block * g.k_blocks + b]);
  return unsafe;
}
// Such a row's product with a row of W over these blocks, by one thread and as slow as it is rare.  The rows of codes start on 16 bytes.
__device__ __forceinline__ float f8_dot(const F8Args& g, long long row, int col, int begin, int end) {
  const uint8_t *a = g.a + row * g.lda, *w = g.w + (long long)col * g.ldw;
  float sum = 0.f;
#pragma unroll 1
  for (int b = begin; b < end; ++b) {
    float part = 0.f;
    const int last = min(g.k, (b + 1) * F8_BLOCK);
    int k = b * F8_BLOCK;
#pragma unroll 1
    for (; k + 16 <= last; k += 16) {
      const SbPack<uint16_t, 8> pa = *reinterpret_cast<const SbPack<uint16_t, 8>*>(a + k), pw = *reinterpret_cast<const SbPack<uint16_t, 8>*>(w + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 va = f8_unpack2(pa.v[i]), vw = f8_unpack2(pw.v[i]);
        part = fmaf(va.y, vw.y, fmaf(va.x, vw.x, part));
      }
    }
#pragma unroll 1
    for (; k < last; ++k) part = fmaf(f8_to_f32(a[k]), f8_to_f32(w[k]), part);
    const F8Scale f = f8_scale(g.sa[(long long)b * g.m + row], g.sw[(long long)(col / F8_BLOCK) * g.k_blocks + b]);
    sum = fmaf(part * f.first, f.second, sum);
  }
  return sum;
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
        const F8Scale s = f8_scale(sa, sw);
        acc[i][j] = fmaf(part[i][j] * s.first, s.second, acc[i][j]);
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


// The tensor-core form: persistent CTAs, a tile of 128 x BN values each.  A stage of the ring is one 128-byte block of K of
// both operands, brought by TMA.  The scales change with every block of K, so every block's MMAs start a fresh accumulator
// in TMEM, and eight warps add it, times its two scales, to sums in registers (packed fp32 multiply-adds) while the MMAs of
// the next block run into another accumulator.  A thread owns one row and half of the columns, which lie in one 128-block
// of N: the product of the scales is one number per thread and block.  At BN = 256 the two halves of the columns are
// products of their own with two accumulators each, so that the adding warps of a half wait for their own MMAs only.
//
// Bound by the operands' way from L2 into shared memory: at BN = 256 a block is 48 KB in 0.55 us per SM, 13 TB/s over the chip
// (8192^3: 530 us, 2070 TFLOP/s, the same without the multiply-adds).  Pairs of CTAs (cta_group::2, 256 x 256) load a third
// less and were slower, 16384 x 4096 x 4096 in short bursts 320 us against 271: the round trip from the MMAs over both CTAs' adding
// warps back to the issuer is longer than two accumulators cover.  Four stages instead of three 288 us, sixteen adding warps, whose
// 112 registers spill, 327 (in pairs), measured alike.  Back to back, that is under the power cap, this form takes 275 us on codes of
// normal values and 308 on codes of random bits.
constexpr int F8_STAGES_MAX = 12;
constexpr int F8_WARPS = 8;                                  // that add
constexpr int F8_FIRST = 4;                                  // the first of them: warp 0 loads, warp 1 issues
constexpr int F8_THREADS = 32 * (F8_FIRST + F8_WARPS);
constexpr int F8_SMEM = 225 * 1024;
constexpr uint32_t F8_BOX = 4096;                            // a warp's staging box: 32 rows x 128 bytes
// Boxes of a warp: where it fills several per tile, one is read by its store while the next is filled.
__host__ __device__ constexpr int f8_boxes(int bn) { return bn == 256 ? 2 : 1; }
constexpr int F8_AHEAD = 4;                                  // blocks whose scales are on their way or in use
constexpr uint32_t F8_SCALES = F8_WARPS * 32 * 8;            // bytes of one block's: a pair per adding thread

__device__ __forceinline__ void f8_mma(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate, bool issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"((uint32_t)issue) : "memory");
}
// One block of K: four MMAs of 32 elements into a fresh accumulator.
__device__ __forceinline__ void f8_block(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                         bool issue) {
  f8_mma(d, a_lo, a_hi, b_lo, b_hi, idesc, 0u, issue);
  f8_mma(d, a_lo + 2u, a_hi, b_lo + 2u, b_hi, idesc, 1u, issue);
  f8_mma(d, a_lo + 4u, a_hi, b_lo + 4u, b_hi, idesc, 1u, issue);
  f8_mma(d, a_lo + 6u, a_hi, b_lo + 6u, b_hi, idesc, 1u, issue);
}
// kind::f8f6f4, E4M3 x E4M3 (formats 0), fp32 accumulator, M = 128; the fields are those of sb_umma_idesc.
__host__ __device__ constexpr uint32_t f8_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24); }

struct F8Plan {
  int stages, tiles_m, tiles_n, tiles;
  int tma_store;
};

__device__ __forceinline__ void f8_tile(const F8Plan& p, int tile, int& m_blk, int& n_blk) {
  constexpr int GROUP = 8;                                   // tiles that run at the same time share operands through L2
  const int per_group = GROUP * p.tiles_n;
  const int g = tile / per_group;
  const int rows = min(GROUP, p.tiles_m - g * GROUP);
  const int r = tile - g * per_group;
  m_blk = g * GROUP + r % rows;
  n_blk = r / rows;
}

__shared__ int g_f8_abort;

__device__ __forceinline__ void f8_copy4(uint32_t dst, const float* src, uint32_t bytes) {   // bytes 0: a zero is written
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float f8_lds(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
// N columns of an accumulator added to the sums: sum += scale * part.
template <int N>
__device__ __forceinline__ void f8_add(unsigned long long* sum, const uint32_t* part, unsigned long long scale) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j)
    fma_f32x2(sum[j], pack_f32x2(__uint_as_float(part[2 * j]), __uint_as_float(part[2 * j + 1])), scale);
}

// A box of 32 rows -> C with plain stores.  Lane l has columns l, l + 32, ... of a row; the places of 8 rows repeat with the
// swizzle, so the loop over rows knows them as constants.  9653 x 1114 x 1008 bf16 27 us (24 for the 1120 columns that TMA stores),
// 42 with an element's row and place worked out one by one; 3778 x 2006 x 2496 fp32 35.5 and 44.
template <typename O, int BOX_COLS>
__device__ __forceinline__ void f8_write_rows(O* to, long long ldc, int rows, int cols, uint32_t box, int lane) {
  constexpr int PER = 16 / sizeof(O), ROW_BYTES = BOX_COLS * sizeof(O), PIECES = ROW_BYTES / 16;
  constexpr int EACH = (BOX_COLS + 31) / 32;
  static_assert(BOX_COLS >= 32, "");
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += 8, to += 8 * ldc, box += 8 * ROW_BYTES) {
    O v[8][EACH];
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const uint32_t c = (uint32_t)(lane + 32 * e), key = ROW_BYTES == 128 ? (uint32_t)r : (uint32_t)(r >> 1) & 3u;
        const uint32_t at = box + (uint32_t)r * ROW_BYTES + (((c / PER ^ key) & (PIECES - 1)) << 4) + (c % PER) * (uint32_t)sizeof(O);
        if constexpr (sizeof(O) == 4) {
          uint32_t w;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
          memcpy(&v[r][e], &w, 4);
        } else {
          uint16_t w;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(at) : "memory");
          memcpy(&v[r][e], &w, 2);
        }
      }
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        if (r0 + r < rows && lane + 32 * e < cols) to[r * ldc + lane + 32 * e] = v[r][e];
  }
}

// Finished values of this warp's 32 rows and COLS columns (their biases in shared memory) -> C, a box of 32 rows x 128 bytes at a time (64 bytes where the
// columns are no more): by a TMA store, or by coalesced stores where C's rows are not whole 16-byte pieces.
template <typename O, int COLS, int BOXES>
__device__ __forceinline__ void f8_write(const F8Args& g, const CUtensorMap* tmap_c, bool tma, const unsigned long long* sum,
                                         long long row0, int col0, uint32_t boxes, uint32_t bias, int lane) {
  constexpr int BOX_COLS = COLS * sizeof(O) >= 128 ? 128 / sizeof(O) : COLS;
  constexpr int ROW_BYTES = BOX_COLS * sizeof(O), PIECES = ROW_BYTES / 16, PER = 16 / sizeof(O);
#pragma unroll
  for (int b = 0; b < COLS / BOX_COLS; ++b) {
    const int first = col0 + b * BOX_COLS;
    if (first >= g.n) return;
    const uint32_t box = boxes + (uint32_t)(b % BOXES) * F8_BOX;
    if (tma) {                                               // what this box held has been read: all of the tile before, or all but the last
      if (lane == 0) {
        if (b == 0) bulk_wait_group_read<0>();
        else bulk_wait_group_read<BOXES - 1>();
      }
      __syncwarp();
    }
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      float v[PER];
#pragma unroll
      for (int t = 0; t < PER; t += 2) unpack_f32x2(sum[(b * BOX_COLS + q * PER + t) / 2], v[t], v[t + 1]);
      if (g.bias) {
#pragma unroll
        for (int t = 0; t < PER; ++t) v[t] += f8_lds(bias + 4u * (uint32_t)(b * BOX_COLS + q * PER + t));
      }
      if (g.relu) {
#pragma unroll
        for (int t = 0; t < PER; ++t) v[t] = fmaxf(v[t], 0.f);
      }
      SbPack<O, PER> out;
#pragma unroll
      for (int t = 0; t < PER; ++t) out.v[t] = sb_from_f32<O>(v[t]);
      const uint32_t key = ROW_BYTES == 128 ? ((uint32_t)lane & 7u) : (((uint32_t)lane >> 1) & 3u);
      st_shared_v4(box + (uint32_t)lane * ROW_BYTES + ((((uint32_t)q ^ key) & (PIECES - 1)) << 4), *reinterpret_cast<const uint4*>(&out));
    }
    if (tma) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(tmap_c, box, first, (int)row0);
        bulk_commit_group();
      }
    } else {
      __syncwarp();
      f8_write_rows<O, BOX_COLS>((O*)g.c + row0 * g.ldc + first, g.ldc, (int)min(32LL, g.m - row0), g.n - first, box, lane);
      __syncwarp();
    }
  }
}

// An adding thread's rows with scales that f8_scale takes apart, written once more behind the last tile; the loop only notes that there
// may be some.  16384 x 4096 x 4096 308 us, 304 without, 8192^3 629 and 616; two steps in the loop 351, the whole look at a block's scales in the loop 331,
// by the two idle warps beside it 360 (their loads are in the way of the scales').
template <int BN>
__device__ __noinline__ void f8_again(const F8Args g, const F8Plan p) {
  const int t = threadIdx.x;
#pragma unroll 1
  for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
    int m_blk, n_blk;
    f8_tile(p, tile, m_blk, n_blk);
    const long long row = (long long)m_blk * 128 + (t & 127);  // of warp t / 32 modulo 4
    const int col = n_blk * BN + (t / 128 - F8_FIRST / 4) * (BN / 2);
    if (row >= g.m || col >= g.n || !f8_row_unsafe<16>(g, row, col / F8_BLOCK, 0, g.k_blocks)) continue;
#pragma unroll 1
    for (int j = col; j < min(g.n, col + BN / 2); ++j) f8_store(g, row, j, f8_dot(g, row, j, 0, g.k_blocks));
  }
}

template <int BN>
__global__ void __launch_bounds__(F8_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                const __grid_constant__ CUtensorMap tmap_c, const __grid_constant__ F8Args g, const __grid_constant__ F8Plan p) {
  constexpr int PARTS = BN == 256 ? 2 : 1;                   // products with accumulators of their own
  constexpr int PART_N = BN / PARTS;
  constexpr int DEPTH = 4 / PARTS;                           // accumulators of each
  constexpr int COLS = BN / 2;                               // of a thread
  constexpr int BOXES = f8_boxes(BN);
  constexpr uint32_t TMEM_COLS = PARTS * DEPTH * PART_N;
  constexpr uint32_t A_BYTES = 128 * F8_BLOCK, W_BYTES = BN * F8_BLOCK, STAGE = A_BYTES + W_BYTES;
  extern __shared__ uint8_t f8_smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[F8_STAGES_MAX], bar_empty[F8_STAGES_MAX], bar_acc_full[4], bar_acc_empty[4];
  __shared__ uint32_t tmem_slot;
  __shared__ int unsafe_scales;                              // noted by an adding warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t stage0 = (smem_u32(f8_smem_raw) + 1023u) & ~1023u;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), F8_WARPS / PARTS);
    }
    g_f8_abort = 0;
    unsafe_scales = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &g_f8_abort;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const bool one = elect_one_lane();
  // The 384 threads are launched with 168 registers each: 128 x 40 + 256 x 232 = 384 x 168.
  if (warp < F8_FIRST) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      int m_blk, n_blk;
      f8_tile(p, tile, m_blk, n_blk);
      for (int kb = 0; kb < g.k_blocks; ++kb) {
        if (!mbar_wait_warp(empty0 + 8u * (uint32_t)stage, phase ^ 1u, abortp, SB_SITE_PRODUCER_EMPTY)) {
          ok = false;
          break;
        }
        const uint32_t at = stage0 + (uint32_t)stage * STAGE, full = full0 + 8u * (uint32_t)stage;
        if (one) mbar_arrive_expect_tx(full, STAGE);
        tma_load_2d(at, &tmap_a, kb * F8_BLOCK, m_blk * 128, full, one);
        tma_load_2d(at + A_BYTES, &tmap_w, kb * F8_BLOCK, n_blk * BN, full, one);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    const uint64_t a_desc = umma_smem_desc(stage0, 16u, 1024u, 2u), w_desc = umma_smem_desc(stage0 + A_BYTES, 16u, 1024u, 2u);
    const uint32_t a_hi = (uint32_t)(a_desc >> 32), w_hi = (uint32_t)(w_desc >> 32);
    const uint32_t a_lo0 = (uint32_t)a_desc, w_lo0 = (uint32_t)w_desc;
    const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
    const uint32_t acc_full0 = smem_u32(&bar_acc_full[0]), acc_empty0 = smem_u32(&bar_acc_empty[0]);
    uint32_t a_lo = a_lo0, w_lo = w_lo0;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      for (int kb = 0; ok && kb < g.k_blocks; ++kb) {
        ok = mbar_wait_warp(full0 + 8u * (uint32_t)stage, phase, abortp, SB_SITE_MMA_FULL);
#pragma unroll
        for (int h = 0; h < PARTS; ++h) {
          const uint32_t at = (uint32_t)(PARTS * acc + h);
          if (ok) ok = mbar_wait_warp(acc_empty0 + 8u * at, acc_phase ^ 1u, abortp, SB_SITE_MMA_TMEM_EMPTY);
          if (!ok) break;
          tc_fence_after_sync();
          f8_block(tmem + at * PART_N, a_lo, a_hi, w_lo + (uint32_t)h * (W_BYTES / PARTS >> 4), w_hi, f8_idesc(PART_N), one);
          tc_commit(acc_full0 + 8u * at, one);
        }
        if (!ok) break;
        tc_commit(empty0 + 8u * (uint32_t)stage, one);
        a_lo += STAGE >> 4;
        w_lo += STAGE >> 4;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
          a_lo = a_lo0;
          w_lo = w_lo0;
        }
        if (++acc == DEPTH) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
    }
  } else if (warp >= F8_FIRST) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quad = warp & 3, half = (warp - F8_FIRST) >> 2;   // a warp reads the TMEM lanes of its number modulo 4
    const uint32_t boxes = stage0 + (uint32_t)p.stages * STAGE, box = boxes + (uint32_t)(warp - F8_FIRST) * F8_BOX * BOXES;
    const uint32_t scales = boxes + F8_WARPS * BOXES * F8_BOX + (uint32_t)(threadIdx.x - 32 * F8_FIRST) * 4u;
    const uint32_t bias = boxes + F8_WARPS * BOXES * F8_BOX + F8_AHEAD * F8_SCALES + (uint32_t)(warp - F8_FIRST) * 512u;
    const uint32_t acc_full0 = smem_u32(&bar_acc_full[0]), acc_empty0 = smem_u32(&bar_acc_empty[0]);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    // Each thread copies its own scales some blocks ahead, past the registers that the sums need; a tile's first ones before the
    // tile before is written (after it: 16384 x 4096 x 4096 292 us, now 275; 4096^3 88 and 80).
    long long row0 = 0;
    int col0 = 0, ahead = 0;
    bool inside = false;
    const float *sa = g.sa, *sw = g.sw;
    auto fetch = [&]() {
      if (ahead < g.k_blocks) {
        const uint32_t to = scales + (uint32_t)(ahead & (F8_AHEAD - 1)) * F8_SCALES;
        f8_copy4(to, sa, inside ? 4u : 0u);
        f8_copy4(to + F8_SCALES / 2, sw, inside ? 4u : 0u);
        sa += g.m;
        ++sw;
        ++ahead;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto begin = [&](int tile) {
      if (tile >= p.tiles) return;
      int m_blk, n_blk;
      f8_tile(p, tile, m_blk, n_blk);
      row0 = (long long)m_blk * 128 + quad * 32;
      col0 = n_blk * BN + half * COLS;
      inside = row0 + lane < g.m && col0 < g.n;
      sa = g.sa + (inside ? row0 + lane : 0);
      sw = g.sw + (inside ? (long long)(col0 / F8_BLOCK) * g.k_blocks : 0);
      ahead = 0;
#pragma unroll
      for (int i = 0; i < F8_AHEAD - 1; ++i) fetch();
    };
    begin(blockIdx.x);
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      unsigned long long sum[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) sum[j] = 0ull;
      uint32_t noted = 0u;
      // The columns' biases, for when the sums are done.  (Read there one by one they took 33 of 374 us at 16384 x 4096 x 4096.)
      if (g.bias)
#pragma unroll
        for (int j = lane; j < COLS; j += 32) f8_copy4(bias + 4u * (uint32_t)j, g.bias + (col0 + j < g.n ? col0 + j : 0), col0 + j < g.n ? 4u : 0u);
      for (int kb = 0; kb < g.k_blocks; ++kb) {
        const uint32_t at = (uint32_t)(PARTS == 2 ? 2 * acc + half : acc);
        fetch();
        ok = mbar_wait_warp(acc_full0 + 8u * at, acc_phase, abortp, SB_SITE_EPI_TMEM_FULL);
        if (!ok) break;
        asm volatile("cp.async.wait_group %0;" ::"n"(F8_AHEAD - 1) : "memory");
        const uint32_t from = scales + (uint32_t)(kb & (F8_AHEAD - 1)) * F8_SCALES;
        const float scale = f8_lds(from) * f8_lds(from + F8_SCALES / 2);
        noted = max(noted, f8_outside(scale));
        const unsigned long long scale2 = pack_f32x2(scale, scale);
        tc_fence_after_sync();
        const uint32_t t = tmem + ((uint32_t)(quad * 32) << 16) + at * PART_N + (PARTS == 2 ? 0u : (uint32_t)(half * COLS));
        uint32_t part[2][32];
        tmem_ld32(t, part[0]);
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c) {
          tmem_ld_wait32(part[c & 1]);
          if (c + 1 < COLS / 32) {
            tmem_ld32(t + (uint32_t)(c + 1) * 32u, part[(c + 1) & 1]);
          } else {                                           // all of the accumulator is in registers
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty0 + 8u * at);
          }
          f8_add<32>(sum + c * 16, part[c & 1], scale2);
        }
        if (++acc == DEPTH) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) break;
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      if (noted >= F8_OUTSIDE && inside) unsafe_scales = 1;
      const long long row = row0;
      const int col = col0;
      begin(tile + gridDim.x);
      if (row < g.m) {
        if (g.out_dtype == SB_F32) f8_write<float, COLS, BOXES>(g, &tmap_c, p.tma_store != 0, sum, row, col, box, bias, lane);
        else if (g.out_dtype == SB_BF16) f8_write<__nv_bfloat16, COLS, BOXES>(g, &tmap_c, p.tma_store != 0, sum, row, col, box, bias, lane);
        else f8_write<__half, COLS, BOXES>(g, &tmap_c, p.tma_store != 0, sum, row, col, box, bias, lane);
      }
      __syncwarp();                                          // the biases have been read
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
    if (ok && *(volatile int*)&unsafe_scales != 0) f8_again<BN>(g, p);
  }
  // After an expired wait copies and MMAs in flight get time to land before shared and tensor memory are released.
  tc_fence_before_sync();
  __syncthreads();
  if (*abortp != 0) {
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) { }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// The form for few rows of A, and for products whose tiles would leave most of the chip without work: the operands change
// places (M of the MMA is 128 rows of W, N is TN rows of A), and the blocks of K are shared by the CTAs of a cluster, each of
// which loads its part of W at once.  Their sums meet in shared memory: CTA r gets every CTA's sums of the r-th part of the
// columns and adds them in the order of the CTAs.  Bound by reading W, and by the launch.
constexpr int F8_FEW_THREADS = 192;                          // warps 0-3 add, warp 4 loads, warp 5 issues
constexpr int F8_FEW_BLOCKS = 64;                            // blocks of K per CTA at most: their scales are kept
constexpr int F8_FEW_STAGES = 8;

__device__ __forceinline__ void f8_prefetch(const CUtensorMap* tmap, int x, int y, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %3, 0;\n\t"
               "@q cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n\t}"
               ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"((uint32_t)issue) : "memory");
}
// Floats of this thread in another CTA's shared memory, and back from its own.
template <int N>
__device__ __forceinline__ void f8_send(uint32_t cluster_addr, const float* v) {
  if constexpr (N == 2) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_addr), "f"(v[0]), "f"(v[1]) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                   ::"r"(cluster_addr + 4u * (uint32_t)i), "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3]) : "memory");
  }
}

template <int TN, int SPLITS>
__global__ void __launch_bounds__(F8_FEW_THREADS, 1)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ F8Args g,
                    const int stages) {
  constexpr int DEPTH = 4;
  constexpr uint32_t TMEM_COLS = DEPTH * TN;
  constexpr uint32_t W_BYTES = 128 * F8_BLOCK, A_BYTES = TN * F8_BLOCK, STAGE = W_BYTES + A_BYTES;
  extern __shared__ uint8_t f8_smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[F8_FEW_STAGES], bar_empty[F8_FEW_STAGES], bar_acc_full[DEPTH], bar_acc_empty[DEPTH];
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float scales[F8_FEW_BLOCKS][TN];  // of A times of W
  __shared__ int unsafe_scales;                              // some of these products are no normal numbers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int PER = TN / SPLITS;                           // columns that a CTA finishes
  constexpr uint32_t PITCH = 4u * PER + (PER > 4 ? 16u : 0u);   // of a row's sums: 16-byte accesses without bank conflicts
  const int rank = blockIdx.x;                               // a cluster is the splits of one tile
  const int n0 = blockIdx.y * 128, m0 = blockIdx.z * TN;
  const int kb0 = (int)((long long)g.k_blocks * rank / SPLITS), kb1 = (int)((long long)g.k_blocks * (rank + 1) / SPLITS);
  const uint32_t stage0 = (smem_u32(f8_smem_raw) + 1023u) & ~1023u;
  const uint32_t meet = stage0 + (uint32_t)stages * STAGE;   // [SPLITS][128 rows of W][PER] sums
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < DEPTH; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), 4);
    }
    g_f8_abort = 0;
    unsafe_scales = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // Another CTA's shared memory may be written once that CTA has started: all arrive here, and wait before the first such write.
  if (SPLITS > 1) cluster_arrive_relaxed_all();
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &g_f8_abort;
  const bool one = elect_one_lane();
  // The weights' way to L2 can begin while the kernel before this one, which may be making A, still runs: L2 is where all
  // SMs meet, so a line that is written after the prefetch is not stale.
  if (warp == 4)
    for (int kb = kb0; kb < min(kb1, kb0 + stages); ++kb) f8_prefetch(&tmap_w, kb * F8_BLOCK, n0, one);
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  float sum[TN];
  bool again = false;                                        // some rows have scales that f8_scale takes apart
  if (warp == 4) {
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(empty0 + 8u * (uint32_t)stage, phase ^ 1u, abortp, SB_SITE_PRODUCER_EMPTY)) break;
      const uint32_t at = stage0 + (uint32_t)stage * STAGE, full = full0 + 8u * (uint32_t)stage;
      if (one) mbar_arrive_expect_tx(full, STAGE);
      tma_load_2d(at, &tmap_w, kb * F8_BLOCK, n0, full, one);
      tma_load_2d(at + W_BYTES, &tmap_a, kb * F8_BLOCK, m0, full, one);
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  } else if (warp == 5) {
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    const uint64_t w_desc = umma_smem_desc(stage0, 16u, 1024u, 2u), a_desc = umma_smem_desc(stage0 + W_BYTES, 16u, 1024u, 2u);
    const uint32_t w_hi = (uint32_t)(w_desc >> 32), a_hi = (uint32_t)(a_desc >> 32);
    const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
    const uint32_t acc_full0 = smem_u32(&bar_acc_full[0]), acc_empty0 = smem_u32(&bar_acc_empty[0]);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(acc_empty0 + 8u * (uint32_t)acc, acc_phase ^ 1u, abortp, SB_SITE_MMA_TMEM_EMPTY) ||
          !mbar_wait_warp(full0 + 8u * (uint32_t)stage, phase, abortp, SB_SITE_MMA_FULL))
        break;
      tc_fence_after_sync();
      const uint32_t step = (uint32_t)stage * (STAGE >> 4);
      f8_block(tmem + (uint32_t)(acc * TN), (uint32_t)w_desc + step, w_hi, (uint32_t)a_desc + step, a_hi, f8_idesc(TN), one);
      tc_commit(empty0 + 8u * (uint32_t)stage, one);
      tc_commit(acc_full0 + 8u * (uint32_t)acc, one);
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
      if (++acc == DEPTH) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  } else {
    for (int i = threadIdx.x; i < (kb1 - kb0) * TN; i += 128) {
      const int kb = i / TN, j = i % TN;
      const float va = m0 + j < g.m ? g.sa[(long long)(kb0 + kb) * g.m + m0 + j] : 0.f, vw = g.sw[(long long)blockIdx.y * g.k_blocks + kb0 + kb];
      scales[kb][j] = va * vw;
      if (f8_unsafe(va, vw)) unsafe_scales = 1;
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    again = unsafe_scales != 0;
    const uint32_t acc_full0 = smem_u32(&bar_acc_full[0]), acc_empty0 = smem_u32(&bar_acc_empty[0]);
    int acc = 0;
    uint32_t acc_phase = 0;
#pragma unroll
    for (int j = 0; j < TN; ++j) sum[j] = 0.f;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(acc_full0 + 8u * (uint32_t)acc, acc_phase, abortp, SB_SITE_EPI_TMEM_FULL)) break;
      tc_fence_after_sync();
      const uint32_t t = tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)(acc * TN);
      uint32_t part[TN];
#pragma unroll
      for (int c = 0; c < TN; c += 16) tmem_ld16(t + (uint32_t)c, part + c);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" : "+r"(part[j]));   // not read above the wait
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty0 + 8u * (uint32_t)acc);
      const float4* s4 = reinterpret_cast<const float4*>(scales[kb - kb0]);
#pragma unroll
      for (int j = 0; j < TN; j += 4) {
        const float4 s = s4[j / 4];
        sum[j] = fmaf(__uint_as_float(part[j]), s.x, sum[j]);
        sum[j + 1] = fmaf(__uint_as_float(part[j + 1]), s.y, sum[j + 1]);
        sum[j + 2] = fmaf(__uint_as_float(part[j + 2]), s.z, sum[j + 2]);
        sum[j + 3] = fmaf(__uint_as_float(part[j + 3]), s.w, sum[j + 3]);
      }
      if (++acc == DEPTH) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }
  if (again) {
    const int n = n0 + threadIdx.x;
    float total[TN];                                         // by way of local memory: unrolled it would cost everybody registers
#pragma unroll
    for (int j = 0; j < TN; ++j) total[j] = sum[j];
#pragma unroll 1
    for (int j = 0; j < min(TN, g.m - m0) && n < g.n; ++j)
      if (f8_row_unsafe<2>(g, m0 + j, blockIdx.y, kb0, kb1)) total[j] = f8_dot(g, m0 + j, n, kb0, kb1);
#pragma unroll
    for (int j = 0; j < TN; ++j) sum[j] = total[j];
    __syncwarp();
  }
  // Tensor memory goes back as soon as it has been read, whatever the other CTAs do: they may be waiting for tensor memory
  // themselves, and beside a product of CTA pairs on another stream all could else wait for one another.
  tc_fence_before_sync();
  if (warp < 4) {
    asm volatile("bar.arrive 2, 160;" ::: "memory");
  } else if (warp == 5) {
    asm volatile("bar.sync 2, 160;" ::: "memory");
    tc_fence_after_sync();
    if (*abortp != 0) {                                      // as in gemm_fp8_kernel
      const unsigned long long t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000ull) { }
    }
    tmem_dealloc(tmem, TMEM_COLS);
  }
  const int n = n0 + threadIdx.x;
  if constexpr (SPLITS == 1) {
    if (warp < 4) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
        if (n < g.n && m0 + j < g.m) f8_store(g, m0 + j, n, sum[j]);
    }
  } else {
    __syncwarp();
    cluster_wait_all();                                      // for the others' start
    if (warp < 4) {
#pragma unroll
      for (int to = 0; to < SPLITS; ++to)
        f8_send<PER>(map_to_cta(meet + (uint32_t)(rank * 128 + (int)threadIdx.x) * PITCH, (uint32_t)to), sum + to * PER);
    }
    __syncwarp();
    cluster_sync_all();
    if (warp < 4) {
      float total[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) total[j] = 0.f;
#pragma unroll
      for (int r = 0; r < SPLITS; ++r)
#pragma unroll
        for (int j = 0; j < PER; ++j) total[j] += f8_lds(meet + (uint32_t)(r * 128 + (int)threadIdx.x) * PITCH + 4u * (uint32_t)j);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (n < g.n && m0 + rank * PER + j < g.m) f8_store(g, m0 + rank * PER + j, n, total[j]);
    }
  }
}

// Row-major matrix -> tensor map with boxes of box_rows x box_cols, swizzled by 128 bytes (64 where the box is no wider).
int f8_tensor_map(CUtensorMap* map, CUtensorMapDataType type, int item, const void* base, long long rows, long long cols, long long pitch,
                  int box_rows, int box_cols) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return sb_fail(SB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dim[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)(pitch * item)};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, step[2] = {1, 1};
  CUresult r = enc(map, type, 2, const_cast<void*>(base), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   box_cols * item == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return sb_fail(SB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return SB_OK;
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device, once per device (again is harmless).
template <typename K>
int f8_allow_smem(K* kernel, int bytes, std::atomic<bool>* ready) {
  int dev = 0;
  SB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    SB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  return SB_OK;
}

template <int BN>
int launch_fp8(const F8Args& g, cudaStream_t s) {
  constexpr int STAGE = (128 + BN) * F8_BLOCK, REST = 1024 + F8_WARPS * (f8_boxes(BN) * F8_BOX + 512) + F8_AHEAD * F8_SCALES;
  F8Plan p;
  memset(&p, 0, sizeof(p));
  p.tiles_m = (g.m + 127) / 128;
  p.tiles_n = (g.n + BN - 1) / BN;
  p.tiles = p.tiles_m * p.tiles_n;
  p.stages = BN == 256 ? 3 : (F8_SMEM - REST) / STAGE < F8_STAGES_MAX ? (F8_SMEM - REST) / STAGE : F8_STAGES_MAX;
  const int es = sb_dtype_size(g.out_dtype);
  // A TMA store cuts a box off at the row's end by whole 16-byte pieces only: rows of 70 bf16 in a pitch of 72 had the two
  // elements behind them overwritten.
  p.tma_store = reinterpret_cast<uintptr_t>(g.c) % 16 == 0 && (g.ldc * es) % 16 == 0 && ((long long)g.n * es) % 16 == 0;
  CUtensorMap ta, tw, tc;
  memset(&tc, 0, sizeof(tc));
  int rc = f8_tensor_map(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.a, g.m, g.k, g.lda, 128, F8_BLOCK);
  if (rc == SB_OK) rc = f8_tensor_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.w, g.n, g.k, g.ldw, BN, F8_BLOCK);
  if (rc == SB_OK && p.tma_store) {
    const int cols = (BN / 2) * es >= 128 ? 128 / es : BN / 2;
    rc = f8_tensor_map(&tc, g.out_dtype == SB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                            : g.out_dtype == SB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                       es, g.c, g.m, g.n, g.ldc, 32, cols);
  }
  static std::atomic<bool> ready[64];
  if (rc == SB_OK) rc = f8_allow_smem(gemm_fp8_kernel<BN>, F8_SMEM, ready);
  if (rc != SB_OK) return rc;
  const int workers = p.tiles < sb_sm_count() ? p.tiles : sb_sm_count();
  SB_CUDA(sb_launch(gemm_fp8_kernel<BN>, dim3(workers), dim3(F8_THREADS), (size_t)(REST + p.stages * STAGE), s, 1, ta, tw, tc, g, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

// Shared memory of the form for few rows: dynamic bytes and stages; scales and barriers are static (4 to 17 KB).
struct F8FewSize {
  int stages, bytes, fixed;
};
constexpr int F8_FEW_SMEM = F8_SMEM - 20 * 1024;
F8FewSize f8_few_size(int tn, int splits, int k_blocks) {
  const int stage = (128 + tn) * F8_BLOCK, blocks = (k_blocks + splits - 1) / splits;
  const int rest = 1024 + (splits > 1 ? splits * 128 * (4 * (tn / splits) + 16) : 0);
  int stages = (F8_FEW_SMEM - rest) / stage;
  if (stages > F8_FEW_STAGES) stages = F8_FEW_STAGES;
  if (stages > blocks) stages = blocks;
  return {stages, rest + stages * stage, tn * F8_FEW_BLOCKS * 4 + 512};
}

template <int TN, int SPLITS>
int launch_fp8_few(const F8Args& g, cudaStream_t s) {
  const F8FewSize size = f8_few_size(TN, SPLITS, g.k_blocks);
  CUtensorMap ta, tw;
  int rc = f8_tensor_map(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.a, g.m, g.k, g.lda, TN, F8_BLOCK);
  if (rc == SB_OK) rc = f8_tensor_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.w, g.n, g.k, g.ldw, 128, F8_BLOCK);
  static std::atomic<bool> ready[64];
  if (rc == SB_OK) rc = f8_allow_smem(gemm_fp8_few_kernel<TN, SPLITS>, F8_FEW_SMEM, ready);
  if (rc != SB_OK) return rc;
  const dim3 grid(SPLITS, (g.n + 127) / 128, (g.m + TN - 1) / TN);
  SB_CUDA(sb_launch(gemm_fp8_few_kernel<TN, SPLITS>, grid, dim3(F8_FEW_THREADS), (size_t)size.bytes, s, SPLITS, ta, tw, g, size.stages));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <int TN>
int launch_fp8_few(const F8Args& g, int splits, cudaStream_t s) {
  if constexpr (TN == 64)
    if (splits == 1) return launch_fp8_few<TN, 1>(g, s);
  switch (splits) {
    case 2: return launch_fp8_few<TN, 2>(g, s);
    case 4: return launch_fp8_few<TN, 4>(g, s);
    default: return launch_fp8_few<TN, 8>(g, s);
  }
}

// Which form a product takes: the least of rounds over the SMs x (time of a tile + blocks of K x time of a block), in us as
// measured.  Times of back-to-back launches on operands beyond L2, tiles of 256 / 128 / 64 columns: 16384 x 4096 x 4096 275 / 342 /
// 580, 4000 x 3000 x 1008 25.5 / 27.0 / 39.5, 1024^3 9.3 / 6.2 / 5.6.  Few rows, 16 x 4096 x 4096 with K over 1 / 2 / 4 / 8 CTAs: 11.4 /
// 8.1 / 6.4 / 5.7, and 13.6 as 64-column tiles; 64 x 4096 x 4096 20.2 / 12.6 / 9.9 / 21.0 (two rounds), 12.9; 512 x 512 x 4096 18.2 / 11.3 /
// 8.9 / 20.0, 12.3.
struct F8Choice {
  int few, tile, splits;
};
F8Choice f8_choose(int m, int n, int k_blocks) {
  const int sms = sb_sm_count();
  F8Choice best = {0, 256, 1};
  double least = 1e30;
  const struct { int bn; double block, tile; } forms[] = {{256, 0.60, 2.0}, {128, 0.37, 2.0}, {64, 0.35, 1.8}};
  for (const auto& f : forms) {
    const double tiles = (double)((m + 127) / 128) * ((n + f.bn - 1) / f.bn);
    const double t = ceil(tiles / sms) * (k_blocks * f.block + f.tile);
    if (t < least) {
      least = t;
      best = {0, f.bn, 1};
    }
  }
  for (int tn = 16; tn <= 64; tn *= 2) {
    const long long across = (n + 127) / 128, down = (m + tn - 1) / tn;
    if (across > 65535 || down > 65535) continue;
    const double block = tn == 16 ? 0.28 : tn == 32 ? 0.36 : 0.50;
    const double weights = 128e-6 * 128.0 * across * k_blocks / 5.0;           // on their way from DRAM
    // All of K in one CTA pays for many short products only, 64 rows at a time (1856 x 1280 x 384); narrower tiles never won there.
    for (int splits = tn == 64 ? 1 : 2; splits <= 8; splits *= 2) {
      const int blocks = (k_blocks + splits - 1) / splits;
      if (blocks > F8_FEW_BLOCKS || (splits > 1 && k_blocks < 2 * splits)) continue;
      const F8FewSize size = f8_few_size(tn, splits, k_blocks);
      int resident = 227 * 1024 / (size.bytes + size.fixed + 1024);
      if (resident > 2) resident = 2;
      const double ctas = (double)across * down * splits;
      // Clusters do not fill every SM, and a second round of them costs more than it brings.
      if (splits > 1 && ctas > 0.9 * resident * sms) continue;
      const double t = ceil(ctas / (resident * sms)) * (2.2 + blocks * block) + weights;
      if (t < least) {
        least = t;
        best = {1, tn, splits};
      }
    }
  }
  return best;
}

bool f8_aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// TMA takes rows that begin on 16-byte boundaries.
bool f8_tma_rows(const void* a, long long lda, const void* w, long long ldw) {
  return f8_aligned(a, 16) && f8_aligned(w, 16) && lda % 16 == 0 && ldw % 16 == 0;
}

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
  a.across = (unsigned)((cols + F8_BLOCK - 1) / F8_BLOCK);
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
  cudaStream_t s = (cudaStream_t)stream;
  if (k > 0 && f8_tma_rows(a, lda, w, ldw)) {
    const F8Choice f = f8_choose(m, n, g.k_blocks);
    if (f.few) return f.tile == 16 ? launch_fp8_few<16>(g, f.splits, s) : f.tile == 32 ? launch_fp8_few<32>(g, f.splits, s) : launch_fp8_few<64>(g, f.splits, s);
    return f.tile == 256 ? launch_fp8<256>(g, s) : f.tile == 128 ? launch_fp8<128>(g, s) : launch_fp8<64>(g, s);
  }
  const dim3 grid((unsigned)((m + 63) / 64), (unsigned)((n + 63) / 64));
  SB_CUDA(sb_launch(gemm_fp8_simple_kernel, grid, dim3(256), 0, s, 1, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

int sb_matmul_fp8_plan(int m, int n, int k, int* plan) {
  if (!plan) return sb_fail(SB_ERR_BAD_ARG, "sb_matmul_fp8_plan: null output");
  if (m < 1 || n < 1 || k < 1) return sb_fail(SB_ERR_BAD_ARG, "sb_matmul_fp8_plan: sizes must be positive");
  const F8Choice c = f8_choose(m, n, (k + F8_BLOCK - 1) / F8_BLOCK);
  plan[0] = c.few ? c.tile : 128;
  plan[1] = c.few ? 128 : c.tile;
  plan[2] = c.splits;
  return SB_OK;
}

}  // extern "C"
