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


// The tensor-core form.  A tile of 128 x BN values per CTA, or of 256 x 256 per pair of CTAs (cta_group::2: each loads its
// 128 rows of A and half of the rows of W); a stage of the ring is one 128-byte block of K of both operands, brought by TMA.
// The scales change with every block of K, so every block's four MMAs start a fresh accumulator in TMEM, and eight warps
// add it, times its two scales, to sums in registers (packed fp32 multiply-adds) while the MMAs of the next block run into
// another accumulator.  A thread owns one row and half of the columns, which lie in one 128-block of N: the product of the
// scales is one number per thread and block.
constexpr int F8_STAGES_MAX = 12;
constexpr int F8_BUFFERS_MAX = 4;
constexpr int F8_WARPS = 8;                                  // that add
constexpr int F8_FIRST = 4;                                   // the first of them: warp 0 loads, warp 1 issues, a warpgroup adds as a whole
constexpr int F8_THREADS = 32 * (F8_FIRST + F8_WARPS);
constexpr int F8_SMEM = 225 * 1024;
constexpr uint32_t F8_BOX = 4096;                            // a warp's staging box: 32 rows x 128 bytes

template <bool PAIR>
__device__ __forceinline__ void f8_mma(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate, bool issue) {
#define SB_F8_ASM(GROUP)                                                                                               \
  "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"             \
  "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t@q tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4"              \
  " [%0], da, db, %5, p;\n\t}" ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate),      \
  "r"((uint32_t)issue) : "memory"
  if (PAIR) asm volatile(SB_F8_ASM("2"));
  else asm volatile(SB_F8_ASM("1"));
#undef SB_F8_ASM
}

struct F8Plan {
  int pair, block_n, stages, tiles_m, tiles_n, tiles;
  uint32_t idesc;
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

// 32 columns of an accumulator added to the sums: sum += scale * part.
__device__ __forceinline__ void f8_add32(unsigned long long* sum, const uint32_t* part, unsigned long long scale) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    fma_f32x2(sum[j], pack_f32x2(__uint_as_float(part[2 * j]), __uint_as_float(part[2 * j + 1])), scale);
}

// Arrival on another CTA's barrier without a release: what it announces, that an accumulator has been read, is ordered by
// the wait for the loads and the tcgen05 fence before it.  (With a release it waits for the thread's earlier memory
// operations once per block of K: 16384 x 4096 x 4096 took 516 us.)
__device__ __forceinline__ void f8_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Finished values of this warp's 32 rows and COLS columns -> C, a box of 32 rows x 128 bytes at a time (64 bytes where the
// columns are no more): by a TMA store, or by coalesced stores where C's rows are not whole 16-byte pieces.
template <typename O, int COLS>
__device__ __forceinline__ void f8_write(const F8Args& g, const CUtensorMap* tmap_c, bool tma, const unsigned long long* sum,
                                         long long row0, int col0, uint32_t box, int lane) {
  constexpr int BOX_COLS = COLS * sizeof(O) >= 128 ? 128 / sizeof(O) : COLS;
  constexpr int ROW_BYTES = BOX_COLS * sizeof(O), PIECES = ROW_BYTES / 16, PER = 16 / sizeof(O);
#pragma unroll
  for (int b = 0; b < COLS / BOX_COLS; ++b) {
    const int first = col0 + b * BOX_COLS;
    if (first >= g.n) return;
    if (tma) {
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
    }
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      float v[PER];
#pragma unroll
      for (int t = 0; t < PER; t += 2) unpack_f32x2(sum[(b * BOX_COLS + q * PER + t) / 2], v[t], v[t + 1]);
      if (g.bias) {
#pragma unroll
        for (int t = 0; t < PER; ++t) {
          const int col = first + q * PER + t;
          if (col < g.n) v[t] += __ldg(g.bias + col);
        }
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
#pragma unroll 4
      for (int i = lane; i < 32 * BOX_COLS; i += 32) {
        const uint32_t r = (uint32_t)i / BOX_COLS, c = (uint32_t)i % BOX_COLS;
        const uint32_t key = ROW_BYTES == 128 ? (r & 7u) : ((r >> 1) & 3u);
        const uint32_t at = box + r * ROW_BYTES + (((c / PER ^ key) & (PIECES - 1)) << 4) + (c % PER) * (uint32_t)sizeof(O);
        if (row0 + r < g.m && first + (int)c < g.n) {
          O* to = (O*)g.c + (row0 + r) * g.ldc + first + c;
          if (sizeof(O) == 4) {
            uint32_t w;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
            *reinterpret_cast<uint32_t*>(to) = w;
          } else {
            uint16_t w;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(at) : "memory");
            *reinterpret_cast<uint16_t*>(to) = w;
          }
        }
      }
      __syncwarp();
    }
  }
}

template <bool PAIR, int BN>
__global__ void __launch_bounds__(F8_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                const __grid_constant__ CUtensorMap tmap_c, const __grid_constant__ F8Args g, const __grid_constant__ F8Plan p) {
  constexpr int BUFFERS = 512 / BN < F8_BUFFERS_MAX ? 512 / BN : F8_BUFFERS_MAX;
  constexpr int COLS = BN / 2;                               // of a thread
  constexpr int TILE_M = PAIR ? 256 : 128;
  constexpr uint32_t A_BYTES = 128 * 128, W_ROWS = PAIR ? BN / 2 : BN, W_BYTES = W_ROWS * 128, STAGE = A_BYTES + W_BYTES;
  extern __shared__ uint8_t f8_smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[F8_STAGES_MAX], bar_empty[F8_STAGES_MAX];
  __shared__ __align__(8) uint64_t bar_acc_full[F8_BUFFERS_MAX], bar_acc_empty[F8_BUFFERS_MAX];
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_cta_rank() : 0u;
  const int worker = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, workers = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const uint32_t stage0 = (smem_u32(f8_smem_raw) + 1023u) & ~1023u;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < BUFFERS; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), PAIR ? 2 * F8_WARPS : F8_WARPS);
    }
    g_f8_abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(&tmem_slot), BUFFERS * BN);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&tmem_slot), BUFFERS * BN);
      tmem_relinquish();
    }
  }
  tc_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
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
    const uint32_t full_local = smem_u32(&bar_full[0]), full0 = PAIR ? map_to_cta(full_local, 0u) : full_local;
    const uint32_t empty0 = smem_u32(&bar_empty[0]);
    for (int tile = worker; ok && tile < p.tiles; tile += workers) {
      int m_blk, n_blk;
      f8_tile(p, tile, m_blk, n_blk);
      const int m0 = m_blk * TILE_M + (int)rank * 128, n0 = n_blk * BN + (int)rank * (int)W_ROWS;
      for (int kb = 0; kb < g.k_blocks; ++kb) {
        if (!mbar_wait_warp(empty0 + 8u * (uint32_t)stage, phase ^ 1u, abortp, SB_SITE_PRODUCER_EMPTY)) {
          ok = false;
          break;
        }
        // In a pair the leader arms its barrier with the bytes of both CTAs.
        if (one && rank == 0u) mbar_arrive_expect_tx(full_local + 8u * (uint32_t)stage, PAIR ? 2u * STAGE : STAGE);
        const uint32_t at = stage0 + (uint32_t)stage * STAGE, full = full0 + 8u * (uint32_t)stage;
        if (PAIR) {
          tma_load_2d_pair(at, &tmap_a, kb * F8_BLOCK, m0, full, one);
          tma_load_2d_pair(at + A_BYTES, &tmap_w, kb * F8_BLOCK, n0, full, one);
        } else {
          tma_load_2d(at, &tmap_a, kb * F8_BLOCK, m0, full, one);
          tma_load_2d(at + A_BYTES, &tmap_w, kb * F8_BLOCK, n0, full, one);
        }
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0u) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      const uint64_t a_desc = umma_smem_desc(stage0, 16u, 1024u, 2u), w_desc = umma_smem_desc(stage0 + A_BYTES, 16u, 1024u, 2u);
      const uint32_t a_hi = (uint32_t)(a_desc >> 32), w_hi = (uint32_t)(w_desc >> 32);
      const uint32_t a_lo0 = (uint32_t)a_desc, w_lo0 = (uint32_t)w_desc;
      const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
      const uint32_t acc_full0 = smem_u32(&bar_acc_full[0]), acc_empty0 = smem_u32(&bar_acc_empty[0]);
      uint32_t a_lo = a_lo0, w_lo = w_lo0;
      for (int tile = worker; ok && tile < p.tiles; tile += workers) {
        for (int kb = 0; kb < g.k_blocks; ++kb) {
          if (!mbar_wait_warp(acc_empty0 + 8u * (uint32_t)buf, acc_phase ^ 1u, abortp, SB_SITE_MMA_TMEM_EMPTY) ||
              !mbar_wait_warp(full0 + 8u * (uint32_t)stage, phase, abortp, SB_SITE_MMA_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d = tmem + (uint32_t)(buf * BN);
          f8_mma<PAIR>(d, a_lo, a_hi, w_lo, w_hi, p.idesc, 0u, one);
          f8_mma<PAIR>(d, a_lo + 2u, a_hi, w_lo + 2u, w_hi, p.idesc, 1u, one);
          f8_mma<PAIR>(d, a_lo + 4u, a_hi, w_lo + 4u, w_hi, p.idesc, 1u, one);
          f8_mma<PAIR>(d, a_lo + 6u, a_hi, w_lo + 6u, w_hi, p.idesc, 1u, one);
          if (PAIR) {
            tc_commit_pair(empty0 + 8u * (uint32_t)stage, (uint16_t)3, one);
            tc_commit_pair(acc_full0 + 8u * (uint32_t)buf, (uint16_t)3, one);
          } else {
            tc_commit(empty0 + 8u * (uint32_t)stage, one);
            tc_commit(acc_full0 + 8u * (uint32_t)buf, one);
          }
          a_lo += STAGE >> 4;
          w_lo += STAGE >> 4;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
            a_lo = a_lo0;
            w_lo = w_lo0;
          }
          if (++buf == BUFFERS) {
            buf = 0;
            acc_phase ^= 1u;
          }
        }
      }
    }
  } else if (warp >= F8_FIRST) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quad = warp & 3, half = (warp - F8_FIRST) >> 2;   // a warp reads the TMEM lanes of its number modulo 4
    const uint32_t box = stage0 + (uint32_t)p.stages * STAGE + (uint32_t)(warp - F8_FIRST) * F8_BOX;
    const uint32_t acc_full0 = smem_u32(&bar_acc_full[0]);
    const uint32_t acc_empty_local = smem_u32(&bar_acc_empty[0]), acc_empty0 = PAIR ? map_to_cta(acc_empty_local, 0u) : acc_empty_local;
    int buf = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = worker; ok && tile < p.tiles; tile += workers) {
      int m_blk, n_blk;
      f8_tile(p, tile, m_blk, n_blk);
      const long long row0 = (long long)m_blk * TILE_M + (int)rank * 128 + quad * 32;
      const int col0 = n_blk * BN + half * COLS;
      const bool row_ok = row0 + lane < g.m, col_ok = col0 < g.n;
      const float* sa = g.sa + (row_ok ? row0 + lane : 0);
      const float* sw = g.sw + (col_ok ? (long long)(col0 / F8_BLOCK) * g.k_blocks : 0);
      unsigned long long sum[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) sum[j] = 0ull;
      // Scales four blocks ahead: the loads of the next four are on their way while these four are used.
      float next[4];
      auto fetch = [&](int kb0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kb = kb0 + i;
          next[i] = kb < g.k_blocks && row_ok && col_ok ? __ldg(sa + (long long)kb * g.m) * __ldg(sw + kb) : 0.f;
        }
      };
      fetch(0);
      for (int kb0 = 0; ok && kb0 < g.k_blocks; kb0 += 4) {
        float scale[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) scale[i] = next[i];
        fetch(kb0 + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kb0 + i < g.k_blocks && ok) {
            ok = mbar_wait_warp(acc_full0 + 8u * (uint32_t)buf, acc_phase, abortp, SB_SITE_EPI_TMEM_FULL);
            if (ok) {
              tc_fence_after_sync();
              const uint32_t t = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + half * COLS);
              const unsigned long long s2 = pack_f32x2(scale[i], scale[i]);
              uint32_t part[2][32];
              tmem_ld32(t, part[0]);
#pragma unroll
              for (int c = 0; c < COLS / 32; ++c) {
                tmem_ld_wait32(part[c & 1]);
                if (c + 1 < COLS / 32) {
                  tmem_ld32(t + (uint32_t)(c + 1) * 32u, part[(c + 1) & 1]);
                } else {                                     // all of the accumulator is in registers
                  tc_fence_before_sync();
                  __syncwarp();
                  if (lane == 0) {
                    if (PAIR) f8_arrive_cluster(acc_empty0 + 8u * (uint32_t)buf);
                    else mbar_arrive(acc_empty0 + 8u * (uint32_t)buf);
                  }
                }
                f8_add32(sum + c * 16, part[c & 1], s2);
              }
              if (++buf == BUFFERS) {
                buf = 0;
                acc_phase ^= 1u;
              }
            }
          }
        }
      }
      if (!ok) break;
      if (row0 < g.m) {
        if (g.out_dtype == SB_F32) f8_write<float, COLS>(g, &tmap_c, p.tma_store != 0, sum, row0, col0, box, lane);
        else if (g.out_dtype == SB_BF16) f8_write<__nv_bfloat16, COLS>(g, &tmap_c, p.tma_store != 0, sum, row0, col0, box, lane);
        else f8_write<__half, COLS>(g, &tmap_c, p.tma_store != 0, sum, row0, col0, box, lane);
      }
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }
  // After an expired wait copies and MMAs in flight get time to land before shared and tensor memory are released; neither
  // CTA of a pair leaves while the other can still reach it.
  tc_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  if (*abortp != 0) {
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) { }
  }
  if (PAIR) cluster_sync_all(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem, BUFFERS * BN);
    else tmem_dealloc(tmem, BUFFERS * BN);
  }
}

// Row-major matrix -> tensor map with boxes of box_rows x box_bytes, swizzled by 128 bytes (64 where the box is no wider).
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

template <bool PAIR, int BN>
int launch_fp8(const F8Args& g, cudaStream_t s) {
  constexpr uint32_t STAGE = 128 * 128 + (PAIR ? BN / 2 : BN) * 128;
  F8Plan p;
  memset(&p, 0, sizeof(p));
  p.pair = PAIR; p.block_n = BN;
  p.tiles_m = (g.m + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128);
  p.tiles_n = (g.n + BN - 1) / BN;
  p.tiles = p.tiles_m * p.tiles_n;
  const int room = (int)((F8_SMEM - 1024 - F8_WARPS * F8_BOX) / STAGE);
  p.stages = room < F8_STAGES_MAX ? room : F8_STAGES_MAX;
  // kind::f8f6f4, E4M3 x E4M3 (formats 0), fp32 accumulator: see sb_umma_idesc for the fields.
  p.idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((PAIR ? 256u : 128u) >> 4 << 24);
  const int es = sb_dtype_size(g.out_dtype);
  // A TMA store cuts a box off at the row's end by whole 16-byte pieces only: rows of 70 bf16 in a pitch of 72 had the two
  // elements behind them overwritten.
  p.tma_store = reinterpret_cast<uintptr_t>(g.c) % 16 == 0 && (g.ldc * es) % 16 == 0 && ((long long)g.n * es) % 16 == 0;
  CUtensorMap ta, tw, tc;
  memset(&tc, 0, sizeof(tc));
  int rc = f8_tensor_map(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.a, g.m, g.k, g.lda, 128, 128);
  if (rc == SB_OK) rc = f8_tensor_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.w, g.n, g.k, g.ldw, PAIR ? BN / 2 : BN, 128);
  if (rc == SB_OK && p.tma_store) {
    const int cols = (BN / 2) * es >= 128 ? 128 / es : BN / 2;
    rc = f8_tensor_map(&tc, g.out_dtype == SB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                            : g.out_dtype == SB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                       es, g.c, g.m, g.n, g.ldc, 32, cols);
  }
  if (rc != SB_OK) return rc;
  const size_t smem = 1024 + (size_t)p.stages * STAGE + F8_WARPS * F8_BOX;
  static std::atomic<bool> ready[64];
  int dev = 0;
  SB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {   // setting it twice is harmless
    SB_CUDA(cudaFuncSetAttribute(gemm_fp8_kernel<PAIR, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, F8_SMEM));
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  const int most = PAIR ? sb_sm_count() / 2 : sb_sm_count();
  const int workers = p.tiles < most ? p.tiles : most;
  SB_CUDA(sb_launch(gemm_fp8_kernel<PAIR, BN>, dim3(PAIR ? 2 * workers : workers), dim3(F8_THREADS), smem, s, PAIR ? 2 : 1, ta, tw, tc, g, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
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
  cudaStream_t s = (cudaStream_t)stream;
  // TMA takes rows that begin on 16-byte boundaries.
  if (k > 0 && f8_aligned(a, 16) && f8_aligned(w, 16) && lda % 16 == 0 && ldw % 16 == 0) {
    const long long sms = sb_sm_count();
    const long long pairs = ((m + 255) / 256LL) * ((n + 255) / 256LL), singles = ((m + 127) / 128LL) * ((n + 127) / 128LL);
    if (getenv("F8V")) {
      const int v = atoi(getenv("F8V"));
      return v == 0 ? launch_fp8<true, 256>(g, s) : v == 1 ? launch_fp8<false, 128>(g, s) : launch_fp8<false, 64>(g, s);
    }
    if (pairs >= sms / 2) return launch_fp8<true, 256>(g, s);
    if (singles >= sms / 2) return launch_fp8<false, 128>(g, s);
    return launch_fp8<false, 64>(g, s);
  }
  const dim3 grid((unsigned)((m + 63) / 64), (unsigned)((n + 63) / 64));
  SB_CUDA(sb_launch(gemm_fp8_simple_kernel, grid, dim3(256), 0, s, 1, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

}  // extern "C"
