// Gated layers: h = act(x Wg^T) * (x Wu^T), both projections, the activation and their product in one kernel, and the gradient.
//
// With g = x Wg^T, u = x Wu^T and a the activation:
//   dg = dh u a'(g)   du = dh a(g)   dx = dg Wg + du Wu   dWg = dg^T x   dWu = du^T x
//   silu: a = g s(g), a' = s (1 + g (1 - s)) with s = 1 / (1 + exp(-g));  gelu: a = g P(g), a' = P(g) + g exp(-g^2 / 2) / sqrt(2 pi)
//   with the normal distribution P(g) = (1 + erf(g / sqrt 2)) / 2;  relu: a = max(0, g), a' = [g > 0].
#include "common.cuh"
#include "few_rows.cuh"
#include "vector_io.cuh"

#include <type_traits>

namespace {

enum GatedAct { ACT_SILU = SB_ACT_SILU, ACT_GELU = SB_ACT_GELU, ACT_RELU = SB_ACT_RELU };

// 1 / (1 + exp(-g)), from exp(-|g|), which no g takes out of range: the quick division gives 0 for divisors above 2^126.
__device__ __forceinline__ float gated_sigmoid(float g) {
  const float e = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + e);
  return g < 0.f ? e * r : r;
}

// The normal distribution's P(g) and exp(-g^2 / 2), which its tails are made of: with t = 1 / (1 + |g| / sqrt 8) P(-|g|) = t (a1 + t (a2 + ... + t
// a7)) exp(-g^2 / 2).  The coefficients are a fit of this file's own, the least largest error on 0 <= |g| <= 14.4 relative to exp(g^2 / 2) P(-|g|), which
// falls like 1 / |g|: with all roundings 6e-7 up to |g| = 1, 1e-6 up to 2, 7e-6 up to 12, so that the smallest values have all the digits of the storage
// types.
__device__ __forceinline__ float2 gated_normal(float g) {
  const float t = __fdividef(1.f, fmaf(0.35355339059327376f, fabsf(g), 1.f)), e = __expf(-0.5f * g * g);
  float q = fmaf(t, 0.04597611858848591f, -0.18459764335694676f);
  q = fmaf(t, q, 0.20273347957186824f);
  q = fmaf(t, q, 0.013682007891541514f);
  q = fmaf(t, q, 0.1425210676958373f);
  q = fmaf(t, q, 0.13850115379783598f);
  q = fmaf(t, q, 0.14118375197936758f);
  q *= t * e;
  return make_float2(g > 0.f ? 1.f - q : q, e);
}

template <int ACT>
__device__ __forceinline__ float gated_act(float g) {
  if (ACT == ACT_SILU) return g * gated_sigmoid(g);
  if (ACT == ACT_GELU) return g * gated_normal(g).x;
  return g > 0.f ? g : (g != g ? g : 0.f);
}
// The activation and its derivative.  A gate that the storage type rounded to an infinity counts as the number next to it: far below zero both are 0,
// not 0 times infinity (the layer's output was finite there), and far above the derivative is 1.
template <int ACT>
__device__ __forceinline__ float2 gated_act_grad(float g) {
  constexpr float MOST = 3.402823466e38f;
  g = min_nan(max_nan(g, -MOST), MOST);
  if (ACT == ACT_SILU) {
    const float s = gated_sigmoid(g);
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  if (ACT == ACT_GELU) {
    const float2 n = gated_normal(g);
    return make_float2(g * n.x, fmaf(g * 0.39894228040143268f, n.y, n.x));
  }
  return make_float2(gated_act<ACT_RELU>(g), g > 0.f ? 1.f : 0.f);
}

// Any sizes, pitches and alignments, on the CUDA cores: 64 x 64 outputs per block, 16 of K at a time.
constexpr int GS_TILE = 64, GS_K = 16;

// A matrix by the distances of neighbours in a column and in a row; `lo`: what its rounding left off, laid out the same, where that is kept.
struct Strided {
  const void* p;
  long long down, across;
  const void* lo;
};

template <typename T>
__device__ __forceinline__ float strided_at(const Strided& m, long long i, long long j) {
  const long long at = i * m.down + j * m.across;
  const float v = sb_to_f32<T>(reinterpret_cast<const T*>(m.p)[at]);
  return m.lo ? v + sb_to_f32<T>(reinterpret_cast<const T*>(m.lo)[at]) : v;
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
  const Strided x = {p.x, p.ldx, 1, nullptr}, g = {p.w, p.ldw, 1, nullptr}, u = {reinterpret_cast<const T*>(p.w) + (long long)p.f * p.ldw, p.ldw, 1, nullptr};
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

// ---- tensor cores ----------------------------------------------------------------------------------------------
// One persistent kernel: tiles of 128 rows (256 for a pair of CTAs) and `bf` columns of h.  A tile's accumulator has 2 bf columns, the
// gate's and beside them the other projection's, from one sequence of MMAs with N = 2 bf whose B operand is bf rows of each half of w: in
// a pair the leader brings the gate's and its peer the other's.  The epilogue finds both values of an output in one TMEM lane.
//   warp 0: TMA of x      warp 10: TMA of w      warp 1: MMAs      warps 2 .. 9: epilogue, two per lane quadrant on alternate 32-column chunks
// Two accumulators let the epilogue of a tile run beside the MMAs of the next.  Bound by the tensor cores where rows are on 32 bytes; calls one after
// the other, all with saved: 16384 x 4096 x 1024 (silu) 233 to 249 us, 1.1 to 1.2 PFLOP/s under the power cap, 4001 x 3000 x 1024 (gelu) 52 to 58.
// Rows of 2000 bytes, whose pieces of 128 lie in five sectors of L2 each, take 61 to 71 for 4001 x 3000 x 1000.
constexpr int GU_EPI_WARPS = 8;
constexpr int GU_THREADS = 96 + 32 * GU_EPI_WARPS;
constexpr int GU_MAX_STAGES = 8;
constexpr int GU_BOX = 32 * 64;                 // 32 rows of 32 16-bit columns on their way to memory
constexpr int GU_BOXES = 3;                     // per epilogue warp: h, g, u of a chunk
constexpr int GU_STAGING = GU_EPI_WARPS * GU_BOXES * GU_BOX;
constexpr int GU_SMEM = 225 * 1024;

struct GatedMaps {
  CUtensorMap x, w, w_half, h, g, u;            // w_half: boxes of half as many rows, for the half tiles; g, u: the halves of saved
};
struct GatedPlan {
  int bf, tiles_m, tiles_f, k_blocks, stages, acc_stride, tmem_cols;
  int items, half_first;                        // items from half_first on are the halves of tiles
  uint32_t idesc, idesc_half, b_bytes;          // of w per stage and CTA
  int boxes_out;                                // 1: outputs leave as TMA boxes
};

// An item's row block, first column of h and columns.
__device__ __forceinline__ void gated_item(const GatedPlan& q, int item, int& mb, int& f0, int& bf) {
  const int tile = item < q.half_first ? item : q.half_first + (item - q.half_first) / 2;
  bf = item < q.half_first ? q.bf : q.bf / 2;
  // Eight row blocks at a time: the CTAs that run together share rows of w and of x in L2.
  const int per_group = 8 * q.tiles_f, group = tile / per_group, first = 8 * group;
  const int rows = min(8, q.tiles_m - first), r = tile - group * per_group;
  mb = first + r % rows;
  f0 = r / rows * q.bf + (item < q.half_first ? 0 : (item - q.half_first) % 2 * bf);
}

template <typename T>
__device__ __forceinline__ uint32_t gated_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t gated_pack<__nv_bfloat16>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <>
__device__ __forceinline__ uint32_t gated_pack<__half>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// A lane's row of 32 values into its row of a swizzled box.
template <typename T>
__device__ __forceinline__ void gated_to_box(uint32_t box, int lane, const float* v) {
  const uint32_t row = box + 64u * (uint32_t)lane, key = ((uint32_t)lane >> 1) & 3u;
#pragma unroll
  for (uint32_t q = 0; q < 4; ++q)
    st_shared_v4(row + ((q ^ key) << 4), make_uint4(gated_pack<T>(v[8 * q], v[8 * q + 1]), gated_pack<T>(v[8 * q + 2], v[8 * q + 3]),
                                                    gated_pack<T>(v[8 * q + 4], v[8 * q + 5]), gated_pack<T>(v[8 * q + 6], v[8 * q + 7])));
}

// For outputs that no box takes: lanes' rows of 32 values to 4 KB of shared memory, from where the lanes take a row's columns.
__device__ __forceinline__ void gated_turn(uint32_t to, int lane, const float* v) {
#pragma unroll
  for (int j = 0; j < 32; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + 128u * (uint32_t)lane + 4u * (uint32_t)(j ^ lane)), "f"(v[j]) : "memory");
  __syncwarp();
}
__device__ __forceinline__ float gated_turned(uint32_t at, int lane, int row) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at + 128u * (uint32_t)row + 4u * (uint32_t)(lane ^ row)) : "memory");
  return v;
}

template <bool PAIR, typename T, int ACT>
__global__ void __launch_bounds__(GU_THREADS, 1) gated_umma_kernel(const __grid_constant__ GatedMaps maps, const GatedArgs p, const GatedPlan q) {
  extern __shared__ uint8_t gu_smem[];
  __shared__ __align__(8) uint64_t bar_full[GU_MAX_STAGES], bar_empty[GU_MAX_STAGES], bar_acc_full[2], bar_acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  constexpr uint32_t A_BYTES = 128 * 128;
  constexpr int TILE_M = PAIR ? 256 : 128;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = PAIR ? cluster_cta_rank() : 0u;
  const int worker = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, workers = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const uint32_t base = (smem_u32(gu_smem) + 1023u) & ~1023u;
  const uint32_t stage_bytes = A_BYTES + q.b_bytes;
  if (tid == 0) {
    for (int i = 0; i < q.stages; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), (PAIR ? 2 : 1) * GU_EPI_WARPS);
    }
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.x);
    tma_prefetch_desc(&maps.w);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(&tmem_slot), (uint32_t)q.tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&tmem_slot), (uint32_t)q.tmem_cols);
      tmem_relinquish();
    }
  }
  tc_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &abort_flag;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();

  const bool one = elect_one_lane();
  if (warp == 0 || warp == 2 + GU_EPI_WARPS) {
    const bool do_x = warp == 0;
    const uint32_t full_local = smem_u32(&bar_full[0]), full0 = PAIR ? map_to_cta(full_local, 0u) : full_local, empty0 = smem_u32(&bar_empty[0]);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = worker; ok && item < q.items; item += workers) {
      int mb, f0, bf;
      gated_item(q, item, mb, f0, bf);
      const int m0 = mb * TILE_M + (int)rank * 128;
      const CUtensorMap* w = bf == q.bf ? &maps.w : &maps.w_half;
      const uint32_t b_bytes = bf == q.bf ? q.b_bytes : q.b_bytes / 2u, tx = (PAIR ? 2u : 1u) * (A_BYTES + b_bytes);
      for (int kb = 0; kb < q.k_blocks; ++kb) {
        if (!mbar_wait_warp(empty0 + 8u * (uint32_t)stage, phase ^ 1u, abortp, SB_SITE_PRODUCER_EMPTY)) {
          ok = false;
          break;
        }
        const uint32_t full = full0 + 8u * (uint32_t)stage, dst = base + (uint32_t)stage * stage_bytes;
        if (do_x) {
          // In a pair the leader arms its barrier with the bytes of both CTAs.
          if (one && rank == 0u) mbar_arrive_expect_tx(full_local + 8u * (uint32_t)stage, tx);
          if (PAIR) tma_load_2d_pair(dst, &maps.x, kb * 64, m0, full, one);
          else tma_load_2d(dst, &maps.x, kb * 64, m0, full, one);
        } else if (PAIR) {
          // (Rows of the gate beyond f are the other projection's: outputs that are not written.)
          tma_load_2d_pair(dst + A_BYTES, w, kb * 64, rank == 0u ? f0 : p.f + f0, full, one);
        } else {
          tma_load_2d(dst + A_BYTES, w, kb * 64, f0, full, one);
          tma_load_2d(dst + A_BYTES + (uint32_t)bf * 128u, w, kb * 64, p.f + f0, full, one);
        }
        if (++stage == q.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0u) {
      const uint64_t a_desc = umma_smem_desc(base, 16u, 1024u, 2u), b_desc = umma_smem_desc(base + A_BYTES, 16u, 1024u, 2u);
      const uint32_t a_hi = (uint32_t)(a_desc >> 32), b_hi = (uint32_t)(b_desc >> 32), a_lo0 = (uint32_t)a_desc, b_lo0 = (uint32_t)b_desc;
      const uint32_t step = stage_bytes >> 4, full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
      uint32_t a_lo = a_lo0, b_lo = b_lo0, phase = 0, acc_phase = 0;
      int stage = 0, acc = 0;
      bool ok = true;
      for (int item = worker; ok && item < q.items; item += workers) {
        const uint32_t idesc = item < q.half_first ? q.idesc : q.idesc_half;
        if (!mbar_wait_warp(smem_u32(&bar_acc_empty[acc]), acc_phase ^ 1u, abortp, SB_SITE_MMA_TMEM_EMPTY)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + (uint32_t)(acc * q.acc_stride);
        for (int kb = 0; kb < q.k_blocks; ++kb) {
          if (!mbar_wait_warp(full0 + 8u * (uint32_t)stage, phase, abortp, SB_SITE_MMA_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) umma_issue<PAIR, false>(d, a_lo + 2u * i, a_hi, b_lo + 2u * i, b_hi, idesc, kb > 0 || i > 0 ? 1u : 0u, one);
          if (PAIR) tc_commit_pair(empty0 + 8u * (uint32_t)stage, (uint16_t)3, one);
          else tc_commit(empty0 + 8u * (uint32_t)stage, one);
          a_lo += step;
          b_lo += step;
          if (++stage == q.stages) {
            stage = 0;
            phase ^= 1u;
            a_lo = a_lo0;
            b_lo = b_lo0;
          }
        }
        if (!ok) break;
        if (PAIR) tc_commit_pair(smem_u32(&bar_acc_full[acc]), (uint16_t)3, one);
        else tc_commit(smem_u32(&bar_acc_full[acc]), one);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  } else if (warp < 2 + GU_EPI_WARPS) {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const uint32_t boxes = base + (uint32_t)q.stages * stage_bytes + (uint32_t)(warp - 2) * (GU_BOXES * GU_BOX);
    const bool keep = p.saved != nullptr;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int item = worker; item < q.items; item += workers) {
      int mb, f0, bf;
      gated_item(q, item, mb, f0, bf);
      const int row0 = mb * TILE_M + (int)rank * 128 + quad * 32;
      const uint32_t t_row = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * q.acc_stride);
      if (!mbar_wait(smem_u32(&bar_acc_full[acc]), acc_phase, abortp, SB_SITE_EPI_TMEM_FULL)) break;
      tc_fence_after_sync();
      for (int c = 32 * half; c < bf; c += 64) {
        uint32_t raw_g[32], raw_u[32];
        tmem_ld32(t_row + (uint32_t)c, raw_g);
        tmem_ld32(t_row + (uint32_t)(bf + c), raw_u);
        tmem_ld_wait();
        if (c + 64 >= bf) {                       // this warp's last: the accumulator is free
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if (PAIR) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_acc_empty[acc]), 0u));
            else mbar_arrive(smem_u32(&bar_acc_empty[acc]));
          }
        }
        const int col0 = f0 + c;
        if (row0 >= p.m || col0 >= p.f) continue;
        float* g = reinterpret_cast<float*>(raw_g);
        float* u = reinterpret_cast<float*>(raw_u);
        if (q.boxes_out) {
          if (lane == 0) bulk_wait_group_read<0>();            // the boxes of the chunk before have been read
          __syncwarp();
          if (keep) {
            gated_to_box<T>(boxes + GU_BOX, lane, g);
            gated_to_box<T>(boxes + 2 * GU_BOX, lane, u);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = gated_act<ACT>(g[j]) * u[j];
          gated_to_box<T>(boxes, lane, g);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&maps.h, boxes, col0, row0);
            if (keep) {
              tma_store_2d(&maps.g, boxes + GU_BOX, col0, row0);
              tma_store_2d(&maps.u, boxes + 2 * GU_BOX, col0, row0);
            }
            bulk_commit_group();
          }
        } else {
          const bool mine = col0 + lane < p.f;
          const int rows = min(32, p.m - row0);
          T* saved = reinterpret_cast<T*>(p.saved) + (long long)row0 * p.lds + col0 + lane;
          T* h = reinterpret_cast<T*>(p.h) + (long long)row0 * p.ldh + col0 + lane;
          if (keep) {
            gated_turn(boxes, lane, g);
            for (int i = 0; i < rows; ++i) {
              const float v = gated_turned(boxes, lane, i);
              if (mine) saved[(long long)i * p.lds] = sb_from_f32<T>(v);
            }
            __syncwarp();
            gated_turn(boxes, lane, u);
            for (int i = 0; i < rows; ++i) {
              const float v = gated_turned(boxes, lane, i);
              if (mine) saved[(long long)i * p.lds + p.f] = sb_from_f32<T>(v);
            }
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = gated_act<ACT>(g[j]) * u[j];
          gated_turn(boxes, lane, g);
          for (int i = 0; i < rows; ++i) {
            const float v = gated_turned(boxes, lane, i);
            if (mine) h[(long long)i * p.ldh] = sb_from_f32<T>(v);
          }
          __syncwarp();
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }
  // After an expired wait, copies and MMAs in flight get time to land before shared and tensor memory go back; in a pair neither CTA
  // leaves while its peer can still touch its memory.
  tc_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  if (*abortp != 0) {
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) { }
  }
  if (PAIR) cluster_sync_all(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem, (uint32_t)q.tmem_cols);
    else tmem_dealloc(tmem, (uint32_t)q.tmem_cols);
  }
}

// ---- few rows --------------------------------------------------------------------------------------------------
// Up to 8 NT rows: a block has 16 columns of h, 16 rows of each half of w, and its eight warps share K, UNROLL blocks of 32 on their way at a
// time.  Their sums are joined in the order of the warps.  1 x 4096 x 1024: 3.3 to 3.7 us, of which the 16.8 MB of weights take 2.6.
constexpr int GF_ROWS = 16, GF_WARPS = 8;
constexpr long long GF_NO_END = 1LL << 60;

template <typename T, int ACT, int NT>
__global__ void __launch_bounds__(32 * GF_WARPS) gated_few_kernel(GatedArgs p) {
  constexpr int UNROLL = 4;
  __shared__ float part[GF_WARPS][2][NT][GF_ROWS][9];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int f0 = blockIdx.x * GF_ROWS, n0 = blockIdx.y * 8 * NT;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const T* w = reinterpret_cast<const T*>(p.w);
  const T* x = reinterpret_cast<const T*>(p.x);
  // Rows of w that are not there give outputs that are not written: they read row 0 of their half.
  const T* rows[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int f = f0 + g + 8 * (i & 1);
    rows[i] = w + (long long)((i >> 1) * (long long)p.f + (f < p.f ? f : 0)) * p.ldw;
  }
  float acc[2][NT][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.f;
  for (int k0 = warp * 32 * UNROLL; k0 < p.k; k0 += GF_WARPS * 32 * UNROLL) {
    uint4 a[UNROLL][4], b[UNROLL][NT];
    if (k0 + 32 * UNROLL <= p.k) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[u][i] = load_eight<false>(rows[i], k0 + 32 * u + 8 * t, GF_NO_END, true);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n) b[u][n] = load_eight<true>(x + (long long)(n0 + 8 * n + g) * p.ldx, k0 + 32 * u + 8 * t, GF_NO_END, n0 + 8 * n + g < p.m);
    } else {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[u][i] = load_eight<false>(rows[i], k0 + 32 * u + 8 * t, p.k, true);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n) b[u][n] = load_eight<true>(x + (long long)(n0 + 8 * n + g) * p.ldx, k0 + 32 * u + 8 * t, p.k, n0 + 8 * n + g < p.m);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mma_16x8x16<T>(acc[i][n], a[u][2 * i].x, a[u][2 * i + 1].x, a[u][2 * i].y, a[u][2 * i + 1].y, b[u][n].x, b[u][n].y);
          mma_16x8x16<T>(acc[i][n], a[u][2 * i].z, a[u][2 * i + 1].z, a[u][2 * i].w, a[u][2 * i + 1].w, b[u][n].z, b[u][n].w);
        }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[warp][i][n][g + 8 * (j >> 1)][2 * t + (j & 1)] = acc[i][n][j];
  __syncthreads();
  for (int e = threadIdx.x; e < GF_ROWS * 8 * NT; e += 32 * GF_WARPS) {
    const int f = e % GF_ROWS, c = e / GF_ROWS, row = n0 + c;
    if (f0 + f >= p.f || row >= p.m) continue;
    float gate = 0.f, up = 0.f;
#pragma unroll
    for (int v = 0; v < GF_WARPS; ++v) {
      gate += part[v][0][c / 8][f][c % 8];
      up += part[v][1][c / 8][f][c % 8];
    }
    reinterpret_cast<T*>(p.h)[(long long)row * p.ldh + f0 + f] = sb_from_f32<T>(gated_act<ACT>(gate) * up);
    if (p.saved) {
      T* saved = reinterpret_cast<T*>(p.saved) + (long long)row * p.lds + f0 + f;
      saved[0] = sb_from_f32<T>(gate);
      saved[p.f] = sb_from_f32<T>(up);
    }
  }
}

struct GatedGradArgs {
  const void* dh;
  const void* saved;
  void* d;                        // [m, 2 f]: dg, du
  void* lo;                       // what their rounding left off, where it is kept
  long long lddh, lds, ldd;
  int m, f;
};

// V columns per thread, every access as wide as they are.  Bound by memory: 8192 x 4096 54 us, 6.2 TB/s.
template <typename T, int ACT, int V>
__global__ void __launch_bounds__(256) gated_act_grad_kernel(GatedGradArgs p) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int across = p.f / V;
  const long long total = (long long)p.m * across;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
    const long long r = e / across, c = (e - r * across) * V;
    const T* saved = reinterpret_cast<const T*>(p.saved) + r * p.lds + c;
    SbWords<sizeof(T) * V> dh_w, g_w, u_w;
    sb_load_words(dh_w, reinterpret_cast<const T*>(p.dh) + r * p.lddh + c, true);
    sb_load_words(g_w, saved, true);
    sb_load_words(u_w, saved + p.f, true);
    float dh[V], g[V], u[V];
    sb_unpack_words<T, V>(dh_w, dh);
    sb_unpack_words<T, V>(g_w, g);
    sb_unpack_words<T, V>(u_w, u);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 a = gated_act_grad<ACT>(g[i]);
      g[i] = dh[i] * u[i] * a.y;
      u[i] = dh[i] * a.x;
    }
    T* d = reinterpret_cast<T*>(p.d) + r * p.ldd + c;
    sb_store_f32<T, V>(d, g);
    sb_store_f32<T, V>(d + p.f, u);
    if (p.lo) {
      T* lo = reinterpret_cast<T*>(p.lo) + r * p.ldd + c;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float hg = sb_to_f32<T>(sb_from_f32<T>(g[i])), hu = sb_to_f32<T>(sb_from_f32<T>(u[i]));
        g[i] = fabsf(hg) < INFINITY ? g[i] - hg : 0.f;
        u[i] = fabsf(hu) < INFINITY ? u[i] - hu : 0.f;
      }
      sb_store_f32<T, V>(lo, g);
      sb_store_f32<T, V>(lo + p.f, u);
    }
  }
}

// ---- the gradient's products -----------------------------------------------------------------------------------
// dx = d w (d [m, 2 f], w [2 f, k]) and dw (+)= d^T x in one persistent launch of pairs of CTAs on tiles of 256 x bn, 128 of K per stage.  B has
// rows of K in both; A does in dw alone.  As many tiles as fill the workers are whole; the rest are cut into parts of K, which leave fp32 sums for
// the launch that joins them: one wave of short parts where two launches would have had a wave of few tiles each.  Bound by the tensor cores: 0.78 us
// per 128 of K and 256 x 256 sums, 1.6 PFLOP/s over the card.  With the launch before and the join one call after the other under the power cap: 8192 x
// 4096 x 1024 279 to 305 us, 4001 x 3000 x 1000 122 to 129, 2048^3 59.  Against a launch for each product with K cut there, single launches at the
// full clock (in series the largest gains nothing): 8192 x 4096 x 1024 249 -> 230, 4001 x 3000 x 1000 122 -> 110, 2048^3 73 -> 65, 4096 x 512 x 2048 62 -> 44, 4096 x 2048 x 512 88 -> 50,
// 512^3 24 -> 17, 65536 x 256 x 216 87 -> 89, 128 x 4096 x 1024 35 -> 35.
//   warp 0: TMA of A      warp 10: TMA of B      warp 1: MMAs      warps 2 .. 9: epilogue, as above
constexpr int GP_BOX = 32 * 128;                // 32 rows of 32 fp32 columns on their way to memory
constexpr int GP_STAGING = GU_EPI_WARPS * GP_BOX;
constexpr uint32_t GP_A_BYTES = 128 * 256;      // of a stage and CTA: 128 rows (or columns) by 128 of K

struct ProductsMaps {
  CUtensorMap a[2], a_lo[2], b[2], out[2];      // dx, dw
};
struct GatedProduct {
  void* out;
  long long ld;
  int rows, cols;
  int tiles_m, tiles_n, whole, parts;           // tiles from `whole` on are cut into `parts`
  int k_blocks;
  int a_mn, f32, accumulate, boxes;             // boxes: outputs leave as TMA boxes
  uint32_t idesc;
};
struct ProductsPlan {
  GatedProduct p[2];
  int bn, stages, items;
  int twice;                                    // 1: every block of K once with d and once with what its rounding left off
  uint32_t b_bytes;                             // of a stage and CTA
  float* partial;
};
struct ProductsItem {
  int which, tile, kb0, kb1;
  long long part;                               // of all parts, -1: a whole tile
};

__device__ __forceinline__ ProductsItem products_item(const ProductsPlan& q, int item) {
  ProductsItem t;
  const int w0 = q.p[0].whole, w1 = q.p[1].whole;
  if (item < w0 + w1) {
    t.which = item < w0 ? 0 : 1;
    t.tile = t.which == 0 ? item : item - w0;
    t.kb0 = 0;
    t.kb1 = q.p[t.which].k_blocks;
    t.part = -1;
    return t;
  }
  int r = item - w0 - w1;
  const int first = (q.p[0].tiles_m * q.p[0].tiles_n - w0) * q.p[0].parts;
  t.which = r < first ? 0 : 1;
  t.part = r;
  if (t.which == 1) r -= first;
  const GatedProduct& p = q.p[t.which];
  t.tile = p.whole + r / p.parts;
  const int part = r % p.parts;
  t.kb0 = (int)((long long)p.k_blocks * part / p.parts);
  t.kb1 = (int)((long long)p.k_blocks * (part + 1) / p.parts);
  if (p.parts == 1) t.part = -1;
  return t;
}
// Eight row blocks at a time, as above.
__device__ __forceinline__ void products_tile(const GatedProduct& p, int bn, int tile, int& row0, int& col0) {
  const int per_group = 8 * p.tiles_n, group = tile / per_group, first = 8 * group;
  const int rows = min(8, p.tiles_m - first), r = tile - group * per_group;
  row0 = (first + r % rows) * 256;
  col0 = r / rows * bn;
}

template <typename T>
__global__ void __launch_bounds__(GU_THREADS, 1) gated_products_kernel(const __grid_constant__ ProductsMaps maps, const __grid_constant__ ProductsPlan q) {
  extern __shared__ uint8_t gu_smem[];
  __shared__ __align__(8) uint64_t bar_full[GU_MAX_STAGES], bar_empty[GU_MAX_STAGES], bar_acc_full[2], bar_acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_cta_rank();
  const int worker = (int)(blockIdx.x >> 1), workers = (int)(gridDim.x >> 1);
  const uint32_t base = (smem_u32(gu_smem) + 1023u) & ~1023u;
  const uint32_t stage_bytes = GP_A_BYTES + q.b_bytes;
  if (tid == 0) {
    for (int i = 0; i < q.stages; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), 2 * GU_EPI_WARPS);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&tmem_slot), (uint32_t)(2 * q.bn));
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &abort_flag;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();

  const bool one = elect_one_lane();
  if (warp == 0 || warp == 2 + GU_EPI_WARPS) {
    const bool do_a = warp == 0;
    const uint32_t full_local = smem_u32(&bar_full[0]), full0 = map_to_cta(full_local, 0u), empty0 = smem_u32(&bar_empty[0]);
    const uint32_t tx = 2u * stage_bytes;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = worker; ok && item < q.items; item += workers) {
      const ProductsItem t = products_item(q, item);
      const GatedProduct& p = q.p[t.which];
      int m0, n0;
      products_tile(p, q.bn, t.tile, m0, n0);
      m0 += (int)rank * 128;
      n0 += (int)rank * (q.bn / 2);
      const CUtensorMap* b = &maps.b[t.which];
      for (int block = t.kb0; block < t.kb1; ++block) {
        const int kb = block >> q.twice;
        const CUtensorMap* a = block & q.twice ? &maps.a_lo[t.which] : &maps.a[t.which];
        if (!mbar_wait_warp(empty0 + 8u * (uint32_t)stage, phase ^ 1u, abortp, SB_SITE_PRODUCER_EMPTY)) {
          ok = false;
          break;
        }
        const uint32_t full = full0 + 8u * (uint32_t)stage, dst = base + (uint32_t)stage * stage_bytes;
        if (do_a) {
          // The leader arms its barrier with the bytes of both CTAs.
          if (one && rank == 0u) mbar_arrive_expect_tx(full_local + 8u * (uint32_t)stage, tx);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            tma_load_2d_pair(dst + (uint32_t)i * (GP_A_BYTES / 2), a, p.a_mn ? m0 + 64 * i : kb * 128 + 64 * i, p.a_mn ? kb * 128 : m0, full, one);
        } else {
          for (int i = 0; i < q.bn / 128; ++i)
            tma_load_2d_pair(dst + GP_A_BYTES + (uint32_t)i * 16384u, b, n0 + 64 * i, kb * 128, full, one);
        }
        if (++stage == q.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0u) {
      // Rows of K: segments of 64 columns 16384 bytes apart, 16 of K 2048.  Otherwise 16 of K are 32 bytes apart, 64 a slab.
      const uint64_t a_cols = umma_smem_desc(base, 16u, 1024u, 2u), a_rows = umma_smem_desc(base, 16384u, 1024u, 2u),
                     b_rows = umma_smem_desc(base + GP_A_BYTES, 16384u, 1024u, 2u);
      const uint32_t hi = (uint32_t)(a_cols >> 32);            // the same in all three
      const uint32_t step = stage_bytes >> 4, full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);
      uint32_t phase = 0, acc_phase = 0, at = 0;
      int stage = 0, acc = 0;
      bool ok = true;
      for (int item = worker; ok && item < q.items; item += workers) {
        const ProductsItem t = products_item(q, item);
        const bool mn = q.p[t.which].a_mn != 0;
        const uint32_t idesc = q.p[t.which].idesc, a_lo0 = mn ? (uint32_t)a_rows : (uint32_t)a_cols, near = mn ? 128u : 2u, far = mn ? 512u : 1024u;
        if (!mbar_wait_warp(smem_u32(&bar_acc_empty[acc]), acc_phase ^ 1u, abortp, SB_SITE_MMA_TMEM_EMPTY)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + (uint32_t)(acc * q.bn);
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!mbar_wait_warp(full0 + 8u * (uint32_t)stage, phase, abortp, SB_SITE_MMA_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a_lo = a_lo0 + at, b_lo = (uint32_t)b_rows + at;
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i)
            umma_issue<true, false>(d, a_lo + (i / 4) * far + (i % 4) * near, hi, b_lo + 128u * i, hi, idesc, kb > t.kb0 || i > 0 ? 1u : 0u, one);
          tc_commit_pair(empty0 + 8u * (uint32_t)stage, (uint16_t)3, one);
          at += step;
          if (++stage == q.stages) {
            stage = 0;
            phase ^= 1u;
            at = 0;
          }
        }
        if (!ok) break;
        tc_commit_pair(smem_u32(&bar_acc_full[acc]), (uint16_t)3, one);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  } else if (warp < 2 + GU_EPI_WARPS) {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const uint32_t box = base + (uint32_t)q.stages * stage_bytes + (uint32_t)(warp - 2) * GP_BOX;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int item = worker; item < q.items; item += workers) {
      const ProductsItem t = products_item(q, item);
      const GatedProduct& p = q.p[t.which];
      int row0, n0;
      products_tile(p, q.bn, t.tile, row0, n0);
      row0 += (int)rank * 128 + quad * 32;
      const uint32_t t_row = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * q.bn);
      if (!mbar_wait(smem_u32(&bar_acc_full[acc]), acc_phase, abortp, SB_SITE_EPI_TMEM_FULL)) break;
      tc_fence_after_sync();
      for (int c = 32 * half; c < q.bn; c += 64) {
        uint32_t raw[32];
        tmem_ld32(t_row + (uint32_t)c, raw);
        tmem_ld_wait();
        if (c + 64 >= q.bn) {                     // this warp's last: the accumulator is free
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_acc_empty[acc]), 0u));
        }
        const int col0 = n0 + c;
        if (row0 >= p.rows || col0 >= p.cols) continue;
        float* v = reinterpret_cast<float*>(raw);
        if (t.part >= 0) {                        // by columns, so that the lanes' stores are neighbours
          float* to = q.partial + ((2 * t.part + rank) * q.bn + c) * 128 + quad * 32 + lane;
#pragma unroll
          for (int j = 0; j < 32; ++j) to[128 * j] = v[j];
          continue;
        }
        // Sums in fp32 are added by the memory system, one addition per element; 16-bit ones here, rounded once.
        if (p.accumulate && !p.f32 && row0 + lane < p.rows) {
          const T* old = reinterpret_cast<const T*>(p.out) + (long long)(row0 + lane) * p.ld + col0;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (col0 + j < p.cols) v[j] += sb_to_f32<T>(old[j]);
        }
        if (p.boxes) {
          if (lane == 0) bulk_wait_group_read<0>();            // the box of the chunk before has been read
          __syncwarp();
          if (p.f32) {
            const uint32_t row = box + 128u * (uint32_t)lane, key = (uint32_t)lane & 7u;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) st_shared_v4(row + ((i ^ key) << 4), make_uint4(raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]));
          } else {
            gated_to_box<T>(box, lane, v);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (p.accumulate && p.f32) tma_reduce_add_2d(&maps.out[t.which], box, col0, row0);
            else tma_store_2d(&maps.out[t.which], box, col0, row0);
            bulk_commit_group();
          }
        } else {
          gated_turn(box, lane, v);
          for (int i = 0; i < 32 && row0 + i < p.rows; ++i) {
            const float value = gated_turned(box, lane, i);
            if (col0 + lane >= p.cols) continue;
            const long long e = (long long)(row0 + i) * p.ld + col0 + lane;
            if (p.f32) reinterpret_cast<float*>(p.out)[e] = p.accumulate ? reinterpret_cast<float*>(p.out)[e] + value : value;
            else reinterpret_cast<T*>(p.out)[e] = sb_from_f32<T>(value);
          }
          __syncwarp();
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }
  // The end, as above.
  tc_fence_before_sync();
  cluster_sync_all();
  if (*abortp != 0) {
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) { }
  }
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, (uint32_t)(2 * q.bn));
  }
}

// Tiles cut into parts: their sums, in the order of the parts.  A block has 32 rows of 32 columns, read along the parts' columns and written along
// the rows.
template <typename T>
__global__ void __launch_bounds__(256) gated_join_kernel(const __grid_constant__ ProductsPlan q) {
  __shared__ float tile[32][33];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int chunks = q.bn / 32, cut0 = q.p[0].parts > 1 ? q.p[0].tiles_m * q.p[0].tiles_n - q.p[0].whole : 0;
  const long long first1 = (long long)(q.p[0].tiles_m * q.p[0].tiles_n - q.p[0].whole) * q.p[0].parts;
  const int c = (int)(blockIdx.x % chunks) * 32, sub = (int)(blockIdx.x / chunks) & 7;          // the eighths of a tile's rows, four to a CTA
  int r = (int)(blockIdx.x / chunks) >> 3;
  const int which = r < cut0 ? 0 : 1;
  if (which == 1) r -= cut0;
  const GatedProduct& p = q.p[which];
  int row0, col0;
  products_tile(p, q.bn, p.whole + r, row0, col0);
  row0 += 32 * sub;
  col0 += c;
  if (row0 >= p.rows || col0 >= p.cols) return;
  const long long part0 = (which == 1 ? first1 : 0) + (long long)r * p.parts;
  const int row = threadIdx.x % 32, first = threadIdx.x / 32 * 4;
  const float* from = q.partial + ((2 * part0 + sub / 4) * q.bn + c + first) * 128 + sub % 4 * 32 + row;
  float sum[4] = {};
#pragma unroll 8
  for (int i = 0; i < p.parts; ++i) {
    const float* part = from + (long long)i * (2 * q.bn * 128);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += __ldcs(part + 128 * j);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) tile[first + j][row] = sum[j];
  __syncthreads();
  const int lane = threadIdx.x % 32;
  if (col0 + lane >= p.cols) return;
  for (int i = threadIdx.x / 32; i < 32 && row0 + i < p.rows; i += 8) {
    const long long at = (long long)(row0 + i) * p.ld + col0 + lane;
    const float v = tile[lane][i];
    if (p.f32) {
      float* o = reinterpret_cast<float*>(p.out) + at;
      *o = p.accumulate ? *o + v : v;
    } else {
      T* o = reinterpret_cast<T*>(p.out) + at;
      *o = sb_from_f32<T>(p.accumulate ? v + sb_to_f32<T>(*o) : v);
    }
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
  if (m > (1 << 30)) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most 2^30 rows", who);
  return SB_OK;
}

template <typename T>
constexpr int gated_code() { return std::is_same<T, __half>::value ? SB_F16 : SB_BF16; }

// Tiles of `rows` x `columns`: whole ones, and behind them halves of columns for the rest.
struct GatedTiles {
  int tiles_m, tiles_f, half_first, items;
};
GatedTiles gated_tiles(long long m, long long f, int rows, int columns) {
  const int most = rows == 256 ? sb_sm_count() / 2 : sb_sm_count();
  GatedTiles t;
  t.tiles_m = (int)((m + rows - 1) / rows);
  t.tiles_f = (int)((f + columns - 1) / columns);
  const int tiles = t.tiles_m * t.tiles_f, rest = tiles % most;
  // A last wave of at most half the workers is cut into halves.
  t.half_first = rows == 256 && tiles > most && 2 * rest <= most ? tiles - rest : tiles;
  t.items = 2 * tiles - t.half_first;
  return t;
}

template <bool PAIR, typename T, int ACT>
int launch_gated_umma(const GatedArgs& p, int bf, cudaStream_t s) {
  const CUtensorMapDataType type = gated_code<T>() == SB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  GatedPlan q;
  memset(&q, 0, sizeof(q));
  const int tile_m = PAIR ? 256 : 128;
  const int most = PAIR ? sb_sm_count() / 2 : sb_sm_count();
  q.bf = bf;
  if (((long long)p.m + tile_m - 1) / tile_m * (((long long)p.f + bf - 1) / bf) > 0x3fffffff) return sb_fail(SB_ERR_TOO_LARGE, "sb_gated: too many outputs");
  const GatedTiles t = gated_tiles(p.m, p.f, tile_m, bf);
  q.tiles_m = t.tiles_m;
  q.tiles_f = t.tiles_f;
  q.half_first = t.half_first;
  q.items = t.items;
  q.k_blocks = (p.k + 63) / 64;
  q.acc_stride = bf > 64 ? 256 : 2 * bf;
  q.tmem_cols = 2 * q.acc_stride;
  q.b_bytes = (uint32_t)bf * 128u * (PAIR ? 1u : 2u);
  q.idesc = sb_umma_idesc(gated_code<T>(), 0, 0, tile_m, 2 * bf);
  q.idesc_half = sb_umma_idesc(gated_code<T>(), 0, 0, tile_m, bf);
  q.stages = (GU_SMEM - 1024 - GU_STAGING) / (int)(128 * 128 + q.b_bytes);
  if (q.stages > GU_MAX_STAGES) q.stages = GU_MAX_STAGES;
  T* saved = reinterpret_cast<T*>(p.saved);
  GatedMaps maps;
  memset(&maps, 0, sizeof(maps));
  int rc = sb_tensor_map(&maps.x, type, 2, p.x, p.m, p.k, p.ldx, 128, 64);
  if (rc == SB_OK) rc = sb_tensor_map(&maps.w, type, 2, p.w, 2LL * p.f, p.k, p.ldw, bf, 64);
  if (rc == SB_OK && q.items > q.half_first) rc = sb_tensor_map(&maps.w_half, type, 2, p.w, 2LL * p.f, p.k, p.ldw, bf / 2, 64);
  q.boxes_out = gated_rows16(p.h, p.ldh, gated_code<T>()) && (!saved || (gated_rows16(saved, p.lds, gated_code<T>()) && p.f % 8 == 0)) ? 1 : 0;
  if (q.boxes_out) {
    if (rc == SB_OK) rc = sb_tensor_map(&maps.h, type, 2, p.h, p.m, p.f, p.ldh, 32, 32);
    if (rc == SB_OK && saved) rc = sb_tensor_map(&maps.g, type, 2, saved, p.m, p.f, p.lds, 32, 32);
    if (rc == SB_OK && saved) rc = sb_tensor_map(&maps.u, type, 2, saved + p.f, p.m, p.f, p.lds, 32, 32);
  }
  static std::atomic<bool> ready[64];
  if (rc == SB_OK) rc = sb_allow_smem(gated_umma_kernel<PAIR, T, ACT>, GU_SMEM, ready);
  if (rc != SB_OK) return rc;
  const int workers = q.items < most ? q.items : most;
  const size_t smem = 1024 + (size_t)q.stages * (128 * 128 + q.b_bytes) + GU_STAGING;
  SB_CUDA(sb_launch(gated_umma_kernel<PAIR, T, ACT>, dim3((unsigned)(PAIR ? 2 * workers : workers)), dim3(GU_THREADS), smem, s, PAIR ? 2 : 1, maps, p, q));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int ACT, int NT>
int launch_gated_few(const GatedArgs& p, cudaStream_t s) {
  const dim3 grid((unsigned)((p.f + GF_ROWS - 1) / GF_ROWS), (unsigned)((p.m + 8 * NT - 1) / (8 * NT)));
  SB_CUDA(sb_launch(gated_few_kernel<T, ACT, NT>, grid, dim3(32 * GF_WARPS), 0, s, 1, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

// Rows and columns of h that a block, or a pair of them, makes where rows of x and w start on 16 bytes; up to 16 rows are for the few.
struct GatedForm {
  int rows, columns;
};
GatedForm gated_form(int m, int f, int k) {
  if (m <= 16) return {m <= 8 ? 8 : 16, GF_ROWS};
  // Pairs of CTAs on 256 rows and 128 columns of h, or CTAs on 128 rows and 128 or 64 columns: the least of waves x time of a tile, in us as
  // measured.  Pairs / 128 / 64: 16384 x 4096 x 1024 176 / 198 / 238, 16384 x 512 x 512 23.2 / 23.2 / 19.5, 512 x 4096 x 1024 12.0 / 10.6 / 11.4,
  // 256 x 4096 x 1024 11.5 / 10.0 / 9.7, 1000^3 13.3 / 14.7 / 10.7, 128 x 512 x 4096 28 / 29 / 16.
  const int sms = sb_sm_count(), blocks = (k + 63) / 64;
  const long long wide = (f + 127) / 128, tall = (m + 127) / 128, pairs = (m + 255) / 256 * wide, half = sms / 2;
  const double pair_waves = (double)(pairs / half) + (pairs % half == 0 ? 0.0 : pairs > half && 2 * (pairs % half) <= half ? 0.5 : 1.0);
  const double pair = 6.0 + pair_waves * (2.9 + 0.21 * blocks), single = 4.0 + (double)((tall * wide + sms - 1) / sms) * (2.55 + 0.28 * blocks),
               narrow = 4.0 + (double)((tall * ((f + 63) / 64) + sms - 1) / sms) * (0.15 + 0.256 * blocks);
  if (m > 128 && pair <= single && pair <= narrow) return {256, 128};
  return {128, single <= narrow ? 128 : 64};
}

template <typename T, int ACT>
int launch_gated(const GatedArgs& p, cudaStream_t s) {
  if (p.k > 0 && gated_rows16(p.x, p.m == 1 ? 8 : p.ldx, gated_code<T>()) && gated_rows16(p.w, p.ldw, gated_code<T>())) {
    const GatedForm form = gated_form(p.m, p.f, p.k);
    if (form.rows == 8) return launch_gated_few<T, ACT, 1>(p, s);
    if (form.rows == 16) return launch_gated_few<T, ACT, 2>(p, s);
    return form.rows == 256 ? launch_gated_umma<true, T, ACT>(p, form.columns, s) : launch_gated_umma<false, T, ACT>(p, form.columns, s);
  }
  const dim3 grid((unsigned)((p.m + GS_TILE - 1) / GS_TILE), (unsigned)((p.f + GS_TILE - 1) / GS_TILE));
  SB_CUDA(sb_launch(gated_simple_kernel<T, ACT>, grid, dim3(256), 0, s, 1, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int ACT, int V>
int launch_gated_act_grad(const GatedGradArgs& p, cudaStream_t s) {
  const long long blocks = ((long long)p.m * (p.f / V) + 255) / 256, most = 32LL * sb_sm_count();
  SB_CUDA(sb_launch(gated_act_grad_kernel<T, ACT, V>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, s, 1, p));
  SB_COUNT_LAUNCH();
  return SB_OK;
}
template <typename T, int ACT>
int launch_gated_act_grad(const GatedGradArgs& p, cudaStream_t s) {
  constexpr int CODE = gated_code<T>();
  const bool wide = p.f % 8 == 0 && gated_rows16(p.dh, p.lddh, CODE) && gated_rows16(p.saved, p.lds, CODE);
  return wide ? launch_gated_act_grad<T, ACT, 8>(p, s) : launch_gated_act_grad<T, ACT, 1>(p, s);
}

// What is whole and what is cut, for the products that are not empty (rows, cols and the length of K of each; 0 rows: none): the least of the modelled
// times, in us as measured (74 tiles of 2 / 8 / 64 times 128 of K: 9.7 / 14.4 / 73 with 256 columns, 8.2 / 10.9 / 66 with 128).  A tile takes 1.5 and
// per 128 of K 0.78 or 0.45; parts another 4 for the launch that joins them, and their bytes to memory and back.  Returns the parts' bytes.
struct ProductSize {
  long long rows, cols, k;
};
long long gated_products_plan(const ProductSize* size, int twice, ProductsPlan* q) {
  const long long workers = sb_sm_count() / 2;
  long long bytes = 0;
  double least = 1e30;
  for (int bn = 256; bn >= 128; bn -= 128) {
    const double block = bn == 256 ? 0.78 : 0.45;
    long long tiles[2], blocks[2];
    for (int i = 0; i < 2; ++i) {
      tiles[i] = (size[i].rows + 255) / 256 * ((size[i].cols + bn - 1) / bn);
      blocks[i] = ((size[i].k + 127) / 128) << twice;
    }
    const long long full = (tiles[0] + tiles[1]) / workers, most = blocks[0] > blocks[1] ? blocks[0] : blocks[1];
    for (int first = 0; first < 2; ++first) {     // the product whose tiles are whole first
      long long whole[2];
      whole[first] = tiles[first] < full * workers ? tiles[first] : full * workers;
      whole[1 - first] = full * workers - whole[first];
      const int slow = blocks[0] >= blocks[1] ? 0 : 1;
      const long long slow_waves = (whole[slow] + workers - 1) / workers;
      const double waves = slow_waves * (1.5 + block * blocks[slow]) + (full - slow_waves) * (1.5 + block * blocks[1 - slow]);
      for (int s = 1; s <= 128 && (s == 1 || 2 * s <= most); s += s < 32 ? 1 : 16) {
        long long parts[2], items = 0, cut = 0;
        double longest = 0.0, sum = 0.0;
        for (int i = 0; i < 2; ++i) {
          parts[i] = most > 0 ? (blocks[i] * s + most - 1) / most : 1;
          if (parts[i] < 1) parts[i] = 1;
          const long long left = tiles[i] - whole[i];
          const double t = 1.5 + block * ((blocks[i] + parts[i] - 1) / parts[i]);
          items += left * parts[i];
          sum += t * left * parts[i];
          if (parts[i] > 1) cut += left * parts[i];
          if (left > 0 && t > longest) longest = t;
        }
        const double rest = items > 0 ? sum / items * ((items + workers - 1) / workers) : 0.0;
        const double t = waves + (rest > longest ? rest : longest) + (cut > 0 ? 4.0 + 2.0e-6 * 256 * bn * cut : 0.0);
        if (t >= least) continue;
        least = t;
        bytes = cut > 0 ? items * 256 * bn * 4 : 0;            // (a rest that is whole has its places in the order)
        q->bn = bn;
        for (int i = 0; i < 2; ++i) {
          GatedProduct& p = q->p[i];
          p.tiles_m = (int)((size[i].rows + 255) / 256);
          p.tiles_n = (int)((size[i].cols + bn - 1) / bn);
          p.k_blocks = (int)blocks[i];
          p.whole = (int)whole[i];
          p.parts = (int)parts[i];
        }
        q->items = (int)(full * workers + items);
      }
    }
  }
  return bytes;
}

template <typename T, typename Out>
int launch_product_simple(const Strided& a, const Strided& b, void* c, long long ldc, long long m, long long n, long long k, int accumulate, cudaStream_t s) {
  const dim3 grid((unsigned)((m + GS_TILE - 1) / GS_TILE), (unsigned)((n + GS_TILE - 1) / GS_TILE));
  SB_CUDA(sb_launch(gated_product_simple_kernel<T, Out>, grid, dim3(256), 0, s, 1, a, b, reinterpret_cast<Out*>(c), ldc, m, n, k, accumulate));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

struct GatedGradOut {
  const void* x;
  const void* w;
  void* dx;
  void* dw;
  long long ldx, ldw, lddx, lddw;
  int dw_dtype, accumulate, k;
  float* partial;
};

// dx and dw, those that are wanted and whose operands have rows on 16 bytes, on the tensor cores.
template <typename T>
int launch_gated_products(const GatedGradArgs& g, const GatedGradOut& o, bool dx, bool dw, cudaStream_t s) {
  constexpr int CODE = gated_code<T>();
  const CUtensorMapDataType type = CODE == SB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const long long f2 = 2LL * g.f, ldx = g.m == 1 ? (o.k + 7) / 8 * 8 : o.ldx;
  const ProductSize size[2] = {{dx ? g.m : 0, o.k, f2}, {dw ? f2 : 0, o.k, g.m}};
  ProductsPlan q;
  ProductsMaps maps;
  memset(&q, 0, sizeof(q));
  memset(&maps, 0, sizeof(maps));
  if ((size[0].rows + 255) / 256 * ((o.k + 127) / 128) + (size[1].rows + 255) / 256 * ((o.k + 127) / 128) > 0x1fffffff)
    return sb_fail(SB_ERR_TOO_LARGE, "sb_gated_grad: too many outputs");
  q.twice = g.lo ? 1 : 0;
  gated_products_plan(size, q.twice, &q);
  q.partial = o.partial;
  q.b_bytes = (uint32_t)q.bn * 128u;
  q.stages = (GU_SMEM - 1024 - GP_STAGING) / (int)(GP_A_BYTES + q.b_bytes);
  int rc = SB_OK;
  for (int i = 0; i < 2; ++i) {
    GatedProduct& p = q.p[i];
    p.rows = (int)size[i].rows;
    p.cols = o.k;
    if (p.rows == 0) continue;
    p.out = i == 0 ? o.dx : o.dw;
    p.ld = i == 0 ? o.lddx : o.lddw;
    p.a_mn = i;
    p.f32 = i == 1 && o.dw_dtype == SB_F32 ? 1 : 0;
    p.accumulate = i == 1 ? o.accumulate : 0;
    p.boxes = gated_rows16(p.out, p.ld, p.f32 ? SB_F32 : CODE) ? 1 : 0;
    p.idesc = sb_umma_idesc(CODE, p.a_mn, 1, 256, q.bn);
    if (rc == SB_OK) rc = sb_tensor_map(&maps.a[i], type, 2, g.d, g.m, f2, g.ldd, 128, 64);
    if (rc == SB_OK && q.twice) rc = sb_tensor_map(&maps.a_lo[i], type, 2, g.lo, g.m, f2, g.ldd, 128, 64);
    if (rc == SB_OK) rc = i == 0 ? sb_tensor_map(&maps.b[i], type, 2, o.w, f2, o.k, o.ldw, 128, 64) : sb_tensor_map(&maps.b[i], type, 2, o.x, g.m, o.k, ldx, 128, 64);
    if (rc == SB_OK && p.boxes)
      rc = p.f32 ? sb_tensor_map(&maps.out[i], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.out, p.rows, p.cols, p.ld, 32, 32)
                 : sb_tensor_map(&maps.out[i], type, 2, p.out, p.rows, p.cols, p.ld, 32, 32);
  }
  static std::atomic<bool> ready[64];
  if (rc == SB_OK) rc = sb_allow_smem(gated_products_kernel<T>, GU_SMEM, ready);
  if (rc != SB_OK) return rc;
  const int most = sb_sm_count() / 2, workers = q.items < most ? q.items : most;
  const size_t smem = 1024 + (size_t)q.stages * (GP_A_BYTES + q.b_bytes) + GP_STAGING;
  SB_CUDA(sb_launch(gated_products_kernel<T>, dim3((unsigned)(2 * workers)), dim3(GU_THREADS), smem, s, 2, maps, q));
  SB_COUNT_LAUNCH();
  long long cut = 0;
  for (const GatedProduct& p : q.p) cut += p.parts > 1 ? p.tiles_m * p.tiles_n - p.whole : 0;
  if (cut > 0) {
    SB_CUDA(sb_launch(gated_join_kernel<T>, dim3((unsigned)(cut * 8 * (q.bn / 32))), dim3(256), 0, s, 1, q));
    SB_COUNT_LAUNCH();
  }
  return SB_OK;
}

template <typename T>
int gated_grad_products(const GatedGradArgs& g, const GatedGradOut& o, cudaStream_t s) {
  constexpr int CODE = gated_code<T>();
  const int f2 = 2 * g.f;
  if (o.k == 0) return SB_OK;
  const bool dx = o.dx && g.m > 0, dw = o.dw && f2 > 0;
  const bool fast_dx = dx && f2 > 0 && gated_rows16(o.w, o.ldw, CODE), fast_dw = dw && g.m > 0 && gated_rows16(o.x, g.m == 1 ? 8 : o.ldx, CODE);
  int rc = SB_OK;
  if (fast_dx || fast_dw) rc = launch_gated_products<T>(g, o, fast_dx, fast_dw, s);
  if (rc == SB_OK && dx && !fast_dx) rc = launch_product_simple<T, T>({g.d, g.ldd, 1, g.lo}, {o.w, 1, o.ldw, nullptr}, o.dx, o.lddx, g.m, o.k, f2, 0, s);
  if (rc != SB_OK || !dw || fast_dw) return rc;
  const Strided a = {g.d, 1, g.ldd, g.lo}, b = {o.x, 1, o.ldx, nullptr};
  return o.dw_dtype == SB_F32 ? launch_product_simple<T, float>(a, b, o.dw, o.lddw, f2, o.k, g.m, o.accumulate, s)
                              : launch_product_simple<T, T>(a, b, o.dw, o.lddw, f2, o.k, g.m, o.accumulate, s);
}

// The workspace: dg and du [m, 2 f] with rows on 16 bytes, and behind them the parts of a product.
long long gated_grad_pitch(int f) { return (2LL * f + 7) / 8 * 8; }
// Rounding dg and du to 16 bits adds as much to the error of a gradient as rounding that itself does: sqrt(2) of it in all.  With few rows, whose few
// values of dg and du need not average, it was up to twice: there what their rounding left off is kept too and multiplied beside them, at the time of
// the launches (64 rows at most: no more than one block of K more for dw, and every block of w twice, the second time from L2).  With more rows it
// takes as long again as the products themselves, and is the caller's choice: 8192 x 4096 x 1024 281 -> 518 us, 4001 x 3000 x 1000 122 -> 220, 128 x
// 4096 x 1024 25 -> 31; errors 0.0023 -> 0.0017 in bf16, 0.00029 -> 0.00021 in f16, and of an fp32 dw 0.0017 -> 0.00002.
int gated_grad_twice(int m, bool exact) { return m <= 64 || exact ? 1 : 0; }
size_t gated_grad_first(int m, int f, bool exact) { return (((size_t)m << gated_grad_twice(m, exact)) * (size_t)gated_grad_pitch(f) * 2 + 255) / 256 * 256; }

int gated_grad_bytes(const char* who, int m, int f, int k, bool exact, size_t* bytes) {
  if (!bytes) return sb_fail(SB_ERR_BAD_ARG, "%s: null output", who);
  if (m < 0 || f < 0 || k < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  long long most = 0;                             // of both products or either
  for (int want = 1; want < 4; ++want) {
    const ProductSize size[2] = {{want & 1 ? m : 0, k, 2LL * f}, {want & 2 ? 2LL * f : 0, k, m}};
    ProductsPlan q;
    const long long parts = m > 0 && f > 0 && k > 0 ? gated_products_plan(size, gated_grad_twice(m, exact), &q) : 0;
    if (parts > most) most = parts;
  }
  *bytes = gated_grad_first(m, f, exact) + (size_t)most;
  return SB_OK;
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
  if (h == x || h == w || h == saved || (saved && (saved == x || saved == w))) return sb_fail(SB_ERR_BAD_ARG, "%s: outputs in the place of an input", who);
  if (!gated_element_aligned(x, dtype) || !gated_element_aligned(w, dtype) || !gated_element_aligned(h, dtype) || !gated_element_aligned(saved, dtype))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  const GatedArgs p = {x, w, h, saved, ldx, ldw, ldh, lds, m, f, k};
  cudaStream_t s = (cudaStream_t)stream;
#define SB_GATED_CALL(ACT) (dtype == SB_BF16 ? launch_gated<__nv_bfloat16, ACT>(p, s) : launch_gated<__half, ACT>(p, s))
  return activation == SB_ACT_SILU ? SB_GATED_CALL(ACT_SILU) : activation == SB_ACT_GELU ? SB_GATED_CALL(ACT_GELU) : SB_GATED_CALL(ACT_RELU);
#undef SB_GATED_CALL
}

int sb_gated_plan(int m, int f, int k, int* plan) {
  const char* who = "sb_gated_plan";
  int rc = gated_args_ok(who, m, f, k, SB_BF16, SB_ACT_SILU);
  if (rc != SB_OK) return rc;
  if (!plan) return sb_fail(SB_ERR_BAD_ARG, "%s: null output", who);
  if (m == 0 || f == 0 || k == 0) return sb_fail(SB_ERR_BAD_ARG, "%s: sizes of nothing", who);
  const GatedForm form = gated_form(m, f, k);
  if (((long long)m + form.rows - 1) / form.rows * (((long long)f + form.columns - 1) / form.columns) > 0x3fffffff) return sb_fail(SB_ERR_TOO_LARGE, "%s: too many outputs", who);
  const GatedTiles t = gated_tiles(m, f, form.rows, form.columns);
  plan[0] = form.rows;
  plan[1] = form.columns;
  plan[2] = t.half_first;
  plan[3] = t.items - t.half_first;
  return SB_OK;
}

int sb_gated_grad_plan(int m, int f, int k, int which, int* plan) {
  const char* who = "sb_gated_grad_plan";
  int rc = gated_args_ok(who, m, f, k, SB_BF16, SB_ACT_SILU);
  if (rc != SB_OK) return rc;
  if (!plan) return sb_fail(SB_ERR_BAD_ARG, "%s: null output", who);
  if (m == 0 || f == 0 || k == 0 || which < 1 || which > 3) return sb_fail(SB_ERR_BAD_ARG, "%s: sizes of nothing, or neither product", who);
  if (((long long)m + 255) / 256 * ((k + 127) / 128) + (2LL * f + 255) / 256 * ((k + 127) / 128) > 0x1fffffff) return sb_fail(SB_ERR_TOO_LARGE, "%s: too many outputs", who);
  const ProductSize size[2] = {{which & 1 ? m : 0, k, 2LL * f}, {which & 2 ? 2LL * f : 0, k, m}};
  ProductsPlan q;
  memset(&q, 0, sizeof(q));
  gated_products_plan(size, gated_grad_twice(m, false), &q);
  plan[0] = q.bn;
  for (int i = 0; i < 2; ++i) {
    plan[1 + 3 * i] = q.p[i].whole;
    plan[2 + 3 * i] = q.p[i].tiles_m * q.p[i].tiles_n - q.p[i].whole;
    plan[3 + 3 * i] = q.p[i].parts;
  }
  return SB_OK;
}

int sb_gated_grad_workspace_bytes(int m, int f, int k, size_t* bytes) {
  return gated_grad_bytes("sb_gated_grad_workspace_bytes", m, f, k, false, bytes);
}

int sb_gated_grad_exact_workspace_bytes(int m, int f, int k, size_t* bytes) {
  return gated_grad_bytes("sb_gated_grad_exact_workspace_bytes", m, f, k, true, bytes);
}

int sb_gated_grad(const void* dh, long long lddh, const void* x, long long ldx, const void* w, long long ldw, const void* saved, long long lds,
                  void* dx, long long lddx, void* dw, long long lddw, int dw_dtype, int accumulate, int m, int f, int k, int dtype,
                  int activation, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "sb_gated_grad";
  const bool exact = (activation & SB_GATED_EXACT) != 0;
  activation &= ~SB_GATED_EXACT;
  int rc = gated_args_ok(who, m, f, k, dtype, activation);
  if (rc != SB_OK) return rc;
  if (dw && dw_dtype != dtype && dw_dtype != SB_F32) return sb_fail(SB_ERR_UNSUPPORTED, "%s: dw holds f32 or the storage type (got %d)", who, dw_dtype);
  const bool any = m > 0 && f > 0;
  if (any && (!dh || !saved || !workspace)) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (any && ((dx && k > 0 && !w) || (dw && k > 0 && !x))) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if ((any && (lddh < f || lds < 2LL * f)) || (x && ldx < k) || (w && ldw < k) || (dx && lddx < k) || (dw && lddw < k))
    return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than its rows", who);
  // Tiles of both products are written while others are still made.
  if (any && ((dx && dx == w) || (dw && dw == x))) return sb_fail(SB_ERR_BAD_ARG, "%s: dx or dw in the place of what it is made from", who);
  if (dx && dw && (dx == x || dw == w || dx == dw)) return sb_fail(SB_ERR_BAD_ARG, "%s: dx or dw in the place of what the other is made from", who);
  if (any && (workspace == dh || workspace == saved || workspace == x || workspace == w || workspace == dx || workspace == dw))
    return sb_fail(SB_ERR_BAD_ARG, "%s: the workspace in the place of an input or output", who);
  if (!gated_element_aligned(dh, dtype) || !gated_element_aligned(saved, dtype) || !gated_element_aligned(x, dtype) || !gated_element_aligned(w, dtype) ||
      !gated_element_aligned(dx, dtype) || (dw && !gated_element_aligned(dw, dw_dtype)) || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size, or the workspace not to 256 bytes", who);
  size_t need = 0;
  if ((rc = gated_grad_bytes(who, m, f, k, exact, &need)) != SB_OK) return rc;
  if (any && workspace_bytes < need) return sb_fail(SB_ERR_BAD_ARG, "%s: the workspace has %zu bytes, %zu are needed", who, workspace_bytes, need);
  if (!dx && !dw) return SB_OK;
  char* const lo = gated_grad_twice(m, exact) ? reinterpret_cast<char*>(workspace) + (size_t)m * (size_t)gated_grad_pitch(f) * 2 : nullptr;
  const GatedGradArgs g = {dh, saved, workspace, lo, lddh, lds, gated_grad_pitch(f), m, f};
  const GatedGradOut o = {x, w, dx, dw, ldx, ldw, lddx, lddw, dw_dtype, accumulate, k, reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + gated_grad_first(m, f, exact))};
  cudaStream_t s = (cudaStream_t)stream;
#define SB_GATED_CALL(ACT) (dtype == SB_BF16 ? launch_gated_act_grad<__nv_bfloat16, ACT>(g, s) : launch_gated_act_grad<__half, ACT>(g, s))
  if (any) rc = activation == SB_ACT_SILU ? SB_GATED_CALL(ACT_SILU) : activation == SB_ACT_GELU ? SB_GATED_CALL(ACT_GELU) : SB_GATED_CALL(ACT_RELU);
#undef SB_GATED_CALL
  if (rc != SB_OK) return rc;
  return dtype == SB_BF16 ? gated_grad_products<__nv_bfloat16>(g, o, s) : gated_grad_products<__half>(g, o, s);
}

}  // extern "C"
