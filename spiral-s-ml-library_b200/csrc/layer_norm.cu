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

// Rows that fit into registers.  LANES threads share a row (a part of a warp, a warp, or W warps), each with NV packs of V
// elements, R rows at a time.  In the backward pass the running column sums stay in registers over all rows of a thread.
// The arithmetic is packed, two fp32 operations per instruction: with 12 operations per element and 16 warps per SM the
// scalar form was bound by issue (65536 x 1024 bf16: 97 us forward, 107 backward; now 65 and 79, fp32 91 and 127, 6 TB/s).  What bounds
// the 16-bit types is still issue (62 % backward) and, forward, the weights' way from L1.
constexpr int LN_THREADS = 512;                              // of a block at most
struct NormShape {
  int warps;                     // per row; 1: `lanes` threads of a warp
  int lanes;                     // threads per row
  int groups;                    // of threads with rows of their own, per block
  int span;                      // packs of a warp, a multiple of 32, where warps have packs of their own
};
// Which packs of a row a thread has.  APART: warps have neighbouring packs of their own, and a thread's are 32 apart: a number
// that the compiler knows, so that all of a thread's addresses are one register and a constant (20000 x 1501 forward, single
// elements: fp32 84 -> 67 us, bf16 83 -> 60, against the row's number of threads as the distance, which took 53 instructions per
// element).  Else the row's `lanes` threads take turns.
template <int V, int NV, bool APART>
struct LnPlace {
  int first, count, apart;       // packs `first` + i * `apart`, i < `count`
  bool full;                     // all threads of the warp have NV
  __device__ __forceinline__ LnPlace(const NormShape& s, int lane, int cols) {
    const int packs = (cols + V - 1) / V;
    int end = packs, begin = 0;
    if constexpr (APART) {
      apart = 32;
      begin = (lane >> 5) * s.span;
      end = min(packs, begin + s.span);
      first = begin + (lane & 31);
    } else {
      apart = s.lanes;
      first = lane;
    }
    const int left = end - first + apart - 1;
    count = left <= 0 ? 0 : APART ? left >> 5 : left / apart;
    full = end - begin == NV * apart;
  }
  __device__ __forceinline__ int stride() const { return (APART ? 32 : apart) * V; }   // elements
};
typedef unsigned long long Pair; // two fp32 values
__device__ __forceinline__ Pair ln_pair(float v) { return pack_f32x2(v, v); }
__device__ __forceinline__ float ln_both(Pair v) {
  float lo, hi;
  unpack_f32x2(v, lo, hi);
  return lo + hi;
}

// K sums over the threads that share a row; the two buffers of `slots` take turns, so that one barrier per call is enough.
template <int K>
__device__ __forceinline__ void ln_row_sums(float (&v)[K], const NormShape& s, int group, float4* slots) {
  static_assert(K <= 4, "");
  const int from = s.warps > 1 ? 16 : s.lanes >> 1;
  for (int o = from; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  if (s.warps > 1) {
    const int warp = threadIdx.x >> 5, first = group * s.warps;
    if ((threadIdx.x & 31) == 0) slots[warp] = make_float4(v[0], K > 1 ? v[K > 1 ? 1 : 0] : 0.f, K > 2 ? v[K > 2 ? 2 : 0] : 0.f, K > 3 ? v[K > 3 ? 3 : 0] : 0.f);
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(s.warps * 32) : "memory");
    float4 t = slots[first];
    for (int w = 1; w < s.warps; ++w) {
      const float4 u = slots[first + w];
      t.x += u.x; t.y += u.y; t.z += u.z; t.w += u.w;
    }
    v[0] = t.x;
    if (K > 1) v[K > 1 ? 1 : 0] = t.y;
    if (K > 2) v[K > 2 ? 2 : 0] = t.z;
    if (K > 3) v[K > 3 ? 3 : 0] = t.w;
  }
}

// Rows on their way.  Packs of 4 bytes and more travel by cp.async, DEPTH turns of R rows ahead: every thread copies what it
// will itself read into its own places in shared memory, so nothing needs a barrier, and the rows in flight need no
// registers.  Packs of 2 bytes (16-bit rows whose pitch or base is odd), which cp.async does not take, are loaded one turn
// ahead into registers.
template <typename T, int V, int NV, int R, int MATRICES, int DEPTH>
struct LnAhead {
  static constexpr bool RING = sizeof(T) * V >= 4;
  static constexpr uint32_t PACK = sizeof(T) * V, TURN = MATRICES * R * NV;   // packs per thread and turn
  SbPack<T, V> held[RING ? 1 : TURN];
  uint32_t mine, stride;         // this thread's first place; bytes between its places
  int slot;

  static __host__ __device__ constexpr size_t bytes(int threads) { return RING ? (size_t)DEPTH * TURN * PACK * threads : 0; }
  __device__ __forceinline__ void start(uint32_t smem) {
    stride = blockDim.x * PACK;
    mine = smem + threadIdx.x * PACK;
    slot = 0;
    if constexpr (RING)                                      // places behind a row's end stay zero
      for (uint32_t k = 0; k < DEPTH * TURN; ++k)
#pragma unroll
        for (uint32_t w = 0; w < PACK; w += 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(mine + k * stride + w), "r"(0) : "memory");
  }
  // Rows `row` .. `row` + R - 1; `from` points at this thread's first element of the first.
  template <typename Place>
  __device__ __forceinline__ void fetch(int matrix, const T* from, long long row, long long ld, const NormArgs& a, const Place& place, int to) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int count = row + r < a.rows ? place.count : 0;
      const T* at = from + (row + r < a.rows ? r * ld : 0);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (matrix * R + r) * NV + i;
        if constexpr (RING) {
          const uint32_t dst = mine + (uint32_t)(to * (int)TURN + k) * stride;
          if constexpr (PACK == 16)
            asm volatile("{\n\t.reg .pred q;\n\tsetp.lt.s32 q, %2, %3;\n\t@q cp.async.cg.shared.global [%0], [%1], 16;\n\t}"
                         ::"r"(dst), "l"(at + i * place.stride()), "r"(i), "r"(count) : "memory");
          else
            asm volatile("{\n\t.reg .pred q;\n\tsetp.lt.s32 q, %2, %3;\n\t@q cp.async.ca.shared.global [%0], [%1], 4;\n\t}"
                         ::"r"(dst), "l"(at + i * place.stride()), "r"(i), "r"(count) : "memory");
        } else {
          held[k] = i < count ? sb_load_pack<T, V>(at + i * place.stride()) : sb_zero_pack<T, V>();
        }
      }
    }
  }
  __device__ __forceinline__ void read(int matrix, int r, int i, float* x) const {
    static_assert(!RING || PACK == 4 || PACK == 16, "");
    const int k = (matrix * R + r) * NV + i;
    SbPack<T, V> p;
    if constexpr (RING) {
      const uint32_t src = mine + (uint32_t)(slot * (int)TURN + k) * stride;
      if constexpr (PACK == 16) {
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
        p = *reinterpret_cast<const SbPack<T, V>*>(&v);
      } else {
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(src) : "memory");
        p = *reinterpret_cast<const SbPack<T, V>*>(&v);
      }
    } else {
      p = held[k];
    }
    sb_unpack<T, V>(p, x);
  }
  __device__ __forceinline__ void next() {
    if (++slot == DEPTH) slot = 0;
  }
};

// V weights (16-byte loads where V allows them); `other` where there are none (`have`: the row goes that far).
template <int V>
__device__ __forceinline__ void ln_weights(const float* w, int col, bool have, float other, float* to) {
  if (!w || !have) {
#pragma unroll
    for (int k = 0; k < V; ++k) to[k] = other;
  } else if constexpr (V >= 4) {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(w + col + k));
      to[k] = f.x; to[k + 1] = f.y; to[k + 2] = f.z; to[k + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) to[k] = __ldg(w + col + k);
  }
}

// NV x V values of a thread as pairs.
template <typename A, int V, int NV>
__device__ __forceinline__ void ln_read(const A& rows, int matrix, int r, Pair* x) {
  float v[NV * V];
#pragma unroll
  for (int i = 0; i < NV; ++i) rows.read(matrix, r, i, v + i * V);
#pragma unroll
  for (int j = 0; j < NV * V / 2; ++j) x[j] = pack_f32x2(v[2 * j], v[2 * j + 1]);
}
template <typename T, int V>
__device__ __forceinline__ void ln_store(T* to, const Pair* x, int i) {
  float v[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    float lo, hi;
    unpack_f32x2(x[(i * V + k) / 2], lo, hi);
    v[k] = (i * V + k) & 1 ? hi : lo;
  }
  sb_store_f32<T, V>(to, v);
}

constexpr int LN_DEPTH = 3;

// Weights are read for every row, from L1: in registers they would cost half of the warps.
template <typename T, int V, int NV, int R, bool APART>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_kernel(NormArgs a, NormShape s) {
  constexpr int E = NV * V;
  __shared__ float4 slots[2][LN_THREADS / 32];
  extern __shared__ __align__(16) uint8_t ln_smem[];
  const int group = threadIdx.x / s.lanes, lane = threadIdx.x % s.lanes;
  const LnPlace<V, NV, APART> place(s, lane, a.cols);
  const int stride = place.stride();
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const long long step = (long long)R * gridDim.x * s.groups;
  long long row = (long long)R * ((long long)blockIdx.x * s.groups + group);
  // All groups of a warp stay together: they end when the last has no row left.
  const long long last = s.warps > 1 ? row : row - (long long)R * (group % (32 / s.lanes));
  LnAhead<T, V, NV, R, 1, LN_DEPTH> rows;
  constexpr bool RING = decltype(rows)::RING;
  rows.start(smem_u32(ln_smem));
  const T* x_at = (const T*)a.x + row * a.ldx + place.first * V;
  T* y_at = (T*)a.out + row * a.ldout + place.first * V;
  constexpr int FIRST = RING ? LN_DEPTH - 1 : 1;
#pragma unroll
  for (int d = 0; d < FIRST; ++d) {
    rows.fetch(0, x_at + d * step * a.ldx, row + d * step, a.ldx, a, place, d);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (long long at = last; at < a.rows; at += step, row += step, x_at += step * a.ldx, y_at += step * a.ldout) {
    if (RING) {
      rows.fetch(0, x_at + (LN_DEPTH - 1) * step * a.ldx, row + (LN_DEPTH - 1) * step, a.ldx, a, place,
                 rows.slot == 0 ? LN_DEPTH - 1 : rows.slot - 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group %0;" ::"n"(LN_DEPTH - 1) : "memory");
    }
    Pair x[R][E / 2];
    float v[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ln_read<decltype(rows), V, NV>(rows, 0, r, x[r]);
      Pair t = x[r][0];
#pragma unroll
      for (int j = 1; j < E / 2; ++j) t = add_f32x2(t, x[r][j]);
      v[r] = ln_both(t);
    }
    if (!RING) rows.fetch(0, x_at + step * a.ldx, row + step, a.ldx, a, place, 0);
    rows.next();
    ln_row_sums<R>(v, s, group, slots[0]);
    float mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = v[r] * a.inv_cols;
      const Pair m = ln_pair(mean[r]);
      Pair t = 0ull;
#pragma unroll
      for (int j = 0; j < E / 2; ++j) x[r][j] = sub_f32x2(x[r][j], m);
      if (!place.full) {                                           // what lies behind the row's end deviates by nothing
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          float lo, hi;
          unpack_f32x2(x[r][j], lo, hi);
          if (2 * j / V >= place.count) lo = 0.f;
          if ((2 * j + 1) / V >= place.count) hi = 0.f;
          x[r][j] = pack_f32x2(lo, hi);
        }
      }
#pragma unroll
      for (int j = 0; j < E / 2; ++j) fma_f32x2(t, x[r][j], x[r][j]);
      v[r] = ln_both(t);
    }
    ln_row_sums<R>(v, s, group, slots[1]);
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rstd[r] = 1.f / sqrtf(v[r] * a.inv_cols + a.eps);
      const Pair f = ln_pair(rstd[r]);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) x[r][j] = mul_f32x2(x[r][j], f);
    }
#pragma unroll
    for (int i = 0; i < NV; i += V == 1 ? 2 : 1) {           // pairs of packs where a pack is one element
      constexpr int P = V == 1 ? 2 : 1;
      float w[P * V], b[P * V];
#pragma unroll
      for (int q = 0; q < P; ++q) {
        ln_weights<V>(a.weight, place.first * V + (i + q) * stride, i + q < place.count, 1.f, w + q * V);
        ln_weights<V>(a.bias, place.first * V + (i + q) * stride, i + q < place.count, 0.f, b + q * V);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int k = 0; k < P * V; k += 2) {
          Pair y = pack_f32x2(b[k], b[k + 1]);
          fma_f32x2(y, x[r][(i * V + k) / 2], pack_f32x2(w[k], w[k + 1]));
          x[r][(i * V + k) / 2] = y;
        }
#pragma unroll
        for (int q = 0; q < P; ++q)
          if (row + r < a.rows && i + q < place.count)
            ln_store<T, V>(y_at + r * a.ldout + (i + q) * stride, x[r], i + q);
      }
    }
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row + r < a.rows) {
          if (a.mean) a.mean[row + r] = mean[r];
          if (a.rstd) a.rstd[row + r] = rstd[r];
        }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// dx of a thread's rows whose mean times rstd is infinite, over its own packs; the sums over whole rows.
template <typename T, int V>
__device__ __forceinline__ void ln_grad_again(const NormArgs& a, long long row, long long step, int r, int col, int count, int stride) {
#pragma unroll 1
  for (; row < a.rows; row += step)
#pragma unroll 1
    for (long long at = row; at < row + r && at < a.rows; ++at) {
      const float mean = a.mean[at], rstd = a.rstd[at];
      if (fabsf(mean * rstd) != INFINITY || !(rstd < INFINITY)) continue;
      const T *x = (const T*)a.x + at * a.ldx, *dy = (const T*)a.dy + at * a.lddy;
      T* dx = (T*)a.out + at * a.ldout;
      auto g_of = [&](int j) { return sb_to_f32<T>(dy[j]) * (a.weight ? a.weight[j] : 1.f); };
      auto h_of = [&](int j) { return (sb_to_f32<T>(x[j]) - mean) * rstd; };
      float s1 = 0.f, s2 = 0.f;
#pragma unroll 1
      for (int j = 0; j < a.cols; ++j) {
        const float g = g_of(j);
        s1 += g;
        s2 = fmaf(g, h_of(j), s2);
      }
      s1 *= a.inv_cols;
      s2 *= a.inv_cols;
#pragma unroll 1
      for (int i = 0; i < count; ++i)
        for (int k = 0; k < V; ++k) {
          const int j = col + i * stride + k;
          dx[j] = sb_from_f32<T>((g_of(j) - s1 - h_of(j) * s2) * rstd);
        }
    }
}

// The backward pass: x and dy are read once for dx and the column sums together.
template <typename T, int V, int NV, int R, bool APART>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_grad_kernel(NormArgs a, NormShape s) {
  constexpr int E = NV * V;
  __shared__ float4 slots[2][LN_THREADS / 32];
  __shared__ float stats[LN_DEPTH][LN_THREADS / 4][2 * R];   // mean and rstd of the rows on their way, per warp or group
  extern __shared__ __align__(16) uint8_t ln_smem[];
  float* columns = reinterpret_cast<float*>(ln_smem);        // [2][cols], where several groups of a block add up at the end
  const int group = threadIdx.x / s.lanes, lane = threadIdx.x % s.lanes;
  const int unit = s.warps > 1 ? threadIdx.x >> 5 : group, member = s.warps > 1 ? threadIdx.x & 31 : lane;
  const LnPlace<V, NV, APART> place(s, lane, a.cols);
  const int stride = place.stride();
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const long long step = (long long)R * gridDim.x * s.groups;
  long long row = (long long)R * ((long long)blockIdx.x * s.groups + group);
  const long long last = s.warps > 1 ? row : row - (long long)R * (group % (32 / s.lanes));
  LnAhead<T, V, NV, R, 2, LN_DEPTH> rows;
  constexpr bool RING = decltype(rows)::RING;
  rows.start(smem_u32(ln_smem));
  const T* x_at = (const T*)a.x + row * a.ldx + place.first * V;
  const T* dy_at = (const T*)a.dy + row * a.lddy + place.first * V;
  T* dx_at = (T*)a.out + row * a.ldout + place.first * V;
  auto fetch = [&](int turns, int to) {
    const long long at = row + turns * step;
    rows.fetch(0, x_at + turns * step * a.ldx, at, a.ldx, a, place, RING ? to : 0);
    rows.fetch(1, dy_at + turns * step * a.lddy, at, a.lddy, a, place, RING ? to : 0);
    if (member < 2 * R) {
      const bool in = at + member % R < a.rows;
      const float* from = (member < R ? a.mean : a.rstd) + (in ? at + member % R : 0);
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(&stats[to][unit][member])), "l"(from), "r"(in ? 4u : 0u) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int FIRST = RING ? LN_DEPTH - 1 : 1;
#pragma unroll
  for (int d = 0; d < FIRST; ++d) fetch(d, d);
  Pair w[E / 2], dw[E / 2], db[E / 2];
  {
    float f[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) ln_weights<V>(a.weight, place.first * V + i * stride, i < place.count, 1.f, f + i * V);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      w[j] = pack_f32x2(f[2 * j], f[2 * j + 1]);
      dw[j] = db[j] = 0ull;
    }
  }
  int turn = 0;
  // A place behind a row's end deviates by -mean, and where that times rstd is infinite (constant rows of very large values) its zero of
  // a gradient makes a NaN of the row's sum.  Packs of 16 bytes and short rows: such places are masked for such a row.  Others: such rows are
  // noted and done once more at the end, each thread its own values.  (Masks there: 20000 x 1501 bf16 74.5 -> 78.1 us.  Once more here: 65536 x
  // 1024 bf16 78.3 -> 83.9, 200000 x 62 27.7 -> 29.7.)
  constexpr bool MASKS = sizeof(T) * V == 16 || !APART;
  float beyond = 0.f;
  for (long long at = last; at < a.rows; at += step, turn ^= 1) {
    if (RING) {
      fetch(LN_DEPTH - 1, rows.slot == 0 ? LN_DEPTH - 1 : rows.slot - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(LN_DEPTH - 1) : "memory");
    } else {
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __syncwarp();                                            // the statistics were copied by other lanes
    Pair h[R][E / 2], g[R][E / 2];
    float v[2 * R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mean = *(volatile float*)&stats[rows.slot][unit][r];
      rstd[r] = *(volatile float*)&stats[rows.slot][unit][R + r];
      const Pair m = ln_pair(mean), f = ln_pair(rstd[r]);
      if (row + r < a.rows) {                                // else the places hold an earlier row
        ln_read<decltype(rows), V, NV>(rows, 0, r, h[r]);
        ln_read<decltype(rows), V, NV>(rows, 1, r, g[r]);
      } else {
#pragma unroll
        for (int j = 0; j < E / 2; ++j) h[r][j] = g[r][j] = 0ull;
      }
      if constexpr (!MASKS) {
        beyond = fmaxf(beyond, fabsf(mean * rstd[r]));
      } else if (!place.full && !(fabsf(mean * rstd[r]) < INFINITY)) {
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          float lo, hi;
          unpack_f32x2(h[r][j], lo, hi);
          if (2 * j / V >= place.count) lo = mean;
          if ((2 * j + 1) / V >= place.count) hi = mean;
          h[r][j] = pack_f32x2(lo, hi);
        }
      }
      Pair s1 = 0ull, s2 = 0ull;
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        h[r][j] = mul_f32x2(sub_f32x2(h[r][j], m), f);
        fma_f32x2(dw[j], g[r][j], h[r][j]);
        db[j] = add_f32x2(db[j], g[r][j]);
        g[r][j] = mul_f32x2(g[r][j], w[j]);
        s1 = add_f32x2(s1, g[r][j]);
        fma_f32x2(s2, g[r][j], h[r][j]);
      }
      v[2 * r] = ln_both(s1);
      v[2 * r + 1] = ln_both(s2);
    }
    __syncwarp();                                            // the statistics have been read
    rows.next();
    if (!RING) fetch(1, rows.slot);
    if (a.out) {
      ln_row_sums<2 * R>(v, s, group, slots[turn]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Pair s1 = ln_pair(-v[2 * r] * a.inv_cols), s2 = ln_pair(-v[2 * r + 1] * a.inv_cols), f = ln_pair(rstd[r]);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          Pair t = add_f32x2(g[r][j], s1);
          fma_f32x2(t, h[r][j], s2);
          g[r][j] = mul_f32x2(t, f);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (row + r < a.rows && i < place.count) ln_store<T, V>(dx_at + r * a.ldout + i * stride, g[r], i);
      }
    }
    row += step;
    x_at += step * a.ldx;
    dy_at += step * a.lddy;
    dx_at += step * a.ldout;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!MASKS && beyond == INFINITY && a.out && a.cols != E * s.lanes)
    ln_grad_again<T, V>(a, (long long)R * ((long long)blockIdx.x * s.groups + group), step, R, place.first * V, place.count, stride);
  if (!a.partial) return;
  float sums[2][E];
#pragma unroll
  for (int j = 0; j < E / 2; ++j) {
    unpack_f32x2(dw[j], sums[0][2 * j], sums[0][2 * j + 1]);
    unpack_f32x2(db[j], sums[1][2 * j], sums[1][2 * j + 1]);
  }
  float* part = a.partial + (long long)blockIdx.x * 2 * a.cols;
  if (s.groups == 1) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int col = place.first * V + j / V * stride + j % V;
      if (j / V < place.count) {
        part[col] = sums[0][j];
        part[a.cols + col] = sums[1][j];
      }
    }
    return;
  }
  // Groups of one warp add up by shuffles, then the block's in their order through shared memory.
  for (int o = 16; o >= s.lanes; o >>= 1)
#pragma unroll
    for (int j = 0; j < E; ++j) {
      sums[0][j] += __shfl_xor_sync(0xffffffffu, sums[0][j], o);
      sums[1][j] += __shfl_xor_sync(0xffffffffu, sums[1][j], o);
    }
  const bool mine = s.warps > 1 || (threadIdx.x & 31) < s.lanes;
  const int turns = s.warps > 1 ? s.groups : blockDim.x / 32, my_turn = s.warps > 1 ? group : threadIdx.x >> 5;
  __syncthreads();                                           // every group's rows have been read
  for (int t = 0; t < turns; ++t) {
    if (t == my_turn && mine) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int col = place.first * V + j / V * stride + j % V;
        if (j / V < place.count) {
          columns[col] = (t ? columns[col] : 0.f) + sums[0][j];
          columns[a.cols + col] = (t ? columns[a.cols + col] : 0.f) + sums[1][j];
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * a.cols; i += blockDim.x) part[i] = columns[i];
}

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

// Any row length and alignment: a block per row, the row read three times (the second and third time from L2), element by element.
// Rows that no register form takes: past 8192 columns (16384 of 16 bits in 16-byte packs), backward past 4096 in fp32 and 8192 in 16 bits
// (or 8192 single elements).  4096 x 16384 forward fp32 249 us (floor 82), backward fp32 446 and bf16 434 (123 and 62); 8192 x 8192 fp32
// backward 411, where rows of 4096 take 144 for twice as many.
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

// Blocks with partial column sums, at most.
constexpr int LN_BLOCKS_PER_SM = 8;
constexpr int LN_SMEM = 200 * 1024;
int ln_columns_blocks(long long rows) {
  const long long most = LN_BLOCKS_PER_SM * (long long)sb_sm_count();
  return (int)(rows < 1 ? 1 : rows < most ? rows : most);
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

// How many threads share a row, for packs of v elements and nv of them per thread (whole warps where these have packs of their
// own); false: the row does not fit.
bool norm_shape(int cols, int v, int nv, bool apart, NormShape* s) {
  const int packs = (cols + v - 1) / v, most = LN_THREADS * nv;
  if (packs > most) return false;
  s->warps = (packs + 32 * nv - 1) / (32 * nv);
  s->lanes = 32 * s->warps;
  if (s->warps == 1 && !apart) {
    s->lanes = 4;
    while (s->lanes * nv < packs) s->lanes *= 2;
  }
  s->groups = s->lanes < 256 ? 256 / s->lanes : 1;
  s->span = ((packs + s->warps - 1) / s->warps + 31) / 32 * 32;
  return true;
}

// Blocks of KERNEL that are resident on the device at a time (at most LN_BLOCKS_PER_SM per SM), asked once per device and
// block size; the kernel may use `smem` bytes of shared memory.
template <auto KERNEL>
cudaError_t norm_resident(int threads, size_t smem, int* blocks) {
  static std::atomic<int> known[64][LN_THREADS / 32 + 1];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool keep = dev >= 0 && dev < 64;
  int per_sm = keep ? known[dev][threads / 32].load(std::memory_order_acquire) : 0;
  if (per_sm == 0) {
    if ((e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, LN_SMEM)) != cudaSuccess) return e;
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, KERNEL, threads, smem)) != cudaSuccess) return e;
    per_sm = per_sm < 1 ? 1 : per_sm > LN_BLOCKS_PER_SM ? LN_BLOCKS_PER_SM : per_sm;
    if (keep) known[dev][threads / 32].store(per_sm, std::memory_order_release);
  }
  *blocks = per_sm * sb_sm_count();
  return cudaSuccess;
}

// The groups of a block, and the blocks: as many threads as fit at a time.  Numbers of threads per row that do not divide 256
// may do better in blocks of up to 512 (96 threads per row at 128 registers: one block of five rows, two of two).
template <auto KERNEL, typename Smem>
cudaError_t norm_groups(NormShape* s, const Smem& smem, int* blocks) {
  cudaError_t e = norm_resident<KERNEL>(s->lanes * s->groups, smem(*s), blocks);
  if (e != cudaSuccess || 256 % s->lanes == 0 || LN_THREADS / s->lanes <= s->groups) return e;
  NormShape other = *s;
  other.groups = LN_THREADS / s->lanes;
  int more = 0;
  if ((e = norm_resident<KERNEL>(other.lanes * other.groups, smem(other), &more)) != cudaSuccess) return e;
  if (more * other.groups > *blocks * s->groups) {
    *s = other;
    *blocks = more;
  }
  return e;
}

int norm_grid(const NormArgs& a, const NormShape& s, int r, int most) {
  const long long at_once = (long long)r * s.groups, want = (a.rows + at_once - 1) / at_once;
  return (int)(want < most ? want : most);
}

template <typename T, int V, int NV, int R, bool APART>
bool try_norm(const NormArgs& a, cudaStream_t s, cudaError_t* e) {
  NormShape shape;
  if (!norm_shape(a.cols, V, NV, APART, &shape)) return false;
  const auto smem = [](const NormShape& s) { return LnAhead<T, V, NV, R, 1, LN_DEPTH>::bytes(s.lanes * s.groups); };
  int blocks = 0;
  if ((*e = norm_groups<layer_norm_kernel<T, V, NV, R, APART>>(&shape, smem, &blocks)) == cudaSuccess)
    *e = sb_launch(layer_norm_kernel<T, V, NV, R, APART>, dim3(norm_grid(a, shape, R, blocks)), dim3(shape.lanes * shape.groups), smem(shape), s,
                   1, a, shape);
  return true;
}

// Pack width of rows and weights: 16 bytes, 4 bytes, or one element.
int norm_width(int v, int item, const NormArgs& a) {
  if (v * item == 16 && (reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.bias)) % 16 == 0) return v;
  return v * item >= 4 ? 4 / item : 1;
}

template <typename T>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(T), WORD = 4 / sizeof(T);
  int v = sb_vector_width(a.x, a.ldx, a.cols, sizeof(T), MOST);
  v = norm_width(sb_vector_width(a.out, a.ldout, a.cols, sizeof(T), v), sizeof(T), a);
  cudaError_t e = cudaSuccess;
  if (v == MOST) {
    // Two rows share a load of their weights: 16384 x 4096 bf16 72 us, 79 with twice the columns of one row.
    if (a.cols <= 32 * MOST && try_norm<T, MOST, 1, 2, false>(a, s, &e)) return e;
    if (try_norm<T, MOST, 2, 2, true>(a, s, &e)) return e;
    if (try_norm<T, MOST, 4, 1, true>(a, s, &e)) return e;
  } else if (v == WORD && WORD > 1) {
    if (a.cols <= 128 * WORD && try_norm<T, WORD, 4, 2, false>(a, s, &e)) return e;
    if (try_norm<T, WORD, 8, 2, true>(a, s, &e)) return e;
    if (try_norm<T, WORD, 16, 1, true>(a, s, &e)) return e;
  } else {
    if (a.cols <= 128 && try_norm<T, 1, 4, 2, false>(a, s, &e)) return e;
    if (try_norm<T, 1, 8, 2, true>(a, s, &e)) return e;
    if (try_norm<T, 1, 16, 1, true>(a, s, &e)) return e;
  }
  const int threads = a.cols >= 1024 ? 1024 : (a.cols + 31) / 32 * 32;
  const long long most = 16LL * sb_sm_count();
  return sb_launch(layer_norm_wide_kernel<T>, dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(threads), 0, s, 1, a);
}

// Writes the partial sums' number to *parts where the row fits into registers.
template <typename T, int V, int NV, int R, bool APART>
bool try_norm_grad(const NormArgs& a, cudaStream_t s, cudaError_t* e, int* parts) {
  NormShape shape;
  if (!norm_shape(a.cols, V, NV, APART, &shape)) return false;
  const auto smem = [&a](const NormShape& s) {
    const size_t ahead = LnAhead<T, V, NV, R, 2, LN_DEPTH>::bytes(s.lanes * s.groups);
    const size_t sums = s.groups > 1 ? 2 * sizeof(float) * (size_t)a.cols : 0;     // at most 32 KB: two groups share 512 threads
    return ahead > sums ? ahead : sums;
  };
  int blocks = 0;
  if ((*e = norm_groups<layer_norm_grad_kernel<T, V, NV, R, APART>>(&shape, smem, &blocks)) != cudaSuccess) return true;
  *parts = norm_grid(a, shape, R, blocks);
  *e = sb_launch(layer_norm_grad_kernel<T, V, NV, R, APART>, dim3(*parts), dim3(shape.lanes * shape.groups), smem(shape), s, 1, a, shape);
  return true;
}

template <typename T>
cudaError_t launch_norm_grad(const NormArgs& a, cudaStream_t s, int* parts) {
  constexpr int MOST = 16 / sizeof(T), WORD = 4 / sizeof(T);
  int v = sb_vector_width(a.x, a.ldx, a.cols, sizeof(T), MOST);
  v = sb_vector_width(a.dy, a.lddy, a.cols, sizeof(T), v);
  if (a.out) v = sb_vector_width(a.out, a.ldout, a.cols, sizeof(T), v);
  v = norm_width(v, sizeof(T), a);
  cudaError_t e = cudaSuccess;
  // Short rows two at a time (65536 x 1024 fp32 147 -> 127 us, bf16 82 -> 80, against one pack per thread and more warps per row).
  if (v == MOST) {
    if (a.cols <= 64 * MOST && try_norm_grad<T, MOST, 1, 2, false>(a, s, &e, parts)) return e;
    if (try_norm_grad<T, MOST, 2, 1, true>(a, s, &e, parts)) return e;
  } else if (v == WORD && WORD > 1) {
    if (a.cols <= 128 * WORD && try_norm_grad<T, WORD, 4, 1, false>(a, s, &e, parts)) return e;
    // Two rows at a time here as well (20000 x 1502 bf16 66 -> 54 us, 65536 x 1002 126 -> 105); of 128 packs and fewer one (200000 x 62
    // 27.7, with two 29.1), and of single elements too (65536 x 1001 bf16 130, with two 138).
    if (try_norm_grad<T, WORD, 4, 2, true>(a, s, &e, parts)) return e;
    if (try_norm_grad<T, WORD, 8, 1, true>(a, s, &e, parts)) return e;
  } else {
    if (a.cols <= 256 && try_norm_grad<T, 1, 8, 1, false>(a, s, &e, parts)) return e;
    if (try_norm_grad<T, 1, 8, 1, true>(a, s, &e, parts)) return e;
    // Sixteen single 16-bit elements spill 168 bytes at 128 registers; more warps per row do not fit.
    if (try_norm_grad<T, 1, 16, 1, true>(a, s, &e, parts)) return e;
  }
  *parts = 0;
  if (!a.out) return cudaSuccess;
  const int threads = a.cols >= 1024 ? 1024 : (a.cols + 31) / 32 * 32;
  const long long most = 16LL * sb_sm_count();
  e = sb_launch(layer_norm_grad_wide_kernel<T>, dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(threads), 0, s, 1, a);
  SB_COUNT_LAUNCH();
  return e;
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
  if (!columns) a.partial = nullptr;
  int parts = 0;
  cudaError_t e = dtype == SB_F32 ? launch_norm_grad<float>(a, s, &parts)
                                  : dtype == SB_BF16 ? launch_norm_grad<__nv_bfloat16>(a, s, &parts) : launch_norm_grad<__half>(a, s, &parts);
  SB_CUDA(e);
  if (parts > 0) SB_COUNT_LAUNCH();
  if (columns) {
    if (parts == 0) {
      parts = ln_columns_blocks(rows);
      const dim3 grid((cols + 255) / 256, parts);
      e = dtype == SB_F32 ? sb_launch(layer_norm_columns_kernel<float>, grid, dim3(256), 0, s, 1, a)
          : dtype == SB_BF16 ? sb_launch(layer_norm_columns_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, 1, a)
                             : sb_launch(layer_norm_columns_kernel<__half>, grid, dim3(256), 0, s, 1, a);
      SB_COUNT_LAUNCH();
      SB_CUDA(e);
    }
    e = sb_launch(layer_norm_partials_kernel, dim3((cols + 31) / 32, 2), dim3(1024), 0, s, 1, (const float*)workspace, parts, cols,
                  dweight, dbias, accumulate);
    SB_COUNT_LAUNCH();
    SB_CUDA(e);
  }
  return SB_OK;
}

}  // extern "C"
