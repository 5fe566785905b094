// Log probabilities of given tokens under row distributions, their entropy and likeliest alternatives, and the gradient: what
// a policy gradient needs of a policy head, or a token loss of a large vocabulary.
//
// With s the scale (one over the temperature), x a row's legal logits, M their largest and S = sum exp(s (x_j - M)):
//   log p_j = s (x_j - M) - log S        H = log S - s sum exp(s (x_j - M)) (x_j - M) / S
//   d x_j = s (a ([j = t] - p_j) - h p_j (log p_j + H))      for the gradients a of log p_t and h of H.
#include "common.cuh"
#include "vector_io.cuh"

#include <type_traits>

namespace {

constexpr int LP_MAX_TOP = 64;
constexpr float LP_LOG2E = 1.4426950408889634f;

struct LogProbArgs {
  const void* logits;
  long long ld, rows;
  int cols;                      // legal columns end here (the prefix), <= mask_cols
  int mask_cols;
  const uint8_t* mask;
  float scale;
  const void* tokens;
  int wide_tokens;               // 64-bit tokens
  float* out;
  float* entropy;
  float* stats;
  int top;
  float* top_values;
  int32_t* top_tokens;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float LP_LOWEST = -3.402823466e38f;
// What a distance from the largest logit counts as at least where it is multiplied by its own probability: 0, not NaN, for -inf.
constexpr float LP_FAR = -1e30f;

__device__ __forceinline__ long long lp_token(const void* tokens, int wide, long long row) {
  return wide ? reinterpret_cast<const long long*>(tokens)[row] : (long long)reinterpret_cast<const int*>(tokens)[row];
}

// Largest logit so far (NaN left out: it shows in the sum), sum = S and dist = sum exp(s (x - top)) (x - top).  Of nothing: the lowest
// number, which no -inf reaches, and zeros.
struct RowSums {
  float top, sum, dist;
};
// The same, seen from `top`, which is not below its own.
__device__ __forceinline__ void lp_raise(RowSums& r, float top, float c) {
  const float d = fmaxf(r.top - top, LP_FAR), f = exp2_approx(d * c);
  r.dist = fmaf(r.sum, d, r.dist) * f;
  r.sum *= f;
  r.top = top;
}
// In N values, whose largest is not above r.top.
template <int N>
__device__ __forceinline__ void lp_take(RowSums& r, const float* x, float c) {
  if constexpr (N % 2 == 0) {
    const unsigned long long top2 = pack_f32x2(r.top, r.top), c2 = pack_f32x2(c, c);
    unsigned long long sum2 = 0ull, dist2 = 0ull;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      float d0, d1, a0, a1;
      unpack_f32x2(sub_f32x2(pack_f32x2(x[i], x[i + 1]), top2), d0, d1);
      const unsigned long long d2 = pack_f32x2(max_nan(d0, LP_FAR), max_nan(d1, LP_FAR));
      unpack_f32x2(mul_f32x2(d2, c2), a0, a1);
      const unsigned long long e2 = pack_f32x2(exp2_approx(a0), exp2_approx(a1));
      sum2 = add_f32x2(sum2, e2);
      fma_f32x2(dist2, e2, d2);
    }
    float s0, s1, d0, d1;
    unpack_f32x2(sum2, s0, s1);
    unpack_f32x2(dist2, d0, d1);
    r.sum += s0 + s1;
    r.dist += d0 + d1;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = max_nan(x[i] - r.top, LP_FAR), e = exp2_approx(d * c);
      r.sum += e;
      r.dist = fmaf(e, d, r.dist);
    }
  }
}

// What a row's sums give: the logarithm of S and the entropy; a row of nothing has the sum 0.
__device__ __forceinline__ void lp_finish(const LogProbArgs& g, long long row, const RowSums& r, float log_sum, float token_logit, long long token) {
  const bool empty = r.sum == 0.f;
  if (g.out)
    g.out[row] = token < 0 || token >= g.mask_cols ? 0.f : token >= g.cols || empty ? -INFINITY : g.scale * (token_logit - r.top) - log_sum;
  if (g.entropy) g.entropy[row] = empty ? 0.f : log_sum - g.scale * (r.dist / r.sum);
  if (g.stats) {
    g.stats[2 * row] = empty ? 0.f : r.top;
    g.stats[2 * row + 1] = log_sum;
  }
}
__device__ __forceinline__ void lp_alternative(const LogProbArgs& g, long long row, int place, float x, int column, float top, float log_sum) {
  const bool none = column < 0;
  if (g.top_values) g.top_values[row * g.top + place] = none ? -INFINITY : g.scale * (x - top) - log_sum;
  if (g.top_tokens) g.top_tokens[row * g.top + place] = none ? -1 : column;
}

// A logit by itself; -inf where the mask forbids it.
template <typename T>
__device__ __forceinline__ float lp_logit(const T* x, const uint8_t* mask, int j) {
  const float v = sb_to_f32<T>(x[j]);
  return mask && mask[j] == 0 ? -INFINITY : v;
}

// Rows of up to G E columns: G lanes per row, E columns each, in registers.  Alternatives by rounds: every lane offers its best.
template <typename T, int G, int E>
__global__ void __launch_bounds__(128) log_probs_short_kernel(LogProbArgs g) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x % G;
  const float c = g.scale * LP_LOG2E;
  const long long groups = (long long)gridDim.x * (128 / G);
  // Whole warps go round together.
  const long long first = (long long)blockIdx.x * (128 / G) + threadIdx.x / G, warp_first = first - (threadIdx.x % 32) / G;
  for (long long at = 0; warp_first + at < g.rows; at += groups) {
    const long long row = first + at;
    const bool there = row < g.rows;
    const T* logits = reinterpret_cast<const T*>(g.logits) + (there ? row : 0) * g.ld;
    const uint8_t* mask = g.mask ? g.mask + (there ? row : 0) * g.mask_cols : nullptr;
    const long long token = there && g.out ? lp_token(g.tokens, g.wide_tokens, row) : -1;
    float x[E];
    RowSums r = {LP_LOWEST, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = lane + G * e;
      x[e] = there && j < g.cols ? sb_to_f32<T>(logits[j]) : -INFINITY;
    }
    if (mask) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int j = lane + G * e;
        if (there && j < g.cols && mask[j] == 0) x[e] = -INFINITY;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) r.top = fmaxf(r.top, x[e]);
#pragma unroll
    for (int o = G / 2; o; o >>= 1) r.top = fmaxf(r.top, __shfl_xor_sync(0xffffffffu, r.top, o));
    lp_take<E>(r, x, c);
#pragma unroll
    for (int o = G / 2; o; o >>= 1) {
      r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
      r.dist += __shfl_xor_sync(0xffffffffu, r.dist, o);
    }
    const float log_sum = r.sum == 0.f ? INFINITY : logf(r.sum);
    if (there && lane == 0) {
      const bool legal = token >= 0 && token < g.cols;
      lp_finish(g, row, r, log_sum, legal ? lp_logit<T>(logits, mask, (int)token) : 0.f, token);
    }
    if (g.top > 0) {
      float best = -INFINITY;
      int column = 0x7fffffff;
      auto offer = [&]() {
        best = -INFINITY;
        column = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (x[e] > best) {
            best = x[e];
            column = lane + G * e;
          }
      };
      offer();
      for (int i = 0; i < g.top; ++i) {
        float v = best;
        int j = column;
#pragma unroll
        for (int o = G / 2; o; o >>= 1) {
          const float w = __shfl_xor_sync(0xffffffffu, v, o);
          const int k = __shfl_xor_sync(0xffffffffu, j, o);
          if (w > v || (w == v && k < j)) {
            v = w;
            j = k;
          }
        }
        if (there && lane == i % G) lp_alternative(g, row, i, v, j == 0x7fffffff ? -1 : j, r.top, log_sum);
        if (j == column && j != 0x7fffffff) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (lane + G * e == j) x[e] = -INFINITY;
          offer();
        }
      }
    }
  }
}

// A row's place in memory: single elements up to the first 16-byte boundary, packs of 16 bytes, single elements behind them.
template <typename T>
struct RowShape {
  static constexpr int V = 16 / sizeof(T);
  int head, packs, tail;
  __device__ __forceinline__ RowShape(const T* x, int cols) {
    head = (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (int)sizeof(T);
    head = head < cols ? head : cols;
    packs = (cols - head) / V;
    tail = cols - head - packs * V;
  }
  __device__ __forceinline__ int column(int pack) const { return head + pack * V; }
  // The i-th of the head + tail single elements.
  __device__ __forceinline__ int single(int i) const { return i < head ? i : packs * V + i; }
};

template <typename T>
__device__ __forceinline__ float lp_largest(const SbWords<16>& w);
template <>
__device__ __forceinline__ float lp_largest<float>(const SbWords<16>& w) {
  return fmaxf(fmaxf(__uint_as_float(w.v.x), __uint_as_float(w.v.y)), fmaxf(__uint_as_float(w.v.z), __uint_as_float(w.v.w)));
}
template <>
__device__ __forceinline__ float lp_largest<__nv_bfloat16>(const SbWords<16>& w) {
  __nv_bfloat162 v[4];
  memcpy(v, &w, 16);
  const float2 m = __bfloat1622float2(__hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
  return fmaxf(m.x, m.y);
}
template <>
__device__ __forceinline__ float lp_largest<__half>(const SbWords<16>& w) {
  __half2 v[4];
  memcpy(v, &w, 16);
  const float2 m = __half22float2(__hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
  return fmaxf(m.x, m.y);
}

template <typename T>
__device__ __forceinline__ void lp_mask_pack(float* x, const uint8_t* mask) {
#pragma unroll
  for (int i = 0; i < RowShape<T>::V; ++i)
    if (mask[i] == 0) x[i] = -INFINITY;
}

// An order of floats as unsigned numbers.
__device__ __forceinline__ uint32_t lp_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// An order of alternatives: by their logits (zeros of both signs are equal), the lower column first.
__device__ __forceinline__ unsigned long long lp_place(float x, int column) {
  return (unsigned long long)lp_key(x + 0.f) << 32 | (uint32_t)~column;
}
__device__ __forceinline__ float lp_place_logit(unsigned long long place) {
  const uint32_t key = (uint32_t)(place >> 32);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ int lp_place_column(unsigned long long place) { return (int)~(uint32_t)place; }

constexpr int LP_CANDIDATES = 512;
// The `top` best of n candidates in their order: each counts those before it. 
__device__ __forceinline__ void lp_rank(unsigned long long* candidates, int n, unsigned long long* best, int top, int threads) {
  for (int i = threadIdx.x; i < n; i += threads) {
    const unsigned long long mine = candidates[i];
    int before = 0, k = 0;
    for (; k + 8 <= n; k += 8) {
#pragma unroll
      for (int u = 0; u < 8; u += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(candidates + k + u);
        before += (two.x > mine ? 1 : 0) + (two.y > mine ? 1 : 0);
      }
    }
    for (; k < n; ++k) before += candidates[k] > mine ? 1 : 0;
    if (before < top) best[before] = mine;
  }
}

// Longer rows: a block per row, or a cluster of blocks that share one, in one pass over memory.  Each thread keeps its own
// sums and raises their reference when a batch of packs brings a larger logit.
//
// Alternatives: the top-th largest of the threads' own largest logits is a bound that `top` logits at least reach and few others do.  Only
// the threads that reach it hold alternatives; the block reads their share of the row once more, from L2, and ranks what reaches
// the bound.  Rows with more of those than there is room for (long runs of equal logits) find them one after the other.
template <typename T, int NT, bool MASKED, bool CLUSTER>
__global__ void __launch_bounds__(NT) log_probs_long_kernel(LogProbArgs g) {
  constexpr int V = RowShape<T>::V, WARPS = NT / 32, UNROLL = 4;
  __shared__ RowSums part[WARPS];
  __shared__ RowSums whole;                      // of this block's share
  __shared__ float largest[NT];
  __shared__ int hot[NT];
  __shared__ __align__(16) unsigned long long candidates[LP_CANDIDATES];
  __shared__ unsigned long long best[LP_MAX_TOP];      // 0: none
  __shared__ int hot_count, candidate_count;
  __shared__ float bound;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blocks = CLUSTER ? (int)gridDim.x : 1, rank = CLUSTER ? (int)blockIdx.x : 0;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const float c = g.scale * LP_LOG2E;
  for (long long row = blockIdx.y; row < g.rows; row += gridDim.y) {
    const T* x = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const uint8_t* mask = MASKED ? g.mask + row * g.mask_cols : nullptr;
    const RowShape<T> shape(x, g.cols);
    const int stride = NT * blocks, first = rank * NT + tid;
    const int singles = shape.head + shape.tail;               // fewer than 2 V: the first threads of the first block have one each
    RowSums r = {LP_LOWEST, 0.f, 0.f};
    if (first < singles) {
      const float v = lp_logit<T>(x, mask, shape.single(first));
      r.top = fmaxf(r.top, v);
      lp_take<1>(r, &v, c);
    }
    for (int p0 = first; p0 < shape.packs; p0 += UNROLL * stride) {
      SbWords<16> w[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        // Packs that are not there hold -inf.
        w[u].v = sizeof(T) == 4 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u)
                 : std::is_same<T, __half>::value ? make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u)
                                                  : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
        sb_load_words(w[u], x + shape.column(p0 + u * stride < shape.packs ? p0 + u * stride : 0), p0 + u * stride < shape.packs);
      }
      float top = r.top;
      if constexpr (!MASKED) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) top = fmaxf(top, lp_largest<T>(w[u]));
        lp_raise(r, top, c);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          float v[V];
          sb_unpack_words<T, V>(w[u], v);
          lp_take<V>(r, v, c);
        }
      } else {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          float v[V];
          sb_unpack_words<T, V>(w[u], v);
          if (p0 + u * stride < shape.packs) lp_mask_pack<T>(v, mask + shape.column(p0 + u * stride));
          float most = r.top;
#pragma unroll
          for (int i = 0; i < V; ++i) most = fmaxf(most, v[i]);
          lp_raise(r, most, c);
          lp_take<V>(r, v, c);
        }
      }
    }
    const float mine = r.top;
    float top = r.top;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    lp_raise(r, top, c);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
      r.dist += __shfl_xor_sync(0xffffffffu, r.dist, o);
    }
    __syncthreads();                             // what the row before left has been read
    if (lane == 0) part[warp] = r;
    if (g.top > 0) largest[tid] = mine;
    if (tid == 0) hot_count = candidate_count = 0;
    __syncthreads();
    if (warp == 0) {
      RowSums all = lane < WARPS ? part[lane] : RowSums{LP_LOWEST, 0.f, 0.f};
      float most = all.top;
#pragma unroll
      for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      lp_raise(all, most, c);
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        all.sum += __shfl_xor_sync(0xffffffffu, all.sum, o);
        all.dist += __shfl_xor_sync(0xffffffffu, all.dist, o);
      }
      if (lane == 0) whole = all;
    }
    if (g.top > 0) {
      if (warp == WARPS - 1) {
        // Bit by bit the largest key that `top` of the threads reach; near it is near enough.
        uint32_t keys[NT / 32], low = 0xffffffffu, high = 0u;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) {
          keys[i] = lp_key(largest[lane + 32 * i]);
          low = min(low, keys[i]);
          high = max(high, keys[i]);
        }
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        const int alike = __clz((int)(low ^ high));    // leading bits that all keys share: 32 where they are equal
        uint32_t key = alike == 32 ? low : low & ~(0xffffffffu >> alike);
        for (int bit = 31 - alike; bit >= 0; --bit) {
          const uint32_t tried = key | 1u << bit;
          int reach = 0;
#pragma unroll
          for (int i = 0; i < NT / 32; ++i) reach += keys[i] >= tried ? 1 : 0;
          reach = (int)__reduce_add_sync(0xffffffffu, (unsigned)reach);
          if (reach >= g.top) {
            key = tried;
            if (reach <= g.top + 4) break;
          }
        }
        // The key as a number; below the lowest number's (fewer threads than alternatives have a logit) everything counts.
        const float b = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
        if (lane == 0) bound = key <= lp_key(LP_LOWEST) ? LP_LOWEST : b;
      }
      __syncthreads();
      const float least = bound;
      if (mine >= least) hot[atomicAdd(&hot_count, 1)] = tid;
      __syncthreads();
      // A thread's share: its packs, then its single element.
      const int each = (shape.packs + stride - 1) / stride + 1, items = hot_count * each;
      for (int item = tid; item < items; item += NT) {
        const int who = hot[item / each], k = item % each;
        const int pack = rank * NT + who + k * stride;
        auto candidate = [&](float v, int j) {
          if (v >= least && v > -INFINITY) {
            const int at = atomicAdd(&candidate_count, 1);
            if (at < LP_CANDIDATES) candidates[at] = lp_place(v, j);
          }
        };
        if (k == each - 1) {
          if (rank * NT + who < singles) {
            const int j = shape.single(rank * NT + who);
            candidate(lp_logit<T>(x, mask, j), j);
          }
        } else if (pack < shape.packs) {
          SbWords<16> w;
          sb_load_words(w, x + shape.column(pack), true);
          if (MASKED || lp_largest<T>(w) >= least) {
            float v[V];
            sb_unpack_words<T, V>(w, v);
            if (MASKED) lp_mask_pack<T>(v, mask + shape.column(pack));
#pragma unroll
            for (int i = 0; i < V; ++i) candidate(v[i], shape.column(pack) + i);
          }
        }
      }
      if (tid < LP_MAX_TOP) best[tid] = 0ull;
      __syncthreads();
      const int n = candidate_count;
      if (n <= LP_CANDIDATES) {
        lp_rank(candidates, n, best, g.top, NT);
        __syncthreads();
      } else {
        unsigned long long last = ~0ull;
        for (int i = 0; i < g.top; ++i) {
          unsigned long long next = 0ull;
          auto look = [&](float v, int j) {
            const unsigned long long place = lp_place(v, j);
            if (v > -INFINITY && place < last && place > next) next = place;
          };
          if (first < singles) look(lp_logit<T>(x, mask, shape.single(first)), shape.single(first));
          for (int p = first; p < shape.packs; p += stride) {
            SbWords<16> w;
            sb_load_words(w, x + shape.column(p), true);
            float v[V];
            sb_unpack_words<T, V>(w, v);
            if (MASKED) lp_mask_pack<T>(v, mask + shape.column(p));
#pragma unroll
            for (int e = 0; e < V; ++e) look(v[e], shape.column(p) + e);
          }
#pragma unroll
          for (int o = 16; o; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, next, o);
            next = other > next ? other : next;
          }
          __syncthreads();
          if (lane == 0) candidates[warp] = next;
          __syncthreads();
          for (int w = 0; w < WARPS; ++w) next = candidates[w] > next ? candidates[w] : next;
          if (tid == 0) best[i] = next;
          last = next;
        }
        __syncthreads();
      }
    } else {
      __syncthreads();
    }
    RowSums all = whole;
    if constexpr (CLUSTER) {
      // The first block joins the others' sums and alternatives, in their order.
      cluster_sync_all();
      if (rank == 0) {
        if (tid == 0) candidate_count = 0;
        __syncthreads();
        RowSums parts[8];
        float most = LP_LOWEST;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          parts[b] = {LP_LOWEST, 0.f, 0.f};
          if (b < blocks) {
            const uint32_t at = map_to_cta(smem_u32(&whole), (uint32_t)b);
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(parts[b].top) : "r"(at) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(parts[b].sum) : "r"(at + 4u) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(parts[b].dist) : "r"(at + 8u) : "memory");
          }
          most = fmaxf(most, parts[b].top);
        }
        all = {most, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          lp_raise(parts[b], most, c);
          all.sum += parts[b].sum;
          all.dist += parts[b].dist;
        }
        for (int i = tid; i < blocks * g.top; i += NT) {
          unsigned long long place;
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(place) : "r"(map_to_cta(smem_u32(&best[i % g.top]), (uint32_t)(i / g.top))) : "memory");
          if (place != 0ull) candidates[atomicAdd(&candidate_count, 1)] = place;
        }
        __syncwarp();
      }
      cluster_arrive_relaxed_all();              // what was read has been used: the others may go on
      cluster_wait_all();
      if (rank == 0 && g.top > 0) {
        const int n = candidate_count;
        if (tid < LP_MAX_TOP) best[tid] = 0ull;
        __syncthreads();
        lp_rank(candidates, n, best, g.top, NT);
        __syncthreads();
      }
    }
    if (rank == 0) {
      const float log_sum = all.sum == 0.f ? INFINITY : logf(all.sum);
      if (tid == 0) {
        const long long token = g.out ? lp_token(g.tokens, g.wide_tokens, row) : -1;
        lp_finish(g, row, all, log_sum, token >= 0 && token < g.cols ? lp_logit<T>(x, mask, (int)token) : 0.f, token);
      }
      if (tid < g.top) lp_alternative(g, row, tid, lp_place_logit(best[tid]), best[tid] == 0ull ? -1 : lp_place_column(best[tid]), all.top, log_sum);
    }
  }
}

struct LogProbGradArgs {
  const void* logits;
  void* dlogits;
  long long ld, ldd, rows;
  int cols, mask_cols;
  const uint8_t* mask;
  float scale;
  const void* tokens;
  int wide_tokens;
  const float* stats;
  const float* dout;
  const float* entropy;
  const float* dentropy;
};

// What a row's gradient is made of: p_j = exp(s (x_j - top) - log_sum), d_j = -s p_j (c + h log p_j), and `a` more at the token.
struct RowGrad {
  float scale, top, log_sum, c, h, a;
  int token;
};
__device__ __forceinline__ RowGrad lp_row_grad(const LogProbGradArgs& g, long long row) {
  RowGrad r;
  r.scale = g.scale;
  r.top = g.stats[2 * row];
  r.log_sum = g.stats[2 * row + 1];
  const long long t = g.dout ? lp_token(g.tokens, g.wide_tokens, row) : -1;
  const float a = t >= 0 && t < g.mask_cols ? g.dout[row] : 0.f;
  r.h = g.dentropy ? g.dentropy[row] : 0.f;
  r.c = g.dentropy ? fmaf(r.h, g.entropy[row], a) : a;
  r.a = g.scale * a;
  r.token = t >= 0 && t < g.cols && r.log_sum != INFINITY ? (int)t : -1;
  return r;
}
// Logarithms of probabilities at least this far from 1, whose probabilities are 0 in fp32.
constexpr float LP_NOTHING = -1e4f;
__device__ __forceinline__ float lp_grad(const RowGrad& r, float x) {
  const float lp = max_nan(fmaf(r.scale, x - r.top, -r.log_sum), LP_NOTHING);
  return exp2_approx(lp * LP_LOG2E) * fmaf(r.h, lp, r.c) * -r.scale;
}
// A pack of logits whose place the gradient may take: not by the path for data that stays as it is.
__device__ __forceinline__ void lp_load_once(SbWords<16>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t@q ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "+r"(w.v.x), "+r"(w.v.y), "+r"(w.v.z), "+r"(w.v.w) : "l"(from), "r"((uint32_t)issue) : "memory");
}
// Of a single column.
template <typename T>
__device__ __forceinline__ void lp_grad_one(const RowGrad& r, const T* x, const uint8_t* mask, T* d, int j, int cols) {
  float v = 0.f;
  if (j < cols && !(mask && mask[j] == 0)) {
    v = lp_grad(r, sb_to_f32<T>(x[j]));
    if (j == r.token) v += r.a;
  }
  d[j] = sb_from_f32<T>(v);
}

// Short rows: G lanes per row.
template <typename T, int G>
__global__ void __launch_bounds__(256) log_probs_grad_short_kernel(LogProbGradArgs g) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x % G;
  const long long groups = (long long)gridDim.x * (256 / G);
  for (long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; row < g.rows; row += groups) {
    const RowGrad r = lp_row_grad(g, row);
    const T* x = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const uint8_t* mask = g.mask ? g.mask + row * g.mask_cols : nullptr;
    T* d = reinterpret_cast<T*>(g.dlogits) + row * g.ldd;
    for (int j = lane; j < g.mask_cols; j += G) lp_grad_one<T>(r, x, mask, d, j, g.cols);
  }
}

// Long rows: packs of 16 bytes, several on their way; the blocks of a column of the grid share the rows.
template <typename T, bool MASKED>
__global__ void __launch_bounds__(256) log_probs_grad_long_kernel(LogProbGradArgs g) {
  constexpr int V = RowShape<T>::V, UNROLL = 4;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int first = blockIdx.x * 256 + threadIdx.x, stride = gridDim.x * 256;
  for (long long row = blockIdx.y; row < g.rows; row += gridDim.y) {
    const RowGrad r = lp_row_grad(g, row);
    const T* x = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const uint8_t* mask = MASKED ? g.mask + row * g.mask_cols : nullptr;
    T* d = reinterpret_cast<T*>(g.dlogits) + row * g.ldd;
    const RowShape<T> shape(x, g.cols);
    const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15u) == 0;
    if (first < shape.head + shape.tail) lp_grad_one<T>(r, x, mask, d, shape.single(first), g.cols);
    for (int j = g.cols + first; j < g.mask_cols; j += stride) d[j] = sb_from_f32<T>(0.f);
    for (int p0 = first; p0 < shape.packs; p0 += UNROLL * stride) {
      SbWords<16> w[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        w[u].v = make_uint4(0u, 0u, 0u, 0u);
        const bool there = p0 + u * stride < shape.packs;
        lp_load_once(w[u], x + shape.column(there ? p0 + u * stride : 0), there);
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (p0 + u * stride >= shape.packs) break;
        const int j = shape.column(p0 + u * stride);
        float v[V];
        sb_unpack_words<T, V>(w[u], v);
        const unsigned long long top2 = pack_f32x2(r.top, r.top), scale2 = pack_f32x2(r.scale, r.scale), sum2 = pack_f32x2(-r.log_sum, -r.log_sum),
                                 log2 = pack_f32x2(LP_LOG2E, LP_LOG2E), h2 = pack_f32x2(r.h, r.h), c2 = pack_f32x2(r.c, r.c),
                                 minus2 = pack_f32x2(-r.scale, -r.scale);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          unsigned long long lp2 = sum2;
          fma_f32x2(lp2, scale2, sub_f32x2(pack_f32x2(v[i], v[i + 1]), top2));
          float l0, l1;
          unpack_f32x2(lp2, l0, l1);
          lp2 = pack_f32x2(max_nan(l0, LP_NOTHING), max_nan(l1, LP_NOTHING));
          unpack_f32x2(mul_f32x2(lp2, log2), l0, l1);
          unsigned long long q2 = c2;
          fma_f32x2(q2, h2, lp2);
          q2 = mul_f32x2(mul_f32x2(pack_f32x2(exp2_approx(l0), exp2_approx(l1)), q2), minus2);
          unpack_f32x2(q2, v[i], v[i + 1]);
        }
        if ((unsigned)(r.token - j) < (unsigned)V) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (j + i == r.token) v[i] += r.a;
        }
        if (MASKED) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (mask[j + i] == 0) v[i] = 0.f;
        }
        if (alike) {
          sb_store_f32<T, V>(d + j, v);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) d[j + i] = sb_from_f32<T>(v[i]);
        }
      }
    }
  }
}

int lp_args_ok(const char* who, const void* logits, long long ld, int dtype, long long rows, int cols, const uint8_t* mask, int prefix, float scale,
               const void* tokens, int index_dtype) {
  (void)mask;
  if (rows < 0 || cols < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (prefix > cols) return sb_fail(SB_ERR_BAD_ARG, "%s: prefix %d beyond the %d columns", who, prefix, cols);
  if (dtype != SB_F32 && dtype != SB_BF16 && dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: logits are f32, bf16 or f16 (got %d)", who, dtype);
  if (tokens && index_dtype != SB_I32 && index_dtype != SB_I64)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: tokens are int32 or int64 (got %d)", who, index_dtype);
  if (!(scale > 0.f) || scale > 3.402823466e38f) return sb_fail(SB_ERR_BAD_ARG, "%s: the scale must be positive and finite", who);
  if (rows == 0) return SB_OK;
  if (cols > 0 && !logits) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ld < cols) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch of %lld is shorter than the %d columns", who, ld, cols);
  if (rows > (1LL << 40)) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most 2^40 rows", who);
  if (reinterpret_cast<uintptr_t>(logits) % (size_t)sb_dtype_size(dtype) != 0 ||
      (tokens && reinterpret_cast<uintptr_t>(tokens) % (index_dtype == SB_I64 ? 8u : 4u) != 0))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  return SB_OK;
}

bool lp_words(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

template <typename T, int G, int E>
int launch_log_probs_short(const LogProbArgs& g, cudaStream_t s) {
  const long long blocks = (g.rows + 128 / G - 1) / (128 / G), most = 64LL * sb_sm_count();
  SB_CUDA(sb_launch(log_probs_short_kernel<T, G, E>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(128), 0, s, 1, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int NT, bool CLUSTER>
int launch_log_probs_long(const LogProbArgs& g, int blocks, cudaStream_t s) {
  const dim3 grid((unsigned)blocks, (unsigned)(g.rows < 65535 ? g.rows : 65535));
  if (g.mask) SB_CUDA(sb_launch(log_probs_long_kernel<T, NT, true, CLUSTER>, grid, dim3(NT), 0, s, blocks, g));
  else SB_CUDA(sb_launch(log_probs_long_kernel<T, NT, false, CLUSTER>, grid, dim3(NT), 0, s, blocks, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T>
int launch_log_probs(const LogProbArgs& g, cudaStream_t s) {
  if (g.cols <= 16) return launch_log_probs_short<T, 4, 4>(g, s);
  if (g.cols <= 64) return launch_log_probs_short<T, 8, 8>(g, s);
  if (g.cols <= 256) return launch_log_probs_short<T, 32, 8>(g, s);
  if (g.cols <= 1024) return launch_log_probs_short<T, 32, 32>(g, s);
  int blocks = 1;
  while (blocks < 8 && g.rows * blocks * 2 <= 2LL * sb_sm_count() && g.cols / (2 * blocks) >= 4096) blocks *= 2;
  if (blocks > 1) return launch_log_probs_long<T, 512, true>(g, blocks, s);
  if (g.cols <= 4096) return launch_log_probs_long<T, 128, false>(g, 1, s);
  return launch_log_probs_long<T, 256, false>(g, 1, s);
}

template <typename T>
int launch_log_probs_grad(const LogProbGradArgs& g, cudaStream_t s) {
  if (g.mask_cols <= 256) {
    const int lanes = g.mask_cols <= 16 ? 4 : g.mask_cols <= 64 ? 8 : 32;
    const long long blocks = (g.rows * lanes + 255) / 256, most = 32LL * sb_sm_count();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (lanes == 4) SB_CUDA(sb_launch(log_probs_grad_short_kernel<T, 4>, grid, dim3(256), 0, s, 1, g));
    else if (lanes == 8) SB_CUDA(sb_launch(log_probs_grad_short_kernel<T, 8>, grid, dim3(256), 0, s, 1, g));
    else SB_CUDA(sb_launch(log_probs_grad_short_kernel<T, 32>, grid, dim3(256), 0, s, 1, g));
    SB_COUNT_LAUNCH();
    return SB_OK;
  }
  // Enough blocks for the chip where rows are few, each with a batch of packs per thread at least.
  const int batch = 256 * 4 * (16 / (int)sizeof(T));
  long long across = (8LL * sb_sm_count() + g.rows - 1) / g.rows;
  if (across > (g.mask_cols + batch - 1) / batch) across = (g.mask_cols + batch - 1) / batch;
  const dim3 grid((unsigned)across, (unsigned)(g.rows < 65535 ? g.rows : 65535));
  if (g.mask) SB_CUDA(sb_launch(log_probs_grad_long_kernel<T, true>, grid, dim3(256), 0, s, 1, g));
  else SB_CUDA(sb_launch(log_probs_grad_long_kernel<T, false>, grid, dim3(256), 0, s, 1, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

}  // namespace

extern "C" {

int sb_log_probs(const void* logits, long long ld, int dtype, long long rows, int cols, const uint8_t* mask, int prefix, float scale,
                 const void* tokens, int index_dtype, float* out, float* entropy, float* stats, int top, float* top_values,
                 int32_t* top_tokens, void* stream) {
  const char* who = "sb_log_probs";
  int rc = lp_args_ok(who, logits, ld, dtype, rows, cols, mask, prefix, scale, tokens, index_dtype);
  if (rc != SB_OK) return rc;
  if (top < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (top > LP_MAX_TOP) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most %d alternatives (got %d)", who, LP_MAX_TOP, top);
  if (rows == 0) return SB_OK;
  if (out && !tokens) return sb_fail(SB_ERR_BAD_ARG, "%s: log probabilities of no tokens", who);
  if (top > 0 && !top_values && !top_tokens) return sb_fail(SB_ERR_BAD_ARG, "%s: nowhere to put %d alternatives", who, top);
  if (!lp_words(out) || !lp_words(entropy) || !lp_words(stats) || !lp_words(top_values) || !lp_words(top_tokens))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  LogProbArgs g;
  memset(&g, 0, sizeof(g));
  g.logits = logits; g.ld = ld; g.rows = rows; g.cols = prefix >= 0 ? prefix : cols; g.mask_cols = cols;
  g.mask = prefix >= 0 ? nullptr : mask; g.scale = scale; g.tokens = tokens; g.wide_tokens = index_dtype == SB_I64; g.out = out; g.entropy = entropy; g.stats = stats;
  g.top = top; g.top_values = top_values; g.top_tokens = top_tokens;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_F32 ? launch_log_probs<float>(g, s)
         : dtype == SB_BF16 ? launch_log_probs<__nv_bfloat16>(g, s) : launch_log_probs<__half>(g, s);
}

int sb_log_probs_grad(const void* logits, long long ld, int dtype, long long rows, int cols, const uint8_t* mask, int prefix, float scale,
                      const void* tokens, int index_dtype, const float* stats, const float* dout, const float* entropy,
                      const float* dentropy, void* dlogits, long long ldd, void* stream) {
  const char* who = "sb_log_probs_grad";
  int rc = lp_args_ok(who, logits, ld, dtype, rows, cols, mask, prefix, scale, tokens, index_dtype);
  if (rc != SB_OK) return rc;
  if (rows == 0 || cols == 0) return SB_OK;
  if (!dlogits || !stats) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (dout && !tokens) return sb_fail(SB_ERR_BAD_ARG, "%s: a gradient of the log probabilities of no tokens", who);
  if (dentropy && !entropy) return sb_fail(SB_ERR_BAD_ARG, "%s: a gradient of the entropy needs the entropy", who);
  if (ldd < cols) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch of %lld is shorter than the %d columns", who, ldd, cols);
  if (reinterpret_cast<uintptr_t>(dlogits) % (size_t)sb_dtype_size(dtype) != 0 || !lp_words(stats) || !lp_words(dout) || !lp_words(entropy) ||
      !lp_words(dentropy))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  LogProbGradArgs g;
  memset(&g, 0, sizeof(g));
  g.logits = logits; g.ld = ld; g.rows = rows; g.cols = prefix >= 0 ? prefix : cols; g.mask_cols = cols;
  g.mask = prefix >= 0 ? nullptr : mask; g.scale = scale; g.tokens = tokens; g.wide_tokens = index_dtype == SB_I64; g.stats = stats; g.dout = dout; g.entropy = entropy;
  g.dentropy = dentropy; g.dlogits = dlogits; g.ldd = ldd;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_F32 ? launch_log_probs_grad<float>(g, s)
         : dtype == SB_BF16 ? launch_log_probs_grad<__nv_bfloat16>(g, s) : launch_log_probs_grad<__half>(g, s);
}

}  // extern "C"
